"""Corners of the losses of a linear vocabulary head (cacophony_amd.losses, csrc/linear_loss.hip): what is not finite, weights that lie
far apart, confident rows.  Inputs, 64-bit forms and tolerances are those of tests/test_linear_loss.py unless a test derives its own."""
import math

import pytest
import torch

from tests.test_linear_loss import U32, close, dev, expect, loss_of, make, sim, sim_call, targets, with_grad  # noqa: F401


def on_simulator(x, T=1.0, reduction="mean", row_weight=None, **kw):
    return sim_call(x, T, reduction={"none": 0, "mean": 1, "sum": 2}[reduction], row_weight=row_weight, **kw)


def on_gpu(x, T=1.0, reduction="mean", row_weight=None):
    return with_grad(dev(x), T, reduction=reduction, row_weight=None if row_weight is None else row_weight.cuda())._asdict()


# where a case runs: the kernels' sources on the simulator, and the GPU
WHERE = [pytest.param(on_simulator, id="simulator"), pytest.param(on_gpu, id="gpu", marks=pytest.mark.gpu)]


@pytest.fixture
def call(request):
    if request.param is on_simulator:
        request.getfixturevalue("sim")
    return request.param


# ------------------------------------------------------------------------------------------------------------------------------------
# the distillation's d bias: the targets' share
# ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("call", WHERE, indirect=True)
@pytest.mark.parametrize("weight", [1.0 - 2.0 ** -24, 1.0, 2.0 ** 100 * (1 - 2.0 ** -24), 2.0 ** -100])
def test_d_bias_of_entries_of_one_token(call, weight):
    """128 entries that add up to one token's weight: their sum is 1 or a few roundings off it, on either side, in every row."""
    x = make(24, 300, 64, topk=128, seed=70, ignored=0.0)
    x["idx"][:] = torch.arange(24)[:, None] * 5
    wt = torch.full((24,), weight)
    close(call(x, reduction="sum", row_weight=wt), expect(x, reduction="sum", row_weight=wt), f"weight {weight}")


@pytest.mark.parametrize("call", WHERE, indirect=True)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_d_bias_shows_a_teacher_that_is_not_finite(call, bad):
    """One such logit makes the row's softmax NaN, so every gradient that one of the row's entries is part of, and no other."""
    x = make(40, 300, 64, topk=6, seed=71, ignored=0.0)
    x["idx"] = torch.arange(240).reshape(40, 6)
    x["teacher"][7, 2] = bad
    o = call(x, reduction="sum")
    d_bias = o["d_bias"].cpu()
    assert torch.isnan(d_bias[42:48]).all() and torch.isnan(o["d_weight"].cpu()[42:48]).all() and torch.isnan(o["loss"]).all()
    others = torch.cat([torch.arange(42), torch.arange(48, 300)])
    y = dict(x, teacher=torch.where(torch.arange(40)[:, None] == 7, torch.zeros(()), x["teacher"]))      # any finite ones: the other words do not see them
    want, tol = expect(y, reduction="sum")["d_bias"]
    assert ((d_bias.double() - want).abs() <= tol)[others].all()


@pytest.mark.parametrize("call", WHERE, indirect=True)
def test_d_bias_with_weights_that_lie_far_apart(call):
    """Row r has weight +-2^(4 r - 60) and entries of its own, on words whose bias of -200 leaves no row a probability worth mentioning there: the words'
    gradients are -g q, up to 2^156 apart, and each is as exact as if its row were alone."""
    x = make(40, 300, 64, topk=3, seed=72, ignored=0.0)
    x["idx"] = 100 + torch.arange(120).reshape(40, 3)
    x["b"][100:220] = -200.0
    wt = torch.tensor([2.0 ** (4 * r - 60) for r in range(40)]) * torch.where(torch.arange(40) % 3 == 0, -1.0, 1.0)
    o, want = call(x, reduction="sum", row_weight=wt), expect(x, reduction="sum", row_weight=wt)
    val, tol = want["d_bias"]
    q, _ = targets(x, 1.0)
    alone = (wt.double()[:, None] * q).sum(0)
    assert ((val + alone).abs()[100:220] < 1e-6 * alone.abs()[100:220]).all() and (tol[100:220] < 1e-3 * alone.abs()[100:220]).all()
    close(o, want, "weights 2^-60 .. 2^96")
    # the same word in the heaviest and in the lightest row: the sum is as exact as fp32 sums are
    x["idx"][:, 0] = 100
    close(call(x, reduction="sum", row_weight=wt), expect(x, reduction="sum", row_weight=wt), "one word of all rows")


# ------------------------------------------------------------------------------------------------------------------------------------
# confident rows: what is left of 1 - p does not depend on what all logits have in common
# ------------------------------------------------------------------------------------------------------------------------------------
def confident(offset, topk=0, rows=48, vocab=300, dim=64):
    """Rows whose label's logit is about 14 above the others', so that 1 - p is near 1e-5; bias = offset for every word.  Distillation: a teacher
    that is certain of the same word."""
    x = make(rows, vocab, dim, topk=topk, seed=73, ignored=0.0, spread=0.5)
    y = torch.arange(rows) * 3
    w = x["w"].float()
    scale = 20.0 / (w[y] ** 2).sum(1, keepdim=True)
    x["h"] = (0.3 * x["h"].float() + scale * w[y]).bfloat16()
    x["b"] = torch.full((vocab,), float(offset))
    if topk:
        x["idx"] = (y[:, None] + torch.arange(topk)) % vocab
        x["teacher"] = torch.where(torch.arange(topk) == 0, 12.0, -2.0) - torch.linspace(0, 1, topk)[None, :].repeat(rows, 1)
    else:
        x["y"] = y
    return x


def expect_confident(x, row_weight=None):
    """The gradients of the summed loss and what they may be off by when a row's statistics and its probabilities come from the same logits.

    Errors dz of the logits (at most (D + 1) u32 S, S = |h| . |w| + |b|) move p_v by p_v |dz_v - sum_u p_u dz_u|, that is by p_v (1 - p_v) 2 max dz, and
    the loss, sum_k q_k (lse - z_k), by sum_v |p_v - q_v| max dz.  What the logits have in common is only in that.  Exponents are within 2^-22 of
    the difference that they round where it is below 8 (which is where p matters) and within u32 of it elsewhere; the sum of the exponentials is 300 terms in
    at most 24 additions one after the other; exp2, log2 and products are good to 8 u32:  p off by 40 u32 (1 + |log p| / 16) p, the loss by
    40 u32 (1 + sum_k q_k (|log q_k| + |log p_k|)).  q: as in `expect`, 64 u32 (|t| + 8).  Then one rounding to bf16 each, and for the distillation's d bias
    sums of p and of q apart: 64 u32 (p + q)."""
    h, w, b = x["h"].double(), x["w"].double(), x["b"].double()
    R, V, D = h.shape[0], w.shape[0], h.shape[1]
    q, _ = targets(x, 1.0)
    z = h @ w.T + b
    dmax = ((D + 1) * U32 * (h.abs() @ w.abs().T + b.abs())).amax(1, keepdim=True)
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    own = 64 * U32 * (x["teacher"].double().abs().amax(1, keepdim=True) + 8) if x["topk"] else torch.zeros(R, 1, dtype=torch.float64)
    loss = (torch.special.xlogy(q, q) - q * lp).sum(1)
    out = {"row_loss": (loss, ((p - q).abs().sum(1, keepdim=True) * dmax).squeeze(1)
                        + (own * q * (1 - q) * (1 + torch.where(q > 0, torch.log(q.clamp_min(1e-300)) - lp, 0.0).abs())).sum(1)
                        + 40 * U32 * (1 + (torch.special.xlogy(q, q).abs() - q * lp).sum(1)))}
    dL = p - q
    # a word that is certain is off by own * (1 - q), as a probability is
    raw = p * (1 - p) * 2 * dmax * 1.01 + 40 * U32 * (1 + lp.abs() / 16) * p + own * q * (1 - q) + 4 * U32 * q
    dLt = raw + 2.0 ** -8 * (dL.abs() + raw)
    for name, val, tol in (("d_hidden", dL @ w, dLt @ w.abs() + (V + 64) * U32 * (dL.abs() @ w.abs())),
                           ("d_weight", dL.T @ h, dLt.T @ h.abs() + (R + 64) * U32 * (dL.abs().T @ h.abs()))):
        out[name] = (val, tol * (1 + 2.0 ** -8) + 2.0 ** -8 * val.abs() + 1e-38)
    both = 64 * U32 * (p + q).sum(0) if x["topk"] else 0.0
    out["d_bias"] = (dL.sum(0), raw.sum(0) + (R + 64) * U32 * dL.abs().sum(0) + both + 1e-38)
    return out


OFFSETS = [0.0, 60.0, 200.0, 3000.0, -3000.0]


@pytest.mark.parametrize("call", WHERE, indirect=True)
@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("topk", [0, 5])
def test_confident_rows_with_a_common_offset(call, topk, offset):
    x = confident(offset, topk)
    close(call(x, reduction="sum"), expect_confident(x), f"offset {offset}")


def apart_on_simulator(x, T=1.0, reduction="mean", row_weight=None, pair=4):
    """Forward and backward pass as two calls with a workspace each; the backward pass has lse only."""
    from tests import simlib
    lib, P = simlib.load(), simlib.ptr
    R, D, V, K = x["h"].shape[0], x["h"].shape[1], x["w"].shape[0], x["topk"]
    f = lambda *s: torch.full(s, float("nan"))
    o = dict(row_loss=f(R), lse=f(2, R) if pair else f(R), loss=f(1), d_hidden=f(R, D).bfloat16(), d_weight=f(V, D).bfloat16(), d_bias=f(V))
    red = {"none": 0, "mean": 1, "sum": 2}[reduction]
    for what in (1, 2):
        need = lib.caco_linear_loss_workspace(R, V, D, K, 1 << 30, what | pair)
        ws = torch.full((need,), 0xFF, dtype=torch.uint8)
        first = (what | pair, P(x["h"]), D, P(x["w"]), D, P(x["b"]))
        fwd = what == 1
        last = (R, V, D, red, P(row_weight), None, P(o["row_loss"]) if fwd else None, P(o["lse"]), P(o["loss"]) if fwd and red else None, P(o["d_hidden"]), D,
                P(o["d_weight"]), D, P(o["d_bias"]), P(ws), need, None)
        if K:
            rc = lib.caco_linear_distill(*first, P(x["teacher"]), K, P(x["idx"]), K, x["idx"].element_size(), K, T, *last)
        else:
            rc = lib.caco_linear_ce(*first, P(x["y"]), -100, *last)
        simlib.check(rc, "linear loss")
    if pair:
        o["lse"] = o["lse"].double().sum(0)
    if not red:
        del o["loss"]
    return o


def autograd_on_gpu(x, T=1.0, reduction="mean", row_weight=None):
    d = dev(x)
    for k in ("h", "w", "b"):
        d[k].requires_grad_(True)
    loss_of(d, T, reduction=reduction).backward()
    return {"d_hidden": d["h"].grad, "d_weight": d["w"].grad, "d_bias": d["b"].grad}


@pytest.mark.parametrize("offset", [200.0, 3000.0])
@pytest.mark.parametrize("topk", [0, 5])
@pytest.mark.parametrize("call", [pytest.param(apart_on_simulator, id="simulator"), pytest.param(autograd_on_gpu, id="gpu", marks=pytest.mark.gpu)])
def test_confident_rows_with_a_backward_pass_of_its_own(request, call, topk, offset):
    if call is apart_on_simulator:
        request.getfixturevalue("sim")
    x = confident(offset, topk)
    close(call(x, reduction="sum"), expect_confident(x), f"offset {offset}")


@pytest.mark.parametrize("topk", [0, 7])
def test_simulator_two_calls(sim, topk):
    """With the pair and with the single number; rows that do not count, all of them too."""
    x = make(90, 700, 72, topk=topk, seed=74)
    for pair in (4, 0):
        close(apart_on_simulator(x, 2.0 if topk else 1.0, pair=pair), expect(x, 2.0 if topk else 1.0), f"pair {pair}")
    o = apart_on_simulator(make(5, 300, 64, topk=topk, ignored=1.0, seed=5))
    assert not o["lse"].any() and not o["d_weight"].any() and not o["d_bias"].any() and not o["d_hidden"].any()


@pytest.mark.parametrize("call", WHERE, indirect=True)
@pytest.mark.parametrize("rows,vocab,dim", [(70, 300, 72), (20, 2100, 328), (300, 700, 264)])
def test_one_entry_is_the_cross_entropy(call, rows, vocab, dim):
    """A teacher with one entry at T = 1 is a label: the entry's logit has the bits that the label's has in the tiles (whatever the large part that all
    logits share), so the losses are equal bit for bit."""
    x = make(rows, vocab, dim, seed=75)
    x["b"] += 500.0
    y = dict(x, topk=1, idx=x["y"][:, None].clone(), teacher=torch.randn(rows, 1))
    a, b = call(x), call(y)
    assert torch.equal(a["row_loss"], b["row_loss"]) and a["row_loss"].cpu().count_nonzero() == (x["y"] >= 0).sum()
    close({k: v for k, v in b.items() if k != "lse"}, expect(y), "gradients")


@pytest.mark.parametrize("call", WHERE, indirect=True)
@pytest.mark.parametrize("slope", [0.05, 0.5, -0.5])
def test_logits_that_climb_from_tile_to_tile(call, slope):
    """Every tile of the vocabulary lies above (below) the one before, by less and by more than a tile may add before the reference moves."""
    x = make(70, 3000, 64, seed=76)
    x["b"] = slope * torch.arange(3000, dtype=torch.float32)
    close(call(x), expect(x), f"slope {slope}")
    for topk in (0, 3):
        y = confident(0.0, topk, vocab=3000)
        y["b"] = torch.arange(3000).div(128, rounding_mode="floor") * (1.0 / 64)
        close(call(y, reduction="sum"), expect_confident(y), "confident")


# ------------------------------------------------------------------------------------------------------------------------------------
# autograd: what the backward pass holds
# ------------------------------------------------------------------------------------------------------------------------------------
def leaves(x):
    d = dev(x)
    for k in ("h", "w", "b"):
        d[k] = d[k].clone().requires_grad_(True)
    return d


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 6])
def test_saved_tensor_hooks_are_what_the_backward_pass_reads(topk):
    """Hooks that keep copies on the host: the gradients are the same bits.  Hooks that hand back other hidden states: the gradients are another's."""
    x = make(70, 400, 64, topk=topk, seed=77)
    plain = leaves(x)
    loss_of(plain).backward()
    packed = []

    def pack(t):
        packed.append(t.shape)
        return t.cpu()
    d = leaves(x)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        loss = loss_of(d)
    assert {tuple(d[k].shape) for k in ("h", "w", "b")} <= {tuple(s) for s in packed}
    loss.backward()
    for k in ("h", "w", "b"):
        assert torch.equal(d[k].grad, plain[k].grad)
    d = leaves(x)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.zeros_like(t) if t.shape == d["h"].shape else t):
        loss = loss_of(d)
    loss.backward()
    assert not d["w"].grad.any() and d["b"].grad.any()      # d weight = dz^T . hidden


@pytest.mark.gpu
def test_saved_tensors_are_free_after_the_backward_pass():
    """Hidden states that only the loss's graph holds: 4 MiB, free once the backward pass is over, though the loss itself is still there."""
    d = dev(make(4096, 100, 512, seed=78))
    one = torch.ones((), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    middle = d["h"] * one
    loss = loss_of(dict(d, h=middle))
    nbytes = middle.untyped_storage().nbytes()
    del middle
    held = torch.cuda.memory_allocated()
    loss.backward()
    assert one.grad is not None and nbytes == 4 << 20 and held - torch.cuda.memory_allocated() >= nbytes
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


@pytest.mark.gpu
def test_backward_pass_twice():
    d = leaves(make(70, 400, 64, topk=4, seed=79))
    loss = loss_of(d, reduction="sum")
    loss.backward(retain_graph=True)
    first = {k: d[k].grad.clone() for k in ("h", "w", "b")}
    loss.backward()
    for k, g in first.items():
        assert torch.equal(d[k].grad, g + g)


# ------------------------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["h", "w", "b"])
@pytest.mark.parametrize("topk", [0, 3])
def test_forward_mode_is_refused(topk, name):
    """A tangent has nowhere to go; without the refusal it would be dropped where nothing requires a gradient."""
    import torch.autograd.forward_ad as fwd
    x = make(4, 20, 8, topk=topk, seed=80)
    with fwd.dual_level():
        y = dict(x, **{name: fwd.make_dual(x[name], torch.ones_like(x[name]))})
        with pytest.raises(RuntimeError, match="forward-mode"):
            loss_of(y)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            loss_of(y)


@pytest.mark.gpu
def test_inside_a_dual_level_plain_tensors_are_taken():
    import torch.autograd.forward_ad as fwd
    x = make(20, 100, 64, seed=81)
    with fwd.dual_level():
        got = loss_of(dev(x))
    assert torch.equal(got, loss_of(dev(x)))


@pytest.mark.parametrize("change", [dict(h=None), dict(w=None), dict(h="states"), dict(w=torch.zeros(20, 8)), dict(b=torch.zeros(20).double())])
def test_operands_that_are_no_tensors_or_of_another_type(change):
    """Types are looked at before devices: the message names what is wrong wherever the rest lies."""
    x = dict(make(4, 20, 8, seed=82), **change)
    with pytest.raises(ValueError, match="|".join({"h": "hidden", "w": "weight", "b": "bias"}[k] for k in change)):
        loss_of(x)


@pytest.mark.gpu
def test_empty_dimensions_are_refused():
    for shape_h, shape_w in (((4, 0), (20, 0)), ((4, 8), (0, 8)), ((2, 0, 0), (20, 0))):
        h, w = torch.zeros(shape_h, dtype=torch.bfloat16, device="cuda"), torch.zeros(shape_w, dtype=torch.bfloat16, device="cuda")
        y = torch.zeros(shape_h[:-1], dtype=torch.long, device="cuda")
        with pytest.raises(ValueError):
            loss_of(dict(h=h, w=w, y=y, b=None, topk=0))


# ------------------------------------------------------------------------------------------------------------------------------------
# the paths of the large calls against 64 bits
# ------------------------------------------------------------------------------------------------------------------------------------
def expect_on_gpu(d, *args, **kw):
    """`expect` for operands on the GPU, computed there in 64 bits."""
    with torch.device("cuda"):
        out = expect(d, *args, **kw)
    return {k: tuple(t.cpu() for t in v) for k, v in out.items()}


def test_simulator_transposed_weights(sim):
    """2048 rows and more read the weights transposed; with two column blocks, off the tiles in every direction, in one piece and in five."""
    x = make(2304, 1100, 264, seed=90)
    want = expect(x)
    close(sim_call(x), want, "one piece")
    close(sim_call(x, piece=1), want, "pieces")


# d hidden is shared out in whole tiles per workgroup (32 tiles and more) next to a list, and in 8, 4, 2 or 1 slices of the vocabulary (from 32, 64, 128, 256
# tiles of 256 x 256 on); 2048 rows and more read transposed weights, fewer do not
@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dim,topk,T,bias,ignored", [
    (2304, 4200, 264, 0, 1.0, True, 0.0), (2200, 5003, 1288, 0, 1.0, True, 0.0), (2600, 4999, 1544, 20, 2.0, True, 0.0), (1100, 3001, 4104, 0, 1.0, False, 0.0),
    (1200, 2500, 7176, 5, 1.0, True, 0.0), (8192, 300, 2056, 0, 1.0, True, 0.0), (3500, 9001, 520, 40, 1.5, False, 0.3)])
def test_large_calls(rows, vocab, dim, topk, T, bias, ignored):
    d = dev(make(rows, vocab, dim, topk=topk, bias=bias, seed=rows, ignored=ignored))
    want = expect_on_gpu(d, T)
    close(with_grad(d, T)._asdict(), want, "one piece")
    close(with_grad(d, T, piece_bytes=1)._asdict(), want, "pieces of one tile")
    close(with_grad(d, T, piece_bytes=4 * 2048 * rows)._asdict(), want, "pieces of eight tiles")


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 32])
def test_a_full_caption_head(topk):
    """256 captions of 32 tokens, a third of them padding, on the caption decoder's head: the whole vocabulary in one piece, and in nine."""
    d = dev(make(8192, 50265, 768, topk=topk, seed=91))
    T = 2.0 if topk else 1.0
    want = expect_on_gpu(d, T)
    close(with_grad(d, T)._asdict(), want, "one piece")
    close(with_grad(d, T, piece_bytes=192 << 20)._asdict(), want, "nine pieces")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dim", [(700, 17000, 520), (2500, 6000, 776)])
@pytest.mark.parametrize("topk", [0, 9])
def test_autograd_of_large_calls_each_gradient_alone(rows, vocab, dim, topk):
    """More than 128 of the large tiles, three column blocks, in several pieces; the weights as they lie and transposed."""
    x = make(rows, vocab, dim, topk=topk, seed=92)
    want = expect_on_gpu(dev(x))
    names = {"h": "d_hidden", "w": "d_weight", "b": "d_bias"}
    for some in (("h",), ("w",), ("b",), ("w", "b"), ("h", "w", "b")):
        d = dev(x)
        for k in some:
            d[k].requires_grad_(True)
        got = torch.autograd.grad(loss_of(d, piece_bytes=4 * 2048 * rows), [d[k] for k in some])
        close({names[k]: g for k, g in zip(some, got)}, want, str(some))
