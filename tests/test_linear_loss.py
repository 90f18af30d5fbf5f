"""Losses of a linear vocabulary head (cacophony_amd.losses, csrc/linear_loss.hip) against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic alone (u32 = 2^-24, u16 = 2^-8: half a step of fp32 / bf16):
  logits     products of bf16 are exact in fp32; a sum of D of them and the bias, in any order, is off by at most (D + 1) u32 S with
             S = |h| . |w| + |b|; scaling to log2 units and back adds 4 roundings of the value:  dz = (D + 5) u32 S
  row loss   lse and z[y] are each off by max dz; exp2, log2, the joining of partial sums and the final products are good to 16 u32 of
             values no larger than |lse| + |z| + the number of halvings of the sum, 24:          dl = 2 max dz + 16 u32 (|lse| + |z| + 24)
  p          relative error ep = dz + dlse + 8 u32 (|z| + |lse|) (the exponent's rounding) + 8 u32
  d logits   g (p - q) before rounding: g (ep p + 4 u32 (p + q));  rounded to bf16: u16 |dL|
  d hidden   sum over the vocabulary of (u16 |dL| + its error) |w|, fp32 sums (V + 64) u32 |dL| |w|, one rounding u16 |dh|
  d weight   the same over the rows;  d bias: the unrounded values' errors and (rows + 64) u32 sum |dL|
"""
import ctypes as C
import math

import pytest
import torch

from cacophony_amd import _lib

U32, U16 = 2.0 ** -24, 2.0 ** -8


def make(rows, vocab, dim, *, topk=0, bias=True, ignored=0.3, seed=0, spread=1.5, dup=False):
    """Inputs on the CPU.  ignored: share of rows that do not count (the first row counts)."""
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, dim, generator=gen).bfloat16()
    w = (torch.randn(vocab, dim, generator=gen) * spread / math.sqrt(dim)).bfloat16()
    b = torch.randn(vocab, generator=gen) * 0.3 if bias else None
    off = torch.rand(rows, generator=gen) < ignored
    off[:1] = ignored >= 1.0
    x = dict(h=h, w=w, b=b, topk=topk)
    if topk:
        idx = torch.randint(0, max(1, vocab // 8) if dup else vocab, (rows, topk), generator=gen)
        idx[torch.rand(rows, topk, generator=gen) < 0.1] = -1
        idx[off] = -1
        x.update(teacher=torch.randn(rows, topk, generator=gen) * 3, idx=idx)
    else:
        y = torch.randint(0, vocab, (rows,), generator=gen)
        y[off] = -100
        x["y"] = y
    return x


def targets(x, T):
    """q [rows, vocab] in 64 bits and which rows count."""
    R, V = x["h"].shape[0], x["w"].shape[0]
    q = torch.zeros(R, V, dtype=torch.float64)
    if not x["topk"]:
        on = (x["y"] >= 0) & (x["y"] < V) & (x["y"] != x.get("ignore", -100))
        q[on.nonzero()[:, 0], x["y"][on]] = 1.0
        return q, on
    there = (x["idx"] >= 0) & (x["idx"] < V) & (x["teacher"] > -math.inf)
    on = there.any(1)
    t = torch.where(there, x["teacher"].double() / T, -math.inf)
    t = torch.where(on[:, None], t, 0.0).softmax(1) * there
    q.scatter_add_(1, torch.where(there, x["idx"].long(), 0), t)
    return q, on


def expect(x, T=1.0, g=None, reduction="mean", row_weight=None):
    """Everything a call returns, in 64 bits, each with its tolerance."""
    h, w = x["h"].double(), x["w"].double()
    R, V, D = h.shape[0], w.shape[0], h.shape[1]
    q, on = targets(x, T)
    h = torch.where(on[:, None], h, 0.0)
    b = x["b"].double() if x["b"] is not None else torch.zeros(V, dtype=torch.float64)
    z = (h @ w.T + b) / T
    dz = (D + 5) * U32 * ((h.abs() @ w.abs().T + torch.where(b.isfinite(), b, 0.0).abs()) / T)
    lse = torch.logsumexp(z, 1)
    lp = z - lse[:, None]
    loss = T * T * (torch.special.xlogy(q, q) - torch.where(q > 0, q * lp, 0.0)).sum(1) * on
    zmax = torch.where(z.isfinite(), z, 0.0).abs().amax(1) if V else lse * 0
    dmax = dz.amax(1)
    dlse = dmax + 16 * U32 * (lse.abs() + zmax + 24)
    # the distillation's own sum: teacher weights and their logarithms to 64 u32 of entries no larger than |t| / T + log K
    own = 64 * U32 * (x["teacher"].double().abs().nan_to_num(0, 0, 0).amax(1) / T + 8) if x["topk"] else 0.0
    n = int(on.sum())
    wt = torch.ones(R, dtype=torch.float64) if row_weight is None else row_weight.double()
    tot = (loss * wt).sum()
    dl_tol = T * T * (2 * dmax + 16 * U32 * (lse.abs() + zmax + 24) + own)
    out = {"row_loss": (loss, dl_tol * on), "lse": (lse * on, dlse * on)}
    div = n if reduction == "mean" else 1
    if n:
        out["loss"] = (tot / div, (dl_tol * on * wt.abs()).sum() / div + 8 * U32 * (loss * wt).abs().sum() / div)
    gr = (on.double() * wt * T / max(div, 1) * (1.0 if g is None else g))[:, None]
    p = lp.exp()
    dL = gr * (p - q)
    ep = dz + dlse[:, None] + 8 * U32 * (torch.where(z.isfinite(), z, 0.0).abs() + lse.abs()[:, None]) + 8 * U32
    raw = gr.abs() * (ep * p + (4 * U32 + (64 * U32 * (own / U32 / 64) if x["topk"] else 0.0)[:, None] * 2 if x["topk"] else 4 * U32) * (p + q))
    dLt = raw + U16 * (dL.abs() + raw)
    for name, val, a, m in (("d_hidden", dL @ w, dL.abs(), w.abs()), ("d_weight", None, None, None)):
        if name == "d_hidden":
            out[name] = (val, (dLt @ m + (V + 64) * U32 * (a @ m)) * (1 + U16) + U16 * val.abs() + 1e-38)
        else:
            val = dL.T @ h
            out[name] = (val, (dLt.T @ h.abs() + (R + 64) * U32 * (dL.abs().T @ h.abs())) * (1 + U16) + U16 * val.abs() + 1e-38)
    out["d_bias"] = (dL.sum(0), raw.sum(0) + (R + 64) * U32 * dL.abs().sum(0) + 1e-38)
    return out


def close(got, want, what):
    for name, value in got.items():
        if value is None or name not in want:
            continue
        val, tol = want[name]
        v = value.detach().double().cpu().reshape(val.shape)
        assert torch.isfinite(v).all(), f"{what}: {name} has {int((~torch.isfinite(v)).sum())} values that are not finite"
        bad = (v - val).abs() > tol
        assert not bad.any(), f"{what}: {name}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((v - val).abs() / (tol + 1e-300)).max()):.3g} tolerances"


# rows, vocab, dim, topk, temperature, bias: one token; one word; a ragged everything; rows on both sides of the small tile's 64 and of
# the large tile's 256; dims below, at and off the K-tile; a vocabulary below, at and just past a tile
SHAPES = [
    (1, 1, 8, 0, 1.0, True), (1, 257, 64, 0, 1.0, True), (5, 300, 72, 0, 1.0, False), (64, 256, 128, 0, 1.0, True), (65, 513, 136, 0, 1.0, True),
    (256, 255, 64, 0, 1.0, False), (257, 700, 264, 0, 1.0, True),
    # more than 128 of the large tiles; d weight in runs of tokens (1500 rows and more, few tiles)
    (257, 16500, 72, 0, 1.0, True), (130, 33000, 8, 3, 2.0, True), (600, 11100, 136, 0, 1.0, False),
    (1024, 300, 72, 0, 1.0, True), (1500, 257, 264, 4, 1.0, True), (4100, 40, 8, 0, 1.0, True),
    (1, 40, 64, 1, 1.0, True), (7, 500, 64, 5, 2.0, False), (66, 300, 200, 33, 0.5, True), (130, 600, 72, 128, 4.0, True),
]


# ------------------------------------------------------------------------------------------------------------------------------------
# CPU: the kernels' sources on the simulator, the refusals
# ------------------------------------------------------------------------------------------------------------------------------------
def sim_call(x, T=1.0, what=3, reduction=1, piece=1 << 30, row_weight=None, ld=0):
    from tests import simlib
    lib, P = simlib.load(), simlib.ptr
    R, D, V, K = x["h"].shape[0], x["h"].shape[1], x["w"].shape[0], x["topk"]
    f = lambda *s: torch.full(s, float("nan"))
    o = dict(row_loss=f(R), lse=f(R), loss=f(1), d_hidden=f(R, D).bfloat16(), d_weight=f(V, D).bfloat16(), d_bias=f(V))
    need = lib.caco_linear_loss_workspace(R, V, D, K, piece, what)
    guard = 4096
    ws = torch.full((need + guard,), 0xFF, dtype=torch.uint8)
    first = (what, P(x["h"]), D, P(x["w"]), D, P(x["b"]))
    last = (R, V, D, reduction, P(row_weight), None, P(o["row_loss"]), P(o["lse"]), P(o["loss"]), P(o["d_hidden"]), D, P(o["d_weight"]), D,
            P(o["d_bias"]), P(ws), need, None)
    if K:
        rc = lib.caco_linear_distill(*first, P(x["teacher"]), K, P(x["idx"]), K, x["idx"].element_size(), K, T, *last)
    else:
        rc = lib.caco_linear_ce(*first, P(x["y"]), x.get("ignore", -100), *last)
    simlib.check(rc, "linear loss")
    assert (ws[need:] == 0xFF).all(), "wrote past the workspace"
    return o


@pytest.fixture(scope="module")
def sim():
    from tests import simlib
    if not simlib.available():
        pytest.skip("needs ROCm's clang++ for the simulator")
    return simlib.load()


@pytest.mark.parametrize("rows,vocab,dim,topk,T,bias", SHAPES)
def test_losses_and_gradients_on_the_simulator(sim, rows, vocab, dim, topk, T, bias):
    x = make(rows, vocab, dim, topk=topk, bias=bias, seed=rows)
    close(sim_call(x, T, piece=1), expect(x, T), "pieces of one tile")
    close(sim_call(x, T), expect(x, T), "one piece")


def test_simulator_weights_sum_masked_rows_and_repeated_entries(sim):
    x = make(70, 300, 64, topk=20, seed=3, dup=True)
    wt = torch.linspace(-1, 2, 70)
    wt[5] = 0.0
    close(sim_call(x, 1.5, reduction=2, row_weight=wt), expect(x, 1.5, reduction="sum", row_weight=wt), "weights")
    x = make(70, 300, 64, seed=4)
    off = x["y"] < 0
    x["h"][off] = float("nan")
    close(sim_call(x), expect(x), "NaN in rows that do not count")


def test_simulator_no_row_counts(sim):
    for rows in (0, 5):
        x = make(rows, 300, 64, ignored=1.0, seed=5)
        o = sim_call(x)
        assert torch.isnan(o["loss"]).all() and not o["d_weight"].any() and not o["d_bias"].any()
        assert not o["d_hidden"].any() and not o["row_loss"].any() and not o["lse"].any()
        assert float(sim_call(x, reduction=2)["loss"]) == 0.0


def _ce(lib, **kw):
    """caco_linear_ce on host memory with one argument changed; only for calls that are refused before any launch."""
    a = dict(what=3, hidden=1024, ld_h=64, weight=1024, ld_w=64, bias=None, labels=1024, ignore=-100, rows=4, vocab=300, dim=64, reduction=1, row_weight=None,
             scale=None, row_loss=1024, lse=1024, loss=1024, dh=1024, ld_dh=64, dw=1024, ld_dw=64, db=1024, ws=1024, ws_bytes=0, st=None)
    a.update(kw)
    return lib.caco_linear_ce(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(what=0), b"what"), (dict(what=4), b"what"), (dict(reduction=3), b"reduction"), (dict(reduction=-1), b"reduction"),
    (dict(hidden=None), b"null"), (dict(weight=None), b"null"), (dict(labels=None), b"null"), (dict(ws=None), b"null"),
    (dict(rows=-1), b"rows"), (dict(rows=2 ** 24 + 1), b"rows"), (dict(rows=2 ** 22 + 1), b"rows"), (dict(vocab=0), b"vocab"), (dict(vocab=2 ** 24 + 1), b"vocab"),
    (dict(dim=0), b"dim"), (dict(dim=60), b"dim"), (dict(dim=65544), b"dim"), (dict(row_loss=None), b"row_loss"), (dict(reduction=0), b"reduced loss"),
    (dict(what=2, loss=None, lse=None), b"lse"), (dict(dh=None, dw=None, db=None), b"no output"),
    (dict(ld_h=56), b"16 bytes"), (dict(ld_h=65), b"16 bytes"), (dict(ld_w=56), b"16 bytes"), (dict(ld_w=68), b"16 bytes"), (dict(ld_w=1 << 22), b"16 bytes"),
    (dict(hidden=1032), b"16 bytes"), (dict(weight=1032), b"16 bytes"), (dict(dh=1032), b"16 bytes"), (dict(dw=1032), b"16 bytes"), (dict(ld_dh=60), b"16 bytes"),
    (dict(ld_dw=8), b"16 bytes"), (dict(ws=1032), b"workspace must be"), (dict(ws_bytes=1000), b"too small"), (dict(what=1, ws_bytes=1000), b"too small"),
])
def test_calls_that_are_refused(change, message):
    lib = _lib.load()
    assert _ce(lib, **change) == _lib.CACO_ERR_INVALID
    assert message in lib.caco_last_error(), lib.caco_last_error()


def test_distillation_calls_that_are_refused():
    lib = _lib.load()

    def call(topk=4, T=1.0, nbytes=8, ld_t=4, ld_i=4, teacher=1024, idx=1024):
        return lib.caco_linear_distill(3, 1024, 64, 1024, 64, None, teacher, ld_t, idx, ld_i, nbytes, topk, T, 4, 300, 64, 1, None, None, 1024, 1024, 1024,
                                       1024, 64, 1024, 64, 1024, 1024, 0, None)
    for kw in (dict(topk=0), dict(topk=129, ld_t=129, ld_i=129), dict(T=0.0), dict(T=-1.0), dict(T=math.inf), dict(T=math.nan), dict(T=2.0 ** -21), dict(T=2.0 ** 21), dict(T=1e-40), dict(nbytes=2), dict(ld_t=3),
               dict(ld_i=3), dict(teacher=None), dict(idx=None), dict()):
        assert call(**kw) == _lib.CACO_ERR_INVALID, kw
    assert b"too small" in lib.caco_last_error()


def test_workspace_sizes():
    lib = _lib.load()
    size = lib.caco_linear_loss_workspace
    assert size(-1, 300, 64, 0, 1 << 30, 3) == _lib.CACO_ERR_INVALID and size(1, 300, 60, 0, 1 << 30, 3) == _lib.CACO_ERR_INVALID
    fwd, one, many = size(8192, 50265, 768, 0, 1 << 30, 1), size(8192, 50265, 768, 0, 1 << 30, 3), size(8192, 50265, 768, 0, 1, 3)
    assert 0 < fwd < many < one and one < 2 << 30 and fwd < 32 << 20
    assert size(8192, 50265, 768, 128, 1 << 30, 1) > fwd
    # 255 strides of a transposed operand are addressed with 31 bits: no piece has more than 2^22 columns, however much memory there is
    all_of_it = 2 * 2 * 256 * 2 ** 24
    assert size(1, 2 ** 24, 8, 0, 1 << 50, 3) < size(1, 2 ** 22, 8, 0, 1 << 50, 3) + (size(1, 2 ** 24, 8, 0, 1, 3) - size(1, 2 ** 22, 8, 0, 1, 3)) + (1 << 20) < all_of_it
    assert size(2 ** 22, 50265, 768, 0, 1 << 30, 3) > 0 > size(2 ** 22 + 1, 50265, 768, 0, 1 << 30, 3)


@pytest.mark.skipif(torch.cuda.is_available(), reason="exercises the no-GPU failure mode")
def test_python_checks_without_a_gpu():
    from cacophony_amd import losses
    h, w, y = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(10, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="same GPU"):
        losses.linear_cross_entropy(h, w, y)
    with pytest.raises(ValueError, match="reduction"):
        losses.linear_cross_entropy(h, w, y, reduction="max")
    with pytest.raises(ValueError, match="hidden must be"):
        losses.linear_cross_entropy(h.float(), w, y)


# ------------------------------------------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------------------------------------------
def dev(x):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in x.items()}


def with_grad(x, T=1.0, **kw):
    from cacophony_amd import losses
    if x["topk"]:
        return losses.linear_topk_distillation_with_grad(x["h"], x["w"], x["teacher"], x["idx"], x["b"], temperature=T, **kw)
    return losses.linear_cross_entropy_with_grad(x["h"], x["w"], x["y"], x["b"], ignore_index=x.get("ignore", -100), **kw)


def loss_of(x, T=1.0, **kw):
    from cacophony_amd import losses
    if x["topk"]:
        return losses.linear_topk_distillation(x["h"], x["w"], x["teacher"], x["idx"], x["b"], temperature=T, **kw)
    return losses.linear_cross_entropy(x["h"], x["w"], x["y"], x["b"], ignore_index=x.get("ignore", -100), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dim,topk,T,bias", SHAPES + [
    (700, 5003, 768, 0, 1.0, True), (1000, 3001, 520, 100, 1.0, False), (600, 2000, 1032, 0, 1.0, False), (64, 20000, 768, 10, 2.0, True),
    (300, 1500, 4096, 3, 1.0, True)])
def test_losses_and_gradients(rows, vocab, dim, topk, T, bias):
    x = make(rows, vocab, dim, topk=topk, bias=bias, seed=rows)
    want = expect(x, T)
    d = dev(x)
    close(with_grad(d, T)._asdict(), want, "one piece")
    close(with_grad(d, T, piece_bytes=1)._asdict(), want, "pieces")
    rows_only = loss_of(d, T, reduction="none")
    close({"row_loss": rows_only}, want, "losses alone")
    assert rows_only.shape == (rows,) and rows_only.dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 9])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd_gives_the_same_gradients(topk, reduction):
    x = make(90, 700, 136, topk=topk, seed=1)
    d = dev(x)
    wt = torch.linspace(-0.5, 1.5, 90)
    for k in ("h", "w", "b"):
        d[k].requires_grad_(True)
    out = loss_of(d, 2.0 if topk else 1.0, reduction=reduction)
    T = 2.0 if topk else 1.0
    if reduction == "none":
        (out * wt.cuda()).sum().backward()
        want = expect(x, T, reduction="sum", row_weight=wt)
    else:
        (out * 3.0).backward()
        want = expect(x, T, g=3.0, reduction=reduction)
        close({"loss": out}, want, "loss")
    close({"d_hidden": d["h"].grad, "d_weight": d["w"].grad, "d_bias": d["b"].grad}, want, reduction)


@pytest.mark.gpu
def test_autograd_of_some_inputs_only():
    x = make(80, 600, 64, seed=2)
    want = expect(x)
    for names in (("h",), ("w",), ("b",), ("h", "b")):
        d = dev(x)
        for k in names:
            d[k].requires_grad_(True)
        got = torch.autograd.grad(loss_of(d), [d[k] for k in names])
        close({{"h": "d_hidden", "w": "d_weight", "b": "d_bias"}[k]: g for k, g in zip(names, got)}, want, str(names))


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 6])
def test_gradient_against_differences(topk):
    """(l(h + e v) - l(h - e v)) / 2e against d_hidden . v, the steps chosen so that h +- e v is exact in bf16: h on a grid of 2^-4, steps of 2^-4.  The losses are
    off by `row_loss`'s tolerance each; the difference's own error is e^2 / 6 times the third derivative along v, which for a loss of this kind is at most
    2 T^2 (spread / T)^3 with the spread of the logits' slope, max - min of w . v."""
    x = make(12, 90, 64, topk=topk, seed=6, ignored=0.0, spread=0.5)
    T, e = 1.0, 2.0 ** -4
    x["h"] = (x["h"].float() * 16).round().div(16).clamp(-4, 4).bfloat16()
    v = torch.zeros(12, 64)
    v[:, 3], v[:, 40] = 1.0, -1.0
    plus, minus = dict(x, h=(x["h"].float() + e * v).bfloat16()), dict(x, h=(x["h"].float() - e * v).bfloat16())
    assert torch.equal(plus["h"].float() - x["h"].float(), e * v)
    got = (loss_of(dev(plus), T, reduction="none") - loss_of(dev(minus), T, reduction="none")).double().cpu() / (2 * e)
    g = with_grad(dev(x), T, reduction="sum").d_hidden.double().cpu()
    slope = x["w"].double() @ v[0].double()
    tol = (expect(plus)["row_loss"][1] + expect(minus)["row_loss"][1]) / (2 * e) + e * e / 6 * 2 * (slope.max() - slope.min()) ** 3 \
        + (expect(x, reduction="sum")["d_hidden"][1] * v.abs()).sum(1)
    assert ((got - (g * v).sum(1)).abs() <= tol).all()


@pytest.mark.gpu
def test_strides_offsets_and_label_types():
    from cacophony_amd import losses
    x = make(96, 500, 72, seed=8)
    want = expect(x)
    d = dev(x)
    wide_h, wide_w = torch.zeros(96, 160, dtype=torch.bfloat16, device="cuda"), torch.full((500, 88), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_h[:, 8:80], wide_w[:, :72] = d["h"], d["w"]
    nan_bias = torch.full((504,), float("nan"), device="cuda")
    nan_bias[3:503] = d["b"]
    for name, y in (("row strides, read in place", dict(d, h=wide_h[:, 8:80], w=wide_w[:, :72])),
                    ("rows off 16 bytes", dict(d, h=torch.cat([d["h"], d["h"]], 1)[:, 3:75].copy_(d["h"]), b=nan_bias[3:503])),
                    ("transposed storage", dict(d, h=d["h"].t().contiguous().t(), w=d["w"].t().contiguous().t())),
                    ("int32 labels", dict(d, y=d["y"].int()))):
        close(with_grad(y)._asdict(), want, name)
    o = losses.linear_cross_entropy_with_grad(d["h"].view(4, 24, 72), d["w"], d["y"].view(4, 24), d["b"])
    assert o.row_loss.shape == (4, 24) and o.d_hidden.shape == (4, 24, 72)
    close(o._asdict(), want, "leading dimensions")
    one = losses.linear_cross_entropy(d["h"][:1].expand(7, 72), d["w"], d["y"][:1].expand(7), d["b"], reduction="none")
    assert (one == one[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 7])
def test_what_does_not_count_reaches_nothing(topk):
    x = make(150, 700, 64, topk=topk, seed=9, ignored=0.5)
    _, on = targets(x, 1.0)
    for junk in (float("nan"), float("inf"), 3.0e38):
        y = dict(x, h=torch.where(on[:, None], x["h"], torch.tensor(junk).bfloat16()))
        o = with_grad(dev(y))
        close(o._asdict(), expect(x), f"{junk} in rows that do not count")
        assert not o.d_hidden.cpu()[~on].any() and not o.row_loss.cpu()[~on].any()
    # nothing counts at all
    y = dict(x, h=torch.full_like(x["h"], float("nan")))
    if topk:
        y["idx"] = torch.full_like(x["idx"], -1)
    else:
        y["y"] = torch.full_like(x["y"], -100)
    o = with_grad(dev(y))
    assert torch.isnan(o.loss) and not o.d_hidden.any() and not o.d_weight.any() and not o.d_bias.any() and not o.row_loss.any()
    assert float(loss_of(dev(y), reduction="sum")) == 0.0


@pytest.mark.gpu
def test_labels_outside_the_vocabulary_and_another_ignore_index():
    x = make(100, 300, 64, seed=10, ignored=0.0)
    x["y"][::7] = 300
    x["y"][1::7] = -1
    x["y"][2::7] = 2 ** 40
    close(with_grad(dev(x))._asdict(), expect(x), "outside")
    x["ignore"] = int(x["y"][4])
    close(with_grad(dev(x))._asdict(), expect(x), "ignore_index is a word")


@pytest.mark.gpu
def test_banned_words_and_extreme_rows():
    """A bias of -inf or of the lowest fp32 value takes a word out; a row whose logits are thousands apart; labels that are certain."""
    x = make(70, 600, 64, seed=11)
    x["b"][5:400] = -math.inf
    x["b"][400:500] = torch.finfo(torch.float32).min
    x["y"] = torch.where(x["y"] >= 0, 500 + x["y"] % 100, x["y"])
    y = dict(x, b=torch.where(x["b"] < -1e30, torch.tensor(-math.inf), x["b"]))
    close(with_grad(dev(x))._asdict(), expect(y), "banned")
    x = make(70, 600, 64, seed=12)
    x["h"][::3] *= 1000
    close({k: v for k, v in with_grad(dev(x))._asdict().items() if k in ("row_loss", "loss")}, expect(x), "steep")


@pytest.mark.gpu
def test_a_nan_row_is_its_own():
    x = make(70, 300, 64, seed=13, ignored=0.0)
    x["h"][9, 3] = float("nan")
    o = with_grad(dev(x))
    bad = torch.isnan(o.row_loss.cpu())
    assert bad[9] and bad.sum() == 1 and torch.isnan(o.loss)
    keep = torch.arange(70) != 9
    assert torch.isfinite(o.d_hidden.cpu()[keep].float()).all()


@pytest.mark.gpu
def test_teacher_lists_repeated_padded_and_unsorted():
    x = make(90, 800, 64, topk=40, seed=14, dup=True)
    x["teacher"][::5, 1:] = -math.inf
    x["teacher"][3] = -math.inf
    x["idx"][4] = x["idx"][4, 0].clamp_min(0)
    x["idx"][6, ::2] = 800
    want = expect(x, 1.5)
    d = dev(x)
    close(with_grad(d, 1.5)._asdict(), want, "int64")
    close(with_grad(dict(d, idx=d["idx"].int()), 1.5)._asdict(), want, "int32")
    perm = torch.randperm(40, generator=torch.Generator().manual_seed(1)).cuda()
    close(with_grad(dict(d, idx=d["idx"][:, perm], teacher=d["teacher"][:, perm]), 1.5)._asdict(), want, "another order")


@pytest.mark.gpu
def test_row_weights_and_their_zeros():
    x = make(130, 500, 64, seed=15)
    wt = torch.randn(130, generator=torch.Generator().manual_seed(2))
    wt[::4] = 0.0
    d = dev(x)
    for red in ("mean", "sum", "none"):
        close(with_grad(d, row_weight=wt.cuda(), reduction=red)._asdict(), expect(x, reduction=red, row_weight=wt), red)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 12])
def test_equal_calls_give_equal_bits_and_pieces_change_little(topk):
    d = dev(make(520, 3000, 256, topk=topk, seed=16))
    a, b = with_grad(d), with_grad(d)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    c = with_grad(d, piece_bytes=1)
    assert torch.equal(a.d_weight, c.d_weight) and torch.equal(a.d_bias, c.d_bias) and torch.equal(a.row_loss, c.row_loss)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 12])
def test_captured_and_replayed_between_eager_calls(topk):
    xs = [dev(make(200, 900, 128, topk=topk, seed=s)) for s in (20, 21, 22, 23)]
    static = {k: v.clone() if torch.is_tensor(v) else v for k, v in xs[0].items()}
    with_grad(static), loss_of(static, reduction="none")
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = with_grad(static)
    with torch.cuda.graph(g2):
        o2 = loss_of(static, reduction="none")
    for rep in range(2):
        for x in xs:
            for k, v in static.items():
                if torch.is_tensor(v):
                    v.copy_(x[k])
            g1.replay()
            g2.replay()
            torch.cuda.synchronize()
            e = with_grad(x)
            for a, b in zip(o1, e):
                assert torch.equal(a, b)
            assert torch.equal(o2, e.row_loss)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dim,topk", [(2100, 700, 72, 0), (2100, 300, 264, 100), (40, 20000, 64, 7), (900, 17000, 64, 3)])
def test_equal_bits_in_pieces_and_in_a_graph(rows, vocab, dim, topk):
    """d weight in runs of tokens, transposed weights, few words that many teacher entries share; one row to a workgroup at the end."""
    x, y = (dev(make(rows, vocab, dim, topk=topk, seed=s)) for s in (60, 61))
    static = {k: v.clone() if torch.is_tensor(v) else v for k, v in x.items()}
    with_grad(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = with_grad(static)
    for z in (x, y, x):
        for k, v in static.items():
            if torch.is_tensor(v):
                v.copy_(z[k])
        graph.replay()
        torch.cuda.synchronize()
        e = with_grad(z)
        for a, b in zip(out, e):
            assert torch.equal(a, b)
        p = with_grad(z, piece_bytes=1)
        assert torch.equal(p.d_weight, e.d_weight) and torch.equal(p.d_bias, e.d_bias) and torch.equal(p.row_loss, e.row_loss)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["h", "w", "b", "y", "teacher", "idx"])
def test_an_operand_changed_before_the_backward_pass_is_an_error(name):
    from cacophony_amd import losses
    d = dev(make(20, 150, 64, topk=0 if name == "y" else 3, seed=41))
    h = d["h"].clone().requires_grad_()
    if name == "y":
        loss = losses.linear_cross_entropy(h, d["w"], d["y"], d["b"])
    else:
        loss = losses.linear_topk_distillation(h, d["w"], d["teacher"], d["idx"], d["b"])
    with torch.no_grad():
        (h if name == "h" else d[name]).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_autograd_refuses_capture():
    d = dev(make(64, 300, 64, seed=24))
    d["h"].requires_grad_(True)
    live = loss_of(d)                      # an eager graph of the same leaves
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="linear_cross_entropy_with_grad"):
        with torch.cuda.graph(g):
            loss_of(d)
    torch.cuda.synchronize()
    live.backward()
    assert d["h"].grad is not None


@pytest.mark.gpu
def test_a_backward_pass_refuses_capture(monkeypatch):
    """The forward pass ran before the capture; nothing is captured here, the stream only says so."""
    from cacophony_amd import losses
    d = dev(make(20, 150, 64, seed=42))
    h = d["h"].clone().requires_grad_()
    loss = losses.linear_cross_entropy(h, d["w"], d["y"], d["b"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        loss.backward()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    xs = [dev(make(300, 2000, 128, topk=k, seed=30 + k)) for k in (0, 5)]
    want = [with_grad(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(with_grad(xs[i]))
    torch.cuda.synchronize()
    for w, os in zip(want, got):
        for o in os:
            for a, b in zip(w, o):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_python_refusals():
    from cacophony_amd import losses
    d = dev(make(8, 100, 64, topk=3, seed=40))
    h, w, b, t, i = d["h"], d["w"], d["b"], d["teacher"], d["idx"]
    y = torch.zeros(8, dtype=torch.long, device="cuda")
    ce, kd = losses.linear_cross_entropy, losses.linear_topk_distillation
    for exc, call in (
            (ValueError, lambda: ce(h.half(), w, y)), (ValueError, lambda: ce(h, w.float(), y)), (ValueError, lambda: ce(h, w, y, b.bfloat16())),
            (ValueError, lambda: ce(h, w, y.float())), (ValueError, lambda: ce(h, w, y > 0)), (ValueError, lambda: ce(h, w, y[:7])),
            (ValueError, lambda: ce(h, w[:, :32], y)), (ValueError, lambda: ce(h, w, y, b[:50])), (ValueError, lambda: ce(h, w[0], y)),
            (ValueError, lambda: ce(h, w, y, reduction="avg")), (ValueError, lambda: ce(h, w, y, piece_bytes=0)),
            (ValueError, lambda: losses.linear_cross_entropy_with_grad(h, w, y, piece_bytes=0)), (ValueError, lambda: ce(h[:, :60], w[:, :60], y)),
            (RuntimeError, lambda: ce(h.cpu(), w, y)), (RuntimeError, lambda: ce(h, w.cpu(), y)), (RuntimeError, lambda: ce(h, w, y.cpu())),
            (ValueError, lambda: kd(h, w, t, i, temperature=0.0)), (ValueError, lambda: kd(h, w, t, i.float())), (ValueError, lambda: kd(h, w, t.long(), i)),
            (ValueError, lambda: kd(h, w, t[:, :2], i)), (ValueError, lambda: kd(h, w, t[:, :0], i[:, :0])),
            (ValueError, lambda: kd(h, w, t.repeat(1, 50), i.repeat(1, 50))),
            (ValueError, lambda: losses.linear_cross_entropy_with_grad(h, w, y, row_weight=torch.ones(8, device="cuda", dtype=torch.float64)))):
        with pytest.raises(exc):
            call()
    # no rows at all
    o = losses.linear_cross_entropy_with_grad(h[:0], w, y[:0], b, reduction="sum")
    assert float(o.loss) == 0.0 and not o.d_weight.any() and not o.d_bias.any() and o.d_hidden.shape == (0, 64)


@pytest.mark.gpu
def test_teacher_to_student_as_used():
    """The teacher's top logits by `retrieval.topk`, the student's losses and gradients from them, and its likelihoods, in one run."""
    from cacophony_amd import losses, retrieval
    gen = torch.Generator().manual_seed(50)
    x = make(60, 900, 128, seed=51)
    x["y"] = torch.where(x["y"] < 0, torch.zeros_like(x["y"]), x["y"])
    teacher_logits = torch.randn(60, 900, generator=gen) * 2
    idx, val = retrieval.topk(teacher_logits.cuda(), 16)
    x.update(topk=16, idx=idx.cpu().long(), teacher=val.cpu())
    d = dev(x)
    kd = losses.linear_topk_distillation_with_grad(d["h"], d["w"], val, idx, d["b"], temperature=2.0)
    close(kd._asdict(), expect(x, 2.0), "distillation")
    ce = losses.linear_cross_entropy(d["h"], d["w"], d["y"], d["b"], reduction="none")
    close({"row_loss": ce}, expect(dict(x, topk=0)), "likelihood")
