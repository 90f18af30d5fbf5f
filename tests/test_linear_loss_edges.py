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
