"""Likelihoods of given captions (caco_decoder_score, CACO.get_caption_nll, captioning.score_captions): the caption decoder's hidden
states through the linear cross entropy, checked against the cross entropy of the logits the decoder gives for the same captions
(src/caco_torch/caco.py:212-240) and against the reference's own logits."""
import ctypes as C
from dataclasses import replace

import numpy as np
import pytest
import torch

from cacophony_amd import _lib, config, synth
from tests.conftest import load_golden


def _configs():
    a, t, cc = config.tiny_configs(2)
    return a, t, cc, replace(t, num_hidden_layers=2)


@pytest.fixture(scope="module")
def model():
    from cacophony_amd.model import CACO
    a, t, cc, d = _configs()
    return CACO(a, t, cc, decoder_config=d, device="cuda:0").load_state_dict(synth.make_caco_state(a, t, cc, seed=0, decoder_cfg=d))


@pytest.fixture(scope="module")
def clips(model):
    from cacophony_amd import frontend
    ab = frontend.mel_patches_device(torch.from_numpy(synth.make_waveforms(2, start=40)).cuda(), 500, torch.float32)
    _, ah = model.get_audio_embedding(ab["audio_patches"], ab["audio_time_inds"], ab["audio_freq_inds"], ab["audio_mask"])
    return ab, ah


def nll_of(logits, ids, mask):
    """fp64 [B, T - 1] from logits of the first T - 1 tokens"""
    lp = torch.log_softmax(logits.double().cpu(), -1)
    return torch.where(torch.as_tensor(mask)[:, 1:] != 0, -lp.gather(2, torch.as_tensor(ids)[:, 1:, None])[..., 0], 0.0)


def test_refused_without_a_model():
    lib = _lib.load()
    one = C.c_void_p(1024)
    assert lib.caco_decoder_score(None, one, one, one, one, one, -100, 1, 1, 1, one, None) == _lib.CACO_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("n,start", [(2, 40), (9, 7), (33, 100)])
def test_nll_is_the_cross_entropy_of_the_decoders_logits(model, clips, n, start):
    """Same hidden states, bit for bit, on both sides; what differs is the order in which 768 products are added up in fp32, at most
    768 * 2^-24 of the sum of their magnitudes (below 10 here: layer-normed states times 0.02 weights) and twice that for
    logsumexp minus logit: 1e-3."""
    ab, ah = clips
    V = model.text_config.vocab_size
    ids, mask = synth.make_captions(n, 32, V, start=start)
    pick = torch.arange(n, device="cuda") % 2
    ah, am = ah[pick], ab["audio_mask"][pick]
    nll = model.get_caption_nll(ah, am, ids, mask)
    assert nll.shape == (n, 31) and nll.dtype == torch.float32
    want = nll_of(model.get_decoder_logits(ah, am, ids[:, :-1], mask[:, :-1]), ids, mask)
    assert (nll.cpu().double() - want).abs().max() < 1e-3
    assert not nll.cpu()[torch.as_tensor(mask)[:, 1:] == 0].any()
    assert torch.equal(nll, model.get_caption_nll(ah, am, ids, mask))


@pytest.mark.gpu
def test_nll_against_the_references_logits(model, clips):
    """bf16 operands against the reference's fp32: the logits' bar is rel-L2 1e-2; a row's logits have 2-norm |z|, so a logit is off by
    at most 1e-2 |z| and its likelihood by twice that."""
    g = load_golden("decoder_tiny.npz")
    ab, ah = clips
    nll = model.get_caption_nll(ah, ab["audio_mask"], g["ids"], g["tmask"]).cpu().double()
    z = torch.from_numpy(g["logits"][:, :-1])
    bound = 2e-2 * z.double().norm(dim=-1)
    assert ((nll - nll_of(z, g["ids"], g["tmask"])).abs() <= bound).all()


@pytest.mark.gpu
def test_smallest_and_padded_captions(model, clips):
    ab, ah = clips
    am = ab["audio_mask"]
    ids = torch.tensor([[0, 17], [0, 4]])
    nll = model.get_caption_nll(ah, am, ids, torch.ones_like(ids))
    want = nll_of(model.get_decoder_logits(ah, am, ids[:, :1], torch.ones(2, 1)), ids, torch.ones_like(ids))
    assert nll.shape == (2, 1) and (nll.cpu().double() - want).abs().max() < 1e-3
    # a caption of which only BOS exists has no likelihood to add; the other's stays as it is, whatever lies behind its end
    ids, mask = synth.make_captions(2, 16, model.text_config.vocab_size, start=3)
    mask = mask.copy()
    mask[0, 1:] = 0
    mask[1, 9:] = 0
    other = ids.copy()
    other[:, 9:] = 5
    one, two = model.get_caption_nll(ah, am, ids, mask), model.get_caption_nll(ah, am, other, mask)
    assert not one[0].any() and not one[1, 8:].any() and one[1, :8].all() and torch.equal(one[1], two[1])


@pytest.mark.gpu
def test_score_captions_ranks_a_clips_candidates(model, clips):
    from cacophony_amd import captioning
    ab, ah = clips
    ids, mask = synth.make_captions(6, 24, model.text_config.vocab_size, start=60)
    score, count = captioning.score_captions(model, ab, ids, mask, captions_per_clip=3)
    assert score.shape == count.shape == (6,) and count.cpu().tolist() == (mask[:, 1:] != 0).sum(1).tolist()
    for c in range(2):
        for i in range(3):
            r = 3 * c + i
            lg = model.get_decoder_logits(ah[c:c + 1], ab["audio_mask"][c:c + 1], ids[r:r + 1, :-1], mask[r:r + 1, :-1])
            want = -nll_of(lg, ids[r:r + 1], mask[r:r + 1]).sum()
            assert abs(float(score[r]) - float(want)) < 2e-2 * abs(float(want)) + 1e-3      # other row counts, other GEMM tiles: bf16 roundings of the states
    with pytest.raises(ValueError, match="3 captions"):
        captioning.score_captions(model, ab, ids[:5], mask[:5], captions_per_clip=3)
    with pytest.raises(ValueError, match=r"T >= 2"):
        model.get_caption_nll(ah, ab["audio_mask"], ids[:2, :1], mask[:2, :1])
    with pytest.raises(ValueError):
        model.get_caption_nll(ah[:1], ab["audio_mask"][:1], ids[:2], mask[:2])
    bad = ids.copy()
    bad[0, 3] = model.text_config.vocab_size
    with pytest.raises((ValueError, IndexError)):
        model.get_caption_nll(ah, ab["audio_mask"], bad[:2], mask[:2])


@pytest.mark.gpu
def test_models_without_a_decoder_refuse(tiny_state):
    from cacophony_amd import captioning
    from cacophony_amd.model import CACO
    a, t, cc, _ = _configs()
    plain = CACO(a, t, cc, device="cuda:0").load_state_dict(tiny_state)
    with pytest.raises(ValueError, match="Decoder module not initialized"):
        plain.get_caption_nll(torch.zeros(1, 8, 768), torch.ones(1, 8), torch.zeros(1, 4, dtype=torch.long), torch.ones(1, 4))
    with pytest.raises(ValueError, match="use_decoder=True"):
        captioning.score_captions(plain, {}, torch.zeros(1, 4, dtype=torch.long), torch.ones(1, 4))


@pytest.mark.gpu
def test_nll_on_another_stream_and_after_other_work(model, clips):
    """A side stream has an arena of its own; what ran in it before (the decoder's logits, a larger batch) leaves no trace.  Equal calls give
    equal bits.  Equal captions in one call have equal hidden states, but their logits' exponentials are shared out over other workgroups:
    50265 of them added up in parts of at most 197 tiles, 256 words, 8 waves and 512 pairs, each sum off by 2^-24 per addition, below 1000 * 2^-24 =
    6e-5 of the sum and so in its logarithm."""
    ab, ah = clips
    ids, mask = synth.make_captions(2, 20, model.text_config.vocab_size, start=11)
    want = model.get_caption_nll(ah, ab["audio_mask"], ids, mask)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        model.get_decoder_logits(ah, ab["audio_mask"], ids, mask)
        many = torch.as_tensor(ids).repeat(20, 1), torch.as_tensor(mask).repeat(20, 1)
        large = model.get_caption_nll(ah.repeat(20, 1, 1), ab["audio_mask"].repeat(20, 1), *many)
        got = model.get_caption_nll(ah, ab["audio_mask"], ids, mask)
    side.synchronize()
    assert torch.equal(got, want)
    assert (large[:2] - large[38:]).abs().max() < 1e-4


@pytest.mark.gpu
def test_nll_against_the_references_logits_token_by_token(model, clips):
    """The logits' bar of rel-L2 1e-2 spread over a row's V logits is 1e-2 rms(z) for each.  The errors come from bf16 roundings of operands and states, many
    and independent, so a label's is within five times that for every one of the scored tokens (5 sigma: 6e-7 of a normal distribution), the error of
    logsumexp, a mean over the words, well within the same, and the mean over n tokens within 5 / sqrt(n) of it.  What the bound is worth: likelihoods of
    other words - the label 17 words on, the token before instead of the one after, a constant - are outside it for most tokens."""
    g = load_golden("decoder_tiny.npz")
    ab, ah = clips
    nll = model.get_caption_nll(ah, ab["audio_mask"], g["ids"], g["tmask"]).cpu().double()
    z, V = torch.from_numpy(g["logits"][:, :-1]).double(), g["logits"].shape[-1]
    ids, scored = torch.as_tensor(g["ids"]).long(), torch.as_tensor(g["tmask"])[:, 1:] != 0
    lp = torch.log_softmax(z, -1)
    bound = 5e-2 * z.square().mean(-1).sqrt()

    def inside(label):
        return ((nll + lp.gather(2, label[..., None])[..., 0]).abs() <= bound)[scored]
    n = int(scored.sum())
    assert n > 40 and inside(ids[:, 1:]).all()
    err = (nll + lp.gather(2, ids[:, 1:, None])[..., 0])[scored]
    assert abs(err.mean()) <= bound[scored].mean() / n ** 0.5
    for label in ((ids[:, 1:] + 17) % V, ids[:, :-1]):
        assert inside(label).double().mean() < 0.15
    assert ((nll - float(np.log(V))).abs() <= bound)[scored].double().mean() < 0.15


def test_hidden_states_refused_without_a_model():
    lib = _lib.load()
    one = C.c_void_p(1024)
    assert lib.caco_decoder_hidden(None, one, one, one, one, 1, 1, 1, one, None) == _lib.CACO_ERR_INVALID


@pytest.fixture(scope="module")
def head(model):
    a, t, cc, d = _configs()
    state = synth.make_caco_state(a, t, cc, seed=0, decoder_cfg=d)
    get = lambda n: torch.as_tensor(np.asarray(state["decoder_module.decoder_proj." + n])).float().cuda()
    return get("weight").bfloat16(), get("bias")


@pytest.mark.gpu
@pytest.mark.parametrize("n,T", [(2, 24), (9, 1), (5, 33)])
def test_hidden_states_are_what_the_head_projects(model, clips, head, n, T):
    """The head on these states gives the decoder's logits (fp32 sums of the same products: 1e-3, as above), and the cross entropy on them the bits of
    `get_caption_nll`, which does the same inside."""
    from cacophony_amd import losses
    ab, ah = clips
    pick = torch.arange(n, device="cuda") % 2
    ah, am = ah[pick], ab["audio_mask"][pick]
    ids, mask = (torch.as_tensor(x).cuda() for x in synth.make_captions(n, T + 1, model.text_config.vocab_size, start=5))
    h = model.get_decoder_hidden_state(ah, am, ids[:, :-1], mask[:, :-1])
    assert h.shape == (n, T, 768) and h.dtype == torch.bfloat16
    w, b = head
    logits = model.get_decoder_logits(ah, am, ids[:, :-1], mask[:, :-1])
    assert (h.reshape(-1, 768).float() @ w.float().t() + b - logits.reshape(n * T, -1)).abs().max() < 1e-3
    labels = torch.where(mask[:, 1:] != 0, ids[:, 1:], -100)
    nll = losses.linear_cross_entropy(h, w, labels, b, reduction="none")
    assert torch.equal(nll, model.get_caption_nll(ah, am, ids, mask))


@pytest.mark.gpu
def test_a_head_trained_and_distilled_on_the_decoder(model, clips, head):
    """As it is used: the decoder's states, the old head's best logits as a teacher for a new one, the captions as labels; both gradients against 64 bits."""
    from cacophony_amd import losses, retrieval
    from tests.test_linear_loss import close, expect
    ab, ah = clips
    ids, mask = (torch.as_tensor(x).cuda() for x in synth.make_captions(2, 28, model.text_config.vocab_size, start=21))
    args = ah, ab["audio_mask"], ids[:, :-1], mask[:, :-1]
    h, (w, b) = model.get_decoder_hidden_state(*args), head
    idx, val = retrieval.topk(model.get_decoder_logits(*args).reshape(54, -1), 16)
    idx = torch.where((mask[:, 1:] != 0).reshape(-1, 1), idx, -1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    new = (w.float() + 0.02 * torch.randn(w.shape, generator=gen, device="cuda")).bfloat16().requires_grad_(True)
    bias = torch.zeros_like(b, requires_grad=True)
    x = dict(h=h.reshape(54, -1).cpu(), w=new.detach().cpu(), b=bias.detach().cpu())
    loss = losses.linear_topk_distillation(h, new, val.reshape(2, 27, 16), idx.reshape(2, 27, 16), bias, temperature=2.0)
    loss.backward()
    close({"loss": loss, "d_weight": new.grad, "d_bias": bias.grad}, expect(dict(x, topk=16, teacher=val.cpu(), idx=idx.cpu().long()), 2.0), "distilled")
    new.grad = bias.grad = None
    labels = torch.where(mask[:, 1:] != 0, ids[:, 1:], -100)
    loss = losses.linear_cross_entropy(h, new, labels, bias)
    loss.backward()
    close({"loss": loss, "d_weight": new.grad, "d_bias": bias.grad}, expect(dict(x, topk=0, y=labels.reshape(-1).cpu())), "trained")


@pytest.mark.gpu
def test_hidden_states_refusals(model, clips, tiny_state):
    from cacophony_amd.model import CACO
    a, t, cc, _ = _configs()
    ab, ah = clips
    ids = torch.zeros(2, 4, dtype=torch.long)
    plain = CACO(a, t, cc, device="cuda:0").load_state_dict(tiny_state)
    with pytest.raises(ValueError, match="Decoder module not initialized"):
        plain.get_decoder_hidden_state(ah, ab["audio_mask"], ids, torch.ones_like(ids))
    with pytest.raises(ValueError):
        model.get_decoder_hidden_state(ah[:1], ab["audio_mask"][:1], ids, torch.ones_like(ids))
    with pytest.raises((ValueError, IndexError)):
        model.get_decoder_hidden_state(ah, ab["audio_mask"], ids + model.text_config.vocab_size, torch.ones_like(ids))
