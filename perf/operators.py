"""Cases, inputs, plain forms and 64-bit forms of the losses of a linear vocabulary head.

Two operators of `cacophony_amd.losses`, both over logits z = hidden @ weight.T + bias that are never kept whole:

* cross entropy (`linear_cross_entropy`): per row  l = logsumexp(z) - z[label];  rows whose label is `ignore_index` do not count.
* distillation from a teacher's top logits (`linear_topk_distillation`): q = softmax(teacher / T) over the K entries a teacher
  gives for the row (an index < 0 is an absent entry),  l = T^2 * sum_k q_k * (log q_k - log softmax(z / T)[i_k]);  rows with
  no entry do not count.

`op` is "ce" or "distill"; `grad` says whether a pass also returns the gradients of the mean loss with respect to the hidden
states, the weight and the bias (a training step of the head) or the losses alone (scoring captions, measuring a student).
"""
import math

import torch

own = False

IGNORE = -100


def _case(name, op, grad, rows, vocab, dim, bias, ignored, topk=0, temperature=1.0):
    c = {"op": op, "grad": grad, "rows": rows, "vocab": vocab, "dim": dim, "bias": bias, "ignored": ignored, "topk": topk, "temperature": temperature}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the caption head (hidden 768, vocabulary 50265) on a batch of 256 captions of 32 tokens, a third of them padding
        _case("ce-train-256x32", "ce", True, 8192, 50265, 768, True, 0.33),
        # a short batch with an odd number of tokens, no padding and no bias
        _case("ce-train-odd", "ce", True, 1187, 50265, 768, False, 0.0),
        # a wide head with a large vocabulary: the largest matrices
        _case("ce-train-wide", "ce", True, 2048, 131072, 4096, False, 0.1),
        # a toy head, as in the tests of a training loop: launches count, not bytes
        _case("ce-train-small", "ce", True, 37, 1003, 128, True, 0.2),
        # log-likelihoods of 256 candidate captions: losses alone
        _case("ce-score-256x32", "ce", False, 8192, 50265, 768, True, 0.33),
        # the likelihood of one next token: the weights are read once for one row
        _case("ce-score-1", "ce", False, 1, 50265, 768, True, 0.0),
        # one clip's eight candidate captions
        _case("ce-score-8x31", "ce", False, 248, 50265, 768, True, 0.4),
        # a student's step on a teacher's 32 best tokens for every token of a full batch
        _case("distill-train-256x32", "distill", True, 8192, 50265, 768, True, 0.33, 32, 2.0),
        # a narrow student, a deep list of teacher tokens, a ragged vocabulary
        _case("distill-train-k100", "distill", True, 1000, 32007, 520, False, 0.0, 100, 1.0),
        # one short caption on a small head
        _case("distill-train-small", "distill", True, 19, 777, 64, True, 0.1, 5, 4.0),
        # how far a student is from its teacher on a validation batch
        _case("distill-score-64x32", "distill", False, 2048, 50265, 768, True, 0.33, 64, 1.5),
        # one token of a decoding student
        _case("distill-score-1", "distill", False, 1, 50265, 768, True, 0.0, 10, 2.0),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    largest = 2048 * 131072 * 4096
    while True:
        rows = _log_between(rng, 1, 8192)
        vocab = _log_between(rng, 300, 131072)
        dim = 8 * _log_between(rng, 8, 512)
        if rows * vocab * dim <= largest:
            break
    distill = rng.random() < 0.5
    return _case(None, "distill" if distill else "ce", rng.random() < 0.6, rows, vocab, dim, rng.random() < 0.6, rng.choice([0.0, 0.1, 0.33, 0.6]),
                 _log_between(rng, 1, 128) if distill else 0, rng.choice([1.0, 1.5, 2.0, 4.0]) if distill else 1.0)


def _counted(case):
    """Rows that count: the first one always does."""
    return case["rows"] - min(int(case["ignored"] * case["rows"]), case["rows"] - 1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    R, V, D, K = case["rows"], case["vocab"], case["dim"], case["topk"]
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev)
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)
    std = 1.5 / math.sqrt(D)                       # logits spread over +-5, as a trained head's do
    weight = torch.empty(V, D, dtype=torch.bfloat16, device=dev)
    for i in range(0, V, 16384):
        weight[i:i + 16384] = randn(min(16384, V - i), D) * std
    labels = torch.randint(0, V, (R,), generator=gen, device=dev)
    # layer-normed states that lean towards their token: its logit is raised by up to 12
    lean = rand(R, 1) * 12.0 / (D * std * std)
    hidden = (randn(R, D) + lean * weight[labels].float()).to(torch.bfloat16)
    bias = randn(V) * 0.3 if case["bias"] else None
    order = torch.argsort(rand(R - 1)) + 1         # which rows are padding
    padding = order[:R - _counted(case)]
    state = {"case": case, "hidden": hidden, "weight": weight, "bias": bias}
    if case["op"] == "ce":
        labels[padding] = IGNORE
        state["labels"] = labels
    else:
        # K distinct tokens per row, the first one the label; logits in falling order, as a teacher's top-k comes
        step = 1 + (rand(R, 1) * (max(1, (V - 1) // K) - 1)).long()
        k = torch.arange(K, device=dev)
        indices = (labels[:, None] + k * step) % V
        logits = 12.0 - torch.cumsum(rand(R, K) * (24.0 / (K + 2)), dim=1)
        indices[padding] = -1
        state["indices"], state["teacher"] = indices, logits
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from cacophony_amd import losses
    c = state["case"]
    h, w, b = state["hidden"], state["weight"], state["bias"]
    if c["op"] == "ce":
        if not c["grad"]:
            return losses.linear_cross_entropy(h, w, state["labels"], b, ignore_index=IGNORE, reduction="none")
        out = losses.linear_cross_entropy_with_grad(h, w, state["labels"], b, ignore_index=IGNORE, reduction="mean")
    else:
        if not c["grad"]:
            return losses.linear_topk_distillation(h, w, state["teacher"], state["indices"], b, temperature=c["temperature"], reduction="none")
        out = losses.linear_topk_distillation_with_grad(h, w, state["teacher"], state["indices"], b, temperature=c["temperature"], reduction="mean")
    got = [out.loss, out.row_loss, out.d_hidden, out.d_weight]
    return got + [out.d_bias] if b is not None else got


def _plain(state):
    c, w, b = state["case"], state["weight"].float(), state["bias"]
    h = state["hidden"].float()
    T = c["temperature"]
    z = h @ w.t()
    if b is not None:
        z += b
    if T != 1.0:
        z /= T
    z -= z.max(dim=1, keepdim=True).values
    lse = z.exp().sum(dim=1, keepdim=True).log()
    z -= lse                                                   # log-probabilities
    if c["op"] == "ce":
        counts = state["labels"] != IGNORE
        at = torch.where(counts, state["labels"], torch.zeros_like(state["labels"]))[:, None]
        q = counts[:, None].float()
        row = -z.gather(1, at)[:, 0]
    else:
        there = state["indices"] >= 0
        counts = there.any(dim=1)
        at = torch.where(there, state["indices"], torch.zeros_like(state["indices"]))
        t = torch.where(there, state["teacher"] / T, torch.full_like(state["teacher"], -math.inf))
        t = t - torch.where(counts, t.max(dim=1).values, torch.zeros_like(t[:, 0]))[:, None]
        e = t.exp()
        q = e / e.sum(dim=1, keepdim=True).clamp_min(1e-30)
        row = T * T * torch.where(q > 0, q * (q.clamp_min(1e-38).log() - z.gather(1, at)), torch.zeros_like(q)).sum(dim=1)
    row = torch.where(counts, row, torch.zeros_like(row))
    if not c["grad"]:
        return row
    n = counts.sum()
    loss = row.sum() / n
    g = counts.float() * (T / n)                               # T^2 of the loss, 1 / T of the logits' scale
    z.exp_()                                                   # probabilities
    z.scatter_add_(1, at, -q)
    z *= g[:, None]                                            # gradient of the logits
    got = [loss, row, (z @ w).to(torch.bfloat16), (z.t() @ h).to(torch.bfloat16)]
    return got + [z.sum(dim=0)] if b is not None else got


def work(case):
    R, V, D, K = _counted(case), case["vocab"], case["dim"], case["topk"]
    bias = 4 * V if case["bias"] else 0
    read = 2 * R * D + 2 * V * D + bias + case["rows"] * (8 if case["op"] == "ce" else 12 * K)
    write = 4 * case["rows"]
    flops = 2 * R * V * D
    if case["grad"]:
        write += 2 * case["rows"] * D + 2 * V * D + bias
        flops *= 3
    return {"bytes": read + write, "flops": flops}


def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    T, K = case["temperature"], case["topk"]
    W = s["weight"].double()
    H = s["hidden"].double()
    R, V = H.shape[0], W.shape[0]
    row = torch.zeros(R, dtype=torch.float64, device=H.device)
    dh, dw = torch.zeros_like(H), torch.zeros_like(W) if case["grad"] else None
    db = torch.zeros(V, dtype=torch.float64, device=H.device)
    n = float(_counted(case))
    for i in range(0, R, 1024):
        x = H[i:i + 1024]
        logits = torch.matmul(x, W.T)
        if s["bias"] is not None:
            logits = logits + s["bias"].double()
        target = torch.zeros_like(logits)
        r = torch.arange(x.shape[0], device=x.device)
        if case["op"] == "ce":
            y = s["labels"][i:i + 1024]
            alive = y >= 0
            target[r[alive], y[alive]] = 1.0
        else:
            t = s["teacher"][i:i + 1024].double()
            idx = s["indices"][i:i + 1024]
            alive = idx[:, 0] >= 0
            q = torch.softmax(t / T, dim=1) * alive[:, None]
            for k in range(K):
                target[r, idx[:, k].clamp_min(0)] += q[:, k]
        logp = torch.log_softmax(logits / T, dim=1)
        del logits
        kl = torch.special.xlogy(target, target) - target * logp
        row[i:i + 1024] = T * T * kl.sum(dim=1) * alive
        del kl
        if case["grad"]:
            dz = (logp.exp() - target) * (alive.double() * (T / n))[:, None]
            dh[i:i + 1024] = dz @ W
            dw += dz.T @ x
            db += dz.sum(dim=0)
    if not case["grad"]:
        return row
    got = [row.sum() / n, row, dh, dw]
    return got + [db] if s["bias"] is not None else got
