"""The operators of a language model's training step and scoring request whose speed is tracked, each with its plain form.

`linear_act`            y = residual + dropout(act(x . w^T + bias)), with its gradients
`dropout`               y = residual + dropout(x), the mask drawn from a counter and never stored, with its gradient
`linear_cross_entropy`  softmax cross-entropy of x . w^T over a large vocabulary without the logits, with its gradients

The random mask is part of the operators' definition, so that both forms drop the same elements: element i of the flattened
output takes 16 bits of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) at counter (i / 8, step, site) under the key `seed`,
and is kept where they are at least round(65536 p).
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100   # targets that do not count
HIDDEN, FFN, VOCAB = 1024, 4096, 32000   # the decoder of the language clients; BERT: hidden 768, projection 2304, vocabulary 30522


def _linear(train, tokens, k, n, act="none", residual=False, p=0.0):
    return {"op": "linear", "train": train, "tokens": tokens, "k": k, "n": n, "act": act, "residual": residual, "p": p}


def _dropout(tokens, n, p, dtype, residual):
    return {"op": "dropout", "train": True, "tokens": tokens, "n": n, "p": p, "dtype": dtype, "residual": residual}


def _loss(train, tokens, vocab, hidden, ignored):
    return {"op": "loss", "train": train, "tokens": tokens, "vocab": vocab, "hidden": hidden, "ignored": ignored}


def listed():
    return [
        # one new token through the feed-forward block of the decoder: latency
        dict(_linear(False, 1, HIDDEN, FFN, "gelu"), name="linear_1_up_gelu"),
        # sixteen sequences, a token each, on the way back down to the residual stream
        dict(_linear(False, 16, FFN, HIDDEN, "none", True), name="linear_16_down_residual"),
        # one short question of BERT, the attention's output projection
        dict(_linear(False, 77, 768, 768, "none", True), name="linear_77_out_residual"),
        # a batch of full-length sequences, scored: the widest layer of the request
        dict(_linear(False, 16 * 512, HIDDEN, FFN, "gelu"), name="linear_8192_up_gelu"),
        # the same layer in the training step
        dict(_linear(True, 16 * 512, HIDDEN, FFN, "gelu"), name="linear_train_8192_up_gelu"),
        # a small ragged training batch, a residual branch with dropout
        dict(_linear(True, 3 * 200, FFN, HIDDEN, "none", True, 0.1), name="linear_train_600_down_dropout"),
        # embeddings of one short question in float32
        dict(_dropout(77, 768, 0.1, "float32", False), name="dropout_77_f32"),
        # a feed-forward activation of a full batch, added to a stream
        dict(_dropout(16 * 512, FFN, 0.1, "bfloat16", True), name="dropout_8192_residual"),
        # log-likelihood of the last token of sixteen sequences
        dict(_loss(False, 16, VOCAB, HIDDEN, 0.0), name="score_16"),
        # log-likelihoods of a batch of full-length sequences, some of them padded
        dict(_loss(False, 16 * 512, VOCAB, HIDDEN, 0.2), name="score_8192"),
        # the loss of the decoder's training step
        dict(_loss(True, 16 * 512, VOCAB, HIDDEN, 0.0), name="loss_train_8192"),
        # masked-language-model loss of three padded sequences: a vocabulary that divides nothing, most positions not asked for
        dict(_loss(True, 3 * 381, 30522, 768, 0.85), name="loss_train_1143_odd"),
    ]


def _between(rng, low, high):
    """A whole number from low to high, uniform over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "train", "train", "dropout", "score", "loss"))
    if kind in ("linear", "train"):
        # widths in multiples of 8 for the reduction; any for the output
        tokens, k, n = _between(rng, 1, 8192), 8 * _between(rng, 8, 512), _between(rng, 64, 4096)
        if rng.random() < 0.7:
            n = (n + 7) // 8 * 8
        act, residual = rng.choice(("none", "relu", "gelu")), rng.random() < 0.5
        return _linear(kind == "train", tokens, k, n, act, residual, rng.choice((0.0, 0.0, 0.1, 0.25)))
    if kind == "dropout":
        return _dropout(_between(rng, 1, 8192), _between(rng, 64, 4096), round(rng.uniform(0.02, 0.6), 3), rng.choice(("float32", "bfloat16")),
                        rng.random() < 0.5)
    vocab = _between(rng, 500, 32000)
    return _loss(kind == "loss", _between(rng, 1, 8192), vocab, 8 * _between(rng, 8, 128), rng.choice((0.0, 0.1, 0.85)))


def _randn(gen, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = case["tokens"]
    state = dict(case)
    if case["op"] == "loss":
        h, v = case["hidden"], case["vocab"]
        # logits of a spread of about 2, the right token ahead of the others in half of the rows
        state["w"] = _randn(gen, v, h, scale=2.0 / math.sqrt(h))
        target = torch.randint(0, v, (t,), device="cuda", generator=gen)
        sure = torch.rand(t, 1, device="cuda", generator=gen) < 0.5
        state["x"] = (torch.randn(t, h, device="cuda", generator=gen) + sure * 1.5 * state["w"][target].float()).to(torch.bfloat16)
        state["target"] = torch.where(torch.rand(t, device="cuda", generator=gen) < case["ignored"], IGNORE, target)
        state["leaves"] = ["x", "w"]
    else:
        n = case["n"]
        state["rng"] = torch.tensor([seed * 0x5DEECE66D % (1 << 62), 1000 + seed % 1000], dtype=torch.int64, device="cuda")
        state["site"] = 3
        dtype = torch.bfloat16
        if case["op"] == "linear":
            k = case["k"]
            state["x"], state["w"] = _randn(gen, t, k), _randn(gen, n, k, scale=1.0 / math.sqrt(k))
            state["bias"] = _randn(gen, n, scale=0.1)
            state["leaves"] = ["x", "w", "bias"]
        else:
            dtype = getattr(torch, case["dtype"])
            state["x"] = _randn(gen, t, n, dtype=dtype)
            state["leaves"] = ["x"]
        state["residual"] = _randn(gen, t, n, dtype=dtype) if case["residual"] else None
        if case["residual"]:
            state["leaves"] = state["leaves"] + ["residual"]
        if case["train"]:
            state["dy"] = _randn(gen, t, n, dtype=dtype)
    for name in state["leaves"] if case["train"] else ():
        state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------------------ the framework's
def _own(state):
    from orion_b200 import torch_ops
    ops = torch_ops.load()
    leaves = [state[name] for name in state["leaves"]]
    with torch.set_grad_enabled(state["train"]):
        if state["op"] == "loss":
            if not state["train"]:
                return ops.linear_cross_entropy(state["x"], state["w"], state["target"], IGNORE, "none")
            y, dy = ops.linear_cross_entropy(state["x"], state["w"], state["target"], IGNORE, "mean"), None
        elif state["op"] == "linear":
            y = ops.linear_act(state["x"], state["w"], state["bias"], state["residual"], state["act"], state["p"], state["rng"], state["site"])
            if not state["train"]:
                return y
            dy = state["dy"]
        else:
            y, dy = ops.dropout(state["x"], state["p"], state["rng"], state["site"], state["residual"]), state["dy"]
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))


# ------------------------------------------------------------------------------------------------------------ plain forms
def _philox(c, k):
    """Ten rounds on counters c (four int64 tensors holding 32-bit words) under the key k (two of them)."""
    low = 0xFFFFFFFF
    for r in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # the low 64 bits of the product, as a signed number
        k0, k1 = k[0] + r * 0x9E3779B9 & low, k[1] + r * 0xBB67AE85 & low
        c = [p1 >> 32 & low ^ c[1] ^ k0, p1 & low, p0 >> 32 & low ^ c[3] ^ k1, p0 & low]
    return c


def _keep(shape, p, rng, site):
    """The mask of an output of this shape, and what the elements that are kept are multiplied by."""
    n, threshold = math.prod(shape), min(65536, int(p * 65536 + 0.5))
    group = torch.arange((n + 7) // 8, device="cuda")
    low, step = 0xFFFFFFFF, rng[1]
    c = [group & low, group >> 32 & 0xFFFF | (step >> 32 & 0xFFFF) << 16, (step & low).expand_as(group), torch.full_like(group, site)]
    words = torch.stack(_philox(c, [rng[0] & low, rng[0] >> 32 & low]), 1)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).flatten()[:n]
    return (halves >= threshold).view(shape), 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0


def _drop(a, keep, scale):
    return torch.where(keep, a * scale, 0.0)


def _plain_linear(state):
    x, w, bias = (state[n].detach().float() for n in ("x", "w", "bias"))
    z = x @ w.T + bias
    act = state["act"]
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) if act == "gelu" else None
    y = z * cdf if act == "gelu" else z.clamp(min=0.0) if act == "relu" else z
    if state["p"] > 0.0:
        keep, scale = _keep(y.shape, state["p"], state["rng"], state["site"])
        y = _drop(y, keep, scale)
    if state["residual"] is not None:
        y = y + state["residual"].detach().float()
    y = y.to(torch.bfloat16)
    if not state["train"]:
        return y
    dz = state["dy"].float()
    if state["p"] > 0.0:
        dz = _drop(dz, keep, scale)
    if act == "gelu":
        dz = dz * (cdf + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi))
    elif act == "relu":
        dz = torch.where(z > 0.0, dz, 0.0)
    out = [y] + [g.to(torch.bfloat16) for g in (dz @ w, dz.T @ x, dz.sum(0))]
    return out + [state["dy"]] if state["residual"] is not None else out


def _plain_dropout(state):
    x, dtype = state["x"].detach(), state["x"].dtype
    keep, scale = _keep(x.shape, state["p"], state["rng"], state["site"])
    y = _drop(x.float(), keep, scale)
    if state["residual"] is not None:
        y = y + state["residual"].detach().float()
    out = [y.to(dtype), _drop(state["dy"].float(), keep, scale).to(dtype)]
    return out + [state["dy"]] if state["residual"] is not None else out


def _plain_loss(state):
    target = state["target"]
    counts = target != IGNORE
    x, w = torch.where(counts[:, None], state["x"].detach().float(), 0.0), state["w"].detach().float()
    logits = x @ w.T
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    at = target.clamp(min=0)[:, None]
    loss = torch.where(counts, (top + torch.log(total) - logits.gather(1, at))[:, 0], 0.0)
    if not state["train"]:
        return loss
    number = counts.sum().clamp(min=1)
    d = e / total
    d.scatter_add_(1, at, torch.full_like(top, -1.0))
    d = torch.where(counts[:, None], d / number, 0.0)
    return [loss.sum() / number, (d @ w).to(torch.bfloat16), (d.T @ x).to(torch.bfloat16)]


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "dropout": _plain_dropout, "loss": _plain_loss}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    t, train = case["tokens"], case["train"]
    if case["op"] == "loss":
        v, h = case["vocab"], case["hidden"]
        both = 2.0 * (t * h + v * h)   # hidden rows and weights, or their gradients
        return {"bytes": both * (2 if train else 1) + 8.0 * t + (4.0 if train else 4.0 * t), "flops": (6.0 if train else 2.0) * t * v * h}
    n = case["n"]
    out, res = t * n, t * n if case["residual"] else 0
    if case["op"] == "dropout":
        size = 4.0 if case["dtype"] == "float32" else 2.0
        return {"bytes": size * (4 * out + res), "flops": 2.0 * (2 * out + res)}
    k = case["k"]
    both = t * k + n * k + n
    if not train:
        return {"bytes": 2.0 * (both + out + res), "flops": 2.0 * t * n * k}
    return {"bytes": 2.0 * (2 * both + 2 * out + res), "flops": 6.0 * t * n * k}   # dy is read, and is the residual's gradient


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_keep(shape, p, seed, step, site):
    """The mask once more, on the host in unsigned arithmetic."""
    n = int(np.prod(shape))
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    u32, low = np.uint64(32), np.uint64(0xFFFFFFFF)
    w = [g & low, (g >> u32) | np.uint64((step >> 32 & 0xFFFF) << 16), np.full_like(g, step & 0xFFFFFFFF), np.full_like(g, site)]
    key0, key1 = seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF
    for _ in range(10):
        a, b = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(b >> u32) ^ w[1] ^ np.uint64(key0), b & low, (a >> u32) ^ w[3] ^ np.uint64(key1), a & low]
        key0, key1 = (key0 + 0x9E3779B9) & 0xFFFFFFFF, (key1 + 0xBB67AE85) & 0xFFFFFFFF
    bits = np.stack(w, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    limit = min(65536, int(p * 65536 + 0.5))
    factor = 65536.0 / (65536 - limit) if limit < 65536 else 0.0
    return torch.from_numpy((bits.astype(np.int64) >= limit).reshape(shape)).cuda().double() * factor


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        counts = s["target"] != IGNORE
        x, w = s["x"].detach().double()[counts], s["w"].detach().double()
        label = s["target"][counts]
        logits = x @ w.T
        lse = torch.logsumexp(logits, 1)
        rows = torch.zeros(case["tokens"], dtype=torch.float64, device="cuda")
        rows[counts] = lse - logits[torch.arange(len(label), device="cuda"), label]
        if not case["train"]:
            return rows
        number = max(1, len(label))
        prob = logits.sub_(lse[:, None]).exp_()
        prob[torch.arange(len(label), device="cuda"), label] -= 1.0
        prob /= number
        dx = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        dx[counts] = prob @ w
        return [rows.sum() / number, dx, prob.T @ x]
    rng = [int(v) for v in s["rng"].cpu()]
    factor = _exact_keep((case["tokens"], case["n"]), case["p"], rng[0], rng[1], s["site"]) if case["p"] > 0.0 else 1.0
    res = s["residual"].detach().double() if case["residual"] else 0.0
    x = s["x"].detach().double()
    if case["op"] == "dropout":
        out = [x * factor + res, s["dy"].double() * factor]
    else:
        w, b = s["w"].detach().double().requires_grad_(True), s["bias"].detach().double().requires_grad_(True)
        x.requires_grad_(True)
        z = torch.addmm(b, x, w.T)
        a = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[case["act"]](z)
        y = a * factor + res
        if not case["train"]:
            return y.detach()
        out = [y.detach()] + list(torch.autograd.grad(y, (x, w, b), s["dy"].double()))
    return out + [s["dy"].double()] if case["residual"] else out
