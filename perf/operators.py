"""The products of a model that stay in bf16, as training, evaluation and rollout call them: a linear layer with bias, activation, gate
and residual in its epilogue, the cross entropy of the head over the whole vocabulary, and the log-probabilities of sampled tokens.

Sizes are those of the repository's decoder configurations (hidden 1536 and 3584, feed-forward 8960 and 18944, vocabulary 151936 and
152064), of its small test model (hidden 64, vocabulary 97), and odd ones between them."""
import math

import torch

own = False
DEV = torch.device("cuda", 0)


# ---- the cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # Decode of one sequence: the down projection of the larger decoder onto its residual stream.
        dict(name="linear_decode_1_down", kind="linear", tokens=1, k=18944, n=3584, act="none", bias=False, gate=False, residual=True, backward=False),
        # Decode of 16 sequences: an attention projection of the smaller decoder, with its bias.
        dict(name="linear_decode_16_qkv", kind="linear", tokens=16, k=1536, n=1536, act="none", bias=True, gate=False, residual=False, backward=False),
        # Decode of 64 sequences: the gate projection of the larger decoder, silu and the product with `up` behind it.
        dict(name="linear_decode_64_gate", kind="linear", tokens=64, k=3584, n=18944, act="silu", bias=False, gate=True, residual=False, backward=False),
        # A layer of no round size: ragged tokens, odd width, every part of the epilogue.
        dict(name="linear_odd_gelu", kind="linear", tokens=333, k=520, n=1003, act="gelu", bias=True, gate=False, residual=True, backward=True),
        # Prefill: the down projection of the smaller decoder on 16384 tokens.
        dict(name="linear_prefill_16k_down", kind="linear", tokens=16384, k=8960, n=1536, act="none", bias=False, gate=False, residual=True, backward=False),
        # A training step of the gate projection: forward and backward on 8192 tokens.
        dict(name="linear_train_8k_gate", kind="linear", tokens=8192, k=1536, n=8960, act="silu", bias=False, gate=True, residual=False, backward=True),
        # The loss of a small model, where launches are all that counts.
        dict(name="ce_tiny", kind="ce", tokens=24, k=64, vocab=97, reduction="mean", ignored=0.2, backward=True),
        # Evaluation: the loss of 4096 tokens, no gradient.
        dict(name="ce_eval_4k", kind="ce", tokens=4096, k=1536, vocab=151936, reduction="mean", ignored=0.1, backward=False),
        # A training step of the head: loss and both gradients of 8192 tokens, a third of them prompt.
        dict(name="ce_train_8k", kind="ce", tokens=8192, k=1536, vocab=151936, reduction="mean", ignored=0.33, backward=True),
        # A ragged batch over an odd vocabulary, losses summed.
        dict(name="ce_odd", kind="ce", tokens=1021, k=1000, vocab=32003, reduction="sum", ignored=0.1, backward=True),
        # Rollout: log-probabilities and entropies of the tokens that 16 sequences have just sampled.
        dict(name="logprobs_decode_16", kind="logprobs", tokens=16, k=3584, vocab=152064, temperature=1.0, entropy=True, backward=False),
        # Policy update: log-probabilities of 2048 sampled tokens at the sampling temperature, with a gradient for each.
        dict(name="logprobs_grpo_2k", kind="logprobs", tokens=2048, k=1536, vocab=151936, temperature=0.7, entropy=True, backward=True),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


MOST_FLOPS = 6 * 8192 * 1536 * 151936      # of the largest listed case


def draw(rng):
    kind = rng.choice(["linear", "linear", "ce", "logprobs"])
    backward = rng.random() < 0.5
    tokens = _log(rng, 1, 128) if rng.random() < 0.4 else _log(rng, 128, 16384)
    if kind == "linear":
        c = dict(kind=kind, tokens=tokens, k=_log(rng, 64, 18944, 8), n=_log(rng, 33, 18944), act=rng.choice(["none", "silu", "gelu", "gelu_tanh"]),
                 bias=rng.random() < 0.5, gate=rng.random() < 0.4, residual=rng.random() < 0.4, backward=backward)
        most, width = MOST_FLOPS // 4, "n"
    else:
        c = dict(kind=kind, tokens=tokens, k=_log(rng, 64, 3584, 8), vocab=_log(rng, 97, 152064))
        if kind == "ce":
            c.update(reduction=rng.choice(["mean", "sum", "none"]), ignored=rng.choice([0.0, 0.1, 0.5]), backward=backward)
        else:
            c.update(temperature=rng.choice([0.6, 1.0, 1.3]), entropy=rng.random() < 0.5, backward=backward)
        most, width = MOST_FLOPS, "vocab"
    while (6 if backward else 2) * c["tokens"] * c["k"] * c[width] > most:
        c["tokens"] = c["tokens"] // 2 + 1
    return c


# ---- what a program has in hand -----------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=DEV, generator=gen) * scale

    m, k = case["tokens"], case["k"]
    s = dict(case=case)
    if case["kind"] == "linear":
        n = case["n"]
        x = normal(m, k)
        x[:, ::97] *= 8                                     # the few large channels of a hidden state
        s["x"] = x.bfloat16()
        s["weight"] = normal(n, k, scale=0.02).bfloat16()
        s["bias"] = normal(n, scale=0.1).bfloat16() if case["bias"] else None
        s["gate"] = normal(m, n).bfloat16() if case["gate"] else None
        s["residual"] = normal(m, n).bfloat16() if case["residual"] else None
        s["leaves"] = [name for name in ("x", "weight", "bias", "gate", "residual") if s[name] is not None]
        if case["backward"]:
            s["dy"] = normal(m, n, scale=0.1).bfloat16()
    else:
        v = case["vocab"]
        weight = normal(v, k, scale=0.8 / math.sqrt(k))
        target = torch.randint(0, v, (m,), device=DEV, generator=gen)
        # hidden states that lean towards their token, some further than others
        lean = 12.0 * torch.rand(m, 1, device=DEV, generator=gen)
        rows = weight[target]
        s["x"] = (normal(m, k) + lean * rows / rows.norm(dim=1, keepdim=True)).bfloat16()
        s["weight"] = weight.bfloat16()
        if case["kind"] == "ce":
            target = torch.where(torch.rand(m, device=DEV, generator=gen) < case["ignored"], torch.full_like(target, -100), target)
            target[0] = 0                                   # (a batch with nothing to learn has no mean)
            if case["backward"]:
                s["dy"] = normal(m) if case["reduction"] == "none" else torch.ones((), device=DEV)
        elif case["backward"]:
            s["dy"] = normal(m)                             # advantages
        s["target"] = target
        s["leaves"] = ["x", "weight"]
    if case["backward"]:
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from fp4_post_b200 import dense
    c = s["case"]
    if not c["backward"]:
        with torch.no_grad():
            return _call(dense, s, c)
    out = _call(dense, s, c)
    first, rest = (out[0], tuple(out[1:])) if isinstance(out, tuple) else (out, ())
    return (first.detach(), *rest, *torch.autograd.grad(first, [s[name] for name in s["leaves"]], s["dy"]))


def _call(dense, s, c):
    if c["kind"] == "linear":
        return dense.linear(s["x"], s["weight"], s["bias"], activation=None if c["act"] == "none" else c["act"], gate=s["gate"], residual=s["residual"])
    if c["kind"] == "ce":
        return dense.linear_cross_entropy(s["x"], s["weight"], s["target"], reduction=c["reduction"])
    return dense.token_logprobs(s["x"], s["weight"], s["target"], temperature=c["temperature"], entropy=c["entropy"])


def _activation(name, z):
    """act(z) and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    t = torch.tanh(u)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def _plain(s):
    c = s["case"]
    with torch.no_grad():
        return _plain_linear(s, c) if c["kind"] == "linear" else _plain_head(s, c)


def _plain_linear(s, c):
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    a, slope = _activation(c["act"], z)
    y = a
    if s["gate"] is not None:
        y = y * s["gate"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.bfloat16()
    if not c["backward"]:
        return y
    dy = s["dy"].float()
    dz = dy * slope
    if s["gate"] is not None:
        dz = dz * s["gate"].float()
    out = [y, (dz @ w).bfloat16(), (dz.t() @ x).bfloat16()]
    if s["bias"] is not None:
        out.append(dz.sum(dim=0).bfloat16())
    if s["gate"] is not None:
        out.append((dy * a).bfloat16())
    if s["residual"] is not None:
        out.append(s["dy"].clone())
    return tuple(out)


def _plain_head(s, c):
    x, w, target = s["x"].float(), s["weight"].float(), s["target"]
    scale = 1.0 / c.get("temperature", 1.0)
    logits = (x @ w.t()) * scale
    top = logits.max(dim=1, keepdim=True).values
    lse = (logits - top).exp().sum(dim=1, keepdim=True).log() + top
    live = target >= 0
    at = target.clamp(min=0)
    rows = torch.arange(target.numel(), device=target.device)
    nll = torch.where(live, lse[:, 0] - logits[rows, at], torch.zeros_like(lse[:, 0]))
    p = (logits - lse).exp_()
    if c["kind"] == "ce":
        count = live.sum()
        out = [nll if c["reduction"] == "none" else nll.sum() if c["reduction"] == "sum" else nll.sum() / count]
        if c["backward"]:
            g = s["dy"].expand_as(nll) if c["reduction"] != "mean" else (s["dy"] / count).expand_as(nll)
    else:
        out = [-nll]
        if c["entropy"]:
            out.append(lse[:, 0] - (p * logits).sum(dim=1))
        if c["backward"]:
            g = -s["dy"]
    if c["backward"]:
        del logits
        p[rows, at] -= 1
        p *= (torch.where(live, g, torch.zeros_like(g)) * scale)[:, None]
        out += [(p @ w).bfloat16(), (p.t() @ x).bfloat16()]
    return tuple(out) if len(out) > 1 else out[0]


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_linear(s, case) if case["kind"] == "linear" else _exact_head(s, case)


def _exact_linear(s, c):
    """By pieces of the output's columns."""
    x = s["x"].double()
    m, n = x.shape[0], s["weight"].shape[0]
    y = torch.empty(m, n, dtype=torch.float64, device=DEV)
    dx = torch.zeros_like(x) if c["backward"] else None
    dw, db, dgate = [], [], []
    for j in range(0, n, 4096):
        cols = slice(j, min(n, j + 4096))
        w = s["weight"][cols].double()
        z = torch.mm(x, w.t())
        if c["bias"]:
            z += s["bias"][cols].double()
        if c["act"] == "silu":
            phi = torch.sigmoid(z)
            slope = phi + z * phi * torch.sigmoid(-z)
        elif c["act"] == "gelu":
            phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
            slope = phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif c["act"] == "gelu_tanh":
            # (1 + tanh u) / 2 = sigmoid(2 u)
            u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
            phi = torch.sigmoid(u2)
            slope = phi + z * phi * torch.sigmoid(-u2) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
        else:
            phi, slope = torch.ones_like(z), torch.ones_like(z)
        act = z * phi
        gate = s["gate"][:, cols].double() if c["gate"] else 1.0
        y[:, cols] = act * gate + (s["residual"][:, cols].double() if c["residual"] else 0.0)
        if c["backward"]:
            dy = s["dy"][:, cols].double()
            dz = dy * gate * slope
            dx += torch.mm(dz, w)
            dw.append(torch.mm(dz.t(), x))
            db.append(dz.sum(dim=0))
            dgate.append(dy * act)
    if not c["backward"]:
        return y
    out = [y, dx, torch.cat(dw)]
    if c["bias"]:
        out.append(torch.cat(db))
    if c["gate"]:
        out.append(torch.cat(dgate, dim=1))
    if c["residual"]:
        out.append(s["dy"].double())
    return tuple(out)


def _exact_head(s, c):
    """By pieces of the tokens."""
    w = s["weight"].double()
    m = s["x"].shape[0]
    t = c.get("temperature", 1.0)
    live = s["target"] != -100
    weight_of = torch.ones(m, dtype=torch.float64, device=DEV)
    if c["kind"] == "ce" and c["reduction"] == "mean":
        weight_of /= live.sum().double()
    nll = torch.empty(m, dtype=torch.float64, device=DEV)
    entropy = torch.empty_like(nll)
    dx, dw = [], torch.zeros_like(w) if c["backward"] else None
    for i in range(0, m, 1024):
        rows = slice(i, min(m, i + 1024))
        x = s["x"][rows].double()
        logp = torch.log_softmax(torch.mm(x, w.t()) / t, dim=1)
        on = live[rows]
        pick = torch.where(on, s["target"][rows], 0)[:, None]
        nll[rows] = torch.where(on, -logp.gather(1, pick)[:, 0], 0.0)
        p = logp.exp()
        entropy[rows] = -(p * logp).sum(dim=1)
        if c["backward"]:
            dy = s["dy"].double()
            up = (dy[rows] if dy.dim() else dy) * weight_of[rows] * (1.0 if c["kind"] == "ce" else -1.0)
            p.scatter_add_(1, pick, torch.full_like(p[:, :1], -1.0))
            p *= torch.where(on, up, 0.0)[:, None] / t
            dx.append(torch.mm(p, w))
            dw += torch.mm(p.t(), x)
    if c["kind"] == "ce":
        out = [nll if c["reduction"] == "none" else (nll * weight_of).sum()]
    else:
        out = [-nll] + ([entropy] if c["entropy"] else [])
    if c["backward"]:
        out += [torch.cat(dx), dw]
    return tuple(out) if len(out) > 1 else out[0]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    m, k = case["tokens"], case["k"]
    if case["kind"] == "linear":
        n = case["n"]
        elements = case["gate"] + case["residual"] + 1                   # of [tokens, n]: read or written once
        moved = m * k + n * k + n * case["bias"] + m * n * elements
        flops = 2 * m * n * k
        if case["backward"]:
            moved += m * k + n * k + n * case["bias"] + m * n * (1 + case["gate"] + case["residual"])
            flops *= 3
        return {"bytes": 2 * moved, "flops": flops}
    v = case["vocab"]
    moved = 2 * (m * k + v * k) + 8 * m + 4 * m * (1 + case.get("entropy", False))
    if case["backward"]:
        moved += 2 * (m * k + v * k) + 4 * m
    return {"bytes": moved, "flops": (6 if case["backward"] else 2) * m * v * k}
