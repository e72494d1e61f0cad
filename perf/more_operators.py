"""What a rollout takes besides the projections: rotary positions, appending to a paged key-value cache, attention of one new token over it, the pages'
own bookkeeping (a prompt forked for its group's answers, a cache compacted), and sampling.

Sizes are those of the repository's decoder configurations (12 heads on 2 and 28 on 4 key-value heads of 128, 28 layers, vocabulary 151936 and 152064), of
its small test model (vocabulary 97), and odd ones between them."""
import math
import random

import torch

own = False
DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
ORIGINAL = 8192            # positions that a scaled model was trained on


# ---- the cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # A training step of the larger decoder: queries and keys of 4 sequences of 2048, with gradients.
        dict(name="rotary_train_8k", kind="rotary", batch=4, tokens=2048, heads=28, kv_heads=4, head_dim=128, rotary_dim=128, interleaved=False, scaling="none",
             theta=1e6, start=0, dtype="bf16", backward=True),
        # A part of an odd head in neighbouring pairs, far out in a context stretched by yarn, in fp32.
        dict(name="rotary_partial_far", kind="rotary", batch=3, tokens=333, heads=10, kv_heads=5, head_dim=80, rotary_dim=44, interleaved=True, scaling="yarn",
             theta=1e4, start=200000, dtype="fp32", backward=True),
        # Decode of 64 sequences: the new token's keys and values go to the end of each cache.
        dict(name="append_decode_64", kind="append", sequences=64, longest=2048, new=1, heads=28, kv_heads=4, head_dim=128, rotary_dim=128, interleaved=False, scaling="none",
             theta=1e6, page=16, dtype="bf16"),
        # Prefill of 16 prompts of up to 1024 tokens, padded, into an 8-bit cache, with scaled positions.
        dict(name="append_prefill_e4m3", kind="append", sequences=16, longest=1024, new=1024, heads=28, kv_heads=4, head_dim=128, rotary_dim=128, interleaved=False, scaling="llama3",
             theta=1e6, page=64, dtype="e4m3"),
        # One long conversation on the larger decoder.
        dict(name="attend_1_long", kind="attend", sequences=1, longest=32768, ragged=False, heads=28, kv_heads=4, head_dim=128, page=16, dtype="bf16"),
        # A group's answers of all lengths on the smaller decoder, some slots empty.
        dict(name="attend_64_ragged", kind="attend", sequences=64, longest=4000, ragged=True, heads=12, kv_heads=2, head_dim=128, page=16, dtype="bf16"),
        # A full rollout batch over an 8-bit cache.
        dict(name="attend_256_e4m3", kind="attend", sequences=256, longest=2047, ragged=True, heads=28, kv_heads=4, head_dim=128, page=64, dtype="e4m3"),
        # 32 prompts, each forked for 16 answers, and the answers given back at the end.
        dict(name="pages_fork_32x16", kind="pages", op="fork", layers=28, kv_heads=2, head_dim=128, page=16, sequences=32, group=16, longest=500, dtype="bf16"),
        # A batch that ended raggedly: what is left moves to the front of the pool, all layers.
        dict(name="pages_compact", kind="pages", op="compact", layers=28, kv_heads=4, head_dim=128, page=16, sequences=40, group=1, longest=800, dtype="bf16"),
        # One sequence, every filter.
        dict(name="sample_1", kind="sample", rows=1, vocab=152064, dtype="bf16", spread=3.0, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02),
        # A small model's vocabulary, temperature alone.
        dict(name="sample_small", kind="sample", rows=24, vocab=97, dtype="fp32", spread=2.0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # A rollout batch by nucleus.
        dict(name="sample_256_top_p", kind="sample", rows=256, vocab=151936, dtype="bf16", spread=2.5, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 5, 8])
    return dict(heads=kv * rng.choice([1, 2, 3, 6, 7, 8, 12]), kv_heads=kv)


def _angles(rng, head_dim):
    return dict(rotary_dim=head_dim if rng.random() < 0.6 else 2 * rng.randint(1, head_dim // 2), interleaved=rng.random() < 0.4,
                scaling=rng.choice(["none", "linear", "llama3", "yarn"]), theta=rng.choice([1e4, 5e5, 1e6]))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "pages", "sample", "sample"])
    if kind == "rotary":
        d = 8 * _log(rng, 2, 32)
        c = dict(kind=kind, batch=_log(rng, 1, 16), tokens=_log(rng, 1, 4096), **_heads(rng), head_dim=d, **_angles(rng, d), start=rng.choice([0, _log(rng, 1, 1 << 20)]),
                 dtype=rng.choice(["bf16", "fp32"]), backward=rng.random() < 0.6)
        while c["batch"] * c["tokens"] * c["heads"] * d > 30_000_000:
            c["tokens"] = c["tokens"] // 2 + 1
    elif kind == "append":
        d = 8 * _log(rng, 4, 32)
        longest = _log(rng, 1, 4096)
        c = dict(kind=kind, sequences=_log(rng, 1, 256), longest=longest, new=1 if rng.random() < 0.5 else longest, **_heads(rng), head_dim=d, **_angles(rng, d),
                 page=rng.choice([16, 32, 64]), dtype=rng.choice(["bf16", "e4m3"]))
        while c["sequences"] * c["longest"] * c["kv_heads"] * d > 60_000_000 or c["sequences"] * c["new"] * c["heads"] * d > 60_000_000:
            c["sequences"] = c["sequences"] // 2
            if c["sequences"] == 0:
                c["sequences"], c["longest"] = 1, c["longest"] // 2
                c["new"] = min(c["new"], c["longest"])
    elif kind == "attend":
        c = dict(kind=kind, sequences=_log(rng, 1, 512), longest=_log(rng, 1, 65536), ragged=rng.random() < 0.7, **_heads(rng), head_dim=rng.choice([64, 80, 96, 128, 128, 256]),
                 page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "e4m3"]))
        while c["sequences"] * c["longest"] * c["kv_heads"] * c["head_dim"] > 200_000_000 or c["sequences"] * c["longest"] * c["heads"] > 30_000_000:
            c["longest"] = c["longest"] // 2 + 1
            c["sequences"] = (c["sequences"] + 1) // 2
    elif kind == "pages":
        c = dict(kind=kind, op=rng.choice(["fork", "compact"]), layers=_log(rng, 1, 28), kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]),
                 page=rng.choice([16, 32, 64]), sequences=_log(rng, 1, 200), group=_log(rng, 1, 16), longest=_log(rng, 1, 3000), dtype=rng.choice(["bf16", "e4m3"]))
        while c["sequences"] * (c["longest"] + c["group"] * c["page"]) * c["layers"] * c["kv_heads"] * c["head_dim"] > 200_000_000:
            c["sequences"], c["longest"] = (c["sequences"] + 1) // 2, c["longest"] // 2 + 1
            c["layers"] = (c["layers"] + 1) // 2
    else:
        c = dict(kind=kind, rows=_log(rng, 1, 256), vocab=_log(rng, 97, 152064), dtype=rng.choice(["bf16", "fp32"]), spread=rng.choice([0.5, 2.0, 4.0]),
                 temperature=rng.choice([0.0, 0.6, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, 20, 500]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.05]))
    return c


def _lengths(c):
    """Lengths of the sequences of a case, the same for every seed: what a pass has to move goes by them."""
    r = random.Random(c["sequences"] * 100003 + c["longest"])
    if c["kind"] == "attend":
        if not c["ragged"]:
            return [c["longest"]] * c["sequences"]
        return [0 if r.random() < 0.05 else r.randint(1, c["longest"]) for _ in range(c["sequences"] - 1)] + [c["longest"]]
    return [r.randint((c["longest"] + 3) // 4, c["longest"]) for _ in range(c["sequences"])]


def _pages(length, page):
    return -(-length // page)


# ---- what a program has in hand -----------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=DEV, generator=gen) * scale

    c, s = case, dict(case=case)
    kind = c["kind"]
    if kind == "rotary":
        dt = TYPES[c["dtype"]]
        for name, h in (("q", c["heads"]), ("k", c["kv_heads"])):
            s[name] = normal(c["batch"], c["tokens"], h, c["head_dim"]).to(dt)
            if c["backward"]:
                s["d" + name] = normal(c["batch"], c["tokens"], h, c["head_dim"], scale=0.1).to(dt)
                s[name].requires_grad_(True)
        first = torch.arange(c["batch"], device=DEV) * 17 + c["start"] + seed % 1000 * bool(c["start"])
        s["positions"] = first[:, None] + torch.arange(c["tokens"], device=DEV)[None]
    elif kind == "sample":
        # some rows sure of a few tokens, others not
        x = normal(c["rows"], c["vocab"], scale=c["spread"])
        lean = torch.rand(c["rows"], 1, device=DEV, generator=gen) * 2.0
        few = torch.randint(0, c["vocab"], (c["rows"], 8), device=DEV, generator=gen)
        x.scatter_add_(1, few, lean * c["spread"] * torch.rand(c["rows"], 8, device=DEV, generator=gen) * 2)
        s["logits"] = x.to(TYPES[c["dtype"]])
        s["u"] = torch.rand(c["rows"], device=DEV, generator=gen)
    else:
        lengths, page = _lengths(c), c["page"]
        group = c["group"] if kind == "pages" else 1
        held = sum(_pages(n, page) for n in lengths)
        spare = len(lengths) * group if kind == "pages" and c["op"] == "fork" else held // 2
        pages, width = held + spare + 8, _pages(c["longest"], page) + 2
        order = torch.randperm(pages, device=DEV, generator=gen)
        tables = torch.full((len(lengths) * (1 + group if kind == "pages" else 1), width), -1, dtype=torch.int32)
        at, order = 0, order.tolist()
        for i, n in enumerate(lengths):
            for j in range(_pages(n, page)):
                tables[i, j] = order[at]
                at += 1
        s["tables"] = tables.to(DEV)
        s["lengths"] = torch.tensor(lengths + [0] * (tables.shape[0] - len(lengths)), dtype=torch.int32, device=DEV)
        if kind == "pages" and c["op"] == "compact":
            # every third sequence's first pages are also those of a fork of its own
            for i in range(0, len(lengths), 3):
                n = lengths[i] // page * page
                if n:
                    s["tables"][len(lengths) + i, :n // page] = s["tables"][i, :n // page]
                    s["lengths"][len(lengths) + i] = n
        used = s["tables"][s["tables"] >= 0].long()
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEV).index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
        layers = c.get("layers", 1)
        pool = torch.empty(pages, layers, 2, c["kv_heads"], page, c["head_dim"], dtype=TYPES[c["dtype"]], device=DEV)
        for p in pool.split(max(1, (1 << 26) // pool[0].numel())):
            p.copy_(torch.randn(p.shape, device=DEV, generator=gen))
        s["pool"] = pool
        s["scales"] = 0.5 + torch.rand(layers, 2, c["kv_heads"], device=DEV, generator=gen) if c["dtype"] == "e4m3" else None
        if kind == "attend":
            s["q"] = normal(c["sequences"], c["heads"], c["head_dim"], scale=1.5).bfloat16()
        elif kind == "append":
            if c["new"] == 1:
                s["slots"] = torch.randperm(c["sequences"], device=DEV, generator=gen)
                s["positions"] = None                       # each goes to the end of its sequence
            else:
                # padded to the longest; what is behind a prompt belongs to nobody
                n = torch.tensor(lengths, device=DEV)[:, None]
                t = torch.arange(c["new"], device=DEV)[None].expand(c["sequences"], -1)
                s["slots"] = torch.where(t < n, torch.arange(c["sequences"], device=DEV)[:, None], -1).reshape(-1)
                s["positions"] = t.reshape(-1).contiguous()
            count = s["slots"].numel()
            s["q"] = normal(count, c["heads"], c["head_dim"]).bfloat16()
            s["k"], s["v"] = (normal(count, c["kv_heads"], c["head_dim"]).bfloat16() for _ in range(2))
        elif c["op"] == "fork":
            s["src"] = torch.arange(c["sequences"], device=DEV).repeat_interleave(group)
            s["dst"] = torch.arange(group * c["sequences"], device=DEV) + c["sequences"]
        else:
            s["kept"] = s["tables"].clone(), s["refs"].clone()
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _scaling(c):
    return {"none": None, "linear": dict(type="linear", factor=4.0),
            "llama3": dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=ORIGINAL),
            "yarn": dict(type="yarn", factor=4.0, original_max_position=ORIGINAL)}[c["scaling"]]


def _own(s):
    from fp4_post_b200 import rollout
    c = s["case"]
    kind = c["kind"]
    if "theta" in c and "rotary" not in s:
        s["rotary"] = rollout.Rotary(c["head_dim"], theta=c["theta"], rotary_dim=c["rotary_dim"], interleaved=c["interleaved"], scaling=_scaling(c), device=DEV)
    if "pool" in s and "cache" not in s:
        s["cache"] = rollout.PagedCache.of(s["pool"], s["tables"], s["lengths"], s["refs"], scales=s["scales"])
    if kind == "rotary":
        if not c["backward"]:
            return s["rotary"](s["q"], s["k"], s["positions"])
        q, k = s["rotary"](s["q"], s["k"], s["positions"])
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if kind == "sample":
        return rollout.sample(s["logits"], s["u"], temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"], logprobs=True)
    cache = s["cache"]
    if kind == "append":
        return cache.append(0, s["q"], s["k"], s["v"], s["slots"], s["positions"], rotary=s["rotary"]), s["pool"]
    if kind == "attend":
        return cache.attend(0, s["q"], return_lse=True)
    if c["op"] == "fork":
        cache.fork(s["src"], s["dst"])
        out = s["tables"].clone(), s["lengths"].clone(), s["refs"].clone()
        cache.free(s["dst"])
        return (*out, s["tables"], s["lengths"], s["refs"], s["pool"])
    s["tables"].copy_(s["kept"][0])                         # as the batch left it
    s["refs"].copy_(s["kept"][1])
    live = cache.compact()
    return live, s["tables"], s["refs"], s["pool"]


def _frequencies(c):
    """Angles per position of the pairs, in 64 bits, and what the rotated values are multiplied by."""
    n, theta = c["rotary_dim"], c["theta"]
    i = torch.arange(0, n, 2, dtype=torch.float64, device=DEV)
    f = theta ** (-i / n)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "llama3":
        mix = ((ORIGINAL * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        return f / 8.0 * (1 - mix) + f * mix, 1.0
    if c["scaling"] == "yarn":
        low, high = (n * math.log(ORIGINAL / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), n - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f / 4.0 * ramp + f * (1 - ramp), 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _table(c, positions):
    f, m = _frequencies(c)
    angle = positions.double()[..., None, None] * f         # [..., 1, rotary_dim / 2]
    return (angle.cos() * m).float(), (angle.sin() * m).float()


def _rotate(c, x, cos, sin):
    """x [..., heads, head_dim] in fp32."""
    n = c["rotary_dim"]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if c["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * cos - b * sin, b * cos + a * sin
    front = torch.stack((a, b), dim=-1).flatten(-2) if c["interleaved"] else torch.cat((a, b), dim=-1)
    return torch.cat((front, x[..., n:]), dim=-1)


def _plain(s):
    c = s["case"]
    with torch.no_grad():
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "pages": _plain_pages, "sample": _plain_sample}[c["kind"]](s, c)


def _plain_rotary(s, c):
    cos, sin = _table(c, s["positions"])
    dt = TYPES[c["dtype"]]
    out = [_rotate(c, s[n].float(), cos, sin).to(dt) for n in ("q", "k")]
    if c["backward"]:
        out += [_rotate(c, s[n].float(), cos, -sin).to(dt) for n in ("dq", "dk")]
    return tuple(out)


def _plain_append(s, c):
    page, slots = c["page"], s["slots"]
    positions = s["lengths"][slots].long() - 1 if s["positions"] is None else s["positions"]
    cos, sin = _table(c, positions)
    q, k, v = _rotate(c, s["q"].float(), cos, sin), _rotate(c, s["k"].float(), cos, sin), s["v"].float()
    q = torch.where((slots >= 0)[:, None, None], q, torch.zeros_like(q)).bfloat16()
    on = slots >= 0
    slots, positions, k, v = slots[on], positions[on], k[on], v[on]
    pages = s["tables"][slots, positions // page].long()
    if s["scales"] is not None:
        k, v = ((t / s["scales"][0, i][:, None]).clamp(-448.0, 448.0) for i, t in enumerate((k, v)))
    # (8-bit values are put in place as bytes: torch has no indexed writes of the type)
    bits = torch.uint8 if c["dtype"] == "e4m3" else torch.bfloat16
    for i, t in enumerate((k, v)):
        s["pool"].view(bits)[pages, 0, i, :, positions % page] = t.to(TYPES[c["dtype"]]).view(bits)
    return q, s["pool"]


def _plain_attend(s, c):
    b, d, page = c["sequences"], c["head_dim"], c["page"]
    width = _pages(c["longest"], page)
    at = s["tables"][:b, :width].long().clamp(min=0)
    kv = s["pool"][:, 0].view(torch.uint8 if c["dtype"] == "e4m3" else torch.bfloat16)
    there = torch.arange(width * page, device=DEV)[None] < s["lengths"][:b, None]

    def rows(i):
        t = kv[:, i][at].view(TYPES[c["dtype"]]).float()              # [b, width, heads, page, d]
        t = t.transpose(1, 2).reshape(b, c["kv_heads"], width * page, d)
        return t if s["scales"] is None else t * s["scales"][0, i][:, None, None]

    q = s["q"].float().reshape(b, c["kv_heads"], c["heads"] // c["kv_heads"], d)
    scores = torch.matmul(q, rows(0).transpose(2, 3)) * d ** -0.5
    scores = torch.where(there[:, None, None], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = (scores - top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, rows(1)) / total
    out = torch.where((total > 0), out, torch.zeros_like(out))
    return out.reshape(b, c["heads"], d).bfloat16(), (top + total.log())[..., 0].reshape(b, c["heads"])


def _plain_pages(s, c):
    tables, lengths, refs, page = s["tables"], s["lengths"], s["refs"], c["page"]
    pool = s["pool"].view(torch.uint8) if c["dtype"] == "e4m3" else s["pool"]
    column = torch.arange(tables.shape[1], device=DEV)[None]
    if c["op"] == "fork":
        src, dst = s["src"], s["dst"]
        n = lengths[src]
        full, part = n // page, n % page
        new = (refs == 0).nonzero()[:, 0][:int((part > 0).sum())]
        old = tables[src[part > 0], full[part > 0].long()].long()
        rows = torch.where(column < full[:, None], tables[src], torch.full_like(tables[src], -1))
        shared = rows[rows >= 0].long()
        rows[(part > 0).nonzero()[:, 0], full[part > 0].long()] = new.to(torch.int32)
        tables[dst], lengths[dst] = rows, n
        refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
        refs[new] = 1
        filled = (torch.arange(page, device=DEV)[None] < part[part > 0][:, None])[:, None, None, None, :, None]
        pool[new] = torch.where(filled, pool[old], pool[new])
        out = tables.clone(), lengths.clone(), refs.clone()
        given = tables[dst]
        given = given[given >= 0].long()
        refs.index_add_(0, given, -torch.ones_like(given, dtype=torch.int32))
        tables[dst], lengths[dst] = -1, 0
        return (*out, tables, lengths, refs, s["pool"])
    tables.copy_(s["kept"][0])
    refs.copy_(s["kept"][1])
    live = (refs > 0).sum()
    index = torch.arange(refs.numel(), device=DEV)
    holes, movers = ((refs == 0) & (index < live)).nonzero()[:, 0], ((refs > 0) & (index >= live)).nonzero()[:, 0]
    pool[holes] = pool[movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    index[movers] = holes
    tables.copy_(torch.where(tables >= 0, index[tables.long().clamp(min=0)].to(torch.int32), tables))
    return live.to(torch.int32).reshape(1), tables, refs, s["pool"]


def _plain_sample(s, c):
    """The weights in fp32, their sums in 64 bits: a border between two tokens lies where the sums say."""
    x = s["logits"].float()
    n = x.shape[1]
    top = x.amax(dim=1, keepdim=True)
    t = torch.full_like(top, c["temperature"] or 1.0)
    w = ((x - top) * (1.0 / t)).exp()
    log_total = w.double().sum(dim=1, keepdim=True).log()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order).double()
    rank = torch.arange(n, device=DEV)[None]
    k = 1 if c["temperature"] == 0.0 else c["top_k"] or n
    ws = torch.where(rank < k, ws, torch.zeros_like(ws))
    before = ws.cumsum(dim=1)
    total = before[:, -1:].clone()
    before = before - ws
    kept = (rank < k) & (ws >= float(torch.tensor(c["min_p"], dtype=torch.float32)))
    if c["top_p"] < 1.0:
        kept &= before < c["top_p"] * total
    kept[:, 0] = True
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    sums = torch.where(kept, w.double(), torch.zeros((), dtype=torch.float64, device=DEV)).cumsum(dim=1)
    token = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(dim=1)
    logp = ((x.gather(1, token[:, None]).double() - top.double()) / t.double() - log_total)[:, 0]
    return token, logp.float()


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend, "pages": lambda s, c: None, "sample": _exact_sample}[case["kind"]](s, case)


def _exact_angles(c):
    """The same frequencies pair by pair, and as complex numbers of one turn."""
    n, base = c["rotary_dim"], c["theta"]
    freq, m = [], 1.0
    for j in range(n // 2):
        f = math.exp(-2 * j / n * math.log(base))
        if c["scaling"] == "linear":
            f /= 4
        elif c["scaling"] == "llama3":
            turns = ORIGINAL * f / (2 * math.pi)
            f = f / 8 if turns < 1 else f if turns > 4 else f / 8 * (4 - turns) / 3 + f * (turns - 1) / 3
        elif c["scaling"] == "yarn":
            pair = lambda turns: n * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), n - 1)
            slow = min(1.0, max(0.0, (j - lo) / (hi - lo if hi > lo else 0.001)))
            f = f * (1 - slow) + f / 4 * slow
            m = 1 + math.log(4.0) / 10
        freq.append(f)
    return torch.tensor(freq, dtype=torch.float64, device=DEV), m


def _exact_turn(c, x, positions, sign=1.0):
    freq, m = _exact_angles(c)
    n = c["rotary_dim"]
    x = x.detach().double()
    phase = torch.polar(torch.full_like(positions.double()[..., None] * freq, m), sign * positions.double()[..., None] * freq).unsqueeze(-2)
    out = x.clone()
    first, second = (slice(0, n, 2), slice(1, n, 2)) if c["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    z = torch.complex(x[..., first], x[..., second]) * phase
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_rotary(s, c):
    out = [_exact_turn(c, s[n], s["positions"]) for n in ("q", "k")]
    if c["backward"]:
        out += [_exact_turn(c, s["d" + n], s["positions"], -1.0) for n in ("q", "k")]
    return tuple(out)


def _exact_append(s, c):
    """The queries; what the pages hold in 8 bits has one rounding, and no value of its own here."""
    positions = s["lengths"][s["slots"].clamp(min=0)].long() - 1 if s["positions"] is None else s["positions"]
    q = _exact_turn(c, s["q"], positions)
    q[s["slots"] < 0] = 0.0
    if c["dtype"] == "e4m3":
        return q, None
    pool = s["pool"].double()
    k = _exact_turn(c, s["k"], positions)
    on = (s["slots"] >= 0).nonzero()[:, 0]
    flat = s["tables"][s["slots"][on], positions[on] // c["page"]].long()
    pool[flat, 0, 0, :, positions[on] % c["page"]] = k[on]
    pool[flat, 0, 1, :, positions[on] % c["page"]] = s["v"][on].double()
    return q, pool


def _exact_attend(s, c):
    """Sequence by sequence."""
    d, group = c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(c["sequences"], c["heads"], d, dtype=torch.float64, device=DEV)
    lse = torch.full((c["sequences"], c["heads"]), -math.inf, dtype=torch.float64, device=DEV)
    for i, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        own_pages = s["tables"][i, :_pages(n, c["page"])].long()
        kv = s["pool"].view(torch.uint8 if c["dtype"] == "e4m3" else torch.bfloat16)[own_pages, 0].view(TYPES[c["dtype"]]).double()
        if s["scales"] is not None:
            kv = kv * s["scales"][0].double()[None, :, :, None, None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, c["kv_heads"], -1, d)[:, :, :n].repeat_interleave(group, dim=1)
        scores = torch.einsum("hd,hnd->hn", s["q"][i].double(), kv[0]) / math.sqrt(d)
        lse[i] = torch.logsumexp(scores, dim=1)
        out[i] = torch.einsum("hn,hnd->hd", torch.softmax(scores, dim=1), kv[1])
    return out, lse


def _exact_sample(s, c):
    """The log-probabilities of the tokens, row by row: the tokens by thresholds on the logits (no sort), with the operator's weights in fp32."""
    got = []
    t = c["temperature"] or 1.0
    for x, u in zip(s["logits"].float(), s["u"].double()):
        w = ((x - x.max()) * (1.0 / torch.tensor(t, device=DEV))).exp().double()
        kept = torch.ones_like(x, dtype=torch.bool)
        k = 1 if c["temperature"] == 0.0 else c["top_k"]
        if 0 < k < x.numel():
            last = torch.topk(x, k).values[-1]
            over, ties = x > last, x == last
            kept = over | (ties & (ties.cumsum(0) <= k - over.sum()))
        if c["top_p"] < 1.0:
            values, back = torch.unique(x[kept], return_inverse=True)
            mass = torch.zeros_like(values, dtype=torch.float64).index_add_(0, back, w[kept])
            above = mass.flip(0).cumsum(0).flip(0) - mass
            short = above < c["top_p"] * w[kept].sum()              # values of which something is kept: the largest ones
            border = values[short].min()
            over, ties = kept & (x > border), kept & (x == border)
            rest = w[over].sum() + (ties.cumsum(0) - 1) * w[ties][0]
            kept = over | (ties & (rest < c["top_p"] * w[kept].sum()))
        kept &= w >= float(torch.tensor(c["min_p"], dtype=torch.float32))
        sums = torch.where(kept, w, 0.0).cumsum(0)
        token = torch.searchsorted(sums, u * sums[-1], right=True)
        got.append(torch.log_softmax(x.double() / t, dim=0)[token])
    return None, torch.stack(got)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "rotary":
        n = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"])
        size = 2 if c["dtype"] == "bf16" else 4
        passes = 2 if c["backward"] else 1
        return {"bytes": passes * 2 * n * c["head_dim"] * size + 8 * c["batch"] * c["tokens"], "flops": passes * n * 3 * c["rotary_dim"]}
    if kind == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * (2 if c["dtype"] == "bf16" else 4) + 16), "flops": c["rows"] * c["vocab"] * 4}
    lengths, item = _lengths(c), 1 if c["dtype"] == "e4m3" else 2
    if kind == "append":
        live = len(lengths) if c["new"] == 1 else sum(lengths)
        rows = len(lengths) * c["new"]
        read = live * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"] * 2
        return {"bytes": read + rows * c["heads"] * c["head_dim"] * 2 + live * 2 * c["kv_heads"] * c["head_dim"] * item + 8 * rows,
                "flops": live * (c["heads"] + c["kv_heads"]) * 3 * c["rotary_dim"]}
    if kind == "attend":
        total = sum(lengths)
        return {"bytes": 2 * total * c["kv_heads"] * c["head_dim"] * item + len(lengths) * c["heads"] * (c["head_dim"] * 4 + 4) + 4 * sum(_pages(n, c["page"]) for n in lengths),
                "flops": 4 * total * c["heads"] * c["head_dim"]}
    token = c["layers"] * 2 * c["kv_heads"] * c["head_dim"] * item
    held = sum(_pages(n, c["page"]) for n in lengths)
    if c["op"] == "fork":
        parts = sum(n % c["page"] for n in lengths)
        return {"bytes": (1 + c["group"]) * parts * token + 4 * held * (1 + 3 * c["group"]), "flops": 0}
    # a page of `held` among pages in random order is moved where it lies behind the first `held` ones
    pages = held + held // 2 + 8
    return {"bytes": 2 * held * (pages - held) / pages * c["page"] * token + 16 * held + 8 * pages, "flops": 0}
