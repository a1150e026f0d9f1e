"""Operators on a paged key/value cache, as cases that can be timed and compared.

A case is one pass through one operator:

  attend   `paged_attention`: one new token per row over the pages that its table names
  append   `append_kv`: queries and keys of a step turned to their positions, keys and values stored in the cache
  rotary   `rotary`: queries and keys turned to their positions, no cache
  pages    `copy_pages`: pages copied in all layers' pools (a fork's last pages, a compaction)

With `own` false the same is computed from elementary tensor operations in 32 bits (angles in 64).
"""
import math
from functools import lru_cache

import torch

own = False

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # the first tokens of one chat: launch and host latency are the whole of it
        dict(name="attend-1x17", kind="attend", rows=1, longest=17, lengths="equal", heads=32, kv_heads=32, dim=128,
             page=16, window=0, type="f16"),
        # the benchmark's context of 1024 tokens, a small decode batch
        dict(name="attend-32x1024", kind="attend", rows=32, longest=1024, lengths="equal", heads=32, kv_heads=32, dim=128,
             page=16, window=0, type="f16"),
        # one layer of the benchmark's full decode step: 128 sequences, 1025 tokens with the new one
        dict(name="attend-128x1025", kind="attend", rows=128, longest=1025, lengths="equal", heads=32, kv_heads=32, dim=128,
             page=16, window=0, type="f16"),
        # continuous batching: sequences of all ages, padded rows among them, four heads to a key
        dict(name="attend-61-ragged", kind="attend", rows=61, longest=9001, lengths="ragged", heads=32, kv_heads=8, dim=128,
             page=32, window=0, type="bf16"),
        # one long document: rows are few, the length has to be split
        dict(name="attend-1-long", kind="attend", rows=1, longest=131071, lengths="equal", heads=64, kv_heads=8, dim=128,
             page=64, window=0, type="bf16"),
        # a small model with a sliding window that begins inside a page; a head that fills no power of two
        dict(name="attend-24-window", kind="attend", rows=24, longest=2777, lengths="ragged", heads=20, kv_heads=20, dim=80,
             page=8, window=1000, type="f16"),
        # one sequence's new token stored
        dict(name="append-1", kind="append", tokens=1, longest=2000, heads=32, kv_heads=32, dim=128, rot=128, page=16,
             interleaved=False, scaling="none", type="f16"),
        # a full decode batch's new tokens stored
        dict(name="append-128", kind="append", tokens=128, longest=1024, heads=32, kv_heads=32, dim=128, rot=128, page=16,
             interleaved=False, scaling="none", type="f16"),
        # a prefill batch of several prompts stored, positions far beyond the trained ones
        dict(name="append-8192", kind="append", tokens=8192, longest=100000, heads=32, kv_heads=8, dim=128, rot=128, page=64,
             interleaved=False, scaling="yarn", type="bf16"),
        # a ragged prompt of a model that turns part of each head, neighbours paired
        dict(name="rotary-2047", kind="rotary", tokens=2047, longest=5000, heads=20, kv_heads=20, dim=80, rot=32, page=16,
             interleaved=True, scaling="linear", type="f16"),
        # sixteen requests forked (beams, samples of one prompt): their last pages copied in 32 layers
        dict(name="pages-fork", kind="pages", pairs=16, pools=64, pages=256, page_elements=16 * 32 * 128, type="f16"),
        # a cache compacted: live pages moved down in 32 layers
        dict(name="pages-compact", kind="pages", pairs=700, pools=64, pages=1500, page_elements=16 * 8 * 128, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 32), (40, 40), (16, 16), (20, 20), (32, 8), (64, 8), (40, 8), (28, 4), (16, 1), (12, 12)]


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["append"] * 3 + ["rotary"] + ["pages"] * 2)
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([128, 128, 128, 64, 80, 96, 192, 256])
    page, kind_of = rng.choice([8, 16, 16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"])
    if kind == "attend":
        # no dearer than 128 x 1025 tokens of 32 heads of 128
        rows = _log(rng, 1, 256)
        longest = _log(rng, 1, max(2, min(131072, 128 * 1025 * 32 * 128 // (rows * kv * dim))))
        return dict(kind=kind, rows=rows, longest=longest, lengths=rng.choice(["equal", "ragged"]), heads=heads, kv_heads=kv,
                    dim=dim, page=page, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), type=kind_of)
    if kind in ("append", "rotary"):
        rot = rng.choice([dim, dim, dim // 2, 32, 20])
        return dict(kind=kind, tokens=_log(rng, 1, 8192), longest=_log(rng, 64, 200000), heads=heads, kv_heads=kv, dim=dim,
                    rot=rot, page=page, interleaved=rng.random() < 0.4,
                    scaling=rng.choice(["none", "none", "linear", "dynamic", "yarn"]), type=kind_of)
    pools = 2 * rng.choice([1, 2, 12, 24, 32, 40])
    elements = rng.choice([8, 16, 32, 64]) * kv * rng.choice([64, 80, 128])
    pairs = _log(rng, 1, max(2, min(2000, (1 << 29) // (pools * elements))))
    return dict(kind=kind, pairs=pairs, pools=pools, pages=2 * pairs + rng.randrange(1, 100), page_elements=elements, type=kind_of)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _lengths(case, gen):
    """Tokens of each row, the new one among them: a batch of one age, or of all ages with padded (empty) rows."""
    r, n = case["rows"], case["longest"]
    if case["lengths"] == "equal":
        return torch.full((r,), n, dtype=torch.int32, device=DEV)
    u = torch.rand(r, generator=gen, device=DEV)
    lens = torch.exp(u * math.log(n)).round().to(torch.int32).clamp_(1, n)
    lens[torch.arange(r, device=DEV) % 16 == 15] = 0
    lens[0] = n
    return lens


def _scaling(case):
    """The entry of a model's configuration that says how positions are scaled for long contexts."""
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "dynamic": {"type": "dynamic", "factor": 2.0},
            "yarn": {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}}[case["scaling"]]


BASE, TRAINED = 10000.0, 4096


def _frequencies(case):
    """(radians per position of every pair in 64 bits, factor on the turned values)."""
    r = case["rot"]
    i = torch.arange(r // 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "dynamic":          # the base grows with the context, here twice the trained one
        return (BASE * (2.0 * 2.0 - 1.0) ** (r / (r - 2))) ** (-2.0 * i / r), 1.0
    if case["scaling"] == "yarn":             # slow pairs are stretched, fast ones kept, a ramp between
        at = lambda turns: r * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(BASE))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / 16.0 * (1.0 - keep) + f * keep, 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, dtype = case["kind"], TYPES[case["type"]]
    randn = lambda *shape: torch.randn(shape, generator=gen, device=DEV, dtype=dtype)
    if kind == "pages":
        order = torch.randperm(case["pages"], generator=gen, device=DEV)[:2 * case["pairs"]].view(2, -1)
        pools = randn(case["pools"], case["pages"], case["page_elements"])
        src, dst = order[0].contiguous(), order[1].contiguous()
        # the scheduler decides what is copied, on the host
        return dict(case=case, pools=pools, src=src, dst=dst, pairs=torch.stack((src, dst), 1).cpu())
    heads, kv, dim, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if kind == "attend":
        lens = _lengths(case, gen)
        width = -(-case["longest"] // ps)
        used = (lens.long() + ps - 1) // ps
        need = int(used.sum())
        pages = need + need // 8 + 1
        ids = torch.randperm(pages, generator=gen, device=DEV)[:need].to(torch.int32)      # pages come and go: any order
        first = torch.cumsum(used, 0) - used
        column = torch.arange(width, device=DEV)
        at = (first[:, None] + column[None, :]).clamp_(max=max(need - 1, 0))
        tables = torch.where(column[None, :] < used[:, None], ids[at], torch.zeros_like(ids[at])) if need else torch.zeros(
            (case["rows"], width), dtype=torch.int32, device=DEV)
        # keys of a trained model leave some tokens much likelier than others
        return dict(case=case, q=1.5 * randn(case["rows"], heads, dim), k=randn(pages, kv, ps, dim), v=randn(pages, kv, ps, dim),
                    tables=tables.contiguous(), lens=lens, scale=dim ** -0.5)
    tokens = case["tokens"]
    qkv = randn(tokens, (heads + 2 * kv) * dim)                    # what the fused projection gives
    q, k, v = qkv.split((heads * dim, kv * dim, kv * dim), dim=1)
    q, k, v = q.unflatten(1, (heads, dim)), k.unflatten(1, (kv, dim)), v.unflatten(1, (kv, dim))
    if tokens <= 256:                                              # a decode batch: sequences at positions of their own
        positions = torch.randint(0, case["longest"], (tokens,), generator=gen, device=DEV)
        block, offset = torch.arange(tokens, device=DEV), positions % ps
        pages = tokens
    else:                                                          # prompts one after the other
        cuts = torch.randint(0, tokens, (4,), generator=gen, device=DEV)
        t = torch.arange(tokens, device=DEV)
        start = torch.where(cuts[None, :] <= t[:, None], cuts[None, :], torch.zeros_like(cuts)[None, :]).amax(1)
        positions = t - start + int(max(0, case["longest"] - tokens))
        block, offset = t // ps, t % ps
        pages = -(-tokens // ps)
    state = dict(case=case, q=q, k=k, v=v, positions=positions)
    if kind == "append":
        pool = pages + pages // 4 + 1
        where = torch.randperm(pool, generator=gen, device=DEV)
        state.update(slots=where[block] * ps + offset, k_pages=randn(pool, kv, ps, dim), v_pages=randn(pool, kv, ps, dim))
    state["frequencies"], state["factor"] = _frequencies(case)
    if own:                                                        # the same numbers, in the handle that a model keeps
        state["rope"] = _package().RotaryPositions(dim, rotary_dim=case["rot"], base=BASE, max_position=TRAINED,
                                                   interleaved=case["interleaved"], scaling=_scaling(case))
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


@lru_cache(maxsize=1)
def _package():
    import deltazip_amd
    return deltazip_amd


def run(state):
    return {"attend": _attend, "append": _append, "rotary": _rotary, "pages": _pages}[state["case"]["kind"]](state)


def _attend(s):
    case, tables = s["case"], s["tables"]
    if own:
        return _package().paged_attention(s["q"], s["k"], s["v"], tables, s["lens"], scale=s["scale"], window=case["window"])
    rows, heads, dim = s["q"].shape
    kv = case["kv_heads"]
    # pages gathered, in 32 bits: [rows, kv_heads, tokens, dim]
    k, v = (p[tables.long()].permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, dim).float() for p in (s["k"], s["v"]))
    q = s["q"].float().view(rows, kv, heads // kv, dim) * s["scale"]
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous())
    t = torch.arange(scores.shape[-1], device=DEV)
    lens = s["lens"][:, None]
    seen = t < lens
    if case["window"]:
        seen = seen & (t >= lens - case["window"])
    seen = seen[:, None, None, :]
    scores = torch.where(seen, scores, torch.full_like(scores, -3e38))
    p = torch.exp(scores - scores.amax(-1, keepdim=True)) * seen
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(p, v).reshape(rows, heads, dim).to(s["q"].dtype)


def _turn(x, s):
    """The first `rot` values of every head turned by position * frequency, in pairs."""
    case = s["case"]
    r = case["rot"]
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    c, n = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    f = x[..., :r].float()
    if case["interleaved"]:
        a, b = f[..., 0::2], f[..., 1::2]
        y = torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)
    else:
        a, b = f[..., :r // 2], f[..., r // 2:]
        y = torch.cat((a * c - b * n, b * c + a * n), -1)
    return torch.cat((y.to(x.dtype), x[..., r:]), -1)


def _rotary(s):
    if own:
        return _package().rotary(s["q"], s["k"], s["positions"], s["rope"])
    return _turn(s["q"], s), _turn(s["k"], s)


def _append(s):
    if own:
        q = _package().append_kv(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rope"], s["k_pages"], s["v_pages"])
        return q, s["k_pages"], s["v_pages"]
    ps = s["case"]["page"]
    page, offset = s["slots"] // ps, s["slots"] % ps
    s["k_pages"][page, :, offset] = _turn(s["k"], s)
    s["v_pages"][page, :, offset] = s["v"]
    return _turn(s["q"], s), s["k_pages"], s["v_pages"]


def _pages(s):
    if own:
        _package().copy_pages(s["pools"], s["pairs"])
    else:
        s["pools"][:, s["dst"]] = s["pools"][:, s["src"]]
    return s["pools"]


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "pages":
        return dict(bytes=2 * 2 * case["pairs"] * case["pools"] * case["page_elements"], flops=0)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attend":
        rows, n = case["rows"], case["longest"]
        if case["lengths"] == "equal":
            tokens = rows * min(n, case["window"] or n)
        else:                                 # the lengths' distribution in equal steps
            u = [(i + 0.5) / 1000 for i in range(1000)]
            lens = [min(math.exp(x * math.log(n)), case["window"] or n) for x in u]
            tokens = sum(lens) / 1000 * max(rows - 1 - rows // 16, 0) + min(n, case["window"] or n)
        return dict(bytes=2 * 2 * tokens * kv * dim + 2 * 2 * rows * heads * dim + 4 * tokens / case["page"] + 4 * rows,
                    flops=4 * tokens * heads * dim)
    tokens, stored = case["tokens"], case["kind"] == "append"
    values = tokens * (heads + (2 if stored else 1) * kv) * dim
    return dict(bytes=2 * 2 * values + (16 if stored else 8) * tokens, flops=3 * tokens * (heads + kv) * case["rot"])


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        want = s["pools"].clone()
        for a, b in s["pairs"].tolist():
            want[:, b].copy_(s["pools"][:, a])
        return want
    if case["kind"] == "attend":
        rows = []
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                rows.append(torch.zeros(case["heads"], case["dim"], dtype=torch.float64, device=DEV))
                continue
            first = max(0, n - case["window"]) if case["window"] else 0
            t = torch.arange(first, n, device=DEV)
            page = s["tables"][b].long()[t // case["page"]]
            out = []
            for h in range(case["kv_heads"]):
                k, v = (p[page, h, t % case["page"]].double() for p in (s["k"], s["v"]))
                mine = s["q"][b].view(case["kv_heads"], -1, case["dim"])[h].double()
                out.append(torch.softmax(mine @ k.t().contiguous() * s["scale"], -1) @ v)
            rows.append(torch.cat(out))
        return torch.stack(rows)
    r, i = case["rot"], torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
    base, factor = torch.tensor(10000.0, dtype=torch.float64, device=DEV), 1.0
    if case["scaling"] == "dynamic":
        base = base * 3.0 ** (r / (r - 2.0))
    f = torch.exp(-torch.log(base) * 2.0 * i / r)
    if case["scaling"] == "linear":
        f = f * 0.25
    if case["scaling"] == "yarn":
        # the pair that makes `turns` turns within the trained context
        pair = [0.5 * r * math.log(4096 / (2 * math.pi * turns), 10000.0) for turns in (32, 1)]
        lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), r - 1)
        share = torch.clamp((i - lo) / max(hi - lo, 0.001), 0, 1)             # of the stretched frequency
        f = f * (1 - share * (1 - 1 / 16))
        factor = 1 + 0.1 * math.log(16)
    angle = s["positions"].double()[:, None] * f
    z = factor * torch.complex(torch.cos(angle), torch.sin(angle))[:, None, :]

    def turned(x):
        y = x.double().clone()
        if case["interleaved"]:
            w = torch.complex(y[..., 0:r:2].clone(), y[..., 1:r:2].clone()) * z
            y[..., 0:r:2], y[..., 1:r:2] = w.real, w.imag
        else:
            w = torch.complex(y[..., :r // 2].clone(), y[..., r // 2:r].clone()) * z
            y[..., :r // 2], y[..., r // 2:r] = w.real, w.imag
        return y

    q, k = turned(s["q"]), turned(s["k"])
    if case["kind"] == "rotary":
        return q, k
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    page, offset = torch.div(s["slots"], case["page"], rounding_mode="floor"), s["slots"] % case["page"]
    kp[page, :, offset], vp[page, :, offset] = k, s["v"].double()
    return q, kp, vp
