"""Operators on a paged key/value cache whose rows share prefixes, hold prompts and grow on the device, as cases that can be timed
and compared.

A case is one pass through one operator:

  attend   `prefix_attention`: the new tokens of every row over its pages; rows of a group share their first pages
  tables   `extend_tables`: rows given room for new tokens: pages, positions, slots, lengths

With `own` false the same is computed from elementary tensor operations: attention in 32 bits over every row's pages gathered,
tables from running sums.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------
# the cases
#
# attend: `rows` rows in `groups` groups of neighbours whose first `prefix` tokens are the same pages; every row has up to `suffix`
# tokens of its own, of which up to `new` are new (queries); every `pad`-th row is empty (0: none).
# tables: `rows` rows of up to `longest` tokens get up to `new` more; packed: tokens follow each other (prompts), else a place a row.
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # four samples of one chat's short prompt: launch and host latency
        dict(name="samples-4", kind="attend", rows=4, groups=1, prefix=272, suffix=20, new=1, pad=0, heads=32, kv_heads=32, dim=128,
             page=16, type="f16"),
        # samples of one prompt, the benchmark's heads
        dict(name="samples-32", kind="attend", rows=32, groups=1, prefix=2048, suffix=200, new=1, pad=0, heads=32, kv_heads=32, dim=128,
             page=16, type="f16"),
        # the benchmark's batch of 128 chats with four deltas, each with a system prompt of its own
        dict(name="system-128", kind="attend", rows=128, groups=4, prefix=4096, suffix=1025, new=1, pad=0, heads=32, kv_heads=32, dim=128,
             page=16, type="f16"),
        # continuous batching with four heads to a key and more: chats of all ages, padded rows, long instructions
        dict(name="system-203", kind="attend", rows=203, groups=3, prefix=20000, suffix=3001, new=1, pad=16, heads=64, kv_heads=8, dim=128,
             page=32, type="bf16"),
        # questions about one long document
        dict(name="document-16", kind="attend", rows=16, groups=1, prefix=131072, suffix=500, new=1, pad=0, heads=40, kv_heads=8, dim=128,
             page=64, type="bf16"),
        # drafted tokens verified, a small model's heads, which fill no power of two
        dict(name="drafts-48", kind="attend", rows=48, groups=6, prefix=776, suffix=333, new=5, pad=0, heads=20, kv_heads=20, dim=80,
             page=8, type="f16"),
        # a ragged batch of prompts, nothing shared
        dict(name="prompts-9", kind="attend", rows=9, groups=9, prefix=0, suffix=701, new=701, pad=0, heads=32, kv_heads=32, dim=128,
             page=16, type="f16"),
        # one long prompt in one pass
        dict(name="prompt-8192", kind="attend", rows=1, groups=1, prefix=0, suffix=8192, new=8192, pad=0, heads=32, kv_heads=8, dim=128,
             page=16, type="bf16"),
        # a decode step's tables: one token for every sequence
        dict(name="step-16", kind="tables", rows=16, longest=1024, new=1, packed=False, page=16),
        dict(name="step-1777", kind="tables", rows=1777, longest=9001, new=1, packed=False, page=32),
        # prompts taken in: positions and slots of all their tokens
        dict(name="intake-37", kind="tables", rows=37, longest=3001, new=999, packed=True, page=16),
        dict(name="intake-400", kind="tables", rows=400, longest=5000, new=4096, packed=True, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


HEADS = [(32, 32), (40, 40), (16, 16), (20, 20), (32, 8), (64, 8), (40, 8), (28, 4), (16, 1), (12, 12)]


def draw(rng):
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if rng.random() < 0.3:
        packed = rng.random() < 0.5
        rows = _log(rng, 1, 512 if packed else 4096)
        return dict(kind="tables", rows=rows, longest=_log(rng, 1, 20000), new=_log(rng, 1, min(8192, 800000 // rows)) if packed else 1,
                    packed=packed, page=page)
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([128, 128, 128, 64, 80, 96, 192, 256])
    kind_of = rng.choice(["f16", "bf16"])
    what = rng.choice(["samples", "samples", "samples", "drafts", "prompts", "behind"])
    # no dearer than 203 rows of 23000 tokens of 64 heads of 128 (the plain form gathers them all), or 8192 tokens at once
    room = 203 * 23001 * 8 * 128 // (kv * dim)
    if what in ("samples", "drafts"):
        rows = _log(rng, 1, 256)
        groups = _log(rng, 1, max(1, rows // 2))
        total = min(131072, room // rows, 203 * 23001 * 64 * 128 // (rows * heads * dim))
        suffix = _log(rng, 1, max(1, min(4096, total // 4)))
        return dict(kind="attend", rows=rows, groups=groups, prefix=_log(rng, 1, max(1, total * 3 // 4)) // page * page, suffix=suffix,
                    new=1 if what == "samples" else min(suffix, _log(rng, 1, 16)), pad=rng.choice([0, 0, 5, 16]), heads=heads, kv_heads=kv,
                    dim=dim, page=page, type=kind_of)
    rows = _log(rng, 1, 24)
    new = _log(rng, 2, min(4096, 8192 // rows))
    seen = 8192 * 4096 * 32 * 128 // (rows * new * heads * dim)
    earlier = rng.choice([0, 0, _log(rng, 1, max(1, min(2000, seen // 4)))])          # a prompt taken in pieces: tokens in the cache already
    prefix = _log(rng, page, max(page, min(8192, seen // 2))) // page * page if what == "behind" else 0
    return dict(kind="attend", rows=rows, groups=rng.choice([1, max(1, rows // 3)]) if prefix else rows, prefix=prefix, suffix=new + earlier,
                new=new, pad=0, heads=heads, kv_heads=kv, dim=dim, page=page, type=kind_of)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _spread(most, n, even):
    """n lengths up to `most`, the longest among them: of all ages evenly, or spread over their logarithm."""
    u = (np.arange(n, dtype=np.float64) + 1.0) / n
    x = most * u if even else np.exp(u * math.log(most))
    return np.clip(np.ceil(x - 1e-9), 1, most).astype(np.int64)


def _sizes(case):
    """(tokens of their own, new ones) of every row before they are shuffled: the same for every seed, so that the work is."""
    rows = case["rows"]
    suffix = _spread(case["suffix"], rows, even=case["new"] == 1)
    new = np.minimum(_spread(case["new"], rows, even=True), suffix)
    if case["pad"]:
        empty = np.arange(rows) % case["pad"] == case["pad"] - 1
        suffix[empty], new[empty] = 0, 0
    return suffix, new


def _dev(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, dtype)


def prepare(case, seed):
    return (_prepare_attend if case["kind"] == "attend" else _prepare_tables)(case, int(seed))


def _prepare_attend(case, seed):
    gen, rng = torch.Generator(device=DEV).manual_seed(seed), np.random.default_rng(seed)
    dtype, rows, ps, prefix = TYPES[case["type"]], case["rows"], case["page"], case["prefix"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    suffix, new = _sizes(case)
    order = rng.permutation(rows)                                    # padded rows among the others
    suffix, new = suffix[order], new[order]
    lengths = np.where(suffix > 0, prefix + suffix, 0)
    # groups of neighbours, as even as they come; their first pages are the first row's
    bounds = np.arange(case["groups"] + 1, dtype=np.int64) * rows // case["groups"]
    group = np.searchsorted(bounds, np.arange(rows), side="right") - 1
    shared, used = prefix // ps, -(-lengths // ps)
    mine = np.where(lengths > 0, used - shared, 0)
    width = max(1, int(used.max()))
    pages = case["groups"] * shared + int(mine.sum())
    ids = rng.permutation(pages + pages // 8 + 1)                    # pages come and go: any order
    tables = np.zeros((rows, width), dtype=np.int64)
    tables[:, :shared] = ids[:case["groups"] * shared].reshape(case["groups"], shared)[group]
    tables[lengths == 0] = 0
    column = np.arange(width)
    at = case["groups"] * shared + (np.cumsum(mine) - mine)[:, None] + column[None, :] - shared
    own_part = (column[None, :] >= shared) & (column[None, :] < used[:, None])
    tables[own_part] = ids[at[own_part]]
    randn = lambda *shape: torch.randn(shape, generator=gen, device=DEV, dtype=dtype)
    starts = np.concatenate(([0], np.cumsum(new)))
    tokens = rows if case["new"] == 1 else int(starts[-1])
    state = dict(case=case, scale=dim ** -0.5, most=int(new.max()), lens=_dev(lengths, torch.int32), tables=_dev(tables, torch.int32),
                 # keys of a trained model leave some tokens much likelier than others
                 q=1.5 * randn(tokens, heads, dim), k=randn(len(ids), kv, ps, dim), v=randn(len(ids), kv, ps, dim),
                 starts=None if case["new"] == 1 else _dev(starts, torch.int32))
    shares = prefix > 0
    state["groups"] = _dev(bounds, torch.int32) if shares else None
    state["prefixes"] = _dev(np.full(case["groups"], prefix), torch.int32) if shares else None
    return state


def _prepare_tables(case, seed):
    rng = np.random.default_rng(seed)
    rows, ps = case["rows"], case["page"]
    lengths = rng.permutation(_spread(case["longest"], rows, even=False)) - 1          # some are new: no tokens yet
    counts = rng.permutation(_spread(case["new"], rows, even=True))
    if not case["packed"]:
        counts[(np.arange(rows) % 16 == 15) & (rows > 16)] = 0                         # sequences that have ended
    used, after = -(-lengths // ps), -(-(lengths + counts) // ps)
    width = (case["longest"] + case["new"]) // ps + 1
    held = int(used.sum())
    free = int((after - used).sum())
    ids = rng.permutation(held + 2 * free + 7)
    tables = np.zeros((rows, width), dtype=np.int64)
    column = np.arange(width)
    inside = column[None, :] < used[:, None]
    tables[inside] = ids[((np.cumsum(used) - used)[:, None] + column[None, :])[inside]]
    return dict(case=case, tables=_dev(tables, torch.int32), lens=_dev(lengths, torch.int32), counts=_dev(counts, torch.int32),
                free=_dev(ids[held:], torch.int32), taken=_dev(np.array([5]), torch.int32),
                tokens=int(counts.sum()) if case["packed"] else None)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


def run(state):
    return (_attend if state["case"]["kind"] == "attend" else _extend)(state)


def _attend(s):
    if own:
        from deltazip_amd import prefix_attention
        return prefix_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], starts=s["starts"], groups=s["groups"], prefixes=s["prefixes"],
                                scale=s["scale"])
    case, lens = s["case"], s["lens"].long()
    rows, heads, kv, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    # queries of a row side by side: [rows, most, heads, dim]
    if s["starts"] is None:
        q, counts = s["q"][:, None], torch.ones_like(lens)
    else:
        first, counts = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
        i = torch.arange(s["most"], device=DEV)
        real = i[None, :] < counts[:, None]
        at = torch.where(real, first[:, None] + i[None, :], torch.zeros_like(first)[:, None])
        q = s["q"][at]
    q = q.float() * s["scale"]
    n = q.shape[1]
    # [rows, kv_heads, new tokens x heads of a key, dim]
    q = q.view(rows, n, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, dim)
    # pages gathered, in 32 bits: [rows, kv_heads, tokens, dim]
    k = s["k"][s["tables"].long()].permute(0, 2, 4, 1, 3).reshape(rows, kv, dim, -1).float()
    scores = torch.matmul(q, k)
    del k
    t = torch.arange(scores.shape[-1], device=DEV)
    seen = lens[:, None] - counts[:, None] + 1 + torch.arange(n, device=DEV)          # tokens that each new one sees
    seen = torch.where(lens[:, None] > 0, seen, torch.zeros_like(seen))
    hidden = (t >= seen[..., None])[:, None, :, None, :]
    scores = scores.view(rows, kv, n, heads // kv, -1).masked_fill_(hidden, -3e38)
    p = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True))).masked_fill_(hidden, 0.0)
    total = p.sum(-1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    v = s["v"][s["tables"].long()].permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, dim).float()
    y = torch.matmul(p.view(rows, kv, n * (heads // kv), -1), v).view(rows, kv, n, heads // kv, dim) / total
    y = y.permute(0, 2, 1, 3, 4).reshape(rows, n, heads, dim).to(s["q"].dtype)
    if s["starts"] is None:
        return y[:, 0]
    token = torch.arange(s["q"].shape[0], device=DEV)
    row = torch.searchsorted(s["starts"], token, right=True, out_int32=True).long() - 1
    return y[row, token - first[row]]


def _extend(s):
    case, ps = s["case"], s["case"]["page"]
    if own:
        from deltazip_amd import extend_tables
        made = extend_tables(s["tables"], s["lens"], s["counts"], s["free"], s["taken"], ps, tokens=s["tokens"])
        return dict(tables=s["tables"], lengths=made.lengths, taken=made.taken, starts=made.starts, positions=made.positions, slots=made.slots)
    n, c, tables = s["lens"].long(), s["counts"].long(), s["tables"]
    used, after = (n + ps - 1) // ps, (n + c + ps - 1) // ps
    need = after - used
    first = torch.cumsum(need, 0) - need + s["taken"].long()
    column = torch.arange(tables.shape[1], device=DEV)
    added = (column >= used[:, None]) & (column < after[:, None])
    at = torch.where(added, first[:, None] + column - used[:, None], torch.zeros_like(first)[:, None])
    tables.copy_(torch.where(added, s["free"][at], tables))
    starts = torch.cat((torch.zeros_like(c[:1]), torch.cumsum(c, 0)))
    if case["packed"]:
        row = torch.repeat_interleave(torch.arange(case["rows"], device=DEV), c, output_size=s["tokens"])
        positions = n[row] + torch.arange(s["tokens"], device=DEV) - starts[row]
        slots = tables[row, positions // ps].long() * ps + positions % ps
    else:
        starts = torch.arange(case["rows"] + 1, device=DEV)          # a place a row
        positions = torch.where(c > 0, n, torch.zeros_like(n))
        page = torch.gather(tables, 1, (positions // ps)[:, None])[:, 0].long()
        slots = torch.where(c > 0, page * ps + positions % ps, torch.full_like(n, -1))
    return dict(tables=tables, lengths=(n + c).int(), taken=(s["taken"] + need.sum()).int(), starts=starts.int(), positions=positions, slots=slots)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------


def work(case):
    rows, ps = case["rows"], case["page"]
    if case["kind"] == "tables":
        counts = _spread(case["new"], rows, even=True)
        tokens = int(counts.sum()) if case["packed"] else rows
        # lengths and counts read, lengths and starts written; positions and slots; free pages to tables, and the page a token falls in
        return dict(bytes=16 * rows + 16 * tokens + 8 * tokens / ps + 4 * rows, flops=0)
    heads, kv, dim, prefix = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    suffix, new = _sizes(case)
    alive = suffix > 0
    stored = case["groups"] * prefix + int(suffix.sum())
    # a row's new tokens see its prefix, its older tokens and each other, one more each
    pairs = int((new * (prefix + suffix) - new * (new - 1) // 2)[alive].sum())
    tokens = rows if case["new"] == 1 else int(new.sum())
    return dict(bytes=4 * stored * kv * dim + 4 * tokens * heads * dim + 4 * stored / ps + 8 * rows, flops=4 * pairs * heads * dim)


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_extend(s)


def _exact_attend(s):
    case = s["case"]
    heads, kv, dim, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows = case["rows"]
    starts = list(range(rows + 1)) if s["starts"] is None else s["starts"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, n in enumerate(s["lens"].tolist()):
        a, b = starts[r], starts[r + 1]
        if n == 0 or b == a:
            continue
        t = torch.arange(n, device=DEV)
        page = s["tables"][r].long()[t // ps]
        for h in range(kv):
            k, v = (p[page, h, t % ps].double() for p in (s["k"], s["v"]))
            kt = k.t().contiguous()
            for j in range(h * (heads // kv), (h + 1) * (heads // kv)):
                x = s["q"][a:b, j].double() @ kt * s["scale"]
                if b - a > 1:
                    x.masked_fill_(t[None, :] > torch.arange(n - (b - a), n, device=DEV)[:, None], -math.inf)
                out[a:b, j] = torch.softmax(x, -1) @ v
    return out


def _exact_extend(s):
    case, ps = s["case"], s["case"]["page"]
    tables, lens, counts = s["tables"].cpu().numpy().copy(), s["lens"].tolist(), s["counts"].tolist()
    free, taken = s["free"].tolist(), s["taken"].tolist()[0]
    starts, positions, slots = [0], [], []
    for r, (n, c) in enumerate(zip(lens, counts)):
        for t in range(n, n + c):
            if t % ps == 0:
                tables[r, t // ps] = free[taken]
                taken += 1
            positions.append(t)
            slots.append(int(tables[r, t // ps]) * ps + t % ps)
        if not case["packed"] and c == 0:
            positions.append(0)
            slots.append(-1)
        starts.append(len(positions))
    return dict(tables=torch.from_numpy(tables), lengths=torch.tensor([n + c for n, c in zip(lens, counts)], dtype=torch.int32),
                taken=torch.tensor([taken], dtype=torch.int32), starts=torch.tensor(starts, dtype=torch.int32),
                positions=torch.tensor(positions), slots=torch.tensor(slots))
