"""Attention of several new tokens of a row behind prefixes that rows share, and tables made on the device, against restatements in 64 bits
(oracle/paged_ref.py)."""
import ctypes as C
import random

import pytest
import torch

from oracle import paged_ref as ref

TYPES = [torch.float16, torch.bfloat16]


# ---------------------------------------------------------------------------------------------
# the restatement's own pins, and the C entries' checks
# ---------------------------------------------------------------------------------------------


def test_oracle_of_tokens_as_rows():
    tables = torch.tensor([[5, 1], [6, 2], [7, 3], [0, 0]], dtype=torch.int32)
    row, length, tab = ref.tokens_as_rows([0, 2, 3, 6, 6], [10, 9, 12, 0], tables, torch.tensor([0, 2, 4]), torch.tensor([8, 100]), 8)
    assert row == [0, 0, 1, 2, 2, 2] and length.tolist() == [9, 10, 9, 10, 11, 12]
    assert tab.tolist() == [[5, 1], [5, 1], [5, 2], [7, 3], [7, 3], [7, 3]]
    row, length, _ = ref.tokens_as_rows([0, 3], [2], tables[:1])
    assert length.tolist() == [0, 1, 2]


def test_oracle_of_tables():
    got = ref.extend_tables([[4, 0, 0], [0, 0, 0]], [6, 0], [4, 1], [9, 8, 7], 1, 8, tokens=7)
    assert got == ([[4, 8, 0], [7, 0, 0]], [10, 1], 3, [0, 4, 5], [6, 7, 8, 9, 0, 0, 0], [38, 39, 64, 65, 56, -1, -1])
    assert ref.extend_tables([[4, 0]], [8], [1], [9], 1, 8) is None and ref.extend_tables([[4]], [8], [1], [9], 0, 8) is None
    assert ref.extend_tables([[4, 0], [0, 0]], [7, 0], [1, 0], [], 0, 8) == ([[4, 0], [0, 0]], [8, 0], 0, [0, 1, 2], [7, 0], [39, -1])


def test_c_entry_points_check_their_arguments(dzlib):
    from deltazip_amd import paged
    P = 0x1000
    names = ("bytes q k v tables lengths starts groups prefixes out work status work_bytes num_pages q_row q_head k_page k_head k_token v_page v_head "
             "v_token out_row out_head table_row tokens rows groups_n heads kv_heads dim page_size pages_per_row dtype scale").split()
    ok = dict(zip(names, [paged._PREFIX.size] + [P] * 11 + [1 << 34, 10] + [4096, 128, 65536, 2048, 128, 65536, 2048, 128, 4096, 128, 4]
                  + [5, 3, 1, 32, 32, 128, 16, 40, 0, 0.1]))
    call = lambda **kw: dzlib.dz_prefix_attention(paged._PREFIX.pack(*{**ok, **kw}.values()), None)
    assert dzlib.dz_prefix_attention(None, None) == -1 and call(bytes=8) == -1
    for name in ("q", "k", "v", "tables", "lengths", "starts", "groups", "prefixes", "out", "status"):
        assert call(**{name: 0}) == -1, name
    for kw in (dict(heads=33), dict(kv_heads=0), dict(dim=130), dict(dim=264), dict(dim=0), dict(page_size=12), dict(page_size=4), dict(page_size=2048),
               dict(rows=-1), dict(rows=(1 << 20) + 1), dict(tokens=-1), dict(tokens=1 << 26), dict(groups_n=-1), dict(groups_n=2049), dict(pages_per_row=-1),
               dict(pages_per_row=1 << 28), dict(num_pages=0), dict(num_pages=1 << 31), dict(table_row=-1), dict(heads=8192, kv_heads=8192)):
        assert call(**kw) == -12, kw
    for kw in (dict(q=P + 8), dict(k=P + 2), dict(out=P + 4), dict(lengths=P + 2), dict(starts=P + 1), dict(prefixes=P + 2), dict(k_token=132), dict(v_page=-8)):
        assert call(**kw) == -10, kw
    assert call(dtype=2) == -1 and call(work=0) == -8 and call(work_bytes=64) == -8 and call(work=P + 4) == -8
    assert call(tokens=0, q=0) == 0 and call(tokens=0, rows=0, starts=0, q=0) == 0
    need = lambda *a: dzlib.dz_prefix_attention_bytes(*a)
    assert need(5, 3, 1, 32, 32, 128) >= need(5, 3, 0, 32, 32, 128) > 0 == need(5, 3, 1, 33, 32, 128) == need(-1, 3, 1, 32, 32, 128)

    names = ("bytes tables lengths counts free taken lengths_out taken_out starts positions slots status table_row rows pages_per_row page_size free_n "
             "tokens packed").split()
    ok = dict(zip(names, [paged._EXTEND.size] + [P] * 11 + [4, 3, 4, 16, 20, 7, 1]))
    call = lambda **kw: dzlib.dz_extend_tables(paged._EXTEND.pack(*{**ok, **kw}.values()), None)
    assert dzlib.dz_extend_tables(None, None) == -1 and call(bytes=8) == -1
    for name in ("tables", "lengths", "counts", "free", "taken", "lengths_out", "taken_out", "starts", "positions", "slots", "status"):
        assert call(**{name: 0}) == -1, name
    for kw in (dict(rows=-1), dict(rows=(1 << 20) + 1), dict(pages_per_row=-1), dict(pages_per_row=1 << 27), dict(page_size=12), dict(page_size=4),
               dict(page_size=2048), dict(free_n=-1), dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(packed=0), dict(table_row=-1)):
        assert call(**kw) == -12, kw
    for kw in (dict(tables=P + 2), dict(lengths=P + 1), dict(taken=P + 2), dict(slots=P + 4), dict(positions=P + 4)):
        assert call(**kw) == -10, kw


def test_host_tensors_are_refused(dzlib):
    from deltazip_amd import extend_tables, prefix_attention
    q, pages = torch.zeros(2, 2, 16, dtype=torch.float16), torch.zeros(3, 2, 8, 16, dtype=torch.float16)
    i32 = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: prefix_attention(q, pages, pages, i32[:, None], i32), lambda: extend_tables(i32[:, None], i32, i32, i32, i32[:1], 16)):
        with pytest.raises(ValueError, match="GPU"):
            call()


# ---------------------------------------------------------------------------------------------
# the cache: groups, several new tokens, runs
# ---------------------------------------------------------------------------------------------


def _cache(device="cpu", pages=200, page_size=8, monkeypatch=None, **kw):
    from deltazip_amd import PagedKVCache, kv_cache
    if monkeypatch is not None:
        def copy(pool, pairs):
            pool[:, [b for _, b in pairs]] = pool[:, [a for a, _ in pairs]]

        def extend(tables, lengths, counts, free, taken, page_size, tokens=None, out=None):
            made = ref.extend_tables(tables.tolist(), lengths.tolist(), counts.tolist(), free.tolist(), int(taken), page_size, tokens)
            if made is None:
                made = tables.tolist(), lengths.tolist(), int(taken), [0] * (len(lengths) + 1), [0] * len(out.slots), [-1] * len(out.slots)
            tables.copy_(torch.tensor(made[0], dtype=torch.int32).view_as(tables))
            for t, x in zip(out, (made[1], [made[2]], *made[3:])):
                t.copy_(torch.tensor(x, dtype=t.dtype))
            return out
        monkeypatch.setattr(kv_cache, "copy_pages", copy)
        monkeypatch.setattr(kv_cache, "extend_tables", extend)
    return PagedKVCache(1, pages, page_size, 1, 8, max_tokens=400, device=device, **kw)


def test_neighbours_that_share_pages_are_groups(monkeypatch):
    cache = _cache(monkeypatch=monkeypatch)
    cache.add("a", 40)
    cache.add("z", 40)
    for i in range(4):
        cache.fork("a", i)
    cache.extend([0, 1, 2, 3], 9)                    # (their sixth pages are their own)
    cache.fork(3, "late")
    cache.extend(["late", "z"])
    b = cache.batch([0, 1, 2, "z", 3, "late", None], prefix=True)
    assert b.groups.tolist() == [0, 3, 4, 6, 7, 7, 7, 7] and b.prefixes.tolist() == [40, 0, 48, 0, 0, 0, 0] and b.starts is None
    # a row joins where that spares as many pages as the group without it did
    b = cache.batch([3, "late", 0, 1], prefix=True)
    assert b.groups.tolist() == [0, 4, 4, 4, 4] and b.prefixes.tolist() == [40, 0, 0, 0]
    again = cache.batch([1, None, "z", 2], prefix=True, out=b)
    assert again.groups is b.groups and b.groups.tolist() == [0, 4, 4, 4, 4] and b.prefixes.tolist() == [0, 0, 0, 0]
    assert cache.batch([0, 1]).groups is None and cache.batch([], prefix=True).groups.tolist() == [0]
    for bad in (dict(out=b), dict(out=cache.batch([0, 1, 2, 3]), prefix=True), dict(out=b, prefix=True, tokens=[1] * 4)):
        with pytest.raises(ValueError):
            cache.batch([1, None, "z", 2], **bad)


def test_more_groups_than_a_call_takes(monkeypatch):
    from deltazip_amd import kv_cache
    monkeypatch.setattr(kv_cache, "MAX_GROUPS", 2)
    cache = _cache(monkeypatch=monkeypatch)
    for i in range(3):
        cache.add(("p", i), 16)
        for j in range(2):
            cache.fork(("p", i), (i, j))
    seqs = [(i, j) for i in range(3) for j in range(2)]
    run = cache.run(seqs, 1, prefix=True)
    b = run.step()
    assert b.groups.tolist() == [0, 2, 4] and b.prefixes.tolist() == [16, 16]            # (the others read their own)
    run.finish()
    b = cache.batch(seqs, prefix=True)
    assert b.groups.tolist() == [0, 2, 4] and b.prefixes.tolist() == [16, 16]


@pytest.mark.parametrize("seed", range(10))
def test_groups_hold_what_their_rows_share(seed):
    cache, rng = _cache(), random.Random(seed)
    rows, w = rng.randrange(1, 30), 12
    import numpy as np
    used = np.array([rng.choice([0, rng.randrange(1, w + 1)]) for _ in range(rows)])
    tables = np.zeros((rows, w), dtype=np.int32)
    for r in range(rows):
        if used[r]:
            keep = rng.choice([0, rng.randrange(0, used[r] + 1)]) if r and used[r - 1] else 0
            tables[r, :used[r]] = [tables[r - 1, i] if i < min(keep, used[r - 1]) else 100 * r + i + 1 for i in range(used[r])]
    bounds, sizes = cache._groups_of(tables, used)
    assert bounds[0] == 0 and bounds[-1] == rows and len(sizes) == len(bounds) - 1 and (np.diff(bounds) > 0).all()
    for a, b, n in zip(bounds, bounds[1:], sizes):
        assert n % 8 == 0 and (n == 0 or (b - a > 1 and (used[a:b] >= n // 8).all() and (tables[a:b, :n // 8] == tables[a, :n // 8]).all()))


def test_batches_of_several_new_tokens(monkeypatch):
    cache = _cache(monkeypatch=monkeypatch)
    cache.add("p", 21)
    cache.add("q", 5)
    cache.extend(["q"], 4)
    b = cache.batch(["p", None, "q"], tokens=[21, 0, 4])
    assert b.starts.tolist() == [0, 21, 21, 25] and b.lengths.tolist() == [21, 0, 9]
    assert b.positions.tolist() == list(range(21)) + [5, 6, 7, 8]
    where = {x: cache.slots(x)[1].tolist() for x in "pq"}
    assert b.slots.tolist() == where["p"] + where["q"][5:]
    assert cache.batch([None, "q"], tokens=[0, 0]).positions.numel() == 0
    for bad in ([22, 0, 1], [1, 1, 1], [1, 0], [-1, 0, 1]):
        with pytest.raises(ValueError):
            cache.batch(["p", None, "q"], tokens=bad)
    cache.fork("p", "r")
    with pytest.raises(ValueError, match="other sequences"):
        cache.batch(["r"], tokens=[3])
    cache.extend(["r"], 12)
    assert cache.batch(["r"], tokens=[12]).positions.tolist() == list(range(21, 33))


@pytest.mark.parametrize("seed", range(6))
def test_runs_give_back_what_they_were(monkeypatch, seed):
    """Against the same steps by the host: the same tokens in the same places of each sequence, and the same number of free pages."""
    rng = random.Random(seed)
    cache = _cache(monkeypatch=monkeypatch)
    for i in range(5):
        cache.add(i, rng.randrange(0, 30))
    cache.add("base", 20)
    for x in "ab":
        cache.fork("base", x)
    seqs = ["a", 0, None, 1, "b", 2]
    before = {x: cache.length(x) for x in seqs if x is not None}
    steps = rng.randrange(1, 40)
    kept = {x: cache.pages(x) for x in ("base", 3, 4)}
    free = cache.free_pages
    run = cache.run(seqs, steps)
    lost = rng.randrange(0, steps + 1)
    for i in range(lost):
        if i == lost // 2:
            run.counts[3] = 0
        b = run.step()
        assert b.block_tables is run._tables
        for r, x in enumerate(seqs):
            n = int(b.lengths[r])
            if x is None or (r == 3 and i >= lost // 2):
                assert int(b.slots[r]) == -1
            else:
                assert n == before[x] + i + 1 and int(b.positions[r]) == n - 1
                assert int(b.slots[r]) == int(b.block_tables[r, (n - 1) // 8]) * 8 + (n - 1) % 8
    for call in (lambda: cache.extend(["a"]), lambda: cache.free(0), lambda: cache.fork(1, "new"), lambda: cache.batch(["b"]), lambda: cache.compact(),
                 lambda: cache.truncate(2, 0), lambda: cache.run([0], 1), lambda: cache.length("a"), lambda: cache.slots(0)):
        with pytest.raises(ValueError, match="run"):
            call()
    cache.extend([3, 4], 2)                          # others go on
    cache.truncate(3, cache.length(3) - 2)
    cache.truncate(4, cache.length(4) - 2)
    run.finish()
    run.finish()
    with pytest.raises(ValueError, match="finished"):
        run.step()
    held = [p for x in list(before) + ["base", 3, 4] for p in cache.pages(x)]
    for x, n in before.items():
        assert cache.length(x) == n + (lost // 2 if x == 1 else lost)
        assert len(cache.pages(x)) == -(-cache.length(x) // 8)
    assert {x: cache.pages(x) for x in kept} == kept
    assert cache.free_pages == cache.num_pages - len(set(held))
    for x in list(before) + ["base", 3, 4]:
        cache.free(x)
    assert cache.free_pages == cache.num_pages and sorted(cache._free) == list(range(cache.num_pages)) and cache._spared == 0


def test_runs_that_do_not_fit_change_nothing(monkeypatch):
    from deltazip_amd import kv_cache
    cache = _cache(monkeypatch=monkeypatch, pages=6)
    cache.add("a", 20)
    cache.add("b", 3)
    with pytest.raises(kv_cache.OutOfPages):
        cache.run(["a", "b"], 30)
    for call in (lambda: cache.run(["a"], 0), lambda: cache.run(["a", "a"], 1), lambda: cache.run(["x"], 1), lambda: cache.run(["a"], 1000)):
        with pytest.raises(ValueError):
            call()
    monkeypatch.setattr(kv_cache, "TableStep", None)               # (as where the device has no memory left)
    with pytest.raises(TypeError):
        cache.run(["a", "b"], 8)
    assert cache.free_pages == 2 and cache.length("a") == 20 and cache.length("b") == 3
    cache.extend(["a", "b"])


# ---------------------------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------------------------


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _tables_problem(rng, rows, longest, most, ps, packed, spare=0):
    lengths = [rng.choice([0, 1, ps - 1, ps, ps + 1, rng.randrange(0, longest + 1)]) for _ in range(rows)]
    lengths = [min(n, longest) for n in lengths]
    counts = [rng.choice([0, 1, most, rng.randrange(0, most + 1)]) if packed else rng.randrange(0, 2) for _ in range(rows)]
    width = max([1] + [-(-(n + c) // ps) for n, c in zip(lengths, counts)]) + rng.randrange(0, 2)
    used = [-(-n // ps) for n in lengths]
    need = sum(-(-(n + c) // ps) - u for n, c, u in zip(lengths, counts, used))
    ids = rng.sample(range(1 << 20), sum(used) + need + 8)
    tables, at = [], 0
    for u in used:
        tables.append(ids[at:at + u] + [-7] * (width - u))
        at += u
    taken = rng.randrange(0, 4)
    return tables, lengths, counts, ids[at:at + need + taken + spare], taken


def _hold_tables(dev, tables, lengths, counts, free, taken, ps, tokens):
    from deltazip_amd import extend_tables, ops
    want = ref.extend_tables(tables, lengths, counts, free, taken, ps, tokens)
    width = len(tables[0]) if tables else 1
    wide = torch.full((len(tables), width + 3), 99, dtype=torch.int32, device=dev)       # (rows of a wider tensor)
    wide[:, :width] = _i32(tables, dev).view(len(tables), width)
    ins = [_i32(x, dev) for x in (lengths, counts, free, [taken])]
    got = extend_tables(wide[:, :width], *ins, ps, tokens=tokens)
    assert [t.tolist() for t in ins] == [lengths, counts, free, [taken]] and (wide[:, width:] == 99).all()
    n = len(got.slots)
    if want is None:
        with pytest.raises(ops.DeltaKernelError, match="paged"):
            ops.poll_status(wait=True)
        want = tables, lengths, taken, [0] * (len(tables) + 1), [0] * n, [-1] * n
    else:
        ops.poll_status(wait=True)
    assert wide[:, :width].tolist() == want[0] and got.lengths.tolist() == want[1] and got.taken.tolist() == [want[2]]
    assert got.starts.tolist() == want[3] and got.positions.tolist() == want[4] and got.slots.tolist() == want[5]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1, 2, 63, 64, 65, 300, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("packed", [False, True])
def test_tables(dev, rows, packed):
    rng = random.Random(rows + packed)
    for ps in (8, 64):
        p = _tables_problem(rng, rows, 300, 40, ps, packed, spare=rng.randrange(0, 3))
        _hold_tables(dev, *p, ps, sum(p[2]) + rng.choice([0, 0, 13]) if packed else None)


@pytest.mark.gpu
def test_tables_of_long_prompts(dev):
    rng = random.Random(3)
    for rows, most, ps in ((1, 9000, 16), (1, 4096, 1024), (1, 4097, 8), (5, 5000, 32), (2, 20000, 8), (40, 700, 16)):
        p = _tables_problem(rng, rows, 3000, most, ps, True)
        p[2][0] = most
        width = max(-(-(n + c) // ps) for n, c in zip(p[1], p[2]))
        p = ([t + [-7] * (width - len(t)) for t in p[0]], p[1], p[2], list(range(5000, 5000 + 2 * width * rows)), p[4])
        _hold_tables(dev, *p, ps, sum(p[2]) + 5)


@pytest.mark.gpu
def test_tables_that_do_not_fit_are_left_as_they_were(dev):
    base = ([[1, 2, -7], [3, -7, -7], [4, 5, 6]], [9, 8, 17], [1, 1, 1], [10, 11, 12], 0)
    _hold_tables(dev, *base, 8, None)
    for change in ({2: [1, 2, 1]}, {2: [1, -1, 1]}, {1: [9, -1, 17]}, {1: [9, 8, 24]}, {3: []}, {4: 3}, {4: -1}, {4: 2**31 - 1}, {1: [9, 2**31 - 1, 3]},
                   {2: [2**31 - 1] * 3}):
        p = [change.get(i, x) for i, x in enumerate(base)]
        _hold_tables(dev, *p, 8, None)
        _hold_tables(dev, *p, 8, 3)
    _hold_tables(dev, *base, 8, 3)
    _hold_tables(dev, *base, 8, 2)
    _hold_tables(dev, [[-7] * 600] * 3, [0, 0, 0], [4700, 4700, 1], list(range(1200)), 0, 8, 9400)      # one place short, three workgroups
    _hold_tables(dev, [[-7] * 600] * 3, [0, 0, 0], [4700, 4700, 1], list(range(1200)), 0, 8, 9401)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [256, 512, 1024])
def test_tables_of_counts_whose_sum_passes_32_bits(dev, rows):
    """2^24 tokens a row: 256 rows' sum is 2^32, which 32 bits would take for 0, and there are pages for them."""
    from deltazip_amd import extend_tables, ops
    most, ps = 1 << 24, 1024
    tables = torch.full((rows, most // ps), -7, dtype=torch.int32, device=dev)
    lengths, counts = (torch.full((rows,), x, dtype=torch.int32, device=dev) for x in (0, most))
    free, taken = torch.arange(rows * (most // ps), dtype=torch.int32, device=dev), _i32([0], dev)
    got = extend_tables(tables, lengths, counts, free, taken, ps, tokens=most)
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(wait=True)
    assert bool((tables == -7).all()) and got.lengths.tolist() == [0] * rows and got.taken.tolist() == [0]
    assert got.starts.tolist() == [0] * (rows + 1) and not bool(got.positions.any()) and bool((got.slots == -1).all())


@pytest.mark.gpu
def test_tables_a_page_below_zero_stores_nothing(dev):
    from deltazip_amd import extend_tables, ops
    tables = _i32([[-3, 0], [1, 0]], dev)
    got = extend_tables(tables, _i32([4, 8], dev), _i32([1, 1], dev), _i32([-1], dev), _i32([0], dev), 8)
    assert got.slots.tolist() == [-1, -1]
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(wait=True)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [None, 10000])
def test_tables_step_in_place_and_from_a_graph(dev, tokens):
    """Lengths and pages taken over the inputs: every call, and every replay, goes one step on."""
    from deltazip_amd import TableStep, extend_tables
    rng = random.Random(7)
    rows, ps, width = 37, 8, 400
    lengths = [rng.randrange(0, 30) for _ in range(rows)]
    counts = [rng.randrange(0, 2) if tokens is None else rng.randrange(0, 200) for _ in range(rows)]
    used = [-(-n // ps) for n in lengths]
    free = rng.sample(range(1 << 20), 6000)
    tables = [[1000000 + 400 * r + i if i < u else -7 for i in range(width)] for r, u in enumerate(used)]
    places = rows if tokens is None else tokens
    tab, ln, ct, fr, tk = (_i32(x, dev) for x in (tables, lengths, counts, free, [0]))
    out = TableStep(ln, tk, torch.empty(rows + 1, dtype=torch.int32, device=dev), *torch.empty(2, places, dtype=torch.int64, device=dev))
    step = lambda: extend_tables(tab, ln, ct, fr, tk, ps, tokens=tokens, out=out)
    assert step() is out
    graph, state = torch.cuda.CUDAGraph(), (tables, lengths, 0)
    for i in range(6):
        state = ref.extend_tables(state[0], state[1], counts, free, state[2], ps, tokens)
        if i:
            graph.replay()
        assert tab.tolist() == state[0] and ln.tolist() == state[1] and tk.tolist() == [state[2]]
        assert out.starts.tolist() == state[3] and out.positions.tolist() == state[4] and out.slots.tolist() == state[5]
        if i == 0:
            with torch.cuda.graph(graph):
                step()


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------


def _problem(dev, dtype, prefixes, suffixes, news, groups, heads, kv, dim, ps, seed=0, spread=1.5, poison=True):
    """Pages in random order; what no row sees holds NaN, what tables hold behind a length -- or under a prefix that is read through another row's -- is no page.
    prefixes: of each group; suffixes, news: of each row (a suffix of None: an empty row)."""
    g = torch.Generator().manual_seed(seed)
    rows = len(suffixes)
    lengths = [0] * rows
    for a, b, p in zip(groups, groups[1:], prefixes):
        for r in range(a, b):
            lengths[r] = 0 if suffixes[r] is None else p + suffixes[r]
    for r in list(range(groups[0])) + list(range(groups[-1], rows)):
        lengths[r] = suffixes[r] or 0
    used = [-(-n // ps) for n in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g)
    k, v = (torch.randn(pages, kv, ps, dim, generator=g).to(dtype) for _ in range(2))
    width = max(used + [0]) + 2
    tables = torch.full((rows, width), 0x7fffffff, dtype=torch.int32)
    seen = torch.zeros(pages, ps, dtype=torch.bool)
    at = 0
    for r, (n, u) in enumerate(zip(lengths, used)):
        tables[r, :u] = order[at:at + u].int()
        at += u
    starts = [0]
    for c in news:
        starts.append(starts[-1] + c)
    for a, b, p in zip(groups, groups[1:], prefixes):
        alive = [r for r in range(a, b) if lengths[r] > 0 and news[r] > 0]
        for r in alive[1:]:
            tables[r, :p // ps] = tables[alive[0], :p // ps]
            if p % ps:                                       # a copy of the page that the prefix ends in
                for x in (k, v):
                    x[tables[r, p // ps].long(), :, :p % ps] = x[tables[alive[0], p // ps].long(), :, :p % ps]
    for r, n in enumerate(lengths):
        t = torch.arange(n)
        seen[tables[r].long()[t // ps], t % ps] = True
    if poison:
        for x in (k, v):
            x.masked_fill_(~seen[:, None, :, None], float("nan"))
    q = (spread * torch.randn(starts[-1], heads, dim, generator=g)).to(dtype)
    return [x.to(dev) for x in (q, k, v, tables, torch.tensor(lengths, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32),
                                torch.tensor(groups, dtype=torch.int32), torch.tensor(prefixes, dtype=torch.int32))]


def _hold(got, q, k, v, tables, lengths, starts, groups=None, prefixes=None, scale=None, most_rows=10**9):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    row, length, tab = ref.tokens_as_rows(starts, lengths, tables, groups, prefixes, k.shape[2])
    pick = list(range(len(row))) if len(row) <= most_rows else sorted(random.Random(1).sample(range(len(row)), most_rows))
    want, size, most = ref.attention(q[pick], k, v, tab[pick], length[pick], scale)
    largest = max([float(x.nan_to_num(0, 0, 0).abs().max()) for x in v.split(4096)])
    bound = ref.prefix_bound(want, size, most, q.dtype, q.shape[2], max(1, int(length.max()) if len(length) else 1), largest)
    y = got.double().cpu()[pick]
    off = (y - want).abs()
    assert torch.isfinite(y).all()
    assert (off <= bound).all(), f"off by up to {(off / bound).max():.2f} of the bound at {(off / bound).argmax()}"
    assert (got[len(row):] == 0).all()


def _run(p, single=False, shared=True, **kw):
    from deltazip_amd import prefix_attention
    q, k, v, tables, lengths, starts, groups, prefixes = p
    return prefix_attention(q, k, v, tables, lengths, starts=None if single else starts, groups=groups if shared else None,
                            prefixes=prefixes if shared else None, **kw)


HEADS = [(4, 4, 128), (8, 2, 64), (7, 1, 80), (20, 1, 128), (6, 3, 256), (33, 1, 8), (5, 5, 96), (32, 2, 192), (3, 1, 24), (16, 1, 256), (6, 2, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("ps", [8, 16, 64])
def test_prefix_of_single_tokens(dev, dtype, heads, kv, dim, ps):
    suffixes = [1, 5, None, 9, 64, 65, 300, 1, 1, 130, None, 7, 40, 3]
    p = _problem(dev, dtype, [96, 333, 64], suffixes, [1] * 14, [0, 7, 10, 13], heads, kv, dim, ps)
    for single in (True, False):                                   # (starts that say the same; without them so few rows go one by one)
        got = _run(p, single=single)
        _hold(got, *p)
        assert torch.equal(got, _run(p, single=single))
    assert torch.equal(_run(p, single=True, shared=False), _run(p[:3] + [p[3].clone()] + p[4:], single=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("ps", [8, 64])
def test_prefix_of_several_tokens(dev, dtype, heads, kv, dim, ps):
    suffixes, news = [5, 70, None, 130, 8, 300, 2, 33], [5, 6, 0, 130, 2, 17, 0, 33]
    p = _problem(dev, dtype, [200, 77], suffixes, news, [0, 5, 8], heads, kv, dim, ps)
    _hold(_run(p), *p)
    _hold(_run(p, shared=False), *p[:6])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,prefix,heads,kv,dim,ps", [(40, 5003, 8, 8, 128, 16), (3, 20011, 8, 1, 128, 16), (17, 9000, 4, 4, 64, 256), (64, 3000, 16, 2, 256, 8),
                                                       (2, 40000, 2, 2, 80, 1024)])
def test_prefix_of_long_contexts(dev, dtype, rows, prefix, heads, kv, dim, ps):
    rng = random.Random(rows)
    p = _problem(dev, dtype, [prefix], [rng.randrange(1, 600) for _ in range(rows)], [1] * rows, [0, rows], heads, kv, dim, ps)
    _hold(_run(p), *p)
    _hold(_run(p, single=True), *p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,earlier,heads,kv,dim", [(1000, 0, 4, 4, 128), (1025, 513, 8, 1, 64), (2047, 0, 6, 2, 80), (600, 5000, 2, 2, 256)])
def test_prompts(dev, dtype, new, earlier, heads, kv, dim):
    p = _problem(dev, dtype, [0], [new + earlier], [new], [0, 1], heads, kv, dim, 16)
    _hold(_run(p, shared=False), *p[:6], most_rows=150)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025, 1500])
def test_prefix_of_any_number_of_rows(dev, rows):
    rng = random.Random(rows)
    p = _problem(dev, torch.float16, [48], [rng.choice([None, 1, 2, 30]) for _ in range(rows)], [1] * rows, [0, rows], 2, 1, 32, 8)
    _hold(_run(p), *p, most_rows=200)
    _hold(_run(p, single=True), *p, most_rows=200)


@pytest.mark.gpu
def test_prefix_of_many_groups(dev):
    rng = random.Random(1)
    rows, n = 1500, 700
    groups = [0] + sorted(rng.choices(range(rows + 1), k=n - 1)) + [rows]          # empty ones among them
    p = _problem(dev, torch.bfloat16, [rng.randrange(0, 90) for _ in range(n)], [rng.choice([None, 1, 20]) for _ in range(rows)],
                 [rng.randrange(0, 3) for _ in range(rows)], groups, 2, 1, 16, 8)
    # (a row's new tokens may be more than its own: the prefix is cut)
    _hold(_run(p), *p, most_rows=300)


@pytest.mark.gpu
def test_prefix_longer_than_rows_see_is_cut(dev):
    # (one of row 0's new tokens is in the prefix: of its 101 tokens the first of them sees 100, and no more are the same as the others')
    p = _problem(dev, torch.float16, [100], [1, 4, 30], [2, 4, 2], [0, 3], 4, 2, 64, 8)
    for prefix in (100, 101, 104, 129, 100000, 2**31 - 1):
        p[-1] = torch.tensor([prefix], dtype=torch.int32, device=dev)
        _hold(_run(p), *p)
    for prefix in (0, -5, 1, 7, 8, 63, 64, 65, 99):
        p[-1] = torch.tensor([prefix], dtype=torch.int32, device=dev)
        _hold(_run(p), *p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (40, 2, 128), (6, 3, 200)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", ["keys", "values", "both"])
def test_what_a_token_does_not_see_does_not_reach_it(dev, dtype, heads, kv, dim, bad, which):
    """Values that are not finite in a row's newest tokens: the older ones' outputs are what they are without them, the others' are not finite."""
    for news, suffixes, prefixes, groups, at in (([40, 3], [70, 9], [64], [0, 2], 60), ([200], [200], [0], [0, 1], 130), ([20] * 9, [20] * 9, [128], [0, 9], 13)):
        p = _problem(dev, dtype, prefixes, suffixes, news, groups, heads, kv, dim, 8)
        clean = _run(p)
        prefix, n = prefixes[0], int(p[4][0])
        t = prefix + at                                            # of row 0
        page = int(p[3][0, t // 8])
        for x in ((p[1],) if which == "keys" else (p[2],) if which == "values" else p[1:3]):
            x[page, 0, t % 8, 3] = bad
        got = _run(p)
        first = max(0, t - (n - news[0]))                          # the first of row 0's new tokens that sees it
        share = heads // kv
        assert torch.equal(got[:first], clean[:first]) and torch.equal(got[news[0]:], clean[news[0]:]) and torch.equal(got[:, share:], clean[:, share:])
        mine = got[first:news[0], :share]
        if which == "values":
            assert not torch.isfinite(mine[..., 3]).any() and torch.equal(mine[..., :3], clean[first:news[0], :share, :3])
            assert torch.equal(torch.isnan(mine[..., 3]), torch.full_like(mine[..., 3], bad != bad, dtype=torch.bool))
        elif bad != bad or which == "both":
            assert torch.isnan(mine).any(-1).all() or which == "both"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (40, 2, 128), (6, 3, 200)])
def test_queries_that_are_not_finite_stay_with_themselves(dev, dtype, heads, kv, dim):
    """Those of padded rows and behind the last row, and one head of one token among the others of its tile."""
    p = _problem(dev, dtype, [300], [5, None, 9, 70, None, 3], [2, 1, 1, 30, 3, 3], [0, 6], heads, kv, dim, 8)
    p[0] = torch.cat((p[0], p[0][:4]))
    want = _run(p)
    assert (want[40:] == 0).all() and (want[2:3] == 0).all() and (want[34:37] == 0).all()
    for bad in (float("nan"), float("inf")):
        p[0][40:], p[0][2:3], p[0][34:37] = bad, bad, -bad
        assert torch.equal(_run(p), want)
    p[0][8, 1] = float("nan")
    got = _run(p)
    assert torch.isnan(got[8, 1]).all()
    got[8, 1] = want[8, 1]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_prefix_scores_far_apart(dev, dtype):
    """Scores that rise, fall, are far from each other, all alike or all far below zero: the maximum of each piece is its own.  (In powers of two a
    score of -2^126 is -1.4427 2^126, which 32 bits hold; bfloat16's lowest, -2^128, is none that they hold.)"""
    from deltazip_amd import prefix_attention
    for kind in ("rising", "falling", "alike", "spike", "lowest"):
        p = _problem(dev, dtype, [700], [90] * 20, [2] * 20, [0, 20], 4, 2, 64, 16, poison=False)
        q, k = p[0], p[1]
        q.zero_()
        q[..., 0] = 1.0
        k.zero_()
        n = int(p[4][0])
        for r in range(20):
            t = torch.arange(n, device=dev)
            s = {"rising": t * 0.05, "falling": -t * 0.05, "alike": t * 0 + 3.0, "spike": (t == 350) * 60.0, "lowest": t * 0 + max(torch.finfo(dtype).min, -2.0**126)}[kind]
            k[p[3][r].long()[t // 16], :, t % 16, 0] = s.to(dtype)[:, None]
        got = _run(p, scale=1.0)
        _hold(got, *p, scale=1.0)
        _hold(_run(p, scale=-0.5), *p, scale=-0.5)
        _hold(_run(p, scale=0.0), *p, scale=0.0)


@pytest.mark.gpu
def test_prefix_strides_orders_and_places(dev):
    """Queries sliced from a projection, pages as [pages, tokens, heads, dim] and of a pool of keys and values, outputs into a wider tensor, tables into
    wider ones."""
    p = _problem(dev, torch.float16, [64], [5, 20, 70], [5, 3, 1], [0, 3], 6, 3, 64, 16)
    want = _run(p)
    q, k, v, tables = p[:4]
    wide = torch.zeros(9, 12, 80, dtype=q.dtype, device=dev)
    wide[:, 2:8, 8:72] = q
    pool = torch.zeros(k.shape[0], 16, 2, 3, 72, dtype=q.dtype, device=dev)
    pool[:, :, 0, :, :64], pool[:, :, 1, :, :64] = k.transpose(1, 2), v.transpose(1, 2)
    tab = torch.full((3, tables.shape[1] + 5), -1, dtype=torch.int32, device=dev)
    tab[:, 2:2 + tables.shape[1]] = tables
    into = torch.full((9, 12, 64), 7.0, dtype=q.dtype, device=dev)
    other = [wide[:, 2:8, 8:72], pool[:, :, 0, :, :64].transpose(1, 2), pool[:, :, 1, :, :64].transpose(1, 2), tab[:, 2:2 + tables.shape[1]]] + p[4:]
    got = _run(other, out=into[:, ::2])
    assert torch.equal(got, want) and torch.equal(into[:, ::2], want) and (into[:, 1::2] == 7.0).all()


@pytest.mark.gpu
def test_prefix_far_into_a_large_pool(dev):
    """Pages beyond 2^31 values, tables of one row far apart."""
    pages, kv, ps, dim = 70000, 2, 64, 256
    k = torch.zeros(pages, kv, ps, dim, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(0)
    far = [69999, 12, 40000, 69000, 33333, 65535]
    tables = torch.tensor([far[:3] + [far[3]], far[:3] + [far[4]]], dtype=torch.int32, device=dev)
    for page in far:
        k[page] = torch.randn(kv, ps, dim, generator=g).to(dev).bfloat16()
    q = torch.randn(2, 4, dim, generator=g).to(dev).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    from deltazip_amd import prefix_attention
    got = prefix_attention(q, k, k, tables, i32(200, 256), starts=i32(0, 1, 2), groups=i32(0, 2), prefixes=i32(192))
    _hold(got, q, k, k, tables, i32(200, 256), i32(0, 1, 2), i32(0, 2), i32(192))


@pytest.mark.gpu
def test_prefix_of_nothing(dev):
    from deltazip_amd import prefix_attention
    h = lambda *s: torch.full(s, float("nan"), dtype=torch.float16, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    kp = h(3, 2, 8, 16)
    empty = torch.zeros(0, dtype=torch.int32, device=dev)
    assert prefix_attention(h(0, 4, 16), kp, kp, i32(0, 0).view(2, 1), i32(3, 3), starts=i32(0, 0, 0)).shape == (0, 4, 16)
    assert prefix_attention(h(0, 4, 16), kp, kp, empty.view(0, 1), empty).shape == (0, 4, 16)
    # tokens of no row, rows without tokens or a table
    for got in (prefix_attention(h(5, 4, 16), kp, kp, empty.view(0, 1), empty, starts=i32(0)), prefix_attention(h(2, 4, 16), kp, kp, i32(0, 0).view(2, 1), i32(0, 0)),
                prefix_attention(h(2, 4, 16), kp, kp, empty.view(2, 0), i32(0, -3)),
                prefix_attention(h(5, 4, 16), kp, kp, i32(0, 0).view(2, 1), i32(0, 0), starts=i32(1, 2, 4), groups=i32(0, 2), prefixes=i32(8))):
        assert (got == 0).all()
    kp[1] = 0.5
    got = prefix_attention(torch.ones(6, 4, 16, dtype=torch.float16, device=dev), kp, kp, i32(1, 1).view(2, 1), i32(2, 8), starts=i32(1, 4, 5))
    assert got[:, 0, 0].tolist() == [0, 0, 0.5, 0.5, 0.5, 0]       # (three new tokens of a row of two: the first sees nothing)


@pytest.mark.gpu
def test_what_only_the_device_sees_is_reported(dev):
    from deltazip_amd import ops, prefix_attention
    p = _problem(dev, torch.float16, [64], [5, 20, 70], [5, 3, 1], [0, 3], 4, 2, 64, 16, poison=False)
    q, k, v, tables, lengths, starts, groups, prefixes = p
    want = _run(p)
    ops.poll_status(wait=True)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)

    def told():
        with pytest.raises(ops.DeltaKernelError, match="paged"):
            ops.poll_status(wait=True)

    for bad in (i32(0, 5, 4, 9), i32(-1, 5, 8, 9), i32(0, 5, 8, 10), i32(0, 5, 8, -2**31), i32(2**31 - 1, 5, 8, 9)):
        assert (prefix_attention(q, k, v, tables, lengths, starts=bad, groups=groups, prefixes=prefixes) == 0).all()
        told()
    apart = prefix_attention(q, k, v, tables, lengths, starts=starts)
    ops.poll_status(wait=True)
    for bad in (i32(0, 4), i32(-1, 3), i32(2, 1), i32(0, 2**31 - 1)):
        assert torch.equal(prefix_attention(q, k, v, tables, lengths, starts=starts, groups=bad, prefixes=prefixes), apart)
        told()
    for page in (k.shape[0], -1, 2**31 - 1):
        t = tables.clone()
        t[0, 1] = page                                             # (the prefix's: page 0 is read)
        other = tables.clone()
        other[:, 1] = 0
        assert torch.equal(_run([q, k, v, t] + p[4:]), _run([q, k, v, other] + p[4:]))
        told()
    long = lengths.clone()
    long[2] = tables.shape[1] * 16 + 1
    t = tables.clone()
    t[2, -2:] = 0
    got = _run([q, k, v, t, long] + p[5:])
    told()
    long[2] -= 1
    assert torch.equal(got, _run([q, k, v, t, long] + p[5:]))
    ops.poll_status(wait=True)
    assert torch.equal(_run(p), want)


@pytest.mark.gpu
def test_arguments_that_do_not_fit_are_refused(dev):
    from deltazip_amd import TableStep, extend_tables, prefix_attention
    h = lambda *s: torch.zeros(s, dtype=torch.float16, device=dev)
    i32, i64 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev), lambda *s: torch.zeros(s, dtype=torch.int64, device=dev)
    ok = dict(q=h(3, 4, 16), k=h(3, 2, 8, 16), v=h(3, 2, 8, 16), tab=i32(2, 3), ln=i32(2), starts=i32(3), groups=i32(2), prefixes=i32(1), out=None)
    call = lambda a: prefix_attention(a["q"], a["k"], a["v"], a["tab"], a["ln"], starts=a["starts"], groups=a["groups"], prefixes=a["prefixes"], out=a["out"])
    call(ok)
    q = ok["q"]
    for bad in (dict(q=q.float()), dict(q=h(3, 3, 16)), dict(q=h(3, 4, 12)), dict(q=h(3, 4, 32)[..., ::2]), dict(q=q[0]), dict(q=q.bfloat16()), dict(starts=None),
                dict(starts=i32(2)), dict(starts=i64(3)), dict(starts=i32(6)[::2]), dict(groups=None), dict(prefixes=None), dict(groups=i32(3)), dict(groups=i64(2)),
                dict(prefixes=i64(1)), dict(prefixes=i32(1, 1)), dict(groups=i32(2050), prefixes=i32(2049)), dict(k=h(3, 2, 12, 16), v=h(3, 2, 12, 16)),
                dict(k=h(4, 2, 8, 16)), dict(k=h(3, 2, 8, 32)), dict(k=h(0, 2, 8, 16), v=h(0, 2, 8, 16)), dict(tab=ok["tab"].long()), dict(tab=i32(3, 3)),
                dict(tab=i32(3, 2).t()), dict(ln=i64(2)), dict(ln=i32(4)[::2]), dict(out=h(3, 4, 8)), dict(out=q), dict(out=h(3, 1, 16).expand(3, 4, 16)),
                dict(out=h(3, 4, 16).cpu()), dict(starts=i32(3).cpu()), dict(q=h(3, 4, 20)[..., 4:]), dict(out=ok["k"].view(-1)[:192].view(3, 4, 16))):
        with pytest.raises(ValueError):
            call({**ok, **bad})
    ok = dict(tab=i32(2, 3), ln=i32(2), ct=i32(2), free=i32(4), taken=i32(1), ps=8, tokens=5, out=None)
    call = lambda a: extend_tables(a["tab"], a["ln"], a["ct"], a["free"], a["taken"], a["ps"], tokens=a["tokens"], out=a["out"])
    call(ok)
    made = lambda **kw: TableStep(i32(2), i32(1), i32(3), i64(5), i64(5))._replace(**kw)
    both, one = i32(4), i64(5)
    for bad in (dict(tab=i32(2)), dict(tab=i64(2, 3)), dict(tab=i32(3, 3)), dict(tab=i32(3, 2).t()), dict(tab=i32(1, 3).expand(2, 3)), dict(ln=i64(2)), dict(ct=i32(3)),
                dict(free=i64(4)), dict(free=i32(2, 2)), dict(taken=i32(2)), dict(ps=12), dict(ps=4), dict(ps=2048), dict(tokens=-1), dict(tokens=(1 << 24) + 1),
                dict(ct=i32(2).cpu()), dict(tab=both.view(2, 2), ln=both[:2]), dict(out=made(lengths=i32(3))), dict(out=made(slots=i32(5))),
                dict(out=made(positions=one, slots=one)), dict(out=made(lengths=ok["ct"])), dict(out=made(starts=ok["free"][:3])), dict(out=made(taken=ok["ln"][:1])),
                dict(out=made(lengths=ok["tab"].view(-1)[:2])), dict(tokens=None, out=made())):
        with pytest.raises(ValueError):
            call({**ok, **bad})
    got = call({**ok, "out": made(lengths=ok["ln"], taken=ok["taken"])})
    assert got.lengths is ok["ln"]


@pytest.mark.gpu
def test_captured_calls_replay_beside_eager_ones(dev):
    """Two graphs and eager calls in any order: every one has room of its own; lengths, starts and prefixes are the replay's."""
    ps = [_problem(dev, torch.bfloat16, [900, 100], [30, 7, 200, 5, 9], [3, 1, 40, 5, 1], [0, 3, 5], 8, 2, 128, 16, seed=s) for s in range(3)]
    want = [_run(p) for p in ps]
    for w, p in zip(want, ps):
        _hold(w, *p)
    graphs = []
    for p in ps[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(p)
        graphs.append((graph, out))
    for order in ((0, 1, 2), (1, 0, 0), (2, 1, 0), (1, 1, 2)):
        for i in order:
            if i < 2:
                graphs[i][1].zero_()
                graphs[i][0].replay()
                assert torch.equal(graphs[i][1], want[i])
            else:
                assert torch.equal(_run(ps[2]), want[2])
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for (graph, out), stream in zip(graphs, (torch.cuda.current_stream(), side)):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for (_, out), w in zip(graphs, want))
    q, k, v, tables, lengths, starts, groups, prefixes = ps[0]
    lengths[1] -= 3
    starts.copy_(_i32([0, 2, 3, 43, 48, 49], dev))
    prefixes[0] -= 300
    graphs[0][0].replay()
    _hold(graphs[0][1], *ps[0])
    assert torch.equal(graphs[0][1], _run(ps[0]))


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_meet(dev):
    ps = [_problem(dev, torch.float16, [1500], [30] * 40, [1] * 40, [0, 40], 8, 8, 64, 16, seed=s) for s in range(2)]
    want = [_run(p) for p in ps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, p in zip(streams, ps):
            with torch.cuda.stream(s):
                got.append(_run(p))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(60))
def test_prefix_over_drawn_sizes(dev, seed):
    rng = random.Random(seed)
    heads, kv, dim = rng.choice(HEADS + [(8, 8, 128), (16, 2, 128), (12, 12, 64)])
    ps, dtype = rng.choice([8, 16, 32, 128]), rng.choice(TYPES)
    rows = int(2 ** rng.uniform(0, 6.5))
    many = rng.random() < 0.5
    n = rng.randrange(1, max(2, rows // 2 + 1))
    groups = [rng.randrange(0, 2)] + sorted(rng.choices(range(1, rows + 1), k=n - 1)) + [rows - rng.randrange(0, 2) if rows > 1 else 1]
    groups = sorted(min(max(g, 0), rows) for g in groups)
    news = [rng.choice([0, 1, 2, rng.randrange(1, 60)]) if many else 1 for _ in range(rows)]
    suffixes = [rng.choice([None, c, c + 1, c + rng.randrange(0, 400)]) for c in news]
    suffixes = [None if s == 0 else s for s in suffixes]
    prefixes = [rng.choice([0, 1, ps, int(2 ** rng.uniform(0, 11))]) for _ in range(n)]
    p = _problem(dev, dtype, prefixes, suffixes, news, groups, heads, kv, dim, ps, seed=seed)
    _hold(_run(p), *p, most_rows=200)
    if not many:
        _hold(_run(p, single=True), *p, most_rows=200)


@pytest.mark.gpu
def test_steps_prompts_and_runs_of_a_model(dev):
    """Prompts taken in one pass, chats that share a prefix and a captured step of a run, against the same tokens one at a time."""
    from test_llama_step import BITS, H, HEADS, LAYERS, V, I, _close, _delta_state_dict
    from deltazip_amd import CompressionConfig, DeltaConfig, DeltaMapping, DeltaModel, create_delta_manager, ops
    from deltazip_amd.llama_step import LlamaForDecodeStep, LlamaStepConfig
    cfg = LlamaStepConfig(hidden_size=H, intermediate_size=I, num_attention_heads=HEADS, num_hidden_layers=LAYERS, vocab_size=V, max_position_embeddings=96)
    model = LlamaForDecodeStep(cfg, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    mgr = create_delta_manager(model, max_num_seqs=64, max_num_batched_tokens=64, vocab_size=V, delta_config=DeltaConfig(max_deltas=3, max_bitwidth=BITS))
    for d in (1, 2):
        mgr.add_delta(DeltaModel.from_tensors(_delta_state_dict(1000 * d)[0], d, CompressionConfig(bits=BITS, prunen=2, prunem=4, sparsity=0.5), pin_memory=False))
        mgr.activate_delta(d)

    def ids(deltas):
        mgr.set_delta_mapping(DeltaMapping(tuple(deltas), tuple(deltas)))

    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, V, (n,), generator=g).to(dev) for n in (19, 1, 24)]
    slow, fast = model.make_paged_cache(60, page_size=8, device=dev), model.make_paged_cache(60, page_size=8, device=dev)
    for c in (slow, fast):
        c.pool.fill_(float("nan"))
    want = []
    for d, p in enumerate(prompts):                  # token by token
        slow.add(d)
        ids([d])
        for t in range(len(p)):
            slow.extend([d])
            last = model.paged_step(p[t:t + 1], slow, slow.batch([d]))
        want.append(last)
    for d, p in enumerate(prompts):
        fast.add(d, len(p))
    ids([d for d, p in enumerate(prompts) for _ in p])
    b = fast.batch([0, 1, 2], tokens=[len(p) for p in prompts])
    got = model.paged_step(torch.cat(prompts), fast, b, sample_rows=(b.starts[1:] - 1).long())
    assert _close(got.float().cpu().numpy(), torch.cat(want).float().cpu().numpy())

    # chats behind the first and the third prompt
    for c in (slow, fast):
        for name, parent in (("a", 0), ("b", 0), ("c", 2), ("d", 2), ("e", 2)):
            c.fork(parent, name)
    seqs, deltas = ["a", "b", "c", "d", "e", None], [0, 0, 2, 2, 2, 0]
    ids(deltas)
    steps = torch.randint(0, V, (12, 6), generator=g).to(dev)
    want, got = [], []
    for t in steps[:2]:
        for c, kept, prefix in ((slow, want, False), (fast, got, True)):
            c.extend(seqs[:5])
            kept.append(model.paged_step(t, c, c.batch(seqs, prefix=prefix)))
    assert fast.batch(seqs, prefix=True).prefixes.tolist()[:2] == [16, 24]
    run = fast.run(seqs, 10, prefix=True)
    batch, words = run.step(), torch.empty(6, dtype=torch.long, device=dev)
    words.copy_(steps[2])
    got.append(model.paged_step(words, fast, batch))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.paged_step(words, fast, run.step())
    for t in steps[3:]:
        words.copy_(t)
        graph.replay()
        got.append(logits.clone())
    for t in steps[2:]:
        slow.extend(seqs[:5])
        want.append(model.paged_step(t, slow, slow.batch(seqs)))
    for x, y in zip(got, want):
        assert _close(x[:5].float().cpu().numpy(), y[:5].float().cpu().numpy())
    ops.poll_status(wait=True)
    run.finish()
    assert [fast.length(x) for x in seqs[:5]] == [slow.length(x) for x in seqs[:5]] and fast.free_pages == slow.free_pages
    for x in seqs[:5]:
        (p, s), (_, z) = fast.slots(x, 24), slow.slots(x, 24)
        for layer in range(LAYERS):
            for a, c in ((fast.keys[layer], slow.keys[layer]), (fast.values[layer], slow.values[layer])):
                x1, x2 = a[s // 8, :, s % 8], c[z // 8, :, z % 8]
                assert torch.isfinite(x1).all() and _close(x1.float().flatten(1).cpu().numpy(), x2.float().flatten(1).cpu().numpy())
    # more steps than there are pages for: nothing goes on
    run, n = fast.run(["a"], 1), fast.num_pages
    assert fast.free_pages == slow.free_pages
    for _ in range(3):
        b = run.step()
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(wait=True)
    assert b.slots.tolist() == [-1] and b.lengths.tolist() == [32]
    run.finish()
    assert fast.length("a") == 32
