"""The paged key/value cache and its operators: rotary positions, keys and values stored, attention of one new token,
pages copied, and the host's bookkeeping, against restatements in 64 bits (oracle/paged_ref.py)."""
import ctypes as C
import math
import random
import struct
import threading

import numpy as np
import pytest
import torch

from oracle import paged_ref as ref

TYPES = [torch.float16, torch.bfloat16]


# ---------------------------------------------------------------------------------------------
# the restatement's own pins
# ---------------------------------------------------------------------------------------------


def test_oracle_rotary_closed_forms():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 9.0]]])
    # a quarter turn of the first pair, none of the second
    y = ref.rotary(x, torch.tensor([1]), [math.pi / 2, 0.0])
    assert torch.allclose(y, torch.tensor([[[-3.0, 2.0, 1.0, 4.0, 9.0]]], dtype=torch.float64))
    y = ref.rotary(x, torch.tensor([2]), [math.pi / 2, 0.0], factor=2.0, interleaved=True)
    assert torch.allclose(y, torch.tensor([[[-2.0, -4.0, 6.0, 8.0, 9.0]]], dtype=torch.float64))


def test_oracle_attention_closed_forms():
    # equal scores: the mean of the tokens seen; one score far above: that token; nothing seen: zero
    k, v = torch.zeros(3, 1, 8, 8), torch.arange(24.0).view(3, 1, 8, 1).expand(3, 1, 8, 8).contiguous()
    q = torch.ones(3, 2, 8)
    tables, lengths = torch.tensor([[2, 0], [1, 0], [0, 0]], dtype=torch.int32), torch.tensor([10, 8, 0], dtype=torch.int32)
    out, size, _ = ref.attention(q, k, v, tables, lengths, 1.0)
    assert torch.allclose(out[0], torch.tensor((sum(range(16, 24)) + 0 + 1) / 10).double())
    assert torch.allclose(out[1], torch.tensor(11.5).double()) and (out[2] == 0).all() and torch.equal(out, size)
    out, _, _ = ref.attention(q, k, v, tables, lengths, 1.0, window=3)
    assert torch.allclose(out[0], torch.tensor((23 + 0 + 1) / 3).double()) and torch.allclose(out[1], torch.tensor(14.0).double())
    k[1, 0, 4] = 100.0
    out, _, _ = ref.attention(q, k, v, tables, lengths, 1.0)
    assert torch.allclose(out[1], torch.tensor(12.0).double())


# ---------------------------------------------------------------------------------------------
# positions
# ---------------------------------------------------------------------------------------------


def test_frequencies_of_the_scalings():
    from deltazip_amd import RotaryPositions
    i = np.arange(64)
    plain = 10000.0 ** (-i / 64)
    f = lambda **kw: RotaryPositions(128, **kw).frequencies.numpy()
    assert np.allclose(f(), plain, rtol=1e-14)
    assert np.allclose(f(scaling={"type": "linear", "factor": 4.0}), plain / 4, rtol=1e-14)
    assert np.allclose(f(rotary_dim=32), 10000.0 ** (-np.arange(16) / 16), rtol=1e-14)
    # dynamic, twice the trained length: the base times (2 * 2 - 1)^(128 / 126)
    assert np.allclose(f(scaling={"type": "dynamic", "factor": 2.0}), (10000.0 * 3 ** (128 / 126)) ** (-i / 64), rtol=1e-13)
    # yarn: pairs that turn often within the trained length are kept, those that turn less than once stretched
    r = RotaryPositions(128, scaling={"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096})
    got, turns = r.frequencies.numpy(), 4096 * plain / (2 * math.pi)
    assert np.allclose(got[turns > 34], plain[turns > 34], rtol=1e-14) and (turns > 34).sum() > 10
    assert np.allclose(got[turns < 0.9], plain[turns < 0.9] / 8, rtol=1e-14) and (turns < 0.9).sum() > 10
    assert (np.diff(got) < 0).all() and abs(r.attention_factor - (1 + 0.1 * math.log(8))) < 1e-12
    for bad in (dict(head_dim=127), dict(head_dim=300), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=7),
                dict(head_dim=64, base=0.0), dict(head_dim=64, scaling={"type": "linear", "factor": 0.5}),
                dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "beta_fast": 3}),
                dict(head_dim=64, rotary_dim=2, scaling={"type": "dynamic", "factor": 2.0}),
                dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0, "beta_fast": 1, "beta_slow": 2})):
        with pytest.raises(ValueError):
            RotaryPositions(**bad)
    with pytest.raises(NotImplementedError):
        RotaryPositions(64, scaling={"type": "other", "factor": 2.0})


@pytest.mark.parametrize("scaling", [{"factor": 4.0}, {"type": None, "factor": 4.0}, {"type": "linear"}, {"type": "dynamic"}, {"rope_type": "yarn"},
                                     {"original_max_position_embeddings": 4096}, {"type": "linear", "factor": math.inf},
                                     {"type": "yarn", "factor": math.nan}, {"type": "linear", "factor": None}])
def test_scalings_that_say_too_little_are_refused(scaling):
    """An entry without a type or a factor would leave positions as they are, and no one would know."""
    from deltazip_amd import RotaryPositions
    with pytest.raises(ValueError, match="scaling must"):
        RotaryPositions(64, scaling=scaling)
    assert torch.equal(RotaryPositions(64, scaling={}).frequencies, RotaryPositions(64).frequencies)


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle"])
def test_positions_that_were_copied_are_their_own(how):
    """What a call is handed points into the copy, not into what it was copied from."""
    import copy
    import pickle
    from deltazip_amd import RotaryPositions
    first = RotaryPositions(64, rotary_dim=20, interleaved=True, scaling={"type": "yarn", "factor": 4.0})
    made = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x))}[how](first)
    assert made._packed[0] == made._turns.ctypes.data and made._packed[1:] == first._packed[1:]
    got = np.ctypeslib.as_array(C.cast(made._packed[0], C.POINTER(C.c_double)), (10,))
    assert np.array_equal(got, first.frequencies.numpy() / (2 * math.pi)) and torch.equal(made.frequencies, first.frequencies)
    if how != "copy":
        assert made._packed[0] != first._packed[0]


# ---------------------------------------------------------------------------------------------
# the host's bookkeeping
# ---------------------------------------------------------------------------------------------


def _plain_copy(pool, pairs):
    pool[:, [b for _, b in pairs]] = pool[:, [a for a, _ in pairs]]


def _cache_on(device, monkeypatch=None, pages=40, page_size=8, layers=2, **kw):
    from deltazip_amd import PagedKVCache, kv_cache
    if monkeypatch is not None:
        monkeypatch.setattr(kv_cache, "copy_pages", _plain_copy)
    return PagedKVCache(layers, pages, page_size, 1, 8, max_tokens=200, device=device, **kw)


def _seen(cache, seq):
    """The first value of every token of a sequence, per pool, by its table."""
    b = cache.batch([seq])
    n, ps = int(b.lengths[0]), cache.page_size
    t = torch.arange(n)
    page = b.block_tables[0].cpu().long()[t // ps]
    return cache.pool[:, page.to(cache.pool.device), 0, (t % ps).to(cache.pool.device), 0].cpu()


def _store(cache, seqs, values):
    """What append_kv does: the newest token of every sequence."""
    b = cache.batch(seqs)
    for slot, value in zip(b.slots.tolist(), values):
        cache.pool[:, slot // cache.page_size, :, slot % cache.page_size] = value


def _check(cache, model):
    users = [0] * cache.num_pages
    for seq, tokens in model.items():
        assert cache.length(seq) == len(tokens) and len(cache.pages(seq)) == -(-len(tokens) // cache.page_size)
        for p in cache.pages(seq):
            users[p] += 1
    assert cache._spared == sum(u - 1 for u in users if u)
    assert cache._users == users and sorted(cache._free) == [p for p in range(cache.num_pages) if not users[p]]
    assert len(cache) == len(model) and cache.free_pages == users.count(0)


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_against_lists_of_tokens(monkeypatch, seed):
    """Random sequences that come, grow, fork, are cut, compacted and go: every one still holds its own tokens."""
    from deltazip_amd.kv_cache import OutOfPages
    rng = random.Random(seed)
    cache, model, fresh, full = _cache_on("cpu", monkeypatch), {}, 0, 0
    for step in range(300):
        act = rng.choice(["add", "extend", "extend", "extend", "extend", "fork", "free", "truncate", "compact"])
        names = list(model)
        try:
            if act == "add":
                n = rng.randrange(0, 30)
                cache.add(fresh, n)
                model[fresh] = [1000 * (fresh % 50) + i % 50 for i in range(n)]
                if n:
                    pos, slots = cache.slots(fresh)
                    assert pos.tolist() == list(range(n))
                    for slot, value in zip(slots.tolist(), model[fresh]):
                        cache.pool[:, slot // 8, :, slot % 8] = value
                fresh += 1
            elif act == "extend" and names:
                some = rng.sample(names, rng.randrange(1, len(names) + 1))
                cache.extend(some)
                values = [rng.randrange(0, 2000) for _ in some]
                _store(cache, some, values)
                for s, value in zip(some, values):
                    model[s].append(value)
            elif act == "fork" and names:
                parent = rng.choice(names)
                cache.fork(parent, fresh)
                model[fresh] = list(model[parent])
                fresh += 1
            elif act == "free" and names:
                s = rng.choice(names)
                cache.free(s)
                del model[s]
            elif act == "truncate" and names:
                s = rng.choice(names)
                n = rng.randrange(0, len(model[s]) + 1)
                cache.truncate(s, n)
                del model[s][n:]
            elif act == "compact":
                n = cache.compact()
                assert all(p < n for s in model for p in cache.pages(s)) and cache.free_pages == cache.num_pages - n
        except OutOfPages:
            full += 1
            if names:
                s = rng.choice(names)
                cache.free(s)
                del model[s]
        _check(cache, model)
        for s, tokens in model.items():
            if tokens and cache._users[cache.pages(s)[-1]] == 1:      # (batch refuses a shared newest page)
                assert torch.equal(_seen(cache, s), torch.tensor(tokens, dtype=torch.float16).expand(4, -1))
    assert fresh > 20


def test_pages_are_shared_until_written(monkeypatch):
    cache = _cache_on("cpu", monkeypatch)
    cache.add("a", 11)
    cache.pool[:, list(cache.pages("a"))] = 5.0
    cache.fork("a", "b")
    cache.fork("a", "c")
    assert cache.pages("a") == cache.pages("b") == cache.pages("c") and cache.free_pages == 38
    cache.add("alone", 160)
    cache.extend(["alone"])
    assert not cache.batch(["alone"]).shared
    cache.free("alone")
    cache.extend(["a", "b", "c"])              # two of three are given copies of the last page, the last keeps it
    assert cache.free_pages == 36 and len({cache.pages(s)[1] for s in "abc"}) == 3 and len({cache.pages(s)[0] for s in "abc"}) == 1
    _store(cache, ["a", "b", "c"], [1.0, 2.0, 3.0])
    assert cache.batch(["a"]).shared and not cache.batch(["a", "b", "c"]).shared      # (two spared of two seen, of six)
    for s, value in zip("abc", (1.0, 2.0, 3.0)):
        assert _seen(cache, s)[0].tolist() == [5.0] * 11 + [value]
    with pytest.raises(ValueError, match="other sequences"):
        cache.slots("a")
    assert cache.slots("a", 8)[0].tolist() == [8, 9, 10, 11]
    cache.free("a")
    cache.free("b")
    cache.free("c")
    assert cache.free_pages == 40 and len(cache) == 0


def test_rows_are_shared_among_those_of_the_batch(monkeypatch):
    """What sequences outside the batch share has no part in it."""
    cache = _cache_on("cpu", monkeypatch, pages=200)
    for parent in ("a", "b"):
        cache.add(parent, 83)
        for i in range(5):
            cache.fork(parent, f"{parent}{i}")
    cache.add("x", 9)
    cache.add("y", 20)
    cache.extend(["a", "b", "x", "y", *(f"{p}{i}" for p in "ab" for i in range(5))])
    shared = lambda *seqs: cache.batch(list(seqs)).shared
    assert not shared("x", "y") and not shared("x", None) and not shared("a", None, None) and not shared("a", "b")
    assert not shared("a", "b", "x", "y") and not shared("a", "a0")          # (ten pages of 22 are met twice)
    assert shared("a", "a0", "a1") and shared(*(f"b{i}" for i in range(5)), "x", None) and shared("a", "a0", "a1", "b", "b0", "b1", "y")
    out = cache.batch(["a", "a0", "a1"])
    assert out.shared and not cache.batch(["a", "b", "x"], out=out).shared


def test_a_copy_that_fails_changes_nothing(monkeypatch):
    """extend and compact of a pool that copy_pages refuses (it is on the host): every sequence has the pages it had."""
    from deltazip_amd import kv_cache
    cache = _cache_on("cpu")
    model = {}
    for s, n in (("gone", 20), ("a", 11), ("c", 8)):
        cache.add(s, n)
        model[s] = [0] * n
    for s in ("b", "d"):
        cache.fork("a", s)
        model[s] = [0] * 11
    cache.free("gone")
    del model["gone"]
    state = lambda: ({s: (cache.pages(s), cache.length(s)) for s in model}, sorted(cache._free), list(cache._users), cache._spared)
    before = state()
    for call in (lambda: cache.extend(["a", "c", "b", "d"], 9), cache.compact):
        with pytest.raises(ValueError, match="GPU"):
            call()
        assert state() == before
        _check(cache, model)
    monkeypatch.setattr(kv_cache, "copy_pages", _plain_copy)
    cache.extend(["a", "c", "b", "d"], 9)
    for s in model:
        model[s] = model[s] + [0] * 9
    _check(cache, model)
    assert cache.compact() == 10 and len({cache.pages(s)[1] for s in "abd"}) == 3
    _check(cache, model)


def test_calls_that_do_not_fit_change_nothing(monkeypatch):
    from deltazip_amd.kv_cache import OutOfPages
    cache = _cache_on("cpu", monkeypatch, pages=4)
    cache.add("a", 9)
    cache.add("b", 8)
    before = (cache.pages("a"), cache.pages("b"), cache.free_pages, cache.length("a"))
    with pytest.raises(OutOfPages):
        cache.extend(["a", "b"], 17)
    with pytest.raises(OutOfPages):
        cache.add("c", 9)
    with pytest.raises(ValueError):
        cache.extend(["a", "a"])
    with pytest.raises(ValueError):
        cache.extend(["a", "nobody"])
    with pytest.raises(ValueError):
        cache.extend(["a"], 192)               # beyond max_tokens
    with pytest.raises(ValueError):
        cache.add("a")
    with pytest.raises(ValueError):
        cache.fork("a", "b")
    with pytest.raises(ValueError):
        cache.truncate("a", 10)
    with pytest.raises(ValueError):
        cache.free("nobody")
    with pytest.raises(ValueError):
        cache.slots("a", 3, 10)
    with pytest.raises(ValueError):
        cache.batch(["a"], width=1)
    with pytest.raises(ValueError, match="twice"):
        cache.batch(["a", None, "a"])
    cache.add("empty")
    with pytest.raises(ValueError):
        cache.batch(["empty"])
    assert before == (cache.pages("a"), cache.pages("b"), cache.free_pages, cache.length("a"))
    b = cache.batch(["a", None, "b"], width=5)
    assert b.positions.tolist() == [8, 0, 7] and b.lengths.tolist() == [9, 0, 8] and b.slots[1] == -1
    assert b.block_tables.shape == (3, 5) and b.block_tables[0, :2].tolist() == list(cache.pages("a"))
    again = cache.batch([None, "b", "a"], out=b)
    assert all(x is y for x, y in zip(again[:4], b)) and b.lengths.tolist() == [0, 8, 9]
    for bad in (dict(page_size=12), dict(page_size=4), dict(pages=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            _cache_on("cpu", **bad)


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------


def test_c_entry_points_check_their_arguments(dzlib):
    """On the host, before anything is launched: no pointer below is dereferenced."""
    from deltazip_amd import paged
    P = 0x1000
    names = ("bytes q k v tables lengths out work counters status work_bytes num_pages q_row q_head k_page k_head k_token v_page v_head v_token "
             "out_row out_head table_row rows heads kv_heads dim page_size pages_per_row window dtype scale shared").split()
    ok = dict(zip(names, [paged._ATTENTION.size] + [P] * 9 + [1 << 30, 10] + [4096, 128, 65536, 2048, 128, 65536, 2048, 128, 4096, 128, 4]
                  + [2, 32, 32, 128, 16, 40, 0, 0, 0.1, 0]))
    attend = lambda **kw: dzlib.dz_paged_attention(paged._ATTENTION.pack(*{**ok, **kw}.values()), None)
    assert dzlib.dz_paged_attention(None, None) == -1 and attend(bytes=8) == -1
    for name in ("q", "k", "v", "tables", "lengths", "out", "status"):
        assert attend(**{name: 0}) == -1, name
    for kw in (dict(heads=33), dict(kv_heads=0), dict(dim=130), dict(dim=264), dict(dim=0), dict(page_size=12), dict(page_size=4),
               dict(page_size=2048), dict(rows=-1), dict(pages_per_row=-1), dict(pages_per_row=1 << 28), dict(num_pages=0),
               dict(num_pages=1 << 31), dict(table_row=-1), dict(heads=8192, kv_heads=8192)):
        assert attend(**kw) == -12, kw
    for kw in (dict(q=P + 8), dict(k=P + 2), dict(out=P + 4), dict(lengths=P + 2), dict(k_token=132), dict(v_page=-8)):
        assert attend(**kw) == -10, kw
    assert attend(dtype=2) == -1 and attend(window=-1) == -1
    assert attend(work=0) == -8 and attend(work_bytes=64) == -8 and attend(counters=0) == -8 and attend(counters=P + 2) == -8
    assert attend(rows=0, q=0) == 0
    assert dzlib.dz_paged_attention_bytes(2, 32, 32, 128, 16, 40) > 0 == dzlib.dz_paged_attention_bytes(2, 32, 32, 128, 16, 4) and dzlib.dz_paged_attention_bytes(2, 33, 32, 128, 16, 4) == 0

    names = ("bytes q k v q_out k_out v_out positions slots turns status num_pages q_row q_head k_row k_head v_row v_head q_out_row "
             "q_out_head k_out_page k_out_head k_out_token v_out_page v_out_head v_out_token tokens heads kv_heads dim rot neighbours "
             "page_size dtype factor reserved").split()
    ok = dict(zip(names, [paged._ROTARY.size] + [P] * 10 + [10] + [4096, 128] * 4 + [65536, 2048, 128] * 2
                  + [3, 32, 32, 128, 128, 0, 16, 0, 1.0, 0]))
    turn = lambda **kw: dzlib.dz_rotary(paged._ROTARY.pack(*{**ok, **kw}.values()), None)
    assert dzlib.dz_rotary(None, None) == -1 and turn(bytes=8) == -1
    for kw in (dict(q=0), dict(q_out=0), dict(k_out=0), dict(v_out=0), dict(positions=0), dict(turns=0), dict(slots=0), dict(dtype=3)):
        assert turn(**kw) == -1, kw
    for kw in (dict(dim=127), dict(dim=258), dict(rot=130), dict(rot=7), dict(tokens=-1), dict(heads=5000), dict(num_pages=0),
               dict(page_size=12), dict(status=0)):
        assert turn(**kw) == -12, kw
    for kw in (dict(q=P + 2), dict(k_row=129), dict(v_out_page=-2)):
        assert turn(**kw) == -10, kw
    assert turn(tokens=0, q=0) == 0

    pools, pairs = (C.c_void_p * 2)(P, P), (C.c_int32 * 4)(0, 1, 2, 3)
    copy = lambda pools=pools, n=2, stride=4096, size=4096, pages=4, pairs=pairs, npairs=2: dzlib.dz_copy_pages(
        pools, n, stride, size, pages, pairs, npairs, None)
    assert copy(pools=None) == -1 and copy(pairs=None) == -1 and copy(pages=3) == -1 and copy(pairs=(C.c_int32 * 4)(0, -1, 2, 3)) == -1
    assert copy(size=24) == -12 and copy(stride=2048) == -12 and copy(n=-1) == -12 and copy(stride=4104) == -12
    assert copy(pools=(C.c_void_p * 2)(P, P + 8)) == -10 and copy(pools=(C.c_void_p * 2)(P, None)) == -10
    assert copy(n=0) == 0 and copy(npairs=0) == 0


def test_host_tensors_are_refused(dzlib):
    from deltazip_amd import RotaryPositions, append_kv, copy_pages, paged_attention, rotary
    q, pages = torch.zeros(2, 2, 16, dtype=torch.float16), torch.zeros(3, 2, 8, 16, dtype=torch.float16)
    pos, i32 = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    rope = RotaryPositions(16)
    for call in (lambda: paged_attention(q, pages, pages, i32[:, None], i32), lambda: rotary(q, q, pos, rope),
                 lambda: append_kv(q, q, q, pos, pos, rope, pages, pages), lambda: copy_pages(pages[None], [(0, 1)])):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("seed", range(8))
def test_tensors_that_share_elements_are_told_from_those_that_do_not(seed):
    """Against the elements themselves: no two that share one are taken for apart, and where strides step over what is inside them, none
    that are apart are taken for sharing."""
    from deltazip_amd.paged import _meet
    rng, store = random.Random(seed), torch.arange(4000, dtype=torch.int16)
    met = apart = 0
    for _ in range(600):
        inner = rng.choice([1, 2, 3, 8])
        head = inner * rng.randrange(1, 4)
        heads = rng.randrange(1, 6)
        row = head * heads * rng.randrange(1, 3) + rng.randrange(0, 9)
        views = []
        for _ in range(2):
            n, h, d = rng.randrange(1, 6), rng.randrange(1, heads + 1), rng.randrange(1, inner + 1)
            at = rng.randrange(0, 2 * row) + 500
            shape, strides = (n, h, d), (row, head, 1)
            order = rng.choice([(0, 1, 2), (1, 0, 2), (2, 0, 1)])
            views.append(store.as_strided([shape[i] for i in order], [strides[i] for i in order], at))
        a, b = views
        share = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert _meet(a, b) == _meet(b, a) == share
        met, apart = met + share, apart + (not share)
        # any strides at all: never taken for apart wrongly
        c, d = (store.as_strided([rng.randrange(1, 5) for _ in range(3)], [rng.randrange(0, 30) for _ in range(3)], rng.randrange(0, 60)) for _ in range(2))
        if set(c.flatten().tolist()) & set(d.flatten().tolist()):
            assert _meet(c, d)
    assert met > 50 and apart > 50
    assert not _meet(store[:0], store) and not _meet(store[:10], store[10:]) and _meet(store[:10], store.view(torch.int32)[4:])


def test_pools_that_share_memory_are_told_from_those_that_do_not():
    from deltazip_amd.paged import _pools_meet
    rng = random.Random(5)
    for _ in range(3000):
        pages, size = rng.randrange(1, 6), rng.randrange(1, 5)
        stride = size + rng.choice([0, 0, 3, 2 * size, 3 * size])
        at = [rng.randrange(0, 60) for _ in range(rng.randrange(1, 4))]
        cells = [{a + p * stride + i for p in range(pages) for i in range(size)} for a in at]
        share = len(set().union(*cells)) < sum(len(c) for c in cells)
        if share:
            assert _pools_meet(at, pages, stride, size)
        elif len(at) == 1 or pages == 1 or all(abs(a - b) >= pages * stride for i, a in enumerate(at) for b in at[:i]):
            assert not _pools_meet(at, pages, stride, size)
    # layers that take turns within a page, keys and values in tensors of their own at any distance
    layers = [base + 16 * i for base in (1000, 1000 + 5 * 64 + 16) for i in range(4)]
    assert not _pools_meet(layers, 5, 64, 16) and _pools_meet(layers + [1008], 5, 64, 16) and _pools_meet(layers + [1064], 5, 64, 16)


def test_status_word_of_a_bad_page():
    from deltazip_amd import ops
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.raise_for_status(ops.STATUS_BAD_PAGE)
    ops.raise_for_status(0)


@pytest.mark.gpu
def test_arguments_that_do_not_fit_are_refused(dev):
    from deltazip_amd import RotaryPositions, append_kv, copy_pages, paged_attention, rotary
    h = lambda *s: torch.zeros(s, dtype=torch.float16, device=dev)
    i32, i64 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev), lambda *s: torch.zeros(s, dtype=torch.int64, device=dev)
    q, kp, vp, tab, ln = h(2, 4, 16), h(3, 2, 8, 16), h(3, 2, 8, 16), i32(2, 3), i32(2)
    paged_attention(q, kp, vp, tab, ln)
    for bad in (dict(q=q.float()), dict(q=h(2, 3, 16)), dict(q=h(2, 4, 12)), dict(q=h(2, 4, 32)[..., ::2]), dict(q=q[0]), dict(q=q.bfloat16()),
                dict(kp=h(3, 2, 12, 16), vp=h(3, 2, 12, 16)), dict(kp=h(4, 2, 8, 16)), dict(kp=h(3, 2, 8, 32)), dict(kp=h(0, 2, 8, 16), vp=h(0, 2, 8, 16)),
                dict(kp=h(3, 0, 8, 16), vp=h(3, 0, 8, 16)), dict(tab=tab.long()), dict(tab=i32(3, 3)), dict(tab=i32(3, 2).t()), dict(ln=ln.long()),
                dict(ln=i32(3)), dict(ln=i32(4)[::2]), dict(window=-1), dict(out=h(2, 4, 8)), dict(out=q), dict(out=h(2, 1, 16).expand(2, 4, 16)),
                dict(out=h(2, 4, 16).cpu()), dict(q=h(2, 4, 20)[..., 4:])):
        a = dict(dict(q=q, kp=kp, vp=vp, tab=tab, ln=ln, window=0, out=None), **bad)
        with pytest.raises(ValueError):
            paged_attention(a["q"], a["kp"], a["vp"], a["tab"], a["ln"], window=a["window"], out=a["out"])
    rope, k, pos = RotaryPositions(16), h(2, 2, 16), i64(2)
    for bad in (dict(q=q.float()), dict(k=h(3, 2, 16)), dict(k=k.bfloat16()), dict(pos=pos.int()), dict(pos=i64(3)), dict(rope=RotaryPositions(32)),
                dict(out=(h(2, 4, 16), None)), dict(out=(h(2, 4, 8), h(2, 2, 16))), dict(out=(h(2, 1, 16).expand(2, 4, 16), h(2, 2, 16))),
                dict(q=h(3, 4, 16)[:2], out="late"), dict(out=(h(2, 4, 16), h(2, 2, 16).cpu()))):
        a = dict(dict(q=q, k=k, pos=pos, rope=rope, out=None), **bad)
        if isinstance(a["out"], str):                # an output that begins inside its input
            whole = h(3, 4, 16)
            a["q"], a["out"] = whole[:2], (whole[1:], h(2, 2, 16))
        with pytest.raises(ValueError):
            rotary(a["q"], a["k"], a["pos"], a["rope"], out=a["out"])
    for bad in (dict(v=h(2, 4, 16)), dict(kp=vp), dict(kp=h(3, 4, 8, 16), vp=h(3, 4, 8, 16)), dict(slots=pos.int()), dict(slots=i64(1)),
                dict(kp=h(1, 2, 8, 16).expand(3, 2, 8, 16)), dict(rope=RotaryPositions(8)), dict(out=kp[:2, :, :2].reshape(2, 4, 16)[:1])):
        a = dict(dict(q=q, k=k, v=k.clone(), slots=pos, rope=rope, kp=kp, vp=vp, out=None), **bad)
        with pytest.raises(ValueError):
            append_kv(a["q"], a["k"], a["v"], pos, a["slots"], a["rope"], a["kp"], a["vp"], out=a["out"])
    pool = h(2, 6, 64)
    for pools, pairs in ((pool, [(0, 6)]), (pool, [(-1, 2)]), (pool, [(0, 1), (2, 1)]), (pool, [(0, 1), (1, 2)]), (pool, [(3, 3)]), (pool, [0, 1]),
                         (pool, [(0.0, 1.0)]), (pool, torch.zeros(1, 2, dtype=torch.int64, device=dev)), (h(2, 6, 5), [(0, 1)]),
                         ([pool[0], pool[0]], [(0, 1)]), ([pool[0], h(5, 64)], [(0, 1)]), (h(2, 6, 4, 32)[..., :16], [(0, 1)]),
                         (h(2, 1, 64).expand(2, 6, 64), [(0, 1)])):
        with pytest.raises(ValueError):
            copy_pages(pools, pairs)


@pytest.mark.gpu
def test_outputs_that_share_memory_with_what_is_read_are_refused(dev):
    """Kernels read and write side by side: a key that is turned in place must not be a query's memory, and the like."""
    from deltazip_amd import RotaryPositions, append_kv, paged_attention, rotary
    h = lambda *s: torch.randn(s, device=dev).half()
    rope, pos, slots = RotaryPositions(16), torch.arange(3, device=dev), torch.tensor([0, 9, 17], device=dev)
    x, wide = h(3, 4, 16), h(3, 8, 16)
    for q, k, out in ((x, x, (x, x)), (x, x, (x, h(3, 4, 16))), (x, x, (h(3, 4, 16), x)), (x, x[:, 1:3], (x, x[:, 1:3])),
                      (wide[:, :4], wide[:, 3:6], (wide[:, :4], wide[:, 3:6])), (x, h(3, 2, 16), (wide[:, :4], wide[:, 3:5]))):
        with pytest.raises(ValueError, match="own"):
            rotary(q, k, pos, rope, out=out)
    pool = h(2, 4, 2, 8, 16)
    kp, vp = pool.unbind(0)
    k, v = h(3, 2, 16), h(3, 2, 16)
    for q, kk, vv, kpages, vpages, out in (
            (x, x[:, :2], v, kp, vp, x), (x, k, x[:, 1:3], kp, vp, x), (wide[:, :4], wide[:, 3:5], v, kp, vp, wide[:, :4]),
            (x, kp[:3, :, 2], v, kp, vp, None), (x, k, kp[:3, :, 2], kp, vp, None), (x, k, vp[1:4, :, 7], kp, vp, None),
            (kp[:3, :, :2].reshape(3, 4, 16), k, v, pool.view(8, 2, 8, 16)[:4], pool.view(8, 2, 8, 16)[3:7], None),
            (pool[0].view(-1, 4, 16)[:3], k, v, kp, vp, None), (x, k, v, kp, vp, pool[1].view(-1, 4, 16)[5:8])):
        with pytest.raises(ValueError, match="own"):
            append_kv(q, kk, vv, pos, slots, rope, kpages, vpages, out=out)
    table = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    words = torch.zeros(2, 4, 8, dtype=torch.int32, device=dev)
    for tables, ln in ((table, words.view(-1)[:2]), (words.view(2, 32)[:, :3], table[:, 0].contiguous())):
        with pytest.raises(ValueError, match="own"):
            paged_attention(h(2, 4, 16), kp, vp, tables, ln, out=words.view(torch.float16))
    # slices of one projection, pages of one pool, an output between inputs: apart
    want_q, want_k = rotary(wide[:, :4], wide[:, 4:6], pos, rope)
    both = pool.clone().transpose(0, 1).contiguous()
    for pages in ((pool[0], pool[1]), (both[:, 0], both[:, 1])):
        for into in ("q", "apart", "late"):
            w = torch.cat((wide, h(3, 4, 16)), 1)
            q, kk, vv = w[:, :4], w[:, 4:6], w[:, 6:8]
            out = {"q": q, "apart": w[:, 8:], "late": None}[into]
            rest = w.clone()
            got = append_kv(q, kk, vv, pos, slots, rope, *pages, out=out)
            assert torch.equal(got, want_q) and torch.equal(w[:, 4:8], rest[:, 4:8])
            for p, want in zip(pages, (want_k, wide[:, 6:8])):
                assert torch.equal(p[slots // 8, :, slots % 8], want)
    w = wide.clone()
    rotary(w[:, :4], w[:, 4:6], pos, rope, out=(w[:, :4], w[:, 4:6]))
    assert torch.equal(w[:, :4], want_q) and torch.equal(w[:, 4:6], want_k) and torch.equal(w[:, 6:], wide[:, 6:])
    assert append_kv(x, k, x[:, :2], pos, slots, None, kp, vp) is x               # (a query that nothing turns is not touched)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------


def _problem(dev, dtype, lengths, heads, kv, dim, ps, seed, poison=True, spread=1.5):
    """Pages in random order; what no row sees holds NaN, what tables hold behind a length is no page."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-max(n, 0) // ps) for n in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g)
    k, v = (torch.randn(pages, kv, ps, dim, generator=g).to(dtype) for _ in range(2))
    width = max(used) + 2
    tables = torch.full((len(lengths), width), 0x7fffffff, dtype=torch.int32)
    seen = torch.zeros(pages, ps, dtype=torch.bool)
    at = 0
    for r, (n, u) in enumerate(zip(lengths, used)):
        tables[r, :u] = order[at:at + u].int()
        t = torch.arange(max(n, 0))
        seen[tables[r].long()[t // ps], t % ps] = True
        at += u
    if poison:
        for p in (k, v):
            p.masked_fill_(~seen[:, None, :, None], float("nan"))
    q = (spread * torch.randn(len(lengths), heads, dim, generator=g)).to(dtype)
    return [x.to(dev) for x in (q, k, v, tables, torch.tensor(lengths, dtype=torch.int32))]


def _hold(got, q, k, v, tables, lengths, scale, window=0):
    want, size, most = ref.attention(q, k, v, tables, lengths, scale, window)
    bound = ref.attention_bound(want, size, most, q.dtype, q.shape[2], max(1, int(lengths.max()) if lengths.numel() else 1))
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"off by up to {(off / bound).max():.2f} of the bound at {(off / bound).argmax()}"


HEADS = [(4, 4, 128), (8, 2, 64), (7, 1, 80), (20, 1, 128), (6, 3, 256), (33, 1, 8), (5, 5, 96), (32, 2, 192), (3, 1, 24), (16, 1, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("ps", [8, 16, 64])
def test_attention_of_ragged_rows(dev, dtype, heads, kv, dim, ps):
    from deltazip_amd import paged_attention
    lengths = [1, 0, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, -3, 1000, 0]
    p = _problem(dev, dtype, lengths, heads, kv, dim, ps, 7 * dim + ps)
    got = paged_attention(*p)
    _hold(got, *p, dim ** -0.5)
    assert (got[1] == 0).all() and (got[18] == 0).all() and (got[20] == 0).all()
    assert torch.equal(got, paged_attention(*p))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 5, 32, 33, 100, 511, 100000, 1 << 40])
def test_attention_window(dev, dtype, window):
    """The window begins inside a tile and a page; what is in front of it may be NaN and its pages given away."""
    from deltazip_amd import paged_attention
    lengths = [1, 0, 5, 6, 33, 64, 100, 101, 133, 512, 700, 1500]
    q, k, v, tables, ln = _problem(dev, dtype, lengths, 6, 2, 128, 16, window % 97)
    for r, n in enumerate(lengths):
        gone = max(0, n - window)
        for t in range(gone):
            page = int(tables[r, t // 16])
            k[page, :, t % 16] = v[page, :, t % 16] = float("inf")
        tables[r, :gone // 16] = -77
    _hold(paged_attention(q, k, v, tables, ln, scale=0.3, window=window), q, k, v, tables, ln, 0.3, min(window, 1 << 30))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,heads,kv,dim,ps", [(1, 20011, 8, 1, 128, 16), (1, 9000, 4, 4, 64, 256), (3, 5003, 16, 2, 256, 8), (2, 40000, 2, 2, 80, 1024)])
def test_attention_of_few_long_rows(dev, dtype, rows, n, heads, kv, dim, ps):
    """The length is split over workgroups and joined."""
    from deltazip_amd import paged_attention
    p = _problem(dev, dtype, [n - 37 * r for r in range(rows)], heads, kv, dim, ps, n)
    got = paged_attention(*p)
    _hold(got, *p, dim ** -0.5)
    assert torch.equal(got, paged_attention(*p))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_many_rows(dev, dtype):
    """More rows than a launch takes, some long ones among short ones; rows that share all their pages."""
    from deltazip_amd import paged_attention
    rng = random.Random(5)
    lengths = [rng.choice([0, 1, 3, 17, 40]) for _ in range(600)]
    lengths[300], lengths[599] = 3000, 700
    p = _problem(dev, dtype, lengths, 2, 1, 64, 8, 11)
    _hold(paged_attention(*p), *p, 0.125)
    q, k, v, tables, ln = _problem(dev, dtype, [90], 2, 1, 64, 16, 12)
    q = torch.randn(90, 2, 64, device=dev).to(dtype)
    shared = q, k, v, tables.expand(90, -1), torch.arange(1, 91, dtype=torch.int32, device=dev)
    _hold(paged_attention(*shared), *shared, 0.125)
    assert torch.equal(paged_attention(*shared, shared=True), paged_attention(*shared))
    p = _problem(dev, dtype, [900] * 24, 16, 8, 128, 16, 13)                 # (past the caches, unless it is said to be shared)
    assert torch.equal(paged_attention(*p, shared=True), paged_attention(*p))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scores_far_apart(dev, dtype):
    """Scores that rise along the sequence (the maximum moves at every step), fall, and one far above the rest; a long flat tail
    far below the maximum still counts with its sum."""
    from deltazip_amd import paged_attention
    n, dim = 1200, 64
    q, k, v, tables, ln = _problem(dev, dtype, [n] * 4, 1, 1, dim, 16, 3, spread=0.0)
    q[:, 0, 0] = torch.tensor([1.0, -1.0, 1.0, 4.0], device=dev).to(dtype)
    for r in range(4):
        at = tables[r].long()[torch.arange(n, device=dev) // 16], 0, torch.arange(n, device=dev) % 16
        ramp = torch.linspace(-40, 40, n, device=dev)
        k[at[0], 0, at[2], 0] = (ramp if r < 2 else torch.full_like(ramp, -3.0)).to(dtype)
        if r >= 2:
            k[tables[r, 30].long(), 0, 5, 0] = 9.0
            v[at[0], 0, at[2]] = (1.0 + 0.1 * v[at[0], 0, at[2]].float()).to(dtype)
    _hold(paged_attention(q, k, v, tables, ln, scale=1.0), q, k, v, tables, ln, 1.0)
    # a negative scale, and scores beyond the type's range
    q[:, 0, 1] = 50.0
    _hold(paged_attention(q, k, v, tables, ln, scale=-2.0), q, k, v, tables, ln, -2.0)


@pytest.mark.gpu
def test_attention_of_values_that_are_not_finite(dev):
    """What a row sees is not masked: NaN stays in its row and head, an infinite score too; other rows are untouched."""
    from deltazip_amd import paged_attention
    q, k, v, tables, ln = p = _problem(dev, torch.float16, [40, 70, 40], 4, 2, 64, 16, 9)
    clean = paged_attention(*p)
    k[tables[1, 0].long(), 0, 3] = float("nan")
    got = paged_attention(*p)
    assert torch.isnan(got[1, :2]).all() and torch.equal(got[1, 2:], clean[1, 2:]) and torch.equal(got[[0, 2]], clean[[0, 2]])
    k[tables[1, 0].long(), 0, 3] = 1.0
    v[tables[1, 4].long(), 1, 5, 7] = float("nan")
    got = paged_attention(*p)
    assert torch.isnan(got[1, 2:, 7]).all() and torch.isfinite(got[1, 2:, :7]).all() and torch.equal(got[[0, 2]], clean[[0, 2]])
    v[tables[1, 4].long(), 1, 5, 7] = 1.0
    k[tables[1, 2].long(), 1, :, 0] = float("-inf")       # sixteen tokens with a score of -inf (or inf), the others count
    q[1, 2, 0], q[1, 3, 0] = 1.0, -1.0
    got = paged_attention(*p)
    keep = [t for t in range(70) if t // 16 != 2]
    kk, vv = (x[tables[1].long()[torch.tensor(keep, device=dev) // 16], 1, torch.tensor(keep, device=dev) % 16].double() for x in (k, v))
    want = torch.softmax(kk @ q[1, 2].double() / 8, 0) @ vv
    assert (got[1, 2].double() - want).abs().max() < 4e-3 and torch.isnan(got[1, 3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 2, 8), (6, 3, 256), (20, 2, 128)])
@pytest.mark.parametrize("n,first,last", [(7, 0, 7), (33, 32, 33), (65, 64, 65), (97, 96, 97), (100, 32, 64), (128, 96, 128), (2048, 512, 640),
                                          (2048, 1920, 2048), (5000, 4999, 5000), (20480, 4096, 6144), (40000, 39999, 40000)])
def test_attention_keeps_nan_of_pieces_without_a_maximum(dev, dtype, heads, kv, dim, n, first, last):
    """Keys that are NaN in all that a wavefront, or a part of a split row, sees: the newest token alone in its tile, whole tiles,
    whole parts (of 4 tiles), all 16 parts that are joined first.  Their heads are NaN; the other heads and rows have the bits that they had."""
    from deltazip_amd import paged_attention
    q, k, v, tables, ln = p = _problem(dev, dtype, [40, n, 300], heads, kv, dim, 16, 90)
    clean = paged_attention(*p)
    t = torch.arange(first, last, device=dev)
    k[tables[1].long()[t // 16], 0, t % 16] = float("nan")
    got = paged_attention(*p)
    share = heads // kv
    assert torch.isnan(got[1, :share]).all()
    assert torch.equal(got[1, share:], clean[1, share:]) and torch.equal(got[[0, 2]], clean[[0, 2]])


@pytest.mark.gpu
def test_attention_strides_and_orders(dev):
    """Queries as slices of a wider projection, pages with tokens in front of heads, keys and values in one tensor, out in
    a wider one: the same bits as the plain layouts."""
    from deltazip_amd import paged_attention
    for dtype in TYPES:
        q, k, v, tables, ln = _problem(dev, dtype, [5, 300, 64, 0, 1000], 6, 2, 80, 16, 21)
        want = paged_attention(q, k, v, tables, ln)
        wide = torch.full((5, 9, 88), float("nan"), dtype=dtype, device=dev)
        wide[:, 2:8, :80] = q
        both = torch.stack((k.transpose(1, 2), v.transpose(1, 2)), 1).contiguous()      # [pages, 2, tokens, kv, dim]
        out = torch.full((6, 5, 96), 7.0, dtype=dtype, device=dev)
        tab = torch.cat((tables, tables), 1)[:, :tables.shape[1]]
        got = paged_attention(wide[:, 2:8, :80], both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), tab, ln, out=out.transpose(0, 1)[..., 8:88])
        assert torch.equal(got, want) and (out[..., :8] == 7).all() and (out[..., 88:] == 7).all()


@pytest.mark.gpu
def test_attention_far_into_a_large_pool(dev):
    """Pages beyond 2^32 bytes and 2^31 values."""
    from deltazip_amd import append_kv, copy_pages, paged_attention
    pages, kv, ps, dim = 36000, 8, 64, 128
    k, v = (torch.empty(pages, kv, ps, dim, dtype=torch.float16, device=dev) for _ in range(2))
    assert k.numel() > 1 << 31
    q, ks, vs, tables, ln = _problem(dev, torch.float16, [200, 64, 5], 16, kv, dim, ps, 31)
    far = torch.arange(pages - len(ks), pages, device=dev)
    k[far], v[far] = ks, vs
    moved = torch.where(tables == 0x7fffffff, tables, (tables + (pages - len(ks))).int())
    assert torch.equal(paged_attention(q, k, v, moved, ln), paged_attention(q, ks, vs, tables, ln))
    x = torch.randn(1, kv, dim, device=dev).half()
    slots = torch.tensor([(pages - 1) * ps + 63], device=dev)
    append_kv(x, x, 2 * x, slots, slots, None, k, v)
    assert torch.equal(k[pages - 1, :, 63], x[0]) and torch.equal(v[pages - 1, :, 63], 2 * x[0])
    copy_pages([k, v], [(pages - 1, pages - 30000), (pages - 2, 0)])
    for t in (k, v):
        assert torch.equal(t[pages - 30000, :, 63], t[pages - 1, :, 63])
        assert torch.equal(t[0].view(torch.int16), t[pages - 2].view(torch.int16))


@pytest.mark.gpu
def test_attention_of_nothing(dev):
    from deltazip_amd import paged_attention
    k = torch.full((2, 2, 8, 16), float("nan"), dtype=torch.float16, device=dev)
    q = torch.ones(0, 4, 16, dtype=torch.float16, device=dev)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    assert paged_attention(q, k, k, i(0, 3), i(0)).shape == (0, 4, 16)
    q = torch.ones(3, 4, 16, dtype=torch.float16, device=dev)
    assert (paged_attention(q, k, k, i(3, 0), i(3)) == 0).all()         # tables without pages
    assert (paged_attention(q, k, k, i(3, 1), i(3)) == 0).all()


@pytest.mark.gpu
def test_pages_outside_the_pool_are_reported(dev):
    from deltazip_amd import append_kv, ops, paged_attention
    ops.poll_status(dev, wait=True)
    q, k, v, tables, ln = _problem(dev, torch.float16, [40, 20], 2, 2, 64, 16, 41)
    paged_attention(q, k, v, tables, ln)
    ops.poll_status(dev, wait=True)                       # behind the lengths anything may stand
    for bad in (len(k), -1):
        t = tables.clone()
        t[0, 1] = bad
        got = paged_attention(q, k, v, t, ln)
        assert torch.equal(got[1], paged_attention(q, k, v, tables, ln)[1])
        with pytest.raises(ops.DeltaKernelError, match="paged"):
            ops.poll_status(dev, wait=True)
        ops.poll_status(dev, wait=True)
    long = tables[:, :2].contiguous(), torch.tensor([40, 20], dtype=torch.int32, device=dev)
    got = paged_attention(q, k, v, *long)                 # 40 tokens in a table of 32
    cut = torch.tensor([32, 20], dtype=torch.int32, device=dev)
    assert torch.equal(got, paged_attention(q, k, v, long[0], cut))
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(dev, wait=True)
    x = torch.randn(3, 2, 64, device=dev).half()
    before = k.clone(), v.clone()
    pos = torch.arange(3, device=dev)
    append_kv(x, x, x, pos, torch.full((3,), -1, device=dev), None, k, v)
    ops.poll_status(dev, wait=True)                       # padded rows are no fault
    append_kv(x, x, x, pos, torch.tensor([-(1 << 62), len(k) * 16, 1 << 62], device=dev), None, k, v)
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(dev, wait=True)
    for a, b in zip(before, (k, v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


# ---------------------------------------------------------------------------------------------
# rotary positions, and keys and values stored
# ---------------------------------------------------------------------------------------------

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 2048}]


def _turned(got, x, pos, rope):
    """Half a step of the output, and of fp32: cosine, sine (2 steps each of values up to the factor), products and sum."""
    want = ref.rotary(x, pos, rope.frequencies.numpy(), rope.attention_factor, rope.interleaved)
    half = torch.finfo(x.dtype).eps / 2
    size = x.double().cpu().abs().amax(-1, keepdim=True)
    bound = half * want.abs() + 16 * 2.0 ** -24 * rope.attention_factor * 2 * size + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((got.double().cpu() - want).abs() <= bound).all()
    assert torch.equal(got[..., rope.rotary_dim:], x[..., rope.rotary_dim:])


def _qkv(dev, dtype, tokens, heads, kv, dim, seed):
    """Views of one fused projection."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(tokens, (heads + 2 * kv) * dim, generator=g, device=dev).to(dtype)
    q, k, v = x.split((heads * dim, kv * dim, kv * dim), 1)
    return q.unflatten(1, (heads, dim)), k.unflatten(1, (kv, dim)), v.unflatten(1, (kv, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 32), (80, 20), (64, 64), (96, 48), (256, 256), (6, 2), (70, 70), (16, 10), (256, 6)])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_rotary(dev, dtype, interleaved, dim, rot, scaling):
    from deltazip_amd import RotaryPositions, rotary
    rope = RotaryPositions(dim, rotary_dim=rot, interleaved=interleaved, scaling=scaling)
    for tokens, heads, kv in ((1, 1, 1), (3, 5, 2), (37, 12, 4)):
        q, k, v = _qkv(dev, dtype, tokens, heads, kv, dim, dim + rot)
        pos = torch.randint(0, 1 << 20, (tokens,), device=dev)
        pos[0], pos[-1] = 0, (1 << 20) + 1
        a, b = rotary(q, k, pos, rope)
        _turned(a, q, pos, rope)
        _turned(b, k, pos, rope)
        assert torch.equal(rotary(q, None, pos, rope)[0], a)
        # in place, within the fused projection: the values stay as they were
        vs = v.clone()
        got = rotary(q, k, pos, rope, out=(q, k))
        assert got[0] is q and torch.equal(q, a) and torch.equal(k, b) and torch.equal(v, vs)


@pytest.mark.gpu
def test_rotary_far_and_negative_positions(dev):
    """Angles hold at positions whose product with the frequency has no fraction left in 32 bits."""
    from deltazip_amd import RotaryPositions, rotary
    rope = RotaryPositions(128)
    q, k, _ = _qkv(dev, torch.float16, 6, 3, 1, 128, 5)
    pos = torch.tensor([1 << 24, (1 << 30) + 7, -5, -(1 << 20), 99999999, 1], device=dev)
    a, b = rotary(q, k, pos, rope)
    _turned(a, q, pos, rope)
    _turned(b, k, pos, rope)
    assert rotary(q[:0], k[:0], pos[:0], rope)[0].shape == (0, 3, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,rot,ps,interleaved", [(4, 4, 128, 128, 16, False), (8, 2, 80, 32, 8, True), (3, 1, 64, 20, 64, False),
                                                           (7, 7, 30, 30, 8, False), (40, 8, 128, 128, 256, True)])
@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_append(dev, dtype, heads, kv, dim, rot, ps, interleaved, tokens):
    """Every slot named holds its token, every other what it held; padded tokens are turned and not stored."""
    from deltazip_amd import RotaryPositions, append_kv, rotary
    rope = RotaryPositions(dim, rotary_dim=rot, interleaved=interleaved)
    q, k, v = _qkv(dev, dtype, tokens, heads, kv, dim, tokens)
    pages = -(-tokens // ps) + 3
    g = torch.Generator(device=dev).manual_seed(1)
    kp, vp = (torch.randn(pages, kv, ps, dim, generator=g, device=dev).to(dtype) for _ in range(2))
    slots = torch.randperm(pages * ps, generator=g, device=dev)[:tokens]
    if tokens > 1:
        slots[1::4] = -1
    pos = torch.randint(0, 5000, (tokens,), generator=g, device=dev)
    wk, wv = kp.clone(), vp.clone()
    tq, tk = rotary(q, k, pos, rope)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            wk[s // ps, :, s % ps], wv[s // ps, :, s % ps] = tk[t], v[t]
    before = q.clone()
    got = append_kv(q, k, v, pos, slots, rope, kp, vp)
    assert torch.equal(got, tq) and torch.equal(kp, wk) and torch.equal(vp, wv) and torch.equal(q, before)
    # pages with tokens in front of heads, q in place
    kt, vt = (torch.zeros(pages, ps, kv, dim, dtype=dtype, device=dev).transpose(1, 2) for _ in range(2))
    assert append_kv(q, k, v, pos, slots, rope, kt, vt, out=q) is q and torch.equal(q, tq)
    for s in slots.tolist():
        if s >= 0:
            assert torch.equal(kt[s // ps, :, s % ps], wk[s // ps, :, s % ps]) and torch.equal(vt[s // ps, :, s % ps], wv[s // ps, :, s % ps])
    # no positions: copied as they are
    kp.zero_()
    assert append_kv(q, k, v, pos, slots, None, kp, vp) is q
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            assert torch.equal(kp[s // ps, :, s % ps], k[t])


# ---------------------------------------------------------------------------------------------
# pages copied
# ---------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("pools,pages,shape,pairs", [(2, 6, (2, 8, 16), 1), (5, 900, (1, 8, 8), 400), (140, 20, (1, 8, 8), 7), (300, 700, (8,), 333),
                                                   (2, 9, (5, 64, 104), 4)])
def test_copy_pages(dev, pools, pages, shape, pairs):
    from deltazip_amd import copy_pages
    g = torch.Generator().manual_seed(pairs)
    pool = torch.randn(pools, pages, *shape, generator=g).half().to(dev)
    order = torch.randperm(pages, generator=g)[:2 * pairs].view(-1, 2)
    want = pool.clone()
    want[:, order[:, 1].to(dev)] = pool[:, order[:, 0].to(dev)]
    got = pool.clone()
    copy_pages(got, order)
    assert torch.equal(got, want)
    # pools apart, pages with a gap between them, pairs as a list
    wide = torch.zeros(pools, pages, 2, *shape, dtype=torch.float16, device=dev)
    wide[:, :, 0] = pool
    copy_pages([w[:, 0] for w in wide], order.tolist())
    assert torch.equal(wide[:, :, 0], want) and (wide[:, :, 1] == 0).all()
    copy_pages(got, [])
    copy_pages([], order)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_pools_that_share_memory_are_refused(dev):
    """Every pool's copies run beside the others': a page of one that lies in another's would be read as it is written."""
    from deltazip_amd import copy_pages
    flat = torch.randn(12, 64, device=dev).half()
    for pools in ([flat[:6], flat[1:7]], [flat[:6], flat[:6]], [flat[6:], flat[:8][2:]], flat.as_strided((2, 6, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="share memory"):
            copy_pages(pools, [(0, 1)])
    # keys and values of layers that take turns within a page
    keys, values = (torch.randn(6, 4, 64, device=dev).half() for _ in range(2))
    want = [t.clone() for t in (keys, values)]
    for w in want:
        w[[1, 3]] = w[[0, 5]]
    copy_pages(list(keys.unbind(1)) + list(values.unbind(1)), [(0, 1), (5, 3)])
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_a_run_of_steps_with_forks_and_compaction(dev):
    """Sequences that come, step, fork, go and are compacted: every step's attention against all tokens of each sequence."""
    from deltazip_amd import PagedKVCache, RotaryPositions, append_kv, paged_attention, rotary
    heads, kv, dim, layers = 8, 2, 64, 2
    cache = PagedKVCache(layers, 60, 16, kv, dim, max_tokens=256, device=dev)
    cache.pool.fill_(float("nan"))
    rope = RotaryPositions(dim, rotary_dim=32, interleaved=True)
    rng, seed, model = random.Random(3), 0, {}
    def tokens(n):
        nonlocal seed
        seed += 1
        return _qkv(dev, torch.float16, n, heads, kv, dim, seed)
    for name in range(4):                               # prompts
        n = rng.randrange(1, 50)
        cache.add(name, n)
        pos, slots = cache.slots(name)
        model[name] = []
        for layer in range(layers):
            q, k, v = tokens(n)
            append_kv(q, k, v, pos, slots, rope, cache.keys[layer], cache.values[layer])
            model[name].append([rotary(k, None, pos, rope)[0].cpu(), v.cpu()])
    fresh = 4
    for step in range(40):
        if step % 7 == 3:
            parent = rng.choice(list(model))
            cache.fork(parent, fresh)
            model[fresh] = [[t.clone() for t in kv_] for kv_ in model[parent]]
            fresh += 1
        if step % 11 == 8:
            gone = rng.choice(list(model))
            cache.free(gone)
            del model[gone]
            cache.compact()
        rows = [s for s in model if rng.random() < 0.8] or list(model)[:1]
        cache.extend(rows)
        padded = rows + [None]
        b = cache.batch(padded)
        for layer in range(layers):
            q, k, v = tokens(len(padded))
            got = paged_attention(append_kv(q, k, v, b.positions, b.slots, rope, cache.keys[layer], cache.values[layer]), cache.keys[layer],
                                  cache.values[layer], b.block_tables, b.lengths)
            tq, tk = rotary(q, k, b.positions, rope)
            assert (got[-1] == 0).all()
            for r, s in enumerate(rows):
                kv_ = model[s][layer]
                kv_[0], kv_[1] = torch.cat((kv_[0], tk[r:r + 1].cpu())), torch.cat((kv_[1], v[r:r + 1].cpu()))
                n = len(kv_[0])
                assert n == cache.length(s)
                one = kv_[0].transpose(0, 1)[None], kv_[1].transpose(0, 1)[None]      # one page of all tokens
                _hold(got[r:r + 1], tq[r:r + 1], *one, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([n]), dim ** -0.5)


@pytest.mark.gpu
def test_captured_steps_follow_the_tables_of_the_replay(dev):
    """Two graphs of a step each, replayed in turn with other tables, lengths and slots, eager work between them."""
    from deltazip_amd import PagedKVCache, RotaryPositions, append_kv, paged_attention
    heads, kv, dim, rows = 4, 2, 128, 5
    cache = PagedKVCache(1, 400, 16, kv, dim, max_tokens=4096, device=dev)
    cache.pool.normal_()
    rope = RotaryPositions(dim)
    names = list(range(rows))
    for s, n in zip(names, (3, 700, 64, 15, 2000)):
        cache.add(s, n)
    q, k, v = _qkv(dev, torch.float16, rows, heads, kv, dim, 1)
    fixed = cache.batch(names, width=256)

    def step(c):
        turned = append_kv(q, k, v, fixed.positions, fixed.slots, rope, c.keys[0], c.values[0])
        return paged_attention(turned, c.keys[0], c.values[0], fixed.block_tables, fixed.lengths), paged_attention(
            turned, c.keys[0], c.values[0], fixed.block_tables, fixed.lengths, window=40)

    step(cache)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            made = step(cache)
        graphs.append((g, made))
    for n in range(6):
        cache.extend(names, 1 + 13 * n)
        if n == 3:
            cache.free(4)
            cache.add(4, 9)
        cache.batch(names, out=fixed)
        k.normal_()
        g, made = graphs[n % 2]
        for t in made:
            t.fill_(float("nan"))
        g.replay()
        other = [t.clone() for t in made]
        torch.cuda.synchronize()
        for a, b in zip(other, step(cache)):
            assert torch.equal(a, b)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(other, made):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_meet(dev):
    """Long rows, split and joined, on two streams at once: each call has a workspace of its own."""
    from deltazip_amd import paged_attention
    problems = [_problem(dev, torch.float16, [6000 + i, 300], 8, 2, 128, 16, 50 + i) for i in range(2)]
    want = [paged_attention(*p) for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for p, s in zip(problems, streams):
            with torch.cuda.stream(s):
                got.append(paged_attention(*p))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_room_for_parts_outlives_a_larger_call_of_another_thread(dev):
    """Two host threads on one stream: while a call of many launches is under way, another thread's call puts larger room in the
    place of its own, and tensors made then may lie where the first call's parts are."""
    from deltazip_amd import paged_attention
    rows, n = 1 << 17, 1000
    q = torch.randn(256, 1, 8, dtype=torch.float16, device=dev).repeat(rows // 256, 1, 1)
    k, v = (torch.randn(256, 1, 1024, 8, dtype=torch.float16, device=dev) for _ in range(2))
    tables = torch.arange(256, dtype=torch.int32, device=dev).repeat(rows // 256)[:, None].contiguous()
    ln = torch.full((rows,), n, dtype=torch.int32, device=dev)
    want = paged_attention(q[:256].contiguous(), k, v, tables[:256], ln[:256])
    wide = torch.zeros(256, 512, 256, dtype=torch.float16, device=dev)
    pages = torch.zeros(1, 32, 1024, 256, dtype=torch.float16, device=dev)
    none = torch.zeros(256, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    for _ in range(4):
        stream, under_way, got, after = torch.cuda.Stream(), threading.Event(), [], []

        def many():
            with torch.cuda.stream(stream):
                paged_attention(q[:512], k, v, tables[:512], ln[:512])     # (the stream has room for this size)
                under_way.set()
                got.append(paged_attention(q, k, v, tables, ln))

        def larger():
            with torch.cuda.stream(stream):
                under_way.wait()
                after.append(paged_attention(wide, pages, pages, none[:, None], none))
                for _ in range(8):
                    after.append(torch.full((1 << 20,), 7, dtype=torch.uint8, device=dev))

        threads = [threading.Thread(target=f) for f in (many, larger)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert torch.equal(got[0].view(-1, 256, 1, 8), want.expand(rows // 256, -1, -1, -1)) and (after[0] == 0).all()
        assert all((t == 7).all() for t in after[1:])


@pytest.mark.gpu
def test_llama_steps_over_the_paged_cache(dev):
    """Sequences at positions of their own: every row's logits are those of the padded cache at its position, in a step and
    after a fork; both round to fp16 between their operators, at other places."""
    from test_llama_step import BITS, CTX, H, HEADS, LAYERS, V, I, _close, _delta_state_dict
    from deltazip_amd import CompressionConfig, DeltaConfig, DeltaMapping, DeltaModel, create_delta_manager
    from deltazip_amd.llama_step import LlamaForDecodeStep, LlamaStepConfig
    B, nd = 12, 2
    cfg = LlamaStepConfig(hidden_size=H, intermediate_size=I, num_attention_heads=HEADS, num_hidden_layers=LAYERS, vocab_size=V,
                          max_position_embeddings=64)
    model = LlamaForDecodeStep(cfg, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    mgr = create_delta_manager(model, max_num_seqs=64, max_num_batched_tokens=64, vocab_size=V,
                               delta_config=DeltaConfig(max_deltas=nd + 1, max_bitwidth=BITS))
    for d in range(1, nd + 1):
        mgr.add_delta(DeltaModel.from_tensors(_delta_state_dict(1000 * d)[0], d,
                                              CompressionConfig(bits=BITS, prunen=2, prunem=4, sparsity=0.5), pin_memory=False))
        mgr.activate_delta(d)
    ids = tuple(b % (nd + 1) for b in range(B))
    mgr.set_delta_mapping(DeltaMapping(ids, ids))
    rng = np.random.default_rng(3)
    tokens = torch.from_numpy(rng.integers(0, V, B)).to(dev)
    padded = model.make_kv_cache(B, CTX, dev, fill=0.5)
    before = [CTX, 0, 7, 16] * 3                        # tokens in front of the new one
    cache = model.make_paged_cache(40, page_size=8, device=dev)
    cache.pool.fill_(float("nan"))
    for b, n in enumerate(before):
        cache.add(b, n)
        _, slots = cache.slots(b)
        for layer, kv in enumerate(padded):
            for pages, t in zip((cache.keys[layer], cache.values[layer]), kv):
                pages[slots // 8, :, slots % 8] = t[b, :, :n].transpose(0, 1)
    cache.extend(range(B))
    got = model.paged_step(tokens, cache, cache.batch(list(range(B))))
    assert got.shape == (B, V)
    for n in set(before):
        want = model.decode_step(tokens, [(k[:, :, :n + 1].clone(), v[:, :, :n + 1].clone()) for k, v in padded], n)
        rows = [b for b in range(B) if before[b] == n]
        assert _close(got[rows].float().cpu().numpy(), want[rows].float().cpu().numpy())
    # a fork steps on from the same tokens: equal logits where parent and child have one delta, and sampled rows alone
    cache.fork(0, "child")
    names = ["child"] + list(range(1, B - 1)) + [0]
    same = (ids[0],) + ids[1:B - 1] + (ids[0],)
    mgr.set_delta_mapping(DeltaMapping(same, same))
    cache.extend(names)
    step = torch.cat((tokens[:B - 1], tokens[:1]))
    got = model.paged_step(step, cache, cache.batch(names), sample_rows=torch.tensor([0, B - 1], device=dev))
    assert got.shape == (2, V) and torch.equal(got[0], got[1]) and torch.isfinite(got).all()


@pytest.mark.gpu
def test_a_graph_replayed_before_others_and_after_eager_calls(dev):
    """Graphs share nothing: the second is replayed first, with rows that are split, and the first behind it; the number of a
    capture is its own."""
    from deltazip_amd import _lib, ops, paged_attention
    p = _problem(dev, torch.float16, [5000, 40, 9000], 8, 2, 128, 16, 77)
    want = paged_attention(*p)
    torch.cuda.synchronize()
    graphs, seen = [], []
    for _ in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            seen.append(_lib.lib().dz_capture_id(ops._stream()))
            made = [paged_attention(*p) for _ in range(3)]
        graphs.append((g, made))
    assert 0 not in seen and len(set(seen)) == 3 and _lib.lib().dz_capture_id(ops._stream()) == 0
    for n in (1, 0, 2, 0, 1, 1):
        g, made = graphs[n]
        for t in made:
            t.zero_()
        g.replay()
        assert torch.equal(paged_attention(*p), want)
        torch.cuda.synchronize()
        for t in made:
            assert torch.equal(t, want)


@pytest.mark.gpu
def test_a_bad_page_of_a_replay_is_reported_once(dev):
    from deltazip_amd import ops, paged_attention
    q, k, v, tables, ln = _problem(dev, torch.float16, [40, 20], 2, 2, 64, 16, 41)
    fixed = tables.clone()
    paged_attention(q, k, v, fixed, ln)
    ops.poll_status(dev, wait=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, fixed, ln)
    for bad in (False, True, False, True):
        fixed.copy_(tables)
        if bad:
            fixed[1, 0] = len(k) + 5
        g.replay()
        if bad:
            with pytest.raises(ops.DeltaKernelError, match="paged"):
                ops.poll_status(dev, wait=True)
        else:
            ops.poll_status(dev, wait=True)
    fixed[1, 0] = -9
    g.replay()
    torch.cuda.synchronize()
    ops.poll_status(dev)                       # starts the look,
    torch.cuda.synchronize()
    with pytest.raises(ops.DeltaKernelError, match="paged"):
        ops.poll_status(dev)                   # which the next call takes in
    ops.poll_status(dev, wait=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 192, 193, 255, 256, 257, 300])
def test_attention_of_any_number_of_rows(dev, rows):
    """Lengths that are cut into one part, several, and more than are joined at once, in any order of the rows."""
    from deltazip_amd import paged_attention
    rng = random.Random(rows)
    lengths = [rng.choice([0, 1, 5, 30, 64, 100, 383, 384, 385, 400, 600]) for _ in range(rows)]
    lengths[rng.randrange(rows)] = 7000 + 2000 * (rows % 3)
    if rows > 3:
        lengths[rng.randrange(rows)] = 17000
    p = _problem(dev, torch.float16, lengths, 2, 1, 32, 32, rows)
    got = paged_attention(*p)
    _hold(got, *p, 32 ** -0.5)
    assert torch.equal(got, paged_attention(*p))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(60))
def test_attention_over_drawn_sizes(dev, seed):
    from deltazip_amd import paged_attention
    rng = random.Random(1000 + seed)
    kv = rng.choice([1, 1, 2, 3, 5, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 7, 8, 16, 17, 24])
    dim, ps, rows = 8 * rng.randrange(1, 33), 8 << rng.randrange(0, 8), rng.choice([1, 2, 3, 7, 20, 40])
    most = max(2, 60000 // (rows * heads))
    lengths = [rng.choice([0, 1, rng.randrange(1, 40), rng.randrange(1, most), most]) for _ in range(rows)]
    q, k, v, tables, ln = _problem(dev, rng.choice(TYPES), lengths, heads, kv, dim, ps, seed)
    window = rng.choice([0, 0, 1, 7, 64, rng.randrange(1, most + 1), 2 * most])
    if rng.random() < 0.5:                              # tokens in front of heads, and both pools in one
        both = torch.stack((k.transpose(1, 2), v.transpose(1, 2)), 1).contiguous()
        k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    scale = rng.choice([dim ** -0.5, 1.0, -0.1, 0.0])
    _hold(paged_attention(q, k, v, tables, ln, scale=scale, window=window), q, k, v, tables, ln, scale, window)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(30))
def test_append_over_drawn_sizes(dev, seed):
    """Against the restatement: turned queries, and every slot of the pools, those that nothing was stored at included."""
    from deltazip_amd import RotaryPositions, append_kv
    rng = random.Random(2000 + seed)
    heads, kv, dim = rng.randrange(1, 30), rng.randrange(1, 9), 2 * rng.randrange(1, 129)
    rot, ps, tokens, dtype = 2 * rng.randrange(1, dim // 2 + 1), 8 << rng.randrange(0, 6), rng.choice([1, 2, 9, 64, 333]), rng.choice(TYPES)
    rope = RotaryPositions(dim, rotary_dim=rot, interleaved=rng.random() < 0.5, base=rng.choice([100.0, 10000.0, 1e6]))
    q, k, v = _qkv(dev, dtype, tokens, heads, kv, dim, seed)
    pages = -(-tokens // ps) + 2
    kp, vp = (torch.randn(pages, kv, ps, dim, device=dev).to(dtype) for _ in range(2))
    slots, pos = torch.randperm(pages * ps, device=dev)[:tokens], torch.randint(-50, 1 << 22, (tokens,), device=dev)
    wk, wv = kp.clone(), vp.clone()
    _turned(append_kv(q, k, v, pos, slots, rope, kp, vp), q, pos, rope)
    page, place = slots // ps, slots % ps
    _turned(kp[page, :, place], k, pos, rope)
    assert torch.equal(vp[page, :, place], v)
    wk[page, :, place], wv[page, :, place] = kp[page, :, place], v
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
