"""Attention behind prefixes, batches and runs of the paged cache: what tests/test_prefix.py leaves open."""
import random
import types

import pytest
import torch

from oracle import paged_ref as ref
from test_prefix import HEADS, TYPES, _cache, _problem, _run


# ---------------------------------------------------------------------------------------------
# attention: weights
# ---------------------------------------------------------------------------------------------


def _two_values_bound(want, size, most, dtype, dim, tokens, largest):
    """How far outputs may be off where weights are held in two values of the type.  A weight p (1 + m) is cut to the type and what is left, at most
    a step (eps) and m of p, rounded to half a step of itself: p (1 + m) (1 + d) with d up to half (eps + m), in the sum of values and in
    that of weights, so that m cancels and d counts for the sum of p |v| and |o|.  m is eps / 4; below 2^-39 of the largest float16 holds nothing."""
    half = torch.finfo(dtype).eps / 2
    d = half * (2 * half + half / 2) * (1 + 2 * half)
    lost = 2 * tokens * 2.0 ** -39 * largest if dtype == torch.float16 else 0.0
    return ref.attention_bound(want, size, most, dtype, dim, tokens) + d * (size + want.abs()) + lost


def _hold_two_values(got, q, k, v, tables, lengths, starts, groups=None, prefixes=None):
    row, length, tab = ref.tokens_as_rows(starts, lengths, tables, groups, prefixes, k.shape[2])
    want, size, most = ref.attention(q, k, v, tab, length, q.shape[2] ** -0.5)
    bound = _two_values_bound(want, size, most, q.dtype, q.shape[2], int(length.max()), float(v.nan_to_num(0, 0, 0).abs().max()))
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), f"off by up to {(off / bound).max():.2f} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,new,heads,kv,dim,prefix", [(32, 1, 2, 2, 128, 700), (64, 1, 3, 3, 64, 3000), (17, 1, 2, 2, 80, 90), (5, 3, 12, 3, 96, 400), (13, 1, 8, 2, 256, 1000),
                                                          (3, 20, 2, 2, 192, 64), (1, 64, 2, 2, 128, 0)])
def test_weights_of_up_to_64_queries_are_held_in_two_values(dev, dtype, rows, new, heads, kv, dim, prefix):
    """Units of few queries and tiles alike, and the join of both."""
    rng = random.Random(rows)
    p = _problem(dev, dtype, [prefix], [new + rng.randrange(0, 90) for _ in range(rows)], [new] * rows, [0, rows], heads, kv, dim, 16)
    _hold_two_values(_run(p), *p)


# ---------------------------------------------------------------------------------------------
# attention: what others hold
# ---------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 128), (4, 2, 64), (3, 1, 200)])
@pytest.mark.parametrize("news,groups,prefix", [([1] * 4, [0, 4], 2000), ([2, 1], [0, 2], 900), ([3], [0, 1], 0), ([5], [0, 1], 0), ([1] * 30, [0, 30], 1500)])
def test_finite_queries_and_keys_of_others_change_no_bit(dev, dtype, heads, kv, dim, news, groups, prefix):
    """Of units of few queries and of tiles: a query's sums go by its own scores."""
    p = _problem(dev, dtype, [prefix], [c + 700 for c in news], news, groups, heads, kv, dim, 16)
    want, last = _run(p), sum(news)
    for token, factor in ((0, 9.0), (last - 1, 0.0), (last // 2, -30.0)):
        q = p[0].clone()
        q[token] = q[token] * factor
        got = _run([q] + p[1:])
        keep = torch.arange(last, device=dev) != token
        assert torch.equal(got[keep], want[keep]) and not torch.equal(got[token], want[token])
    if news[0] > 1:
        # the newest key of row 0, which its other tokens do not see
        n = int(p[4][0])
        k = p[1].clone()
        k[int(p[3][0, (n - 1) // 16]), :, (n - 1) % 16] *= 20.0
        got = _run([p[0], k] + p[2:])
        keep = torch.arange(last, device=dev) != news[0] - 1
        assert torch.equal(got[keep], want[keep]) and not torch.equal(got[news[0] - 1], want[news[0] - 1])


def _one_sided(dev, dtype, tokens, scores, extra=None):
    """Tokens of 300 (256 of them a prefix) whose keys hold `scores` in their first value and `extra` in their second, which queries of ones pick."""
    from deltazip_amd import paged_attention, prefix_attention
    g = torch.Generator().manual_seed(tokens)
    k, v = torch.zeros(38 * 8, 2, 64, dtype=dtype), torch.randn(38 * 8, 2, 64, generator=g).to(dtype)
    k[:300, :, 0] = scores.to(dtype)[:, None]
    if extra is not None:
        k[:300, :, 1] = extra.to(dtype)[:, None]
    k, v = (x.view(38, 8, 2, 64).transpose(1, 2).contiguous().to(dev) for x in (k, v))
    q = torch.zeros(tokens, 2, 64, dtype=dtype)
    q[..., :2] = 1.0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    p = [q.to(dev), k, v, i32([list(range(38))] * tokens), i32([300] * tokens), i32(list(range(tokens + 1))), i32([0, tokens]), i32([256])]
    return p, lambda scale: prefix_attention(*p[:5], starts=p[5], groups=p[6], prefixes=p[7], scale=scale), lambda scale: paged_attention(*p[:5], scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 3, 40, 64, 100, 300])
def test_scores_of_any_size(dev, dtype, tokens):
    """Of 2^11 to 2^126: four tokens have the largest, alike, and their values' mean is the output, or all but four have it.  (Weights alike are rounded
    alike; sums of 300 are off by 300 2^-24 twice.)"""
    g = torch.Generator().manual_seed(5)
    for e in list(range(11, 40)) + [60, 90, 124]:
        top = torch.empty(1).uniform_(1.0, 1.9, generator=g).to(dtype)
        scores = (top / 2).repeat(300)
        where = [5, 77, 190, 290]
        scores[where] = top
        p, behind, single = _one_sided(dev, dtype, tokens, scores)
        v = p[2].transpose(1, 2).reshape(304, 2, 64)[:300].double().cpu()
        for sign in (1.0, -1.0):
            pick = torch.zeros(300, dtype=torch.bool)
            pick[where] = True
            want = v[pick if sign > 0 else ~pick].mean(0)
            for y in (behind(sign * 0.7123 * 2.0 ** e), single(sign * 0.7123 * 2.0 ** e)):
                off = (y.double().cpu() - want).abs()
                assert (off <= torch.finfo(dtype).eps / 2 * want.abs() + 600 * 2.0 ** -24 * v.abs().max() + 2.0 ** -24).all(), (e, sign)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [3, 40, 100])
@pytest.mark.parametrize("base", [1000, 2830, 2840, 2848, -2848, 20000])
def test_scores_around_where_differences_are_taken_by_themselves(dev, dtype, tokens, base):
    """Large sums with small differences, maxima of pieces on either side of the border: a score is rounded by up to 2^-23 of its size twice, whichever way it goes."""
    g = torch.Generator().manual_seed(base % 97)
    for extra in (torch.randn(300, generator=g), torch.linspace(-6, 6, 300), torch.linspace(6, -6, 300)):
        scores = torch.full((300,), float(base))
        p, behind, single = _one_sided(dev, dtype, tokens, scores, extra)
        q, k, v, tables, lengths = p[:5]
        want, size, most = ref.attention(q[:1], k, v, tables[:1], lengths[:1], 1.0)
        bound = ref.prefix_bound(want, size, most / 17, dtype, 64, 300, float(v.abs().max()))           # (4 roundings of a score, not 68)
        for y in (behind(1.0), single(1.0)):
            off = (y.double().cpu() - want).abs()
            assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [3, 40, 100, 300])
@pytest.mark.parametrize("first,then", [(-30000.0, 0.0), (-4000.0, 3.0), (-50.0, 4000.0), (-20000.0, -3000.0), (-30000.0, 30000.0)])
def test_scores_that_come_from_where_differences_are_taken_by_themselves(dev, dtype, tokens, first, then):
    """The first 130 tokens' far below the others', whose differences are small: maxima pass the border within a piece."""
    g = torch.Generator().manual_seed(3)
    scores = torch.where(torch.arange(300) < 130, torch.tensor(first), torch.tensor(then))
    p, behind, single = _one_sided(dev, dtype, tokens, scores, torch.randn(300, generator=g))
    q, k, v, tables, lengths = p[:5]
    want, size, most = ref.attention(q[:1], k, v, tables[:1], lengths[:1], 1.0)
    most = torch.full_like(most, 2 * abs(then) + 20.0)             # (of the scores that count)
    bound = ref.prefix_bound(want, size, most / 17, dtype, 64, 300, float(v.abs().max()))
    for y in (behind(1.0), single(1.0)):
        off = (y.double().cpu() - want).abs()
        assert (off <= bound).all(), float((off / bound).max())


SMALL = [([3], [3], [0], [0, 1]), ([4], [90], [0], [0, 1]), ([2] * 4, [2, 30, 2, 9], [64], [0, 4]), ([5, 1], [5, 1], [40], [0, 2]), ([1] * 8, [1, None, 7, 1, 3, None, 1, 90], [200], [0, 8])]
LARGE = [([40, 3], [70, 9], [64], [0, 2]), ([200], [200], [0], [0, 1]), ([20] * 9, [20] * 9, [128], [0, 9])]


def _hold_not_finite(got, p, spoilt):
    """Outputs of keys or values that are not finite: not finite where the definition says so, and elsewhere within the bound of the scores that are."""
    q, k, v, tables, lengths, starts, groups, prefixes = p
    row, length, tab = ref.tokens_as_rows(starts, lengths, tables, groups, prefixes, k.shape[2])
    _, _, most = ref.attention(q, k, v, tab, length, q.shape[2] ** -0.5)
    _, size, _ = ref.attention(q, spoilt[0], v, tab, length, q.shape[2] ** -0.5)
    want, _, _ = ref.attention(q, *spoilt, tab, length, q.shape[2] ** -0.5)
    bound = ref.prefix_bound(want, size, most, q.dtype, q.shape[2], int(length.max()), float(v.nan_to_num(0, 0, 0).abs().max()))
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite) and ((got - want).abs()[finite] <= bound[finite]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (4, 2, 128), (6, 3, 200), (3, 1, 256)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_who_sees_them(dev, dtype, heads, kv, dim, bad):
    """In the newest token of a row, one of the older new ones and one that all of its new ones see; units of few queries and tiles."""
    for news, suffixes, prefixes, groups in SMALL + LARGE:
        p = _problem(dev, dtype, prefixes, suffixes, news, groups, heads, kv, dim, 8)
        clean = _run(p)
        n, c, share = int(p[4][0]), news[0], heads // kv
        for t in {n - 1, n - c, n - (c + 1) // 2, max(prefixes[0], n - c - 1)}:
            v = p[2].clone()
            v[int(p[3][0, t // 8]), 0, t % 8, 3] = bad
            got = _run([p[0], p[1], v] + p[3:])
            first = max(0, t - (n - c))                            # the first of row 0's new tokens that sees it
            seen = torch.zeros_like(clean, dtype=torch.bool)
            seen[first:c, :share, 3] = True
            assert torch.equal(got[~seen], clean[~seen]) and not torch.isfinite(got[seen]).any()
            if t > n - c:                                          # (in a step that some do not see: as it is)
                assert torch.equal(torch.isnan(got[seen]), torch.full_like(got[seen], bad != bad, dtype=torch.bool))
                assert bad != bad or (got[seen] == bad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (6, 3, 200)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", ["keys", "both"])
def test_keys_that_are_not_finite_reach_who_sees_them(dev, dtype, heads, kv, dim, bad, which):
    """As scores that are not finite do in the definition: NaN, or, far below all others, no weight."""
    for news, suffixes, prefixes, groups in SMALL + LARGE:
        p = _problem(dev, dtype, prefixes, suffixes, news, groups, heads, kv, dim, 8, poison=False)
        clean = _run(p)
        n, c, share = int(p[4][0]), news[0], heads // kv
        for t in {n - 1, n - (c + 1) // 2, max(prefixes[0], n - c - 1)}:
            if n == 1 or (t == 0 and bad == bad):
                continue                                           # (a token's only score)
            k, v = p[1].clone(), p[2].clone()
            for x in (k, v)[:1 if which == "keys" else 2]:
                x[int(p[3][0, t // 8]), 0, t % 8, 3] = bad
            got = _run([p[0], k, v] + p[3:])
            first = max(0, t - (n - c))
            assert torch.equal(got[:first], clean[:first]) and torch.equal(got[c:], clean[c:]) and torch.equal(got[:, share:], clean[:, share:])
            if bad != bad:
                assert torch.isnan(got[first:c, :share]).all()
            _hold_not_finite(got, p, (k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (4, 2, 128), (3, 3, 200)])
def test_queries_of_padded_rows_that_are_not_finite_stay_with_themselves(dev, dtype, heads, kv, dim):
    """In a group's unit of few queries, among the others of a matrix instruction."""
    for prefix in (40, 700):
        p = _problem(dev, dtype, [prefix], [1, None, 7, 1, 3, None, 1, 90], [1] * 8, [0, 8], heads, kv, dim, 8)
        want = _run(p)
        assert (want[[1, 5]] == 0).all()
        for bad in (float("nan"), float("inf")):
            p[0][1], p[0][5] = bad, -bad
            assert torch.equal(_run(p), want)
        for bad in (float("nan"), float("inf"), 6e4):
            q = p[0].clone()
            q[6] = bad
            got = _run([q] + p[1:])
            keep = torch.arange(8, device=dev) != 6
            assert torch.equal(got[keep], want[keep])
            assert bad == 6e4 or torch.isnan(got[6]).all()


@pytest.mark.gpu
def test_more_workgroups_than_a_line_of_a_grid_has(dev):
    """Rows times key heads beyond 2^24: every output, against the same in 32 bits."""
    from deltazip_amd import prefix_attention
    rows, heads, dim, ps = 530001, 32, 8, 8
    g = torch.Generator(device=dev).manual_seed(0)
    k, v = (torch.randn(3, heads, ps, dim, generator=g, device=dev).half() for _ in range(2))
    q = torch.randn(rows, heads, dim, generator=g, device=dev).half()
    lengths = torch.randint(0, ps + 1, (rows,), generator=g, device=dev, dtype=torch.int32)
    tables = torch.tensor([[2]], dtype=torch.int32, device=dev).expand(rows, 1)
    got = prefix_attention(q, k, v, tables, lengths, starts=torch.arange(rows + 1, dtype=torch.int32, device=dev))
    half = torch.finfo(torch.float16).eps / 2
    for h in range(heads):
        s = dim ** -0.5 * (q[:, h].float() @ k[2, h].float().t().contiguous())
        p = torch.softmax(s.masked_fill(torch.arange(ps, device=dev) >= lengths[:, None], -1e30), 1)
        want = (p @ v[2, h].float()) * (lengths > 0)[:, None]
        # (both sides' sums of 8 in 32 bits, and exponentials: 2^-19 of the largest value)
        assert ((got[:, h].float() - want).abs() <= half * want.abs() + 2.0 ** -19 * 5 + 2.0 ** -24).all(), h


@pytest.mark.gpu
@pytest.mark.parametrize("into", [False, True])
def test_calls_of_several_threads_on_one_stream(dev, into):
    """Plans, sums and joins of a call lie in the stream's room: no other's launch may come between them."""
    import threading
    from deltazip_amd import paged_attention
    few = _problem(dev, torch.float16, [600], [30] * 5, [1] * 5, [0, 5], 4, 2, 64, 16, seed=1)
    many = _problem(dev, torch.float16, [40, 900], [9] * 300, [2] * 300, [0, 200, 300], 8, 2, 64, 16, seed=2)
    long = _problem(dev, torch.float16, [0], [9000] * 3, [1] * 3, [0, 3], 8, 2, 64, 16, seed=3)
    calls = [lambda out: _run(few, out=out), lambda out: _run(many, out=out), lambda out: paged_attention(*long[:5], out=out)]
    want = [call(None) for call in calls]
    stream, got = torch.cuda.Stream(), [[] for _ in calls]
    torch.cuda.synchronize()

    def repeat(call, like, kept):
        with torch.cuda.stream(stream):
            for _ in range(150):
                kept.append(call(torch.empty_like(like) if into else None))

    threads = [threading.Thread(target=repeat, args=x) for x in zip(calls, want, got)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(kept) == 150 and all(torch.equal(x, w) for x in kept) for kept, w in zip(got, want))


# ---------------------------------------------------------------------------------------------
# groups
# ---------------------------------------------------------------------------------------------


def test_padded_rows_do_not_cut_a_group(monkeypatch):
    cache = _cache(monkeypatch=monkeypatch, pages=400)
    cache.add("p", 80)
    rows = [None if i % 16 == 15 else i for i in range(60)]
    for i in rows:
        if i is not None:
            cache.fork("p", i)
    cache.extend([i for i in rows if i is not None])
    for seqs, bounds, sizes in ((rows, [0, 60], [80]), ([None, None] + rows + [None] * 3, [0, 2, 62, 65], [0, 80, 0]), ([None, 1, None], [0, 3], [0]), ([None] * 3, [0, 3], [0])):
        b = cache.batch(seqs, prefix=True)
        n = len(bounds)
        assert b.groups.tolist()[:n] == bounds and set(b.groups.tolist()[n:]) <= {len(seqs)}
        assert b.prefixes.tolist()[:n - 1] == sizes and not any(b.prefixes.tolist()[n - 1:])
    assert cache.batch([None, None], width=0, prefix=True).prefixes.tolist() == [0, 0]
    run = cache.run([0, None, None, 1, 2], 1, prefix=True)
    b = run.step()
    assert b.groups.tolist() == [0, 5] and b.prefixes.tolist() == [80] and b.shared
    run.finish()
    run = cache.run([0] + [None] * 40, 1, prefix=True)
    assert not run.step().shared
    run.finish()


@pytest.mark.parametrize("seed", range(20))
def test_groups_over_padded_rows_hold_what_their_rows_share(seed):
    """And are those of the rows without the padded ones."""
    import numpy as np
    cache, rng = _cache(), random.Random(seed)
    rows, w = rng.randrange(1, 30), 6
    used = np.array([rng.choice([0, rng.randrange(1, w + 1)]) for _ in range(rows)])
    tables, last = np.zeros((rows, w), dtype=np.int32), None
    for r in np.flatnonzero(used):
        keep = 0 if last is None else min(rng.randrange(0, w + 1), used[r], used[last])
        tables[r, :used[r]] = [tables[last, i] if i < keep else 100 * r + i + 1 for i in range(used[r])]
        last = r
    bounds, sizes = cache._groups_of(tables, used)
    assert bounds[0] == 0 and bounds[-1] == rows and len(sizes) == len(bounds) - 1 and (np.diff(bounds) > 0).all()
    alive = np.flatnonzero(used)
    for a, b, n in zip(bounds, bounds[1:], sizes):
        mine = [r for r in range(a, b) if used[r]]
        assert n % 8 == 0 and (n == 0 or (len(mine) > 1 and used[a] and used[b - 1] and all(used[r] >= n // 8 and (tables[r, :n // 8] == tables[a, :n // 8]).all() for r in mine)))
    packed, shares = cache._groups_of(tables[alive], used[alive])
    assert [(list(alive[a:b]), n) for a, b, n in zip(packed, packed[1:], shares) if n] == [
        ([r for r in range(a, b) if used[r]], n) for a, b, n in zip(bounds, bounds[1:], sizes) if n]


# ---------------------------------------------------------------------------------------------
# batches
# ---------------------------------------------------------------------------------------------


def test_a_batch_is_five_items_whatever_it_holds_besides():
    import copy
    import pickle
    from deltazip_amd import PagedBatch
    cache = _cache()
    cache.add("a", 21)
    cache.add("b", 4)
    for kw in (dict(), dict(prefix=True), dict(tokens=[3, 2]), dict(tokens=[1, 0], prefix=True)):
        b = cache.batch(["a", "b"], **kw)
        positions, slots, tables, lengths, shared = b
        assert positions is b.positions and lengths.tolist() == [21, 4] and shared is False and len(b) == 5
        assert (b.starts is not None) == ("tokens" in kw) and (b.groups is not None) == (b.prefixes is not None) == ("prefix" in kw)
        other = b._replace(shared=True)
        assert type(other) is PagedBatch and other.shared and other.starts is b.starts and other.groups is b.groups and other.slots is slots
        for same in (pickle.loads(pickle.dumps(b)), copy.copy(b), copy.deepcopy(b)):
            for name in ("positions", "slots", "block_tables", "lengths", "starts", "groups", "prefixes"):
                x, y = getattr(b, name), getattr(same, name)
                assert (x is None and y is None) or torch.equal(x, y)
    b = cache.batch(["a", None], prefix=True)
    again = cache.batch([None, "b"], prefix=True, out=b)
    assert again.groups is b.groups and again.lengths is b.lengths and b.lengths.tolist() == [0, 4]
    assert PagedBatch(positions, slots, tables, lengths, True, b.starts, b.groups, b.prefixes).prefixes is b.prefixes


# ---------------------------------------------------------------------------------------------
# runs
# ---------------------------------------------------------------------------------------------


def test_a_run_is_finished_once_the_device_is_done(monkeypatch):
    """Not when the current stream is: steps may be on others."""
    cache = _cache(monkeypatch=monkeypatch)
    cache.add("a", 8)
    run = cache.run(["a"], 9)
    run.step()
    before = run._lengths.clone()

    def wait(device):
        if (run._lengths == before).all():
            run.step()                                 # (what was still under way)
    monkeypatch.setattr(torch.cuda, "synchronize", wait)
    cache.pool = types.SimpleNamespace(is_cuda=True, device="cuda:0")
    run.finish()
    assert cache.length("a") == 10 and len(cache.pages("a")) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_runs_whose_steps_are_on_another_stream(dev, captured):
    """Behind long work on that stream, finished from the current one."""
    from deltazip_amd import PagedKVCache
    cache = PagedKVCache(1, 60, 8, 1, 8, max_tokens=200, device=dev)
    for x, n in (("a", 7), ("b", 16)):
        cache.add(x, n)
    run = cache.run(["a", "b"], 20)
    work, side, graph = torch.randn(4096, 4096, device=dev), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        run.step()
        if captured:
            with torch.cuda.graph(graph, stream=side):
                run.step()
        for _ in range(20):
            work = work @ work / 64.0
        for _ in range(19):
            graph.replay() if captured else run.step()
    run.finish()
    assert cache.length("a") == 27 and cache.length("b") == 36 and cache.free_pages == 60 - 4 - 5
    held = [p for x in "ab" for p in cache.pages(x)]
    assert len(set(held)) == 9 and sorted(held + cache._free) == list(range(60))


def test_a_run_that_is_dropped_gives_its_sequences_back(monkeypatch):
    cache = _cache(monkeypatch=monkeypatch)
    cache.add("a", 10)
    cache.add("b", 3)
    with pytest.raises(KeyError):
        with cache.run(["a"], 20) as run:
            run.step()
            raise KeyError
    assert cache.length("a") == 11 and cache.runs == () and cache.free_pages == 200 - 3
    cache.run(["a", None], 20).step()
    cache.run(["b"], 1)
    with pytest.raises(ValueError, match="runs"):
        cache.free("a")
    for run in cache.runs:
        run.finish()
        run.finish()
    assert cache.runs == () and cache.length("a") == 12 and cache.length("b") == 3
    cache.free("a")
    cache.free("b")
    assert cache.free_pages == 200


# ---------------------------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [256, 257, 600, 1025, 1777])
def test_steps_of_many_rows_over_their_inputs(dev, rows):
    """A place a row, as a run steps: more than one workgroup, lengths and pages taken left to a launch of their own; by calls and by replays, until the
    pages are at an end and nothing goes on."""
    from deltazip_amd import TableStep, extend_tables, ops
    rng = random.Random(rows)
    ps, width, steps = 8, 8, 12
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    lengths, counts = [rng.randrange(0, 40) for _ in range(rows)], [rng.choice([0, 1, 1, 1]) for _ in range(rows)]
    tables = [[100000 + width * r + i if i < -(-n // ps) else -7 for i in range(width)] for r, n in enumerate(lengths)]
    state, free = (tables, lengths, 0), rng.sample(range(90000), 2 * rows)
    for _ in range(steps):
        state = ref.extend_tables(state[0], state[1], counts, free, state[2], ps)
    free = free[:state[2]]                             # (just enough for so many steps)
    tab, ln, ct, fr, tk = (i32(x) for x in (tables, lengths, counts, free, [0]))
    out = TableStep(ln, tk, torch.empty(rows + 1, dtype=torch.int32, device=dev), *torch.empty(2, rows, dtype=torch.int64, device=dev))
    step = lambda: extend_tables(tab, ln, ct, fr, tk, ps, out=out)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    state = ref.extend_tables(tables, lengths, counts, free, 0, ps)
    for i in range(1, steps + 30):
        assert tab.tolist() == state[0] and ln.tolist() == state[1] and tk.tolist() == [state[2]]
        if i <= steps:
            assert [out.starts.tolist(), out.positions.tolist(), out.slots.tolist()] == list(state[3:])
        graph.replay() if i % 2 else step()
        after = ref.extend_tables(state[0], state[1], counts, free, state[2], ps)
        if after is None:
            assert i >= steps and out.slots.tolist() == [-1] * rows and ln.tolist() == state[1] and tab.tolist() == state[0] and tk.tolist() == [state[2]]
            with pytest.raises(ops.DeltaKernelError, match="paged"):
                ops.poll_status(wait=True)
            return
        state = after
    raise AssertionError("steps without an end")
