"""Paged attention of requests that continue others, whose tokens are held
once: the plan exactly, the attention against 64 bits."""

import random

import paged_scores_reference as R
import pytest
import torch

import sunshape_mlx_amd as S
from test_gpu_paged_scores import BF16, DEV, F16, SHAPES, ints, pool, queries, slopes_of

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the plan


def plan_of(parents, lengths, starts, n):
    """(group starts, rows, parents, positions) as plain lists."""
    r = len(parents)
    bad = any(b < a for a, b in zip(starts, starts[1:]))
    of = [-1 if bad or not 0 <= p < r or p == i or starts[i] < 0 else p for i, p in enumerate(parents)]
    groups = [[] for _ in range(r)]
    positions = [-1] * n
    for i in range(0 if bad else r):
        for t in range(max(0, starts[i]), min(starts[i + 1], n)):
            own = lengths[i] - (starts[i + 1] - t)
            if of[i] >= 0:
                groups[of[i]].append((t, own))
            positions[t] = max(-1, own + (lengths[of[i]] if of[i] >= 0 else 0))
    out = [0]
    for g in groups:
        out.append(out[-1] + len(g))
    return out, [x for g in groups for x in g], of, positions


def check_plan(parents, lengths, starts, n):
    got = S.build_shared_plan(ints(parents), ints(lengths), ints(starts), n)
    groups, rows, of, positions = plan_of(parents, lengths, starts, n)
    assert got.group_starts.cpu().tolist() == groups
    assert got.rows.cpu().tolist()[:len(rows)] == [list(x) for x in rows]
    assert got.parents.cpu().tolist() == of
    assert got.positions.cpu().tolist() == positions


@pytest.mark.parametrize("r,most,pad", [(1, 3, 0), (2, 1, 2), (3, 9, 0), (64, 1, 0), (65, 4, 3), (130, 2, 0),
                                        (1024, 3, 5), (1025, 1, 0), (4096, 2, 1), (700, 20, 7)])
def test_plans(r, most, pad):
    """Few parents and many, up to the most requests and more tokens than one
    workgroup writes."""
    rng = random.Random(r)
    for few in (True, False):
        parents = [rng.choice([-1, 0, r // 2, r - 1] if few else [rng.randint(-3, r + 3)]) for _ in range(r)]
        new = [rng.randint(0, most) for _ in range(r)]
        lengths = [n + rng.randint(0, 1000) for n in new]
        starts = [sum(new[:i]) for i in range(r + 1)]
        check_plan(parents, lengths, starts, starts[-1] + pad)


def test_plans_of_odd_starts():
    check_plan([1, -1, 1], [5, 9, 7], [2, 4, 5, 8], 10)          # rows before the first request
    check_plan([1, -1, 1], [5, 9, 7], [0, 2, 1, 4], 6)           # starts that descend: no rows
    check_plan([1, -1, 1], [5, 9, 7], [0, 2, 4, 9], 6)           # more rows than there are
    check_plan([-(2 ** 31), 2 ** 31 - 1, 2], [1, 1, 1], [0, 1, 2, 3], 3)
    check_plan([1, 0, 0], [4, 4, 4], [0, 2, 4, 6], 6)            # each other's: one level is followed
    many = [sum([61, 0, 93][i % 3] for i in range(j)) for j in range(301)]
    check_plan([i % 2 * 7 for i in range(300)], [200] * 300, many, many[-1] + 9)
    many[5] = many[4] - 1
    check_plan([i % 2 * 7 for i in range(300)], [200] * 300, many, many[-1] + 9)


# ----------------------------------------------------------- the attention


def run(seed, lengths, new, parents, hq=8, hkv=2, d=128, group=64, page=16, dtype=F16, pad=0, hints=True,
        ordinary=True, out=None, scale=None, causal=True, **kw):
    """A call against the reference."""
    store, table = pool(seed, lengths, hkv, d, group, page, dtype)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    n = starts[-1] + pad
    q, le, st = queries(seed + 1, n, hq, d, dtype), ints(lengths), ints(starts)
    scale = d ** -0.5 if scale is None else scale
    more, groups = {}, 1
    if hints:
        kids = [p for p in parents if p >= 0]
        groups = max(1, len(set(kids)))
        more = dict(max_new=max(1, max(new)),
                    max_length=max([x for i, x in enumerate(lengths) if i not in kids] or [1]))
    plan = S.build_shared_plan(ints(parents), le, st, n, n_groups=groups,
                               max_shared=max([lengths[p] for p in parents if p >= 0] or [0]) if hints else None)
    got = S.paged_attention(q, store, table, le, st, scale, shared=plan, causal=causal, out=out, **more, **kw)
    want = R.attend(q, store, table, le, st, scale, parents=parents, causal=causal, **kw)
    error = R.check(got[:starts[-1]], [x[:starts[-1]] for x in want], ordinary)
    assert not error, error
    if out is None:
        assert not bool(got[starts[-1]:].any())
    return got


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("many", [False, True])
def test_one_prefix(many, dtype, d, group):
    """Steps of a few requests behind one prefix, and of so many that the
    prompt kernel takes the prefix."""
    b = 40 if many else 3
    rng = random.Random(b)
    own = [rng.randint(1, 90) for _ in range(b)]
    for prefix in (700, 2600):
        run(prefix, [prefix, *own], [0] + [1] * b, [-1] + [0] * b, d=d, group=group, dtype=dtype, pad=2)


@pytest.mark.parametrize("hints", [False, True])
@pytest.mark.parametrize("page", [16, 128])
def test_several_prefixes_and_requests_without(hints, page):
    """Children of three prefixes in any order, requests that continue nothing,
    and prefixes that nobody continues; drafts and prompts among them."""
    lengths = [300, 5, 900, 40, 1, 33, 400, 70, 7, 2, 260]
    new = [0, 0, 0, 3, 1, 7, 130, 1, 2, 1, 64]
    parents = [-1, -1, -1, 2, 0, -1, 2, 2, 0, 6, -1]
    run(3, lengths, new, parents, page=page, hints=hints)
    run(4, lengths, new, parents, page=page, hints=hints, d=64, group=32, hq=8, dtype=BF16, pad=4,
        softcap=6.0, slopes=slopes_of(8, 0.1))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 127, 128, 129, 1024, 1025, 5000])
def test_prefix_lengths(prefix):
    run(prefix + 1, [prefix, 1, 20, 9], [0, 1, 2, 9], [-1, 0, 0, 0])
    b = 33
    run(prefix + 2, [prefix] + [3] * b, [0] + [3] * b, [-1] + [0] * b, hq=4, hkv=1, page=64)


@pytest.mark.parametrize("own", [1, 130, 1100, 4000])
def test_own_tokens_of_any_length(own):
    """Columns of own tokens that stay whole and that are cut."""
    run(own, [500, own, own // 2 + 1, 5], [0, 1, 1, 2], [-1, 0, 0, 0], page=64)
    run(own + 1, [3000, own, 200, 7], [0, min(own, 200), 150, 7], [-1, 0, 0, 0], page=64, hints=False)


@pytest.mark.parametrize("kw", [dict(softcap=4.0), dict(slopes=0.3), dict(softcap=20.0, slopes=0.02)])
@pytest.mark.parametrize("many", [False, True])
def test_with_caps_and_distances(kw, many):
    """Distances count the prefix."""
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(8, kw["slopes"])
    b = 30 if many else 2
    run(5, [1500] + [50] * b, [0] + [3] * b, [-1] + [0] * b, **kw)


def test_all_own_tokens_seen():
    run(6, [300, 40, 50], [0, 4, 5], [-1, 0, 0], causal=False)


@pytest.mark.parametrize("kw", [dict(scale=100.0), dict(scale=1e4, slopes=1.0), dict(scale=0.0),
                                dict(slopes=200.0), dict(scale=-0.2)])
@pytest.mark.parametrize("many", [False, True])
def test_scores_of_any_size(kw, many):
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(8, kw["slopes"])
    b = 40 if many else 3
    run(7, [1300] + [70] * b, [0] + [1] * b, [-1] + [0] * b, ordinary=False, **kw)


def test_parents_that_add_tokens_and_children_that_hold_none():
    """A prefix that grows in the same step; rows in front of their request's
    tokens see the prefix alone."""
    run(8, [200, 0, 3], [5, 2, 4], [-1, 0, 0])
    run(9, [0, 0, 3], [0, 2, 1], [-1, 0, 0])


@pytest.mark.parametrize("hq,hkv", [(2, 2), (71, 1), (28, 4)])
def test_head_groups(hq, hkv):
    run(10, [700, 33, 1, 90], [0, 1, 1, 4], [-1, 0, 0, 0], hq=hq, hkv=hkv, d=64, group=64)


def test_values_of_bfloat16_of_any_size():
    """Sums of either pass keep bfloat16's range."""
    store, table = pool(11, [600] + [40] * 30, 2, 128, 64, 16, BF16)
    for f in (2.0 ** 100, 2.0 ** -90):
        s2 = S.PagedKVStore(store.k_codes, store.v_codes, store.k_meta, store.v_meta * f)
        n = 30
        q, le, st = queries(12, n, 8, 128, BF16), ints([600] + [40] * n), ints([0] + list(range(n + 1)))
        plan = S.build_shared_plan(ints([-1] + [0] * n), le, st, n)
        got = S.paged_attention(q, s2, table, le, st, 0.1, shared=plan)
        error = R.check(got, R.attend(q, s2, table, le, st, 0.1, parents=[-1] + [0] * n))
        assert not error, error


def test_rows_of_no_request_are_left_with_out():
    out = torch.full((7, 8, 128), 7.0, dtype=F16, device=DEV)
    got = run(13, [90, 4, 5], [0, 2, 3], [-1, 0, 0], pad=2, out=out)
    assert got is out and bool((out[5:] == 7.0).all())


def test_wrong_hints_change_roundings_only():
    lengths, new, parents = [2500, 300, 60, 9, 20], [0, 90, 1, 1, 1], [-1, -1, 0, 0, 1]
    store, table = pool(14, lengths, 2, 128, 64, 64, F16)
    starts = ints([0, 0, 90, 91, 92, 93])
    q, le = queries(15, 93, 8, 128, F16), ints(lengths)
    want = R.attend(q, store, table, le, starts, 0.1, parents=parents)
    plan = S.build_shared_plan(ints(parents), le, starts, 93)
    for groups, most in ((1, None), (5, 1), (100, 10 ** 6), (2, 2500)):
        for hints in (dict(), dict(max_new=1, max_length=1), dict(max_new=1000, max_length=10 ** 6)):
            got = S.paged_attention(q, store, table, le, starts, 0.1,
                                    shared=plan._replace(n_groups=groups, max_shared=most), **hints)
            error = R.check(got, want)
            assert not error, (groups, most, hints, error)


@pytest.mark.parametrize("d,group", [(128, 64), (64, 32)])
def test_many_prefixes_where_one_is_expected(d, group):
    """More columns than workgroups, which then take several one after the other."""
    rng = random.Random(d)
    lengths = [2500] + [rng.randint(1, 300) for _ in range(63)] + [rng.randint(8, 40) for _ in range(64)]
    new, parents = [0] * 64 + [8] * 64, [-1] * 64 + rng.sample(range(64), 64)
    store, table = pool(33, lengths, 8, d, group, 16, F16, width=1 << 12)
    starts = ints([sum(new[:i]) for i in range(129)])
    q, le = queries(34, 512, 32, d, F16), ints(lengths)
    plan = S.build_shared_plan(ints(parents), le, starts, 512, n_groups=1)
    got = S.paged_attention(q, store, table, le, starts, 0.1, shared=plan, max_new=8, max_length=40)
    error = R.check(got, R.attend(q, store, table, le, starts, 0.1, parents=parents))
    assert not error, error


@pytest.mark.parametrize("prefix", [33 * 64 * 8, 40000])
def test_a_prefix_in_more_parts_than_are_joined_at_once(prefix):
    lengths = [prefix] + [5 + i % 7 for i in range(64)]
    for d, group, dtype, kw in ((128, 64, BF16, {}), (64, 64, F16, dict(softcap=7.0))):
        run(35, lengths, [0] + [1] * 64, [-1] + [0] * 64, hq=4, hkv=1, d=d, group=group, page=128, dtype=dtype, **kw)


def test_graphs_follow_the_plan():
    """The plan and the attention captured, replayed with other parents and
    lengths and eager work between."""
    store, table = pool(16, [800, 500, 70, 70, 70], 2, 128, 64, 16, F16)
    parents, le = ints([-1, -1, 0, 0, 1]), ints([800, 500, 70, 70, 70])
    starts, q = ints([0, 0, 0, 1, 3, 4]), queries(17, 4, 8, 128, F16)

    def call():
        plan = S.build_shared_plan(parents, le, starts, 4, n_groups=2)
        return plan.positions, S.paged_attention(q, store, table, le, starts, 0.1, shared=plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i, p in enumerate(([-1, -1, 1, 1, 0], [-1] * 5, [-1, -1, -1, 0, 0], [-1, -1, 0, 0, 0])):
        parents.copy_(ints(p))
        le.copy_(ints([800 - i, 500 - 9 * i, 70, 60 + i, 70]))
        q.copy_(queries(20 + i, 4, 8, 128, F16))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        error = R.check(out[1], R.attend(q, store, table, le, starts, 0.1, parents=p))
        assert not error, error


# -------------------------------------------------------------- the cache


def serve(cache, table, step, new, **kw):
    """One step of the layer: (queries, output)."""
    n = sum(max(0, x) for x in new)
    q, k, v = (queries(100 * step + i, n, h, 64, F16) for i, h in enumerate((8, 2, 2)))
    cache.step(new)
    q = cache.append_rotated(q, k, v, table)
    return q, cache.attend(q, 0.125, **kw)


@pytest.mark.parametrize("on_gpu", [False, True])
def test_a_cache_shares(on_gpu):
    """Requests fork behind a prompt, go on, end and fork again; every step's
    attention is that over the prompt's tokens and their own, at positions that
    follow the prompt's."""
    cache = S.PagedKVCache(n_requests=6, n_kv_heads=2, head_dim=64, max_tokens=400, page_size=16, device=DEV)
    turn = S.rotary_table(1000, 64, device=DEV)
    if on_gpu:  # the host no longer knows the lengths
        cache.step(ints([0] * 6), 0)
    serve(cache, turn, 1, [333, 0, 0, 0, 0, 50])
    cache.share([1, 2, 4], 0)
    cache.share([3], 5)
    parents = [-1, 0, 0, 5, 0, -1]
    for step, new in enumerate(([0, 3, 90, 5, 1, 0], [0, 1, 1, 1, 1, 1], [0, 4, 4, 4, 4, 0])):
        q, got = serve(cache, turn, step + 2, new, softcap=10.0)
        want = R.attend(q, cache.store, cache.block_table, cache.lengths, cache.plan.token_starts, 0.125,
                        parents=parents, softcap=10.0)
        error = R.check(got, want)
        assert not error, error
        lengths, starts = cache.lengths.cpu().tolist(), cache.plan.token_starts.cpu().tolist()
        assert cache.plan.positions.cpu().tolist() == plan_of(parents, lengths, starts, sum(new))[3]
    with pytest.raises(ValueError):
        cache.release([0])
    cache.trim(2)
    assert cache.lengths.cpu().tolist() == [333, 6, 93, 8, 4, 51]
    cache.release([1, 2])
    assert cache.lengths.cpu().tolist() == [333, 0, 0, 8, 4, 51]
    cache.release([0, 4])
    parents = [-1, -1, -1, 5, -1, -1]
    q, got = serve(cache, turn, 9, [20, 1, 0, 1, 2, 0])
    want = R.attend(q, cache.store, cache.block_table, cache.lengths, cache.plan.token_starts, 0.125,
                    parents=parents)
    error = R.check(got, want)
    assert not error, error
    cache.release(range(6))
    assert int(cache.n_free) == cache.free_pages.shape[0] and cache.shared is not None
    serve(cache, turn, 10, [1] * 6)
    assert cache.shared is None
