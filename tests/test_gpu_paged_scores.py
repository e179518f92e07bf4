"""Paged attention with capped and biased scores, windows and open prefixes,
against 64 bits."""

import math
import random

import paged_scores_reference as R
import pytest
import torch

import sunshape_mlx_amd as S

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPES = [(128, 64), (128, 128), (128, 32), (64, 64), (64, 32)]
F16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def slopes_of(hq, most=0.5):
    return most * 2.0 ** (-8.0 * torch.arange(hq, device=DEV) / hq)


def pool(seed, lengths, hkv, d, group, page, dtype, spare=2, width=None):
    """A filled store and the block table of requests of these lengths."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    have = [-(-n // page) for n in lengths]
    total = sum(have) + spare
    store = S.PagedKVStore.zeros(total, hkv, d, page_size=page, group_size=group, dtype=dtype, device=DEV)
    s = 0.5 + 3.5 * torch.rand((d,), generator=g, device=DEV)
    n = total * page
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    S.append_paged(store, (torch.randn((n, hkv, d), generator=g, device=DEV) * s).to(dtype),
                   torch.randn((n, hkv, d), generator=g, device=DEV).to(dtype), slots)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), width or max(1, max(have))), -1, dtype=torch.int32)
    for r, k in enumerate(have):
        for j in range(k):
            table[r, j] = order.pop()
    return store, table.to(DEV)


def queries(seed, n, hq, d, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((n, hq, d), generator=g, device=DEV).to(dtype)


def run(seed, lengths, new, hq, hkv, d, group, page, dtype, scale=None, hints=True, pad=0,
        ordinary=True, **kw):
    """One call against the reference."""
    store, table = pool(seed, lengths, hkv, d, group, page, dtype)
    n = sum(new) + pad
    q = queries(seed + 1, n, hq, d, dtype)
    starts = ints([sum(new[:i]) for i in range(len(new) + 1)])
    scale = d ** -0.5 if scale is None else scale
    call = dict(kw)
    if call.get("prefix") is not None:
        call["prefix_lengths"] = ints(call.pop("prefix"))
    else:
        call.pop("prefix", None)
    if hints:
        call.update(max_new=max(new), max_length=max(lengths))
    got = S.paged_attention(q, store, table, ints(lengths), starts, scale, **call)
    want = R.attend(q, store, table, ints(lengths), starts, scale, **kw)
    error = R.check(got, want, ordinary)
    assert not error, error
    assert not bool(got[sum(new):].any())
    return got


CASES = {
    "cap": dict(softcap=5.0),
    "high cap": dict(softcap=50.0),
    "slopes": dict(slopes=0.5),
    "cap and slopes": dict(softcap=8.0, slopes=0.25),
    "window": dict(window=37),
    "one token": dict(window=1),
    "window and cap": dict(window=130, softcap=5.0),
    "prefix": dict(prefix=[64, 5, 0]),
    "prefix, window and slopes": dict(prefix=[90, 1000, -3], window=100, slopes=0.1),
    "all, in a window": dict(causal=False, window=50, slopes=0.1),
    "all, capped": dict(causal=False, softcap=3.0),
}


def options(name, hq):
    kw = dict(CASES[name])
    if "slopes" in kw:
        kw["slopes"] = slopes_of(hq, kw["slopes"])
    return kw


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_steps(dtype, d, group, name):
    """Decode steps and drafts: the few rows of the decode kernel, whole columns
    and cut ones."""
    kw = options(name, 8)
    run(1, [509, 33, 700], [1, 1, 1], 8, 2, d, group, 16, dtype, **kw)
    run(2, [2600, 300, 1], [4, 7, 1], 8, 2, d, group, 64, dtype, pad=3, **kw)


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompts(dtype, d, group, name):
    """Prompts and chunks beside steps: the prompt kernel, whole columns and cut
    ones, takes the many rows."""
    forced(4, [421, 900, 77], [421, 130, 1], 8, 2, d, group, 32, dtype, **options(name, 8))


def forced(seed, lengths, new, hq, hkv, d, group, page, dtype, **kw):
    """A call whose hints are those of a large one: rows past 64 a KV head are
    the prompt kernel's."""
    store, table = pool(seed, lengths, hkv, d, group, page, dtype)
    n = sum(new)
    q = queries(seed + 1, n, hq, d, dtype)
    starts = ints([sum(new[:i]) for i in range(len(new) + 1)])
    call = dict(kw)
    prefix = call.pop("prefix", None)
    if prefix is not None:
        call["prefix_lengths"] = ints(prefix)
    wide = torch.full((table.shape[0], 1 << 14), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    got = S.paged_attention(q, store, wide, ints(lengths), starts, d ** -0.5, **call)
    want = R.attend(q, store, table, ints(lengths), starts, d ** -0.5, **kw)
    error = R.check(got, want)
    assert not error, error
    return got


@pytest.mark.parametrize("hq,hkv", [(4, 4), (7, 1), (28, 4), (71, 1)])
@pytest.mark.parametrize("name", ["cap and slopes", "prefix, window and slopes"])
def test_head_groups(hq, hkv, name):
    kw = options(name, hq)
    run(5, [700, 90, 3], [1, 2, 3], hq, hkv, 64, 32, 16, F16, **kw)
    forced(6, [300, 90, 333], [300, 2, 200], hq, hkv, 128, 64, 16, F16, **kw)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 127, 128, 129, 500, 4095, 1 << 40])
def test_windows_at_tile_and_page_ends(window):
    run(7, [1023, 1024, 1025, 129], [1, 1, 3, 129], 8, 2, 128, 64, 64, F16, window=window)
    forced(8, [1024, 1537, 400], [300, 128, 400], 8, 2, 128, 64, 64, F16, window=window)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 255, 257, 2047, 2049, 5000])
def test_lengths(length):
    for kw in (dict(softcap=10.0, slopes=slopes_of(8)), dict(window=200), dict(prefix=[40, 40])):
        run(length, [length, 1], [1, 1], 8, 2, 128, 64, 16, BF16, **kw)
        run(length, [length, 20], [min(length, 5), 20], 8, 2, 64, 64, 16, F16, **kw)


def test_no_tokens_and_rows_before_them():
    """Requests that hold nothing, and more new tokens than tokens: rows in
    front see nothing, but for an open prefix."""
    for kw in (dict(softcap=4.0), dict(window=9), dict(prefix=[3, 3, 3]),
               dict(prefix=[3, 0, 9], slopes=slopes_of(4))):
        run(9, [0, 5, 100], [2, 9, 1], 4, 2, 128, 32, 16, F16, **kw)


@pytest.mark.parametrize("kw", [dict(window=70), dict(window=70, softcap=5.0), dict(window=600)])
@pytest.mark.parametrize("many", [False, True])
def test_what_a_window_hides_may_hold_anything(kw, many):
    """NaN and infinities before the window and behind the request do not reach
    a row; inside it they do."""
    lengths, new = ([400, 1000], [200, 300]) if many else ([400, 1000], [1, 3])
    store, table = pool(10, lengths, 2, 128, 64, 16, F16, width=1 << 12 if many else None)
    last = table[1, 62].item()
    for r, n in enumerate(lengths):
        # tokens before what the request's first new one sees
        gone = max(0, n - new[r] + 1 - kw["window"])
        for t in range(gone):
            p, i = int(table[r, t // 16]), t % 16
            for x, m in enumerate((store.k_meta, store.v_meta)):
                m[p, :, :, i] = [math.nan, math.inf, -math.inf][(t + x) % 3]
    store.k_meta[last, :, :, 8:], store.v_meta[last, :, :, 8:] = math.nan, math.inf
    q = queries(11, sum(new), 8, 128, F16)
    starts = ints([0, new[0], sum(new)])
    got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **kw)
    assert bool(got.isfinite().all())
    clean = [t.nan_to_num(0.0, 0.0, 0.0) if t.dtype == F16 else t for t in store]
    error = R.check(got, R.attend(q, clean, table, ints(lengths), starts, 0.1, **kw))
    assert not error, error
    at = lengths[1] - 2
    store.v_meta[int(table[1, at // 16]), 1, 0, at % 16] = math.nan
    got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **kw)
    seen = torch.zeros_like(got, dtype=torch.bool)
    seen[-2:, 4:, :64] = True
    assert torch.equal(got.isnan(), seen)


@pytest.mark.parametrize("many", [False, True])
def test_large_values_before_a_window_cost_nothing(many):
    """Finite ones too: the row's values keep their bits."""
    lengths, new = ([400, 1000], [200, 300]) if many else ([400, 1000], [1, 3])
    store, table = pool(29, lengths, 2, 128, 64, 16, BF16, width=1 << 12 if many else None)
    for r, n in enumerate(lengths):
        for t in range(max(0, n - new[r] + 1 - 75)):
            store.v_meta[int(table[r, t // 16]), :, :, t % 16] = 1e37
    q = queries(30, sum(new), 8, 128, BF16)
    starts = ints([0, new[0], sum(new)])
    for kw in (dict(window=75), dict(window=75, softcap=4.0)):
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **kw)
        error = R.check(got, R.attend(q, store, table, ints(lengths), starts, 0.1, **kw))
        assert not error, error


@pytest.mark.parametrize("many", [False, True])
def test_a_steep_bias_keeps_the_scores_of_near_tokens(many):
    """Biases of 10^5 and more beside scores of a few units, with a cap and
    without."""
    lengths, new = ([9000, 800], [150, 90]) if many else ([9000, 800], [1, 5])
    store, table = pool(31, lengths, 2, 128, 64, 64, F16, width=1 << 12 if many else None)
    # nothing is held near the rows: their largest scores are far below 0
    table[0, 130:] = -1
    q = queries(32, sum(new), 8, 128, F16)
    starts, slopes = ints([0, new[0], sum(new)]), torch.full((8,), 0.0, device=DEV)
    slopes[:] = torch.tensor([300.0, 40.0, 7.0, 1.0, 0.3, 0.01, 150.0, 2.0])
    for kw in (dict(slopes=slopes), dict(slopes=slopes, softcap=5.0)):
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **kw)
        want = R.attend(q, store, table, ints(lengths), starts, 0.1, **kw)
        error = R.check(got, want, False)
        assert not error, error


@pytest.mark.parametrize("many", [False, True])
def test_pages_outside_the_pool(many):
    lengths, new = ([300, 500], [100, 90]) if many else ([300, 500], [1, 2])
    store, table = pool(12, lengths, 2, 64, 32, 16, BF16, width=1 << 12 if many else None)
    table[0, 3], table[0, 18], table[1, 30], table[1, 0] = -1, 1 << 30, -(1 << 31), store[0].shape[0]
    q = queries(13, sum(new), 8, 64, BF16)
    starts = ints([0, new[0], sum(new)])
    for kw in (dict(softcap=6.0), dict(window=40), dict(prefix=[90, 90]), dict(slopes=slopes_of(8))):
        call = dict(kw)
        if "prefix" in kw:
            call["prefix_lengths"] = ints(call.pop("prefix"))
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.125, **call)
        error = R.check(got, R.attend(q, store, table, ints(lengths), starts, 0.125, **kw))
        assert not error, error


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("kw", [dict(softcap=1e-3), dict(softcap=3e4), dict(softcap=50.0, scale=40.0),
                                dict(slopes=300.0), dict(slopes=-0.05), dict(softcap=2.0, slopes=1e4),
                                dict(scale=1e4, slopes=1.0), dict(scale=0.0, slopes=0.01),
                                dict(scale=-0.3, softcap=4.0), dict(scale=1e-30, softcap=20.0)])
def test_scores_of_any_size(kw, many):
    """Far scores keep a reference of their row; negative scales and slopes."""
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(8, kw["slopes"])
    lengths, new = ([3000, 800], [150, 90]) if many else ([3000, 800], [1, 5])
    run(14, lengths, new, 8, 2, 128, 64, 64, F16, ordinary=False, **kw)


def test_a_scale_that_is_nan():
    store, table = pool(15, [50], 1, 64, 64, 16, F16)
    q = queries(16, 1, 2, 64, F16)
    got = S.paged_attention(q, store, table, ints([50]), ints([0, 1]), math.nan, softcap=5.0)
    assert bool(got.isnan().all())


def test_rows_of_no_request_are_left_with_out():
    store, table = pool(17, [50, 60], 2, 128, 64, 16, F16)
    q = queries(18, 9, 4, 128, F16)
    for kw in (dict(softcap=5.0), dict(window=20), dict(prefix_lengths=ints([9, 9]))):
        out = torch.full_like(q, 7.0)
        starts = ints([2, 3, 5])
        got = S.paged_attention(q, store, table, ints([50, 60]), starts, 0.1, out=out, **kw)
        assert got is out and bool((out[:2] == 7.0).all()) and bool((out[5:] == 7.0).all())
        fresh = S.paged_attention(q, store, table, ints([50, 60]), starts, 0.1, **kw)
        assert torch.equal(fresh[2:5], out[2:5]) and not bool(fresh[:2].any() | fresh[5:].any())
        # starts that descend name no rows
        bad = S.paged_attention(q, store, table, ints([50, 60]), ints([0, 5, 3]), 0.1, **kw)
        assert not bool(bad.any())


def test_wrong_hints_change_roundings_only():
    lengths, new = [3000, 200, 900], [90, 1, 300]
    store, table = pool(19, lengths, 2, 128, 64, 64, F16)
    q, starts = queries(20, sum(new), 8, 128, F16), ints([0, 90, 91, 391])
    for kw in (dict(softcap=9.0, slopes=slopes_of(8, 0.02)), dict(window=300), dict(prefix=[50, 50, 500])):
        want = R.attend(q, store, table, ints(lengths), starts, 0.1, **kw)
        call = dict(kw)
        if "prefix" in kw:
            call["prefix_lengths"] = ints(call.pop("prefix"))
        for hints in (dict(max_new=1, max_length=1), dict(max_new=1, max_length=10 ** 6), dict(),
                      dict(max_new=300, max_length=3000), dict(max_new=10 ** 6, max_length=5)):
            got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **hints, **call)
            error = R.check(got, want)
            assert not error, (hints, error)


@pytest.mark.parametrize("held", [0, 1, 700])
@pytest.mark.parametrize("new,hkv,d", [(1100, 8, 128), (1090, 8, 64), (2041, 4, 128), (2300, 8, 64)])
def test_one_prompt_whose_columns_fill_the_device_once(new, hkv, d, held):
    """The longer ones are halved, where rows see little beside their own."""
    store, table = pool(37, [held + new], hkv, d, 64, 64, F16)
    q, starts = queries(38, new + 3, 4 * hkv, d, F16), ints([0, new])
    for call, kw in ((dict(softcap=8.0), dict(softcap=8.0)),
                     (dict(prefix_lengths=ints([300])), dict(prefix=[300])),
                     (dict(prefix_lengths=ints([900])), dict(prefix=[900])),
                     (dict(slopes=slopes_of(4 * hkv)), dict(slopes=slopes_of(4 * hkv)))):
        got = S.paged_attention(q, store, table, ints([held + new]), starts, 0.1, **call)
        error = R.check(got, R.attend(q, store, table, ints([held + new]), starts, 0.1, **kw))
        assert not error, (kw, error)
        assert not bool(got[new:].any())


@pytest.mark.parametrize("real", [0, 1, 300, 1100, 1500])
def test_one_prompt_that_fills_its_batch_in_part(real):
    """A step sized for 1500 tokens of which fewer come (a captured one, say)."""
    n, hkv = 1500, 8
    store, table = pool(39, [max(real, 1)], hkv, 128, 64, 64, F16, width=40)
    q = queries(40, n, 4 * hkv, 128, F16)
    for starts in ([0, real], [n - real, n]) if real else ([0, 0], [7, 7], [9, 5]):
        st, le = ints(starts), ints([real])
        got = S.paged_attention(q, store, table, le, st, 0.1, softcap=8.0, max_new=n, max_length=n)
        at = slice(starts[0], starts[0] + real)
        if real:
            want = R.attend(q, store, table, le, st, 0.1, softcap=8.0)
            error = R.check(got[at], [x[at] for x in want])
            assert not error, error
        assert not bool(got[:at.start].any() | got[at.stop:].any())


@pytest.mark.parametrize("new", [0, 1, 5, 40, 300])
@pytest.mark.parametrize("kw", [dict(softcap=9.0), dict(window=100), dict(prefix_lengths=None)])
def test_one_request_with_hints_of_many_rows(kw, new):
    """One request's rows are one kernel's, whichever the hints name; rows in
    front of it and behind it are zeroed there too."""
    store, table = pool(27, [700], 2, 128, 64, 16, F16, width=1 << 13)
    q, starts = queries(28, new + 5, 8, 128, F16), ints([2, 2 + new])
    call = dict(kw)
    if "prefix_lengths" in kw:
        call, kw = dict(prefix_lengths=ints([600])), dict(prefix=[600])
    for hints in (dict(max_new=10 ** 5, max_length=10 ** 6), dict(max_new=1, max_length=700), dict()):
        got = S.paged_attention(q, store, table, ints([700]), starts, 0.1, **hints, **call)
        error = R.check(got, R.attend(q, store, table, ints([700]), starts, 0.1, **kw))
        assert not error, (hints, error)
        assert not bool(got[:2].any() | got[2 + new:].any())
        out = torch.full_like(q, 7.0)
        S.paged_attention(q, store, table, ints([700]), starts, 0.1, out=out, **hints, **call)
        assert torch.equal(out[2:2 + new], got[2:2 + new])
        assert bool((out[:2] == 7.0).all()) and bool((out[2 + new:] == 7.0).all())


def test_strided_and_unaligned_queries():
    lengths, new = [300, 40], [3, 2]
    store, table = pool(21, lengths, 2, 64, 32, 16, F16)
    wide = queries(22, 5, 9, 65, F16)
    q = wide[:, 1:, 1:]
    starts = ints([0, 3, 5])
    for kw in (dict(softcap=9.0), dict(window=30)):
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.125, **kw)
        error = R.check(got, R.attend(q, store, table, ints(lengths), starts, 0.125, **kw))
        assert not error, error


def test_many_uneven_requests():
    rng = random.Random(3)
    lengths = [rng.randint(0, 900) for _ in range(300)]
    new = [min(n, rng.choice([0, 1, 1, 2, 5])) for n in lengths]
    run(23, lengths, new, 8, 2, 64, 64, 16, BF16, softcap=6.0, window=333)
    run(24, lengths, new, 4, 2, 128, 64, 32, F16, prefix=[rng.randint(-5, 950) for _ in lengths])


def test_a_cache_attends_with_options():
    cache = S.PagedKVCache(n_requests=2, n_kv_heads=2, head_dim=64, max_tokens=300, page_size=16, device=DEV)
    for step, new in enumerate(([130, 60], [1, 1], [3, 2])):
        n = sum(new)
        cache.step(new)
        cache.append(queries(step, n, 2, 64, F16), queries(step + 10, n, 2, 64, F16))
        q = queries(step + 20, n, 8, 64, F16)
        for kw in (dict(softcap=3.0, slopes=slopes_of(8)), dict(window=50),
                   dict(prefix=[20, 40])):
            call = dict(kw)
            if "prefix" in kw:
                call["prefix_lengths"] = ints(call.pop("prefix"))
            got = cache.attend(q, 0.125, **call)
            want = R.attend(q, cache.store, cache.block_table, cache.lengths, cache.plan.token_starts, 0.125, **kw)
            error = R.check(got, want)
            assert not error, error


def test_graphs_and_streams():
    """Two calls captured in one graph, replayed with eager calls between, on
    another stream too."""
    lengths, new = [3000, 900], [1, 2]
    store, table = pool(25, lengths, 2, 128, 64, 64, F16)
    q, starts, le = queries(26, 3, 8, 128, F16), ints([0, 1, 3]), ints(lengths)
    sl = slopes_of(8, 0.1)

    def calls():
        return (S.paged_attention(q, store, table, le, starts, 0.1, softcap=20.0, slopes=sl),
                S.paged_attention(q, store, table, le, starts, 0.1, window=700))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for i in range(4):
        q.copy_(queries(30 + i, 3, 8, 128, F16))
        le.copy_(ints([3000 - 100 * i, 900 - 7 * i]))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = calls()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
