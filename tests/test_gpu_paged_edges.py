"""The paged 4-bit cache's operators at the ends of what their calls allow:
starts, lengths, magnitudes and counts that the ordinary cases do not reach,
against the 64-bit restatement (tests/paged_reference.py)."""

import math

import paged_reference as R
import pytest
import torch
from test_gpu_paged import DEV, HALF, check_attention, fresh, ints, rows, wide, world  # noqa: F401

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

pytestmark = pytest.mark.gpu


def poisoned(shape, dtype):
    """Leaves NaN in memory that the next tensor of this size will get."""
    torch.full(shape, math.nan, dtype=dtype, device=DEV)


@pytest.mark.parametrize("new", [(3, 1, 2), (3, 70, 30)])
def test_rows_before_the_first_request_are_zero(new):
    """Some of a plan's requests over all of its packed queries: starts that
    begin above 0."""
    store, table, le, starts = world(31, [40, 120, 35], new, 2, 64, 32, 16, torch.float16)
    n = sum(new) + 2
    q = rows(32, n, 4, 64, torch.float16, False)
    for some in (slice(1, 3), slice(1, 2), slice(2, 3)):
        part = (table[some].contiguous(), le[some].contiguous(), starts[some.start:some.stop + 1].contiguous())
        poisoned(q.shape, q.dtype)
        out = S.paged_attention(q, store, *part, 0.125)
        check_attention(out, q, store, *part, 0.125)
        assert (out[:sum(new[:some.start])] == 0).all() and (out[sum(new[:some.stop]):] == 0).all()
        given = torch.full_like(q, 7.0)
        S.paged_attention(q, store, *part, 0.125, out=given)
        at = slice(sum(new[:some.start]), sum(new[:some.stop]))
        assert torch.equal(given[at], out[at])
        assert (given[:at.start] == 7).all() and (given[at.stop:] == 7).all()
    # starts past the queries: no request has a row, so all are zero
    poisoned(q.shape, q.dtype)
    assert (S.paged_attention(q, store, table, le, starts + 10 ** 6, 0.125) == 0).all()


def beside_a_large_value(dtype, factor, new, d=64, group=32, n=300):
    """(call arguments, the output in 64 bits, the scale of its values'
    groups) of rows that rest on one ordinary token, 2^-40 of them on each of
    the others, one of which, in another tile, holds `factor` times the
    ordinary values."""
    g = [rows(40 + i, n, 1, d, torch.float32, False) for i in range(2)]
    k = torch.zeros((n, 1, d), device=DEV)
    k[150, 0, 0] = 1.0
    v = g[0].to(dtype)
    v[9] = (g[1][9] * factor).to(dtype)
    store = fresh(dtype, 19, 1, d, group, 16)
    S.append_paged(store, k.to(dtype), v, torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(19, dtype=torch.int32, device=DEV)[None]
    q = torch.zeros((new, 4, d), dtype=dtype, device=DEV)
    q[..., 0] = 8.0
    args = (q, store, table, ints([n]), ints([0, new]), 5 * math.log(2))
    scale = R.unpack(store)[3][150, 0, :, 0].double().repeat_interleave(group)
    return args, R.attend(*args)[0], scale


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("factor", [64.0, 256.0, 1000.0])
def test_ordinary_values_keep_their_bits_beside_a_large_one(factor, dtype):
    """p scale is rounded to fp16 (2^-11) and meets code - 7.5; 299 tokens of
    2^-40, one of them `factor` times as large as 4, are below 2^-28."""
    args, want, scale = beside_a_large_value(dtype, factor, 2)
    err = (S.paged_attention(*args).cpu().double() - want).abs()
    assert (err <= (R.U16[dtype] + 2.0 ** -20) * want.abs() + 2.0 ** -11 * 7.5 * scale + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("factor", [64.0, 256.0, 1000.0])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (128, 128), (128, 32), (64, 64)])
def test_large_attention_and_ordinary_values_beside_a_large_one(wide, d, group, factor, dtype):
    """The probability and the value are rounded to fp16, 2^-11 of each and
    their product 2^-22 more."""
    args, want, _ = beside_a_large_value(dtype, factor, 80, d, group)
    err = (S.paged_attention(*args).cpu().double() - want).abs()
    assert (err <= (R.U16[dtype] + 2.001 * 2.0 ** -11) * want.abs() + 2.0 ** -24).all(), \
        f"{float((err / want.abs().clamp(min=1e-3)).max()):.1e}"


def check_some_rows(out, q, store, table, lengths, starts, scale, some, bound=2.0 ** -9):
    """Rows (request, new token, KV head) against the 64-bit form: relative
    L2 error of each query head.  fp16: 2^-11 each of the output, the
    probabilities and the values is below 2^-9."""
    rep = q.shape[1] // store.n_kv_heads
    at, le = starts.tolist(), lengths.tolist()
    for r, i, h in some:
        row, n, heads = at[r] + i, at[r + 1] - at[r], slice(h * rep, (h + 1) * rep)
        one = S.PagedKVStore(*(t[:, h:h + 1] for t in store))
        want, _ = R.attend(q[row:row + 1, heads], one, table[r:r + 1], ints([le[r] - n + i + 1]), ints([0, 1]), scale)
        err = (out[row:row + 1, heads].cpu().double() - want).norm(dim=-1)
        assert (err <= bound * want.norm(dim=-1)).all(), (r, i, h, float((err / want.norm(dim=-1)).max()))


@pytest.mark.parametrize("n,hq,hkv,d,max_new", [(33001, 8, 2, 128, None), (32768, 64, 64, 64, 1)])
def test_long_prompts_in_tables_of_many_pages(n, hq, hkv, d, max_new):
    """Prompts in tables of 2^20 tokens a row, with and without the hint that
    there are many rows."""
    page = 128
    store, table, le, starts = world(51, [n], [n], hkv, d, 64, page, torch.float16)
    table = torch.nn.functional.pad(table, (0, 2 ** 20 // page - table.shape[1]), value=-1)
    q = rows(52, n, hq, d, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, d ** -0.5, max_new=max_new)
    some = [(0, i, h) for i in (0, 5, 130, n // 2, n - 1) for h in (0, hkv - 1)]
    check_some_rows(out, q, store, table, le, starts, d ** -0.5, some)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_list_step_in_a_capture_is_refused():
    """The capture ends, cache and device go on."""
    c = S.PagedKVCache(n_requests=2, n_kv_heads=1, head_dim=64, max_tokens=64)
    c.step([5, 9])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            c.step([1, 1])
    assert c._host == [5, 9]
    c.step([1, 2])
    assert c.lengths.tolist() == [6, 11] == c._host


@pytest.mark.parametrize("new", [1, 128])
def test_a_request_of_2_to_the_30_tokens(new):
    """The longest table row, whose every page is the same: the page's own
    attention, but for sums of up to 2^17 float32 numbers, 2^-7 of their size
    each (values around 3, so that the sums are of one sign).  Memory that no
    part writes is NaN."""
    d, page, width = 64, 1024, 2 ** 20
    store = fresh(torch.float16, 1, 1, d, 64, page)
    k, v = rows(61, page, 1, d, torch.float16, False), 3 + 0.25 * rows(62, page, 1, d, torch.float16, False)
    S.append_paged(store, k, v, torch.arange(page, dtype=torch.int32, device=DEV))
    q = rows(63, new, 1, d, torch.float16, False)
    table = torch.zeros((1, width), dtype=torch.int32, device=DEV)
    want, _ = R.attend(q, store, table, ints([page]), ints([0, new]), 0.125, causal=False)
    need = paged._workspace_bytes(0, (1, 1, d, 64, page, _hip.SS_F16), new, 1, 1, new, page * width)
    assert need > 0
    poisoned((need // 2,), torch.float16)
    out = S.paged_attention(q, store, table, ints([page * width]), ints([0, new]), 0.125)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -6 * want.abs()).all()


def small_against_large(q_size, k_size, new):
    """Call arguments, without the scale, of bfloat16 queries and keys of
    these sizes."""
    n, d = 200, 64
    store = fresh(torch.bfloat16, 13, 1, d, 32, 16)
    k = (rows(71, n, 1, d, torch.float32, False).clamp(-4, 4) * k_size).to(torch.bfloat16)
    v = rows(72, n, 1, d, torch.bfloat16, False)
    S.append_paged(store, k, v, torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(13, dtype=torch.int32, device=DEV)[None]
    q = (rows(73, new, 4, d, torch.float32, False) * q_size).to(torch.bfloat16)
    return q, store, table, ints([n]), ints([0, new])


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("q_size,k_size", [(1e-30, 1e30), (1e-33, 1e31), (1e-36, 1e31), (1e30, 1e-30),
                                           (1e36, 1e-36)])
def test_small_queries_against_large_keys(q_size, k_size, new):
    args = (*small_against_large(q_size, k_size, new), 0.125)
    check_attention(S.paged_attention(*args), *args)


@pytest.mark.parametrize("q_size,k_size", [(1e-30, 1e30), (1e-33, 1e31)])
def test_large_attention_of_small_queries(wide, q_size, k_size):
    test_small_queries_against_large_keys(q_size, k_size, 80)


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, -1e-40])
def test_a_scale_of_nothing_gives_the_mean(scale, new):
    """... of the tokens that a row sees, whatever the keys."""
    for sizes in ((1.0, 1.0), (1.0, 1e30)):
        args = (*small_against_large(*sizes, new), scale if sizes[1] == 1.0 else 0.0)
        check_attention(S.paged_attention(*args), *args)


@pytest.mark.parametrize("new", [1, 80])
def test_a_scale_that_is_no_number_gives_none(new):
    args = small_against_large(1.0, 1.0, new)
    assert S.paged_attention(*args, math.nan).isnan().all()


def test_large_attention_with_scales_of_nothing(wide):
    test_a_scale_of_nothing_gives_the_mean(0.0, 80)
    test_a_scale_that_is_no_number_gives_none(80)


def far_scores(dtype, size, new, d=128, n=400):
    """Call arguments of scores that differ by `size` log2 units from token to
    token, all of them exact (keys 0 .. 14 in one dim, scale 1), and the 64-bit
    output: each row's largest tokens alone."""
    store = fresh(dtype, 25, 1, d, 64, 16)
    k = torch.zeros((n, 1, d), device=DEV)
    k[:, 0, 0] = torch.arange(n, device=DEV) * 7 % 15
    k[:, 0, 1] = 15.0  # (the group's scale)
    v = rows(81, n, 1, d, dtype, False)
    S.append_paged(store, k.to(dtype), v, torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(25, dtype=torch.int32, device=DEV)[None]
    q = torch.zeros((new, 4, d), dtype=dtype, device=DEV)
    q[..., 0] = torch.tensor([1.0, -1.0, 3.0, -0.5], device=DEV)
    args = (q, store, table, ints([n]), ints([0, new]), size * math.log(2))
    return args, R.attend(*args)[0]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("size", [300.0, 2.0 ** 13, 2.0 ** 22, 2.0 ** 27, 2.0 ** 40, 2.0 ** 90])
def test_scores_of_any_size(size, new, dtype):
    """The largest scores' tokens are averaged: p is 1 or 0, so only the
    values' roundings are left, 2^-11 of p scale times 7.5 codes here, 2^-11 of
    p and of the value in the kernel for large calls."""
    args, want = far_scores(dtype, size, new)
    out = S.paged_attention(*args)
    store = args[1]
    terms = want.abs() + 7.5 * R.unpack(store)[3][:400, 0, :, 0].double().amax(0).repeat_interleave(64)
    err = (out.cpu().double() - want).abs()
    assert (err <= R.U16[dtype] * want.abs() + 2.001 * 2.0 ** -11 * terms + 2.0 ** -16).all(), float(err.max())


@pytest.mark.parametrize("dtype", HALF)
def test_large_attention_with_scores_of_any_size(wide, dtype):
    for size in (300.0, 2.0 ** 13, 2.0 ** 22, 2.0 ** 27, 2.0 ** 40, 2.0 ** 90):
        test_scores_of_any_size(size, 80, dtype)


@pytest.mark.parametrize("new", [1, 80])
def test_far_scores_of_small_queries_against_large_keys(new):
    args = (*small_against_large(1e-20, 1e31, new), 0.125)
    check_attention(S.paged_attention(*args), *args)


SIZES = {"constant": lambda v: torch.ones_like(v) * 1e20, "largest": lambda v: torch.full_like(v, 3.3e38),
         "smallest": lambda v: v * 1e-30, "wide": lambda v: v * 1e37, "raised": lambda v: 1e25 + v * 1e20,
         "one": lambda v: torch.where(torch.arange(v.shape[0], device=DEV)[:, None, None] == 77, v * 3e37, v)}


@pytest.mark.parametrize("new", [1, 3, 80])
@pytest.mark.parametrize("size", SIZES)
def test_values_of_any_size(size, new, lengths=(300, 2500)):
    """bfloat16 values of one size or of all: groups whose scale is 0 or small
    beside their zero, the largest and the smallest numbers, one token that is
    far larger than the others.  Keys of 0: every token counts the same."""
    d, group, page = 64, 32, 16
    for n in lengths:
        store = fresh(torch.bfloat16, -(-n // page), 1, d, group, page)
        v = SIZES[size](rows(91, n, 1, d, torch.float32, False).clamp(-3, 3)).to(torch.bfloat16)
        S.append_paged(store, torch.zeros_like(v), v, torch.arange(n, dtype=torch.int32, device=DEV))
        table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None]
        q = rows(92, new, 4, d, torch.bfloat16, False)
        args = (q, store, table, ints([n]), ints([0, new]), 0.125)
        check_attention(S.paged_attention(*args), *args)


@pytest.mark.parametrize("size", SIZES)
def test_large_attention_with_values_of_any_size(wide, size):
    test_values_of_any_size(size, 80, (300,))


@pytest.mark.parametrize("n_new", [1, 5000])
def test_pages_of_no_pool_give_no_slots(n_new):
    """Page numbers whose slots pass 32 bits do not come back as slots of other
    pages; for few new tokens and, by the second launch, for many."""
    page, big = 64, 2 ** 26
    width = 1 + -(-n_new // page)
    for number in (big + 3, -big, -1, -big + 3, 2 ** 31 - 1, big // 2 - 1, 7):
        table = ints([[number] + [-1] * (width - 1), list(range(width))])
        free = torch.arange(100, 100 + 2 * width, dtype=torch.int32, device=DEV)
        plan = S.build_block_tables(ints([5, 5]), ints([n_new, 1]), table, free, ints([2 * width]), page, n_new + 1)
        S.check_plan(plan)
        slots, first = plan.slots.tolist(), min(n_new, page - 5)
        real = number >= 0 and (number + 1) * page <= 2 ** 31
        assert slots[:first] == [number * page + 5 + i if real else -1 for i in range(first)], number
        assert slots[-1] == 5 and all(s >= 0 for s in slots[first:])
        assert plan.positions.tolist() == list(range(5, 5 + n_new)) + [5]


@pytest.mark.parametrize("max_new", [1, 64])
def test_starts_that_descend_name_no_rows(max_new):
    """Requests that overlap; as many as pass 32 bits of blocks among them."""
    store, table, le, _ = world(101, [64, 64, 64], [1, 1, 1], 2, 64, 64, 16, torch.float16)
    q = rows(102, 40, 8, 64, torch.float16, False)
    for starts in ([0, 30, 10, 40], [40, 30, 20, 0], [0, 0, 40, 39], [0, 40, -2 ** 31, 40], [5, -2 ** 31, 40, 40]):
        poisoned(q.shape, q.dtype)
        assert (S.paged_attention(q, store, table, le, ints(starts), 0.125, max_new=max_new) == 0).all(), starts
        given = torch.full_like(q, 7.0)
        S.paged_attention(q, store, table, le, ints(starts), 0.125, max_new=max_new, out=given)
        assert (given == 7).all()
    many, page = 4000, 1024
    big = fresh(torch.float16, 1, 2, 64, 64, page)
    table = torch.zeros((many, 2 ** 20 // page), dtype=torch.int32, device=DEV)
    out = S.paged_attention(q, big, table, ints([2 ** 20] * many), ints([0, 40] * (many // 2) + [40]), 0.125,
                            max_new=max_new)
    assert (out == 0).all()


def test_large_attention_of_starts_that_descend(wide):
    test_starts_that_descend_name_no_rows(64)


def test_attention_captured_without_its_step():
    """append and attend of an eager step in a graph: replays give the same
    after other steps have come and their plans gone."""
    hq, hkv, d = 8, 2, 64
    c = S.PagedKVCache(n_requests=2, n_kv_heads=hkv, head_dim=d, max_tokens=900, page_size=16)
    c.step([300, 500])
    c.append(rows(111, 800, hkv, d, torch.float16), rows(112, 800, hkv, d, torch.float16, False))
    c.step([1, 3])
    k, v, q = (rows(113 + i, 4, h, d, torch.float16) for i, h in enumerate((hkv, hkv, hq)))
    c.append(k, v)
    want = c.attend(q, 0.125)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.append(k, v)
        out = c.attend(q, 0.125)
    for _ in range(4):
        c.step([2, 1])  # other plans, and back again
        c.step([-2, -1])
        junk = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in (13, 15, 17, 19)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del junk
