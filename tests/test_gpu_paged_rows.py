"""The paged attention's rows within the L2 bound of their roundings: the
ordinary cases, and the launch shapes of the kernel for large calls: whole
prompts whose columns are not cut, more columns than parts are cut for, more
requests than a wave has lanes."""

import random

import paged_reference as R
import pytest
import torch
from test_gpu_paged import CASES, DEV, HALF, ints, rows, wide, world  # noqa: F401

import sunshape_mlx_amd as S

pytestmark = pytest.mark.gpu
SHAPES = [(128, 64), (64, 32), (128, 32), (128, 128), (64, 64)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("lengths,new,hq,hkv,page", CASES)
def test_rows(lengths, new, hq, hkv, page, d, group, dtype):
    store, table, le, starts = world(len(lengths) + d, lengths, new, hkv, d, group, page, dtype)
    q = rows(9, sum(new), hq, d, dtype, False)
    want, bound = R.attend_l2(q, store, table, le, starts, d ** -0.5)
    for hints in ({}, dict(max_new=max(1, max(new)), max_length=max(lengths))):
        assert R.within_l2(S.paged_attention(q, store, table, le, starts, d ** -0.5, **hints), want, bound)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("lengths,new,hq,hkv,page",
                         [c for c in CASES if max(c[1]) * c[2] // c[3] > 64] + [([500, 65], [400, 65], 4, 4, 16)])
def test_rows_of_large_calls(wide, lengths, new, hq, hkv, page, d, group, dtype):  # noqa: F811
    test_rows(lengths, new, hq, hkv, page, d, group, dtype)


@pytest.mark.parametrize("dtype", HALF)
def test_rows_of_long_decodes(dtype):
    test_rows([12345, 1000, 3], [1, 2, 1], 8, 2, 16, 128, 64, dtype)


def check_some(out, q, store, table, lengths, starts, scale, some):
    """Rows (request, new token, KV head)."""
    rep = q.shape[1] // store.n_kv_heads
    at, le = starts.tolist(), lengths.tolist()
    for r, i, h in some:
        row, heads = at[r] + i, slice(h * rep, (h + 1) * rep)
        one = S.PagedKVStore(*(t[:, h:h + 1] for t in store))
        seen = le[r] - (at[r + 1] - at[r]) + i + 1
        want, bound = R.attend_l2(q[row:row + 1, heads], one, table[r:r + 1], ints([seen]), ints([0, 1]), scale)
        err = (out[row:row + 1, heads].cpu().double() - want).norm(dim=-1)
        assert (err <= bound).all(), (r, i, h, float((err / bound).max()))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group,n,hq,hkv", [(128, 64, 4093, 32, 8), (64, 32, 2041, 32, 16), (128, 128, 1501, 16, 16),
                                              (64, 64, 4093, 32, 8), (128, 32, 1999, 28, 14)])
def test_whole_prompts(d, group, n, hq, hkv, dtype):
    """More columns than compute units: none is cut, a workgroup takes up to
    64 tiles."""
    store, table, le, starts = world(7, [n], [n], hkv, d, group, 64, dtype)
    q = rows(8, n, hq, d, dtype, False)
    out = S.paged_attention(q, store, table, le, starts, d ** -0.5)
    some = [(0, i, h) for i in (0, 1, 63, 64, 130, 1000, n - 1) for h in (0, hkv // 2, hkv - 1)]
    check_some(out, q, store, table, le, starts, d ** -0.5, some)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", HALF)
def test_more_columns_than_are_cut(dtype):
    """40 requests of 80 rows a KV head: the sizes leave room for parts, the
    tables name too many columns for them."""
    new = [20] * 40
    lengths = [20 + 17 * i for i in range(40)]
    store, table, le, starts = world(9, lengths, new, 8, 128, 64, 32, dtype)
    q = rows(10, sum(new), 32, 128, dtype, False)
    out = S.paged_attention(q, store, table, le, starts, 128 ** -0.5)
    some = [(r, i, h) for r in (0, 1, 20, 39) for i in (0, 19) for h in (0, 7)]
    check_some(out, q, store, table, le, starts, 128 ** -0.5, some)


@pytest.mark.parametrize("b", [65, 200])
def test_large_calls_of_more_requests_than_a_wave_has_lanes(b):
    """Prompts, chunks and decode steps of many requests, some of which add
    nothing."""
    rng = random.Random(b)
    lengths = [rng.randint(1, 900) for _ in range(b)]
    new = [min(n, rng.choice([0, 1, 1, 4, 20, 33, 150])) for n in lengths]
    store, table, le, starts = world(11, lengths, new, 4, 64, 32, 16, torch.float16)
    q = rows(12, sum(new), 16, 64, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125)
    some = [(r, i, r % 4) for r in range(0, b, 3) if new[r] for i in (0, new[r] - 1)]
    check_some(out, q, store, table, le, starts, 0.125, some)
    given = torch.full((sum(new) + 3, 16, 64), 7.0, dtype=torch.float16, device=DEV)
    S.paged_attention(torch.nn.functional.pad(q, (0, 0, 0, 0, 0, 3)), store, table, le, starts, 0.125, out=given,
                      max_new=150, max_length=900)
    check_some(given, q, store, table, le, starts, 0.125, some)
    assert (given[sum(new):] == 7).all()


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("dtype,other", [HALF, HALF[::-1]])
@pytest.mark.parametrize("d,group", [(128, 64), (64, 32)])
def test_queries_of_the_other_type(request, d, group, dtype, other, large):
    """Queries and stores need not share a type; the output has the queries'."""
    if large:
        request.getfixturevalue("wide")
    store, table, le, starts = world(15, [150, 33, 90], [70, 1, 3], 2, d, group, 16, dtype)
    q = rows(16, 74, 8, d, other, False)
    out = S.paged_attention(q, store, table, le, starts, d ** -0.5)
    assert out.dtype is other and R.within_l2(out, *R.attend_l2(q, store, table, le, starts, d ** -0.5))


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("page", [256, 512, 1024])
def test_large_pages(request, page, large):
    if large:
        request.getfixturevalue("wide")
    store, table, le, starts = world(17, [1500, 1025, 1024, 3], [90, 1, 4, 3], 2, 64, 64, page, torch.float16)
    q = rows(18, 98, 4, 64, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125)
    assert R.within_l2(out, *R.attend_l2(q, store, table, le, starts, 0.125))


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("hq", [96, 128, 1024])
def test_many_query_heads_to_one(request, hq, large):
    """More rows of one token than a block, or a tile, has."""
    if large:
        request.getfixturevalue("wide")
    store, table, le, starts = world(19, [300, 77], [1, 3], 1, 64, 32, 16, torch.bfloat16)
    q = rows(20, 4, hq, 64, torch.bfloat16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125)
    assert R.within_l2(out, *R.attend_l2(q, store, table, le, starts, 0.125))


@pytest.mark.parametrize("large", [False, True])
def test_more_new_tokens_than_a_request_holds(request, large):
    """Rows before the request's first token see nothing and are zero."""
    if large:
        request.getfixturevalue("wide")
    store, table, le, starts = world(21, [3, 40, 1], [70, 2, 100], 2, 64, 64, 16, torch.float16)
    q = rows(22, 172, 4, 64, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125)
    assert R.within_l2(out, *R.attend_l2(q, store, table, le, starts, 0.125))
    assert (out[:67] == 0).all() and (out[72:171] == 0).all() and (out[67:72] != 0).any(-1).all()


def test_thousands_of_requests():
    """Dozens of requests a lane, most of them without new tokens."""
    rng = random.Random(3)
    lengths = [rng.choice([0, 1, 5, 30]) for _ in range(5000)]
    new = [min(n, rng.choice([0, 0, 0, 1])) for n in lengths]
    store, table, le, starts = world(23, lengths, new, 2, 64, 64, 16, torch.float16)
    q = rows(24, sum(new), 4, 64, torch.float16, False)
    want, bound = R.attend_l2(q, store, table, le, starts, 0.125)
    for hints in ({}, dict(max_new=1, max_length=30)):
        assert R.within_l2(S.paged_attention(q, store, table, le, starts, 0.125, **hints), want, bound)


def test_requests_that_share_pages():
    """Two requests over the same first pages, as after a fork of a prompt."""
    store, table, le, starts = world(25, [64, 90], [1, 1], 2, 64, 64, 16, torch.float16)
    table[0, :3], le = table[1, :3], ints([48, 90])
    q = rows(26, 2, 4, 64, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125)
    assert R.within_l2(out, *R.attend_l2(q, store, table, le, starts, 0.125))
