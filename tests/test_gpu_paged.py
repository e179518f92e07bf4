"""GPU parity of the paged 4-bit cache's operators with their 64-bit
restatement (tests/paged_reference.py): page bookkeeping and codes exactly,
attention within the derived bound of its roundings."""

import math
import random

import numpy as np
import paged_reference as R
import pytest
import torch

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPES = [(128, 64), (128, 128), (128, 32), (64, 64), (64, 32)]
HALF = [torch.float16, torch.bfloat16]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(seed, n, h, d, dtype, spread=True):
    g = gen(seed)
    s = 0.5 + 3.5 * torch.rand((d,), generator=g, device=DEV) if spread else 1.0
    return (torch.randn((n, h, d), generator=g, device=DEV) * s).to(dtype)


# ------------------------------------------------------------ block tables


def tables(lengths, new, page, width, n_pages, n_tokens, seed=0, in_place=False):
    """(plan, table, free pages, the reference's bookkeeping after the step)."""
    rng = random.Random(seed)
    order = list(range(n_pages))
    rng.shuffle(order)
    ref = R.Pages(page, width, [])
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)
    for r, n in enumerate(lengths):
        ref.add()
        ref.lengths[r] = n
        for j in range(-(-n // page)):
            ref.rows[r].append(order.pop())
            table[r, j] = ref.rows[r][-1]
    ref.free = list(order)
    free = torch.full((n_pages,), -9, dtype=torch.int32)
    free[:len(order)] = torch.tensor(order, dtype=torch.int32)
    t, f, n_free, le = table.to(DEV), free.to(DEV), ints([len(order)]), ints(lengths)
    kw = dict(lengths_out=le, n_free_out=n_free) if in_place else {}
    plan = S.build_block_tables(le, ints(new), t, f, n_free, page, n_tokens, **kw)
    if in_place:
        assert plan.lengths is le and plan.n_free is n_free
    return plan, t, f, ref, table


def check_tables(plan, t, f, ref, before, new, n_tokens):
    assert int(plan.status) == 0
    S.check_plan(plan)
    slots, positions = ref.step(new)
    total = len(slots)
    got = plan.slots.cpu().numpy()
    assert np.array_equal(got[:total], slots) and (got[total:] == -1).all()
    got = plan.positions.cpu().numpy()
    assert np.array_equal(got[:total], positions) and (got[total:] == -1).all()
    assert plan.lengths.cpu().tolist() == ref.lengths
    starts = np.concatenate([[0], np.cumsum([max(0, x) for x in new])])
    assert np.array_equal(plan.token_starts.cpu().numpy(), starts)
    assert int(plan.n_free) == len(ref.free)
    assert f.cpu().tolist()[:len(ref.free)] == ref.free
    want = before.clone()
    for r, row in enumerate(ref.rows):
        for j, x in enumerate(row):
            want[r, j] = x
    assert torch.equal(t.cpu(), want)  # (entries past a row's pages as they were)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,new,page,extra", [
    ([0], [1], 16, 0), ([0], [0], 64, 2), ([16], [1], 16, 0), ([15], [1], 16, 3),
    ([509], [-509], 64, 0), ([33, 0, 64], [-20, 100, 0], 32, 5),
    ([1, 2, 3, 4], [4, 3, -3, -1], 128, 1),
])
def test_block_tables_small(lengths, new, page, extra, in_place):
    n = sum(max(0, x) for x in new) + extra
    plan, t, f, ref, before = tables(lengths, new, page, 16, 64, n, in_place=in_place)
    check_tables(plan, t, f, ref, before, new, n)


@pytest.mark.parametrize("b,most,add,page", [(257, 700, 1, 16), (1025, 90, 2, 16), (4096, 40, 1, 16),
                                             (61, 0, 411, 64), (7, 5000, 2300, 32)])
def test_block_tables_of_many_requests(b, most, add, page):
    """Requests that enter, go on, shrink and end; more tokens than the table
    kernel itself fills among them."""
    rng = random.Random(b)
    lengths = [rng.randint(0, most) for _ in range(b)]
    new = [rng.choice([-n, -(n // 2), 0, add, add, rng.randint(0, add)]) for n in lengths]
    n = sum(max(0, x) for x in new) + 11
    need = sum(-(-(x + max(0, y)) // page) for x, y in zip(lengths, new))
    plan, t, f, ref, before = tables(lengths, new, page, -(-(most + add) // page), need + 3, n, seed=b)
    check_tables(plan, t, f, ref, before, new, n)


@pytest.mark.parametrize("b,page", [(64, 16), (4096, 32)])
def test_block_tables_of_which_few_requests_move(b, page):
    """The pages given back and taken lie far apart, in runs from one page to
    many times what the lanes of a wave hold."""
    lengths, new = [5] * b, [0] * b
    lengths[0], new[0] = 700 * page + 1, -(700 * page)
    lengths[1], new[1] = 2 * page, -page
    lengths[b // 2], new[b // 2] = 3, 130 * page
    lengths[b - 2], new[b - 2] = page, 1
    lengths[b - 1], new[b - 1] = 300 * page - 7, -(300 * page - 7)
    n = 130 * page + 1
    plan, t, f, ref, before = tables(lengths, new, page, 701, 1200 + 5 * b, n, seed=page)
    check_tables(plan, t, f, ref, before, new, n)


@pytest.mark.parametrize("lengths,new,pages,n,bits", [
    ([5], [-6], 4, 9, 1), ([-1], [0], 4, 9, 1), ([100], [200], 4, 300, 2), ([16, 16], [40, 40], 6, 99, 4),
    ([16, 0], [3, 5], 4, 7, 8), ([2000000000], [2000000000], 4, 9, 2 + 8),
    # (one that gives pages back first makes room for the other: no failure)
    ([64, 0], [-64, 64], 4, 64, 0)])
def test_block_tables_that_cannot_be_done_change_nothing(lengths, new, pages, n, bits):
    page, width = 16, 8
    table = torch.full((len(lengths), width), -7, dtype=torch.int32, device=DEV)
    used = 0
    for r, x in enumerate(lengths):
        for j in range(min(width, max(0, -(-x // page)))):
            table[r, j], used = used, used + 1
    free = torch.arange(pages, dtype=torch.int32, device=DEV)
    n_free = ints([max(0, pages - used)])
    t0, f0 = table.clone(), free.clone()
    plan = S.build_block_tables(ints(lengths), ints(new), table, free, n_free, page, n)
    assert int(plan.status) & ~4 == bits & ~4 and (int(plan.status) != 0) == (bits != 0)
    if not bits:
        return
    with pytest.raises(RuntimeError):
        S.check_plan(plan)
    assert torch.equal(table, t0) and torch.equal(free, f0)
    assert plan.lengths.cpu().tolist() == lengths and int(plan.n_free) == int(n_free)
    assert (plan.slots == -1).all() and (plan.positions == -1).all()
    assert (plan.token_starts == 0).all()


def test_a_stack_count_out_of_range_is_reported():
    for count in (-1, 5):
        plan = S.build_block_tables(ints([1]), ints([0]), ints([[0]]), ints([0, 1, 2, 3]),
                                    ints([count]), 16, 1)
        assert int(plan.status) == 16 and int(plan.n_free) == count


# ------------------------------------------------------------------ append


def check_slots(store, k, v, slots, group):
    """The slots hold exactly the reference's codes, scales and zeros."""
    got = R.unpack(store)
    at = slots.cpu().long()
    real = (at >= 0) & (at < store.k_codes.shape[0] * store.page_size)
    for x, codes, meta in ((k, got[0], got[2]), (v, got[1], got[3])):
        code, scale, zero = R.quantize(x.to(store.dtype).cpu()[real], group)
        assert torch.equal(codes[at[real]], code)
        for mine, want in ((meta[at[real]][..., 0], scale), (meta[at[real]][..., 1], zero)):
            assert torch.equal(mine.isnan(), want.isnan())
            assert torch.equal(mine.nan_to_num(0.0), want.nan_to_num(0.0))


def fresh(dtype, n_pages, h, d, group, page, seed=None):
    """A store of zeros, or one whose every bit is random."""
    store = S.PagedKVStore.zeros(n_pages, h, d, page_size=page, group_size=group, dtype=dtype, device=DEV)
    if seed is not None:
        for t in store:
            t.view(torch.int32).random_(-2 ** 31, 2 ** 31 - 1, generator=gen(seed))
    return store


@pytest.mark.parametrize("in_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group", SHAPES)
def test_append_stores_the_nearest_codes(d, group, dtype, in_dtype):
    h, page, n = 3, 16, 77
    store = fresh(dtype, 9, h, d, group, page, seed=5)
    before = [t.clone() for t in R.unpack(store)]
    k, v = rows(1, n, h, d, in_dtype), rows(2, n, h, d, in_dtype)
    # runs of slots (aligned, not aligned), single ones, left-out ones
    free = torch.randperm(9 * page, generator=torch.Generator().manual_seed(3))
    slots = torch.cat((torch.arange(16, 48), torch.arange(53, 66), torch.tensor([-1, 144, 2 ** 31 - 1]),
                       free[~((free >= 16) & (free < 66))][:29])).to(torch.int32).to(DEV)
    assert slots.numel() == n
    S.append_paged(store, k, v, slots)
    check_slots(store, k, v, slots, group)
    # everything else as it was
    rest = torch.ones(9 * page, dtype=torch.bool)
    rest[slots.cpu()[(slots.cpu() >= 0) & (slots.cpu() < 144)].long()] = False
    for a, b in zip(R.unpack(store), before):
        a, b = (x.view(torch.int16) if x.is_floating_point() else x for x in (a, b))
        assert torch.equal(a[rest], b[rest])
    # and read back as held, one rounding to the store's type
    rk, rv = S.read_paged(store, slots)
    real = (slots >= 0) & (slots < 144)
    for x, got in ((k, rk), (v, rv)):
        want = R.held(x.to(dtype).cpu(), group)
        assert (got[~real] == 0).all()
        err = (got.cpu().double() - want).abs()[real.cpu()]
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
        # (the product is exact in float32, the sum rounds at 2^-24 of the result and of its terms)
        assert (err <= (R.U16[dtype] + 2.0 ** -22) * want.abs()[real.cpu()] + tiny + 2.0 ** -22 *
                x.to(dtype).cpu().double().abs().amax()).all()


@pytest.mark.parametrize("dtype", HALF)
def test_append_of_extreme_groups(dtype):
    """Constant and zero groups, the type's largest and smallest values,
    subnormals, ties, infinities and NaN."""
    d, group, h, page = 64, 32, 1, 16
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    n = 12
    x = torch.zeros((n, h, d), dtype=torch.float32)
    x[0] = 3.25
    x[1, 0, :32] = torch.linspace(-big, big, 32)
    x[2, 0, :32] = torch.linspace(0, 15, 32)            # halves: ties to even
    x[2, 0, 32:] = torch.arange(32) % 16 * 0.5
    x[3, 0, 5] = tiny / 8
    x[4, 0, 7] = math.inf
    x[5, 0, 40] = math.nan
    x[6, 0, 3], x[6, 0, 9] = -math.inf, math.inf
    x[7, 0, :32] = torch.arange(32) * tiny / 64
    x[8] = -0.0
    x[9, 0, 0], x[9, 0, 1] = 60000.0, -60000.0
    x[10, 0, 2] = 1e-6
    x[11, 0, ::2] = 1.0
    x = x.to(dtype).to(DEV)
    store = fresh(dtype, 1, h, d, group, page)
    slots = ints([3, 2, 1, 0, 4, 5, 6, 7, 8, 9, 10, 15])
    S.append_paged(store, x, x.flip(0).contiguous(), slots)
    check_slots(store, x, x.flip(0), slots, group)
    assert S.read_paged(store, ints([4]))[0][0, 0, :32].isnan().all()


@pytest.mark.parametrize("offset,step,pad", [(1, 1, 0), (0, 3, 0), (0, 1, 8)])
def test_append_takes_rows_of_any_stride_and_alignment(offset, step, pad):
    d, group, h, page, n = 128, 64, 2, 32, 9
    store, same = (fresh(torch.float16, 2, h, d, group, page) for _ in range(2))
    base = rows(4, n * step, h, d + pad + 1, torch.float16)
    k = base[::step, :, offset:offset + d]
    v = base.transpose(0, 1).contiguous().transpose(0, 1)[::step, :, :d]
    slots = torch.arange(5, 5 + n, dtype=torch.int32, device=DEV)
    S.append_paged(store, k, v, slots)
    S.append_paged(same, k.contiguous(), v.contiguous(), slots)
    for a, b in zip(store, same):
        assert torch.equal(a, b)
    check_slots(store, k, v, slots, group)


def test_append_of_nothing():
    store = fresh(torch.float16, 1, 2, 64, 64, 16)
    e = torch.empty((0, 2, 64), dtype=torch.float16, device=DEV)
    S.append_paged(store, e, e, ints([]))
    k, v = S.read_paged(store, ints([]))
    assert k.shape == v.shape == (0, 2, 64)
    S.append_paged(store, rows(1, 3, 2, 64, torch.float16), rows(2, 3, 2, 64, torch.float16), ints([-1] * 3))
    assert all((t == 0).all() for t in store)


# --------------------------------------------------------------- attention


def world(seed, lengths, new, hkv, d, group, page, dtype, spare=2, noise=True):
    """A store whose requests hold quantised rows (and whose other slots hold
    anything, NaN scales among them), with its tables."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    width = max(max(need), 1) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    store = fresh(dtype, total, hkv, d, group, page, seed=seed if noise else None)
    if noise:
        store.k_meta[:] = math.nan
        store.v_meta[:] = math.nan
    slots = torch.cat([R.slots_of(table[r], n, page) for r, n in enumerate(lengths)] or [torch.zeros(0)])
    n = slots.numel()
    S.append_paged(store, rows(seed + 1, n, hkv, d, dtype), rows(seed + 2, n, hkv, d, dtype, False),
                   slots.to(torch.int32).to(DEV))
    starts = ints([0] + list(np.cumsum(new)))
    return store, table.to(DEV), ints(lengths), starts


def check_attention(out, q, store, table, lengths, starts, scale, causal=True):
    want, tol = R.attend(q, store, table, lengths, starts, scale, causal)
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    assert (err <= tol).all(), f"{float((err / tol.clamp(min=1e-30)).max()):.2f} of the bound"


CASES = [  # lengths, new tokens, query / KV heads, page
    ([1], [1], 4, 1, 16), ([509], [1], 32, 8, 64), ([16, 17, 31, 33], [1, 1, 1, 1], 8, 2, 16),
    ([300, 0, 5, 129], [1, 0, 1, 1], 16, 16, 32), ([700, 64], [4, 4], 16, 4, 32),
    ([40, 3], [7, 3], 28, 4, 128), ([9], [9], 16, 2, 16), ([2100, 100], [1, 2], 8, 1, 16),
    ([90, 200], [33, 70], 8, 2, 64), ([5], [0], 4, 4, 16),
    # prompts, chunks, and decode steps beside them
    ([129], [129], 8, 2, 16), ([65, 300, 1, 200], [65, 100, 1, 2], 16, 4, 32), ([333], [90], 7, 1, 128),
    ([150, 0, 66], [150, 0, 66], 4, 4, 16),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("lengths,new,hq,hkv,page", CASES)
def test_attention(lengths, new, hq, hkv, page, d, group, dtype):
    store, table, le, starts = world(len(lengths) + d, lengths, new, hkv, d, group, page, dtype)
    n = sum(new) + 3
    q = rows(9, n, hq, d, dtype, False)
    scale = 1.0 / math.sqrt(d)
    out = S.paged_attention(q, store, table, le, starts, scale)
    check_attention(out, q, store, table, le, starts, scale)
    assert (out[sum(new):] == 0).all()
    # the launch's hints change nothing but roundings; given rows are left alone
    given = torch.full_like(out, 7.0)
    S.paged_attention(q, store, table, le, starts, scale, max_new=max(1, max(new)),
                      max_length=max(1, max(lengths)), out=given)
    assert (given[sum(new):] == 7.0).all()
    given[sum(new):] = 0
    check_attention(given, q, store, table, le, starts, scale)


@pytest.mark.parametrize("new", [1, 5, 70])
def test_attention_without_a_causal_limit(new):
    store, table, le, starts = world(3, [77, 400], [new, new], 2, 128, 64, 16, torch.float16)
    q = rows(9, 2 * new, 8, 128, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.1, causal=False)
    check_attention(out, q, store, table, le, starts, 0.1, causal=False)


@pytest.mark.parametrize("length", [4000, 12345])
def test_attention_over_many_splits(length):
    store, table, le, starts = world(4, [length, 1000, 3], [1, 1, 1], 2, 128, 64, 16, torch.bfloat16)
    q = rows(9, 3, 8, 128, torch.bfloat16, False)
    first = S.paged_attention(q, store, table, le, starts, 0.09, max_new=1, max_length=length)
    check_attention(first, q, store, table, le, starts, 0.09)
    for _ in range(3):  # bit for bit the same again
        assert torch.equal(S.paged_attention(q, store, table, le, starts, 0.09, max_new=1,
                                             max_length=length), first)
    for hint in (1, 200, 513, 100000):  # (too short ones too: whole columns, then)
        out = S.paged_attention(q, store, table, le, starts, 0.09, max_length=hint)
        check_attention(out, q, store, table, le, starts, 0.09)


@pytest.mark.parametrize("hint", [None, 100])
@pytest.mark.parametrize("b,most", [(70, 300), (300, 40), (150, 900)])
def test_attention_of_many_requests(b, most, hint):
    """More requests than a wave has lanes, more columns than workgroups."""
    rng = random.Random(b)
    lengths = [rng.choice([0, 1, rng.randint(1, most), rng.randint(1, most)]) for _ in range(b)]
    new = [min(n, rng.choice([0, 1, 1, 1, 2])) for n in lengths]
    store, table, le, starts = world(5, lengths, new, 4, 64, 64, 16, torch.float16)
    q = rows(9, sum(new), 8, 64, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.125, max_new=2, max_length=hint)
    check_attention(out, q, store, table, le, starts, 0.125)


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("step", [40.0, 600.0])
def test_attention_with_scores_that_rise_along_the_cache(step, new):
    """Scores that climb by `step` log2 units: the running maximum moves all
    the way, and the last tokens alone count."""
    d, n, page = 64, 600, 16
    store = fresh(torch.bfloat16, 38, 1, d, 64, page)
    k = torch.zeros((n, 1, d), device=DEV)
    k[:, 0, 0] = torch.linspace(0, 1, n, device=DEV)
    v = rows(1, n, 1, d, torch.float32, False)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    S.append_paged(store, k, v, slots)
    table = torch.arange(38, dtype=torch.int32, device=DEV)[None]
    q = torch.zeros((new, 4, d), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 8.0
    scale = step / 8 * math.log(2)
    for sign in (1, -1):
        args = (sign * q, store, table, ints([n]), ints([0, new]), scale)
        check_attention(S.paged_attention(*args), *args)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_with_value_scales_of_all_sizes(new):
    """Value groups from 1e-30 to 1e30 (bfloat16): what is added to what is
    far smaller swallows it, and nothing overflows on the way."""
    d, n, page = 128, 256, 16
    store = fresh(torch.bfloat16, 16, 1, d, 64, page)
    k = rows(1, n, 1, d, torch.float32)
    v = rows(2, n, 1, d, torch.float32, False)
    for order in (1, -1):
        f = 10.0 ** torch.linspace(-30 * order, 30 * order, n, device=DEV)[:, None]
        v2 = v.clone()
        v2[:, 0, :64] *= f
        S.append_paged(store, k, v2, torch.arange(n, dtype=torch.int32, device=DEV))
        table = torch.arange(16, dtype=torch.int32, device=DEV)[None]
        q = rows(3, new, 4, d, torch.bfloat16, False)
        args = (q, store, table, ints([n]), ints([0, new]), 0.05)
        check_attention(S.paged_attention(*args), *args)


@pytest.mark.parametrize("new", [1, 33])
def test_attention_with_queries_of_all_sizes(new):
    for dtype, sizes in ((torch.float16, (6e-8, 1e-4, 1.0, 6e4)), (torch.bfloat16, (1e-30, 1e-3, 1e4, 1e20))):
        store, table, le, starts = world(6, [200], [new], 1, 64, 32, 16, dtype)
        for size in sizes:
            q = (rows(3, new, 4, 64, torch.float32, False).clamp(-1, 1) * size).to(dtype)
            scale = 0.125 / max(1.0, size)
            out = S.paged_attention(q, store, table, le, starts, scale)
            check_attention(out, q, store, table, le, starts, scale)


@pytest.mark.parametrize("new", [4, 50])
@pytest.mark.parametrize("dtype", HALF)
def test_what_a_row_does_not_see_does_not_reach_it(dtype, new):
    """A NaN key or value of a later token, or behind the request's end,
    stays out of the rows before it and makes the others NaN: all dims for a
    key, its group's for a value."""
    n, d, group = 90, 128, 64
    ok = new - 2
    for where in ("k", "v"):
        store, table, le, starts = world(8, [n], [new], 2, d, group, 16, dtype)
        x = rows(1, 1, 2, d, dtype)
        bad = x.clone()
        bad[0, :, group + 3] = math.inf
        at = R.slots_of(table[0], n, 16)[n - 2:n - 1].to(torch.int32).to(DEV)
        S.append_paged(store, bad if where == "k" else x, bad if where == "v" else x, at)
        q = rows(3, new, 4, d, dtype, False)
        out = S.paged_attention(q, store, table, le, starts, 0.1)
        assert torch.isfinite(out[:ok]).all() and out[ok:, :, group:].isnan().all()
        assert out[ok:, :, :group].isnan().all() if where == "k" else out[ok:, :, :group].isfinite().all()
        good = S.paged_attention(q[:ok].contiguous(), store, table, le - 2, ints([0, ok]), 0.1)
        want, tol = R.attend(q[:ok], store, table, le - 2, ints([0, ok]), 0.1)
        for o in (out[:ok], good):
            assert ((o.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("new", [(1, 2), (80, 40)])
def test_pages_outside_the_pool_hold_no_tokens(new):
    store, table, le, starts = world(11, [100, 40], new, 2, 128, 64, 16, torch.float16)
    table[0, 2], table[0, 5], table[1, 0], table[1, 1], table[1, 2] = -1, 10 ** 6, -5, 99, 2 ** 31 - 1
    q = rows(3, sum(new), 4, 128, torch.float16, False)
    out = S.paged_attention(q, store, table, le, starts, 0.1)
    check_attention(out, q, store, table, le, starts, 0.1)
    assert (out[new[0]:] == 0).all()


def test_counts_that_do_not_fit_are_cut_to_the_memory_there_is():
    """Starts and lengths past the tensors: rows and tokens that exist are
    computed, nothing else is read or written."""
    store, table, le, _ = world(12, [64, 64], [1, 1], 2, 64, 64, 16, torch.float16)
    q = rows(3, 2, 4, 64, torch.float16, False)
    out = torch.full_like(q, 7.0)
    S.paged_attention(q, store, table, ints([64, 10 ** 9]), ints([0, 1, 10 ** 9]), 0.1, out=out)
    one = S.paged_attention(q[:1].contiguous(), store, table[:1].contiguous(), ints([64]), ints([0, 1]), 0.1)
    assert torch.equal(out[:1], one)
    S.paged_attention(q, store, table, ints([-4, 64]), ints([-3, -3, 2]), 0.1, out=out)


def test_attention_takes_queries_of_any_stride_and_alignment():
    store, table, le, starts = world(13, [70, 50], [2, 3], 2, 64, 32, 16, torch.bfloat16)
    base = rows(3, 5, 8, 67, torch.bfloat16, False)
    want = S.paged_attention(base[..., 1:65].contiguous(), store, table, le, starts, 0.1)
    assert torch.equal(S.paged_attention(base[..., 1:65], store, table, le, starts, 0.1), want)
    flip = base[..., 1:65].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(S.paged_attention(flip, store, table, le, starts, 0.1), want)
    last = base[..., 1:65].transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(S.paged_attention(last, store, table, le, starts, 0.1), want)


# ---------------------------------------------------------------- together


def test_steps_of_requests_that_come_and_go():
    """Scheduling, appends and attention as a server runs them: prompts enter,
    requests decode, speculate and give drafts back, end, and their pages go
    to others; every step's outputs against all that the requests hold."""
    hq, hkv, d, group, page, dtype = 8, 2, 64, 32, 16, torch.float16
    n_pages, slots_, width = 40, 4, 12
    store = fresh(dtype, n_pages, hkv, d, group, page, seed=1)
    table = torch.full((slots_, width), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(n_pages, dtype=torch.int32, device=DEV)
    lengths, n_free = ints([0] * slots_), ints([n_pages])
    held = [[torch.zeros((0, hkv, d)).double()] * 2 for _ in range(slots_)]
    steps = [[5, 0, 0, 0], [1, 100, 0, 17], [1, 1, 0, 1], [4, 4, 33, 4], [-2, -3, 1, -1],
             [1, 1, 1, 1], [0, -98, 1, 1], [64, 1, 0, -22], [1, 30, 1, 160], [-73, 1, 1, 1]]
    for i, new in enumerate(steps):
        n = sum(max(0, x) for x in new)
        plan = S.build_block_tables(lengths, ints(new), table, free, n_free, page, n + 2,
                                    lengths_out=lengths, n_free_out=n_free)
        S.check_plan(plan)
        k, v = rows(10 + i, n + 2, hkv, d, dtype), rows(50 + i, n + 2, hkv, d, dtype, False)
        S.append_paged(store, k, v, plan.slots)
        q = rows(90 + i, n + 2, hq, d, dtype, False)
        out = S.paged_attention(q, store, table, lengths, plan.token_starts, 0.125,
                                max_new=max(1, max(new)))
        check_attention(out, q, store, table, lengths, plan.token_starts, 0.125)
        at = 0
        for r, x in enumerate(new):
            for j, rows_ in enumerate((k, v)):
                keep = held[r][j][:max(0, held[r][j].shape[0] + min(0, x))]
                fresh_ = R.held(rows_[at:at + max(0, x)].cpu(), group)
                held[r][j] = torch.cat((keep, fresh_))
            at += max(0, x)
            assert int(lengths[r]) == held[r][0].shape[0]
            got = S.read_paged(store, R.slots_of(table[r], int(lengths[r]), page).to(torch.int32).to(DEV))
            for j in range(2):
                assert (got[j].cpu().double() - held[r][j]).abs().max().item() <= 2.0 ** -10 * 16 \
                    if held[r][j].numel() else True
    owned = sum(-(-int(x) // page) for x in lengths)
    assert int(n_free) == n_pages - owned


def test_a_step_replays_from_a_graph():
    """A decode step captured once and replayed: lengths, pages and stack step
    on the device, and every replay equals the same steps run eagerly."""
    hq, hkv, d, group, page, dtype, b = 8, 2, 128, 64, 16, torch.bfloat16, 3
    n_pages = 64

    def state():
        store = fresh(dtype, n_pages, hkv, d, group, page)
        table = torch.full((b, 24), -1, dtype=torch.int32, device=DEV)
        free = torch.arange(n_pages, dtype=torch.int32, device=DEV)
        st = dict(store=store, table=table, free=free, lengths=ints([0] * b), n_free=ints([n_pages]),
                  new=ints([1] * b), k=torch.zeros((b, hkv, d), dtype=dtype, device=DEV),
                  v=torch.zeros((b, hkv, d), dtype=dtype, device=DEV),
                  q=torch.zeros((b, hq, d), dtype=dtype, device=DEV),
                  out=torch.zeros((b, hq, d), dtype=dtype, device=DEV))
        prompt = ints([40, 15, 200])
        plan = S.build_block_tables(st["lengths"], prompt, table, free, st["n_free"], page, 255,
                                    lengths_out=st["lengths"], n_free_out=st["n_free"])
        S.append_paged(store, rows(1, 255, hkv, d, dtype), rows(2, 255, hkv, d, dtype, False), plan.slots)
        return st

    def step(st):
        plan = S.build_block_tables(st["lengths"], st["new"], st["table"], st["free"], st["n_free"],
                                    page, b, lengths_out=st["lengths"], n_free_out=st["n_free"])
        S.append_paged(st["store"], st["k"], st["v"], plan.slots)
        S.paged_attention(st["q"], st["store"], st["table"], st["lengths"], plan.token_starts, 0.1,
                          max_new=1, max_length=384, out=st["out"])

    eager, other = state(), state()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(other)
    for i in range(20):
        for st in (eager, other):
            st["k"].copy_(rows(100 + i, b, hkv, d, dtype))
            st["v"].copy_(rows(200 + i, b, hkv, d, dtype, False))
            st["q"].copy_(rows(300 + i, b, hq, d, dtype, False))
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert eager["lengths"].tolist() == [41 + i, 16 + i, 201 + i] == other["lengths"].tolist()
        assert torch.equal(eager["out"], other["out"])
        assert torch.equal(eager["table"], other["table"])
        torch.empty(1 << 20, device=DEV).random_()  # the program's own work between
    starts = ints([0, 1, 2, 3])
    check_attention(other["out"], other["q"], other["store"], other["table"], other["lengths"], starts, 0.1)


# ------------------------------------- the same, in a call that looks large


@pytest.fixture
def wide(monkeypatch):
    """Tables of 2^20 tokens a row and no hint of the lengths: requests of many
    rows go to the kernel that is for large calls."""
    narrow = S.paged_attention

    def call(q, store, table, lengths, starts, scale, *, max_length=None, **kw):
        more = (1 << 20) // store.page_size - table.shape[1]
        table = torch.nn.functional.pad(table, (0, more), value=-1)
        return narrow(q, store, table, lengths, starts, scale, **kw)

    monkeypatch.setattr(S, "paged_attention", call)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("lengths,new,hq,hkv,page",
                         [c for c in CASES if max(c[1]) * c[2] // c[3] > 64] +
                         [([500, 65], [400, 65], 4, 4, 16), ([1100], [1030], 2, 1, 64)])
def test_large_attention(wide, lengths, new, hq, hkv, page, d, group, dtype):
    test_attention(lengths, new, hq, hkv, page, d, group, dtype)


def test_large_attention_without_a_causal_limit(wide):
    test_attention_without_a_causal_limit(70)


@pytest.mark.parametrize("step", [40.0, 600.0])
def test_large_attention_with_scores_that_rise(wide, step):
    test_attention_with_scores_that_rise_along_the_cache(step, 80)


def test_large_attention_with_values_and_queries_of_all_sizes(wide):
    test_attention_with_value_scales_of_all_sizes(40)
    test_attention_with_queries_of_all_sizes(33)


@pytest.mark.parametrize("dtype", HALF)
def test_large_attention_and_what_a_row_does_not_see(wide, dtype):
    test_what_a_row_does_not_see_does_not_reach_it(dtype, 50)
    test_pages_outside_the_pool_hold_no_tokens((80, 40))


@pytest.mark.parametrize("max_length", [100, 1100, 3000])
def test_more_rows_than_the_hint_says(max_length):
    """Columns beyond those that the merge is launched for, cut and whole."""
    new = [15, 9, 0, 1, 60]
    store, table, le, starts = world(21, [3000, 2000, 700, 1500, 1300], new, 2, 128, 64, 16, torch.float16)
    q = rows(22, sum(new), 8, 128, torch.float16, False)
    for max_new in (1, 4, 16):
        out = S.paged_attention(q, store, table, le, starts, 0.1, max_new=max_new, max_length=max_length)
        check_attention(out, q, store, table, le, starts, 0.1)


def test_a_cache_steps_in_a_graph():
    """Lengths on the GPU, columns cut and joined, and every replay the same as
    the steps run eagerly; then eager sdpa calls beside a captured one."""
    hq, hkv, d, b = 8, 2, 128, 2
    caches = [S.PagedKVCache(n_requests=b, n_kv_heads=hkv, head_dim=d, max_tokens=4096, page_size=32)
              for _ in range(2)]
    given = [torch.zeros((b, h, d), dtype=torch.float16, device=DEV) for h in (hkv, hkv, hq)]
    new, outs = ints([1] * b), [None, None]
    for c in caches:
        c.step(ints([2500, 2500]), 5000)
        c.append(rows(1, 5000, hkv, d, torch.float16), rows(2, 5000, hkv, d, torch.float16, False))

    def step(i):
        caches[i].step(new, b, max_new=1)
        caches[i].append(given[0], given[1])
        outs[i] = caches[i].attend(given[2], 0.1)
        return caches[i].sdpa(given[2].view(b, 1, hq, d).transpose(1, 2), 0.1)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        last = step(1)
    for i in range(6):
        for j, h in enumerate((hkv, hkv, hq)):
            given[j].copy_(rows(30 * j + i, b, h, d, torch.float16, j == 0))
        step(0)
        graph.replay()
        torch.cuda.synchronize()
        c = caches[1]
        assert c.lengths.tolist() == [2501 + i] * b == caches[0].lengths.tolist()
        starts = ints([0, 1, 2])
        for out in (outs[0], outs[1], last.transpose(1, 2).reshape(b, hq, d)):
            check_attention(out, given[2], c.store, c.block_table, c.lengths, starts, 0.1)
        beside = c.sdpa(given[2].view(b, 1, hq, d).transpose(1, 2), 0.1)
        check_attention(beside.transpose(1, 2).reshape(b, hq, d), given[2], c.store, c.block_table,
                        c.lengths, starts, 0.1)
        torch.empty(1 << 20, device=DEV).random_()


def test_calls_on_other_streams():
    """Two streams at once over one store, each with its own workspace."""
    store, table, le, starts = world(14, [3000, 500], [1, 1], 2, 128, 64, 16, torch.float16)
    qs = [rows(20 + i, 2, 8, 128, torch.float16, False) for i in range(2)]
    want = [S.paged_attention(q, store, table, le, starts, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(S.paged_attention(qs[i], store, table, le, starts, 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_refusals_on_the_device():
    store, table, le, starts = world(15, [20], [1], 2, 64, 64, 16, torch.float16)
    q = rows(1, 1, 4, 64, torch.float16, False)
    with pytest.raises(ValueError, match="no backward"):
        S.paged_attention(q.clone().requires_grad_(), store, table, le, starts, 0.1)
    with torch.no_grad():
        S.paged_attention(q.clone().requires_grad_(), store, table, le, starts, 0.1)
    with pytest.raises(_hip.SunShapeUnsupported):
        S.build_block_tables(le, ints([1]), table, ints([0]), ints([1]), 24, 1)
    with pytest.raises(ValueError):
        S.paged_attention(q, store, table, le, starts.cpu(), 0.1)


# ------------------------------------------------------------------- cache


def test_a_trim_of_a_negative_number_gives_nothing_back():
    c = S.PagedKVCache(n_requests=2, n_kv_heads=1, head_dim=64, max_tokens=64)
    c.step([5, 9])
    c.trim(-3)
    assert c.lengths.tolist() == [5, 9]
    c.step(ints([1, 1]), 2)
    c.trim(-3)
    c.trim(0)
    assert c.lengths.tolist() == [6, 10]


def test_cache_serves_requests_of_their_own_lengths():
    """Steps given as lists and as tensors, speculation, trims, releases: the
    outputs and what the cache holds against everything appended."""
    hq, hkv, d, group, page = 8, 2, 128, 64, 32
    c = S.PagedKVCache(n_requests=3, n_kv_heads=hkv, head_dim=d, max_tokens=400, n_pages=20,
                       page_size=page, group_size=group, dtype=torch.bfloat16)
    lengths = [0, 0, 0]

    def go(new, n_tokens=None, seed=0):
        total = sum(max(0, x) for x in new)
        plan = c.step(ints(new), n_tokens) if n_tokens is not None else c.step(new)
        c.check()
        n = plan.slots.numel()
        k, v = rows(seed, n, hkv, d, torch.bfloat16), rows(seed + 50, n, hkv, d, torch.bfloat16, False)
        c.append(k, v)
        q = rows(seed + 90, n, hq, d, torch.bfloat16, False)
        out = c.attend(q, 0.09)
        check_attention(out, q, c.store, c.block_table, c.lengths, plan.token_starts, 0.09)
        assert (out[total:] == 0).all()
        for r, x in enumerate(new):
            lengths[r] += x
        assert c.lengths.tolist() == lengths
        check_slots(c.store, k, v, plan.slots, group)

    go([70, 1, 0], seed=1)
    go([1, 1, 150], seed=2)
    go([4, 4, 4], seed=3)
    go([-3, 0, -1], seed=4)
    c.release([1])
    lengths[1] = 0
    assert c.lengths.tolist() == lengths
    with pytest.raises(RuntimeError, match="no one length"):
        c.offset
    go([1, 33, 1], 40, seed=5)   # from here on the host does not know the lengths
    go([2, -33, 1], 3, seed=6)
    c.release([0])
    lengths[0] = 0
    c.trim(5)
    lengths = [max(0, x - 5) for x in lengths]
    assert c.lengths.tolist() == lengths
    go([9, 9, 1], 19, seed=7)
    assert int(c.n_free) == 20 - sum(-(-x // page) for x in lengths)
    # 9 + 400 tokens fit the 13 pages of a row (416) and the 13 that are free
    # beside the one held; 8 more do not
    c.step(ints([0, 400, 0]), 400)
    c.check()
    lengths[1] += 400
    assert c.lengths.tolist() == lengths
    c.step(ints([0, 8, 0]), 8)
    with pytest.raises(RuntimeError, match="row holds"):
        c.check()
    assert c.lengths.tolist() == lengths and (c.plan.slots == -1).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("t", [1, 3, 40])
def test_cache_in_the_router(t, dtype):
    """update_and_fetch and the SDPA router, as a model calls them."""
    b, hq, hkv, d, group = 2, 8, 2, 64, 32
    c = S.PagedKVCache(n_requests=b, n_kv_heads=hkv, head_dim=d, max_tokens=300, group_size=group,
                       dtype=dtype)
    k, v = (rows(i, b * (90 + t), hkv, d, dtype).view(b, -1, hkv, d).transpose(1, 2) for i in (1, 2))
    c.update_and_fetch(k[:, :, :90], v[:, :, :90])
    ks, vs = c.update_and_fetch(k[:, :, 90:], v[:, :, 90:])
    assert ks.shape == vs.shape == (b, hkv, 90 + t, d) and c.offset == 90 + t
    for got, x in ((ks, k), (vs, v)):
        want = R.held(x.cpu(), group)
        assert ((got.cpu().double() - want).abs() <= R.U16[dtype] * want.abs() + 2.0 ** -22 * 16).all()
    q = rows(3, b * t, hq, d, dtype, False).view(b, t, hq, d).transpose(1, 2)
    starts = ints([0, t, 2 * t])
    for mask in ("causal", None):
        out = S.patch.scaled_dot_product_attention(q, ks, vs, c, 0.125, mask)
        assert out.shape == q.shape
        packed = out.transpose(1, 2).reshape(b * t, hq, d)
        check_attention(packed, q.transpose(1, 2).reshape(b * t, hq, d), c.store, c.block_table,
                        c.lengths, starts, 0.125, mask == "causal")
    c.trim(t)
    assert c.offset == 90
    with pytest.raises(RuntimeError, match="changed"):
        ks2, _ = c.update_and_fetch(k[:, :, 90:], v[:, :, 90:])
        c.trim(1)
        ks2 + 0
    none = S.sunshape_sdpa(q[:, :, :0], c, 0.125)
    assert none.shape == (b, hq, 0, d)
    stats = S.get_kernel_stats()
    assert stats["paged_attn_hip"] > 0 and stats["block_tables_hip"] > 0


def test_cache_decode_step_replays_from_a_graph():
    b, hq, hkv, d = 2, 8, 2, 128
    c = S.PagedKVCache(n_requests=b, n_kv_heads=hkv, head_dim=d, max_tokens=900)
    n = 700
    c.step([n, 300])
    c.append(rows(1, n + 300, hkv, d, torch.float16), rows(2, n + 300, hkv, d, torch.float16, False))
    one = ints([1] * b)
    k, v, q = (torch.zeros((b, h, d), dtype=torch.float16, device=DEV) for h in (hkv, hkv, hq))
    out = torch.zeros_like(q)

    def step():
        c.step(one, b, max_new=1)
        c.append(k, v)
        c.attend(q, 0.1, out=out)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        for j, x in enumerate((k, v, q)):
            x.copy_(rows(10 * i + j, b, x.shape[1], d, torch.float16, j == 0))
        graph.replay()
        torch.cuda.synchronize()
        assert c.lengths.tolist() == [n + i + 1, 301 + i]
        check_attention(out, q, c.store, c.block_table, c.lengths, ints([0, 1, 2]), 0.1)
        torch.empty(1 << 20, device=DEV).random_()
