"""The rotated append of the paged 4-bit cache against a restatement that
rounds every operation to float32 as it does (queries and codes exactly), and
against 64 bits (within the roundings' sum)."""

import math

import paged_reference as R
import pytest
import torch

import sunshape_mlx_amd as S

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPES = [(128, 64), (128, 128), (128, 32), (64, 64), (64, 32)]
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rows(seed, n, h, d, dtype, size=1.0):
    g = torch.Generator().manual_seed(seed)
    s = 0.5 + 3.5 * torch.rand((d,), generator=g)
    return (torch.randn((n, h, d), generator=g) * s * size).to(dtype).to(DEV)


def pairs(y, rdim, neighbours):
    if neighbours:
        return y[..., :rdim:2], y[..., 1:rdim:2]
    return y[..., :rdim // 2], y[..., rdim // 2:rdim]


def joined(a, b, neighbours):
    return torch.stack((a, b), -1).flatten(-2) if neighbours else torch.cat((a, b), -1)


def rotated(x, positions, table, weight, eps, neighbours, dtype):
    """(the operator's result in ``dtype``, the same in 64 bits, its tolerance)
    on the CPU; every float32 operation below is one rounding."""
    x, table, rdim = x.cpu(), table.cpu(), 2 * table.shape[1]
    y, y64 = x.float(), x.double()
    if weight is not None:
        mean = y64.square().mean(-1, keepdim=True) + eps
        r64 = 1.0 / mean.sqrt()
        y, y64 = (y * r64.float()) * weight.cpu().float(), y64 * r64 * weight.cpu().double()
    turn = table[positions.cpu().long().clamp(0, table.shape[0] - 1)][:, None]
    a, b = pairs(y, rdim, neighbours)
    c, s = turn[..., 0], turn[..., 1]
    z = torch.cat((joined(a * c - b * s, b * c + a * s, neighbours), y[..., rdim:]), -1)
    a, b = pairs(y64, rdim, neighbours)
    c, s = c.double(), s.double()
    z64 = torch.cat((joined(a * c - b * s, b * c + a * s, neighbours), y64[..., rdim:]), -1)
    # y: three roundings; a product one more, their sum one
    size = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    size = torch.cat((joined(*size, neighbours), y64[..., rdim:].abs()), -1)
    u = R.U16[dtype]
    tiny = 2.0 ** -24 if dtype == F16 else 0.0  # half a step of its subnormals, and more
    return z.to(dtype), z64, 1.01 * (5 * 2.0 ** -24 * size * (1 + u) + u * z64.abs()) + tiny


def held_codes(store, slots):
    """Codes and (scale, zero) of these slots, on the CPU."""
    k, v, km, vm = R.unpack(store)
    at = slots.cpu().long()
    return k[at], v[at], km[at], vm[at]


def check_stored(store, slots, k, v, group):
    """Keys and values (N, H, D) of the store's type are in these slots."""
    kc, vc, km, vm = held_codes(store, slots)
    for x, code, meta in ((k, kc, km), (v, vc, vm)):
        want, scale, zero = R.quantize(x, group)
        assert torch.equal(meta[..., 0].isnan(), scale.isnan())
        ok = ~scale.isnan()
        assert torch.equal(meta[..., 0][ok], scale[ok]) and torch.equal(meta[..., 1][ok], zero[ok])
        assert torch.equal(code, want)


def case(seed, n, hq, hkv, d, group, dtype, store_dtype, page=16, norm=True, span=100):
    store = S.PagedKVStore.zeros(-(-n // page) + 3, hkv, d, page_size=page, group_size=group,
                                 dtype=store_dtype, device=DEV)
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(store.k_codes.shape[0] * page, generator=g)[:n].int()
    positions = torch.randint(0, span, (n,), generator=g).int()
    w = (1.0 + 0.2 * torch.randn((2, d), generator=g)).to(dtype).to(DEV)
    return dict(store=store, q=rows(seed + 1, n, hq, d, dtype), k=rows(seed + 2, n, hkv, d, dtype),
                v=rows(seed + 3, n, hkv, d, dtype), slots=slots.to(DEV), positions=positions.to(DEV),
                qw=w[0] if norm else None, kw=w[1] if norm else None)


def run_and_check(s, table, eps=1e-6, neighbours=False, **kw):
    store, dtype = s["store"], s["q"].dtype
    q_type = store.dtype if dtype == F32 else dtype
    args = (s["positions"], table)
    k_in, v_in, q_in = s["k"].clone(), s["v"].clone(), s["q"].clone()
    got = S.append_rotated_paged(store, s["q"], s["k"], s["v"], s["slots"], *args, q_weight=s["qw"],
                                 k_weight=s["kw"], eps=eps, neighbours=neighbours, **kw)
    assert got.dtype == q_type and got.shape == q_in.shape
    want, exact, tol = rotated(q_in, *args, s["qw"], eps, neighbours, q_type)
    assert torch.equal(got.cpu(), want)
    assert bool(((got.cpu().double() - exact).abs() <= tol).all())
    k = rotated(k_in, *args, s["kw"], eps, neighbours, store.dtype)[0]
    check_stored(store, s["slots"], k, v_in.cpu().to(store.dtype), store.head_dim // store.k_meta.shape[2])
    return got


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,store_dtype", [(F16, F16), (BF16, BF16), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("d,group", SHAPES)
def test_rotated_append_is_its_formula(d, group, dtype, store_dtype, norm, neighbours):
    table = S.rotary_table(100, d, device=DEV)
    for n, hq, hkv in ((1, 4, 2), (9, 8, 2), (67, 3, 1)):
        s = case(n, n, hq, hkv, d, group, dtype, store_dtype, norm=norm)
        run_and_check(s, table, neighbours=neighbours)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("d,rdim", [(128, 16), (128, 48), (128, 64), (128, 112), (64, 16), (64, 48)])
def test_heads_rotated_in_part(d, rdim, neighbours):
    table = S.rotary_table(300, rdim, 500000.0, device=DEV)
    s = case(rdim, 21, 6, 3, d, 32, BF16, BF16, span=300)
    run_and_check(s, table, neighbours=neighbours)


@pytest.mark.parametrize("n,hq,hkv", [(8, 32, 8), (130, 32, 8), (513, 28, 4), (40, 1, 1), (300, 71, 1),
                                      (2041, 16, 4)])
def test_runs_of_heads_and_tokens(n, hq, hkv):
    table = S.rotary_table(5000, 128, device=DEV)
    run_and_check(case(n, n, hq, hkv, 128, 64, F16, F16, page=64, span=5000), table)


def test_one_weight_alone_and_other_types_of_weights():
    table = S.rotary_table(100, 64, device=DEV)
    for q, k in ((True, False), (False, True)):
        s = case(5, 19, 4, 2, 64, 32, F16, F16)
        s["qw"], s["kw"] = s["qw"].float() if q else None, s["kw"].float() if k else None
        run_and_check(s, table)
    s = case(6, 19, 4, 2, 64, 32, F16, F16)
    s["qw"], s["kw"] = s["qw"].bfloat16(), s["kw"].bfloat16()
    run_and_check(s, table, eps=0.5)


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_slices_of_one_projection(shift):
    """Queries, keys and values as a model's joint projection leaves them: rows
    of a larger stride, at odd addresses too."""
    n, hq, hkv, d = 37, 8, 2, 128
    wide = rows(3, n, 1, (hq + 2 * hkv) * d + 8, BF16)[:, 0, shift:]
    s = case(4, n, hq, hkv, d, 64, BF16, BF16)
    at = [0, hq * d, (hq + hkv) * d, (hq + 2 * hkv) * d]
    s["q"], s["k"], s["v"] = (wide[:, a:b].unflatten(1, (-1, d)) for a, b in zip(at, at[1:]))
    run_and_check(s, S.rotary_table(100, d, device=DEV))


def test_heads_last_and_reversed_rows():
    s = case(7, 20, 4, 2, 64, 64, F16, F16)
    for x in "qkv":
        s[x] = s[x].permute(1, 2, 0).contiguous().permute(2, 0, 1)
    run_and_check(s, S.rotary_table(100, 64, device=DEV))


def test_queries_turned_in_place():
    s = case(8, 45, 8, 2, 128, 64, F16, F16)
    got = run_and_check(s, S.rotary_table(100, 128, device=DEV), out=s["q"])
    assert got.data_ptr() == s["q"].data_ptr()


@pytest.mark.parametrize("n", [5, 8, 29])
def test_tokens_without_a_position_or_a_slot(n):
    """Negative positions: query zero (or left), nothing stored, whatever the
    slot; slots outside the pool: the query is turned, nothing stored."""
    s = case(9, n, 4, 2, 128, 32, BF16, BF16)
    store, table = s["store"], S.rotary_table(100, 128, device=DEV)
    for t in store:
        t.view(torch.int16 if t.dtype == BF16 else torch.int32).fill_(0x1234)
    before = [t.clone() for t in store]
    gone, unslotted = [0, n - 1], [1, 3]
    s["positions"][gone] = ints([-1, -(2 ** 31)])
    s["slots"][unslotted] = ints([-1, store.k_codes.shape[0] * 16])
    left = torch.full_like(s["q"], 7.0)
    kw = dict(q_weight=s["qw"], k_weight=s["kw"])
    args = (store, s["q"], s["k"], s["v"], s["slots"], s["positions"], table)
    zeroed = S.append_rotated_paged(*args, **kw)
    S.append_rotated_paged(*args, **kw, out=left)
    want = rotated(s["q"], s["positions"], table, s["qw"], 1e-6, False, BF16)[0]
    stays = torch.ones(n, dtype=torch.bool)
    stays[gone] = False
    for got, rest in ((zeroed, 0.0), (left, 7.0)):
        assert torch.equal(got.cpu()[stays], want[stays])
        assert bool((got.cpu()[gone] == rest).all())
    stored = stays.clone()
    stored[unslotted] = False
    k = rotated(s["k"], s["positions"], table, s["kw"], 1e-6, False, BF16)[0]
    check_stored(store, s["slots"][stored.to(DEV)], k[stored], s["v"].cpu()[stored], 32)
    other = torch.ones(store.k_codes.shape[0] * 16, dtype=torch.bool)
    other[s["slots"].cpu().long()[stored]] = False
    for a, b in zip(R.unpack(store), R.unpack(before)):
        a, b = (x.view(torch.int16) if x.dtype == BF16 else x for x in (a, b))
        assert torch.equal(a[other], b[other])


def test_positions_past_the_table_are_nan():
    s = case(10, 6, 2, 2, 128, 64, F16, F16, norm=False)
    s["positions"][:] = ints([99, 100, 2 ** 31 - 1, 0, 98, 101])
    got = S.append_rotated_paged(s["store"], s["q"], s["k"], s["v"], s["slots"], s["positions"],
                                 S.rotary_table(100, 64, device=DEV)).cpu()
    bad = torch.tensor([False, True, True, False, False, True])
    assert bool(got[bad][..., :64].isnan().all()) and not bool(got[~bad].isnan().any())
    assert torch.equal(got[..., 64:], s["q"].cpu()[..., 64:])
    km = held_codes(s["store"], s["slots"])[2]
    assert bool(km[bad][:, :, 0].isnan().all()) and not bool(km[bad][:, :, 1].isnan().any())
    assert not bool(km[~bad].isnan().any())


@pytest.mark.parametrize("norm", [False, True])
def test_infinities_nans_zeros_and_large_values(norm):
    """A key that is not finite spoils its head's turned groups and, under a
    norm, its row; the other rows keep their bits.  Large values are squared
    in 64 bits."""
    s = case(11, 8, 2, 2, 128, 32, BF16, BF16, norm=norm)
    s["k"][0, 0, 3], s["k"][1, 1, 100], s["q"][2, 0, 5] = math.inf, math.nan, math.nan
    s["k"][3], s["q"][3] = 0.0, 0.0
    s["k"][4] *= 1e37
    s["q"][5] *= 2.0 ** 100
    s["q"][6] *= 2.0 ** -100
    table = S.rotary_table(100, 128, device=DEV)
    got = S.append_rotated_paged(s["store"], s["q"], s["k"], s["v"], s["slots"], s["positions"], table,
                                 q_weight=s["qw"], k_weight=s["kw"]).cpu()
    args = (s["positions"], table)
    want = rotated(s["q"], *args, s["qw"], 1e-6, False, BF16)[0]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    k = rotated(s["k"], *args, s["kw"], 1e-6, False, BF16)[0]
    check_stored(s["store"], s["slots"], k, s["v"].cpu(), 32)


def test_zero_rows_without_eps():
    s = case(12, 2, 2, 1, 64, 64, F16, F16)
    s["q"][0] = 0.0
    got = S.append_rotated_paged(s["store"], s["q"], s["k"], s["v"], s["slots"], s["positions"],
                                 S.rotary_table(100, 64, device=DEV), q_weight=s["qw"], eps=0.0).cpu()
    assert bool(got[0].isnan().all()) and not bool(got[1].isnan().any())


def test_nothing_to_append():
    s = case(13, 1, 2, 1, 64, 64, F16, F16)
    empty = [s[x][:0] for x in ("q", "k", "v", "slots", "positions")]
    out = S.append_rotated_paged(s["store"], *empty, S.rotary_table(100, 64, device=DEV))
    assert out.shape == (0, 2, 64)


def test_rotary_tables():
    t = S.rotary_table(70000, 64, 500000.0, device=DEV).cpu().double()
    p, i = torch.arange(70000, dtype=torch.float64)[:, None], torch.arange(32, dtype=torch.float64)
    angle = p * 500000.0 ** (-i / 32)
    # the angle's own rounding in 64 bits, and one of the result
    assert bool(((t[..., 0] - angle.cos()).abs() <= 2.0 ** -24).all())
    assert bool(((t[..., 1] - angle.sin()).abs() <= 2.0 ** -24).all())
    f = torch.linspace(0.1, 1.0, 8)
    t = S.rotary_table(9, 16, frequencies=f, device=DEV).cpu().double()
    assert bool(((t[8, :, 1] - (8 * f.double()).sin()).abs() <= 2.0 ** -24).all())


def test_offsets_past_32_bits():
    """Queries and results of more than 2^31 elements."""
    n, hq, d = 66000, 256, 128
    s = case(14, 16, hq, 1, d, 128, F16, F16, norm=False)
    q = torch.zeros((n, hq, d), dtype=F16, device=DEV)
    q[-16:] = s["q"]
    k = torch.zeros((n, 1, d), dtype=F16, device=DEV)
    slots = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    positions = torch.zeros((n,), dtype=torch.int32, device=DEV)
    positions[-16:] = s["positions"]
    table = S.rotary_table(100, d, device=DEV)
    out = S.append_rotated_paged(s["store"], q, k, k, slots, positions, table, out=torch.full_like(q, 3.0))
    assert torch.equal(out[-16:].cpu(), rotated(s["q"], s["positions"], table, None, 0, False, F16)[0])
    assert not bool(out[:-16].any())


# -------------------------------------------------------------- the cache


def cache_of(**kw):
    return S.PagedKVCache(n_requests=3, n_kv_heads=2, head_dim=128, max_tokens=200, page_size=16,
                          dtype=BF16, device=DEV, **kw)


def test_a_cache_steps_rotates_and_attends():
    """append_rotated is the norm, the rotation and append one after the other."""
    table = S.rotary_table(200, 128, device=DEV)
    a, b = cache_of(), cache_of()
    w = rows(20, 1, 2, 128, BF16)[0].abs()
    for step, new in enumerate(([5, 0, 33], [1, 1, 1], [-2, 17, 4])):
        n = sum(max(0, x) for x in new)
        q, k, v = (rows(30 + 3 * step + i, n, h, 128, BF16) for i, h in enumerate((8, 2, 2)))
        a.step(new)
        b.step(new)
        positions = b.plan.positions
        got = a.append_rotated(q, k, v, table, q_weight=w[0], k_weight=w[1])
        turned = [rotated(x, positions, table, y, 1e-6, False, BF16)[0].to(DEV) for x, y in
                  ((q, w[0]), (k, w[1]))]
        b.append(turned[1], v)
        assert torch.equal(got, turned[0])
        assert all(torch.equal(x, y) for x, y in zip(a.store, b.store))
        assert torch.equal(a.attend(got, 0.1), b.attend(turned[0], 0.1))


def test_captured_steps_and_another_stream():
    """A step, its rotated append and its attention in a graph, replayed with
    eager work between, are what the eager calls give; on another stream too."""
    table = S.rotary_table(200, 128, device=DEV)
    graphed, eager = cache_of(), cache_of()
    new = ints([1, 2, 0])
    q, k, v = (torch.empty((3, h, 128), dtype=BF16, device=DEV) for h in (8, 2, 2))

    def one(cache):
        cache.step(new, 3, max_new=2)
        return cache.attend(cache.append_rotated(q, k, v, table), 0.1)

    for x, seed in ((q, 1), (k, 2), (v, 3)):
        x.copy_(rows(seed, 3, x.shape[1], 128, BF16))
    warm = cache_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(graphed)
    for i in range(4):
        for x, seed in ((q, 10), (k, 20), (v, 30)):
            x.copy_(rows(seed + i, 3, x.shape[1], 128, BF16))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = one(eager)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(x, y) for x, y in zip(graphed.store, eager.store))
        assert torch.equal(graphed.lengths, eager.lengths)
