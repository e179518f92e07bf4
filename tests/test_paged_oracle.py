"""The paged cache's L2 check, on the CPU: right results, rounded as the
kernels round them, pass it, and results that are a little wrong do not."""

import paged_reference as R
import pytest
import torch

import sunshape_mlx_amd as S

CASES = [  # lengths, new tokens, query / KV heads, page, causal prompt
    ([509], [1], 32, 8, 64), ([2100, 100], [1, 2], 8, 1, 16), ([12345, 1000, 3], [1, 1, 1], 8, 2, 16),
    ([333], [90], 7, 1, 128),
]


def packed(codes):
    """(..., 8) codes as int32 words."""
    sh = torch.tensor([R.bit(j) for j in range(8)])
    return (codes.long() << sh).sum(-1).to(torch.int32)


def rows(seed, n, h, d, dtype, spread=True):
    g = torch.Generator().manual_seed(seed)
    s = 0.5 + 3.5 * torch.rand((d,), generator=g) if spread else 1.0
    return (torch.randn((n, h, d), generator=g) * s).to(dtype)


def world(case, dtype, d=128, group=64):
    """A store on the CPU whose requests hold quantised rows, its tables, queries."""
    lengths, new, hq, hkv, page = case
    need = [-(-n // page) for n in lengths]
    total, width = sum(need), max(need)
    store = S.PagedKVStore.zeros(total, hkv, d, page_size=page, group_size=group, dtype=dtype, device="cpu")
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = order[sum(need[:r]):sum(need[:r + 1])]
    n = total * page  # (every slot holds something)
    for x, codes, meta in ((rows(2, n, hkv, d, dtype), store.k_codes, store.k_meta),
                           (rows(3, n, hkv, d, dtype, False), store.v_codes, store.v_meta)):
        code, scale, zero = (t.unflatten(0, (total, page)).transpose(1, 2) for t in R.quantize(x, group))
        words = code.unflatten(-1, (-1, 8)) if codes is store.k_codes else \
            code.unflatten(2, (-1, 8)).transpose(3, 4)
        codes.copy_(packed(words))
        meta.copy_(torch.stack((scale, zero), -1).transpose(2, 3))
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    q = rows(4, sum(new), hq, d, dtype, False)
    return q, store, table, torch.tensor(lengths, dtype=torch.int32), starts, d ** -0.5


def attend(q, store, table, lengths, starts, scale, form=None, drop=None, half=0.0):
    """The attention in 64 bits, rounded as a kernel rounds it (``form``), with
    a page of every request left out (``drop``), or values half a code off."""
    k_c, v_c, k_m, v_m = R.unpack(store)
    k_all, v_all = R.values_of(k_c, k_m), R.values_of(v_c + half, v_m)
    page, rep = store.page_size, q.shape[1] // store.n_kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    for r, length in enumerate(lengths.tolist()):
        at, pos = R.slots_of(table[r], length, page), torch.arange(length)
        for h in range(store.n_kv_heads):
            for i in range(int(starts[r + 1] - starts[r])):
                see = pos <= length - int(starts[r + 1] - starts[r]) + i
                if drop is not None:
                    see = see & (pos // page != drop)
                heads, row = slice(h * rep, (h + 1) * rep), int(starts[r]) + i
                s = q[row, heads].double() @ k_all[at, h][see].t() * scale
                e = torch.exp(s - s.amax(-1, keepdim=True))
                v, total = v_all[at, h][see], e.sum(-1, keepdim=True)
                if form == "prompt":
                    e, v = (e * 1024).half().double() / 1024, v.half().double()
                if form == "decode":
                    vs = v_m[at, h][see][..., 0].double()
                    mid = (vs * 7.5 + v_m[at, h][see][..., 1].double()).repeat_interleave(q.shape[2] // vs.shape[1], 1)
                    c = v_c[at, h][see].double().unflatten(-1, (vs.shape[1], -1)) - 7.5
                    ps = (e[..., None] * vs).half().double()             # (heads, T, G)
                    out[row, heads] = (e @ mid + torch.einsum("htg,tgd->hgd", ps, c).flatten(1)) / total
                else:
                    out[row, heads] = e @ v / total
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_the_l2_check_tells_right_from_wrong(case, dtype):
    args = world(case, dtype)
    want, bound = R.attend_l2(*args)
    assert (bound <= (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -9) * want.norm(dim=-1)).all()
    right = attend(*args)
    assert (right - want).abs().max() <= 1e-12
    for form in ("decode", "prompt"):
        assert R.within_l2(attend(*args, form=form).to(dtype), want, bound)
    q, scale = args[0], args[-1]
    fp8 = (q.to(torch.float8_e4m3fn).to(dtype), *args[1:])
    wrong = dict(
        loss=0.97 * want, scale=attend(*args[:-1], 1.01 * scale), page=attend(*args, drop=1),
        half_code=attend(*args, half=0.5), queries=attend(*fp8), none=torch.zeros_like(want))
    for name, out in wrong.items():
        if name != "page" or max(case[0]) > case[-1]:
            assert not R.within_l2(out.to(dtype), want, bound), name
