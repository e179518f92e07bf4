"""Rows of one large score and very many small ones, each below what fp16 holds as a
normal number, which together are 1 % of the row's sum."""

import math

import paged_scores_reference as R
import pytest
import torch

import sunshape_mlx_amd as S
from test_gpu_paged_scores import F16, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(window=1 << 30), dict(softcap=1e3)], ids=["plain", "window", "cap"])
@pytest.mark.parametrize("new", [1, 70])
def test_a_long_flat_tail_is_in_the_rows_sum(new, kw):
    """Token 0 scores 24.6 log2 units above all others, 2^18 of them at 2^-24.6: their
    probabilities enter the products, and have to enter the sum, 1.0104 with them.  All
    tokens hold the same, so that a row is that whatever its probabilities: off by the
    output's rounding (2^-11), the 16-bit operands' (2^-11 of 1.5, the largest), and two
    sums of a rounding a 32-token tile and 64 more."""
    n, d, page = (1 << 18) + new, 64, 1024
    pages = -(-n // page)
    dev = torch.device("cuda:0")
    store = S.PagedKVStore.zeros(pages, 1, d, page_size=page, group_size=64, device=dev)
    k = torch.zeros((n, 1, d), dtype=F16, device=dev)
    k[0, 0, 0] = 1.0
    v = torch.full((n, 1, d), 1.5, dtype=F16, device=dev)
    v[:, :, 1::2] = -0.75
    S.append_paged(store, k, v, torch.arange(n, dtype=torch.int32, device=dev))
    # (a table that may hold more: the rows of 70 tokens are the prompt kernel's)
    table = torch.full((1, 1 << 19), -1, dtype=torch.int32, device=dev)
    table[0, :pages] = torch.arange(pages, dtype=torch.int32, device=dev)
    held = S.read_paged(store, ints([0]))[0][0, 0, 0].item()
    q = torch.zeros((new, 1, d), dtype=F16, device=dev)
    q[..., 0] = 1.0
    scale = 24.6 * math.log(2.0) / held
    args = (q, store, table, ints([n]), ints([0, new]), scale)
    got = S.paged_attention(*args, **kw)
    want = R.attend(*args, **kw)[0]
    tol = 2.0 ** -11 * want.abs() + 1.5 * (2.0 ** -11 + 2 * (n / 32 + 64) * 2.0 ** -24)
    missed = want * (1 + 2.0 ** (18 - 24.6))
    assert bool(((missed - want).abs() > 1.5 * tol).all())
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (off / tol).max().item()
