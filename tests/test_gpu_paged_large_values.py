"""Paged attention over many values next to bfloat16's largest: sums over tokens
pass float32's range unless they are kept below it, whichever kernel takes the
rows, whole or in parts."""

import paged_reference
import paged_scores_reference as R
import paged_strict_check as strict
import pytest
import torch

import sunshape_mlx_amd as S
from test_gpu_paged_scores import BF16, ints, pool, queries

pytestmark = pytest.mark.gpu


def large(seed, lengths, hkv, page=64, d=128, size=1.0, **kw):
    """A pool whose values are 1e38 to 3e38 (times size), of either sign by the dim."""
    store, table = pool(seed, lengths, hkv, d, 64, page, BF16, **kw)
    n = store[0].shape[0] * page
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    v = 1e38 + 2e38 * torch.rand((n, hkv, d), generator=g, device="cuda")
    v = v * size * torch.where(torch.arange(d, device="cuda") // 64 == 1, -1.0, 1.0)
    k = torch.randn((n, hkv, d), generator=g, device="cuda")
    S.append_paged(store, k.to(BF16), v.to(BF16), torch.arange(n, dtype=torch.int32, device="cuda"))
    return store, table


def shared(lengths, new, parents, hkv, hq, hints, size=1.0, **kw):
    store, table = large(51, lengths, hkv, size=size, width=kw.pop("width", None))
    n = sum(new)
    q, le = queries(52, n, hq, 128, BF16), ints(lengths)
    starts = ints([sum(new[:i]) for i in range(len(new) + 1)])
    most = max(lengths[p] for p in parents if p >= 0)
    want = R.attend(q, store, table, le, starts, 0.09, parents=parents, **kw)
    for h in hints:
        plan = S.build_shared_plan(ints(parents), le, starts, n, max_shared=h.get("max_shared", most))
        got = S.paged_attention(q, store, table, le, starts, 0.09, shared=plan, **kw,
                                **{k: v for k, v in h.items() if k != "max_shared"})
        error = strict.check(got, want)
        assert not error, (h, error)


@pytest.mark.parametrize("size", [1.0, 2.0 ** -220])
@pytest.mark.parametrize("kw", [{}, dict(softcap=20.0)])
def test_a_long_prefix(kw, size):
    """Of 64 requests, in parts; in one where the hints are of short ones.  (Small values
    keep their bits in the same scale.)"""
    shared([12000] + [40] * 64, [0] + [1] * 64, [-1] + [0] * 64, 8, 32,
           [dict(max_new=1, max_length=40), dict(max_new=1, max_length=40, max_shared=1), dict()], size, **kw)


def test_a_prefix_of_more_columns_than_are_cut():
    n = 1100
    shared([4000] + [3] * n, [0] + [1] * n, [-1] + [0] * n, 2, 32, [dict(max_new=1, max_length=3)])


@pytest.mark.parametrize("kw", [{}, dict(softcap=20.0)])
def test_many_own_rows_behind_a_prefix(kw):
    """Own tokens that the prompt kernel takes, whole and in parts."""
    shared([5000, 400, 30], [0, 300, 1], [-1, 0, 0], 2, 8, [{}], width=1 << 10, **kw)
    shared([5000, 12000, 30], [0, 70, 1], [-1, 0, 0], 2, 8, [{}], width=1 << 10, **kw)


@pytest.mark.parametrize("kw,prefix", [(dict(softcap=8.0), None), ({}, 300)])
@pytest.mark.parametrize("new", [1100, 2041])
def test_halved_columns_of_one_prompt(new, kw, prefix):
    store, table = large(53, [new], 8)
    q, starts = queries(54, new, 32, 128, BF16), ints([0, new])
    call = dict(kw, prefix_lengths=ints([prefix])) if prefix else kw
    got = S.paged_attention(q, store, table, ints([new]), starts, 0.09, max_new=new, max_length=new, **call)
    error = strict.check(got, R.attend(q, store, table, ints([new]), starts, 0.09, prefix=prefix and [prefix], **kw))
    assert not error, error


@pytest.mark.parametrize("window", [None, 30000])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -220])
def test_long_columns_in_parts(window, size):
    """Of a chunk behind many tokens, without other options too."""
    lengths, new = [33000, 9000], [70, 65]
    store, table = large(55, lengths, 2, size=size)
    q, starts = queries(56, sum(new), 8, 128, BF16), ints([0, 70, 135])
    want = R.attend(q, store, table, ints(lengths), starts, 0.09, window=window)
    for hints in ({}, dict(max_new=70, max_length=33000), dict(max_new=1, max_length=1)):
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.09, window=window, **hints)
        error = strict.check(got, want)
        assert not error, (hints, error)


def test_the_two_restatements_agree_on_large_values():
    store, table = large(57, [300], 1)
    q, starts = queries(58, 2, 4, 128, BF16), ints([0, 2])
    a = R.attend(q, store, table, ints([300]), starts, 0.09)[0]
    b = paged_reference.attend(q, store, table, ints([300]), starts, 0.09)[0]
    assert torch.allclose(a.cpu(), b, rtol=1e-12, atol=0.0) and bool((a.abs() > 1e37).all())
