"""Capped scores of the paged attention: what a row does not see and what other
rows score changes nothing of it."""

import paged_scores_reference as R
import paged_strict_check as strict
import pytest
import torch

import sunshape_mlx_amd as S
from test_gpu_paged_scores import BF16, F16, ints, pool, queries

pytestmark = pytest.mark.gpu


def page_0_unused(store, table):
    """Page 0, which is read where a table names none of the pool, holds no
    request's tokens."""
    free = next(p for p in range(store[0].shape[0]) if p not in set(table.flatten().tolist()))
    if free:
        for t in store:
            t[free] = t[0].clone()
        table[table == 0] = free


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("hidden", ["behind", "window", "outside"])
@pytest.mark.parametrize("d,group", [(128, 64), (64, 32)])
def test_hidden_keys_have_no_say(d, group, hidden, many):
    """Large finite keys behind a request's tokens, before its window, and in
    pages that it does not have leave every bit as it is."""
    lengths, new = ([399, 1001], [200, 300]) if many else ([399, 1001], [1, 3])
    store, table = pool(41, lengths, 2, d, group, 16, F16, width=1 << 12 if many else None)
    page_0_unused(store, table)
    q, starts = queries(42, sum(new), 8, d, F16), ints([0, new[0], sum(new)])
    kw = dict(softcap=3e4, window=75 if hidden == "window" else None)
    if hidden == "outside":
        table[0, 5], table[0, 24], table[1, 61] = -1, 1 << 30, -7

    def attend():
        return S.paged_attention(q, store, table, ints(lengths), starts, 0.1, **kw)

    clean = attend()
    want = R.attend(q, store, table, ints(lengths), starts, 0.1, **kw)
    assert not strict.check(clean, want), strict.check(clean, want)
    m = store.k_meta
    if hidden == "outside":
        m[0] = 5e4
    for r, n in enumerate(lengths):
        if hidden == "behind":
            m[int(table[r, n // 16]), :, :, n % 16:] = 5e4
        elif hidden == "window":
            for t in range(n - new[r] + 1 - 75):
                m[int(table[r, t // 16]), :, :, t % 16] = 5e4
    assert torch.equal(attend(), clean)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("large", [0, 5])
def test_rows_of_small_scores_beside_rows_of_large_ones(large, many):
    """One head's scores reach the cap, 2^20; the others', a few units, keep
    theirs to 2^-21 of themselves."""
    lengths, new = ([399, 1001], [200, 300]) if many else ([399, 1001], [1, 3])
    store, table = pool(43, lengths, 2, 128, 64, 16, F16, width=1 << 12 if many else None)
    q, starts = queries(44, sum(new), 8, 128, BF16), ints([0, new[0], sum(new)])
    q[:, large] *= 2.0 ** 21
    for cap in (2.0 ** 20, 3e4):
        got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, softcap=cap)
        want = R.attend(q, store, table, ints(lengths), starts, 0.1, softcap=cap)
        rest = [h for h in range(8) if h != large]
        error = strict.check(got[:, rest], [x[:, rest] for x in want])
        assert not error, error
        error = strict.check(got, want, False)
        assert not error, error


def test_a_prefix_of_many_rows_beside_a_row_of_large_scores():
    n, cap = 40, 2.0 ** 20
    lengths, parents = [1500] + [50] * n, [-1] + [0] * n
    store, table = pool(45, lengths, 2, 128, 64, 16, F16)
    q, starts = queries(46, n, 8, 128, BF16), ints([0, *range(n + 1)])
    q[7, 3] *= 2.0 ** 21
    plan = S.build_shared_plan(ints(parents), ints(lengths), starts, n, max_shared=1500)
    got = S.paged_attention(q, store, table, ints(lengths), starts, 0.1, shared=plan, max_new=1, max_length=50,
                            softcap=cap)
    want = R.attend(q, store, table, ints(lengths), starts, 0.1, parents=parents, softcap=cap)
    rest = [i for i in range(n) if i != 7]
    error = strict.check(got[rest], [x[rest] for x in want])
    assert not error, error


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("q_size,k_size,scale,cap", [
    (1e24, 1.0, 1.0, 2.0 ** -60), (1e30, 1e-30, 1.0, 2.0 ** -60), (1e30, 1e-30, 1.0, 0.5), (1e20, 1e10, 1.0, 2.0 ** 60),
    (2.0 ** -60, 2.0 ** 97, 2.0 ** -40, 2.0 ** 60), (2.0 ** -100, 2.0 ** 100, 0.5, 2.0 ** 40),
    (1.0, 1.0, 1.0, 2.0 ** -60), (1.0, 1.0, 1.0, 2.0 ** 60)])
def test_caps_of_any_size(q_size, k_size, scale, cap, many):
    """The factor of a product over the cap may pass float32 either way; half of the
    tokens' keys are 0, and score 0."""
    lengths, new = ([399, 1001], [200, 300]) if many else ([399, 1001], [1, 3])
    store, table = pool(47, lengths, 2, 128, 64, 16, BF16, width=1 << 12 if many else None)
    n = store[0].shape[0] * 16
    g = torch.Generator(device="cuda").manual_seed(48)
    k, v = (torch.randn((n, 2, 128), generator=g, device="cuda").to(BF16) for _ in range(2))
    k[::2] = 0
    S.append_paged(store, k * k_size, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    q, starts = queries(49, sum(new), 8, 128, BF16) * q_size, ints([0, new[0], sum(new)])
    got = S.paged_attention(q, store, table, ints(lengths), starts, scale, softcap=cap)
    want = R.attend(q, store, table, ints(lengths), starts, scale, softcap=cap)
    error = strict.check(got, want, False)
    assert not error, error
