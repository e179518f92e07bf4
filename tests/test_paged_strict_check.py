"""What the strict bounds of paged attention's tests refuse: the restatement
passes for itself, and with a NaN or a mistake planted in it does not."""

import math

import paged_scores_reference as R
import paged_strict_check as strict
import pytest
import torch
from test_paged_scores_refusals import MISTAKES, example


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("right,wrong", MISTAKES)
def test_mistakes_are_refused(right, wrong, dtype):
    args = example(dtype=dtype)
    want = R.attend(*args, **right)
    assert not strict.check(want[0].to(dtype), want)
    assert strict.check(R.attend(*args, **wrong)[0].to(dtype), want)


@pytest.mark.parametrize("ordinary", [False, True])
@pytest.mark.parametrize("at", [(3, 1, 5), (7,), ()])
def test_nans_are_refused_on_either_side(at, ordinary):
    """One element, one token's rows, all of them."""
    want = R.attend(*example(), softcap=5.0)
    got = want[0].half()
    got[at] = math.nan
    assert strict.check(got, want, ordinary)
    out = want[0].clone()
    out[at] = math.nan
    assert strict.check(want[0].half(), (out, *want[1:]), ordinary)
    assert not strict.check(got, (out, *want[1:]), ordinary)
    got[at] = math.inf
    assert strict.check(got, want, ordinary) and strict.check(got, (out, *want[1:]), ordinary)


def test_a_bound_that_is_nan_shows_nothing():
    out, tol, l2 = R.attend(*example(), softcap=5.0)
    got = out.half()
    assert strict.check(got, (out, tol * math.nan, l2))
    assert strict.check(got, (out, tol, l2 * math.nan)) and not strict.check(got, (out, tol, l2 * math.nan), False)
