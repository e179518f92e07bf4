"""The paged 4-bit cache's operators at the ends of what their calls allow:
starts, lengths, magnitudes and counts that the ordinary cases do not reach,
against the 64-bit restatement (tests/paged_reference.py)."""

import math

import pytest
import torch
from test_gpu_paged import DEV, check_attention, ints, rows, world

import sunshape_mlx_amd as S

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
