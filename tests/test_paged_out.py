"""What autograd learns of tensors that a paged call writes into, on the CPU:
nothing is launched."""

import pytest
import torch

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

F16 = torch.float16


@pytest.fixture(autouse=True)
def nothing_runs(monkeypatch):
    monkeypatch.setattr(_hip, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    monkeypatch.setattr(paged, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(paged, "_scored_workspace_bytes", lambda *a: 0)


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def rotate(q, out):
    store = S.PagedKVStore.zeros(4, 2, 128, page_size=16, device="cpu")
    k = torch.zeros((3, 2, 128), dtype=F16)
    return S.append_rotated_paged(store, q, k, k, ints([0] * 3), ints([0] * 3), torch.zeros((9, 64, 2)), out=out)


def attend(q, out, **kw):
    store = S.PagedKVStore.zeros(4, 2, 128, page_size=16, device="cpu")
    return S.paged_attention(q, store, ints([[0, 1]]), ints([9]), ints([0, 3]), 0.1, out=out, **kw)


CALLS = {"rotate": rotate, "attend": attend, "capped": lambda q, out: attend(q, out, softcap=5.0)}


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_a_graph_that_saved_what_is_written_has_no_backward_pass(call):
    """Its gradient would be that of other values."""
    w = torch.ones((3, 4, 128), dtype=F16, requires_grad=True)
    q, out = torch.zeros((3, 4, 128), dtype=F16), torch.zeros((3, 4, 128), dtype=F16)
    loss = (out * w).sum()
    assert call(q, out) is out
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_queries_turned_in_place_too():
    w = torch.ones((3, 4, 128), dtype=F16, requires_grad=True)
    q = torch.zeros((3, 4, 128), dtype=F16)
    loss = (q * w).sum()
    rotate(q, q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_out_under_autograd_is_refused(call):
    q = torch.zeros((3, 4, 128), dtype=F16)
    out = torch.zeros((3, 4, 128), dtype=F16, requires_grad=True)
    with pytest.raises(ValueError, match="no backward"):
        call(q, out)
    with torch.no_grad():
        assert call(q, out) is out


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_new_outputs_and_inference_tensors_pass(call):
    q = torch.zeros((3, 4, 128), dtype=F16)
    assert call(q, None)._version == 0 and q._version == 0
    with torch.inference_mode():
        call(torch.zeros_like(q), torch.zeros_like(q))
        call(q, torch.zeros_like(q))
