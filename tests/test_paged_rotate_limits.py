"""How many tokens the rotated append takes, on the CPU: sizes are checked before
pointers, and these are null, so nothing is launched on either side.  And what of
autograd it refuses."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

FAKE = 1 << 20  # an address that nothing reads
HEADS = (1, 2, 3, 5, 8, 28, 32, 64, 71, 128, 1024)


def status(n, hq, hkv, d):
    st = paged._Store(FAKE, FAKE, FAKE, FAKE, 4, hkv, d, 64, 64, _hip.SS_F16)
    ro = paged._Rotation(FAKE, 9, d, 0, None, None, 1e-6, 0)
    return _hip.load_library().ss_append_rotated_paged(
        ctypes.addressof(st), None, None, None, _hip.SS_F16, n, hq, hq * d, d, hkv * d, d, hkv * d, d, None, None,
        ctypes.addressof(ro), None, 0, None)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq", HEADS)
def test_the_stated_size_is_taken_with_any_heads(hq, d):
    for hkv in HEADS:
        blocks = (1 << 27) // (hq + hkv) // 8
        for n in (1, 8 * blocks - 7, 8 * blocks):
            assert status(n, hq, hkv, d) == -1, (n, hkv)  # (null pointers)
        assert status((1 << 31) // (hq + hkv) + 8, hq, hkv, d) == -2, hkv
        assert b"too many" in _hip.load_library().ss_last_error()


# ------------------------------------------------- a table under autograd


class Launched(Exception):
    pass


def append(rotary):
    store = S.PagedKVStore.zeros(4, 2, 128, page_size=16, device="cpu")
    q, k = (torch.zeros((3, h, 128), dtype=torch.float16) for h in (4, 2))
    at = torch.zeros(3, dtype=torch.int32)
    return S.append_rotated_paged(store, q, k, k, at, at, rotary)


def test_a_table_under_autograd_is_refused(monkeypatch):
    """Of learned frequencies, say: their gradient would be dropped."""
    def launch(name, dev, *args):
        raise Launched(name)

    monkeypatch.setattr(_hip, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "_launch", launch)
    learned = S.rotary_table(9, 128, frequencies=torch.ones(64, requires_grad=True), device="cpu")
    with pytest.raises(ValueError, match="no backward"):
        append(learned)
    for rotary in (learned.detach(), S.rotary_table(9, 128, device="cpu")):
        with pytest.raises(Launched):
            append(rotary)
    with torch.no_grad(), pytest.raises(Launched):
        append(learned)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        append(forward_ad.make_dual(learned.detach(), torch.ones_like(learned)))
