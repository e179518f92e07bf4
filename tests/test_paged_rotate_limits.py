"""How many tokens the rotated append takes, on the CPU: sizes are checked before
pointers, and these are null, so nothing is launched on either side."""

import ctypes

import pytest

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
