"""What the rotated append refuses, on the CPU: the C ABI checks sizes before
any launch, the Python layer checks tensors before it calls."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

FAKE = 1 << 20  # an address that nothing reads


def call(q=FAKE, dtype=_hip.SS_F16, n=1, hq=2, slots=FAKE, positions=FAKE, out=FAKE, rotation=None,
         heads=2, **kw):
    st = paged._Store(FAKE, FAKE, FAKE, FAKE, 4, heads, 128, 64, 64, _hip.SS_F16)
    f = dict(table=FAKE, n_positions=9, rotary_dim=128, neighbours=0, q_weight=None, k_weight=None,
             eps=1e-6, weight_dtype=0)
    f.update(kw)
    ro = paged._Rotation(*f.values())
    return _hip.load_library().ss_append_rotated_paged(
        ctypes.addressof(st), q, FAKE, FAKE, dtype, n, hq, 256, 128, 256, 128, 256, 128, slots,
        positions, ctypes.addressof(ro) if rotation is None else None, out, 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), -1), (dict(dtype=7), -1), (dict(n=-1), -1), (dict(hq=0), -1),
    (dict(slots=None), -1), (dict(positions=None), -1), (dict(out=None), -1),
    (dict(out=FAKE + 8), -1), (dict(rotation=0), -1), (dict(table=None), -1),
    (dict(table=FAKE + 4), -1), (dict(n_positions=0), -1), (dict(rotary_dim=8), -2),
    (dict(rotary_dim=24), -2), (dict(rotary_dim=144), -2), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(q_weight=FAKE, weight_dtype=5), -1), (dict(n=1 << 31), -2),
    (dict(n=1 << 26, hq=1 << 10), -2), (dict(n=1 << 24, heads=1 << 10), -2), (dict(n=0, q=None), 0),
])
def test_calls_that_are_refused(kw, status):
    assert call(**kw) == status
    assert status == 0 or _hip.load_library().ss_last_error()


class Launched(Exception):
    pass


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass for GPU ones; a call that would launch raises Launched."""
    def launch(name, dev, *args):
        raise Launched(name)

    monkeypatch.setattr(_hip, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "_launch", launch)


def args(**kw):
    n = kw.pop("n", 3)
    store = S.PagedKVStore.zeros(4, 2, 128, page_size=16, device="cpu")
    half = torch.float16
    f = dict(store=store, queries=torch.zeros((n, 4, 128), dtype=half),
             keys=torch.zeros((n, 2, 128), dtype=half), values=torch.zeros((n, 2, 128), dtype=half),
             slots=torch.zeros(n, dtype=torch.int32), positions=torch.zeros(n, dtype=torch.int32),
             rotary=torch.zeros((9, 64, 2)))
    f.update(kw)
    return f


def test_a_call_that_is_taken(on_cpu):
    w = torch.ones(128)
    with pytest.raises(Launched, match="ss_append_rotated_paged"):
        S.append_rotated_paged(**args(q_weight=w, k_weight=w))


@pytest.mark.parametrize("kw,error", [
    (dict(queries=torch.zeros((3, 4, 128))), TypeError),
    (dict(queries=torch.zeros((3, 4, 64), dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros((2, 4, 128), dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros((3, 0, 128), dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros((3, 128), dtype=torch.float16)), ValueError),
    (dict(keys=torch.zeros((3, 1, 128), dtype=torch.float16)), ValueError),
    (dict(values=torch.zeros((3, 2, 128), dtype=torch.bfloat16)), TypeError),
    (dict(slots=torch.zeros((3, 1), dtype=torch.int32)), ValueError),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(rotary=torch.zeros((9, 64, 2), dtype=torch.float64)), TypeError),
    (dict(rotary=torch.zeros((9, 128))), ValueError),
    (dict(rotary=torch.zeros((9, 64, 3))), ValueError),
    (dict(rotary=torch.zeros((9, 128, 2))[:, ::2]), ValueError),
    (dict(q_weight=torch.ones(64)), ValueError),
    (dict(q_weight=torch.ones(256)[::2]), ValueError),
    (dict(q_weight=torch.ones(128), k_weight=torch.ones(128, dtype=torch.float16)), TypeError),
    (dict(k_weight=torch.ones(128, dtype=torch.float64)), (TypeError, ValueError)),
    (dict(out=torch.zeros((3, 4, 128))), ValueError),
    (dict(out=torch.zeros((3, 2, 128), dtype=torch.float16)), ValueError),
    (dict(out=torch.zeros((3, 4, 256), dtype=torch.float16)[..., ::2]), ValueError),
    (dict(queries=torch.zeros((3, 4, 128), dtype=torch.float16, requires_grad=True)), ValueError),
    (dict(q_weight=torch.nn.Parameter(torch.ones(128))), ValueError),
    (dict(k_weight=torch.nn.Parameter(torch.ones(128))), ValueError),
])
def test_tensors_that_are_refused(on_cpu, kw, error):
    with pytest.raises(error):
        S.append_rotated_paged(**args(**kw))


def test_parameters_are_taken_without_autograd(on_cpu):
    with torch.no_grad(), pytest.raises(Launched):
        S.append_rotated_paged(**args(q_weight=torch.nn.Parameter(torch.ones(128))))


def test_forward_mode_is_refused(on_cpu):
    f = args()
    with forward_ad.dual_level():
        f["queries"] = forward_ad.make_dual(f["queries"], torch.ones_like(f["queries"]))
        with pytest.raises(ValueError, match="forward-mode"):
            S.append_rotated_paged(**f)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU fallback"):
        S.append_rotated_paged(**args())


@pytest.mark.parametrize("kw", [dict(n_positions=0), dict(rotary_dim=8), dict(rotary_dim=40),
                                dict(base=0.0), dict(base=float("inf")), dict(base=float("nan")),
                                dict(frequencies=torch.ones(9))])
def test_rotary_tables_that_are_refused(kw):
    with pytest.raises(ValueError):
        S.rotary_table(**{**dict(n_positions=5, rotary_dim=16, device="cpu"), **kw})


def test_a_cache_needs_a_step_before_it_rotates():
    cache = S.PagedKVCache(n_requests=1, n_kv_heads=2, max_tokens=64, device="cpu")
    f = args()
    with pytest.raises(RuntimeError, match="step first"):
        cache.append_rotated(f["queries"], f["keys"], f["values"], f["rotary"])
