"""What paged attention with other scores and masks, and over shared tokens,
refuses, on the CPU; and what the GPU tests' bounds refuse: the restatement
with a mistake planted in it does not pass for itself."""

import ctypes
import math

import paged_reference
import paged_scores_reference as R
import pytest
import torch

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

FAKE = 1 << 20  # an address that nothing reads


def scores(**kw):
    f = dict(softcap=0.0, slopes=None, window=0, prefix_lengths=None, group_starts=None, group_rows=None,
             parents=None, n_groups=1, max_shared=100)
    f.update(kw)
    return paged._Scores(*f.values())


def shared(**kw):
    return scores(**{**dict(group_starts=FAKE, group_rows=FAKE, parents=FAKE), **kw})


def store():
    return paged._Store(FAKE, FAKE, FAKE, FAKE, 4, 2, 128, 64, 64, _hip.SS_F16)


def attention(sc, n=1, hq=2, r=1, width=4, max_new=1, max_length=256, ws=None, ws_bytes=0, **kw):
    f = dict(q=FAKE, table=FAKE, lengths=FAKE, starts=FAKE, out=FAKE, q_dtype=_hip.SS_F16)
    f.update(kw)
    st = store()
    return _hip.load_library().ss_paged_attn_scored(
        ctypes.addressof(st), f["q"], f["q_dtype"], n, hq * 128, 128, hq, f["table"], width,
        f["lengths"], f["starts"], r, 0.1, 1, max_new, max_length, f["out"], 0,
        ctypes.addressof(sc) if sc is not None else None, ws, ws_bytes, None)


@pytest.mark.parametrize("sc,status", [
    (scores(softcap=-1.0), -1), (scores(softcap=math.nan), -1), (scores(softcap=math.inf), -1),
    (scores(softcap=2.0 ** -61), -1), (scores(window=-1), -1), (shared(group_rows=None), -1),
    (shared(group_starts=None), -1), (shared(parents=None), -1), (shared(group_rows=FAKE + 4), -1),
    (shared(window=5), -2), (shared(prefix_lengths=FAKE), -2), (shared(max_shared=0), -1),
    (shared(n_groups=0), -1), (shared(max_shared=1 << 31), -1), (shared(), -4),
])
def test_calls_that_are_refused(sc, status):
    assert attention(sc) == status
    assert _hip.load_library().ss_last_error()


@pytest.mark.parametrize("kw,status", [(dict(q=None), -1), (dict(q_dtype=_hip.SS_F32), -2), (dict(hq=3), -1),
                                       (dict(r=0), -1), (dict(out=None), -1), (dict(n=0), 0),
                                       (dict(max_length=5000, width=100), -4)])
def test_other_arguments_are_checked_as_ever(kw, status):
    for sc in (scores(softcap=5.0), None):
        assert attention(sc, **kw) == status


def test_a_window_and_shared_tokens_size_the_workspace():
    lib, st = _hip.load_library(), store()

    def need(sc, length=20000, n=1):
        return lib.ss_paged_attn_scored_workspace_bytes(ctypes.addressof(st), n, 1, 2, 1, length,
                                                        ctypes.addressof(sc))

    plain = lib.ss_paged_attn_workspace_bytes(ctypes.addressof(st), 1, 1, 2, 1, 20000)
    assert need(scores(softcap=2.0)) == plain and need(scores(window=500)) == 0
    part = 2 * 130 * 4
    assert need(shared(max_shared=20000)) == plain + part and need(shared(), 100) == part
    assert need(shared(max_shared=20000), 100) == plain + part
    assert attention(shared(), max_length=100, ws=FAKE, ws_bytes=part - 1) == -4
    assert need(scores(softcap=-1.0)) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(r=0), -1), (dict(n=-1), -1), (dict(r=4097), -2), (dict(n=1 << 31), -2),
    (dict(parents=None), -1), (dict(rows=None), -1), (dict(rows=FAKE + 4), -1), (dict(of=None), -1)])
def test_shared_plans_that_are_refused(kw, status):
    f = dict(parents=FAKE, r=2, n=3, rows=FAKE, of=FAKE)
    f.update(kw)
    assert _hip.load_library().ss_shared_plan(f["parents"], FAKE, FAKE, f["r"], f["n"], FAKE, f["rows"],
                                              f["of"], FAKE, None, None) == status


# ------------------------------------------------------------ Python layer


class Launched(Exception):
    pass


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass for GPU ones; a call that would launch raises Launched."""
    def launch(name, dev, *args):
        raise Launched(name)

    monkeypatch.setattr(_hip, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "_launch", launch)
    monkeypatch.setattr(paged, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(paged, "_scored_workspace_bytes", lambda *a: 0)


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def attend(**kw):
    pool = S.PagedKVStore.zeros(4, 2, 128, page_size=16, device="cpu")
    return S.paged_attention(torch.zeros((3, 4, 128), dtype=torch.float16), pool, ints([[0, 1], [2, 3]]),
                             ints([5, 9]), ints([0, 1, 3]), 0.1, **kw)


def plan(**kw):
    return S.SharedPlan(ints([0, 0, 0]), ints([[0, 0]] * 3), ints([-1, -1]), ints([0] * 3))._replace(**kw)


@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(slopes=torch.ones(4)), dict(window=7),
                                dict(prefix_lengths=ints([1, 2])), dict(shared=plan())])
def test_calls_that_are_taken(on_cpu, kw):
    with pytest.raises(Launched, match="ss_paged_attn_scored"):
        attend(**kw)


def test_a_call_without_options_is_the_plain_one(on_cpu):
    with pytest.raises(Launched, match="ss_paged_attn$"):
        attend()


@pytest.mark.parametrize("kw,error", [
    (dict(softcap=0.0), ValueError), (dict(softcap=-3.0), ValueError),
    (dict(softcap=math.nan), ValueError), (dict(softcap=math.inf), ValueError),
    (dict(softcap=1e30), ValueError), (dict(slopes=torch.ones(2)), ValueError),
    (dict(slopes=torch.ones(4, dtype=torch.float16)), TypeError),
    (dict(slopes=torch.ones(8)[::2]), ValueError),
    (dict(slopes=torch.ones(4, requires_grad=True)), ValueError),
    (dict(window=0), ValueError), (dict(window=-5), ValueError),
    (dict(prefix_lengths=ints([1])), ValueError),
    (dict(prefix_lengths=torch.tensor([1, 2])), TypeError),
    (dict(shared=plan(rows=ints([[0, 0]] * 2))), ValueError),
    (dict(shared=plan(group_starts=ints([0, 0]))), ValueError),
    (dict(shared=plan(parents=ints([-1]))), ValueError),
    (dict(shared=plan(rows=torch.zeros((3, 2)))), TypeError),
    (dict(shared=plan(), window=4), ValueError),
    (dict(shared=plan(), prefix_lengths=ints([1, 2])), ValueError),
])
def test_options_that_are_refused(on_cpu, kw, error):
    with pytest.raises(error):
        attend(**kw)


@pytest.mark.parametrize("args,kw,error", [
    ((ints([[0]]), ints([1]), ints([0, 1]), 1), {}, ValueError),
    ((torch.tensor([0]), ints([1]), ints([0, 1]), 1), {}, TypeError),
    ((ints([0]), ints([1, 2]), ints([0, 1]), 1), {}, ValueError),
    ((ints([0]), ints([1]), ints([0]), 1), {}, ValueError),
    ((ints([0]), ints([1]), ints([0, 1]), -1), {}, ValueError),
    ((ints([0]), ints([1]), ints([0, 1]), 1), dict(n_groups=0), ValueError),
    ((ints([0]), ints([1]), ints([0, 1]), 1), dict(max_shared=-1), ValueError),
])
def test_plan_arguments_that_are_refused(on_cpu, args, kw, error):
    with pytest.raises(error):
        S.build_shared_plan(*args, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU fallback"):
        S.build_shared_plan(ints([-1]), ints([1]), ints([0, 1]), 1)


# -------------------------------------------------------------- the cache


def cache(**kw):
    return S.PagedKVCache(**{**dict(n_requests=4, n_kv_heads=2, max_tokens=64, device="cpu"), **kw})


def test_who_may_continue_whom():
    c = cache()
    c.share([1, 2], 0)
    assert c.parents.tolist() == [-1, 0, 0, -1]
    for requests, parent in (([3], 1), ([0], 3), ([3], 3), ([4], 0), ([-1], 0), ([3], 4), ([3], -1)):
        with pytest.raises(ValueError):
            c.share(requests, parent)
        assert c.parents.tolist() == [-1, 0, 0, -1]
    c.share([1], None)
    c.share([3], 0)
    assert c.parents.tolist() == [-1, -1, 0, 0]


def test_requests_that_hold_tokens_keep_what_they_continue():
    c = cache()
    c._host = [5, 0, 3, 0]
    c.share([1], 0)
    with pytest.raises(ValueError, match="hold tokens"):
        c.share([2, 3], 0)
    assert c.parents.tolist() == [-1, 0, -1, -1]


def test_a_prefix_does_not_end_before_its_children(on_cpu):
    c = cache()
    c.share([1], 0)
    with pytest.raises(ValueError, match="others continue"):
        c.release([0])
    with pytest.raises(Launched):
        c.release([0, 1])


def test_batches_of_equal_steps_are_refused_where_requests_share(on_cpu):
    c = cache()
    c.share([1], 0)
    x = torch.zeros((4, 2, 1, 128), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="alike"):
        c.update_and_fetch(x, x)
    with pytest.raises(RuntimeError, match="alike"):
        S.sunshape_sdpa(x, c, 0.1, "causal")
    c.share([1], None)
    with pytest.raises(Launched):
        c.update_and_fetch(x, x)


# --------------------------------------- what the GPU tests' bounds refuse


def example(seed=0, dtype=torch.float16):
    """A cache on the CPU that holds quantised tokens."""
    g = torch.Generator().manual_seed(seed)
    page, hkv, d, group = 16, 2, 64, 32
    pool = S.PagedKVStore.zeros(60, hkv, d, page_size=page, group_size=group, dtype=dtype, device="cpu")
    n = 60 * page
    sh = torch.tensor([paged_reference.bit(j) for j in range(8)])
    for x, codes, meta, values in ((torch.randn((n, hkv, d), generator=g) * 2, 0, 2, False),
                                   (torch.randn((n, hkv, d), generator=g), 1, 3, True)):
        c, s, z = paged_reference.quantize(x.to(dtype), group)
        c = c.view(60, page, hkv, d).transpose(1, 2)
        c = c.unflatten(2, (-1, 8)).transpose(3, 4) if values else c.unflatten(3, (-1, 8))
        words = (c << sh).sum(-1)
        pool[codes].copy_(torch.where(words >= 1 << 31, words - (1 << 32), words).int())
        m = torch.stack((s, z), -1).view(60, page, hkv, d // group, 2)
        pool[meta].copy_(m.permute(0, 2, 3, 1, 4))
    table = torch.randperm(60, generator=g).int().view(3, 20)
    q = torch.randn((24, 8, d), generator=g).to(dtype)
    return q, pool, table, ints([300, 41, 77]), ints([0, 3, 7, 24]), 0.125


MISTAKES = [
    (dict(softcap=5.0), dict(softcap=5.2)), (dict(softcap=5.0), dict()),
    (dict(slopes=torch.full((8,), 0.05)), dict(slopes=torch.full((8,), 0.051))),
    (dict(slopes=2.0 ** -torch.arange(8.0)), dict(slopes=2.0 ** -torch.arange(8.0).flip(0))),
    (dict(window=20), dict(window=21)), (dict(window=20), dict(window=19)),
    (dict(prefix=[290, 40, 70]), dict(prefix=[290, 40, 69])), (dict(prefix=[299, 40, 70]), dict()),
    (dict(parents=[-1, 0, 0]), dict()), (dict(parents=[-1, 0, 0]), dict(parents=[-1, 0, -1])),
    (dict(parents=[-1, 0, 0], slopes=torch.full((8,), 0.02)),
     dict(parents=[-1, 0, 0], slopes=torch.full((8,), 0.0205))),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("right,wrong", MISTAKES)
def test_bounds_refuse_mistakes(right, wrong, dtype):
    args = example(dtype=dtype)
    want = R.attend(*args, **right)
    assert not R.check(want[0].to(dtype), want)
    assert R.check(R.attend(*args, **wrong)[0].to(dtype), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_restatement_is_the_plain_one_without_options(dtype):
    args = example(1, dtype)
    want, _ = paged_reference.attend(*args)
    assert torch.allclose(R.attend(*args)[0], want, rtol=1e-12, atol=1e-14)
