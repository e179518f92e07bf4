"""What the paged cache's entry points refuse, on the CPU: the C ABI checks
sizes before any launch, the Python layer checks tensors before it calls."""

import ctypes

import pytest
import torch

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged

FAKE = 1 << 20  # an address that nothing reads


def store(**kw):
    f = dict(k_codes=FAKE, v_codes=FAKE, k_meta=FAKE, v_meta=FAKE, n_pages=4, n_kv_heads=2,
             head_dim=128, group_size=64, page_size=64, dtype=_hip.SS_F16)
    f.update(kw)
    return paged._Store(**f)


BAD_STORES = [
    (dict(k_codes=None), -1), (dict(v_meta=FAKE + 4), -1), (dict(n_pages=0), -1),
    (dict(n_kv_heads=0), -1), (dict(dtype=_hip.SS_F32), -2), (dict(head_dim=96), -2),
    (dict(head_dim=256), -2), (dict(group_size=16), -2), (dict(head_dim=64, group_size=128), -2),
    (dict(page_size=8), -2), (dict(page_size=48), -2), (dict(page_size=2048), -2),
    (dict(n_pages=1 << 26), -2),
]


@pytest.mark.parametrize("kw,status", BAD_STORES)
def test_stores_that_are_refused(kw, status):
    lib, st = _hip.load_library(), store(**kw)
    at = ctypes.addressof(st)
    assert lib.ss_append_paged(at, FAKE, FAKE, 1, 1, 256, 128, 256, 128, FAKE, None) == status
    assert lib.ss_read_paged(at, FAKE, 1, FAKE, FAKE, None) == status
    assert attention(st) == status
    assert lib.ss_paged_attn_workspace_bytes(at, 1, 1, 2, 1, 1000) == 0


def attention(st=None, q=FAKE, q_dtype=_hip.SS_F16, n=1, hq=2, table=FAKE, width=4, lengths=FAKE,
              starts=FAKE, r=1, max_new=1, max_length=256, out=FAKE, ws=None, ws_bytes=0):
    st = store() if st is None else st
    return _hip.load_library().ss_paged_attn(
        ctypes.addressof(st), q, q_dtype, n, hq * 128, 128, hq, table, width, lengths, starts, r,
        0.1, 1, max_new, max_length, out, 0, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), -1), (dict(q_dtype=_hip.SS_F32), -2), (dict(q_dtype=7), -2), (dict(n=-1), -1),
    (dict(hq=3), -1), (dict(hq=0), -1), (dict(hq=2048), -2), (dict(table=None), -1),
    (dict(width=0), -1), (dict(width=1 << 30), -2), (dict(lengths=None), -1),
    (dict(starts=None), -1), (dict(r=0), -1), (dict(r=70000), -1), (dict(max_new=0), -1),
    (dict(max_length=0), -1), (dict(out=None), -1), (dict(out=FAKE + 2), -1),
    (dict(n=1 << 31), -2), (dict(max_length=5000, width=100), -4),
    (dict(max_length=5000, width=100, ws=FAKE, ws_bytes=64), -4), (dict(n=0), 0),
])
def test_attention_calls_that_are_refused(kw, status):
    assert attention(**kw) == status
    assert status == 0 or _hip.load_library().ss_last_error()


def test_workspace_is_what_the_call_asks_for():
    lib = _hip.load_library()
    for n, r, hq, new, length in ((1, 1, 2, 1, 512), (1, 1, 2, 1, 513), (1, 1, 2, 1, 1024),
                                  (1, 1, 2, 1, 1025), (300, 2, 8, 200, 4000),
                                  (4096, 256, 32, 1, 131072)):
        st = store()
        need = lib.ss_paged_attn_workspace_bytes(ctypes.addressof(st), n, r, hq, new, length)
        # (few columns of at most 8 units of 128 tokens are not cut)
        assert (need == 0) == (length <= 8 * 128 and new == 1)
        if need:
            assert attention(n=n, r=r, hq=hq, max_new=new, max_length=length, width=4000,
                             ws=FAKE, ws_bytes=need - 1) == -4


@pytest.mark.parametrize("kw,status", [
    (dict(n_tokens=-1), -1), (dict(n_requests=0), -1), (dict(n_requests=4097), -2),
    (dict(width=0), -1), (dict(pool=0), -1), (dict(page_size=24), -2), (dict(page_size=8), -2),
    (dict(pool=1 << 28), -2), (dict(lengths=None), -1), (dict(slots=None), -1),
])
def test_block_table_calls_that_are_refused(kw, status):
    f = dict(lengths=FAKE, n_requests=2, width=4, pool=8, page_size=64, n_tokens=3, slots=FAKE)
    f.update(kw)
    assert _hip.load_library().ss_block_tables(
        f["lengths"], FAKE, f["n_requests"], FAKE, f["width"], FAKE, f["pool"], FAKE,
        f["page_size"], f["n_tokens"], FAKE, FAKE, FAKE, f["slots"], None, FAKE, None) == status


@pytest.mark.parametrize("n,dtype,keys,status", [(-1, 1, FAKE, -1), (1, 9, FAKE, -1), (1, 1, None, -1), (0, 1, None, 0)])
def test_append_calls_that_are_refused(n, dtype, keys, status):
    st = store()
    assert _hip.load_library().ss_append_paged(ctypes.addressof(st), keys, FAKE, dtype, n, 256, 128,
                                               256, 128, FAKE, None) == status


def test_more_tokens_than_a_launch_counts_are_refused():
    """Pairs of (token, head) are counted in 32 bits when read back, blocks of
    8 tokens of a head when written."""
    lib, st = _hip.load_library(), store(n_kv_heads=1024, n_pages=64)
    at = ctypes.addressof(st)
    assert lib.ss_read_paged(at, FAKE, 1 << 21, FAKE, FAKE, None) == -2
    assert lib.ss_append_paged(at, FAKE, FAKE, 1, 1 << 24, 256, 128, 256, 128, FAKE, None) == -2


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


def pool(n=3, h=2, d=128, **kw):
    return S.PagedKVStore.zeros(n, h, d, device="cpu", **kw)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def call(store=None, n=2, **kw):
    store = pool() if store is None else store
    f = dict(queries=torch.zeros(n, 4, 128, dtype=torch.float16), store=store,
             block_table=torch.zeros(1, 3, dtype=torch.int32), lengths=ints(5),
             token_starts=ints(0, n), scale=0.1)
    f.update(kw)
    return S.paged_attention(**f)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU fallback"):
        call()
    with pytest.raises(ValueError, match="no CPU fallback"):
        S.build_block_tables(ints(1), ints(1), torch.zeros(1, 1, dtype=torch.int32), ints(0), ints(1), 16, 1)
    with pytest.raises(ValueError, match="no CPU fallback"):
        S.read_paged(pool(), ints(0))


def test_a_good_call_gets_to_its_launch(on_cpu):
    with pytest.raises(Launched, match="ss_paged_attn"):
        call()
    z = torch.zeros(2, 2, 128)
    with pytest.raises(Launched, match="ss_append_paged"):
        S.append_paged(pool(), z, z, ints(0, 1))


@pytest.mark.parametrize("kw,error", [
    (dict(queries=torch.zeros(2, 4, 128)), TypeError),
    (dict(queries=torch.zeros(2, 3, 128, dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros(2, 4, 64, dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros(2, 4, dtype=torch.float16)), ValueError),
    (dict(queries=torch.zeros(2, 4, 128, dtype=torch.float16, requires_grad=True)), ValueError),
    (dict(lengths=torch.tensor([5])), TypeError), (dict(lengths=ints(5, 6)), ValueError),
    (dict(token_starts=ints(0)), ValueError), (dict(token_starts=ints(0, 1, 2)), ValueError),
    (dict(block_table=torch.zeros(1, 6, dtype=torch.int32)[:, ::2]), ValueError),
    (dict(out=torch.zeros(2, 4, 128)), ValueError), (dict(out=torch.zeros(1, 4, 128, dtype=torch.float16)), ValueError),
])
def test_attention_arguments_that_are_refused(on_cpu, kw, error):
    with pytest.raises(error):
        call(**kw)


def test_stores_whose_tensors_do_not_agree(on_cpu):
    good = pool()
    for i, t in enumerate(good):
        for bad in (t[:2], t.transpose(0, 1), t.double() if t.is_floating_point() else t.long()):
            with pytest.raises((ValueError, TypeError)):
                S.read_paged(S.PagedKVStore(*good[:i], bad, *good[i + 1:]), ints(0))
    with pytest.raises((ValueError, TypeError)):
        S.read_paged(S.PagedKVStore(good[0], good[1], good[2], good[3].bfloat16()), ints(0))


def test_appends_that_are_refused(on_cpu):
    z = torch.zeros(2, 2, 128)
    for k, v, s in ((z[:1], z, ints(0, 1)), (z, z[:, :1], ints(0, 1)), (z, z.half(), ints(0, 1)),
                    (z.double(), z.double(), ints(0, 1)), (z, z, torch.tensor([0, 1])), (z, z, ints(0, 1, 2))):
        with pytest.raises((ValueError, TypeError)):
            S.append_paged(pool(), k, v, s)


@pytest.mark.parametrize("kw,error", [
    (dict(head_dim=96), ValueError), (dict(group_size=48), ValueError), (dict(page_size=40), ValueError),
    (dict(dtype=torch.float32), TypeError), (dict(n_requests=0), ValueError),
    (dict(max_tokens=0), ValueError), (dict(n_pages=0), ValueError), (dict(n_kv_heads=0), ValueError),
])
def test_caches_that_are_refused(kw, error):
    f = dict(n_requests=2, n_kv_heads=2, head_dim=128, max_tokens=100, device="cpu")
    f.update(kw)
    with pytest.raises(error):
        S.PagedKVCache(**f)


def test_cache_steps_that_are_refused(on_cpu, monkeypatch):
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c = S.PagedKVCache(n_requests=2, n_kv_heads=2, head_dim=128, max_tokens=100, n_pages=3,
                       page_size=32, device="cpu")
    z = torch.zeros(1, 2, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="step first"):
        c.append(z, z)
    with pytest.raises(RuntimeError, match="step first"):
        c.attend(z, 0.1)
    for bad in ([1], [1, 2, 3], [101, 0], [-1, 0]):
        with pytest.raises(ValueError):
            c.step(bad)
    with pytest.raises(RuntimeError, match="pages"):
        c.step([64, 64])
    with pytest.raises(ValueError):
        c.step([5, 5], 9)
    with pytest.raises(ValueError, match="n_tokens"):
        c.step(ints(1, 1))
    c.step([5, 3])
    with pytest.raises(RuntimeError, match="one length"):
        c.offset
    q = torch.zeros(2, 4, 1, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="mask"):
        S.sunshape_sdpa(q, c, 0.1, torch.zeros(1))
    with pytest.raises(ValueError):
        S.sunshape_sdpa(q[:1], c, 0.1)
    with pytest.raises(ValueError, match="dtype"):
        S.sunshape_sdpa(q, c, 0.1, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        c.update_and_fetch(q, q)
    with pytest.raises(ValueError):
        c.release([2])
    with pytest.raises(ValueError):
        c.make_mask(1, return_array=True)
    with pytest.raises(TypeError):
        S.save_cache("/nonexistent", c)


@pytest.mark.parametrize("shape", [(2, 4, 128), (0, 4, 128)])
def test_queries_with_a_tangent_are_refused(on_cpu, shape):
    """Forward mode: the kernel would drop the tangent.  Queries without one
    pass, inside a level too."""
    from torch.autograd import forward_ad

    q = torch.zeros(shape, dtype=torch.float16)
    n = shape[0]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for grad in (True, False):  # (no_grad does not reach forward mode)
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                call(n=n, queries=dual)
        if n:
            with pytest.raises(Launched):
                call(n=n, queries=q)
            with pytest.raises(Launched):
                call(n=n, queries=forward_ad.unpack_dual(dual).primal)


def test_sdpa_queries_with_a_tangent_are_refused(on_cpu, monkeypatch):
    from torch.autograd import forward_ad

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = S.PagedKVCache(n_requests=2, n_kv_heads=2, head_dim=128, max_tokens=100, device="cpu")
    q = torch.zeros(2, 4, 1, 128, dtype=torch.float16)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError, match="forward-mode"):
            S.sunshape_sdpa(dual, c, 0.1, "causal")
        with pytest.raises(Launched):
            S.sunshape_sdpa(q, c, 0.1, "causal")


def sized(n, r, tokens, hq=32, hkv=8, page=64, max_new=None, max_length=None, **kw):
    """Status of a call of these sizes that has no workspace: -4 where the
    sizes are taken."""
    return attention(store(n_kv_heads=hkv, page_size=page, **kw), n=n, r=r, hq=hq, width=tokens // page,
                     max_new=max_new or n - r + 1, max_length=max_length or tokens)


@pytest.mark.parametrize("n,r,tokens,hq", [
    # prompts and chunks of tables that hold 131072 and 2^20 tokens a row
    (65536, 1, 131072, 32), (65536, 16, 131072, 32), (65536, 32, 131072, 32), (131072, 1, 131072, 32),
    (32768, 1, 131072, 64), (32768, 8, 131072, 64), (92161, 1, 131072, 32), (8192, 1, 1 << 20, 32),
    (1 << 20, 1, 1 << 20, 32), (1 << 22, 1, 1 << 22, 32), (3000, 1000, 1 << 20, 32), (1000, 1000, 1 << 20, 32),
    (4096, 4096, 131072, 32), (65535, 65535, 16384, 32),
])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_prompts_and_batches_that_are_taken(n, r, tokens, hq, group):
    assert sized(n, r, tokens, hq, group_size=group) == -4
    # hints that are too low for these tables cost time, not the call
    assert sized(n, r, tokens, hq, group_size=group, max_new=1) == -4


def test_counts_past_32_bits_are_refused():
    """128 requests of one row a KV head, 8 rows a block: at most 128 + 128/8
    blocks of rows, over as many blocks of 128 tokens as fit 32 bits, and one more."""
    for heads in (2, 4):
        most = (2 ** 31 - 1) // ((128 + 16) * heads)
        for blocks, status in ((most, -4), (most + 1, -2)):
            assert sized(128, 128, blocks * 128, heads, heads, page=16, max_new=1) == status
    # the decode kernel's part of many long prompts: 16 blocks a request at most
    assert sized(1 << 20, 1000, 1 << 20, group_size=32) == -4
    assert sized(1 << 20, 4097, 1 << 20, group_size=32) == -2
    assert b"32 bits" in _hip.load_library().ss_last_error()


def known(c):
    """What a cache knows on the host."""
    return c._host, c._bound, c._max_new, c._version, c.plan


def small_cache(**kw):
    f = dict(n_requests=2, n_kv_heads=2, head_dim=128, max_tokens=100, page_size=32, device="cpu")
    f.update(kw)
    return S.PagedKVCache(**f)


@pytest.mark.parametrize("step", [
    lambda c: c.step(torch.tensor([1, 1]), 2), lambda c: c.step(ints(1), 2), lambda c: c.step(ints(1, 1, 1), 3),
    lambda c: c.step(ints(1, 2)[::2], 2), lambda c: c.step(ints(1, 1), -1), lambda c: c.step(ints(1, 1)),
    lambda c: c.step([1, 1], 1), lambda c: c.step([1, "x"]), lambda c: c.step([200, 0]), lambda c: c.step([1, 1]),
    lambda c: c.step(ints(1, 1), 2), lambda c: c.trim(1), lambda c: c.release([0]),
])
def test_steps_that_fail_leave_the_cache_as_it_was(on_cpu, monkeypatch, step):
    """Refused arguments, and launches that raise."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    refuse = paged._launch
    c = small_cache()
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c.step([5, 3])
    c.step([-2, 1])
    monkeypatch.setattr(paged, "_launch", refuse)
    before = known(c)
    assert before[:3] == ([3, 4], 4, 1)
    with pytest.raises((ValueError, TypeError, Launched)):
        step(c)
    assert known(c) == before
    assert c.plan is before[-1]


def test_steps_given_as_lists_are_not_captured(on_cpu, monkeypatch):
    launch = paged._launch
    c = small_cache()
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c.step([5, 5])
    monkeypatch.setattr(paged, "_launch", launch)
    monkeypatch.setattr(paged, "_capturing", lambda t: True)
    before = known(c)
    z = torch.zeros(2, 2, 1, 128, dtype=torch.float16)
    for call_ in (lambda: c.step([1, 1]), lambda: c.trim(1), lambda: c.release([0]),
                  lambda: c.update_and_fetch(z, z)):
        with pytest.raises(RuntimeError, match="captured"):
            call_()
        assert known(c) == before


@pytest.mark.parametrize("k,v", [
    (torch.float16, torch.float32), (torch.float64, torch.float64), (torch.int32, torch.int32), ("meta", None),
    (None, "meta"),
])
def test_updates_that_are_refused_add_no_tokens(monkeypatch, k, v):
    """Types that the append does not take, keys or values on another device."""
    def one_device(*tensors):
        if any(t.is_meta for t in tensors):
            raise ValueError("another device")

    monkeypatch.setattr(_hip, "require_gpu", one_device)
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c = small_cache()
    c.step([5, 5])
    before = known(c)
    good = torch.zeros(2, 2, 3, 128, dtype=torch.float16)

    def other(x):
        return good if x is None else good.to("meta") if x == "meta" else good.to(x)

    with pytest.raises((ValueError, TypeError)):
        c.update_and_fetch(other(k), other(v))
    assert known(c) == before
    c.update_and_fetch(good, good)
    assert c.offset == 8


@pytest.mark.parametrize("kw", [
    dict(n_requests=4097), dict(max_tokens=2 ** 30 + 1, n_pages=1), dict(page_size=0), dict(n_pages=2 ** 26),
    dict(n_pages=2 ** 21, n_kv_heads=1024, page_size=16), dict(n_requests=4096, max_tokens=2 ** 26, n_pages=1),
])
def test_caches_that_no_step_would_take_are_not_built(kw, monkeypatch):
    def zeros(*a, **k):  # (a pool of this size is not made)
        raise Launched

    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch, "full", zeros)
    with pytest.raises(ValueError):
        small_cache(**dict(dict(page_size=32), **kw))


def test_the_largest_number_of_requests_is_taken(on_cpu):
    c = small_cache(n_requests=4096, n_pages=1)
    with pytest.raises(Launched, match="ss_block_tables"):
        c.step([0] * 4096)


@pytest.mark.parametrize("big", [1 << 62, (1 << 62) + 1, (1 << 60) + 3, (1 << 63) - 1, 1 << 32])
def test_counts_whose_products_pass_64_bits_are_refused(big):
    """Products of two sizes that come out small, or negative, in 64 bits."""
    lib = _hip.load_library()
    st = store(n_pages=big)
    at = ctypes.addressof(st)
    assert lib.ss_read_paged(at, FAKE, 1, FAKE, FAKE, None) == -2
    assert lib.ss_append_paged(at, FAKE, FAKE, 1, 1, 256, 128, 256, 128, FAKE, None) == -2
    assert attention(st) == -2

    def tables(r=2, width=4, pool=8, n=3):
        return lib.ss_block_tables(FAKE, FAKE, r, FAKE, width, FAKE, pool, FAKE, 64, n, FAKE, FAKE, FAKE, FAKE, None,
                                   FAKE, None)

    assert tables(pool=big) == tables(width=big) == tables(r=4096, width=big) == tables(n=big) == -2
    st = store()
    at = ctypes.addressof(st)
    assert lib.ss_append_paged(at, FAKE, FAKE, 1, big, 256, 128, 256, 128, FAKE, None) == -2
    assert lib.ss_read_paged(at, FAKE, big, FAKE, FAKE, None) == -2
    assert attention(n=big) == attention(width=big) == -2
    assert attention(max_new=big) == attention(max_length=big) == -1
    for n in (big, -big, -1):
        assert lib.ss_paged_attn_workspace_bytes(at, n, 1, 2, 1, 100000) == 0


@pytest.mark.parametrize("heads", [1, 3, 8])
def test_more_threads_than_a_launch_counts_are_refused(heads):
    """2^32 threads: 8 of a wave's tokens and a head each in appends, 8 dims of
    a token and a head in reads."""
    lib = _hip.load_library()
    for d, read in ((128, 2 ** 28), (64, 2 ** 29)):
        st = store(n_kv_heads=heads, head_dim=d)
        at = ctypes.addressof(st)
        for n in (-(-2 ** 29 // heads), 2 ** 31 - 1):
            assert lib.ss_append_paged(at, FAKE, FAKE, 1, n, 256, 128, 256, 128, FAKE, None) == -2
        for n in (-(-read // heads), 2 ** 31 // heads, 2 ** 31 - 1):
            assert lib.ss_read_paged(at, FAKE, n, FAKE, FAKE, None) == -2
        assert b"too many" in lib.ss_last_error()


def test_a_cache_says_whether_it_is_empty(on_cpu, monkeypatch):
    """As the other caches do; with lengths that the host knows or not."""
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c = small_cache()
    assert c.empty()
    c.step([0, 2])
    assert not c.empty()
    c.release([1])
    assert c.empty()
    c.step(ints(1, 0), 1)  # (nothing runs here: the lengths on the device are still 0)
    assert c.empty()
    c.lengths[1] = 3
    assert not c.empty()


def test_the_bound_follows_what_tensor_steps_may_add(on_cpu, monkeypatch):
    """Lengths given on the GPU are held to a table row's whole pages, which
    may pass max_tokens; launches are sized for as many."""
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    for captured, bounds in ((False, (90, 128, 128)), (True, (128, 128, 128))):
        monkeypatch.setattr(paged, "_capturing", lambda t: captured)
        c = small_cache()  # (100 tokens, pages of 32)
        for bound in bounds:
            c.step(ints(90, 1), 91, max_new=90)
            assert c._bound == bound
    monkeypatch.setattr(paged, "_capturing", lambda t: False)
    with pytest.raises(ValueError, match="within 0 .. 100"):
        small_cache().step([101, 0])


def test_a_plan_that_a_graph_reads_stays(on_cpu, monkeypatch):
    """append and attend captured after an eager step read its plan at every
    replay: its memory is not given back when the next step replaces it."""
    import weakref

    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    c = small_cache()
    z, q = torch.zeros(2, 2, 128), torch.zeros(2, 4, 128, dtype=torch.float16)

    def slots_after(captured):
        c.step([1, 1])
        monkeypatch.setattr(paged, "_capturing", lambda t: captured)
        c.append(z, z)
        c.attend(q, 0.1)
        c.attend(q, 0.1)
        monkeypatch.setattr(paged, "_capturing", lambda t: False)
        slots = weakref.ref(c.plan.slots)
        c.step([1, 1])
        return slots()

    assert slots_after(False) is None
    assert slots_after(True) is not None and len(c._kept) == 1
    with pytest.raises(RuntimeError, match="attend needs a step"):
        small_cache().attend(q, 0.1)
