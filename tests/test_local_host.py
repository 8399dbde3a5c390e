"""Refusals of the local attention and page cache entry points that need no GPU: every argument is checked before any CUDA call."""
import contextlib
import ctypes
import threading
import time

import pytest
import torch

import fast_memory_b200 as fm
from fast_memory_b200 import _lib as L
from fast_memory_b200 import cache as cache_module

FAKE = 1 << 20            # an address that is only ever compared with null


def _attn(**kw):
    a = L.LocalAttnArgs(q=FAKE, k=FAKE, v=FAKE, q_stride_head=640, q_stride_row=64, k_stride_head=640, k_stride_row=64, v_stride_head=640,
                        v_stride_row=64, n_q_rows=10, n_k_rows=10, dtype=L.BF16, d=64, n_q_heads=2, n_kv_heads=1, n_docs=1, window=0, causal=1,
                        sm_scale=1.0, softcap=0.0)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


BAD = -1
UNSUPPORTED = -2
WORKSPACE = -3


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=7), BAD, "element type"), (dict(d=48), UNSUPPORTED, "head dim"), (dict(n_q_heads=3, n_kv_heads=2), BAD, "evenly"),
    (dict(n_kv_heads=0), BAD, "evenly"), (dict(n_docs=0), BAD, "document"), (dict(window=-1), BAD, "window"), (dict(softcap=-1.0), BAD, "cap"),
    (dict(n_q_rows=-1), BAD, "row counts"), (dict(n_q_rows=1 << 30), BAD, "row counts"), (dict(n_docs=2), BAD, "cu_q"),
    (dict(n_q_heads=1 << 20, n_q_rows=1 << 20), BAD, "2^31"), (dict(q=None), BAD, "null"), (dict(k=None), BAD, "null"),
    (dict(page_table=FAKE), BAD, "lengths"),
    (dict(page_table=FAKE, lengths=FAKE, n_seqs=1, n_pages=1, page_size=24, page_table_width=1, cu_q=FAKE), UNSUPPORTED, "page size"),
    (dict(page_table=FAKE, lengths=FAKE, n_seqs=1, n_pages=1, page_size=16, page_table_width=1 << 29, cu_q=FAKE), BAD, "too wide"),
    (dict(page_table=FAKE, lengths=FAKE, n_seqs=1, n_pages=1, page_size=16, page_table_width=1), BAD, "one query a sequence"),
])
def test_forward_refuses(kw, status, text):
    lib = L.lib()
    rc = lib.fm_local_attn_fwd(ctypes.byref(_attn(**kw)), FAKE, FAKE, FAKE, 1 << 30, None)
    assert rc == status and text.encode() in lib.fm_last_error(), lib.fm_last_error()


@pytest.mark.parametrize("cap", [float("inf"), float("nan")])
def test_a_cap_that_is_not_finite_is_refused(cap):
    lib = L.lib()
    assert lib.fm_local_attn_fwd(ctypes.byref(_attn(softcap=cap)), FAKE, FAKE, FAKE, 1 << 30, None) == BAD
    assert b"finite" in lib.fm_last_error()


def test_other_refusals():
    lib = L.lib()
    ref = ctypes.byref
    assert lib.fm_local_attn_fwd(None, FAKE, FAKE, FAKE, 1 << 30, None) == BAD
    assert lib.fm_local_attn_fwd(ref(_attn()), None, FAKE, FAKE, 1 << 30, None) == BAD
    assert lib.fm_local_attn_fwd(ref(_attn(n_q_rows=0)), None, None, None, 0, None) == 0            # nothing to do
    assert lib.fm_local_attn_bwd(ref(_attn()), FAKE, FAKE, FAKE, 640, 64, None, FAKE, FAKE, FAKE, FAKE, 8, None) == WORKSPACE
    assert lib.fm_local_attn_bwd(ref(_attn()), FAKE, FAKE, FAKE, 640, 64, None, FAKE, None, FAKE, FAKE, 1 << 30, None) == BAD
    for kw in (dict(n_q_rows=0), dict(n_k_rows=0), dict(n_q_heads=300), dict(n_q_rows=0, n_k_rows=0), dict(d=48), dict(n_kv_heads=0)):
        lib.fm_local_attn_workspace_bytes(ref(_attn(**kw)))                                           # any numbers: a size, no crash
        lib.fm_local_attn_bwd_workspace_bytes(ref(_attn(**kw)))
    assert lib.fm_local_attn_fwd(ref(_attn(q=FAKE + 2)), FAKE, FAKE, FAKE, 1 << 30, None) == BAD
    assert lib.fm_local_attn_fwd(ref(_attn(k_stride_row=60)), FAKE, FAKE, FAKE, 1 << 30, None) == BAD
    paged = _attn(page_table=FAKE, lengths=FAKE, n_seqs=1, n_pages=1, page_size=16, page_table_width=1, cu_q=FAKE)
    assert lib.fm_local_attn_bwd(ref(paged), FAKE, FAKE, FAKE, 640, 64, None, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == UNSUPPORTED


def _cache(**kw):
    a = L.PageCacheArgs(k_pages=FAKE, v_pages=FAKE, page_table=FAKE, lengths=FAKE, refcounts=FAKE, status=FAKE, n_pages=4, width=2,
                        dtype=L.BF16, d=64, n_heads=1, page_size=16, n_seqs=3)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,status,text", [
    (dict(k_pages=None), BAD, "null"), (dict(status=None), BAD, "null"), (dict(dtype=9), BAD, "element type"), (dict(n_pages=0), BAD, "sizes"),
    (dict(page_size=8), UNSUPPORTED, "page size"), (dict(page_size=512), UNSUPPORTED, "page size"), (dict(page_size=0), UNSUPPORTED, "page size"),
    (dict(d=12), UNSUPPORTED, "multiple of 16"), (dict(k_pages=FAKE + 8), BAD, "aligned"), (dict(width=1 << 40), BAD, "wide"),
])
def test_cache_refuses(kw, status, text):
    lib = L.lib()
    c = ctypes.byref(_cache(**kw))
    calls = [lib.fm_cache_append(c, FAKE, 1, FAKE, FAKE, FAKE, 1, 64, 64, 64, 64, FAKE, 1 << 30, None),
             lib.fm_cache_fork(c, FAKE, FAKE, 1, FAKE, 1 << 30, None), lib.fm_cache_free(c, FAKE, 1, FAKE, 1 << 30, None),
             lib.fm_cache_compact(c, FAKE, 1 << 30, None), lib.fm_cache_copy_pages(c, FAKE, FAKE, 1, None),
             lib.fm_cache_gather(c, FAKE, FAKE, None, 1, 1, FAKE, FAKE, None)]
    assert calls == [status] * 6 and text.encode() in lib.fm_last_error(), lib.fm_last_error()


def test_cache_calls_refuse():
    lib = L.lib()
    c = ctypes.byref(_cache())
    need = lib.fm_page_cache_workspace_bytes(c, 2)
    assert lib.fm_cache_append(c, FAKE, 2, FAKE, FAKE, FAKE, 5, 64, 64, 64, 64, FAKE, need - 1, None) == WORKSPACE
    assert lib.fm_cache_append(c, FAKE, 4, FAKE, FAKE, FAKE, 5, 64, 64, 64, 64, FAKE, 1 << 30, None) == BAD      # more than there are
    assert lib.fm_cache_append(c, FAKE, 2, None, FAKE, FAKE, 5, 64, 64, 64, 64, FAKE, need, None) == BAD         # one token each
    assert lib.fm_cache_append(c, FAKE, 2, FAKE, FAKE, FAKE, 5, 64, 60, 64, 64, FAKE, need, None) == BAD         # rows off the 16-byte grid
    assert lib.fm_cache_append(c, FAKE, 0, None, None, None, 0, 64, 64, 64, 64, None, 0, None) == 0
    assert lib.fm_cache_fork(c, FAKE, FAKE, 2, FAKE, need - 1, None) == WORKSPACE
    assert lib.fm_cache_free(c, None, 2, FAKE, need, None) == BAD
    assert lib.fm_cache_free(c, FAKE, 2, FAKE, need - 1, None) == WORKSPACE


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 64)
    with pytest.raises(fm.FastMemError):
        fm.local_attention(q, q, q, 1.0)
    with pytest.raises(fm.FastMemError):
        fm.local_attention_backward(q, q, q, 1.0, q, q[..., 0], q)
    with pytest.raises(fm.FastMemError):
        fm.PagedCache(1, 64, n_pages=2, n_seqs=1, max_len=10, device="cpu")
    with pytest.raises(fm.FastMemError):
        fm.paged_attention(q, q[None], q[None], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0)


def _one_head(dtype=torch.bfloat16, n=3):                 # one head's rows cut from a buffer of odd width: the head stride is the buffer's
    return torch.randn(4, n * 64 + 1).to(dtype)[:, :n * 64].unflatten(1, (n, 64))[:1]


def _one_row(dtype=torch.bfloat16):                       # the first row of one head of a buffer of odd width
    return torch.randn(3, 1, 131).to(dtype)[:, :, :64][:1]


@pytest.mark.parametrize("make", [_one_head, _one_row, lambda: torch.randn(5, 7, 131)[:, :0, :64], lambda: torch.randn(3, 5, 64)[:, :1],
                                  lambda: torch.randn(2, 9, 131)[..., :64], lambda: torch.randn(4, 6, 64).transpose(0, 1), lambda: torch.randn(2, 8, 64)])
def test_rows_have_strides_the_library_takes(make):
    """Any view's rows, whatever the strides of its dims of size one."""
    from fast_memory_b200.local import _rows
    t = make()
    r = _rows(t)
    assert torch.equal(r, t)
    assert all(s * r.element_size() % 16 == 0 for s in r.stride()[:2]) and r.stride(2) == 1


def test_calls_that_pytorch_has_to_see_are_noticed():
    """Under tracing, a dispatch mode or a functorch transform a call must go by way of the registered operator."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    from fast_memory_b200.local import _observed
    x = torch.ones(2, 3)
    saw = []

    def look(t):
        saw.append(_observed(t))
        return t * 2

    look(x)
    look(torch.nn.Parameter(x))
    with torch.no_grad(), torch.device("cpu"):
        look(x)
    assert saw == [False] * 3
    saw.clear()
    make_fx(look)(x)
    make_fx(look, pre_dispatch=True)(x)
    make_fx(look, tracing_mode="fake")(x)
    torch.func.vmap(look)(x)
    torch.func.grad(lambda t: look(t).sum())(x)
    with FlopCounterMode(display=False):
        look(x)
    assert saw == [True] * 6

    class Sub(torch.Tensor):
        pass

    assert _observed(None, x.as_subclass(Sub))


def test_a_forward_mode_derivative_is_refused_not_dropped():
    from torch.autograd import forward_ad
    from fast_memory_b200.local import _refuse_tangents
    x = torch.ones(3)
    with forward_ad.dual_level():
        _refuse_tangents(x, x)                             # inside a level, but no tangent
        with pytest.raises(fm.FastMemError, match="forward-mode"):
            _refuse_tangents(x, forward_ad.make_dual(x, x))

    def f(t):
        _refuse_tangents(t)
        return t

    with pytest.raises(fm.FastMemError, match="forward-mode"):
        torch.func.jvp(f, (x,), (x,))


def _host_cache(monkeypatch):
    """A cache whose operations reach their native call without a device."""
    lib = type("Lib", (), {"fm_page_cache_workspace_bytes": lambda self, *a: 16})()
    cache = fm.PagedCache.__new__(fm.PagedCache)
    cache.device, cache.n_seqs, cache._ws, cache._ref, cache._lock = torch.device("cpu"), 1, {}, b"", threading.Lock()
    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(cache_module, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(cache_module, "_stream", lambda dev: 0)
    monkeypatch.setattr(cache_module, "_capturing", lambda: False)
    return cache


def test_page_operations_of_two_host_threads_do_not_interleave(monkeypatch):
    """An operation enqueues a plan and a copy that share the stream's workspace."""
    cache, marks = _host_cache(monkeypatch), []

    def call(ref, who, ws, nbytes, stream):
        marks.append((who, "plan"))
        time.sleep(0.002)                                  # (a native call lets other threads run)
        marks.append((who, "copy"))

    threads = [threading.Thread(target=lambda who=who: [cache._run(call, who) for _ in range(20)]) for who in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(marks) == 120
    assert all(a[0] == b[0] and (a[1], b[1]) == ("plan", "copy") for a, b in zip(marks[::2], marks[1::2]))


def test_page_operations_refuse_to_be_traced(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    cache, calls = _host_cache(monkeypatch), []

    def f(t):
        cache._run(lambda *a: calls.append(a))
        return t * 2

    f(torch.ones(1))
    with FlopCounterMode(display=False):                   # a mode that only watches
        f(torch.ones(1))
    for kw in ({}, {"pre_dispatch": True}):
        with pytest.raises(fm.FastMemError, match="traced"):
            make_fx(f, **kw)(torch.ones(1))
    assert len(calls) == 2


def test_wide_numbers_do_not_wrap():
    """2^32 + 1 is no name of sequence 1."""
    from fast_memory_b200.local import _int32
    t = _int32(torch.tensor([2 ** 32 + 1, -2 ** 40, 7, -1, 2 ** 31]), torch.device("cpu"), "seqs")
    assert t.dtype is torch.int32 and t.tolist() == [2 ** 31 - 1, -2 ** 31, 7, -1, 2 ** 31 - 1]
