"""Local attention: the near context whose (O, LSE) a memory's result is merged with.

The reference calls it ``attention_forward`` (mem:302) and does not ship it.  Two forms of one operator:

  * :func:`local_attention` over packed documents, with :func:`local_attention_backward` and autograd,
  * :func:`paged_attention` of new tokens (one or a chunk a sequence) over the pages of a cache.

For query i of a document with n_q queries and n_k keys, at position p = n_k - n_q + i::

    s = sm_scale q.k;   softcap > 0: s = softcap tanh(s / softcap);   slopes: s -= slopes[head] |p - j|
    key j is visible iff   j < prefix[document]   or   p - window < j <= p   (causal)   /   |p - j| < window   (not causal)
    lse = log sum e^s (fp32, natural log),   o = sum e^(s - lse) v;   a query that sees nothing: o = 0, lse = -inf

so ``merge(o, lse, *memory.query(q, sm_scale))`` is the attention over both.  Everything runs in the CUDA library on the current
stream; nothing is read back, so every call can be captured into a CUDA graph.  A hidden key or value takes no part whatever it
holds (NaN included).
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib as L

Prefix = Union[torch.Tensor, Sequence[int]]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [heads, rows, d] itself if its rows are contiguous, start on 16-byte boundaries and do not overlap, else a copy."""
    sh, st, sd = t.stride()
    if t.is_contiguous() and t.data_ptr() % 16 == 0:             # (a row is a multiple of 16 bytes)
        if not (sh | st) & 7:
            return t
        # contiguous says nothing of the stride of a dim of size one, or of an empty tensor's
        _, n, d = t.shape
        return t.as_strided(t.shape, (n * d, d, 1))
    e = t.element_size()
    d = t.shape[2]
    ok = sd == 1 and (st * e) % 16 == 0 and (sh * e) % 16 == 0 and t.data_ptr() % 16 == 0 and \
        (t.shape[1] == 1 or st >= d) and (t.shape[0] == 1 or sh >= d)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _int32(values: Optional[Prefix], dev: torch.device, name: str, count: Optional[int] = None) -> Optional[torch.Tensor]:
    """A device int32 array from a tensor or a python sequence."""
    if values is None:
        return None
    if isinstance(values, torch.Tensor):
        if values.dtype is torch.int32 and values.dim() == 1 and values.device == dev and values.is_contiguous() and \
                (count is None or values.numel() == count):
            return values                                     # the usual case
        if values.dim() != 1 or values.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name} must be a 1-d int32 or int64 tensor")
        if values.device != dev:
            raise ValueError(f"{name} is on {values.device}, the tensors are on {dev}")
        if values.dtype is torch.int64:                           # a number out of range stays one
            values = values.clamp(-2 ** 31, 2 ** 31 - 1)
        t = values.to(torch.int32).contiguous()
    else:
        t = torch.tensor([int(x) for x in values], dtype=torch.int32, device=dev)
    if count is not None and t.numel() != count:
        raise ValueError(f"{name}: expected {count} entries, got {t.numel()}")
    return t


def _prefix_sums(values: Optional[Prefix], dev: torch.device, name: str, total: int) -> Optional[torch.Tensor]:
    if values is not None and not isinstance(values, torch.Tensor):
        v = [int(x) for x in values]
        if len(v) < 2 or v[0] != 0 or v[-1] > total or any(b < a for a, b in zip(v, v[1:])):
            raise ValueError(f"{name} must rise from 0 to at most {total}")
    t = _int32(values, dev, name)
    if t is not None and t.numel() < 2:
        raise ValueError(f"{name} needs at least two entries")
    return t


def _slopes(slopes: Optional[torch.Tensor], Hq: int, dev: torch.device) -> Optional[torch.Tensor]:
    if slopes is None:
        return None
    if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or slopes.shape != (Hq,):
        raise TypeError(f"slopes must be a float32 tensor [{Hq}], one a query head")
    if slopes.device != dev:
        raise ValueError(f"slopes are on {slopes.device}, the tensors are on {dev}")
    if slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("slopes are constants: no gradient flows to them")
    return slopes.contiguous()


def _check_options(window: int, softcap: float) -> None:
    if int(window) != window or not 0 <= window < 2 ** 30:
        raise ValueError(f"window must be a whole number of keys (0: no bound), got {window}")
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"softcap must be finite and not negative (0: no cap), got {softcap}")


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.device:
    dev = L.require_cuda(q, k, v)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"q [Hq, S, d], k and v [H, N, d] are needed, got {tuple(q.shape)} {tuple(k.shape)} {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v must share a dtype")
    if k.shape[0] == 0 or q.shape[0] == 0 or q.shape[0] % k.shape[0]:
        raise ValueError(f"{q.shape[0]} query heads do not share {k.shape[0]} KV heads evenly")
    if q.shape[2] not in (16, 32, 64, 128, 256):
        raise L.FastMemError(f"local attention: head dim {q.shape[2]} (16, 32, 64, 128 and 256 are built)")
    return dev


_PRE = torch._C.DispatchKey.PreDispatch
_included, _modes = torch._C._dispatch_tls_is_dispatch_key_included, torch._C._len_torch_dispatch_stack
_layers, _compiling = torch._C._functorch.get_dynamic_layer_stack_depth, torch.compiler.is_compiling
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _observed(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether PyTorch has to see this call as an operator: it is traced, watched by a mode or transformed (a call that goes straight to
    the library would leave no mark there), or the tensors are not plain ones.  (0.5 us)"""
    if _compiling() or _modes() or _layers() or _included(_PRE):
        return True
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return True
    return False


def _refuse_tangents(*tensors: torch.Tensor) -> None:
    """No silent loss of a forward-mode derivative: a registered operator without one drops the tangent too."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise L.FastMemError("local attention has no forward-mode derivative (backward-mode gradients only)")


_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """Kernels launch on the tensors' device whatever the current one is."""
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _doc_args(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix) -> bytes:
    """``fm_local_attn_args`` of a call over documents."""
    (qh, qs, _), (kh, ks, _), (vh, vs, _) = q.stride(), k.stride(), v.stride()
    Hq, S, d = q.shape
    H, N, _ = k.shape
    return L.pack_local_attn_args(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qh, qs, kh, ks, vh, vs, S, N, L.dtype_id(q.dtype), d, Hq, H,
        1 if cu_q is None else cu_q.numel() - 1, int(window), 1 if causal else 0, float(sm_scale), float(softcap), L.ptr(cu_q), L.ptr(cu_k),
        L.ptr(prefix), L.ptr(slopes), 0, 0, 0, 0, 0, 0, 0)


def _stream(dev: torch.device) -> int:
    """Handle of the current stream of ``dev`` (the raw form: a tenth of the time of ``torch.cuda.current_stream``)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _scratch(nbytes: int, dev: torch.device) -> Optional[torch.Tensor]:
    """A workspace for one call, or none: a captured graph keeps its own, and no other graph or stream writes it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _forward(args: bytes, q: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    dev = q.device
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(o.size(0), o.size(1), dtype=torch.float32, device=dev)
    lib = L.lib()
    with _on(dev):
        nbytes = lib.fm_local_attn_workspace_bytes(args)
        ws = _scratch(nbytes, dev)
        status = lib.fm_local_attn_fwd(args, o.data_ptr(), lse.data_ptr(), L.ptr(ws), nbytes, _stream(dev))
    if status:
        L.check(status, "fm_local_attn_fwd")
    return o, lse


def _local_fwd(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix):
    q, k, v = _rows(q), _rows(k), _rows(v)
    return _forward(_doc_args(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix), q)


def _local_bwd(q, k, v, out, lse, d_out, d_lse, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix):
    q, k, v, d_out = _rows(q), _rows(k), _rows(v), _rows(d_out)
    if not out.is_contiguous() or out.data_ptr() % 16:
        out = out.clone(memory_format=torch.contiguous_format)
    lse = lse.contiguous()
    d_lse = None if d_lse is None else d_lse.contiguous()
    dev = q.device
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    args = _doc_args(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix)
    lib = L.lib()
    with _on(dev):
        nbytes = lib.fm_local_attn_bwd_workspace_bytes(args)
        ws = _scratch(nbytes, dev)
        status = lib.fm_local_attn_bwd(args, out.data_ptr(), lse.data_ptr(), d_out.data_ptr(), d_out.stride(0), d_out.stride(1),
                                       L.ptr(d_lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), L.ptr(ws), nbytes, _stream(dev))
    if status:
        L.check(status, "fm_local_attn_bwd")
    return dq, dk, dv


def _paged_fwd(q, k_pages, v_pages, page_table, lengths, sm_scale, seqs, cu_q, causal, window, softcap, slopes, prefix):
    q = _rows(q)
    n_pages, H, page, d = k_pages.shape
    args = L.pack_local_attn_args(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), q.stride(0), q.stride(1), 0, 0, 0, 0, q.shape[1], 0, L.dtype_id(q.dtype), d,
        q.shape[0], H, q.shape[1] if cu_q is None else cu_q.numel() - 1, int(window), 1 if causal else 0, float(sm_scale), float(softcap),
        L.ptr(cu_q), 0, L.ptr(prefix), L.ptr(slopes), page_table.data_ptr(), lengths.data_ptr(), L.ptr(seqs), page_table.shape[1], n_pages, page,
        page_table.shape[0])
    return _forward(args, q)


def _check_call(q, k, v, causal, window, softcap, slopes, cu_seqlens_q, cu_seqlens_k, prefix):
    dev = _check_qkv(q, k, v)
    L.dtype_id(q.dtype)
    _check_options(window, softcap)
    if cu_seqlens_q is None and cu_seqlens_k is not None:
        raise ValueError("cu_seqlens_k needs cu_seqlens_q")
    cu_q = _prefix_sums(cu_seqlens_q, dev, "cu_seqlens_q", q.shape[1])
    if cu_q is not None and cu_seqlens_k is None:
        if k.shape[1] != q.shape[1]:
            raise ValueError("queries and keys differ in number: cu_seqlens_k is needed")
        cu_k = cu_q
    else:
        cu_k = _prefix_sums(cu_seqlens_k, dev, "cu_seqlens_k", k.shape[1])
    if cu_q is not None and cu_q.numel() != cu_k.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must name the same documents")
    n_docs = 1 if cu_q is None else cu_q.numel() - 1
    return _slopes(slopes, q.shape[0], dev), cu_q, cu_k, _int32(prefix, dev, "prefix", n_docs)


# ---- registered operators ------------------------------------------------------------------------------------------
@torch.library.custom_op("fast_memory_b200::local_attention", mutates_args=())
def _local_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float, causal: bool, window: int, softcap: float,
                        slopes: Optional[torch.Tensor], cu_q: Optional[torch.Tensor], cu_k: Optional[torch.Tensor],
                        prefix: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The operator behind :func:`local_attention` where gradients or tracing are wanted."""
    return _local_fwd(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix)


@_local_attention_op.register_fake
def _(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.custom_op("fast_memory_b200::local_attention_backward", mutates_args=())
def _local_attention_bwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, d_out: torch.Tensor,
                            d_lse: Optional[torch.Tensor], sm_scale: float, causal: bool, window: int, softcap: float,
                            slopes: Optional[torch.Tensor], cu_q: Optional[torch.Tensor], cu_k: Optional[torch.Tensor],
                            prefix: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _local_bwd(q, k, v, out, lse, d_out, d_lse, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix)


@_local_attention_bwd_op.register_fake
def _(q, k, v, out, lse, d_out, d_lse, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _setup_context(ctx, inputs, output):
    q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix = inputs
    ctx.set_materialize_grads(False)                             # a loss that does not read the LSE makes no gradient of it
    ctx.save_for_backward(q, k, v, *output, slopes, cu_q, cu_k, prefix)
    ctx.how = (sm_scale, causal, window, softcap)


def _backward(ctx, grad_o, grad_lse):
    q, k, v, o, lse, slopes, cu_q, cu_k, prefix = ctx.saved_tensors
    if grad_o is None and grad_lse is None:
        return (None,) * 11
    grad_o = torch.zeros_like(o) if grad_o is None else grad_o
    dq, dk, dv = _local_attention_bwd_op(q, k, v, o, lse, grad_o, grad_lse, *ctx.how, slopes, cu_q, cu_k, prefix)
    return (dq, dk, dv) + (None,) * 8


_local_attention_op.register_autograd(_backward, setup_context=_setup_context)


@torch.library.custom_op("fast_memory_b200::paged_attention", mutates_args=())
def _paged_attention_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        sm_scale: float, seqs: Optional[torch.Tensor], cu_q: Optional[torch.Tensor], causal: bool, window: int, softcap: float,
                        slopes: Optional[torch.Tensor], prefix: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The operator behind :func:`paged_attention` where it is traced or a gradient is wanted: it has none and says so in the backward pass."""
    return _paged_fwd(q, k_pages, v_pages, page_table, lengths, sm_scale, seqs, cu_q, causal, window, softcap, slopes, prefix)


@_paged_attention_op.register_fake
def _(q, k_pages, v_pages, page_table, lengths, sm_scale, seqs, cu_q, causal, window, softcap, slopes, prefix):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


# ---- the functions -------------------------------------------------------------------------------------------------
def local_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float, *, causal: bool = True, window: int = 0,
                    softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, cu_seqlens_q: Optional[Prefix] = None,
                    cu_seqlens_k: Optional[Prefix] = None, prefix: Optional[Prefix] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention over local keys: ``(o [Hq, S, d] in q's dtype, lse [Hq, S] fp32 natural log)``.

    :param q: ``[Hq, S, d]``;  k, v: ``[H, N, d]``, Hq a multiple of H.  Any strides (a view of ``[S, Hq, d]`` activations is
        read as it is; a layout whose rows are not contiguous or not on 16-byte boundaries is copied first)
    :param causal: query at position p sees keys up to p; otherwise both sides
    :param window: keys less than ``window`` positions away only (0: no bound)
    :param softcap: scores are capped smoothly at +-softcap (0: not)
    :param slopes: fp32 ``[Hq]``, distance bias ``-slope |p - j|`` (constants: no gradient)
    :param cu_seqlens_q, cu_seqlens_k: documents packed along S and N (device tensor or python sequence, from 0): a query sees
        keys of its own document only.  ``cu_seqlens_k`` may be left out where both are the same.  The queries are the LAST
        positions of their document's keys.  Rows behind the last document: o = 0, lse = -inf
    :param prefix: per document, the first keys that every query of the document sees

    Differentiable in q, k and v through both results (:func:`local_attention_backward` is the explicit form)."""
    slopes, cu_q, cu_k, prefix = _check_call(q, k, v, causal, window, softcap, slopes, cu_seqlens_q, cu_seqlens_k, prefix)
    _refuse_tangents(q, k, v)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _observed(q, k, v):
        return _local_attention_op(q, k, v, float(sm_scale), bool(causal), int(window), float(softcap), slopes, cu_q, cu_k, prefix)
    return _local_fwd(q, k, v, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix)


def local_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float, out: torch.Tensor, lse: torch.Tensor,
                             d_out: torch.Tensor, *, d_lse: Optional[torch.Tensor] = None, causal: bool = True, window: int = 0,
                             softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, cu_seqlens_q: Optional[Prefix] = None,
                             cu_seqlens_k: Optional[Prefix] = None, prefix: Optional[Prefix] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients ``(dq, dk, dv)`` of :func:`local_attention` in the dtype of q for the output gradient ``d_out``
    ``[Hq, S, d]`` and, where the loss reads the LSE, ``d_lse`` ``[Hq, S]`` fp32.

    ``out`` (q's dtype) and ``lse`` (fp32) are the result the caller ended up with - of this attention alone or merged with a
    memory's, as :meth:`Memory.query_backward` takes them (mem:332, 354-378).  The same call gives the same bits.  The results
    are constants to autograd."""
    slopes, cu_q, cu_k, prefix = _check_call(q, k, v, causal, window, softcap, slopes, cu_seqlens_q, cu_seqlens_k, prefix)
    L.require_cuda(q, out, lse, d_out, d_lse)
    if out.dtype != q.dtype or d_out.dtype != q.dtype:
        raise TypeError("q, k, v, out and d_out must share a dtype")
    if lse.dtype != torch.float32 or (d_lse is not None and d_lse.dtype != torch.float32):
        raise TypeError("lse and d_lse must be float32 (natural log)")
    if out.shape != q.shape or d_out.shape != q.shape or lse.shape != q.shape[:2] or (d_lse is not None and d_lse.shape != lse.shape):
        raise ValueError("out and d_out must be shaped like q, lse and d_lse [Hq, S]")
    _refuse_tangents(q, k, v, out, lse, d_out)
    if _observed(q, k, v, out, lse, d_out, d_lse):
        return _local_attention_bwd_op(q, k, v, out, lse, d_out, d_lse, float(sm_scale), bool(causal), int(window), float(softcap), slopes, cu_q,
                                       cu_k, prefix)
    return _local_bwd(q, k, v, out, lse, d_out, d_lse, sm_scale, causal, window, softcap, slopes, cu_q, cu_k, prefix)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    sm_scale: float, *, seqs: Optional[Prefix] = None, cu_seqlens_q: Optional[Prefix] = None, causal: bool = True,
                    window: int = 0, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, prefix: Optional[Prefix] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of new tokens over a paged cache that already holds them: ``(o [Hq, T, d], lse [Hq, T])``.

    :param q: ``[Hq, T, d]`` the new tokens of all sequences;  ``cu_seqlens_q`` cuts them (left out: one token a sequence)
    :param k_pages, v_pages: ``[n_pages, H, page_size, d]``;  page_table ``[n_seqs, width]`` and lengths ``[n_seqs]`` int32
    :param seqs: which sequence each piece of q belongs to (left out: piece i is sequence i)
    :param prefix: per piece, the first keys that all its tokens see whatever the window

    The other options are those of :func:`local_attention`.  For inference: a backward pass through the result raises."""
    dev = L.require_cuda(q, k_pages, v_pages, page_table, lengths)
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape or q.shape[2] != k_pages.shape[3]:
        raise ValueError(f"q [Hq, T, d] and pages [n_pages, H, page_size, d] are needed, got {tuple(q.shape)} {tuple(k_pages.shape)} "
                         f"{tuple(v_pages.shape)}")
    if not (q.dtype == k_pages.dtype == v_pages.dtype):
        raise TypeError("q and the pages must share a dtype")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32 or page_table.dim() != 2 or lengths.shape != page_table.shape[:1]:
        raise TypeError("page_table [n_seqs, width] and lengths [n_seqs] must be int32")
    H = k_pages.shape[1]
    if H == 0 or q.shape[0] == 0 or q.shape[0] % H:
        raise ValueError(f"{q.shape[0]} query heads do not share {H} KV heads evenly")
    for t in (k_pages, v_pages, page_table, lengths):
        if not t.is_contiguous():
            raise ValueError("the pool, the page table and the lengths must be contiguous")
    _check_options(window, softcap)
    cu_q = _prefix_sums(cu_seqlens_q, dev, "cu_seqlens_q", q.shape[1])
    pieces = q.shape[1] if cu_q is None else cu_q.numel() - 1
    seqs = _int32(seqs, dev, "seqs", pieces)
    if seqs is None and pieces != page_table.shape[0]:
        raise ValueError(f"{pieces} pieces of q for {page_table.shape[0]} sequences: pass seqs")
    slopes, prefix = _slopes(slopes, q.shape[0], dev), _int32(prefix, dev, "prefix", pieces)
    if pieces == 0:
        return torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
    _refuse_tangents(q, k_pages, v_pages)
    if (torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad)) or \
            _observed(q, k_pages, v_pages, page_table, lengths):
        return _paged_attention_op(q, k_pages, v_pages, page_table, lengths, float(sm_scale), seqs, cu_q, bool(causal), int(window),
                                   float(softcap), slopes, prefix)
    return _paged_fwd(q, k_pages, v_pages, page_table, lengths, sm_scale, seqs, cu_q, causal, window, softcap, slopes, prefix)
