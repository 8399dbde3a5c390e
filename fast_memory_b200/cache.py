"""A paged cache of recent keys and values: where a serving process keeps the context that is not (yet) in a memory.

    cache = PagedCache(n_heads=8, d=128, n_pages=4096, n_seqs=64, max_len=16384)
    cache.append(seqs, k_new, v_new, cu_new)                   # k_new, v_new [H, T, d]: the new tokens of some sequences
    o, lse = cache.attend(q, sm_scale, seqs=seqs, cu_seqlens_q=cu_new, window=4096)
    out, lse = merge(o, lse, *mem.query(q, sm_scale))          # with what the memory of older keys answers
    k, v = cache.gather([s], [0, n])                           # keys and values of a sequence, e.g. for Memory.build
    cache.fork(parents, children); cache.free(done); cache.compact()

Pages are shared by reference count; which page a call takes is decided on the device (the lowest free ones), so no call reads
anything back and every call can be captured into a CUDA graph.  A call that cannot be served - too few free pages, a sequence
named twice or out of range, a sequence that would outgrow its table, a fork into a sequence with tokens - changes nothing and
sets a bit that :meth:`PagedCache.check` raises for.  Calls on one cache belong on one stream; host threads may share it.
"""
from __future__ import annotations

import threading
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib as L
from .local import _PRE, _compiling, _included, _int32, _modes, _on, _prefix_sums, _rows, _scratch, _stream, paged_attention

Seqs = Union[torch.Tensor, Sequence[int]]
_capturing = torch._C._cuda_isCurrentStreamCapturing

_STATUS = {1: "a sequence is out of range or named twice, or prefix sums do not rise", 2: "too few free pages",
           4: "a sequence would outgrow its row of the page table", 8: "a fork into a sequence that holds tokens"}


class PagedCache:
    def __init__(self, n_heads: int, d: int, *, n_pages: int, n_seqs: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda"):
        """An empty cache: ``n_pages`` pages of ``page_size`` tokens for ``n_seqs`` sequences of up to ``max_len`` tokens."""
        if torch.device(device).type != "cuda":
            raise L.FastMemError("fast_memory_b200 ops run on CUDA tensors only (there is no CPU path)")
        if page_size <= 0 or n_pages <= 0 or n_seqs <= 0 or max_len <= 0:
            raise ValueError("page_size, n_pages, n_seqs and max_len must be positive")
        pool = (n_pages, n_heads, page_size, d)
        self._init(torch.zeros(pool, dtype=dtype, device=device), torch.zeros(pool, dtype=dtype, device=device),
                   torch.full((n_seqs, -(-max_len // page_size)), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device), torch.zeros(n_pages, dtype=torch.int32, device=device), None)

    @classmethod
    def over(cls, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor,
             status: Optional[torch.Tensor] = None) -> "PagedCache":
        """A cache over tensors the caller holds: pools ``[n_pages, H, page_size, d]``, int32 ``page_table [n_seqs, width]`` (-1
        behind a sequence's last page), ``lengths [n_seqs]``, ``refcounts [n_pages]`` (0 = free; a page that is not full has
        one owner) and optionally the status word ``[1]``."""
        self = cls.__new__(cls)
        self._init(k_pages, v_pages, page_table, lengths, refcounts, status)
        return self

    def _init(self, k_pages, v_pages, page_table, lengths, refcounts, status):
        dev = L.require_cuda(k_pages, v_pages, page_table, lengths, refcounts, status)
        shape = k_pages.shape
        if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != k_pages.dtype:
            raise ValueError("k_pages and v_pages must be [n_pages, n_heads, page_size, d] with equal shapes and dtypes")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=dev)
        i32 = torch.int32
        if page_table.dtype is not i32 or lengths.dtype is not i32 or refcounts.dtype is not i32 or status.dtype is not i32:
            raise TypeError("page_table, lengths, refcounts and status must be int32")
        if page_table.dim() != 2 or lengths.shape != page_table.shape[:1] or refcounts.shape != shape[:1] or status.numel() != 1:
            raise ValueError("page_table [n_seqs, width], lengths [n_seqs], refcounts [n_pages] and status [1] are needed")
        if not (k_pages.is_contiguous() and v_pages.is_contiguous() and page_table.is_contiguous() and lengths.is_contiguous() and
                refcounts.is_contiguous()):
            raise ValueError("the tensors of a cache must be contiguous")
        self.k_pages, self.v_pages, self.page_table, self.lengths, self.refcounts, self.status = \
            k_pages, v_pages, page_table, lengths, refcounts, status
        self.n_pages, self.n_heads, self.page_size, self.d = shape
        self.n_seqs, width = page_table.shape
        self.device = dev
        self._ref = L.pack_page_cache_args(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), refcounts.data_ptr(),
                                           status.data_ptr(), self.n_pages, width, L.dtype_id(k_pages.dtype), self.d, self.n_heads,
                                           self.page_size, self.n_seqs)
        self._ws = {}
        self._lock = threading.Lock()

    def _run(self, call, *args) -> None:
        """One page operation on the current stream.  Operations on a cache follow one another, so they share a
        scratch buffer (one a stream); a captured one gets its own, which lives as long as its graph.  An operation is a plan and
        a copy that reads it: two host threads enqueue theirs one after the other."""
        if not _compiling() and (_modes() or _included(_PRE)):
            self._refuse_tracing()
        dev, lib = self.device, L.lib()
        with self._lock, _on(dev):
            stream = _stream(dev)
            ws = self._ws.get(stream)
            if ws is None or _capturing():
                ws = _scratch(lib.fm_page_cache_workspace_bytes(self._ref, self.n_seqs), dev)
                if not _capturing():
                    self._ws[stream] = ws
            status = call(self._ref, *args, ws.data_ptr(), ws.numel(), stream)
        if status:
            L.check(status, call.__name__)

    @staticmethod
    def _refuse_tracing() -> None:
        """A traced graph would hold nothing of a call that goes straight to the library.  (Called where a mode is active at all.)"""
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if get_proxy_mode() is not None:
            raise L.FastMemError("page operations change the cache in place and cannot be traced")

    def _seqs(self, seqs: Seqs, name: str = "seqs") -> torch.Tensor:
        t = _int32(seqs, self.device, name)
        if t.numel() > self.n_seqs:
            raise ValueError(f"{name}: {t.numel()} entries for {self.n_seqs} sequences")
        return t

    def check(self) -> None:
        """Raise if a call since the last check could not be served (synchronises with the device)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise L.FastMemError("paged cache: " + "; ".join(text for bit, text in _STATUS.items() if bits & bit))

    # ---- page operations ---------------------------------------------------------------------------
    def append(self, seqs: Seqs, k_new: torch.Tensor, v_new: torch.Tensor, cu_new: Optional[Seqs] = None) -> None:
        """Sequence ``seqs[i]`` grows by rows ``cu_new[i]:cu_new[i+1]`` (left out: row i) of ``k_new`` / ``v_new [H, T, d]``."""
        dev = L.require_cuda(self.k_pages, k_new, v_new)
        if k_new.dim() != 3 or v_new.shape != k_new.shape or k_new.shape[0] != self.n_heads or k_new.shape[2] != self.d:
            raise ValueError(f"k_new and v_new must be [{self.n_heads}, T, {self.d}], got {tuple(k_new.shape)} {tuple(v_new.shape)}")
        if not (k_new.dtype == v_new.dtype == self.k_pages.dtype):
            raise TypeError("k_new and v_new must be in the cache's dtype")
        seqs = self._seqs(seqs)
        cu = _prefix_sums(cu_new, dev, "cu_new", k_new.shape[1])
        if (k_new.shape[1] if cu is None else cu.numel() - 1) != seqs.numel():
            raise ValueError("cu_new must have one entry per sequence plus one (left out: one token per sequence)")
        k_new, v_new = _rows(k_new), _rows(v_new)
        (kh, kt, _), (vh, vt, _) = k_new.stride(), v_new.stride()
        self._run(L.lib().fm_cache_append, seqs.data_ptr(), seqs.numel(), L.ptr(cu), k_new.data_ptr(), v_new.data_ptr(), k_new.shape[1],
                  kh, kt, vh, vt)

    def fork(self, parents: Seqs, children: Seqs) -> None:
        """The empty sequence ``children[i]`` becomes a copy of ``parents[i]``: full pages are shared, the rows of a last page
        that is not full are copied.  A parent may have several children."""
        parents, children = _int32(parents, self.device, "parents"), self._seqs(children, "children")
        if parents.numel() != children.numel():
            raise ValueError("parents and children must pair up")
        self._run(L.lib().fm_cache_fork, parents.data_ptr(), children.data_ptr(), children.numel())

    def free(self, seqs: Seqs) -> None:
        """Empty these sequences; pages that no other sequence shares become free."""
        seqs = self._seqs(seqs)
        self._run(L.lib().fm_cache_free, seqs.data_ptr(), seqs.numel())

    def compact(self) -> None:
        """Move the used pages to the low end of the pool (the fewest moves that do it); tables follow."""
        self._run(L.lib().fm_cache_compact)

    def copy_pages(self, src: Seqs, dst: Seqs) -> None:
        """Contents of pages ``src[i]`` to ``dst[i]`` (keys and values), tables untouched.  ``dst`` names no page twice and none
        of ``src``."""
        src, dst = _int32(src, self.device, "src"), _int32(dst, self.device, "dst")
        if src.numel() != dst.numel():
            raise ValueError("src and dst must pair up")
        if not _compiling() and (_modes() or _included(_PRE)):
            self._refuse_tracing()
        with _on(self.device):
            L.check(L.lib().fm_cache_copy_pages(self._ref, src.data_ptr(), dst.data_ptr(), src.numel(), _stream(self.device)),
                    "fm_cache_copy_pages")

    def gather(self, seqs: Seqs, cu: Seqs, starts: Optional[Seqs] = None, n_tokens: Optional[int] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Packed keys and values ``[H, T, d]``: rows ``cu[i]:cu[i+1]`` are tokens ``starts[i] ...`` (left out: 0) of sequence
        ``seqs[i]``; tokens it does not have are zero.  ``n_tokens`` = T is needed where ``cu`` is on the device."""
        if n_tokens is None:
            if isinstance(cu, torch.Tensor):
                raise ValueError("gather: n_tokens is needed with a device cu")
            n_tokens = int(cu[-1])
        seqs = _int32(seqs, self.device, "seqs")
        cu = _prefix_sums(cu, self.device, "cu", n_tokens)
        starts = _int32(starts, self.device, "starts", seqs.numel())
        if cu.numel() != seqs.numel() + 1:
            raise ValueError("cu must have one entry per sequence plus one")
        if not _compiling() and (_modes() or _included(_PRE)):
            self._refuse_tracing()
        k, v = (torch.empty(self.n_heads, n_tokens, self.d, dtype=self.k_pages.dtype, device=self.device) for _ in range(2))
        with _on(self.device):
            L.check(L.lib().fm_cache_gather(self._ref, seqs.data_ptr(), cu.data_ptr(), L.ptr(starts), seqs.numel(), n_tokens, k.data_ptr(),
                                            v.data_ptr(), _stream(self.device)), "fm_cache_gather")
        return k, v

    # ---- attention ---------------------------------------------------------------------------------
    def attend(self, q: torch.Tensor, sm_scale: float, *, seqs: Optional[Seqs] = None, cu_seqlens_q: Optional[Seqs] = None,
               causal: bool = True, window: int = 0, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
               prefix: Optional[Seqs] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """:func:`paged_attention` of the sequences' newest tokens ``q [Hq, T, d]``, which :meth:`append` has already stored."""
        return paged_attention(q, self.k_pages, self.v_pages, self.page_table, self.lengths, sm_scale, seqs=seqs, cu_seqlens_q=cu_seqlens_q,
                               causal=causal, window=window, softcap=softcap, slopes=slopes, prefix=prefix)
