"""Operators of a serving step beside the persistent kernel: K/V rows into a paged cache,
attention of one new token per request over it, log probabilities of given tokens.

The persistent kernel does the first two inside its attention task (paged_attention_layer) and
samples greedily; these calls are for the host around it: a prompt that another engine ran is
handed over with PagedKVCache.append (llama.enter_cached_prompts), a step whose layers the host
runs itself attends with PagedKVCache.decode, and token_logprobs turns logits, the persistent
kernel's own among them (PersistentKernel.token_logprobs), into what a serving API answers with.

They work on the same cache layout and request tables as PersistentKernel, need no handle, are
enqueued on the current stream of the tensors' device, wait for nothing, keep nothing from one
call for the next and can be captured into a CUDA graph.  There is no CPU execution path and no
gradient.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _native as N

_DTYPE = {torch.bfloat16: N.BF16, torch.float16: N.F16}
_binding = None


def _load():
    """The native binding of the calls below (csrc/serving_binding.cpp).  Raises if it is missing."""
    global _binding
    if _binding is None:
        N.load()
        try:
            from . import _serving
        except ImportError as e:
            raise ImportError("yirage_b200/_serving.so is missing or does not load: build it with "
                              f"`python -m yirage_b200.build` (there is no fallback implementation): {e}") from e
        _binding = _serving
    return _binding


def _table(meta, key, n, device):
    t = meta.get(key)
    if t is None:
        raise ValueError(f"meta tensor '{key}' is missing")
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise TypeError(f"meta tensor '{key}' must be a contiguous int32 vector")
    if t.device != device:
        raise ValueError(f"meta tensor '{key}' is on {t.device}, the cache on {device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"meta tensor '{key}' has {t.shape[0]} entries, {n} wanted")
    return t


class PagedKVCache:
    """One layer's paged K/V cache with the tables of the requests in it.

    k_cache, v_cache: [pages, page_size, kv_heads, head_dim], bf16 or fp16, equal strides,
    head_dim contiguous (64, 128 or 256); the layout PersistentKernel.paged_attention_layer
    takes, by any strides that keep rows on 16-byte boundaries.
    meta_tensors: PersistentKernel's dictionary; paged_kv_indptr_buffer [requests + 1],
    paged_kv_indices_buffer and paged_kv_last_page_len_buffer [requests] are read by every
    call, qo_indptr_buffer [requests + 1] by append().  Request r is (its pages - 1) *
    page_size + last_page_len[r] tokens long, new tokens included; no pages: an empty slot.
    The tables' contents may change between calls (and between replays of a graph); the
    tensors themselves stay the caller's, are kept alive by this object and must stay where they
    are: a cache whose memory was exchanged since (resize_, set_) is refused.

    Broken table entries never become addresses: their tokens are left out and a bit is set in
    `status` (int32 [1] on the device), which check() reads."""

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, meta_tensors: dict):
        if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
            raise ValueError("k_cache and v_cache must both be [pages, page_size, kv_heads, head_dim]")
        if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("k_cache and v_cache must both be bfloat16 or float16")
        if k_cache.device != v_cache.device:
            raise ValueError("k_cache and v_cache are on different devices")
        if k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
            raise ValueError("k_cache and v_cache must have the same strides, head_dim contiguous")
        dev = k_cache.device
        last = _table(meta_tensors, "paged_kv_last_page_len_buffer", None, dev)
        requests = last.shape[0]
        indptr = _table(meta_tensors, "paged_kv_indptr_buffer", requests + 1, dev)
        indices = _table(meta_tensors, "paged_kv_indices_buffer", None, dev)
        qo = meta_tensors.get("qo_indptr_buffer")
        if qo is not None:
            qo = _table(meta_tensors, "qo_indptr_buffer", requests + 1, dev)
        self.k_cache, self.v_cache = k_cache, v_cache
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.num_requests = requests
        self._tables = (indptr, indices, last, qo)
        pages, page_size, heads, dim = k_cache.shape
        s = k_cache.stride()
        # a stride over a dimension of one entry is never used: give a valid one
        self._c = N.PagedCache(
            k_cache.data_ptr(), v_cache.data_ptr(), s[0] if pages > 1 else 0, s[1] if page_size > 1 else 0,
            s[2] if heads > 1 else 0, indptr.data_ptr(), indices.data_ptr(), last.data_ptr(),
            qo.data_ptr() if qo is not None else None, self.status.data_ptr(), _DTYPE[k_cache.dtype],
            pages, page_size, heads, dim, requests, indices.shape[0])
        self._at = C.addressof(self._c)
        self._index = dev.index if dev.type == "cuda" else -1
        self._lib = _load()

    def append(self, k: torch.Tensor, v: torch.Tensor, *, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
        """Write the new tokens' rows k, v [tokens, kv_heads, head_dim] to their places: rows
        [qo_indptr[r], qo_indptr[r + 1]) are the last tokens of request r.  On the way k, and q
        ([tokens, heads, dim] or [tokens, kv_heads, group, dim]) if given, are RMS-normalised
        (k_norm / q_norm [head_dim], eps) and rotated by halves with the rows of cos / sin
        [positions, rot] (the cache's type or float32; rot <= head_dim, a multiple of 16) at
        their positions: 32-bit arithmetic, one rounding.  Any strides that keep rows on
        16-byte boundaries.  Returns the rotated q (`q_out`, which may be q itself, or a new
        tensor); its rows behind qo_indptr[requests] are not written."""
        return self._lib.paged_append(self._at, self._index, self.k_cache, self.v_cache, k, v, q, q_out, cos, sin,
                                      q_norm, k_norm, eps)

    def decode(self, q: torch.Tensor, *, out: Optional[torch.Tensor] = None, return_lse: bool = False,
               sm_scale: Optional[float] = None, window: int = 0):
        """Attention of one new token per request: row r of q ([rows, heads, dim] or [rows,
        kv_heads, group, dim], rows <= requests) against all cached positions of request r, or
        the last `window` of them.  Returns out (shaped like q, not sharing memory with it), or
        (out, lse [rows, heads] float32) with lse = ln sum_p exp(sm_scale q.k_p); sm_scale
        defaults to head_dim ** -0.5.  A request without positions gives zeros and -inf; an
        infinity in V of a seen position is one in that dimension of out."""
        return self._lib.paged_decode(self._at, self._index, self.k_cache, self.v_cache, q, out, return_lse, sm_scale,
                                      window)

    def check(self):
        """Wait for the work enqueued so far on the current stream and raise if a call found a
        broken table entry since the last check.  The bits are taken in one step: what a call on
        another stream finds meanwhile is left for the next check."""
        if self._index < 0:
            return
        with torch.cuda.device(self._index):
            taken = torch.empty_like(self.status)
            N.check(None, N.load().ypk_paged_status(C.byref(self._c), C.c_void_p(taken.data_ptr()),
                                                    C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        bits = int(taken.item())
        if not bits:
            return
        what = [text for bit, text in ((N.PAGED_BAD_TABLE, "page offsets or a last page length out of order"),
                                       (N.PAGED_BAD_PAGE, "a page number outside the pool"),
                                       (N.PAGED_BAD_POSITION, "a position outside the rotary tables"),
                                       (N.PAGED_BAD_LENGTH, "more new tokens than a request is long")) if bits & bit]
        raise N.YpkError(N.ERR_INVALID, "paged K/V cache: " + "; ".join(what))


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; the four share one allocation."""
    logprob: torch.Tensor                    # [rows] float32
    entropy: torch.Tensor                    # [rows] float32, nats
    top_logprob: Optional[torch.Tensor]      # [rows, top_k] float32, falling (None: top_k = 0)
    top_token: Optional[torch.Tensor]        # [rows, top_k] int64, the lower id first on ties


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0,
                   valid_cols: Optional[int] = None) -> TokenLogprobs:
    """Log probability of tokens[r] under softmax(logits[r, :valid_cols]), the entropy of that
    distribution and its top_k (0..32) most probable tokens.  logits: [rows, columns] bf16, fp16
    or fp32, rows contiguous, any row stride; columns from valid_cols on (the padding of an
    lm_head) are not looked at.  32-bit arithmetic in one pass over the logits.  A token
    outside [0, valid_cols) and a column of -inf have log probability -inf; a row with a NaN or
    +inf gives NaN."""
    return TokenLogprobs._make((_binding or _load()).token_logprobs(logits, tokens, top_k, valid_cols))
