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

_DTYPE = {torch.bfloat16: N.BF16, torch.float16: N.F16, torch.float32: N.F32}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _call(device, fn, *args):
    """fn(*args, current stream of `device`) with that device current."""
    if device.type != "cuda":
        raise RuntimeError("the serving operators need tensors on a CUDA device (sm_100a); "
                           "there is no CPU execution path")
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != N.YPK_OK:
        N.check(None, rc)


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
    tensors themselves stay the caller's and are kept alive, unmoved, by this object.

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
        self._heads, self._dim, self._dtype, self._device = heads, dim, k_cache.dtype, dev
        s = k_cache.stride()
        # a stride over a dimension of one entry is never used: give a valid one
        self._c = N.PagedCache(
            k_cache.data_ptr(), v_cache.data_ptr(), s[0] if pages > 1 else 0, s[1] if page_size > 1 else 0,
            s[2] if heads > 1 else 0, indptr.data_ptr(), indices.data_ptr(), last.data_ptr(),
            qo.data_ptr() if qo is not None else None, self.status.data_ptr(), _DTYPE[k_cache.dtype],
            pages, page_size, heads, dim, requests, indices.shape[0])
        self._ref = C.byref(self._c)
        self._lib = N.load()
        self._workspace = {}     # bytes by query heads

    # ------------------------------------------------------------------------ operands
    def _operand(self, t, name):
        if t.dtype != self._dtype:
            raise TypeError(f"{name} is {t.dtype}, the cache {self._dtype}")
        if t.device != self._device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self._device}")

    def _queries(self, t, name, written=False):
        """(rows, heads, stride of a row, of a group, of a head) of [rows, heads, dim] or
        [rows, kv_heads, group, dim]."""
        self._operand(t, name)
        shape, stride = t.shape, t.stride()
        if len(shape) == 3:
            rows, heads, dim = shape
            group = heads // self._heads
            st, sh, sd = stride
            sg = sh * group
            good = heads > 0 and heads % self._heads == 0
        elif len(shape) == 4:
            rows, kv, group, dim = shape
            heads = kv * group
            st, sg, sh, sd = stride
            good = kv == self._heads and group > 0
        else:
            good = False
        if not good or dim != self._dim or sd != 1:
            raise ValueError(f"{name} must be [rows, heads, {self._dim}] or [rows, {self._heads}, group, "
                             f"{self._dim}] with heads a multiple of {self._heads} and a contiguous last dimension")
        if written and ((rows > 1 and st < dim) or (self._heads > 1 and sg < dim) or (group > 1 and sh < dim)):
            raise ValueError(f"{name} is written: its rows must not overlap")
        return rows, heads, st if rows > 1 else 0, sg if self._heads > 1 else 0, sh if group > 1 else 0

    def _rows(self, t, name):
        self._operand(t, name)
        if t.dim() != 3 or t.shape[1] != self._heads or t.shape[2] != self._dim or t.stride(2) != 1:
            raise ValueError(f"{name} must be [tokens, {self._heads}, {self._dim}] with a contiguous last dimension")
        s = t.stride()
        return s[0] if t.shape[0] > 1 else 0, s[1] if self._heads > 1 else 0

    # ------------------------------------------------------------------------ operators
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
        if self._tables[3] is None:
            raise ValueError("append needs the meta tensor 'qo_indptr_buffer'")
        kt, kh = self._rows(k, "k")
        vt, vh = self._rows(v, "v")
        tokens = k.shape[0]
        if v.shape[0] != tokens:
            raise ValueError(f"k has {tokens} rows, v {v.shape[0]}")
        a = N.PagedAppendArgs()
        a.k, a.v, a.num_tokens, a.eps = k.data_ptr(), v.data_ptr(), tokens, eps
        a.k_stride_token, a.k_stride_head, a.v_stride_token, a.v_stride_head = kt, kh, vt, vh
        if q is not None:
            rows, heads, a.q_stride_token, a.q_stride_group, a.q_stride_head = self._queries(q, "q")
            if rows != tokens:
                raise ValueError(f"q has {rows} rows, k {tokens}")
            if q_out is None:
                q_out = torch.empty((tokens, heads, self._dim), dtype=self._dtype, device=self._device)
            rows, oh, a.q_out_stride_token, a.q_out_stride_group, a.q_out_stride_head = \
                self._queries(q_out, "q_out", written=True)
            if rows != tokens or oh != heads:
                raise ValueError("q_out must have the rows and heads of q")
            a.q, a.q_out, a.num_q_heads = q.data_ptr(), q_out.data_ptr(), heads
        elif q_out is not None or q_norm is not None:
            raise ValueError("q_out and q_norm come with q")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if cos is not None:
            if cos.dtype not in (self._dtype, torch.float32) or sin.dtype != cos.dtype:
                raise TypeError("cos and sin must both be of the cache's type or float32")
            if cos.dim() != 2 or cos.shape != sin.shape or cos.stride() != sin.stride() or cos.stride(1) != 1:
                raise ValueError("cos and sin must be [positions, rot] alike, rows contiguous")
            if cos.device != self._device or sin.device != self._device:
                raise ValueError("cos and sin must be on the cache's device")
            a.cos, a.sin, a.table_dtype = cos.data_ptr(), sin.data_ptr(), _DTYPE[cos.dtype]
            a.max_positions, a.rot_dim = cos.shape
            a.table_stride = cos.stride(0) if cos.shape[0] > 1 else (cos.shape[1] + 7) // 8 * 8
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None:
                self._operand(w, name)
                if w.dim() != 1 or w.shape[0] != self._dim or not w.is_contiguous():
                    raise ValueError(f"{name} must be a contiguous vector of {self._dim}")
                setattr(a, name, w.data_ptr())
        _call(self._device, self._lib.ypk_paged_append, self._ref, C.byref(a))
        return q_out

    def decode(self, q: torch.Tensor, *, out: Optional[torch.Tensor] = None, return_lse: bool = False,
               sm_scale: Optional[float] = None, window: int = 0):
        """Attention of one new token per request: row r of q ([rows, heads, dim] or [rows,
        kv_heads, group, dim], rows <= requests) against all cached positions of request r, or
        the last `window` of them.  Returns out (shaped like q), or (out, lse [rows, heads]
        float32) with lse = ln sum_p exp(sm_scale q.k_p); sm_scale defaults to head_dim ** -0.5.
        A request without positions gives zeros and -inf."""
        rows, heads, st, sg, sh = self._queries(q, "q")
        if rows > self.num_requests:
            raise ValueError(f"q has {rows} rows, the tables {self.num_requests} requests")
        if out is None:
            out = torch.empty(q.shape, dtype=self._dtype, device=self._device)
        elif out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        _, _, ot, og, oh = self._queries(out, "out", written=True)
        lse = torch.empty((rows, heads), dtype=torch.float32, device=self._device) if return_lse else None
        size = self._workspace.get(heads)
        if size is None:
            need = C.c_uint64()
            N.check(None, self._lib.ypk_paged_decode_workspace(self._ref, heads, C.byref(need)))
            size = self._workspace[heads] = need.value
        # of this call alone, from the caching allocator: calls on several streams and graphs
        # that replay at the same time never share it
        work = torch.empty(size, dtype=torch.uint8, device=self._device)
        a = N.PagedDecodeArgs(
            q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, work.data_ptr(), size,
            st, sg, sh, ot, og, oh, rows, heads, window, self._dim ** -0.5 if sm_scale is None else sm_scale)
        _call(self._device, self._lib.ypk_paged_decode, self._ref, C.byref(a))
        return (out, lse) if return_lse else out

    def check(self):
        """Wait for the work enqueued so far on the current stream and raise if a call found a
        broken table entry since the last check."""
        bits = int(self.status.item())
        if not bits:
            return
        self.status.zero_()
        what = [text for bit, text in ((N.PAGED_BAD_TABLE, "page offsets or a last page length out of order"),
                                       (N.PAGED_BAD_PAGE, "a page number outside the pool"),
                                       (N.PAGED_BAD_POSITION, "a position outside the rotary tables"),
                                       (N.PAGED_BAD_LENGTH, "more new tokens than a request is long")) if bits & bit]
        raise N.YpkError(N.ERR_INVALID, "paged K/V cache: " + "; ".join(what))


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                    # [rows] float32
    entropy: torch.Tensor                    # [rows] float32, nats
    top_logprob: Optional[torch.Tensor]      # [rows, top_k] float32, falling (None: top_k = 0)
    top_token: Optional[torch.Tensor]        # [rows, top_k] int64, the lower id first on ties


def _logprobs(ptr, dtype, rows, vocab, ld, tokens, top_k, device):
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    entropy = torch.empty(rows, dtype=torch.float32, device=device)
    top_logprob = top_token = None
    if top_k > 0:
        top_logprob = torch.empty((rows, top_k), dtype=torch.float32, device=device)
        top_token = torch.empty((rows, top_k), dtype=torch.int64, device=device)
    _call(device, N.load().ypk_token_logprobs, ptr, dtype, rows, vocab, ld, tokens.data_ptr(), top_k,
          logprob.data_ptr(), entropy.data_ptr(), top_logprob.data_ptr() if top_k > 0 else None,
          top_token.data_ptr() if top_k > 0 else None)
    return TokenLogprobs(logprob, entropy, top_logprob, top_token)


def _check_tokens(tokens, rows, device):
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens must be int64, got {tokens.dtype}")
    if tuple(tokens.shape) not in ((rows,), (rows, 1)) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be a contiguous [{rows}] or [{rows}, 1]")
    if tokens.device != device:
        raise ValueError(f"tokens are on {tokens.device}, the logits on {device}")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0,
                   valid_cols: Optional[int] = None) -> TokenLogprobs:
    """Log probability of tokens[r] under softmax(logits[r, :valid_cols]), the entropy of that
    distribution and its top_k (0..32) most probable tokens.  logits: [rows, columns] bf16, fp16
    or fp32, rows contiguous, any row stride; columns from valid_cols on (the padding of an
    lm_head) are not looked at.  32-bit arithmetic in one pass over the logits.  A token
    outside [0, valid_cols) and a column of -inf have log probability -inf; a row with a NaN or
    +inf gives NaN."""
    if logits.dtype not in _DTYPE:
        raise TypeError(f"logits are {logits.dtype}; bfloat16, float16 or float32 wanted")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, columns] with contiguous rows")
    rows, cols = logits.shape
    vocab = cols if valid_cols is None else int(valid_cols)
    if not 1 <= vocab <= cols:
        raise ValueError(f"valid_cols {vocab} of {cols} columns")
    ld = logits.stride(0) if rows > 1 else cols
    if ld < 0 or (0 <= ld < vocab):
        raise ValueError("rows of logits must not overlap")
    _check_tokens(tokens, rows, logits.device)
    return _logprobs(logits.data_ptr(), _DTYPE[logits.dtype], rows, vocab, ld, tokens, top_k, logits.device)
