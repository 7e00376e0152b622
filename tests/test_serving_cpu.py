"""The serving operators without a GPU: what their host side refuses, through Python and through
the C ABI, and the index arithmetic of the paged cache on good and broken tables."""
import ctypes as C
import os
import shutil
import subprocess
import sys

import pytest
import torch

import yirage_b200 as yr
from yirage_b200 import _native as N
from yirage_b200 import llama

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def meta(requests=2, pages=4):
    i32 = dict(dtype=torch.int32)
    return {"qo_indptr_buffer": torch.tensor([0, 1, 2][:requests + 1], **i32),
            "paged_kv_indptr_buffer": torch.tensor([0, 2, 4][:requests + 1], **i32),
            "paged_kv_indices_buffer": torch.arange(pages, **i32),
            "paged_kv_last_page_len_buffer": torch.tensor([3, 5][:requests], **i32)}


def cache(dtype=torch.bfloat16, heads=2, dim=128, **kw):
    k = torch.zeros(4, 16, heads, dim, dtype=dtype)
    return yr.PagedKVCache(k, k.clone(), kw.get("meta", meta()))


def test_cache_refuses_what_it_cannot_address(native_lib):
    k = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    good = meta()
    with pytest.raises(ValueError, match="must both be"):
        yr.PagedKVCache(k, torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), good)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        yr.PagedKVCache(k.float(), k.float(), good)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        yr.PagedKVCache(k, k.half(), good)
    with pytest.raises(ValueError, match="same strides"):
        yr.PagedKVCache(k, k.transpose(1, 2).contiguous().transpose(1, 2), good)
    with pytest.raises(ValueError, match="same strides"):
        t = torch.zeros(4, 16, 128, 128, dtype=torch.bfloat16).transpose(2, 3)
        yr.PagedKVCache(t, t, good)
    for key in ("paged_kv_indptr_buffer", "paged_kv_indices_buffer", "paged_kv_last_page_len_buffer"):
        with pytest.raises(ValueError, match=f"'{key}' is missing"):
            yr.PagedKVCache(k, k, {a: b for a, b in good.items() if a != key})
        with pytest.raises(TypeError, match="int32"):
            yr.PagedKVCache(k, k, dict(good, **{key: good[key].long()}))
    with pytest.raises(ValueError, match="3 wanted"):
        yr.PagedKVCache(k, k, dict(good, paged_kv_indptr_buffer=torch.zeros(4, dtype=torch.int32)))
    with pytest.raises(TypeError, match="int32 vector"):
        yr.PagedKVCache(k, k, dict(good, paged_kv_indices_buffer=torch.zeros(8, dtype=torch.int32)[::2]))


def test_append_refusals(native_lib):
    c = cache()
    r = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    k, q = r(2, 2, 128), r(2, 8, 128)
    table = r(64, 128)
    for err, what, args in (
            (TypeError, "k is torch.float16", dict(k=k.half())),
            (ValueError, "k must be", dict(k=r(2, 3, 128))),
            (ValueError, "k must be", dict(k=r(2, 2, 64))),
            (ValueError, "v has|v 3", dict(v=r(3, 2, 128))),
            (ValueError, "q has 3 rows", dict(q=r(3, 8, 128))),
            (ValueError, "q must be", dict(q=r(2, 7, 128))),
            (ValueError, "q must be", dict(q=r(2, 4, 2, 128))),
            (ValueError, "rows and heads", dict(q=q, q_out=r(2, 4, 128))),
            (ValueError, "must not overlap", dict(q=q, q_out=r(2, 1, 128).expand(2, 8, 128))),
            (ValueError, "come with q", dict(q_out=q)),
            (ValueError, "come with q", dict(q_norm=r(128))),
            (ValueError, "come together", dict(cos=table)),
            (TypeError, "cos and sin must both", dict(cos=table.half(), sin=table.half())),
            (ValueError, "alike", dict(cos=table, sin=r(32, 128))),
            (ValueError, "k_norm must be", dict(k_norm=r(64))),
            (RuntimeError, "no CPU execution path", dict(q=q, cos=table, sin=table))):
        call = dict(dict(k=k, v=k), **args)
        with pytest.raises(err, match=what):
            c.append(call.pop("k"), call.pop("v"), **call)
    no_rows = cache(meta={a: b for a, b in meta().items() if a != "qo_indptr_buffer"})
    with pytest.raises(ValueError, match="qo_indptr_buffer"):
        no_rows.append(k, k)


def test_decode_and_logprob_refusals(native_lib):
    c = cache()
    r = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    q = r(2, 8, 128)
    for err, what, args, kw in (
            (ValueError, "3 rows, the tables 2", (r(3, 8, 128),), {}),
            (TypeError, "q is torch.float16", (q.half(),), {}),
            (ValueError, "shape of q", (q,), dict(out=r(2, 4, 128))),
            (ValueError, "must not overlap", (q,), dict(out=r(1, 8, 128).expand(2, 8, 128)))):
        with pytest.raises(err, match=what):
            c.decode(*args, **kw)
    x, t = r(4, 100), torch.zeros(4, dtype=torch.int64)
    for err, what, args, kw in (
            (TypeError, "logits are torch.int64", (x.long(), t), {}),
            (ValueError, "contiguous rows", (r(100, 4).t(), t), {}),
            (ValueError, "contiguous rows", (r(400), t), {}),
            (ValueError, "valid_cols 101 of 100", (x, t), dict(valid_cols=101)),
            (ValueError, "valid_cols 0 of 100", (x, t), dict(valid_cols=0)),
            (ValueError, "must not overlap", (r(1, 100).expand(4, 100), t), {}),
            (TypeError, "tokens must be int64", (x, t.int()), {}),
            (ValueError, r"tokens must be a contiguous \[4\]", (x, torch.zeros(5, dtype=torch.int64)), {}),
            (RuntimeError, "no CPU execution path", (x, t), dict(top_k=3))):
        with pytest.raises(err, match=what):
            yr.token_logprobs(*args, **kw)


def c_cache(**kw):
    base = dict(k=0x10000, v=0x20000, stride_page=16 * 256, stride_token=256, stride_head=128, indptr=0x30000,
                indices=0x30000, last_page_len=0x30000, qo_indptr=0x30000, status=None, dtype=N.BF16, num_pages=4,
                page_size=16, num_kv_heads=2, head_dim=128, num_requests=2, num_indices=4)
    return N.PagedCache(**dict(base, **kw))


def test_c_abi_refuses_before_it_enqueues(native_lib):
    """The pointers below point nowhere: a call that got past its checks would show."""
    lib = native_lib
    args = N.PagedAppendArgs(k=0x10000, v=0x10000, k_stride_token=256, k_stride_head=128, v_stride_token=256,
                             v_stride_head=128, num_tokens=2)

    def append(c, code, text, **kw):
        a = N.PagedAppendArgs.from_buffer_copy(args)
        for key, v in kw.items():
            setattr(a, key, v)
        assert lib.ypk_paged_append(C.byref(c), C.byref(a), None) == code
        assert text in lib.ypk_last_error(None).decode(), lib.ypk_last_error(None)

    assert lib.ypk_paged_append(None, C.byref(args), None) == N.ERR_INVALID
    assert lib.ypk_paged_append(C.byref(c_cache()), None, None) == N.ERR_INVALID
    append(c_cache(k=0), N.ERR_INVALID, "null cache")
    append(c_cache(qo_indptr=None), N.ERR_INVALID, "row offsets")
    append(c_cache(dtype=N.F32), N.ERR_UNSUPPORTED, "cache type")
    append(c_cache(head_dim=96), N.ERR_UNSUPPORTED, "head_dim 96")
    append(c_cache(page_size=0), N.ERR_INVALID, "0 tokens")
    append(c_cache(num_requests=4097), N.ERR_UNSUPPORTED, "4097 requests")
    append(c_cache(stride_token=260), N.ERR_INVALID, "16-byte")
    append(c_cache(k=0x10008), N.ERR_INVALID, "16-byte")
    append(c_cache(stride_head=0), N.ERR_INVALID, "overlap")
    append(c_cache(), N.ERR_INVALID, "-1 tokens", num_tokens=-1)
    append(c_cache(), N.ERR_INVALID, "come together", q=0x10000, num_q_heads=8)
    append(c_cache(), N.ERR_INVALID, "7 query heads", q=0x10000, q_out=0x10000, num_q_heads=7)
    append(c_cache(), N.ERR_INVALID, "cos and sin", cos=0x10000)
    table = dict(cos=0x10000, sin=0x10000, table_dtype=N.BF16, max_positions=64, table_stride=128)
    append(c_cache(), N.ERR_UNSUPPORTED, "24 rotated", rot_dim=24, **table)
    append(c_cache(), N.ERR_UNSUPPORTED, "256 rotated", rot_dim=256, **table)
    append(c_cache(), N.ERR_UNSUPPORTED, "table type", rot_dim=128, **dict(table, table_dtype=N.F16))
    append(c_cache(), N.ERR_INVALID, "row stride 64", rot_dim=128, **dict(table, table_stride=64))
    append(c_cache(), N.ERR_INVALID, "not 16-byte aligned", k=0x10002)
    append(c_cache(), N.ERR_INVALID, "16-byte boundaries", k_stride_token=260)
    heads = dict(q=0x10000, num_q_heads=8, q_stride_token=1024, q_stride_group=512, q_stride_head=128,
                 q_out_stride_token=1024, q_out_stride_group=512, q_out_stride_head=128)
    append(c_cache(), N.ERR_INVALID, "q_out overlaps q", q_out=0x10010, **heads)
    append(c_cache(), N.ERR_INVALID, "q_out overlaps q", q_out=0x10000, **dict(heads, q_out_stride_token=2048))
    a = N.PagedAppendArgs.from_buffer_copy(args)
    a.num_tokens = 0
    assert lib.ypk_paged_append(C.byref(c_cache()), C.byref(a), None) == N.YPK_OK     # nothing to do

    def decode(c, code, text, **kw):
        base = dict(q=0x10000, out=0x10000, workspace=0x10000, workspace_bytes=1 << 40, q_stride_token=1024,
                    q_stride_group=512, q_stride_head=128, out_stride_token=1024, out_stride_group=512,
                    out_stride_head=128, rows=2, num_q_heads=8, scale=0.1)
        a = N.PagedDecodeArgs(**dict(base, **kw))
        assert lib.ypk_paged_decode(C.byref(c), C.byref(a), None) == code
        assert text in lib.ypk_last_error(None).decode(), lib.ypk_last_error(None)

    decode(c_cache(), N.ERR_INVALID, "out overlaps q")
    decode(c_cache(), N.ERR_INVALID, "out overlaps q", out=0x10000 + 2 * 2 * 1024 - 16)
    decode(c_cache(), N.ERR_INVALID, "3 rows", rows=3)
    decode(c_cache(), N.ERR_INVALID, "7 query heads", num_q_heads=7)
    decode(c_cache(), N.ERR_INVALID, "window -1", window=-1)
    decode(c_cache(), N.ERR_INVALID, "not finite", scale=float("nan"))
    decode(c_cache(), N.ERR_INVALID, "not finite", scale=float("inf"))
    decode(c_cache(), N.ERR_INVALID, "16-byte", q_stride_head=129)
    decode(c_cache(), N.ERR_INVALID, "not 16-byte aligned", out=0x10002)
    decode(c_cache(), N.ERR_INVALID, "null q", q=None)

    def logprobs(code, text, **kw):
        d = dict(dict(logits=0x10000, dtype=N.BF16, rows=2, vocab=100, ld=104, tokens=0x10000, top=2, lp=0x10000,
                      ent=0x10000, tl=0x10000, tt=0x10000), **kw)
        assert lib.ypk_token_logprobs(d["logits"], d["dtype"], d["rows"], d["vocab"], d["ld"], d["tokens"], d["top"],
                                      d["lp"], d["ent"], d["tl"], d["tt"], None) == code
        assert text in lib.ypk_last_error(None).decode(), lib.ypk_last_error(None)

    logprobs(N.ERR_INVALID, "null", logits=None)
    logprobs(N.ERR_INVALID, "null", ent=None)
    logprobs(N.ERR_UNSUPPORTED, "type 955", dtype=N.I32)
    logprobs(N.ERR_INVALID, "row stride 99", ld=99)
    logprobs(N.ERR_INVALID, "vocabulary 0", vocab=0)
    logprobs(N.ERR_UNSUPPORTED, "top_k 33", top=33)
    logprobs(N.ERR_UNSUPPORTED, "top_k 5", top=5, vocab=4)
    logprobs(N.ERR_INVALID, "top alternatives", tt=None)
    logprobs(N.ERR_INVALID, "not aligned", logits=0x10001)
    assert lib.ypk_token_logprobs(0x10000, N.BF16, 0, 100, 100, 0x10000, 0, 0x10000, 0x10000, None, None, None) == 0


HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "paged_index.h"
using namespace ypk;
static void need(bool ok, const char *what) { if (!ok) { std::printf("%s\n", what); std::exit(1); } }
int main() {
  const int big = 0x7fffffff;
  const int offsets[] = {-big - 1, -5, -1, 0, 1, 2, 3, 7, 8, 9, 100, big};
  const int lasts[] = {-big - 1, -1, 0, 1, 5, 16, 17, big};
  const int sizes[] = {1, 3, 16, 64, 4096, big};
  for (int b : offsets) for (int e : offsets) for (int l : lasts) for (int ps : sizes) for (int n : {0, 1, 8, big}) {
    const PagedRun r = paged_run(b, e, l, ps, n);
    need(r.tokens >= 0, "negative length");
    if (b == e) need(r.tokens == 0 && !r.broken, "empty slot");
    if (r.broken) need(r.tokens == 0, "broken run has a length");
    if (r.tokens == 0) continue;
    // the first and the last position look up page numbers inside the list
    need(r.first >= 0 && r.first < n, "first page number");
    const int64_t last = r.first + (r.tokens - 1) / ps;
    need(last >= r.first && last < n && last < e, "last page number");
    for (int qo : offsets) for (int row : {0, 1, 5, big}) {
      const int64_t p = paged_new_position(r, qo, row);
      need(p < r.tokens, "new position behind the end");
      if (row < qo) need(p == r.tokens - (int64_t(qo) - row), "new position");
      else need(p == -1, "row behind the request");
    }
  }
  // rows: inside the pool, at 64-bit offsets, or refused
  for (int page : offsets) for (int pages : {1, 8, big}) for (int ps : {1, 3, 16, 64, 4096}) for (int pos : {0, 1, 15, 16, 1000, big - 255}) {
    const int q = fast_div(pos, fast_divisor(ps)), in = pos - q * ps;
    need(q == pos / ps && in == pos % ps, "page of a position");
    const int64_t st = 1024, sp = st * ps, row = paged_row(page, pages, in, sp, st);
    if (page < 0 || page >= pages) need(row == -1, "page outside the pool");
    else need(row == page * sp + in * st && row >= 0 && row + st <= int64_t(pages) * sp, "row");
  }
  // division without one: every divisor up to 5000 and some large ones, at and around its multiples
  for (int64_t d = 1; d <= big; d = d < 5000 ? d + 1 : d * 3 + 1)
    for (int64_t m : {int64_t(0), int64_t(1), int64_t(2), int64_t(77), big / d - 1, big / d})
      for (int64_t n = m * d - 1; n <= m * d + 1; ++n)
        if (n >= 0 && n <= big) need(fast_div(int(n), fast_divisor(int(d))) == n / d, "fast_div");
  std::puts("ok");
}
"""


def test_paged_index_arithmetic_on_good_and_broken_tables(tmp_path):
    """csrc/paged_index.h, the functions the kernels take every address from, compiled for the
    host: no table, however broken, leads outside the page list or the pool."""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    src = tmp_path / "walk.cpp"
    src.write_text(HARNESS)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "yirage_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip() == "ok"


def test_cached_prompts_that_cannot_enter_are_refused():
    class Kernel:
        max_num_batched_tokens, max_num_batched_requests, max_num_pages, page_size, max_seq_length = 8, 2, 4, 64, 100
    rows = [torch.zeros(60, 2, 128, dtype=torch.bfloat16)]
    state = {"meta": {"prompt_lengths": torch.tensor([70, 70, 70], dtype=torch.int32),
                      "step": torch.zeros(3, dtype=torch.int32)},
             "k_cache": torch.zeros(1, 4, 64, 2, 128, dtype=torch.bfloat16), "q_heads": 8}
    for steps, what in (([60, 0], "one entry per request"), ([70, 0, 0], "less than its prompt"),
                        ([-1, 0, 0], "less than its prompt"), ([0, 0, 60], "request 1 does not fit"),
                        ([30, 20, 20], "60 rows|70 rows")):
        with pytest.raises(ValueError, match=what):
            llama.enter_cached_prompts(Kernel(), state, steps, rows, rows)
    with pytest.raises(ValueError, match="1 layers"):
        llama.enter_cached_prompts(Kernel(), state, [60, 0, 0], rows * 2, rows)


def small_kernel(vocab, **kw):
    ranks = dict(world_size=kw.get("world_size", 1), rank=kw.get("rank", 0))
    shape = llama.LlamaShape(hidden_size=512, intermediate_size=1024, num_hidden_layers=1, num_attention_heads=8,
                             num_key_value_heads=2, vocab_size=vocab)
    return llama.build_decode_kernel(shape, llama.init_weights(shape, "cpu", 0, **ranks),
                                     tokens=torch.zeros(1, 64, dtype=torch.int64),
                                     prompt_lengths=torch.tensor([5], dtype=torch.int32), max_num_batched_requests=1,
                                     max_num_batched_tokens=8, max_num_pages=1, page_size=64, compile=False, **kw)


def test_log_probabilities_of_a_graph_are_over_what_it_samples_from():
    """The lm_head is padded with zero rows to 4096: their logits are no part of the vocabulary."""
    ypk, state = small_kernel(3000)
    logits = state["tensors"]["argmax_in"]
    assert logits.dim(1) == 4096 and ypk._vocabulary_of(logits) == 3000
    other = state["tensors"]["attn_out"]
    assert ypk._vocabulary_of(other) == other.dim(1)              # nothing samples from it
    with pytest.raises(RuntimeError, match="not compiled"):
        ypk.token_logprobs(logits, 1)


@pytest.mark.parametrize("rank", [0, 1])
def test_log_probabilities_of_a_vocabulary_slice_are_refused(rank):
    """Sampled tokens are ids of the whole vocabulary, the logits this rank's part of it."""
    ypk, state = small_kernel(3000, world_size=2, rank=rank)
    with pytest.raises(ValueError, match="split over the ranks"):
        ypk.token_logprobs(state["tensors"]["argmax_in"], 1)
    whole, state = small_kernel(3000, world_size=2, rank=rank, vocab_parallel=False)
    assert whole._vocabulary_of(state["tensors"]["argmax_in"]) == 3000


def test_operators_read_with_loads_that_stay_behind_their_wait():
    """Kernels of op_launch are there while the one before them still writes their inputs.  A load that
    claims read-only data (.nc, __ldg), or inline assembly that the compiler may move, is not held
    by the wait in front of it."""
    csrc = os.path.join(ROOT, "yirage_b200", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        if not name.startswith("op_"):
            continue
        with open(os.path.join(csrc, name)) as f:
            code = "\n".join(line.split("//")[0] for line in f)
        assert "ld.global.nc" not in code and "__ldg(" not in code and "__ldcs(" not in code, name
        for at in range(len(code)):
            if code.startswith("ld.global", at):
                start, end = code.rfind("asm", 0, at), code.index(";", code.index(')', at))
                assert code.startswith("asm volatile", start) and '"memory"' in code[start:end + 1], (name, code[start:end])
                seen += 1
    assert seen >= 3


def test_forward_mode_tangents_are_refused(native_lib):
    """The operators have no derivative: a tangent would be lost without a word."""
    from torch.autograd import forward_ad
    c = cache()
    k, q = torch.zeros(2, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    x, t = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = lambda a: forward_ad.make_dual(a, torch.ones_like(a))
        for call in (lambda: c.append(dual(k), k), lambda: c.append(k, dual(k)), lambda: c.append(k, k, q=dual(q)),
                     lambda: c.append(k, k, q=q, q_out=dual(q)), lambda: c.append(k, k, k_norm=dual(torch.zeros(128).bfloat16())),
                     lambda: c.decode(dual(q)), lambda: c.decode(q, out=dual(q)), lambda: yr.token_logprobs(dual(x), t),
                     lambda: yr.PagedKVCache(dual(c.k_cache), c.v_cache, meta()).decode(q)):
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call()
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            c.decode(forward_ad.unpack_dual(dual(q)).primal)
    grad = yr.PagedKVCache(c.k_cache.requires_grad_(), c.v_cache, meta())
    with pytest.raises(ValueError, match="k_cache requires a gradient"):
        grad.decode(q)


def test_a_cache_that_has_moved_is_refused(native_lib):
    """Calls go where the cache was when it was described: not after its memory was exchanged."""
    k, q = torch.zeros(2, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    for move in (lambda c: c.k_cache.resize_(400, 16, 2, 128), lambda c: c.v_cache.set_(c.v_cache.clone()),
                 lambda c: setattr(c, "k_cache", c.k_cache.clone())):
        c = cache()
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            c.decode(q)
        move(c)
        for call in (lambda: c.decode(q), lambda: c.append(k, k)):
            with pytest.raises(ValueError, match="not where it was"):
                call()


OVERLAPS = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include "strided_rows.h"
using namespace ypk;
static std::set<int64_t> starts(const StridedRows &r, bool &twice) {
  std::set<int64_t> s;
  for (int64_t i = 0; i < r.count[0]; ++i) for (int64_t j = 0; j < r.count[1]; ++j) for (int64_t k = 0; k < r.count[2]; ++k)
    twice |= !s.insert(r.at + i * r.stride[0] + j * r.stride[1] + k * r.stride[2]).second;
  return s;
}
int main() {
  std::mt19937 g(1);
  const auto pick = [&](int lo, int hi) { return int64_t(lo + g() % (hi - lo + 1)); };
  int met = 0, apart = 0, close = 0, loose = 0;
  for (int turn = 0; turn < 60000; ++turn) {
    StridedRows a = {pick(0, 60), pick(1, 8), {}, {}}, b = a;
    for (int k = 0; k < 3; ++k) {
      a.stride[k] = pick(0, turn % 2 ? 40 : 12);
      a.count[k] = pick(1, 5);
      b.stride[k] = pick(0, 3) ? a.stride[k] : pick(0, 40);
      b.count[k] = pick(0, 3) ? a.count[k] : pick(0, 5);
    }
    b.at = pick(0, 120);
    bool twice = false, unused = false;
    const auto sa = starts(a, twice), sb = starts(b, unused);
    for (auto i = sa.begin(); i != sa.end() && std::next(i) != sa.end(); ++i) twice |= *std::next(i) - *i < a.width;
    bool touch = false;
    for (int64_t x : sa) { const auto i = sb.lower_bound(x - a.width + 1); touch |= i != sb.end() && *i < x + a.width; }
    if (rows_distinct(a) == twice || rows_touch(a, b) != touch || rows_touch(b, a) != touch) {
      std::printf("turn %d: distinct %d, by hand %d; touch %d, by hand %d\n", turn, rows_distinct(a), !twice, rows_touch(a, b), touch);
      return 1;
    }
    (touch ? met : apart)++;
    (twice ? close : loose)++;
  }
  // sizes of a cache and of long prompts: answers without a walk over the rows
  const int64_t tokens = 1 << 20, row = 48 * 128;
  const StridedRows q = {0, 128, {row, 6 * 128, 128}, {tokens, 8, 4}}, k = {4 * 128, 128, {row, 6 * 128, 0}, {tokens, 8, 1}};
  const StridedRows v = {64 * 1024, 128, {2 * 64 * 1024, 1024, 128}, {tokens, 64, 8}};
  StridedRows keys = v;
  keys.at = 0;
  const bool far = rows_distinct(q) && !rows_touch(q, k) && rows_distinct(v) && !rows_touch(keys, v);
  keys.at = 1024;
  std::puts(far && rows_touch(keys, v) && met > 1000 && apart > 1000 && close > 1000 && loose > 1000 ? "ok" : "large");
}
"""


def test_rows_that_overlap_are_told_from_rows_that_do_not(tmp_path):
    """csrc/strided_rows.h against sets of small numbers, in any order and nesting of strides."""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(OVERLAPS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "yirage_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout.strip() == "ok"


def test_written_rows_that_share_memory_are_refused(native_lib):
    """Strides that are wide enough one by one and still lead to the same place twice."""
    c, lib = cache(), native_lib
    r = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    q, k = r(2, 8, 128), r(2, 2, 128)
    for out in (r(4096).as_strided((2, 8, 128), (128, 128, 1)), r(4096).as_strided((2, 8, 128), (256, 128, 1)),
                r(4096).as_strided((2, 2, 4, 128), (1024, 384, 128, 1))):
        with pytest.raises(ValueError, match="must not overlap"):
            c.decode(q.view(out.shape), out=out)
        with pytest.raises(ValueError, match="must not overlap"):
            c.append(k, k, q=q.view(out.shape), q_out=out)
    for out in (r(4096).as_strided((2, 8, 128), (128, 256, 1)), r(9000).as_strided((2, 2, 4, 128), (512, 2048, 128, 1))):
        with pytest.raises(RuntimeError, match="no CPU execution path"):      # heads in front of tokens: apart
            c.decode(q.view(out.shape), out=out)

    def append(code, text, c=None, **kw):
        a = N.PagedAppendArgs(k=0x1000000, v=0x1000200, k_stride_token=512, k_stride_head=256, v_stride_token=512,
                              v_stride_head=256, num_tokens=2, **kw)
        assert lib.ypk_paged_append(C.byref(c or c_cache()), C.byref(a), None) == code
        assert text in lib.ypk_last_error(None).decode(), lib.ypk_last_error(None)

    heads = dict(num_q_heads=8, q_stride_token=1024, q_stride_group=512, q_stride_head=128, q_out_stride_token=1024,
                 q_out_stride_group=512, q_out_stride_head=128)
    append(N.ERR_INVALID, "rows of the cache overlap", c_cache(stride_token=128))
    append(N.ERR_INVALID, "rows of the cache overlap", c_cache(stride_page=256))
    append(N.ERR_INVALID, "K and V rows", c_cache(v=0x10000))
    append(N.ERR_INVALID, "K and V rows", c_cache(v=0x10000 + 16 * 512))
    append(N.ERR_INVALID, "rows of q_out overlap", q=0x400000, q_out=0x400000,
           **dict(heads, q_stride_token=0, q_out_stride_token=0))
    append(N.ERR_INVALID, "rows of q_out overlap", q=0x400000, q_out=0x500000, **dict(heads, q_out_stride_token=512))
    append(N.ERR_INVALID, "q_out overlaps q without", q=0x400000, q_out=0x400000 + 2 * 512, **heads)
    append(N.ERR_INVALID, "q_out overlaps k or v", q=0x400000, q_out=0x1000000 - 16, **heads)
    append(N.ERR_INVALID, "q_out overlaps the cache", q=0x400000, q_out=0x20000 + 16, **heads)

    def decode(code, text, **kw):
        a = N.PagedDecodeArgs(**dict(dict(q=0x400000, out=0x500000, q_stride_token=1024, q_stride_group=512,
                                          q_stride_head=128, out_stride_token=1024, out_stride_group=512,
                                          out_stride_head=128, rows=2, num_q_heads=8, scale=0.1), **kw))
        assert lib.ypk_paged_decode(C.byref(c_cache()), C.byref(a), None) == code
        assert text in lib.ypk_last_error(None).decode(), lib.ypk_last_error(None)

    decode(N.ERR_INVALID, "rows of out overlap", out_stride_token=512)
    decode(N.ERR_INVALID, "out overlaps the cache", out=0x10000 + 16)
    decode(N.ERR_INVALID, "out overlaps q", out=0x400000 + 2 * 3 * 128)


def test_launches_are_sized_by_the_device():
    """No SM count stands in the code of the operators: it is the current device's."""
    csrc = os.path.join(ROOT, "yirage_b200", "csrc")
    for name in ("op_paged_append.cu", "op_paged_decode.cu", "op_logprobs.cu"):
        with open(os.path.join(csrc, name)) as f:
            code = "\n".join(line.split("//")[0] for line in f)
        assert "148" not in code and "op_device(" in code, name


def test_the_native_library_builds_without_what_the_python_binding_needs(native_lib, monkeypatch, tmp_path, capsys):
    """A C host has nvcc alone: libypk.so is built, the binding left out with a message; a binding of
    older sources does not stay behind.  A compiler that fails is an error all the same."""
    from yirage_b200 import build
    ran, binding = [], tmp_path / "_serving.so"
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libypk.so"))
    monkeypatch.setattr(build, "BINDING", str(binding))
    monkeypatch.setattr(build, "_run", lambda cmd, verbose, what: ran.append(what))
    which = shutil.which
    monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else which(name))
    binding.write_text("old")
    os.utime(binding, (0, 0))
    assert build.build() == build.LIB and ran == ["nvcc building libypk.so"]
    assert "no g++" in capsys.readouterr().err and not binding.exists()
    monkeypatch.setattr(build.shutil, "which", which)
    for lacking in ("torch", "Python's headers"):
        with monkeypatch.context() as m:
            if lacking == "torch":
                m.setitem(sys.modules, "torch", None)
            else:
                m.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
            assert build._binding_lacks() == lacking
    if which("g++"):
        ran.clear()
        build.build()
        assert ran == ["nvcc building libypk.so", "g++ building _serving.so"]


def test_taking_the_status_refuses_null(native_lib):
    for c, taken in ((None, 0x1000), (c_cache(), 0x1000), (c_cache(status=0x1000), None)):
        assert native_lib.ypk_paged_status(c and C.byref(c), taken, None) == N.ERR_INVALID
        assert "paged_status: null" in native_lib.ypk_last_error(None).decode()
    assert cache().check() is None        # on the CPU nothing has run


def test_table_rows_in_32_bits_start_on_16_byte_boundaries(native_lib):
    """A row stride of 4 x 4 bytes is one; what is behind the check refuses this call (an unaligned k)."""
    for dtype, stride, text in ((N.F32, 132, "not 16-byte aligned"), (N.F32, 130, "row stride 130"),
                                (N.BF16, 132, "row stride 132"), (N.BF16, 136, "not 16-byte aligned")):
        a = N.PagedAppendArgs(k=0x10002, v=0x10000, k_stride_token=256, k_stride_head=128, v_stride_token=256,
                              v_stride_head=128, num_tokens=2, cos=0x10000, sin=0x10000, table_dtype=dtype,
                              max_positions=64, table_stride=stride, rot_dim=128)
        assert native_lib.ypk_paged_append(C.byref(c_cache()), C.byref(a), None) == N.ERR_INVALID
        assert text in native_lib.ypk_last_error(None).decode()


def test_log_probabilities_of_no_rows_are_checked_like_any(native_lib):
    """A call without rows does nothing, with arguments that a call with rows would take."""
    call = lambda **kw: native_lib.ypk_token_logprobs(*dict(dict(
        logits=None, dtype=N.BF16, rows=0, vocab=100, ld=104, tokens=None, top=2, lp=None, ent=None, tl=None, tt=None,
        stream=None), **kw).values())
    assert call() == N.YPK_OK
    for kw, code in ((dict(top=33), N.ERR_UNSUPPORTED), (dict(top=-1), N.ERR_UNSUPPORTED), (dict(top=5, vocab=4), N.ERR_UNSUPPORTED),
                     (dict(dtype=N.I32), N.ERR_UNSUPPORTED), (dict(ld=99), N.ERR_INVALID), (dict(vocab=0), N.ERR_INVALID)):
        assert call(**kw) == code, kw


def test_sizes_past_32_bit_counting_are_refused(native_lib):
    """A loop over columns steps past the last one by the threads of a block, and heads are summed: both
    stay below 2^31.  (What would be behind the checks refuses these calls: null pointers.)"""
    for vocab, code, text in ((2 ** 31 - 1, N.ERR_UNSUPPORTED, "vocabulary 2147483647"), (2 ** 30 + 1, N.ERR_UNSUPPORTED, "at most"),
                              (2 ** 30, N.ERR_INVALID, "null")):
        assert native_lib.ypk_token_logprobs(None, N.BF16, 1, vocab, vocab, None, 0, None, None, None, None, None) == code
        assert text in native_lib.ypk_last_error(None).decode()
    for heads, text in ((2 ** 31 - 2, "query and 2 K/V heads"), (65532, "query and"), (65530, "not 16-byte aligned")):
        a = N.PagedAppendArgs(k=0x10002, v=0x10000, k_stride_token=256, k_stride_head=128, v_stride_token=256,
                              v_stride_head=128, num_tokens=2, q=0x400000, q_out=0x400000, num_q_heads=heads)
        assert native_lib.ypk_paged_append(C.byref(c_cache()), C.byref(a), None) != N.YPK_OK
        assert text in native_lib.ypk_last_error(None).decode()
