// New tokens' K and V rows into a paged cache, with RMS norm and rotation on the way
// (ypk_paged_append), and the host checks that the paged-cache operators share.
#include "op_paged.h"

namespace ypk {

int paged_check(const char *what, const ypk_paged_cache *c, bool append) {
  if (!c) return op_fail(YPK_ERR_INVALID, "%s: null cache", what);
  if (!c->k || !c->v || !c->indptr || (!c->indices && c->num_indices) || !c->last_page_len || (append && !c->qo_indptr))
    return op_fail(YPK_ERR_INVALID, "%s: null cache, page table or row offsets", what);
  if (c->dtype != YPK_BF16 && c->dtype != YPK_F16)
    return op_fail(YPK_ERR_UNSUPPORTED, "%s: cache type %d (bf16 or fp16)", what, c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return op_fail(YPK_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, c->head_dim);
  if (c->num_pages < 1 || c->page_size < 1 || c->num_kv_heads < 1 || c->num_indices < 0)
    return op_fail(YPK_ERR_INVALID, "%s: %d pages of %d tokens, %d K/V heads, %d page numbers", what,
                   c->num_pages, c->page_size, c->num_kv_heads, c->num_indices);
  if (c->num_requests < 1 || c->num_requests > 4096)
    return op_fail(YPK_ERR_UNSUPPORTED, "%s: %d requests (1..4096)", what, c->num_requests);
  if (c->stride_page % 8 || c->stride_token % 8 || c->stride_head % 8 || c->stride_page < 0 ||
      c->stride_token < 0 || c->stride_head < 0 || !op_aligned16(c->k) || !op_aligned16(c->v))
    return op_fail(YPK_ERR_INVALID, "%s: cache rows must start on 16-byte boundaries (strides "
                   "%lld %lld %lld)", what, (long long)c->stride_page, (long long)c->stride_token,
                   (long long)c->stride_head);
  // (rows of a cache may lie in any order, but not on one another: they are written)
  if ((c->num_pages > 1 && c->stride_page < c->head_dim) || (c->page_size > 1 && c->stride_token < c->head_dim) ||
      (c->num_kv_heads > 1 && c->stride_head < c->head_dim))
    return op_fail(YPK_ERR_INVALID, "%s: rows of the cache overlap (strides %lld %lld %lld)", what,
                   (long long)c->stride_page, (long long)c->stride_token, (long long)c->stride_head);
  return YPK_OK;
}

PagedView paged_view(const ypk_paged_cache *c) {
  PagedView v;
  v.k = static_cast<char *>(c->k);
  v.v = static_cast<char *>(c->v);
  v.stride_page = c->stride_page;
  v.stride_token = c->stride_token;
  v.stride_head = c->stride_head;
  v.indptr = c->indptr;
  v.indices = c->indices;
  v.last = c->last_page_len;
  v.qo = c->qo_indptr;
  v.status = c->status;
  v.num_pages = c->num_pages;
  v.page_size = c->page_size;
  v.kv_heads = c->num_kv_heads;
  v.num_requests = c->num_requests;
  v.num_indices = c->num_indices;
  return v;
}

namespace {

struct AppendArgs {
  PagedView c;
  const char *q, *k, *v;
  char *q_out;
  const char *cos, *sin;
  const char *q_norm, *k_norm;
  int64_t k_token, k_head, v_token, v_head;
  int64_t q_token, q_group, q_head, o_token, o_group, o_head;
  int64_t table_stride;
  int tokens, q_heads, group, rot, max_pos;
  float eps;
};

// Eight table values as floats, from 16 or 32 bits.
template <class T, bool WIDE_TABLE>
__device__ __forceinline__ void load_table(const char *base, int64_t element, float (&x)[8]) {
  if (WIDE_TABLE) {
    const float4 *p = reinterpret_cast<const float4 *>(base + element * 4);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    op_widen8<T>(__ldg(reinterpret_cast<const uint4 *>(base + element * 2)), x);
  }
}

// One (token, head) per D / 16 threads; each thread holds two chunks of eight dimensions: the
// pair that a rotation mixes, or two neighbours behind the rotated part.
template <class T, bool WIDE_TABLE, int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a) {
  constexpr int kThreads = D / 16;      // threads per head
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  const int64_t item = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) / kThreads;
  const int lane = threadIdx.x % kThreads;
  if (item >= int64_t(a.tokens) * heads) return;   // whole groups of kThreads threads leave
  const int row = int(item / heads), head = int(item % heads);

  // the request this row belongs to: the last one whose rows begin at or before it
  const int n = a.c.num_requests;
  int lo = 0, hi = n;   // number of requests whose rows end at or before `row`
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.c.qo[mid + 1] <= row) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= n) return;                       // a padding row behind the last request
  const int req = lo;
  const PagedRun run = paged_run(a.c.indptr[req], a.c.indptr[req + 1], a.c.last[req], a.c.page_size,
                                 a.c.num_indices);
  const int64_t pos = paged_new_position(run, a.c.qo[req + 1], row);
  if (a.c.qo[req] > row || run.broken || pos < 0 || pos >= run.tokens) {
    paged_flag(a.c, run.broken ? kPagedBadTable : kPagedBadLength);
    return;
  }
  const bool rotate = a.cos != nullptr;
  if (rotate && pos >= a.max_pos) {
    paged_flag(a.c, kPagedBadPosition);
    return;
  }
  const int64_t slot = paged_row(a.c.indices[run.first + pos / a.c.page_size], a.c.num_pages, pos,
                                 a.c.page_size, a.c.stride_page, a.c.stride_token);
  if (slot < 0) {
    paged_flag(a.c, kPagedBadPage);
    return;
  }

  const bool is_q = head < a.q_heads;
  const int kv = is_q ? 0 : (head - a.q_heads) % a.c.kv_heads;
  const bool is_v = !is_q && head - a.q_heads >= a.c.kv_heads;
  const char *src;
  char *dst;
  if (is_q) {
    const int g = head / a.group, i = head % a.group;
    src = a.q + 2 * (row * a.q_token + g * a.q_group + i * a.q_head);
    dst = a.q_out + 2 * (row * a.o_token + g * a.o_group + i * a.o_head);
  } else {
    src = is_v ? a.v + 2 * (row * a.v_token + kv * a.v_head) : a.k + 2 * (row * a.k_token + kv * a.k_head);
    dst = (is_v ? a.c.v : a.c.k) + 2 * (slot + kv * a.c.stride_head);
  }
  const int pairs = a.rot / 16;                  // threads that hold a rotated pair
  const bool turned = rotate && !is_v && lane < pairs;
  const int c0 = lane < pairs ? lane : a.rot / 8 + 2 * (lane - pairs);
  const int c1 = lane < pairs ? lane + pairs : c0 + 1;
  uint4 x0 = *reinterpret_cast<const uint4 *>(src + 16 * c0);
  uint4 x1 = *reinterpret_cast<const uint4 *>(src + 16 * c1);
  const char *weight = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
  if (weight || turned) {
    float u[8], w[8];
    op_widen8<T>(x0, u);
    op_widen8<T>(x1, w);
    if (weight) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += u[i] * u[i] + w[i] * w[i];
      const unsigned mask = ((kThreads == 32 ? 0u : (1u << kThreads)) - 1u) << (threadIdx.x % 32 / kThreads * kThreads);
#pragma unroll
      for (int o = kThreads / 2; o; o /= 2) ss += __shfl_xor_sync(mask, ss, o);
      const float f = rsqrtf(ss * (1.0f / D) + a.eps);
      float g[8];
      op_widen8<T>(__ldg(reinterpret_cast<const uint4 *>(weight + 16 * c0)), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] *= f * g[i];
      op_widen8<T>(__ldg(reinterpret_cast<const uint4 *>(weight + 16 * c1)), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] *= f * g[i];
    }
    if (turned) {
      float c[8], s[8], c2[8], s2[8];
      const int64_t at = pos * a.table_stride;
      load_table<T, WIDE_TABLE>(a.cos, at + 8 * c0, c);
      load_table<T, WIDE_TABLE>(a.sin, at + 8 * c0, s);
      load_table<T, WIDE_TABLE>(a.cos, at + 8 * c1, c2);
      load_table<T, WIDE_TABLE>(a.sin, at + 8 * c1, s2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // products and sums rounded one by one, as the attention task of the graph does: K rows
        // appended by either are the same bits
        const float y0 = __fadd_rn(__fmul_rn(u[i], c[i]), -__fmul_rn(w[i], s[i]));
        const float y1 = __fadd_rn(__fmul_rn(w[i], c2[i]), __fmul_rn(u[i], s2[i]));
        u[i] = y0;
        w[i] = y1;
      }
    }
    x0 = op_round8<T>(u);
    x1 = op_round8<T>(w);
  }
  *reinterpret_cast<uint4 *>(dst + 16 * c0) = x0;
  *reinterpret_cast<uint4 *>(dst + 16 * c1) = x1;
}

template <class T, bool WIDE_TABLE>
int launch_append(int head_dim, const AppendArgs &a, cudaStream_t st) {
  const int64_t items = int64_t(a.tokens) * (a.q_heads + 2 * a.c.kv_heads);
  const int64_t threads = items * (head_dim / 16);
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return op_fail(YPK_ERR_UNSUPPORTED, "paged_append: %d tokens in one call", a.tokens);
  if (head_dim == 64) paged_append_kernel<T, WIDE_TABLE, 64><<<unsigned(blocks), 256, 0, st>>>(a);
  else if (head_dim == 128) paged_append_kernel<T, WIDE_TABLE, 128><<<unsigned(blocks), 256, 0, st>>>(a);
  else paged_append_kernel<T, WIDE_TABLE, 256><<<unsigned(blocks), 256, 0, st>>>(a);
  return op_launched("paged_append");
}

bool strides_ok(std::initializer_list<int64_t> s) {
  for (int64_t v : s)
    if (v < 0 || v % 8) return false;
  return true;
}

}  // namespace
}  // namespace ypk

using namespace ypk;

extern "C" int ypk_paged_append(const ypk_paged_cache *cache, const ypk_paged_append_args *p, void *stream) {
  if (int rc = paged_check("paged_append", cache, true)) return rc;
  if (!p) return op_fail(YPK_ERR_INVALID, "paged_append: null operands");
  if (p->num_tokens < 0) return op_fail(YPK_ERR_INVALID, "paged_append: %d tokens", p->num_tokens);
  if (p->num_tokens == 0) return YPK_OK;
  if (!p->k || !p->v) return op_fail(YPK_ERR_INVALID, "paged_append: null K or V rows");
  if ((p->q == nullptr) != (p->q_out == nullptr))
    return op_fail(YPK_ERR_INVALID, "paged_append: q and q_out come together");
  if (p->q && (p->num_q_heads < 1 || p->num_q_heads % cache->num_kv_heads))
    return op_fail(YPK_ERR_INVALID, "paged_append: %d query heads over %d K/V heads", p->num_q_heads,
                   cache->num_kv_heads);
  if ((p->cos == nullptr) != (p->sin == nullptr))
    return op_fail(YPK_ERR_INVALID, "paged_append: cos and sin come together");
  const bool wide = p->cos && p->table_dtype == YPK_F32;
  if (p->cos) {
    if (p->rot_dim < 16 || p->rot_dim % 16 || p->rot_dim > cache->head_dim)
      return op_fail(YPK_ERR_UNSUPPORTED, "paged_append: %d rotated dimensions of %d (a multiple of 16)",
                     p->rot_dim, cache->head_dim);
    if (!wide && p->table_dtype != cache->dtype)
      return op_fail(YPK_ERR_UNSUPPORTED, "paged_append: table type %d (the cache's or fp32)", p->table_dtype);
    if (p->max_positions < 1 || p->table_stride < p->rot_dim || p->table_stride % 8)
      return op_fail(YPK_ERR_INVALID, "paged_append: tables of %d positions, row stride %lld",
                     p->max_positions, (long long)p->table_stride);
  }
  for (const void *q : {p->k, p->v, p->q, static_cast<const void *>(p->q_out), p->cos, p->sin, p->q_norm, p->k_norm})
    if (!op_aligned16(q)) return op_fail(YPK_ERR_INVALID, "paged_append: an operand is not 16-byte aligned");
  if (!strides_ok({p->k_stride_token, p->k_stride_head, p->v_stride_token, p->v_stride_head}) ||
      (p->q && !strides_ok({p->q_stride_token, p->q_stride_group, p->q_stride_head, p->q_out_stride_token,
                            p->q_out_stride_group, p->q_out_stride_head})))
    return op_fail(YPK_ERR_INVALID, "paged_append: rows must start on 16-byte boundaries");
  AppendArgs a;
  a.c = paged_view(cache);
  a.q = static_cast<const char *>(p->q);
  a.k = static_cast<const char *>(p->k);
  a.v = static_cast<const char *>(p->v);
  a.q_out = static_cast<char *>(p->q_out);
  a.cos = static_cast<const char *>(p->cos);
  a.sin = static_cast<const char *>(p->sin);
  a.q_norm = static_cast<const char *>(p->q_norm);
  a.k_norm = static_cast<const char *>(p->k_norm);
  a.k_token = p->k_stride_token, a.k_head = p->k_stride_head;
  a.v_token = p->v_stride_token, a.v_head = p->v_stride_head;
  a.q_token = p->q_stride_token, a.q_group = p->q_stride_group, a.q_head = p->q_stride_head;
  a.o_token = p->q_out_stride_token, a.o_group = p->q_out_stride_group, a.o_head = p->q_out_stride_head;
  a.table_stride = p->table_stride;
  a.tokens = p->num_tokens;
  a.q_heads = p->q ? p->num_q_heads : 0;
  a.group = p->q ? p->num_q_heads / cache->num_kv_heads : 1;
  a.rot = p->cos ? p->rot_dim : 0;
  a.max_pos = p->max_positions;
  a.eps = p->eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == YPK_BF16)
    return wide ? launch_append<OpBf16, true>(cache->head_dim, a, st) : launch_append<OpBf16, false>(cache->head_dim, a, st);
  return wide ? launch_append<OpF16, true>(cache->head_dim, a, st) : launch_append<OpF16, false>(cache->head_dim, a, st);
}
