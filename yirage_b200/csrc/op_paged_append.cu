// New tokens' K and V rows into a paged cache, with RMS norm and rotation on the way
// (ypk_paged_append), and the host checks that the paged-cache operators share.
#include <algorithm>
#include <initializer_list>

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
  if (!append) return YPK_OK;
  if (!rows_distinct(cache_rows(c, c->k)))
    return op_fail(YPK_ERR_INVALID, "%s: rows of the cache overlap (strides %lld %lld %lld)", what,
                   (long long)c->stride_page, (long long)c->stride_token, (long long)c->stride_head);
  if (rows_touch(cache_rows(c, c->k), cache_rows(c, c->v)))
    return op_fail(YPK_ERR_INVALID, "%s: K and V rows of the cache overlap", what);
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
  int rows_per_cta, rows_at_once;   // tokens a CTA takes; as many of them together
  int heads_per_cta;
  int groups_per_token;             // groups of threads that share a token's heads
  FastDivisor page_div;
  float eps;
};

constexpr int kAppendThreads = 128;
constexpr int kAppendCtas = 4;       // resident per SM
constexpr int kAhead = 3;            // (token, head)s per thread at a time
constexpr int kMaxTurns = 8;         // turns of a CTA
constexpr int kMaxRows = 256;        // tokens of a CTA

// Eight table values as pairs of floats, from 16 or 32 bits.
template <class T, bool WIDE_TABLE>
__device__ __forceinline__ void load_table(const char *base, int64_t element, f32x2 (&x)[4]) {
  if (WIDE_TABLE) {
    const float4 *p = reinterpret_cast<const float4 *>(base + element * 4);
    const float4 a = p[0], b = p[1];
    x[0] = pair(a.x, a.y), x[1] = pair(a.z, a.w), x[2] = pair(b.x, b.y), x[3] = pair(b.z, b.w);
  } else {
    op_widen8<T>(*reinterpret_cast<const uint4 *>(base + element * 2), x);
  }
}

// Where one new token goes.
struct Place {
  int64_t slot;    // element offset of its row for K/V head 0; -1: nowhere
  int64_t table;   // element offset of its row in the rotary tables
};

// The places of the rows of a warp's groups of LANES threads, one row per group; all lanes call.
// Broken entries are reported and give slot -1.
template <int LANES>
__device__ __forceinline__ Place find_place(const AppendArgs &a, int row) {
  const int lane = threadIdx.x % LANES, shift = threadIdx.x % 32 / LANES * LANES;
  // the request whose rows hold this one: rounds of LANES evenly spaced looks at the row offsets
  int lo = 0, n = a.c.num_requests;      // the answer is among requests lo .. lo + n
  while (__any_sync(~0u, n > 0)) {
    const int step = (n + LANES - 1) / LANES, at = lo + (lane + 1) * step;
    const bool before = n > 0 && at <= lo + n && a.c.qo[at] <= row;   // requests lo .. at - 1 end before
    const int skip = __popc(__ballot_sync(~0u, before) >> shift & ((1u << LANES) - 1)) * step;
    lo += skip;
    n = n > 0 ? min(n - skip, step - 1) : 0;
  }
  Place p = {-1, 0};
  if (lo >= a.c.num_requests) return p;                              // a padding row
  const PagedRun run = paged_run(a.c.indptr[lo], a.c.indptr[lo + 1], a.c.last[lo], a.c.page_size, a.c.num_indices);
  const int64_t pos = paged_new_position(run, a.c.qo[lo + 1], row);
  int bad = 0;
  if (run.broken) bad = kPagedBadTable;
  else if (a.c.qo[lo] > row || pos < 0 || pos >= run.tokens) bad = kPagedBadLength;
  else if (a.cos && pos >= a.max_pos) bad = kPagedBadPosition;
  else {
    const int q = fast_div(int(pos), a.page_div), page = a.c.indices[run.first + q];
    p.slot = paged_row(page, a.c.num_pages, int(pos) - q * a.c.page_size, a.c.stride_page, a.c.stride_token);
    p.table = pos * a.table_stride;
    if (p.slot < 0) bad = kPagedBadPage;
  }
  if (bad && lane == 0) paged_flag(a.c, bad);
  return p;
}

// A CTA takes a.rows_per_cta tokens, a.rows_at_once of them together, and of each the heads of
// blockIdx.y's share (q heads, then k, then v).  D / 16 threads move one head, each thread two
// chunks of eight dimensions: the pair that a rotation mixes, or two neighbours behind the rotated
// part.  A thread keeps its kAhead heads from turn to turn, so what belongs to a head
// (addresses, kind, norm weight) is worked out once, and heads of one token share its table
// entries; the next turn's rows are on their way while one is finished, the first ones while
// the places are looked up.
//
// Bytes bound it: rows in and out once, 2 (Hq + 2 Hkv) D elements a token.  At 128 registers four
// CTAs of 128 threads are resident, each thread with 96 bytes in flight and 96 in work; that spills
// 40 bytes a thread, 84 where a CTA has several tokens at once.  Measured
// (32 + 2 x 8 heads of 128, bf16): 32768 tokens called back to back 138 us = 5.8 TB/s, 89 % of the
// copy rate (132 us in a graph); 4498 tokens of 32 + 2 x 4 heads with norms 21.6 us = 4.3 TB/s, in
// one wave, so that nothing covers its first lookups (2 us) and last stores; one token 3.4 us in a
// graph, launch and five dependent loads.  Two heads a
// thread 165 us on 32768 tokens, 256 threads a CTA 171, three CTAs per SM 152.
template <class T, bool WIDE_TABLE, int D, bool TOGETHER>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  op_wait_for_previous();
  constexpr int kLanes = D / 16;                       // threads per head
  constexpr int kItems = kAppendThreads / kLanes;      // heads at a time
  const int at_once = TOGETHER ? a.rows_at_once : 1;
  __shared__ Place s_place[kMaxRows];
  const int64_t row0 = int64_t(blockIdx.x) * a.rows_per_cta;
  const int rows = int(min(int64_t(a.rows_per_cta), a.tokens - row0));
  const int lane = threadIdx.x % kLanes;
  const int pairs = a.rot / 16;                        // threads that hold a rotated pair
  const int c0 = lane < pairs ? lane : a.rot / 8 + 2 * (lane - pairs);
  const int c1 = lane < pairs ? lane + pairs : c0 + 1;
  const unsigned group_mask = ((1u << kLanes) - 1u) << (threadIdx.x % 32 / kLanes * kLanes);
  const bool turns = a.cos && lane < pairs;

  // this thread's heads
  const char *src[kAhead];
  char *dst[kAhead];
  int64_t src_step[kAhead];
  int kind[kAhead];                                    // 0: q, 1: k, 2: v, -1: none
  // a group of threads has heads of one token of the turn, which share its table entries (heads dealt
  // out over the tokens of a turn instead: 12000 tokens of 12 heads 21.9 us, so 18.5)
  const int group = threadIdx.x / kLanes, of_token = TOGETHER ? a.groups_per_token : kItems;
  const int sub = TOGETHER ? group / of_token : 0, head0 = group - sub * of_token;
  const int heads = a.q_heads + 2 * a.c.kv_heads;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int i = head0 + j * of_token, h = blockIdx.y * a.heads_per_cta + i;
    kind[j] = sub >= at_once || i >= a.heads_per_cta || h >= heads ? -1
              : h < a.q_heads ? 0 : h < a.q_heads + a.c.kv_heads ? 1 : 2;
    const int kv = (h - a.q_heads) - (kind[j] == 2 ? a.c.kv_heads : 0);
    if (kind[j] == 0) {
      const int g = h / a.group, i = h - g * a.group;
      src_step[j] = a.q_token;
      src[j] = a.q + 2 * (g * a.q_group + i * a.q_head);
      dst[j] = a.q_out + 2 * (row0 * a.o_token + g * a.o_group + i * a.o_head);
    } else if (kind[j] == 1) {
      src_step[j] = a.k_token;
      src[j] = a.k + 2 * (kv * a.k_head);
      dst[j] = a.c.k + 2 * (kv * a.c.stride_head);
    } else {
      src_step[j] = a.v_token;
      src[j] = a.v + 2 * (kv * a.v_head);
      dst[j] = a.c.v + 2 * (kv * a.c.stride_head);
    }
    src[j] += 2 * (row0 + sub) * src_step[j];
    src_step[j] *= 2 * at_once;
  }
  uint4 n0[kAhead], n1[kAhead];
  const auto fetch = [&](int t) {       // the rows at src, which moves on
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (kind[j] >= 0 && t + sub < rows) {
        n0[j] = op_load_once(reinterpret_cast<const uint4 *>(src[j] + 16 * c0));
        n1[j] = op_load_once(reinterpret_cast<const uint4 *>(src[j] + 16 * c1));
      }
      src[j] += src_step[j];
    }
  };
  fetch(0);
  // (more tokens a CTA: fewer threads per lookup, 12000 tokens of 12 heads 18.5 -> 17.8 us)
  constexpr int kFind = TOGETHER ? 4 : kLanes;
  for (int i0 = 0; i0 < rows; i0 += kAppendThreads / kFind) {
    const int i = i0 + threadIdx.x / kFind;
    const Place p = find_place<kFind>(a, int(row0) + min(i, rows - 1));
    if (threadIdx.x % kFind == 0 && i < rows) s_place[i] = p;
  }
  __syncthreads();

  for (int t = 0; t < rows; t += at_once) {
    uint4 x0[kAhead], x1[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x0[j] = n0[j], x1[j] = n1[j];
    fetch(t + at_once);
    f32x2 cos0[4], sin0[4], cos1[4], sin1[4];         // sin0: negated
    if (TOGETHER && t + sub >= rows) continue;         // (whole groups of kLanes threads together)
    const Place place = s_place[t + sub];
    if (place.slot < 0) continue;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (kind[j] < 0) continue;
      if (turns && j == 0) {
        load_table<T, WIDE_TABLE>(a.cos, place.table + 8 * c0, cos0);
        load_table<T, WIDE_TABLE>(a.sin, place.table + 8 * c0, sin0);
        load_table<T, WIDE_TABLE>(a.cos, place.table + 8 * c1, cos1);
        load_table<T, WIDE_TABLE>(a.sin, place.table + 8 * c1, sin1);
#pragma unroll
        for (int i = 0; i < 4; ++i) sin0[i] ^= 0x8000000080000000ull;
      }
      const char *weight = kind[j] == 0 ? a.q_norm : kind[j] == 1 ? a.k_norm : nullptr;
      if (weight || (turns && kind[j] < 2)) {
        f32x2 u[4], w[4];
        op_widen8<T>(x0[j], u);
        op_widen8<T>(x1[j], w);
        if (weight) {
          f32x2 ss = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) ss = fma2(u[i], u[i], fma2(w[i], w[i], ss));
          const float2 s2 = halves(ss);
          float total = s2.x + s2.y;
#pragma unroll
          for (int o = kLanes / 2; o; o /= 2) total += __shfl_xor_sync(group_mask, total, o);
          const float f = rsqrtf(total * (1.0f / D) + a.eps);
          f32x2 g[4];
          op_widen8<T>(*reinterpret_cast<const uint4 *>(weight + 16 * c0), g);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] = mul2(mul2(u[i], pair(f, f)), g[i]);
          op_widen8<T>(*reinterpret_cast<const uint4 *>(weight + 16 * c1), g);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = mul2(mul2(w[i], pair(f, f)), g[i]);
        }
        if (turns) {
          // products and sums rounded one by one, as the attention task of the graph does: K rows
          // appended by either are the same bits
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2 y = add2(mul2(u[i], cos0[i]), mul2(w[i], sin0[i]));
            w[i] = add2(mul2(w[i], cos1[i]), mul2(u[i], sin1[i]));
            u[i] = y;
          }
        }
        x0[j] = op_round8<T>(u);
        x1[j] = op_round8<T>(w);
      }
      // (stores that leave the L2 first: 137 -> 132 us on 32k tokens)
      char *to = dst[j] + (kind[j] == 0 ? 2 * (t + sub) * a.o_token : 2 * place.slot);
      __stcs(reinterpret_cast<uint4 *>(to + 16 * c0), x0[j]);
      __stcs(reinterpret_cast<uint4 *>(to + 16 * c1), x1[j]);
    }
  }
}

// Few tokens: a CTA takes one token and as many of its heads as it moves at once, so that one
// token's heads spread over the device.  Else all heads that fit, of several tokens together
// where heads are few, and as many turns, at most kMaxTurns, as give whole waves of CTAs.
template <class T, bool WIDE_TABLE, int D>
int launch_shape(AppendArgs &a, cudaStream_t st) {
  constexpr int kItems = kAppendThreads / (D / 16);
  DeviceInfo dev;
  if (int rc = op_device("paged_append", &dev)) return rc;
  const int resident = dev.sms * kAppendCtas;
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  const auto parts = [&](int n) { return (heads + n - 1) / n; };
  const bool few = int64_t(a.tokens) * parts(kItems) <= resident;
  a.heads_per_cta = std::min(heads, few ? kItems : kItems * kAhead);
  a.groups_per_token = (heads + kAhead - 1) / kAhead;
  a.rows_at_once = few ? 1 : std::max(1, kItems / a.groups_per_token);
  const int64_t units = int64_t(a.tokens) * parts(a.heads_per_cta);
  const auto over = [&](int64_t n, int64_t d) { return (n + d * a.rows_at_once - 1) / (d * a.rows_at_once); };
  const int64_t waves = over(units, int64_t(resident) * kMaxTurns);
  a.rows_per_cta = std::min(int(over(units, resident * waves)) * a.rows_at_once, kMaxRows);
  const dim3 grid(unsigned((int64_t(a.tokens) + a.rows_per_cta - 1) / a.rows_per_cta), parts(a.heads_per_cta));
  return op_launch("paged_append",
                   a.rows_at_once > 1 ? paged_append_kernel<T, WIDE_TABLE, D, true>
                                      : paged_append_kernel<T, WIDE_TABLE, D, false>,
                   grid, kAppendThreads, 0, 0, st, a);
}

template <class T, bool WIDE_TABLE>
int launch_append(int head_dim, AppendArgs &a, cudaStream_t st) {
  if (head_dim == 64) return launch_shape<T, WIDE_TABLE, 64>(a, st);
  if (head_dim == 128) return launch_shape<T, WIDE_TABLE, 128>(a, st);
  return launch_shape<T, WIDE_TABLE, 256>(a, st);
}

struct StatusArgs {
  int *status, *taken;
};
__global__ void paged_status_kernel(const __grid_constant__ StatusArgs a) {
  op_wait_for_previous();
  *a.taken = atomicExch(a.status, 0);
}

bool strides_ok(std::initializer_list<int64_t> s) {
  for (int64_t v : s)
    if (v < 0 || v % 8) return false;
  return true;
}

}  // namespace
}  // namespace ypk

using namespace ypk;

extern "C" int ypk_paged_status(const ypk_paged_cache *cache, int32_t *taken, void *stream) {
  if (!cache || !cache->status || !taken) return op_fail(YPK_ERR_INVALID, "paged_status: null cache, status or result");
  return op_launch("paged_status", paged_status_kernel, dim3(1), 1, 0, 0, static_cast<cudaStream_t>(stream),
                   StatusArgs{cache->status, taken});
}

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
  if (int64_t(p->q ? p->num_q_heads : 0) + 2 * int64_t(cache->num_kv_heads) > 65535)      // (sums of them are 32-bit)
    return op_fail(YPK_ERR_UNSUPPORTED, "paged_append: %d query and %d K/V heads", p->q ? p->num_q_heads : 0,
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
    if (p->max_positions < 1 || p->table_stride < p->rot_dim || p->table_stride % (wide ? 4 : 8))
      return op_fail(YPK_ERR_INVALID, "paged_append: tables of %d positions, row stride %lld",
                     p->max_positions, (long long)p->table_stride);
  }
  for (const void *q : {p->k, p->v, p->q, static_cast<const void *>(p->q_out), p->cos, p->sin, p->q_norm, p->k_norm})
    if (!op_aligned16(q)) return op_fail(YPK_ERR_INVALID, "paged_append: an operand is not 16-byte aligned");
  if (!strides_ok({p->k_stride_token, p->k_stride_head, p->v_stride_token, p->v_stride_head}) ||
      (p->q && !strides_ok({p->q_stride_token, p->q_stride_group, p->q_stride_head, p->q_out_stride_token,
                            p->q_out_stride_group, p->q_out_stride_head})))
    return op_fail(YPK_ERR_INVALID, "paged_append: rows must start on 16-byte boundaries");
  const int group = p->q ? p->num_q_heads / cache->num_kv_heads : 1;
  if (p->q) {
    // in place or apart: a row is read by the threads that write it, and ahead of that by nobody
    const auto rows = [&](const void *at, int64_t token, int64_t kv, int64_t head, int heads) {
      return head_rows(at, p->num_tokens, token, cache->num_kv_heads, kv, heads, head, cache->head_dim);
    };
    const StridedRows out = rows(p->q_out, p->q_out_stride_token, p->q_out_stride_group, p->q_out_stride_head, group);
    const bool same = p->q == p->q_out && p->q_stride_token == p->q_out_stride_token &&
                      p->q_stride_group == p->q_out_stride_group && p->q_stride_head == p->q_out_stride_head;
    if (!same && rows_touch(rows(p->q, p->q_stride_token, p->q_stride_group, p->q_stride_head, group), out))
      return op_fail(YPK_ERR_INVALID, "paged_append: q_out overlaps q without being q");
    if (!rows_distinct(out)) return op_fail(YPK_ERR_INVALID, "paged_append: rows of q_out overlap");
    if (rows_touch(rows(p->k, p->k_stride_token, p->k_stride_head, 0, 1), out) ||
        rows_touch(rows(p->v, p->v_stride_token, p->v_stride_head, 0, 1), out))
      return op_fail(YPK_ERR_INVALID, "paged_append: q_out overlaps k or v");
    if (rows_touch(cache_rows(cache, cache->k), out) || rows_touch(cache_rows(cache, cache->v), out))
      return op_fail(YPK_ERR_INVALID, "paged_append: q_out overlaps the cache");
  }
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
  a.group = group;
  a.rot = p->cos ? p->rot_dim : 0;
  a.max_pos = p->max_positions;
  a.eps = p->eps;
  a.page_div = fast_divisor(cache->page_size);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == YPK_BF16)
    return wide ? launch_append<OpBf16, true>(cache->head_dim, a, st) : launch_append<OpBf16, false>(cache->head_dim, a, st);
  return wide ? launch_append<OpF16, true>(cache->head_dim, a, st) : launch_append<OpF16, false>(cache->head_dim, a, st);
}
