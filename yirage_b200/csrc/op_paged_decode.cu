// Attention of one new token per request over a paged cache (ypk_paged_decode).
#include "op_paged.h"

namespace ypk {
namespace {

struct DecodeArgs {
  PagedView c;
  const char *q;
  char *out;
  float *lse;
  int64_t q_token, q_group, q_head, o_token, o_group, o_head;
  int rows, q_heads, group, window;
  float scale;
};

// One CTA of four warps per (request, query head); warp w takes positions w, w + 4, ..., a lane
// holds D / 32 dimensions; running maximum and sum per warp, joined at the end.
template <class T, int D>
__global__ void __launch_bounds__(128) paged_decode_kernel(const DecodeArgs a) {
  constexpr int E = D / 32;     // dimensions per lane: 2, 4 or 8
  const int r = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = h / a.group, i = h % a.group;
  const PagedRun run = paged_run(a.c.indptr[r], a.c.indptr[r + 1], a.c.last[r], a.c.page_size, a.c.num_indices);
  if (run.broken && threadIdx.x == 0) paged_flag(a.c, kPagedBadTable);
  const uint32_t *qp = reinterpret_cast<const uint32_t *>(a.q + 2 * (r * a.q_token + g * a.q_group + i * a.q_head)) + lane * (E / 2);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const float2 f = T::widen(qp[e]);
    q[2 * e] = f.x * a.scale;
    q[2 * e + 1] = f.y * a.scale;
    o[2 * e] = o[2 * e + 1] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int64_t first = a.window > 0 && run.tokens > a.window ? run.tokens - a.window : 0;
  for (int64_t p = first + warp; p < run.tokens; p += 4) {
    const int64_t row = paged_row(a.c.indices[run.first + p / a.c.page_size], a.c.num_pages, p, a.c.page_size,
                                  a.c.stride_page, a.c.stride_token);
    if (row < 0) {
      if (lane == 0) paged_flag(a.c, kPagedBadPage);
      continue;
    }
    const uint32_t *kp = reinterpret_cast<const uint32_t *>(a.c.k + 2 * (row + g * a.c.stride_head)) + lane * (E / 2);
    const uint32_t *vp = reinterpret_cast<const uint32_t *>(a.c.v + 2 * (row + g * a.c.stride_head)) + lane * (E / 2);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 f = T::widen(kp[e]);
      s += q[2 * e] * f.x + q[2 * e + 1] * f.y;
    }
#pragma unroll
    for (int x = 16; x; x /= 2) s += __shfl_xor_sync(~0u, s, x);
    const float top = fmaxf(m, s);
    const float keep = __expf(m - top), w = __expf(s - top);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 f = T::widen(vp[e]);
      o[2 * e] = o[2 * e] * keep + w * f.x;
      o[2 * e + 1] = o[2 * e + 1] * keep + w * f.y;
    }
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w]);
  float f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : __expf(sm[w] - top);
    total += f[w] * sl[w];
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  uint32_t *op = reinterpret_cast<uint32_t *>(a.out + 2 * (r * a.o_token + g * a.o_group + i * a.o_head));
  for (int d = threadIdx.x; d < D / 2; d += 128) {
    float x = 0.f, y = 0.f;
    for (int w = 0; w < 4; ++w) {
      x += f[w] * so[w][2 * d];
      y += f[w] * so[w][2 * d + 1];
    }
    op[d] = T::round2(x * inv, y * inv);
  }
  if (a.lse && threadIdx.x == 0) a.lse[int64_t(r) * a.q_heads + h] = total > 0.f ? top + logf(total) : -INFINITY;
}

template <class T>
int launch_decode(int head_dim, const DecodeArgs &a, cudaStream_t st) {
  const dim3 grid(a.rows, a.q_heads);
  if (head_dim == 64) paged_decode_kernel<T, 64><<<grid, 128, 0, st>>>(a);
  else if (head_dim == 128) paged_decode_kernel<T, 128><<<grid, 128, 0, st>>>(a);
  else paged_decode_kernel<T, 256><<<grid, 128, 0, st>>>(a);
  return op_launched("paged_decode");
}

int check_heads(const ypk_paged_cache *cache, int q_heads) {
  if (q_heads < 1 || q_heads % cache->num_kv_heads || q_heads > 65535)
    return op_fail(YPK_ERR_INVALID, "paged_decode: %d query heads over %d K/V heads", q_heads, cache->num_kv_heads);
  return YPK_OK;
}

}  // namespace
}  // namespace ypk

using namespace ypk;

extern "C" int ypk_paged_decode_workspace(const ypk_paged_cache *cache, int32_t num_q_heads, uint64_t *bytes) {
  if (int rc = paged_check("paged_decode", cache, false)) return rc;
  if (int rc = check_heads(cache, num_q_heads)) return rc;
  if (!bytes) return op_fail(YPK_ERR_INVALID, "paged_decode: null size");
  *bytes = 16;
  return YPK_OK;
}

extern "C" int ypk_paged_decode(const ypk_paged_cache *cache, const ypk_paged_decode_args *p, void *stream) {
  if (int rc = paged_check("paged_decode", cache, false)) return rc;
  if (!p) return op_fail(YPK_ERR_INVALID, "paged_decode: null operands");
  if (int rc = check_heads(cache, p->num_q_heads)) return rc;
  if (p->rows < 0 || p->rows > cache->num_requests)
    return op_fail(YPK_ERR_INVALID, "paged_decode: %d rows for %d requests", p->rows, cache->num_requests);
  if (p->rows == 0) return YPK_OK;
  if (!p->q || !p->out) return op_fail(YPK_ERR_INVALID, "paged_decode: null q or out");
  if (p->window < 0) return op_fail(YPK_ERR_INVALID, "paged_decode: window %d", p->window);
  if (!(p->scale == p->scale) || p->scale - p->scale != 0.f)
    return op_fail(YPK_ERR_INVALID, "paged_decode: scale is not finite");
  for (int64_t s : {p->q_stride_token, p->q_stride_group, p->q_stride_head, p->out_stride_token,
                    p->out_stride_group, p->out_stride_head})
    if (s < 0 || s % 8) return op_fail(YPK_ERR_INVALID, "paged_decode: rows must start on 16-byte boundaries");
  if (!op_aligned16(p->q) || !op_aligned16(p->out) || !op_aligned16(p->workspace))
    return op_fail(YPK_ERR_INVALID, "paged_decode: an operand is not 16-byte aligned");
  uint64_t need = 0;
  if (int rc = ypk_paged_decode_workspace(cache, p->num_q_heads, &need)) return rc;
  if (!p->workspace || p->workspace_bytes < need)
    return op_fail(YPK_ERR_INVALID, "paged_decode: workspace of %llu bytes, %llu needed",
                   (unsigned long long)(p->workspace ? p->workspace_bytes : 0), (unsigned long long)need);
  DecodeArgs a;
  a.c = paged_view(cache);
  a.q = static_cast<const char *>(p->q);
  a.out = static_cast<char *>(p->out);
  a.lse = p->lse;
  a.q_token = p->q_stride_token, a.q_group = p->q_stride_group, a.q_head = p->q_stride_head;
  a.o_token = p->out_stride_token, a.o_group = p->out_stride_group, a.o_head = p->out_stride_head;
  a.rows = p->rows;
  a.q_heads = p->num_q_heads;
  a.group = p->num_q_heads / cache->num_kv_heads;
  a.window = p->window;
  a.scale = p->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == YPK_BF16 ? launch_decode<OpBf16>(cache->head_dim, a, st)
                                  : launch_decode<OpF16>(cache->head_dim, a, st);
}
