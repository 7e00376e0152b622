// Log probabilities of given tokens, with entropy and top alternatives (ypk_token_logprobs).
//
//   m = max x,  s = sum e^(x - m),  u = sum (x - m) e^(x - m)
//   log p(t) = x_t - m - ln s,   entropy = ln s - u / s
//
// One pass over the logits with m, s and u running in each thread's registers (in the base 2:
// y = (x - m) log2 e).  Memory bounds it; next comes the exponential, one per logit: 73 % of the
// special-function rate when 16-bit logits arrive at the copy rate, so everything else is kept
// to packed pairs (two fp32 per instruction, maxima on pairs of 16-bit values).
//
// The top alternatives cost the pass nothing.  Its running maxima m_t, one per thread, give a
// bound: the k-th largest maximum of 64 groups of threads is at most the k-th largest logit.
// Only the columns of the threads whose own maximum reaches the bound (about k of 512) are read
// again, from L2, and what reaches the bound there (a little more than k logits) is ranked.
// Rows full of equal values (a mask that leaves less than k columns) overflow that list; they
// take the logits above the bound and then the lowest columns that equal it.
//
// A row is split over a cluster of CTAs when there are few rows; their sums and lists are
// joined through distributed shared memory, so there is no workspace and no second launch.
#include <cooperative_groups.h>
#include <math.h>

#include <atomic>

#include "op_common.h"
#include "op_num.cuh"

namespace cg = cooperative_groups;

namespace ypk {
namespace {

constexpr int kMaxTop = 32;
constexpr int kThreads = 512;
constexpr int kGroups = 64;        // of 8 threads: what the bound of the top list is taken from
constexpr int kCandidates = 1024;
constexpr int kUnroll = 4;         // 16-byte loads in flight per thread (and as many ahead)
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
// Exponents below this add nothing to a sum that holds a 1; it keeps -infinity out of products.
constexpr float kFloor = -200.f;

struct LogprobArgs {
  const char *logits;
  const long long *tokens;
  float *logprob, *entropy, *top_logprob;
  long long *top_token;
  int64_t ld;
  int vocab, top;
};

// Values as whole numbers in the same order (NaN lowest, -0 and +0 alike), and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0u) return NAN;
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
// Larger key: larger value, then lower column.  No key of a column is 0.
__device__ __forceinline__ unsigned long long key_of(uint32_t order, uint32_t col) {
  return (static_cast<unsigned long long>(order) << 32) | (0xffffffffu - col);
}

// ---- pairs of fp32 in one 64-bit register
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN on either side stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint4 load16(const char *p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One 16-byte vector of logits.
template <int DTYPE>
struct Vec;
template <>
struct Vec<YPK_F32> {
  static constexpr int kN = 4, kBytes = 4;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ float top(const uint4 &v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return i ? make_float2(__uint_as_float(v.z), __uint_as_float(v.w)) : make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
  }
  static __device__ __forceinline__ float one(const char *p) { return __ldg(reinterpret_cast<const float *>(p)); }
};
template <>
struct Vec<YPK_BF16> {
  static constexpr int kN = 8, kBytes = 2;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(const uint4 &v) {
    const float2 f = OpBf16::widen(max2(max2(v.x, v.y), max2(v.z, v.w)));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return OpBf16::widen(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float one(const char *p) {
    return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(p)));
  }
};
template <>
struct Vec<YPK_F16> {
  static constexpr int kN = 8, kBytes = 2;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(const uint4 &v) {
    const float2 f = OpF16::widen(max2(max2(v.x, v.y), max2(v.z, v.w)));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return OpF16::widen(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float one(const char *p) {
    return __half2float(__ldg(reinterpret_cast<const __half *>(p)));
  }
};

// Running maximum and sums.
struct Sums {
  float m, s, u;
};

// To the reference `top` (>= m, or NaN).
__device__ __forceinline__ void move_reference(Sums &a, float top) {
  const float d = fmaxf((a.m - top) * kLog2e, kFloor);   // (-infinity and NaN: no weight is lost, s = 0)
  const float f = exp2_fast(d);
  a.u = a.s == 0.f ? 0.f : (a.u + d * a.s) * f;
  a.s = a.s == 0.f ? 0.f : a.s * f;
  a.m = top;
}

__device__ __forceinline__ void join(Sums &a, Sums b) {
  const float top = max_nan(a.m, b.m);
  move_reference(a, top);
  move_reference(b, top);
  a.s += b.s;
  a.u += b.u;
}

struct Shared {
  Sums warp[kThreads / 32];
  Sums all;                               // of this CTA
  uint32_t group[kGroups];
  uint32_t bound;
  int listed, found;
  int threads[kThreads];                  // whose columns are read again
  unsigned long long cand[kCandidates];
  unsigned long long top[kMaxTop];        // of this CTA, falling; 0: none
  unsigned long long best;
  unsigned long long merged[kMaxCluster * kMaxTop];
  int warp_count[kThreads / 32];
};

// The columns of one CTA: a few single ones, whole 16-byte vectors, a few single ones.
struct Slice {
  const char *row;
  int first, head, vecs, tail;   // columns [first, first + head), vecs vectors, tail columns
};

// Columns of a row at `row` that CTA `rank` of `ctas` takes.
template <int DTYPE>
__device__ __forceinline__ Slice slice_of(const char *row, int vocab, int rank, int ctas) {
  using V = Vec<DTYPE>;
  const int skip = int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / V::kBytes);
  const int head = min(skip, vocab);
  const int vecs = (vocab - head) / V::kN, tail = (vocab - head) % V::kN;
  const int v0 = int(int64_t(vecs) * rank / ctas), v1 = int(int64_t(vecs) * (rank + 1) / ctas);
  Slice s;
  s.row = row;
  s.head = rank == 0 ? head : 0;
  s.first = rank == 0 ? 0 : head + v0 * V::kN;
  s.vecs = v1 - v0;
  s.tail = rank == ctas - 1 ? tail : 0;
  return s;
}

// The k largest of sh.cand[0..n) in order into sh.top; every thread calls.
__device__ void rank_candidates(Shared &sh, int n, int k) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long mine = sh.cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += sh.cand[j] > mine;
    if (above < k) sh.top[above] = mine;
  }
}

template <int DTYPE>
__device__ void top_of_slice(Shared &sh, const Slice &s, float my_max, int k) {
  using V = Vec<DTYPE>;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int first_vec = s.first + s.head;                      // column of the first vector
  const char *vec0 = s.row + int64_t(first_vec) * V::kBytes;
  const int columns = s.head + s.vecs * V::kN + s.tail;
  const uint32_t mine = order_of(my_max);
  uint32_t g = mine;
#pragma unroll
  for (int x = 1; x < kThreads / kGroups; x *= 2) g = max(g, __shfl_xor_sync(~0u, g, x));
  if (tid % (kThreads / kGroups) == 0) sh.group[tid / (kThreads / kGroups)] = g;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.listed = sh.found = 0;
  // a NaN hides its thread's other columns from the maxima
  bool one_by_one = __syncthreads_or(my_max != my_max);
  if (!one_by_one) {
    if (tid < kGroups) {
      const uint32_t gi = sh.group[tid];      // thread i ranks group i
      int above = 0;
      for (int j = 0; j < kGroups; ++j) above += sh.group[j] > gi || (sh.group[j] == gi && j < tid);
      if (above == k - 1) sh.bound = gi;
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (mine >= bound) sh.threads[atomicAdd(&sh.listed, 1)] = tid;
    __syncthreads();
    const int listed = sh.listed;
    const int rounds = (s.vecs + kThreads - 1) / kThreads;
    // logits of at least (strict: above) the bound, in no order
    const auto collect = [&](uint32_t least) {
      const auto offer = [&](float x, int col) {
        const uint32_t o = order_of(x);
        if (o < least) return;
        const int at = atomicAdd(&sh.found, 1);
        if (at < kCandidates) sh.cand[at] = key_of(o, uint32_t(col));
      };
      for (int i = tid; i < listed * rounds; i += kThreads) {
        const int v = i / listed * kThreads + sh.threads[i % listed];
        if (v >= s.vecs) continue;
        const uint4 x = load16(vec0 + int64_t(v) * 16);
        if (order_of(V::top(x)) < least) continue;
#pragma unroll
        for (int e = 0; e < V::kN / 2; ++e) {
          const float2 f = V::two(x, e);
          offer(f.x, first_vec + v * V::kN + 2 * e);
          offer(f.y, first_vec + v * V::kN + 2 * e + 1);
        }
      }
      if (tid < s.head) offer(V::one(s.row + int64_t(s.first + tid) * V::kBytes), s.first + tid);
      if (tid < s.tail) {
        const int col = first_vec + s.vecs * V::kN + tid;
        offer(V::one(s.row + int64_t(col) * V::kBytes), col);
      }
      __syncthreads();
    };
    collect(bound);
    int n = sh.found;
    if (n > kCandidates) {
      // more equal values than the list holds: those above the bound, then the lowest columns
      // that equal it
      __syncthreads();
      if (tid == 0) sh.found = 0;
      __syncthreads();
      collect(bound + 1);
      n = sh.found;
      one_by_one = n > kCandidates;
      if (n < k) {
        int need = k - n;
        for (int c = 0; c < columns && need > 0; c += kThreads) {
          const int i = c + tid;
          const bool tie = i < columns &&
                           order_of(V::one(s.row + int64_t((s.first + i)) * V::kBytes)) == bound;
          const unsigned ties = __ballot_sync(~0u, tie);
          if (lane == 0) sh.warp_count[warp] = __popc(ties);
          __syncthreads();
          int before = 0, total = 0;
          for (int w = 0; w < kThreads / 32; ++w) {
            before += w < warp ? sh.warp_count[w] : 0;
            total += sh.warp_count[w];
          }
          const int at = before + __popc(ties & ((1u << lane) - 1));
          if (tie && at < need) sh.cand[n + at] = key_of(bound, uint32_t((s.first + i)));
          n += min(need, total);
          need -= min(need, total);
          __syncthreads();
        }
      }
    }
    if (!one_by_one) rank_candidates(sh, n, k);
  }
  if (one_by_one) {
    // NaNs, or too many values above the bound: one after the other
    unsigned long long last = ~0ull;
    for (int j = 0; j < k; ++j) {
      if (tid == 0) sh.best = 0;
      __syncthreads();
      unsigned long long best = 0;
      for (int i = tid; i < columns; i += kThreads) {
        const unsigned long long key =
            key_of(order_of(V::one(s.row + int64_t((s.first + i)) * V::kBytes)), uint32_t((s.first + i)));
        if (key < last && key > best) best = key;
      }
#pragma unroll
      for (int x = 16; x; x /= 2) {
        const unsigned long long other = __shfl_xor_sync(~0u, best, x);
        best = other > best ? other : best;
      }
      if (lane == 0) atomicMax(&sh.best, best);
      __syncthreads();
      last = sh.best;
      if (tid == 0) sh.top[j] = last;
      __syncthreads();
      if (last == 0) break;     // the slice has no more columns
    }
  }
  __syncthreads();
}

template <int DTYPE>
__global__ void __launch_bounds__(kThreads, 2) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
  using V = Vec<DTYPE>;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int64_t r = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const char *row = a.logits + r * a.ld * V::kBytes;
  const Slice s = slice_of<DTYPE>(row, a.vocab, rank, ctas);
  const char *vec0 = row + int64_t(s.first + s.head) * V::kBytes;

  // the token's logit is wanted last: ask for it first
  long long token = -1;
  float given = -INFINITY;
  if (rank == 0 && tid == 0) {
    token = a.tokens[r];
    if (token >= 0 && token < a.vocab) given = V::one(row + token * V::kBytes);
  }

  Sums mine = {-INFINITY, 0.f, 0.f};
  {
    f32x2 sum[2] = {0, 0}, prod[2] = {0, 0};
    uint4 next[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int v = j * kThreads + tid;
      next[j] = v < s.vecs ? load16(vec0 + int64_t(v) * 16) : V::none();
    }
    for (int v0 = 0; v0 < s.vecs; v0 += kUnroll * kThreads) {
      uint4 x[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        x[j] = next[j];
        const int v = v0 + (kUnroll + j) * kThreads + tid;
        next[j] = v < s.vecs ? load16(vec0 + int64_t(v) * 16) : V::none();
      }
      float top = V::top(x[0]);
#pragma unroll
      for (int j = 1; j < kUnroll; ++j) top = max_nan(top, V::top(x[j]));
      if (!(top <= mine.m)) {
        const float d = fmaxf((mine.m - top) * kLog2e, kFloor);
        const f32x2 dd = pair(d, d), f = pair(exp2_fast(d), exp2_fast(d));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          prod[i] = mul2(fma2(dd, sum[i], prod[i]), f);
          sum[i] = mul2(sum[i], f);
        }
        mine.m = top;
      }
      const float ref = mine.m == -INFINITY ? 0.f : -mine.m;
      const f32x2 ref2 = pair(ref, ref), scale = pair(kLog2e, kLog2e);
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
#pragma unroll
        for (int e = 0; e < V::kN / 2; ++e) {
          const float2 f = V::two(x[j], e);
          const float2 y = halves(mul2(add2(pair(f.x, f.y), ref2), scale));
          const float y0 = fmaxf(y.x, kFloor), y1 = fmaxf(y.y, kFloor);
          const f32x2 w = pair(exp2_fast(y0), exp2_fast(y1));
          sum[e % 2] = add2(sum[e % 2], w);
          prod[e % 2] = fma2(pair(y0, y1), w, prod[e % 2]);
        }
    }
    const float2 s0 = halves(add2(sum[0], sum[1])), u0 = halves(add2(prod[0], prod[1]));
    mine.s = s0.x + s0.y;
    mine.u = u0.x + u0.y;
  }
  // the single columns at the ends: one per thread
  const auto single = [&](int col) {
    const float x = V::one(row + int64_t(col) * V::kBytes);
    join(mine, Sums{x, x == -INFINITY ? 0.f : 1.f, 0.f});
  };
  if (tid < s.head) single(s.first + tid);
  if (tid < s.tail) single(s.first + s.head + s.vecs * V::kN + tid);

  Sums all = mine;
#pragma unroll
  for (int x = 16; x; x /= 2) {
    Sums o;
    o.m = __shfl_xor_sync(~0u, all.m, x);
    o.s = __shfl_xor_sync(~0u, all.s, x);
    o.u = __shfl_xor_sync(~0u, all.u, x);
    join(all, o);
  }
  if (lane == 0) sh.warp[warp] = all;
  if (a.top > 0) top_of_slice<DTYPE>(sh, s, mine.m, a.top);
  else __syncthreads();
  if (warp == 0) {
    all = lane < kThreads / 32 ? sh.warp[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int x = kThreads / 64; x; x /= 2) {
      Sums o;
      o.m = __shfl_xor_sync(~0u, all.m, x);
      o.s = __shfl_xor_sync(~0u, all.s, x);
      o.u = __shfl_xor_sync(~0u, all.u, x);
      join(all, o);
    }
    if (lane == 0) sh.all = all;
  }

  // ---- join the cluster
  if (ctas > 1) {
    cluster.sync();
    if (rank == 0) {
      if (warp == 0) {
        all = lane < ctas ? cluster.map_shared_rank(&sh, lane)->all : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int x = kMaxCluster / 2; x; x /= 2) {
          Sums o;
          o.m = __shfl_xor_sync(~0u, all.m, x);
          o.s = __shfl_xor_sync(~0u, all.s, x);
          o.u = __shfl_xor_sync(~0u, all.u, x);
          join(all, o);
        }
      }
      for (int i = tid; i < ctas * a.top; i += kThreads)
        sh.merged[i] = cluster.map_shared_rank(&sh, i / a.top)->top[i % a.top];
    }
    cluster.sync();        // nobody leaves while its shared memory is read
    if (rank != 0) return;
    if (warp == 0 && lane == 0) sh.all = all;
    __syncthreads();
    unsigned long long key = 0;
    int above = kMaxTop;
    if (tid < ctas * a.top && (key = sh.merged[tid]) != 0) {
      above = 0;
      for (int j = 0; j < ctas * a.top; ++j) above += sh.merged[j] > key;
    }
    if (above < a.top) sh.top[above] = key;
  }
  __syncthreads();
  all = sh.all;
  const bool bad = !(all.m < INFINITY);                 // a NaN or +infinity in the row
  const bool empty = all.m == -INFINITY;
  const float log_s = log2f(all.s) * kLn2;
  const auto logp = [&](float x) {
    if (bad) return NAN;
    if (empty || x == -INFINITY) return -INFINITY;
    return x - all.m - log_s;
  };
  if (tid == 0) {
    a.logprob[r] = token >= 0 && token < a.vocab ? logp(given) : bad ? NAN : -INFINITY;
    a.entropy[r] = bad ? NAN : empty ? 0.f : kLn2 * (log2f(all.s) - all.u / all.s);
  }
  if (tid < a.top) {
    const unsigned long long key = sh.top[tid];
    a.top_token[r * a.top + tid] = 0xffffffffu - uint32_t(key);
    a.top_logprob[r * a.top + tid] = logp(value_of(uint32_t(key >> 32)));
  }
}

// CTAs per row: as many as fill the device a few times over, none with less than about one
// vector per thread.
int cluster_size(int rows, int vocab, int sms) {
  int c = 1;
  while (c < kMaxCluster && int64_t(rows) * c < 4 * int64_t(sms) && vocab / (2 * c) >= 4096) c *= 2;
  return c;
}

template <int DTYPE>
int launch_logprobs(const LogprobArgs &a, int rows, cudaStream_t st) {
  static std::atomic<int> sms_of[64];
  int device = -1;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || device < 0 || device >= 64)
    return op_fail(YPK_ERR_CUDA, "token_logprobs: no current device (%s)", cudaGetErrorString(e));
  int sms = sms_of[device].load(std::memory_order_relaxed);
  if (!sms) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess)   // clusters of sixteen are an option that has to be asked for
      e = cudaFuncSetAttribute(token_logprobs_kernel<DTYPE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "token_logprobs: set-up: %s", cudaGetErrorString(e));
    sms_of[device].store(sms, std::memory_order_relaxed);
  }
  const int c = cluster_size(rows, a.vocab, sms);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<DTYPE>, a);
  if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "token_logprobs: launch: %s", cudaGetErrorString(e));
  return YPK_OK;
}

}  // namespace
}  // namespace ypk

using namespace ypk;

extern "C" int ypk_token_logprobs(const void *logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t ld,
                                  const int64_t *tokens, int32_t top_k, float *logprob, float *entropy,
                                  float *top_logprob, int64_t *top_token, void *stream) {
  if (rows == 0) return YPK_OK;
  if (!logits || !tokens || !logprob || !entropy)
    return op_fail(YPK_ERR_INVALID, "token_logprobs: null logits, tokens or output");
  if (dtype != YPK_BF16 && dtype != YPK_F16 && dtype != YPK_F32)
    return op_fail(YPK_ERR_UNSUPPORTED, "token_logprobs: type %d (bf16, fp16 or fp32)", dtype);
  if (rows < 0 || vocab < 1 || ld < vocab)
    return op_fail(YPK_ERR_INVALID, "token_logprobs: %d rows, vocabulary %d, row stride %lld", rows, vocab,
                   (long long)ld);
  if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
    return op_fail(YPK_ERR_UNSUPPORTED, "token_logprobs: top_k %d (0..%d, at most the vocabulary)", top_k, kMaxTop);
  if (top_k > 0 && (!top_logprob || !top_token))
    return op_fail(YPK_ERR_INVALID, "token_logprobs: null output of the top alternatives");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == YPK_F32 ? 4 : 2))
    return op_fail(YPK_ERR_INVALID, "token_logprobs: logits are not aligned to their type");
  LogprobArgs a;
  a.logits = static_cast<const char *>(logits);
  a.tokens = reinterpret_cast<const long long *>(tokens);
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_logprob = top_logprob;
  a.top_token = reinterpret_cast<long long *>(top_token);
  a.ld = ld;
  a.vocab = vocab;
  a.top = top_k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == YPK_BF16) return launch_logprobs<YPK_BF16>(a, rows, st);
  if (dtype == YPK_F16) return launch_logprobs<YPK_F16>(a, rows, st);
  return launch_logprobs<YPK_F32>(a, rows, st);
}
