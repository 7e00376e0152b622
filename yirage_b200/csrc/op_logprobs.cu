// Log probabilities of given tokens, with entropy and top alternatives (ypk_token_logprobs).
//
//   y = x log2 e - r,  s = sum 2^y,  u = sum y 2^y      (r: the running maximum's x log2 e)
//   log2 p(t) = y_t - log2 s,   entropy = ln 2 (log2 s - u / s)
//
// One pass over the logits with r, s and u running in each thread's registers.  r is rounded, but
// the same rounded number stands in every y, so it cancels.  Memory bounds the pass only if it
// stays under about seven instructions a logit at 16 bits (four schedulers, 6.5 TB/s), and the
// exponential alone takes 73 % of its unit at that rate: so pairs of fp32 share an instruction
// (fma.f32x2), maxima and the clamp are taken on pairs of 16-bit values.  The clamp keeps
// -infinity out of the products: a column so low adds nothing while the maximum is above kLow; a
// row whose maximum is not, or is above kHigh, has only weights of 0 and 1, and its maxima are
// counted instead.
//
// The top alternatives cost the pass nothing.  Its running maxima, one per thread, give a bound:
// the k-th largest maximum of 64 groups of threads is at most the k-th largest logit.  Each turn
// of the pass also leaves its maximum per thread in shared memory (16 bits, rounded so that
// nothing is missed); only the turns that reach the bound, little more than k, are read
// again, from L2, and what reaches the bound there is ranked.  Rows full of equal values (a mask
// that leaves less than k columns) overflow that list; they take the slow way: the logits above
// the bound and then the lowest columns that equal it.
//
// A row is split over a cluster of CTAs when there are few rows; bounds, sums and candidates
// travel through distributed shared memory, so there is no workspace and no second launch.
//
// Measured, called back to back, bf16 unless said: 4096 x 128256 without alternatives 182 to 194 us
// = 5.4 to 5.8 TB/s, with the SM clock lowered to 1.6 GHz by the card's power cap (special-function
// unit 73 % busy, issue slots 59 %; 161 us, the copy rate, while the clock is up); with 20
// alternatives 187.  333 x 50021 fp32, 8 alternatives 18.7 us: 12 to stream at 2.25 CTAs per SM, as
// a row is one CTA from 223 rows on, then 1.6 for the bound, 1.4 for the candidates.  64 x 151936, 20
// alternatives 12.1 us; 1 x 128256, 5 alternatives 6.35 us, latency.
// Exponentials as polynomials for a quarter of the pairs: 204 against 190 us at the cap.
#include <cooperative_groups.h>
#include <math.h>

#include <atomic>

#include "op_common.h"
#include "op_num.cuh"

namespace cg = cooperative_groups;

namespace ypk {
namespace {

constexpr int kMaxTop = 32;
constexpr int kMaxVocab = 1 << 30;  // columns are counted in 32 bits, a stride of threads past the last one
constexpr int kGroups = 64;        // of threads: what the bound of a top list is taken from
constexpr int kMaxGroups = 128;    // over a cluster
constexpr int kCandidates = 1024;
constexpr int kUnroll = 4;         // 16-byte loads in flight per thread (and as many ahead)
constexpr int kSlots = 32;         // remembered turns of the pass (several share one beyond that)
constexpr int kMaxEntries = 512;   // (thread, slot) pairs to be read again
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
// Exponents below this add nothing to a sum that holds a 1.
constexpr float kFloor = -200.f;
// Beyond kHigh (and below Vec::kLow) neighbouring values are at least 32 apart: weights are 0 or 1.
// Up to there the rounding of the reference shifts every y by at most 2^-24 of it, under 100.
constexpr float kHigh = 0x1p30f;

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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The reference of sums whose largest value is x.  Rounded here and nowhere else: a product that the
// compiler fused into what is subtracted from it would not be the number that stands in every y.
__device__ __forceinline__ float reference(float x) { return __fmul_rn(x, kLog2e); }
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN on either side stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint4 load16(const char *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// Where `valid`; else v stays.  (By a predicate: the asm in four branches cost two kernels a few bytes
// of spills.)
__device__ __forceinline__ void load16_if(uint4 &v, const char *p, bool valid) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
               "@q ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "l"(p), "r"(unsigned(valid)) : "memory");
}

// One 16-byte vector of logits.
template <int DTYPE>
struct Vec;
template <>
struct Vec<YPK_F32> {
  static constexpr int kN = 4, kBytes = 4;
  static constexpr float kLow = -0x1p30f;
  static __device__ __forceinline__ uint32_t clamp1(uint32_t v) {
    return __float_as_uint(fmaxf(__uint_as_float(v), -0x1p34f));
  }
  static __device__ __forceinline__ uint4 clamp(const uint4 &v) {
    return make_uint4(clamp1(v.x), clamp1(v.y), clamp1(v.z), clamp1(v.w));
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ float top(const uint4 &v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint4 larger(const uint4 &a, const uint4 &b) {      // element by element
    return make_uint4(larger1(a.x, b.x), larger1(a.y, b.y), larger1(a.z, b.z), larger1(a.w, b.w));
  }
  static __device__ __forceinline__ uint32_t larger1(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return i ? make_float2(__uint_as_float(v.z), __uint_as_float(v.w)) : make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
  }
  static __device__ __forceinline__ float one(const char *p) { return *reinterpret_cast<const float *>(p); }
};
template <>
struct Vec<YPK_BF16> {
  static constexpr int kN = 8, kBytes = 2;
  static constexpr float kLow = -0x1p30f;
  static __device__ __forceinline__ uint32_t clamp2(uint32_t v) {      // to -2^34
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xd080d080u));
    return r;
  }
  static __device__ __forceinline__ uint4 clamp(const uint4 &v) {
    return make_uint4(clamp2(v.x), clamp2(v.y), clamp2(v.z), clamp2(v.w));
  }
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
  static __device__ __forceinline__ uint4 larger(const uint4 &a, const uint4 &b) {
    return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return OpBf16::widen(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float one(const char *p) {
    return __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(p));
  }
};
template <>
struct Vec<YPK_F16> {
  static constexpr int kN = 8, kBytes = 2;
  static constexpr float kLow = -60000.f;
  static __device__ __forceinline__ uint32_t clamp2(uint32_t v) {      // to the lowest value, -65504
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xfbfffbffu));
    return r;
  }
  static __device__ __forceinline__ uint4 clamp(const uint4 &v) {
    return make_uint4(clamp2(v.x), clamp2(v.y), clamp2(v.z), clamp2(v.w));
  }
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
  static __device__ __forceinline__ uint4 larger(const uint4 &a, const uint4 &b) {
    return make_uint4(max2(a.x, b.x), max2(a.y, b.y), max2(a.z, b.z), max2(a.w, b.w));
  }
  static __device__ __forceinline__ float2 two(const uint4 &v, int i) {
    return OpF16::widen(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float one(const char *p) {
    return __half2float(*reinterpret_cast<const __half *>(p));
  }
};

// Sums against a reference, and the true maximum (NaN if there is one).
struct Sums {
  float r, s, u, top;
};
constexpr Sums kNoSums = {-INFINITY, 0.f, 0.f, -INFINITY};

__device__ __forceinline__ void join(Sums &a, const Sums &b) {
  const float r = fmaxf(a.r, b.r);
  const float da = fmaxf(a.r - r, kFloor), db = fmaxf(b.r - r, kFloor);   // (none yet: NaN or -infinity, s = 0)
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  a.u = (a.u + da * a.s) * fa + (b.u + db * b.s) * fb;
  a.s = a.s * fa + b.s * fb;
  a.r = r;
  a.top = max_nan(a.top, b.top);
}

__device__ __forceinline__ Sums shuffled(const Sums &a, int x) {
  Sums o;
  o.r = __shfl_xor_sync(~0u, a.r, x);
  o.s = __shfl_xor_sync(~0u, a.s, x);
  o.u = __shfl_xor_sync(~0u, a.u, x);
  o.top = __shfl_xor_sync(~0u, a.top, x);
  return o;
}

template <int THREADS>
struct SharedOf {
  Sums warp[THREADS / 32];
  Sums row;                               // of the whole row
  alignas(16) uint32_t part[kGroups];     // maxima of this CTA's groups of threads
  alignas(16) uint32_t group[kMaxGroups]; // of the row's
  uint32_t bound;
  int slow;                               // the row has a NaN, or too many candidates
  int listed, found;
  uint32_t entry[kMaxEntries];            // slot << 16 | thread: columns to be read again
  uint16_t slot_max[kSlots][THREADS];    // upper half of the order of a turn's maximum
  unsigned long long cand[kCandidates];
  unsigned long long top[kMaxTop];        // falling; 0: none
  unsigned long long best;
  unsigned long long merged[kMaxCluster * kMaxTop];
  int warp_count[THREADS / 32];
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

// The k largest of n keys in order into sh.top; every thread calls.
template <int THREADS>
__device__ void rank_keys(SharedOf<THREADS> &sh, const unsigned long long *keys, int n, int k) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long mine = keys[i];
    if (mine == 0) continue;
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < k) sh.top[above] = mine;
  }
}

// Lists the slots of this thread that reach the bound.
template <int THREADS>
__device__ __forceinline__ void list_slots(SharedOf<THREADS> &sh, int slots, uint32_t bound) {
  for (int i0 = 0; i0 < slots; i0 += 4) {
    uint32_t most[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) most[i] = sh.slot_max[min(i0 + i, slots - 1)][threadIdx.x];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + i < slots && most[i] >= bound >> 16) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < kMaxEntries) sh.entry[at] = uint32_t(i0 + i) << 16 | threadIdx.x;
      }
  }
}

// Puts the columns of this CTA's slice that are at least `least` in order into the list of `to`
// (counted in to.found, as far as there is room), from the listed slots of `each` vectors.
template <int DTYPE, int THREADS>
__device__ __forceinline__ void collect(SharedOf<THREADS> &sh, SharedOf<THREADS> &to, const Slice &s, int listed,
                                        int each, uint32_t least) {
  using V = Vec<DTYPE>;
  constexpr int kThreads = THREADS;
  const int tid = threadIdx.x, first_vec = s.first + s.head;
  const char *vec0 = s.row + int64_t(first_vec) * V::kBytes;
  const auto offer = [&](float x, int col) {
    const uint32_t o = order_of(x);
    if (o < least) return;
    const int at = atomicAdd(&to.found, 1);
    if (at < kCandidates) to.cand[at] = key_of(o, uint32_t(col));
  };
  for (int i = tid; i < listed * each; i += kThreads) {
    const int k = each == kUnroll ? i / kUnroll : i / each;
    const uint32_t e = sh.entry[k];
    const int v = (int(e >> 16) * each + i - k * each) * kThreads + int(e & 0xffffu);
    if (v >= s.vecs) continue;
    const uint4 x = load16(vec0 + int64_t(v) * 16);
    if (order_of(V::top(x)) < least) continue;
#pragma unroll
    for (int k = 0; k < V::kN / 2; ++k) {
      const float2 f = V::two(x, k);
      offer(f.x, first_vec + v * V::kN + 2 * k);
      offer(f.y, first_vec + v * V::kN + 2 * k + 1);
    }
  }
  if (tid < s.head) offer(V::one(s.row + int64_t(s.first + tid) * V::kBytes), s.first + tid);
  if (tid < s.tail) {
    const int col = first_vec + s.vecs * V::kN + tid;
    offer(V::one(s.row + int64_t(col) * V::kBytes), col);
  }
}

// The k-th largest of n group maxima, or a little less: the lower bits make way for the group's
// number, so that no two are alike.  Every thread calls; sh.bound is there after a barrier.
template <int THREADS>
__device__ __forceinline__ void find_bound(SharedOf<THREADS> &sh, int n, int k) {
  const int tid = threadIdx.x;
  if (tid >= n) return;
  const uint32_t mine = sh.group[tid];
  int above = 0;
#pragma unroll 8
  for (int j = 0; j < n; j += 4) {
    const uint4 g = *reinterpret_cast<const uint4 *>(sh.group + j);
    above += (g.x > mine) + (g.y > mine) + (g.z > mine) + (g.w > mine);
  }
  if (above == k - 1) sh.bound = mine & ~uint32_t(kMaxGroups - 1);
}
__device__ __forceinline__ uint32_t group_key(uint32_t order, int group) {
  return (order & ~uint32_t(kMaxGroups - 1)) | uint32_t(group);
}

// The slow way: the k largest of this CTA's slice, exactly, into sh.top.
template <int DTYPE, int THREADS>
__device__ __forceinline__ void top_of_slice(SharedOf<THREADS> &sh, const Slice &s, float my_max, int k) {
  using V = Vec<DTYPE>;
  constexpr int kThreads = THREADS, kWarps = THREADS / 32;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int columns = s.head + s.vecs * V::kN + s.tail;
  const uint32_t mine = order_of(my_max);
  uint32_t g = mine;
#pragma unroll
  for (int x = 1; x < kThreads / kGroups; x *= 2) g = max(g, __shfl_xor_sync(~0u, g, x));
  __syncthreads();
  if (tid % (kThreads / kGroups) == 0) sh.group[tid / (kThreads / kGroups)] = g;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.listed = sh.found = 0;
  // a NaN hides its thread's other columns from the maxima
  bool one_by_one = __syncthreads_or(my_max != my_max);
  if (!one_by_one) {
    if (tid < kGroups) {
      // a bound that is one of the values: ties are told from what is above
      const uint32_t gi = sh.group[tid];
      int above = 0;
      for (int j = 0; j < kGroups; ++j) above += sh.group[j] > gi || (sh.group[j] == gi && j < tid);
      if (above == k - 1) sh.bound = gi;
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (mine >= bound) sh.entry[atomicAdd(&sh.listed, 1)] = tid;      // all of its vectors: one slot
    __syncthreads();
    const int listed = sh.listed, rounds = (s.vecs + kThreads - 1) / kThreads;
    collect<DTYPE, THREADS>(sh, sh, s, listed, rounds, bound);
    __syncthreads();
    int n = sh.found;
    if (n > kCandidates) {
      // more equal values than the list holds: those above the bound, then the lowest columns
      // that equal it
      __syncthreads();
      if (tid == 0) sh.found = 0;
      __syncthreads();
      collect<DTYPE, THREADS>(sh, sh, s, listed, rounds, bound + 1);
      __syncthreads();
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
          for (int w = 0; w < kWarps; ++w) {
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
    if (!one_by_one) rank_keys(sh, sh.cand, n, k);
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

// What one thread has seen of its columns.
template <int DTYPE>
struct Running {
  using V = Vec<DTYPE>;
  f32x2 sum[2] = {0, 0}, prod[2] = {0, 0};
  float m = -INFINITY;      // largest value that the reference was taken from
  float r = -INFINITY;      // fl(m log2 e)
  float top = -INFINITY;    // largest value at all, or NaN

  template <int N>
  __device__ __forceinline__ float take(const uint4 (&x)[N]) {      // the largest of x
    uint4 most = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) most = V::larger(most, x[j]);
    const float t = V::top(most);
    top = max_nan(top, t);
    if (!(t >= V::kLow)) return t;      // nothing here that counts beside a higher value
    if (t > m) {
      m = t;
      const float next = reference(t), d = fmaxf(r - next, kFloor);
      const float f = exp2_fast(d);
      const f32x2 dd = pair(d, d), ff = pair(f, f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        prod[i] = mul2(fma2(dd, sum[i], prod[i]), ff);
        sum[i] = mul2(sum[i], ff);
      }
      r = next;
    }
    const f32x2 ref = pair(-r, -r), scale = pair(kLog2e, kLog2e);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint4 c = V::clamp(x[j]);
#pragma unroll
      for (int e = 0; e < V::kN / 2; ++e) {
        const float2 f = V::two(c, e);
        const f32x2 y = fma2(pair(f.x, f.y), scale, ref);
        const float2 yy = halves(y);
        const f32x2 w = pair(exp2_fast(yy.x), exp2_fast(yy.y));
        sum[e % 2] = add2(sum[e % 2], w);
        prod[e % 2] = fma2(y, w, prod[e % 2]);
      }
    }
    return t;
  }

  __device__ __forceinline__ Sums sums() const {
    const float2 s0 = halves(add2(sum[0], sum[1])), u0 = halves(add2(prod[0], prod[1]));
    return Sums{r, s0.x + s0.y, u0.x + u0.y, top};
  }
};

template <int DTYPE, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
  using V = Vec<DTYPE>;
  using Shared = SharedOf<THREADS>;
  constexpr int kThreads = THREADS, kWarps = THREADS / 32;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int64_t r = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const char *row = a.logits + r * a.ld * V::kBytes;
  const Slice s = slice_of<DTYPE>(row, a.vocab, rank, ctas);
  op_wait_for_previous();          // (no memory is touched above)
  const auto meet = [&]() {        // the row's CTAs, or this one's threads
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };

  long long token = -1;
  float given = -INFINITY;
  if (rank == 0 && tid == 0) token = a.tokens[r];
  if (tid == 0) sh.listed = sh.found = sh.slow = 0;

  // ---- the pass: kUnroll vectors per thread at a time, the next ones on their way
  Sums mine;
  const int turns = s.vecs / (kUnroll * kThreads) + 1;               // the last one has bounds to check
  const int turns_per_slot = (turns + kSlots - 1) / kSlots;
  {
    Running<DTYPE> run;
    const char *p = row + int64_t(s.first + s.head) * V::kBytes + tid * 16;
    const int whole = turns - 1;
    float slot_top = -INFINITY;
    int slot = 0, in_slot = 0;
    const auto remember = [&](float t) {
      if (!TOP) return;
      slot_top = fmaxf(slot_top, t);
      if (++in_slot < turns_per_slot) return;
      sh.slot_max[slot++][tid] = uint16_t(order_of(slot_top) >> 16);
      slot_top = -INFINITY;
      in_slot = 0;
    };
    int left = s.vecs - whole * (kUnroll * kThreads) - tid; // of the last turn, for this thread
    uint4 next[kUnroll];
    const auto fetch_whole = [&]() {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) next[j] = load16(p + j * (kThreads * 16));
      p += kUnroll * kThreads * 16;
    };
    const auto fetch_last = [&]() {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        next[j] = V::none();
        load16_if(next[j], p + j * (kThreads * 16), j * kThreads < left);
      }
    };
    if (whole > 0) fetch_whole();
    else fetch_last();
    for (int i = 0; i < whole; ++i) {
      uint4 x[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) x[j] = next[j];
      if (i + 1 < whole) fetch_whole();
      else fetch_last();
      remember(run.take(x));
    }
    remember(run.take(next));
    if (TOP && in_slot > 0) sh.slot_max[slot][tid] = uint16_t(order_of(slot_top) >> 16);
    mine = run.sums();
  }
  // (wanted at the very end; before the pass its address would have been waited for)
  if (token >= 0 && token < a.vocab) given = V::one(row + token * V::kBytes);
  // the single columns at the ends, one per thread of the first and the second warp: against the
  // reference that Running::take has for such a value, so that the same y of the largest column
  // stands in its weight and in `peak`
  const int behind = tid - 32;
  const int col = tid < s.head ? s.first + tid
                  : behind >= 0 && behind < s.tail ? s.first + s.head + s.vecs * V::kN + behind : -1;
  if (col >= 0) {
    const float x = V::one(row + int64_t(col) * V::kBytes);
    Sums one = {-INFINITY, 0.f, 0.f, x};
    if (x >= V::kLow) {
      const float ref = reference(x), y = fmaf(x, kLog2e, -ref), w = exp2_fast(y);
      one = Sums{ref, w, y * w, x};
    }
    join(mine, one);
  }

  // ---- sums and bounds of the threads, together
  const uint32_t order = order_of(mine.top);
  const int span = min(32, kThreads / kGroups * ctas);     // threads per group: 64 groups a row, or 128
  const int parts = kThreads / span;
  if (TOP) {
    uint32_t g = mine.top != mine.top ? 0xffffffffu : order;    // (a NaN is no order's: it shows)
#pragma unroll
    for (int x = 1; x < 32; x *= 2)
      if (x < span) g = max(g, __shfl_xor_sync(~0u, g, x));
    if (tid % span == 0) sh.part[tid / span] = g;
  }
  Sums all = mine;
#pragma unroll
  for (int x = 16; x; x /= 2) join(all, shuffled(all, x));
  if (lane == 0) sh.warp[warp] = all;
  meet();
  // the last warp joins the row's sums, beside the others' reading
  const auto join_row = [&]() {
    if (rank != 0 || warp != kWarps - 1) return;
    all = kNoSums;
    for (int i = lane; i < ctas * kWarps; i += 32)
      join(all, ctas > 1 ? cluster.map_shared_rank(&sh, i / kWarps)->warp[i % kWarps] : sh.warp[i]);
#pragma unroll
    for (int x = 16; x; x /= 2) join(all, shuffled(all, x));
    if (lane == 0) sh.row = all;
  };
  if (!TOP) join_row();
  if (TOP) {
    Shared *leader = rank > 0 ? cluster.map_shared_rank(&sh, 0) : &sh;
    const int groups = parts * ctas;
    uint32_t g = 0;
    if (tid < groups) {
      g = ctas > 1 ? cluster.map_shared_rank(&sh, tid / parts)->part[tid % parts] : sh.part[tid];
      sh.group[tid] = group_key(g, tid);
      if (g == 0xffffffffu) sh.slow = 1;
    }
    if (tid < kMaxTop) sh.top[tid] = 0;
    __syncthreads();
    find_bound(sh, groups, a.top);
    const bool slow = sh.slow != 0;
    __syncthreads();
    if (!slow) {
      const uint32_t bound = sh.bound;
      if (order >= bound) list_slots(sh, (turns + turns_per_slot - 1) / turns_per_slot, bound);
      __syncthreads();
      const int listed = sh.listed;
      if (listed <= kMaxEntries) collect<DTYPE, THREADS>(sh, *leader, s, listed, turns_per_slot * kUnroll, bound);
      else if (tid == 0) atomicAdd(&leader->found, kCandidates + 1);      // too many: the slow way
    }
    join_row();
    meet();
    const int n = leader->found;
    if (slow || n > kCandidates) {
      // (all CTAs of the row see the same)
      meet();          // everybody has read `found`
      top_of_slice<DTYPE, THREADS>(sh, s, mine.top, a.top);
      meet();
      if (rank == 0) {
        for (int i = tid; i < ctas * a.top; i += kThreads)
          sh.merged[i] = ctas > 1 ? cluster.map_shared_rank(&sh, i / a.top)->top[i % a.top] : sh.top[i];
        __syncthreads();
        rank_keys(sh, sh.merged, ctas * a.top, a.top);
      }
    } else if (rank == 0) {
      rank_keys(sh, sh.cand, n, a.top);
    }
  }
  if (ctas > 1) {
    cluster.sync();          // nobody leaves while its shared memory is read
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // ---- results
  all = sh.row;
  const bool bad = !(all.top < INFINITY);               // a NaN or +infinity in the row
  const bool empty = all.top == -INFINITY;
  const bool ends = !bad && !empty && (all.top < V::kLow || all.top > kHigh);   // weights of 0 and 1
  if (ends) {
    if (tid == 0) sh.found = 0;
    __syncthreads();
    int count = 0;
    for (int i = tid; i < a.vocab; i += kThreads) count += V::one(row + int64_t(i) * V::kBytes) == all.top;
    atomicAdd(&sh.found, count);
    __syncthreads();
    all.s = float(sh.found);
    all.u = 0.f;
  }
  const float log2_s = log2f(all.s);
  // log p of the most probable column; the others lie x - max below it
  const float peak = kLn2 * ((ends ? 0.f : fmaf(all.top, kLog2e, -all.r)) - log2_s);
  const auto logp = [&](float x) {
    if (bad) return NAN;
    if (empty || x == -INFINITY) return -INFINITY;
    return (x - all.top) + peak;
  };
  if (tid == 0) {
    a.logprob[r] = token >= 0 && token < a.vocab ? logp(given) : bad ? NAN : -INFINITY;
    a.entropy[r] = bad ? NAN : empty ? 0.f : fmaxf(0.f, kLn2 * (log2_s - all.u / all.s));
  }
  if (TOP && tid < a.top) {
    const unsigned long long key = sh.top[tid];
    a.top_token[r * a.top + tid] = 0xffffffffu - uint32_t(key);
    a.top_logprob[r * a.top + tid] = logp(value_of(uint32_t(key >> 32)));
  }
}

// CTAs per row: up to three per SM in all (of sixteen a row one: a cluster lies in one GPC, and so
// large ones leave SMs without work), none with less than about two vectors per thread.  (64 x
// 151936: four CTAs a row 11.5 us, eight 12.9; 200 x 128256: two 17.9, one 19.9; sixteen against
// eight: 2 x 128256 6.1 / 6.35 us, 8 6.6 / 6.4, 24 8.6 / 7.55.)
int cluster_size(int rows, int vocab, int sms) {
  int c = 1;
  while (c < kMaxCluster && int64_t(rows) * 2 * c <= (c < kMaxCluster / 2 ? 3 : 1) * int64_t(sms) &&
         vocab / (2 * c) >= 4096)
    c *= 2;
  return c;
}

template <int DTYPE, bool TOP, int THREADS>
int launch_shape(const LogprobArgs &a, int rows, const DeviceInfo &dev, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};      // devices where clusters of sixteen have been asked for
  auto *kernel = token_logprobs_kernel<DTYPE, TOP, THREADS>;
  if (!(ready.load(std::memory_order_relaxed) >> dev.device & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "token_logprobs: set-up: %s", cudaGetErrorString(e));
    ready.fetch_or(uint64_t(1) << dev.device, std::memory_order_relaxed);
  }
  const int c = cluster_size(rows, a.vocab, dev.sms);
  return op_launch("token_logprobs", kernel, dim3(unsigned(rows) * c), THREADS, 0, c, st, a);
}

// With alternatives wanted and more rows than 256-thread CTAs are resident, CTAs of 128 threads:
// their phases without loads overlap with more others' (2000 x 32003 38 us against 46, 4096 x 128256
// 182 against 189; 333 x 50021 19.0 against 18.4).
template <int DTYPE>
int launch_logprobs(const LogprobArgs &a, int rows, cudaStream_t st) {
  DeviceInfo dev;
  if (int rc = op_device("token_logprobs", &dev)) return rc;
  if (!a.top) return launch_shape<DTYPE, false, 256>(a, rows, dev, st);
  return rows > 4 * dev.sms ? launch_shape<DTYPE, true, 128>(a, rows, dev, st)
                        : launch_shape<DTYPE, true, 256>(a, rows, dev, st);
}

}  // namespace
}  // namespace ypk

using namespace ypk;

extern "C" int ypk_token_logprobs(const void *logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t ld,
                                  const int64_t *tokens, int32_t top_k, float *logprob, float *entropy,
                                  float *top_logprob, int64_t *top_token, void *stream) {
  if (dtype != YPK_BF16 && dtype != YPK_F16 && dtype != YPK_F32)
    return op_fail(YPK_ERR_UNSUPPORTED, "token_logprobs: type %d (bf16, fp16 or fp32)", dtype);
  if (rows < 0 || vocab < 1 || ld < vocab)
    return op_fail(YPK_ERR_INVALID, "token_logprobs: %d rows, vocabulary %d, row stride %lld", rows, vocab,
                   (long long)ld);
  if (vocab > kMaxVocab)
    return op_fail(YPK_ERR_UNSUPPORTED, "token_logprobs: vocabulary %d (at most %d)", vocab, kMaxVocab);
  if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
    return op_fail(YPK_ERR_UNSUPPORTED, "token_logprobs: top_k %d (0..%d, at most the vocabulary)", top_k, kMaxTop);
  if (rows == 0) return YPK_OK;      // (nothing to read or write: pointers may be null)
  if (!logits || !tokens || !logprob || !entropy)
    return op_fail(YPK_ERR_INVALID, "token_logprobs: null logits, tokens or output");
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
