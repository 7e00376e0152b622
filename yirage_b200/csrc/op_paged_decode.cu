// Attention of one new token per request over a paged cache (ypk_paged_decode).
//
//   out = sum_p w_p v_p / sum_p w_p,  w_p = 2^(y_p - m),  y_p = scale log2(e) q.k_p
//
// Every K and V row is read once, 2 len Hkv D elements in all, against 4 len Hq D operations: at
// four query heads per K/V head that is 4 operations per byte, so memory bounds it and the
// arithmetic only has to stay out of the way.  It goes to the tensor cores as mma m16n8k16 with
// the sixteen cached tokens on the M side and the query heads of the group as the N side
// (S^T = K Q^T, O^T = V^T P^T): a block of 16 tokens costs the same for one head as for eight.
//
// Work.  The unit is a block of 16 tokens of one (request, K/V head); all units of the call, in
// that order, are cut into equal ranges, one per CTA and one CTA per SM, whatever the lengths
// are: the lengths are read on the device, so the same captured launch serves every step.  (The end
// of a segment counts as work, too: kSegmentUnits.)  A
// (request, head) inside one range is finished there; of one that crosses ranges every CTA
// leaves (m, sum, O) in the workspace and a second, dependent launch joins them in range order.
// No atomics: the result does not depend on who comes first.  (Joining inside the kernel by
// whoever comes last measured 2 to 10 us more than the launch: three round trips to L2 with
// fences between them.)  Where a batch is short, clusters of CTAs take its (request, head)s
// instead and join through distributed shared memory: one launch, no workspace.
//
// Inside a CTA warp w takes the blocks w, w + 8, ...; each warp has its own ring of S blocks in
// shared memory that it fills with 16-byte cp.async and reads with ldmatrix, so no barrier is
// needed until a (request, head) ends and the warps' states are merged; the ring runs on
// across that boundary.  Where the (request, head)s are many and short, each warp has a range of
// its own instead (kManyShort) and only what crosses warps is merged, once, at the end.
//
// Measured, K/V heads of 128, bf16: 64 x 4096 tokens, 32 query / 8 K/V heads 174 to 177 us = 6.1 TB/s
// (93 % of the copy rate; 164 while the SM clock is up); 8 x 4096 30 us = 4.5 TB/s, of which about 8 us are not streaming: launch
// 1, lengths and range 1.5, page numbers 0.6, first rows 1.5, uneven end 2, merge and join 3;
// 1 x 513 6.3 us, latency throughout.  What did not help: warps on different K/V heads
// (64 x 4096 with 64 query heads 184 against 170 us), two CTAs of four warps per SM (8 x 4096 32.6
// against 30.9), a ring of two blocks (64 x 4096 177 against 169).
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "op_paged.h"

namespace cg = cooperative_groups;

namespace ypk {
namespace {

struct DecodeArgs {
  PagedView c;
  const char *q;
  char *out;
  float *lse;
  int64_t q_token, q_group, q_head, o_token, o_group, o_head;
  int rows, q_heads, group, window;
  int ctas;            // per (request, pass) where clusters are used
  int head_blocks;     // passes over a K/V head's rows: ceil(group / (8 NT))
  int heads_per_pass;  // query heads of one pass, at most 8 NT
  FastDivisor page_div;
  float scale_log2;
  // workspace
  int join_heads;      // a block of the join
  int by_segment;      // the segments are few: desc is indexed by segment, not by worker
  int4 *desc;          // {request, pass, parts, worker}: a segment in several parts, the first that
                       // worker's; parts = 0: nothing to join
  float2 *part_ml;     // [workers][2][heads_per_pass] {m, sum}
  float *part_o;       // [workers][2][heads_per_pass][D]
};

constexpr int kBlock = 16;             // tokens per unit of work
// Units a CTA should have at least before the work is spread over more CTAs: two per warp.  (Four:
// the same within 2 % from 1 x 8192 to 16 x 1000 tokens.)
constexpr int kMinUnits = 16;
// Shares shorter than this are cut at the ends of segments if they can be: a second segment in a
// range costs a merge, 2 to 2.5 us.  16 x 1000 tokens (63 blocks a segment) 17.0 us with the cut
// moved, 20.3 with equal shares; from 8 x 4096 on equal shares win.
constexpr int kAlignUnits = 80;
// Segments of at most this many blocks are not cut: they go whole to the range that holds the
// larger part of them (64 x 60 tokens, four blocks a segment: 14.6 us, 18.8 with cuts).
constexpr int kSnapUnits = 16;
// What the end of a segment costs a CTA, its merge, in blocks: so much longer a segment counts when
// the work is cut.  64 requests of 1 to 8192 tokens, where some ranges hold twenty segments and
// some one: 178 us without, 172 at 8, 170 from 12 to 20, 173 at 28; 8 x 4096 29.6 to 28.9.
constexpr int kSegmentUnits = 16;
// Where segments are many and short, each warp has a range of its own and finishes the segments in it
// by itself, without merges: from kManyShort segments a CTA on if they have up to kShortBlocks
// blocks on average, from kManyTiny on if up to kTinyBlocks.  Ranges of CTAs against ranges of
// warps, 8 K/V heads: 256 requests of up to 200 tokens 54.6 / 34.9 us, 148 x 250 39.9 / 33.0, 128 x 512
// 53.8 / 49.3, 74 x 250 24.5 / 23.6, 64 x 60 16.1 / 12.7; but 64 x 300 27.0 / 28.2, 40 x 250
// 19.5 / 22.7, 64 x 700 39.9 / 45.3.
constexpr int kManyShort = 4, kShortBlocks = 32;
constexpr int kManyTiny = 2, kTinyBlocks = 4;
// There, what the end of a segment costs a warp, and what is not cut.  (At 16: 256 requests of up to 500
// tokens 59.7 us against 63.8, but 128 x 512 58.8 against 49.3: merges at every warp's ends.)
constexpr int kApartEndUnits = 2;
constexpr int kApartSnapUnits = 32;
constexpr int kMaxCluster = 8;

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<OpBf16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<OpF16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 8 x 8 matrix of 16-bit values, one row per four lanes: transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Factor of a part's sums when parts are joined.  Never 0 for a part that has weight: an infinity
// among its sums stays one.  (2^-126 of anything finite is nothing beside the largest weight.)
__device__ __forceinline__ float part_factor(float part_sum, float part_max, float top) {
  return part_sum == 0.f ? 0.f : fmaxf(exp2_fast(part_max - top), 0x1p-126f);   // (a NaN sum stays one)
}

// 16 bytes to shared memory; `valid` false writes zeros and reads nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const char *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// 64-bit division is a subroutine of a hundred instructions; the numbers here nearly always fit 32.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : int64_t(uint32_t(a) / uint32_t(b));
}

// The units of a call cut into equal ranges: worker w's begins at floor(total w / workers).  A
// segment's units are its blocks and then kSegmentUnits without work.
struct Ranges {
  int64_t total, each;
  int workers, more;       // total = each workers + more
  __device__ __forceinline__ int64_t start(int w) const {
    return each * w + uint32_t(more) * uint32_t(w) / uint32_t(workers);
  }
  __device__ __forceinline__ int owner(int64_t u) const {   // the worker whose range u lies in
    int w = int(min(int64_t(workers - 1), divide(u, each)));   // (each <= a range: not too low)
    while (start(w) > u) --w;
    return w;
  }
};

// One (request, pass) as far as it lies in a CTA's range: blocks [ja, jb) of its nb.
struct Segment {
  int64_t left;     // units of the range behind this segment
  int r, pass, ja, jb, nb, b0, len, lo, first;
};

template <int NW, int D, int NT, int S>
struct DecodeShape {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTile = kBlock * kRowBytes;     // one of K, V
  static constexpr int kRing = NW * S * 2 * kTile;
  // warps' states at a merge: m and sum, then O
  static int merge_bytes(int heads) { return NW * heads * (8 + D * 4); }
  static int bytes(int heads, int rows) { return kRing + merge_bytes(heads) + NW * S * 4 + rows * 8; }
};

// Infinities of either sign (a NaN counts as both) that V holds for the positions of blocks j0,
// j0 + step, ... < j1 of a request: bit d, bit 16 + d: dimension 16 d + lane / 4, and that + 8.
template <class T, int D>
__device__ __noinline__ uint2 infinities(const DecodeArgs &a, int first_page, int lo, int len, int j0, int j1,
                                         int step, int kv) {
  constexpr uint32_t kExponent = std::is_same<T, OpF16>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x % 32;
  uint2 found = make_uint2(0u, 0u);
  for (int j = j0; j < j1; j += step)
    for (int pos = max(lo, j * kBlock); pos < min(len, (j + 1) * kBlock); ++pos) {
      const int q = fast_div(pos, a.page_div), page = a.c.indices[first_page + q];
      const int64_t row = paged_row(page, a.c.num_pages, pos - q * a.c.page_size, a.c.stride_page, a.c.stride_token);
      if (row < 0) continue;
      const uint16_t *v = reinterpret_cast<const uint16_t *>(a.c.v) + row + kv * a.c.stride_head + lane / 4;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t x = v[8 * i], size = x & 0x7fffu;
        if (size < kExponent) continue;
        const uint32_t bit = 1u << (i / 2 + i % 2 * 16);
        if (size > kExponent || !(x >> 15)) found.x |= bit;
        if (size > kExponent || x >> 15) found.y |= bit;
      }
    }
  return found;
}

// CLUSTER: one cluster of CTAs per (request, pass) instead of equal ranges: the CTAs share its
// blocks evenly and join through distributed shared memory.  One launch, no workspace.
template <class T, int NW, int D, int NT, int S, bool CLUSTER>
__global__ void __launch_bounds__(NW * 32, 1) paged_decode_kernel(const __grid_constant__ DecodeArgs a) {
  using Shape = DecodeShape<NW, D, NT, S>;
  constexpr int kThreads = NW * 32;
  constexpr int kChunks = D / 8;                  // 16-byte chunks per row
  // P in fp16 keeps a few powers of two of head room below: weights down to 2^-31 of the largest
  // survive (bf16 has fp32's range)
  constexpr float kShift = std::is_same<T, OpF16>::value ? 7.f : 0.f;
  extern __shared__ __align__(128) char smem[];
  __shared__ int64_t s_warp_total[NW];
  __shared__ int64_t s_off[NW];      // where a range begins: units into the request,
  __shared__ int s_at[NW];           // the request
  __shared__ int2 s_goes[NW];        // apart: what a warp has of a segment that began before it (Goes, heads)
  __shared__ int4 s_opens[NW];       // and what it leaves open: request (-1: nothing), pass, blocks to come, heads
  __shared__ float2 s_cta[8 * NT];

  op_wait_for_previous();
  // the joining launch may begin to set itself up; it waits for this grid before it reads
  if (!CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int heads = a.heads_per_pass;
  char *ring = smem;
  float2 *m_ml = reinterpret_cast<float2 *>(smem + Shape::kRing);          // [NW][heads]
  float *m_o = reinterpret_cast<float *>(m_ml + NW * heads);               // [NW][heads][D]
  int *s_mask = reinterpret_cast<int *>(m_o + NW * heads * D);             // [NW][S]
  int *s_first = s_mask + NW * S;                                          // [rows]
  int *s_len = s_first + a.rows;                                           // [rows]

  // ---- what this CTA works on: blocks of one (request, pass), or a range of the whole batch's
  const int passes = a.c.kv_heads * a.head_blocks;
  const auto blocks_of = [&](int len) {
    const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
    return (len + kBlock - 1) / kBlock - lo / kBlock;
  };
  int one_first = 0, one_len = 0;       // CLUSTER: of its request
  const auto fill = [&](Segment &s) {   // what follows from the request
    s.first = CLUSTER ? one_first : s_first[s.r];
    s.len = CLUSTER ? one_len : s_len[s.r];
    s.lo = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
    s.b0 = s.lo / kBlock;
    s.nb = blocks_of(s.len);
  };
  bool apart = false;                   // each warp has a range of its own (kManyShort)
  // Both ends of a range inside a short segment move to an end of it, the same way for the two
  // ranges that meet there.
  const auto snap = [&](Segment &s) {
    if (s.nb > (apart ? kApartSnapUnits : kSnapUnits)) return;
    s.jb = s.jb == s.nb || 2 * s.jb > s.nb ? s.nb : 0;
    s.ja = s.ja == 0 || 2 * s.ja <= s.nb ? 0 : s.nb;
    if (s.ja >= s.jb) s.ja = s.jb = 0;
  };
  int end_units = kSegmentUnits;
  // the part of s from unit `at` on, `left` units of the range to go
  const auto enter_at = [&](Segment &s, int at, int64_t left) {
    s.ja = min(at, s.nb);
    s.jb = int(min(int64_t(s.nb), at + left));
    s.left = max(int64_t(0), at + left - (s.nb + end_units));
    snap(s);
  };
  Segment begin;
  Ranges all = {};
  int64_t u0 = 0, u1 = 0;               // this CTA's range, or this warp's
  const int ctas = CLUSTER ? a.ctas : 1, rank = CLUSTER ? int(blockIdx.x) % ctas : 0;
  if (CLUSTER) {
    const int seg = int(blockIdx.x) / ctas;
    begin.r = seg / passes;
    begin.pass = seg % passes;
    const PagedRun run = paged_run(a.c.indptr[begin.r], a.c.indptr[begin.r + 1], a.c.last[begin.r], a.c.page_size,
                                   a.c.num_indices);
    if (run.broken && tid == 0) paged_flag(a.c, kPagedBadTable);
    one_first = int(run.first);
    one_len = int(run.tokens);
    fill(begin);
    begin.ja = int(int64_t(begin.nb) * rank / ctas);
    begin.jb = int(int64_t(begin.nb) * (rank + 1) / ctas);
    begin.left = 0;
  } else {
    const int per = (a.rows + kThreads - 1) / kThreads;
    int64_t mine = 0;             // blocks of a pass, and requests that have positions in the lower 13 bits
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r >= a.rows) break;
      const PagedRun run = paged_run(a.c.indptr[r], a.c.indptr[r + 1], a.c.last[r], a.c.page_size, a.c.num_indices);
      if (run.broken && blockIdx.x == 0) paged_flag(a.c, kPagedBadTable);
      s_first[r] = int(run.first);
      s_len[r] = int(run.tokens);
      mine += (int64_t(blocks_of(int(run.tokens))) << 13) + (run.tokens > 0);
    }
    int64_t before = mine;            // inclusive scan over the threads
  #pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int64_t x = __shfl_up_sync(~0u, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s_warp_total[warp] = before;
    __syncthreads();
    int64_t total = 0;
    before -= mine;
  #pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += s_warp_total[w];
      total += s_warp_total[w];
    }
    const int segments = int(total & 8191) * passes;
    const int most = segments >= kManyShort * int(gridDim.x)  ? kShortBlocks
                     : segments >= kManyTiny * int(gridDim.x) ? kTinyBlocks : 0;
    apart = (total >> 13) * passes <= int64_t(most) * segments;
    if (apart) end_units = kApartEndUnits;
    const auto units = [&](int64_t x) { return ((x >> 13) + (x & 8191) * end_units) * passes; };
    total = units(total);
    before = units(before);
    // As many workers as have kMinUnits each, or as there are segments; and where a worker's share
    // is short, a whole number per segment, so that equal segments are cut at their ends (a
    // second segment in a range costs about as much as kAlignUnits).
    int workers = int(max(int64_t(1), min(max(total / kMinUnits, int64_t(segments)), int64_t(gridDim.x))));
    if (segments > 0 && segments <= workers && total < int64_t(kAlignUnits) * workers)
      workers -= workers % segments;
    all.total = total;
    all.workers = workers;
    all.each = divide(total, all.workers);
    all.more = int(total - all.each * all.workers);
    const bool works = total > 0 && int(blockIdx.x) < all.workers;
    u0 = all.start(blockIdx.x);
    u1 = all.start(blockIdx.x + 1);
    if (works && u0 < before + units(mine) && u1 > before)
      for (int w = 0; w < (apart ? NW : 1); ++w) {
        int64_t off = u0 + (u1 - u0) * w / NW - before;
        if (off < 0 || off >= units(mine)) continue;
        int r = tid * per;
        for (;; ++r) {
          if (s_len[r] == 0) continue;
          const int64_t n = int64_t(blocks_of(s_len[r]) + end_units) * passes;
          if (off < n) break;
          off -= n;
        }
        s_at[w] = r;
        s_off[w] = off;
      }
    if (tid == 0 && !a.by_segment) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    // requests without positions: nobody's range
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
      // (s_len of r was written by this CTA before the barrier above)
      if (s_len[r] != 0) continue;
      if (a.by_segment)
        for (int i = tid; i < passes; i += kThreads) a.desc[r * passes + i] = make_int4(0, 0, 0, 0);
      for (int i = tid; i < a.q_heads * (D / 8); i += kThreads) {
        const int h = i / (D / 8);
        *reinterpret_cast<uint4 *>(a.out + 2 * (r * a.o_token + (h / a.group) * a.o_group + (h % a.group) * a.o_head) +
                                   16 * (i % (D / 8))) = make_uint4(0, 0, 0, 0);
      }
      if (a.lse)
        for (int h = tid; h < a.q_heads; h += kThreads) a.lse[int64_t(r) * a.q_heads + h] = -INFINITY;
    }
    __syncthreads();
    if (!works) return;
    if (apart) {
      const int64_t share = u1 - u0;
      u1 = u0 + share * (warp + 1) / NW;
      u0 = u0 + share * warp / NW;
    }
    begin.ja = begin.jb = 0;
    begin.left = 0;
    if (u0 < u1) {
      const int w = apart ? warp : 0;
      begin.r = s_at[w];
      fill(begin);
      const int each = begin.nb + end_units;
      begin.pass = int(divide(s_off[w], each));
      enter_at(begin, int(s_off[w] - int64_t(begin.pass) * each), u1 - u0);
    }
  }
  const int first = apart ? 0 : warp, step = apart ? 1 : NW;   // blocks of a range that this warp takes

  const auto next_segment = [&](Segment &s) {   // only while s.left > 0
    if (++s.pass == passes) {
      s.pass = 0;
      do ++s.r;
      while (s_len[s.r] == 0);
      fill(s);
    }
    enter_at(s, 0, s.left);
  };

  // ---- filling the ring: this warp's blocks one after the other, across segments
  char *my_ring = ring + warp * (S * 2 * Shape::kTile);
  const uint32_t my_ring32 = static_cast<uint32_t>(__cvta_generic_to_shared(my_ring));
  Segment fs = begin;
  int fj = fs.ja + first;
  int page = 0, in_page = 0;   // of this lane's row (lane % 16) in the block at the cursor; -1: not seen
  int64_t head_at = 0;         // element offset of the segment's K/V head
  bool more = true;            // the cursor stands on a block
  // Page numbers come 32 at a time, a lane each, and the next 32 while these are used: the miss of one
  // load per block shows where pages are short (64 x 4096 in pages of 16: 177 us, so 171).
  int win = 0, win_next = 0;    // this lane's
  int at_win = 0, at_next = 0;  // which page of the run lane 0 has
  int held = 0, last_page = 0;  // blocks that end beyond `held` tokens need other pages; the run's last page
  const auto pages_from = [&](int q) {
    return q + lane <= last_page ? a.c.indices[fs.first + q + lane] : -1;
  };
  const auto enter = [&]() {
    head_at = fs.pass / a.head_blocks * a.c.stride_head;
    at_next = -1;
    held = 0;
    last_page = fast_div(fs.len - 1, a.page_div);
  };
  const auto settle = [&]() {  // move the cursor onto a block, fetch its page numbers
    while (fj >= fs.jb) {
      if (fs.left == 0) {
        more = false;
        return;
      }
      next_segment(fs);
      fj = fs.ja + first;
      enter();
    }
    const int p0 = (fs.b0 + fj) * kBlock, pos = p0 + lane % kBlock;
    const int q = fast_div(pos, a.page_div);
    in_page = pos < fs.len && pos >= fs.lo ? pos - q * a.c.page_size : -1;
    if constexpr (CLUSTER) {
      page = in_page >= 0 ? a.c.indices[fs.first + q] : -1;
    } else {
      if (p0 + kBlock > held) {
        at_win = fast_div(p0, a.page_div);
        win = at_win == at_next ? win_next : pages_from(at_win);
        held = 0x7fffffff;
        if (last_page - at_win >= 32) {
          held = (at_win + 32) * a.c.page_size;     // (in the run, so it fits)
          // the first block of this warp that ends beyond
          const int p1 = p0 + ((held - p0 - kBlock) / (kBlock * step) + 1) * (kBlock * step);
          at_next = -1;
          if (p1 < fs.len) {
            at_next = fast_div(p1, a.page_div);
            win_next = pages_from(at_next);
          }
        }
      }
      page = __shfl_sync(~0u, win, (q - at_win) & 31);
    }
  };
  int fstage = 0;
  const auto issue = [&]() {
    if (more) {
      int64_t row = in_page >= 0 ? paged_row(page, a.c.num_pages, in_page, a.c.stride_page, a.c.stride_token) : -1;
      if (in_page >= 0 && row < 0) paged_flag(a.c, kPagedBadPage);
      const unsigned mask = __ballot_sync(~0u, row >= 0) & 0xffffu;
      if (lane == 0) s_mask[warp * S + fstage] = int(mask);
      if (row >= 0) row = 2 * (row + head_at);
      const uint32_t dst = my_ring32 + fstage * 2 * Shape::kTile;
#pragma unroll
      for (int i = 0; i < kBlock * kChunks / 32; ++i) {
        const int t = i * 32 + lane, rr = t / kChunks, ch = t % kChunks;
        const int64_t at = __shfl_sync(~0u, row, rr);
        const bool valid = at >= 0;
        const int64_t src = valid ? at + ch * 16 : 0;
        const uint32_t to = dst + rr * Shape::kRowBytes + ((ch ^ (rr & 7)) * 16);
        copy16(to, a.c.k + src, valid);
        copy16(to + Shape::kTile, a.c.v + src, valid);
      }
      fstage = fstage + 1 == S ? 0 : fstage + 1;
      fj += step;
      settle();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (CLUSTER || u0 < u1) {
    enter();
    settle();
  } else {
    more = false;
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue();

  // ---- consuming
  int stage = 0;
  Segment cs = begin;
  uint32_t qf[NT][D / 16][2];       // of the segment in work
  const auto load_q = [&](const Segment &s) {
    const int kv = s.pass / a.head_blocks, h0 = (s.pass % a.head_blocks) * heads;
    const int live = min(heads, a.group - h0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = n * 8 + lane / 4;
      const char *qp = a.q + 2 * (s.r * a.q_token + kv * a.q_group + (h0 + h) * a.q_head) + (lane % 4) * 4;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[n][ks][0] = h < live ? *reinterpret_cast<const uint32_t *>(qp + ks * 32) : 0u;
        qf[n][ks][1] = h < live ? *reinterpret_cast<const uint32_t *>(qp + ks * 32 + 16) : 0u;
      }
    }
  };
  const auto advance = [&]() {      // to the next segment that has blocks in this range
    do {
      if (cs.left == 0) return false;
      next_segment(cs);
    } while (cs.ja >= cs.jb);
    return true;
  };
  // The state of a warp by itself that goes into a merge: of a segment that began before the warp's
  // range in its merge area, of one that it opens in its ring, which is empty by then.
  const auto state_o = [&](int w, bool opened) {
    return opened ? reinterpret_cast<float *>(ring + w * (S * 2 * Shape::kTile)) : m_o + w * heads * D;
  };
  const auto state_ml = [&](int w, bool opened) {
    return opened ? reinterpret_cast<float2 *>(state_o(w, true) + heads * D) : m_ml + w * heads;
  };
  enum Goes { kNone, kOn, kEnds, kEmpty };     // no such segment; it goes on behind the warp; it ends; no range
  bool some = CLUSTER || cs.ja < cs.jb || advance();
  if (apart) {
    if (lane == 0) {
      s_goes[warp] = make_int2(some ? kNone : kEmpty, 0);
      s_opens[warp] = make_int4(-1, 0, 0, 0);
    }
  } else if (!some) {
    return;
  }
  const auto finish = [&](int r, int kv, int h0, int h, int d, float top, float sum, const float4 &x) {
    const float inv = sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum;
    const uint2 v = make_uint2(T::round2(x.x * inv, x.y * inv), T::round2(x.z * inv, x.w * inv));
    *reinterpret_cast<uint2 *>(a.out + 2 * (r * a.o_token + kv * a.o_group + (h0 + h) * a.o_head + d)) = v;
    if (a.lse && d == 0)
      a.lse[int64_t(r) * a.q_heads + kv * a.group + h0 + h] =
          sum == 0.f ? -INFINITY : (top - kShift + log2f(sum)) * 0.69314718055994531f;
  };
  while (some) {
    load_q(cs);
    const int kv = cs.pass / a.head_blocks, h0 = (cs.pass % a.head_blocks) * heads;
    const int live = min(heads, a.group - h0);        // query heads of this pass
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
    }
    for (int j = cs.ja + first; j < cs.jb; j += step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
      __syncwarp();
      issue();         // into the stage that the previous block has left
      const uint32_t kt = my_ring32 + stage * 2 * Shape::kTile, vt = kt + Shape::kTile;
      const int mask = s_mask[warp * S + stage];
      stage = stage + 1 == S ? 0 : stage + 1;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t af[4];
        const int row = (lane / 8 % 2) * 8 + lane % 8, ch = ks * 2 + lane / 16;
        ldmatrix4<false>(af, kt + row * Shape::kRowBytes + ((ch ^ (row & 7)) * 16));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<T>(s[n], af, qf[n][ks][0], qf[n][ks][1]);
      }
      const bool v0 = (mask >> (lane / 4)) & 1, v1 = (mask >> (lane / 4 + 8)) & 1;
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = v0 ? s[n][0] * a.scale_log2 : -INFINITY;
        s[n][1] = v0 ? s[n][1] * a.scale_log2 : -INFINITY;
        s[n][2] = v1 ? s[n][2] * a.scale_log2 : -INFINITY;
        s[n][3] = v1 ? s[n][3] * a.scale_log2 : -INFINITY;
        // weights up to 2^8 over the reference are let through: the reference moves rarely
        grows |= fmaxf(s[n][0], s[n][2]) > m[n][0] + 8.f || fmaxf(s[n][1], s[n][3]) > m[n][1] + 8.f;
      }
      if (__any_sync(~0u, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
            for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
            top = fmaxf(top, m[n][c]);
            const float keep = m[n][c] == -INFINITY ? 0.f : exp2_fast(m[n][c] - top);
            m[n][c] = top;
            l[n][c] *= keep;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[n][d][c] *= keep;
              o[n][d][c + 2] *= keep;
            }
          }
      }
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float ref = m[n][c & 1] == -INFINITY ? 0.f : m[n][c & 1];
          p[c] = exp2_fast(s[n][c] - ref + kShift);
        }
        l[n][0] += p[0] + p[2];
        l[n][1] += p[1] + p[3];
        // The weights go into the product as two 16-bit parts, 16 bits of them in all: one part
        // alone would err as much as the rounding of the result itself.
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t h = T::round2(p[2 * c], p[2 * c + 1]);
          const float2 f = T::widen(h);
          hi[n][c] = transpose8(h);
          lo[n][c] = transpose8(T::round2(p[2 * c] - f.x, p[2 * c + 1] - f.y));
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t af[4];
        const int row = (lane / 16) * 8 + lane % 8, ch = d * 2 + lane / 8 % 2;
        ldmatrix4<true>(af, vt + row * Shape::kRowBytes + ((ch ^ (row & 7)) * 16));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<T>(o[n][d], af, hi[n][0], hi[n][1]);
          mma16816<T>(o[n][d], af, lo[n][0], lo[n][1]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 4; x < 32; x *= 2) l[n][c] += __shfl_xor_sync(~0u, l[n][c], x);
    // An infinity in V times a weight's two parts may be a NaN: the low part can be negative or 0, and
    // a weight that is next to nothing has both 0.  Sums that are no numbers though the weights
    // are: this warp's positions are looked through again, and a dimension that holds an infinity
    // gets it, one that holds both or a NaN a NaN.
    float odd[4] = {0.f, 0.f, 0.f, 0.f};       // (four sums: a chain of thirty products showed)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) odd[c] = fmaf(o[n][d][c], 0.f, odd[c]);
    if (__any_sync(~0u, odd[0] + odd[1] + (odd[2] + odd[3]) != 0.f)) {
      const uint2 far = infinities<T, D>(a, cs.first, cs.lo, cs.len, cs.b0 + cs.ja + first, cs.b0 + cs.jb, step, kv);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int bit = d + c / 2 * 16;
            const bool up = far.x >> bit & 1, down = far.y >> bit & 1;
            const float sum = l[n][c & 1];
            if ((up || down) && sum > 0.f) o[n][d][c] = up && down ? NAN : up ? INFINITY : -INFINITY;
          }
    }
    if (!CLUSTER && apart && cs.ja == 0 && cs.jb == cs.nb) {
      // ---- all of the segment: done
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float inv[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float sum = l[n][c];
          inv[c] = sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum;
          const int h = n * 8 + (lane % 4) * 2 + c;
          if (a.lse && lane < 4 && h < live)
            a.lse[int64_t(cs.r) * a.q_heads + kv * a.group + h0 + h] =
                sum == 0.f ? -INFINITY : (m[n][c] - kShift + log2f(sum)) * 0.69314718055994531f;
        }
        const int h = n * 8 + lane / 4;
        char *po = a.out + 2 * (cs.r * a.o_token + kv * a.o_group + (h0 + h) * a.o_head) + (lane % 4) * 4;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const uint32_t x0 = transpose8(T::round2(o[n][d][0] * inv[0], o[n][d][1] * inv[1]));
          const uint32_t x1 = transpose8(T::round2(o[n][d][2] * inv[0], o[n][d][3] * inv[1]));
          if (h < live) {
            *reinterpret_cast<uint32_t *>(po + d * 32) = x0;
            *reinterpret_cast<uint32_t *>(po + d * 32 + 16) = x1;
          }
        }
      }
      some = advance();
      continue;
    }
    // ---- a part of it: left for the merge
    const bool opened = !CLUSTER && apart && cs.ja == 0;
    __syncwarp();
    float2 *ml = state_ml(warp, opened);
    float *so = state_o(warp, opened);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = n * 8 + (lane % 4) * 2 + c;
        if (h < live) {
          if (lane < 4) ml[h] = make_float2(m[n][c], l[n][c]);
          float *po = so + h * D + lane / 4;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            po[d * 16] = o[n][d][c];
            po[d * 16 + 8] = o[n][d][c + 2];
          }
        }
      }
    if (!CLUSTER && apart) {
      if (lane == 0) {
        if (opened) s_opens[warp] = make_int4(cs.r, cs.pass, cs.nb - cs.jb, live);
        else s_goes[warp] = make_int2(cs.jb < cs.nb ? kOn : kEnds, live);
      }
      some = advance();
      continue;
    }
    // ---- merge the warps
    __syncthreads();
    const auto warps_joined = [&](int h, int d, float &top, float &sum, float4 &x) {
      top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, m_ml[w * heads + h].x);
      x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 ml = m_ml[w * heads + h];
        const float f = part_factor(ml.y, ml.x, top);
        const float4 y = *reinterpret_cast<const float4 *>(m_o + (w * heads + h) * D + d);
        sum += f * ml.y;
        x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
      }
    };
    if (CLUSTER) {
      cg::cluster_group cluster = cg::this_cluster();
      // this CTA's state where the first warp's was, then the cluster's CTAs share the output
      for (int i = tid; i < live * (D / 4); i += kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float top, sum;
        float4 x;
        warps_joined(h, d, top, sum, x);
        *reinterpret_cast<float4 *>(m_o + h * D + d) = x;
        if (d == 0) s_cta[h] = make_float2(top, sum);
      }
      cluster.sync();
      for (int i = tid * ctas + rank; i < live * (D / 4); i += kThreads * ctas) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 ml[kMaxCluster];
        float4 y[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
          if (c >= ctas) break;
          ml[c] = cluster.map_shared_rank(s_cta, c)[h];
          y[c] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(m_o, c) + h * D + d);
          top = fmaxf(top, ml[c].x);
        }
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
          if (c >= ctas) break;
          const float f = part_factor(ml[c].y, ml[c].x, top);
          sum += f * ml[c].y;
          x.x += f * y[c].x, x.y += f * y[c].y, x.z += f * y[c].z, x.w += f * y[c].w;
        }
        finish(cs.r, kv, h0, h, d, top, sum, x);
      }
      cluster.sync();     // nobody leaves while its shared memory is read
      return;
    }
    const bool whole = cs.ja == 0 && cs.jb == cs.nb;
    const int slot = 2 * blockIdx.x + (cs.ja == 0);    // 1: the range that begins the segment
    for (int i = tid; i < live * (D / 4); i += kThreads) {
      const int h = i / (D / 4), d = i % (D / 4) * 4;
      float top, sum;
      float4 x;
      warps_joined(h, d, top, sum, x);
      if (whole) {
        finish(cs.r, kv, h0, h, d, top, sum, x);
      } else {
        *reinterpret_cast<float4 *>(a.part_o + (int64_t(slot) * heads + h) * D + d) = x;
        if (d == 0) a.part_ml[int64_t(slot) * heads + h] = make_float2(top, sum);
      }
    }
    if (cs.ja == 0 && tid == 0 && (!whole || a.by_segment)) {
      // this range begins the segment: how many does it run through?
      const int parts = whole ? 0 : all.owner(u1 + (cs.nb - cs.jb) - 1) - int(blockIdx.x) + 1;
      a.desc[a.by_segment ? cs.r * passes + cs.pass : int(blockIdx.x)] = make_int4(cs.r, cs.pass, parts, blockIdx.x);
    }
    some = advance();
    if (some) __syncthreads();      // the merge area is free again
  }
  if (!apart) return;

  // ---- segments that warps share: first (c = -1) the one that an earlier CTA began, then what each
  // warp c opened; in either case with what the next warps have of it
  __syncthreads();
  unsigned none = 0, ending = 0, empty = 0, opened = 0;     // a bit per warp
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int goes = s_goes[w].x;
    none |= unsigned(goes == kNone) << w;
    ending |= unsigned(goes == kEnds) << w;
    empty |= unsigned(goes == kEmpty) << w;
    opened |= unsigned(s_opens[w].x >= 0) << w;
  }
  for (int c = -1; c < NW; ++c) {
    if (c >= 0 && !(opened >> c & 1)) continue;
    // the warps behind c up to the one that has the segment's end, or the last before one without a part
    const unsigned behind = ~0u << (c + 1) & ((1u << NW) - 1);
    const unsigned stop = none & behind, end = ending & behind;
    const bool ends = end && (!stop || __ffs(end) < __ffs(stop));
    const unsigned reach = ends ? (end & -end) * 2 - 1 : stop ? (stop & -stop) - 1 : ~0u;
    const unsigned parts = behind & reach & ~empty;
    if (c < 0 && !parts) continue;
    int4 opens = make_int4(0, 0, 0, 0);
    if (c >= 0) opens = s_opens[c];
    else opens.w = s_goes[__ffs(parts) - 1].y;
    const int live = opens.w;
    const bool whole = c >= 0 && ends;
    const int kv = opens.y / a.head_blocks, h0 = (opens.y % a.head_blocks) * heads;
    const int slot = 2 * blockIdx.x + (c >= 0);    // 1: the range that begins the segment
    for (int i = tid; i < live * (D / 4); i += kThreads) {
      const int h = i / (D / 4), d = i % (D / 4) * 4;
      float2 ml[NW];
      float4 y[NW];
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        ml[w] = make_float2(-INFINITY, 0.f);
        y[w] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (w == c || (parts >> w & 1)) {
          ml[w] = state_ml(w, w == c)[h];
          y[w] = *reinterpret_cast<const float4 *>(state_o(w, w == c) + h * D + d);
        }
        top = fmaxf(top, ml[w].x);
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = part_factor(ml[w].y, ml[w].x, top);
        sum += f * ml[w].y;
        x.x += f * y[w].x, x.y += f * y[w].y, x.z += f * y[w].z, x.w += f * y[w].w;
      }
      if (whole) {
        finish(opens.x, kv, h0, h, d, top, sum, x);
      } else {
        *reinterpret_cast<float4 *>(a.part_o + (int64_t(slot) * heads + h) * D + d) = x;
        if (d == 0) a.part_ml[int64_t(slot) * heads + h] = make_float2(top, sum);
      }
    }
    if (c >= 0 && tid == 0 && !whole) {
      // this CTA begins the segment and others go on: how many?
      const int64_t begins = all.start(blockIdx.x), share = all.start(blockIdx.x + 1) - begins;
      const int n = all.owner(begins + share * (c + 1) / NW + opens.z - 1) - int(blockIdx.x) + 1;
      a.desc[blockIdx.x] = make_int4(opens.x, opens.y, n, blockIdx.x);
    }
  }
}

// Joins the parts of one segment (blockIdx.x: see DecodeArgs::by_segment) for a.join_heads query
// heads of the pass and D / gridDim.z dimensions: parts of workers c (slot 1), c + 1, ...
// (slot 0).  One pass, each group of threads over its own parts, kAhead rows of them in flight.
template <class T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr int kAhead = 8;
  constexpr float kShift = std::is_same<T, OpF16>::value ? 7.f : 0.f;
  __shared__ float2 s_ml[32];
  __shared__ float4 s_o[256];
  op_wait_for_previous();
  const int4 desc = a.desc[blockIdx.x];
  const int parts = desc.z, heads = a.heads_per_pass;
  if (parts == 0) return;
  const int kv = desc.y / a.head_blocks, h0 = (desc.y % a.head_blocks) * heads;
  const int lanes = gridDim.z > 1 ? 8 : D / 4;               // threads per row
  const int groups = 256 / lanes / a.join_heads;             // rows of a head at a time
  const int row0 = threadIdx.x / lanes / groups * groups;    // the head's first group
  const int g = threadIdx.x / lanes - row0, d = blockIdx.z * 8 + threadIdx.x % lanes;
  const int h = blockIdx.y * a.join_heads + row0 / groups;
  const bool mine = h < heads && h0 + h < a.group;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, sum = 0.f;
  for (int i0 = g; mine && i0 < parts; i0 += groups * kAhead) {
    float2 ml[kAhead];
    float4 y[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * groups;
      ml[j] = make_float2(-INFINITY, 0.f);
      y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < parts) {
        const int64_t row = (int64_t(2) * (desc.w + i) + (i == 0)) * heads + h;
        ml[j] = a.part_ml[row];
        y[j] = *reinterpret_cast<const float4 *>(a.part_o + row * D + d * 4);
      }
    }
    float next = top;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) next = fmaxf(next, ml[j].x);
    const float keep = part_factor(sum, top, next);
    sum = sum == 0.f ? 0.f : sum * keep;
    x.x *= keep, x.y *= keep, x.z *= keep, x.w *= keep;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float f = part_factor(ml[j].y, ml[j].x, next);
      sum += f * ml[j].y;
      x.x += f * y[j].x, x.y += f * y[j].y, x.z += f * y[j].z, x.w += f * y[j].w;
    }
    top = next;
  }
  s_o[threadIdx.x] = x;
  if (threadIdx.x % lanes == 0) s_ml[row0 + g] = make_float2(top, sum);
  __syncthreads();
  if (g != 0 || !mine) return;
  const int used = min(groups, parts);
  for (int i = 1; i < used; ++i) top = fmaxf(top, s_ml[row0 + i].x);
  sum = 0.f;
  x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < used; ++i) {
    const float2 ml = s_ml[row0 + i];
    const float f = part_factor(ml.y, ml.x, top);
    const float4 y = s_o[i * lanes + threadIdx.x];
    sum += f * ml.y;
    x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
  }
  const float inv = sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum;
  const uint2 v = make_uint2(T::round2(x.x * inv, x.y * inv), T::round2(x.z * inv, x.w * inv));
  *reinterpret_cast<uint2 *>(a.out + 2 * (desc.x * a.o_token + kv * a.o_group + (h0 + h) * a.o_head + d * 4)) = v;
  if (a.lse && d == 0)
    a.lse[int64_t(desc.x) * a.q_heads + kv * a.group + h0 + h] =
        sum == 0.f ? -INFINITY : (top - kShift + log2f(sum)) * 0.69314718055994531f;
}

// Query heads per pass: eight fill one n-tile of the product.  Sixteen (two n-tiles) read the rows
// once for groups of 9 to 16; at D = 256 the second tile's accumulators do not fit the registers.
int n_tiles(int head_dim, int group) { return head_dim <= 128 && group > 8 ? 2 : 1; }

int pass_heads(int head_dim, int group) { return std::min(group, 8 * n_tiles(head_dim, group)); }

uint64_t workspace_bytes(int workers, int heads, int head_dim) {
  return uint64_t(workers) * (16 + 2 * uint64_t(heads) * (8 + 4 * uint64_t(head_dim)));
}

// CTAs per (request, pass) when each gets a cluster of its own, 0: equal ranges.  A cluster is
// one launch and joins inside it, but a long request among short ones is its cluster's alone.
// How long it can be is known on the host only as far as the page list goes: clusters are used
// where all of them are resident at once (a CTA per SM) and the whole list in one request's hands
// leaves a CTA at most kClusterUnits.  Measured with equal lengths / with everything in one
// request, clusters against ranges: 4 x 500 tokens 6.6 against 9.8 / 9.4 against 9.9 us; one step
// further (a bound of 256) 16 x 100 tokens 5.9 against 7.0 / 20 against 10.
constexpr int kClusterUnits = 64;
int cluster_ctas(const ypk_paged_cache *c, int rows, int passes, int window, int sms) {
  int64_t units = (int64_t(c->num_indices) * c->page_size + kBlock - 1) / kBlock;
  if (window > 0) units = std::min(units, int64_t(window) / kBlock + 2);
  // A cluster lies in one GPC, and GPCs are not multiples of it: of 148 SMs, one CTA each, clusters
  // of four reach 132 and of eight 120 on the card measured.  (16 clusters
  // of eight run in two waves: 1 x 1000 with 16 heads 11.3 us, with four CTAs each 6.4.)
  const auto resident = [&](int ctas) {
    return int64_t(rows) * passes * ctas <= (ctas > 4 ? sms * 4 / 5 : ctas > 2 ? sms * 7 / 8 : sms);
  };
  int ctas = 1;
  while (ctas < kMaxCluster && resident(ctas * 2) && units > 8 * ctas) ctas *= 2;
  return units <= int64_t(kClusterUnits) * ctas && resident(ctas) ? ctas : 0;
}

constexpr int kMaxShared = 232448 - 1024;   // opt-in limit of a block, less the static part

template <class T, int NW, int D, int NT, int S, bool CLUSTER>
int launch_shape(const DecodeArgs &a, const DeviceInfo &dev, cudaStream_t st) {
  using Shape = DecodeShape<NW, D, NT, S>;
  static std::atomic<uint64_t> ready{0};      // devices whose limit has been raised
  auto *kernel = paged_decode_kernel<T, NW, D, NT, S, CLUSTER>;
  if (!(ready.load(std::memory_order_relaxed) >> dev.device & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
    if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "paged_decode: shared memory: %s", cudaGetErrorString(e));
    ready.fetch_or(uint64_t(1) << dev.device, std::memory_order_relaxed);
  }
  const int shared = Shape::bytes(a.heads_per_pass, CLUSTER ? 0 : a.rows);
  const unsigned segments = unsigned(a.rows) * a.c.kv_heads * a.head_blocks;
  if (CLUSTER)
    return op_launch("paged_decode", kernel, dim3(segments * a.ctas), NW * 32, shared, a.ctas, st, a);
  if (int rc = op_launch("paged_decode", kernel, dim3(dev.sms), NW * 32, shared, 0, st, a)) return rc;
  // Few segments: many threads on each (32 dimensions a block), as long as all blocks find a place
  // beside the attention kernel's (two per SM; 4 x 1034 tokens 12.0 us, 13.3 with 512 blocks).  Many:
  // at most one is joined per worker, of two parts as a rule, and blocks for several heads are through
  // sooner (64 x 4096 166.8 -> 164.3 us; 19 x 6 tokens of 64 heads, nothing to join, 11.5 -> 10.5).
  const bool fine = a.by_segment && segments * a.heads_per_pass * (D / 32) <= unsigned(2 * dev.sms);
  DecodeArgs j = a;
  j.join_heads = 1;
  if (!a.by_segment)
    while (j.join_heads < a.heads_per_pass && j.join_heads < 1024 / D) j.join_heads *= 2;
  return op_launch("paged_decode", paged_join_kernel<T, D>,
                   dim3(a.by_segment ? segments : dev.sms, (a.heads_per_pass + j.join_heads - 1) / j.join_heads,
                        fine ? D / 32 : 1), 256, 0, 0, st, j);
}

// Ring depth: three blocks per warp; two where the merge area of sixteen heads or the tables of
// thousands of requests need the room.
template <class T, int NW, int D, int NT>
int launch_ring(const DecodeArgs &a, const DeviceInfo &dev, cudaStream_t st) {
  constexpr int kDeep = NT == 2 && D == 128 ? 2 : 3;
  if (a.ctas) return launch_shape<T, NW, D, NT, kDeep, true>(a, dev, st);
  if (kDeep == 3 && DecodeShape<NW, D, NT, 3>::bytes(a.heads_per_pass, a.rows) <= kMaxShared)
    return launch_shape<T, NW, D, NT, kDeep, false>(a, dev, st);
  return launch_shape<T, NW, D, NT, 2, false>(a, dev, st);
}

template <class T>
int launch_decode(int head_dim, const DecodeArgs &a, const DeviceInfo &dev, cudaStream_t st) {
  const bool two = n_tiles(head_dim, a.group) == 2;
  if (head_dim == 64) return two ? launch_ring<T, 8, 64, 2>(a, dev, st) : launch_ring<T, 8, 64, 1>(a, dev, st);
  if (head_dim == 128) return two ? launch_ring<T, 8, 128, 2>(a, dev, st) : launch_ring<T, 8, 128, 1>(a, dev, st);
  return launch_ring<T, 4, 256, 1>(a, dev, st);
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
  DeviceInfo dev;
  if (int rc = op_device("paged_decode", &dev)) return rc;
  const int group = num_q_heads / cache->num_kv_heads, heads = pass_heads(cache->head_dim, group);
  const int passes = cache->num_kv_heads * ((group + heads - 1) / heads);
  // (fewer rows and a window only make clusters likelier)
  *bytes = cluster_ctas(cache, cache->num_requests, passes, 0, dev.sms) ? 0 : workspace_bytes(dev.sms, heads, cache->head_dim);
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
  if (!(fabsf(p->scale) <= 1e30f)) return op_fail(YPK_ERR_INVALID, "paged_decode: scale is not finite");
  for (int64_t s : {p->q_stride_token, p->q_stride_group, p->q_stride_head, p->out_stride_token,
                    p->out_stride_group, p->out_stride_head})
    if (s < 0 || s % 8) return op_fail(YPK_ERR_INVALID, "paged_decode: rows must start on 16-byte boundaries");
  if (!op_aligned16(p->q) || !op_aligned16(p->out) || !op_aligned16(p->workspace))
    return op_fail(YPK_ERR_INVALID, "paged_decode: an operand is not 16-byte aligned");
  const auto rows = [&](const void *at, int64_t token, int64_t group, int64_t head) {
    return head_rows(at, p->rows, token, cache->num_kv_heads, group, p->num_q_heads / cache->num_kv_heads, head,
                     cache->head_dim);
  };
  const StridedRows out = rows(p->out, p->out_stride_token, p->out_stride_group, p->out_stride_head);
  if (rows_touch(rows(p->q, p->q_stride_token, p->q_stride_group, p->q_stride_head), out))
    return op_fail(YPK_ERR_INVALID, "paged_decode: out overlaps q");
  if (!rows_distinct(out)) return op_fail(YPK_ERR_INVALID, "paged_decode: rows of out overlap");
  if (rows_touch(cache_rows(cache, cache->k), out) || rows_touch(cache_rows(cache, cache->v), out))
    return op_fail(YPK_ERR_INVALID, "paged_decode: out overlaps the cache");
  DeviceInfo dev;
  if (int rc = op_device("paged_decode", &dev)) return rc;
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
  a.heads_per_pass = pass_heads(cache->head_dim, a.group);
  a.head_blocks = (a.group + a.heads_per_pass - 1) / a.heads_per_pass;
  a.page_div = fast_divisor(cache->page_size);
  a.by_segment = int64_t(p->rows) * cache->num_kv_heads * a.head_blocks <= dev.sms;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.ctas = cluster_ctas(cache, p->rows, cache->num_kv_heads * a.head_blocks, p->window, dev.sms);
  const uint64_t need = a.ctas ? 0 : workspace_bytes(dev.sms, a.heads_per_pass, cache->head_dim);
  if (need && (!p->workspace || p->workspace_bytes < need))
    return op_fail(YPK_ERR_INVALID, "paged_decode: workspace of %llu bytes, %llu needed",
                   (unsigned long long)(p->workspace ? p->workspace_bytes : 0), (unsigned long long)need);
  char *w = static_cast<char *>(p->workspace);      // (not used with clusters)
  a.desc = reinterpret_cast<int4 *>(w);
  a.part_o = reinterpret_cast<float *>(w + 16 * uint64_t(dev.sms));
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + 2 * uint64_t(dev.sms) * a.heads_per_pass * cache->head_dim);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == YPK_BF16 ? launch_decode<OpBf16>(cache->head_dim, a, dev, st)
                                  : launch_decode<OpF16>(cache->head_dim, a, dev, st);
}
