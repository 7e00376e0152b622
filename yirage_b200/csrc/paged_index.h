// Index arithmetic of a paged K/V cache: which page and which row of it a position of a
// request lies in.  Plain C++, so that the same functions run in the kernels and in the host
// tests that walk good and broken page tables.
//
// The tables live in device memory and may be anything when a kernel reads them, so every
// value taken from them is checked here before it becomes an address: a broken table gives an
// error bit, never an access out of range.  Sums are taken in 64 bits (pages x page size passes
// 32 bits for tables that are broken, and row offsets do for caches that are not).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define YPK_HD __host__ __device__ __forceinline__
#else
#define YPK_HD inline
#endif

namespace ypk {

// Bits of ypk_paged_cache.status, also in include/ypk.h.
constexpr int kPagedBadTable = 1;      // offsets that run backwards or past the index list
constexpr int kPagedBadPage = 2;       // a page number outside the pool
constexpr int kPagedBadPosition = 4;   // a position outside the rotary tables
constexpr int kPagedBadLength = 8;     // more new tokens than the request is long

// Longest request: positions, and positions rounded up to a block, fit 32 bits.
constexpr int64_t kPagedMaxTokens = 0x7fffff00;

// The run of one request in the list of page numbers, and its length in tokens.
struct PagedRun {
  int64_t first;    // index of its first page number
  int64_t tokens;   // its length, 0 for an empty or a broken run
  bool broken;
};

YPK_HD PagedRun paged_run(int begin, int end, int last_page_len, int page_size, int num_indices) {
  PagedRun r = {begin, 0, false};
  if (begin == end) return r;                       // a slot without a request
  if (begin < 0 || end < begin || end > num_indices || last_page_len < 0 || last_page_len > page_size) {
    r.broken = true;
    return r;
  }
  r.tokens = int64_t(end - begin - 1) * page_size + last_page_len;
  if (r.tokens > kPagedMaxTokens) {                 // no memory holds it: the table is broken
    r.tokens = 0;
    r.broken = true;
  }
  return r;
}

// Position of new token `row` of the call (rows [qo_begin, qo_end) belong to the request):
// the new tokens are the last ones of the request.  Negative: not a position.
YPK_HD int64_t paged_new_position(const PagedRun &run, int qo_end, int row) {
  const int64_t behind = int64_t(qo_end) - row;     // 1 for the last new token
  return behind < 1 ? -1 : run.tokens - behind;
}

// Element offset of a row for K/V head 0, or -1 when the page is not in the pool.  `in_page`: its
// place in the page, in [0, page_size).
YPK_HD int64_t paged_row(int page, int num_pages, int in_page, int64_t stride_page, int64_t stride_token) {
  if (page < 0 || page >= num_pages) return -1;
  return int64_t(page) * stride_page + int64_t(in_page) * stride_token;
}

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 without a division: with l = ceil(log2 d) and
// mul = floor(2^32 (2^l - d) / d) + 1, n / d = (n + mulhi(n, mul)) >> l (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct FastDivisor {
  uint32_t mul, shift;
};
inline FastDivisor fast_divisor(int d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < uint64_t(d)) ++l;
  return {uint32_t((((uint64_t(1) << l) - uint64_t(d)) << 32) / uint64_t(d) + 1), l};
}
YPK_HD int fast_div(int n, const FastDivisor &d) {
#ifdef __CUDA_ARCH__
  const uint32_t hi = __umulhi(uint32_t(n), d.mul);
#else
  const uint32_t hi = uint32_t((uint64_t(uint32_t(n)) * d.mul) >> 32);
#endif
  return int((uint32_t(n) + hi) >> d.shift);
}

}  // namespace ypk
