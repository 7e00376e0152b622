// Log probabilities of given tokens, with entropy and top alternatives (ypk_token_logprobs).
#include "op_common.h"
#include "op_num.cuh"

namespace ypk {
namespace {

constexpr int kMaxTop = 32;

struct LogprobArgs {
  const void *logits;
  const long long *tokens;
  float *logprob, *entropy, *top_logprob;
  long long *top_token;
  int64_t ld;
  int vocab, top;
};

// Values as whole numbers in the same order (NaN lowest, -0 and +0 alike).
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

template <int DTYPE>
__device__ __forceinline__ float logit(const void *row, int64_t i) {
  if (DTYPE == YPK_F32) return static_cast<const float *>(row)[i];
  if (DTYPE == YPK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[i]);
  return __half2float(static_cast<const __half *>(row)[i]);
}

template <class V, class F>
__device__ V block_reduce(V v, V *shared, F f) {
#pragma unroll
  for (int o = 16; o; o /= 2) v = f(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < blockDim.x / 32; ++w) v = f(v, shared[w]);
  return v;
}

// One CTA per row: maximum, then sums, then the k largest one after the other.
template <int DTYPE>
__global__ void __launch_bounds__(512) token_logprobs_kernel(const LogprobArgs a) {
  __shared__ float sf[16];
  __shared__ unsigned long long su[16];
  const int64_t r = blockIdx.x;
  const void *row = static_cast<const char *>(a.logits) + r * a.ld * (DTYPE == YPK_F32 ? 4 : 2);
  float m = -INFINITY;
  bool bad = false;
  for (int i = threadIdx.x; i < a.vocab; i += 512) {
    const float x = logit<DTYPE>(row, i);
    bad |= !(x < INFINITY);
    m = fmaxf(m, x);
  }
  m = block_reduce(m, sf, [](float p, float q) { return fmaxf(p, q); });
  const bool any_bad = __syncthreads_or(bad);
  const bool empty = !any_bad && m == -INFINITY;
  float s = 0.f, u = 0.f;
  if (!any_bad && !empty) {
    for (int i = threadIdx.x; i < a.vocab; i += 512) {
      const float d = logit<DTYPE>(row, i) - m;
      const float e = expf(d);
      s += e;
      u += e > 0.f ? d * e : 0.f;
    }
  }
  s = block_reduce(s, sf, [](float p, float q) { return p + q; });
  u = block_reduce(u, sf, [](float p, float q) { return p + q; });
  const float log_s = logf(s);
  auto logp = [&](float x) {
    if (any_bad) return NAN;
    if (empty || x == -INFINITY) return -INFINITY;
    return x - m - log_s;
  };
  if (threadIdx.x == 0) {
    const long long t = a.tokens[r];
    const bool inside = t >= 0 && t < a.vocab;
    a.logprob[r] = any_bad ? NAN : inside ? logp(logit<DTYPE>(row, t)) : -INFINITY;
    a.entropy[r] = any_bad ? NAN : empty ? 0.f : log_s - u / s;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long best = 0;   // order in the high half, columns from the right in the low one
    for (int i = threadIdx.x; i < a.vocab; i += 512) {
      const unsigned long long key =
          (static_cast<unsigned long long>(order_of(logit<DTYPE>(row, i))) << 32) | (0xffffffffu - unsigned(i));
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, su, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    last = best;
    if (threadIdx.x == 0) {
      const unsigned i = 0xffffffffu - unsigned(best);
      a.top_token[r * a.top + k] = i;
      a.top_logprob[r * a.top + k] = logp(logit<DTYPE>(row, i));
    }
  }
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
  a.logits = logits;
  a.tokens = reinterpret_cast<const long long *>(tokens);
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_logprob = top_logprob;
  a.top_token = reinterpret_cast<long long *>(top_token);
  a.ld = ld;
  a.vocab = vocab;
  a.top = top_k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == YPK_BF16) token_logprobs_kernel<YPK_BF16><<<rows, 512, 0, st>>>(a);
  else if (dtype == YPK_F16) token_logprobs_kernel<YPK_F16><<<rows, 512, 0, st>>>(a);
  else token_logprobs_kernel<YPK_F32><<<rows, 512, 0, st>>>(a);
  return op_launched("token_logprobs");
}
