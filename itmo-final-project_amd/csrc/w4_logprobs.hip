// Log probabilities of given tokens, the entropy of their distributions and the most
// likely alternatives, from rows of logits (int4_hip/scoring.py).
#include <hip/hip_runtime.h>

#include "w4_common.hpp"

namespace w4 {

constexpr int kLogThreads = 256;
constexpr int kMaxTop = 64;

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float *logprob, *entropy, *top_logprob;
  int64_t* top_token;
  int64_t vocab, stride;
  int top;
};

template <int DT>
__device__ __forceinline__ float logit_at(const void* x, int64_t i) {
  if constexpr (DT == W4_DTYPE_FP32) return static_cast<const float*>(x)[i];
  else return act_bits_to_float(static_cast<const uint16_t*>(x)[i], DT);
}

// One workgroup a row: the maximum, the sums, then the alternatives one after the
// other, each the largest (key, lowest index) below the one before.
template <int DT>
__global__ __launch_bounds__(kLogThreads) void logprob_kernel(LogprobArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x, base = row * a.stride;
  __shared__ float red[4], red2[4];
  __shared__ uint64_t best_s[4];
  float m = -__builtin_inff();
  for (int64_t i = tid; i < a.vocab; i += kLogThreads) m = fmaxf(m, logit_at<DT>(a.x, base + i));
  m = wave_max(m);
  if (lane == 0) red[wv] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  float s = 0.f, t = 0.f;
  for (int64_t i = tid; i < a.vocab; i += kLogThreads) {
    const float y = logit_at<DT>(a.x, base + i) - m, e = expf(y);
    s += e;
    t += y == -__builtin_inff() ? 0.f : e * y;
  }
  s = wave_sum(s), t = wave_sum(t);
  if (lane == 0) red[wv] = s, red2[wv] = t;
  __syncthreads();
  s = (red[0] + red[1]) + (red[2] + red[3]);
  t = (red2[0] + red2[1]) + (red2[2] + red2[3]);
  const float ls = logf(s);
  if (tid == 0) {
    a.entropy[row] = ls - t / s;
    if (a.tokens) {
      const int64_t tok = a.tokens[row];
      a.logprob[row] = (uint64_t)tok < (uint64_t)a.vocab ? (logit_at<DT>(a.x, base + tok) - m) - ls : __builtin_nanf("");
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int64_t i = tid; i < a.vocab; i += kLogThreads) {
      const uint64_t key = ((uint64_t)order_key(logit_at<DT>(a.x, base + i)) << 32) | (uint32_t)(~(uint32_t)i);
      if (key < last && key > best) best = key;
    }
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, d);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) best_s[wv] = best;
    __syncthreads();
    for (int w = 0; w < 4; ++w) best = best_s[w] > best ? best_s[w] : best;
    last = best;
    if (tid == 0) {
      const int64_t tok = (int64_t)(uint32_t)~(uint32_t)best;
      a.top_token[row * a.top + k] = tok;
      a.top_logprob[row * a.top + k] = (logit_at<DT>(a.x, base + tok) - m) - ls;
    }
  }
}

}  // namespace w4

// ---------------------------------------------------------------- host side
using namespace w4host;

extern "C" size_t w4_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  (void)rows, (void)vocab, (void)top;
  return 0;
}

extern "C" int w4_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride,
                                 const int64_t* tokens, int64_t top, float* logprob, float* entropy,
                                 float* top_logprob, int64_t* top_token, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  clear_error();
  (void)workspace, (void)workspace_bytes;
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16 && dtype != W4_DTYPE_FP32)
    return fail(W4_ERR_INVALID, "w4_token_logprobs: dtype must be bf16, fp16 or fp32 (got code %d)", dtype);
  if (rows < 0 || vocab < 1 || vocab >= (1ll << 31) || stride < 0 || top < 0 || top > w4::kMaxTop || top > vocab)
    return fail(W4_ERR_INVALID, "w4_token_logprobs: %lld rows of %lld logits, the top %lld (at most %d)",
                (long long)rows, (long long)vocab, (long long)top, w4::kMaxTop);
  if (rows >= (1ll << 24)) return fail(W4_ERR_UNSUPPORTED, "w4_token_logprobs: %lld rows", (long long)rows);
  if (rows == 0) return W4_OK;
  if (!logits || !entropy || (!tokens != !logprob) || (top && (!top_logprob || !top_token)))
    return fail(W4_ERR_INVALID, "w4_token_logprobs: null pointer");
  w4::LogprobArgs a{logits, tokens, logprob, entropy, top_logprob, top_token, vocab, stride, (int)top};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)rows);
  if (dtype == W4_DTYPE_BF16) w4::logprob_kernel<W4_DTYPE_BF16><<<grid, w4::kLogThreads, 0, st>>>(a);
  else if (dtype == W4_DTYPE_FP16) w4::logprob_kernel<W4_DTYPE_FP16><<<grid, w4::kLogThreads, 0, st>>>(a);
  else w4::logprob_kernel<W4_DTYPE_FP32><<<grid, w4::kLogThreads, 0, st>>>(a);
  return check_launch("w4_token_logprobs");
}
