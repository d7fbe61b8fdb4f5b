// What the attention kernels over paged caches share: operands split into 16-bit
// parts, softmax sums that are joined, the order of a wave's LDS accesses.
#pragma once

#include "w4_common.hpp"

namespace w4 {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kPagedBufFlags = 0x00020000;  // raw buffer: the range is checked in bytes
constexpr int kPagedCoherentAux = 16;       // sc1: the cache policy of agent-scope atomic loads and stores

constexpr int kPagedCounters = W4_WORKSPACE_COUNTER_BYTES / 4;

// How an fp32 operand enters 16-bit matrix instructions: as the sum of its roundings.
template <int DT> struct Split;
template <> struct Split<W4_DTYPE_BF16> { static constexpr int N = 3; };  // 8 significant bits each: all 24
template <> struct Split<W4_DTYPE_FP16> { static constexpr int N = 2; };  // 11 each: 22

// QUERY: an infinity or NaN has no small parts.  (A probability is no infinity, and beside a NaN all of its head's
// are.)
template <int DT, bool QUERY>
__device__ __forceinline__ void split8(const float v[8], u32x4* out) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < Split<DT>::N; ++p) {
    out[p] = pack8<DT>(r);
    float t[8];
    unpack8<DT>(out[p], t);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = QUERY && !(__builtin_fabsf(t[e]) < __builtin_inff()) ? 0.f : r[e] - t[e];
  }
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -__builtin_inff() ? 0.f : m; }

// Softmax sums and a quad of outputs, relative to the score M.  (Scores are subtracted before they become exponents:
// past 2^24 the exponent's own rounding would be powers of two.)  A refused part's reference is NaN and stays.
template <bool LOG2>  // scores are exponents of 2 already
struct ShareOf {
  static __device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(LOG2 ? d : d * kLog2e); }
  float M = -__builtin_inff(), L = 0.f;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m, float l, const f32x4& x) {
    const float mn = M != M || m != m ? __builtin_nanf("") : fmaxf(M, m), mz = finite_or_zero(mn);
    const float w0 = weight(M - mz), w1 = weight(m - mz);
    L = __builtin_fmaf(w1, l, L * w0);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = __builtin_fmaf(w1, x[e], t[e] * w0);
    M = mn;
  }
  template <int DT> __device__ __forceinline__ u32x2 out() const {
    const float inv = 1.f / L;
    u32x2 r;
    r[0] = (uint32_t)float_to_act_bits<DT>(t[0] * inv) | ((uint32_t)float_to_act_bits<DT>(t[1] * inv) << 16);
    r[1] = (uint32_t)float_to_act_bits<DT>(t[2] * inv) | ((uint32_t)float_to_act_bits<DT>(t[3] * inv) << 16);
    return r;
  }
};
typedef ShareOf<false> Share;

// Between LDS accesses of one wave whose lanes write what others read: the LDS takes a wave's accesses in their order,
// and the compiler is to leave them in it.  No instruction.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace w4
