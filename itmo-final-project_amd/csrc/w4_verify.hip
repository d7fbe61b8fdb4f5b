// Verification of drafted tokens against the target's probabilities (int4_hip/scoring.py).
#include <hip/hip_runtime.h>

#include "w4_common.hpp"

namespace w4 {

constexpr int kVerThreads = 256;
constexpr int kVerMaxDrafts = 64;
constexpr int kVerMaxParts = 64;
constexpr int kVerBufFlags = 0x00020000;  // raw buffer: the range is checked in bytes
constexpr int kVerCoherentAux = 16;       // sc1: the cache policy of agent-scope atomic loads and stores
constexpr int64_t kVerMaxVocab = 1 << 22;

struct VerifyArgs {
  const void* target;
  const void* draft;  // or null
  const int64_t* tokens;
  const int32_t* counts;  // or null
  const float *accept, *sample;
  int64_t *accepted, *token;
  unsigned* cnt;  // one arrival counter a row
  double* sums;   // [rows, parts, 2]: of the differences' weights and of the target's
  int64_t target_row, target_pos, draft_row, draft_pos;  // strides in elements
  int drafts, vocab, parts, run;  // run: tokens of a part
};

template <int DT>
__device__ __forceinline__ double prob(const void* p, int64_t i) {
  if constexpr (DT == W4_DTYPE_FP32) return (double)static_cast<const float*>(p)[i];
  else return (double)act_bits_to_float(static_cast<const uint16_t*>(p)[i], DT);
}

__device__ __forceinline__ double lane_get(double v, int lane) { return __shfl(v, lane); }

// Inclusive sum over the lanes (as wave_scan of integers: a lane with none before it adds 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan64(double v) {
  v += dpp_or_zero<0x111, 0xF>(v);  // shifted right by 1, 2, 4, 8 in rows of 16
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  v += dpp_or_zero<0x118, 0xF>(v);
  v += dpp_or_zero<0x142, 0xA>(v);  // rows 1, 3 take the last lane before them
  v += dpp_or_zero<0x143, 0xC>(v);  // rows 2, 3 take lane 31
  return v;
}

// Eight probabilities in a row as they are stored (rows need not start on 16 bytes: a vocabulary may be odd), zeros
// where there are fewer.
template <int DT> struct Eight {
  u32x4 v[DT == W4_DTYPE_FP32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i, int n) {
    if constexpr (DT == W4_DTYPE_FP32) {
      typedef u32x4 vec __attribute__((aligned(4)));
      const uint32_t* const q = static_cast<const uint32_t*>(p) + i;
      if (n >= 8) {
        v[0] = *reinterpret_cast<const vec*>(q);
        v[1] = *reinterpret_cast<const vec*>(q + 4);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e >> 2][e & 3] = e < n ? q[e] : 0u;
      }
    } else {
      typedef u32x4 vec __attribute__((aligned(2)));
      const uint16_t* const q = static_cast<const uint16_t*>(p) + i;
      if (n >= 8) {
        v[0] = *reinterpret_cast<const vec*>(q);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[0][e] = (2 * e < n ? (uint32_t)q[2 * e] : 0u) | (2 * e + 1 < n ? (uint32_t)q[2 * e + 1] << 16 : 0u);
      }
    }
  }
  __device__ __forceinline__ void values(double out[8]) const {
    float x[8];
    if constexpr (DT == W4_DTYPE_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(float, (uint32_t)v[e >> 2][e & 3]);
    } else {
      unpack8<DT>(v[0], x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = (double)x[e];
  }
};

// A row's parts of the vocabulary are a workgroup's each, eight tokens in a row a thread (more than once of vocabularies
// past 131072).  Every one of them decides on the drafts (a handful of numbers) and sums its part's weights at the first
// position that is refused, or past the last; the last part to arrive finds the part that the sample falls into and looks
// for it there.  The sums are of 64 bits, so that their order, which is fixed, moves no token but one that the sample
// meets to 2^-50.
//
// What bounds it: one row of 128256 tokens takes 7.5 us, dependent loads (probabilities of the drafts, the weights, the
// arrival, the chosen part again); 48 rows (49 MB) 20 us, 2.5 TB/s: five workgroups a CU of three dependent loads each,
// then the search of the last to arrive (47 us with four tokens a thread, 34 with eight read one by one).
template <int DT>
__global__ __launch_bounds__(kVerThreads, 5) void verify_kernel(VerifyArgs a) {
  __shared__ double sum_s[2][kVerThreads / 64];
  __shared__ unsigned arrived_s;
  __shared__ int found_s;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int n = a.counts ? a.counts[row] : a.drafts;
  if ((unsigned)n > (unsigned)a.drafts) {  // (uniform: a.drafts is not negative)
    if (part == 0 && tid == 0) a.accepted[row] = a.token[row] = -1;
    return;
  }
  bool good = false;
  if (lane < n) {
    const int64_t x = a.tokens[(int64_t)row * a.drafts + lane];
    if ((uint64_t)x < (uint64_t)a.vocab) {
      const double p = prob<DT>(a.target, row * a.target_row + lane * a.target_pos + x);
      const double q = a.draft ? prob<DT>(a.draft, row * a.draft_row + lane * a.draft_pos + x) : 1.0;
      good = (double)a.accept[(int64_t)row * a.drafts + lane] * q < p;
    }
  }
  const uint64_t refused = ~__ballot(good);
  const int r = min(refused ? __builtin_ctzll(refused) : 64, n);
  const int64_t tp = row * a.target_row + r * a.target_pos, dp = row * a.draft_row + r * a.draft_pos;
  // the token that is no choice: the refused draft, where drafts have probability 1
  const int64_t out = r < n && !a.draft ? a.tokens[(int64_t)row * a.drafts + r] : -1;
  const bool minus = r < n && a.draft;
  const int begin = part * a.run, end = min(begin + a.run, a.vocab);
  // Tokens i.. i + 7 below `to`, and their weights: of what is left of the target, and the target's own.  (What is not a
  // number stays one, so that the sum shows it.)
  auto load = [&](int i, int to, Eight<DT>& p, Eight<DT>& q) __attribute__((always_inline)) {
    p.load(a.target, tp + i, to - i);
    if (minus) q.load(a.draft, dp + i, to - i);
  };
  auto weights = [&](int i, const Eight<DT>& pr, const Eight<DT>& qr, double w[8], double p[8]) __attribute__((always_inline)) {
    double d[8];
    pr.values(p);
    if (minus) {
      qr.values(d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = i + e == out ? 1.0 : 0.0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double x = p[e] - d[e];
      w[e] = x < 0.0 ? 0.0 : x;
      p[e] = p[e] < 0.0 ? 0.0 : p[e];
    }
  };
  constexpr int ONCE = kVerThreads * 8;
  double s0 = 0.0, s1 = 0.0;
  auto sum = [&](int i, const Eight<DT>& pr, const Eight<DT>& qr) __attribute__((always_inline)) {
    double w[8], p[8];
    weights(i, pr, qr, w, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) s0 += w[e], s1 += p[e];
  };
  int i = begin + tid * 8;
  Eight<DT> p0, q0, p1, q1;
  for (; i + ONCE + 8 <= end; i += 2 * ONCE) {  // two goes' loads travel together
    load(i, end, p0, q0);
    load(i + ONCE, end, p1, q1);
    sum(i, p0, q0);
    sum(i + ONCE, p1, q1);
  }
  for (; i < end; i += ONCE) {
    load(i, end, p0, q0);
    sum(i, p0, q0);
  }
  s0 = lane_get(wave_scan64(s0), 63);
  s1 = lane_get(wave_scan64(s1), 63);
  if (lane == 0) sum_s[0][wv] = s0, sum_s[1][wv] = s1;
  __syncthreads();
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.sums + (int64_t)row * a.parts * 2), (short)0,
                                                                      a.parts * 16, kVerBufFlags);
  if (tid == 0) {
    double t[2] = {0.0, 0.0};
#pragma unroll
    for (int w = 0; w < kVerThreads / 64; ++w) t[0] += sum_s[0][w], t[1] += sum_s[1][w];
    typedef double f64x2 __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f64x2{t[0], t[1]}), rs, part * 16u, 0, kVerCoherentAux);
    __builtin_amdgcn_s_waitcnt(0);  // at the level all XCDs share
    arrived_s = __hip_atomic_fetch_add(a.cnt + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (arrived_s != (unsigned)(a.parts - 1)) return;
  if (tid == 0) __hip_atomic_store(a.cnt + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // Which weights, their sum, and the part where the sample falls: a lane a part.
  typedef double f64x2 __attribute__((ext_vector_type(2)));
  const f64x2 mine = lane < a.parts ? __builtin_bit_cast(f64x2, __builtin_amdgcn_raw_buffer_load_b128(rs, lane * 16u, 0, kVerCoherentAux))
                                    : f64x2{0.0, 0.0};
  const double u0 = wave_scan64(mine[0]), u1 = wave_scan64(mine[1]);
  const bool rest = lane_get(u0, 63) != 0.0;  // (also where it is NaN)
  const double upto = rest ? u0 : u1, own = rest ? mine[0] : mine[1], all = lane_get(upto, 63);
  if (!(all > 0.0 && all < __builtin_inf())) {
    if (tid == 0) a.accepted[row] = r, a.token[row] = -1;
    return;
  }
  const double aim = (double)a.sample[row] * all;
  // (the last with any weight, should the sample's product round up to the whole sum)
  const uint64_t past = __ballot(upto > aim && own > 0.0), any = __ballot(own > 0.0);
  const int p = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
  const double before = p ? lane_get(upto, p - 1) : 0.0;
  if (tid == 0) found_s = a.vocab;
  // That part once more, in runs of consecutive tokens: the sums up to each thread's eight, then the token.
  const int b = p * a.run, e = min(b + a.run, a.vocab);
  int hit = a.vocab, last = -1;
  double from = before;
  for (int i0 = b; i0 < e; i0 += kVerThreads * 8) {
    const int i = i0 + tid * 8;
    double w[8], t[8], s = 0.0;
    load(min(i, e), e, p0, q0);
    weights(i, p0, q0, w, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (!rest) w[k] = t[k];
      s += w[k];
    }
    const double scan = wave_scan64(s);
    if (i0 != b) __syncthreads();  // the sums before have been read
    if (lane == 63) sum_s[0][wv] = scan;
    __syncthreads();
    double x = from;
#pragma unroll
    for (int k = 0; k < kVerThreads / 64; ++k) {
      x += k < wv ? sum_s[0][k] : 0.0;
      from += sum_s[0][k];
    }
    const double lanes = __shfl_up(scan, 1);  // (of all lanes: one that does not take part gives nothing)
    x += lane ? lanes : 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x += w[k];
      if (w[k] > 0.0) {
        last = i + k;
        if (x > aim) hit = min(hit, i + k);
      }
    }
  }
  if (hit < a.vocab) atomicMin(&found_s, hit);
  __syncthreads();
  const int f = found_s;
  __syncthreads();
  if (f == a.vocab) {  // rounding: the last token of the part that has any weight
    if (tid == 0) found_s = -1;
    __syncthreads();
    atomicMax(&found_s, last);
    __syncthreads();
  }
  if (tid == 0) a.accepted[row] = r, a.token[row] = found_s;
}

}  // namespace w4

// ---------------------------------------------------------------- host side
using namespace w4host;

namespace {

struct VerifyPlan {
  int parts, run;
  int64_t slice;  // rows of a launch
};

// Parts of 2048 tokens, or of a multiple of that where there would be more of them than lanes, or more workgroups than
// the chip holds (five a CU): each begins with three loads that wait for one another.  (48 rows with two a CU
// 21.8 us, five 20.0, ten 22.8; one row in 63 parts 7.6, in sixteen 11.6.)
VerifyPlan verify_plan(int64_t rows, int64_t vocab) {
  VerifyPlan p;
  p.slice = W4_WORKSPACE_COUNTER_BYTES / 4;
  if (p.slice > rows) p.slice = rows;
  const int64_t once = 8 * w4::kVerThreads;
  int64_t parts = 5 * device_cu_count() / p.slice;
  parts = parts < 1 ? 1 : parts > w4::kVerMaxParts ? w4::kVerMaxParts : parts;
  p.run = (int)(((vocab + parts - 1) / parts + once - 1) / once * once);
  p.parts = (int)((vocab + p.run - 1) / p.run);
  return p;
}

}  // namespace

extern "C" size_t w4_verify_drafts_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > w4::kVerMaxVocab) return 0;
  const VerifyPlan p = verify_plan(rows, vocab);
  return W4_WORKSPACE_COUNTER_BYTES + (size_t)(p.slice * p.parts) * 16;
}

extern "C" int w4_verify_drafts(const void* target, const void* draft, int dtype, int64_t rows, int64_t drafts,
                                int64_t vocab, int64_t target_stride_row, int64_t target_stride,
                                int64_t draft_stride_row, int64_t draft_stride, const int64_t* tokens,
                                const int32_t* counts, const float* accept, const float* sample, int64_t* accepted,
                                int64_t* token, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16 && dtype != W4_DTYPE_FP32)
    return fail(W4_ERR_INVALID, "w4_verify_drafts: dtype must be bf16, fp16 or fp32 (got code %d)", dtype);
  if (rows < 0 || drafts < 0 || vocab < 1 || target_stride_row < 0 || target_stride < 0 || draft_stride_row < 0 ||
      draft_stride < 0)
    return fail(W4_ERR_INVALID, "w4_verify_drafts: %lld rows of %lld drafts over %lld tokens", (long long)rows,
                (long long)drafts, (long long)vocab);
  if (rows >= (1ll << 24) || drafts > w4::kVerMaxDrafts || vocab > w4::kVerMaxVocab)
    return fail(W4_ERR_UNSUPPORTED, "w4_verify_drafts: %lld rows of %lld drafts (at most %d) over %lld tokens",
                (long long)rows, (long long)drafts, w4::kVerMaxDrafts, (long long)vocab);
  if (rows == 0) return W4_OK;
  if (!target || !sample || !accepted || !token || (drafts && (!tokens || !accept)))
    return fail(W4_ERR_INVALID, "w4_verify_drafts: null pointer");
  const uintptr_t align = dtype == W4_DTYPE_FP32 ? 4 : 2;
  if ((uintptr_t)target % align || (uintptr_t)draft % align)
    return fail(W4_ERR_INVALID, "w4_verify_drafts: probabilities must be aligned to their size");
  const size_t need = w4_verify_drafts_workspace_bytes(rows, vocab);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return fail(W4_ERR_WORKSPACE, "w4_verify_drafts: needs a 256-byte aligned workspace of %zu bytes (got %zu)", need,
                workspace_bytes);
  const VerifyPlan p = verify_plan(rows, vocab);
  const int64_t bytes = (int64_t)align;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int64_t r = 0; r < rows; r += p.slice) {
    const int64_t n = rows - r < p.slice ? rows - r : p.slice;
    w4::VerifyArgs a{};
    a.target = static_cast<const char*>(target) + r * target_stride_row * bytes;
    a.draft = draft ? static_cast<const char*>(draft) + r * draft_stride_row * bytes : nullptr;
    a.tokens = tokens ? tokens + r * drafts : nullptr;
    a.counts = counts ? counts + r : nullptr;
    a.accept = accept ? accept + r * drafts : nullptr;
    a.sample = sample + r;
    a.accepted = accepted + r;
    a.token = token + r;
    a.cnt = static_cast<unsigned*>(workspace);
    a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + W4_WORKSPACE_COUNTER_BYTES);
    a.target_row = target_stride_row;
    a.target_pos = target_stride;
    a.draft_row = draft_stride_row;
    a.draft_pos = draft_stride;
    a.drafts = (int)drafts;
    a.vocab = (int)vocab;
    a.parts = p.parts;
    a.run = p.run;
    const dim3 grid((unsigned)(n * p.parts));
    if (dtype == W4_DTYPE_BF16) w4::verify_kernel<W4_DTYPE_BF16><<<grid, w4::kVerThreads, 0, st>>>(a);
    else if (dtype == W4_DTYPE_FP16) w4::verify_kernel<W4_DTYPE_FP16><<<grid, w4::kVerThreads, 0, st>>>(a);
    else w4::verify_kernel<W4_DTYPE_FP32><<<grid, w4::kVerThreads, 0, st>>>(a);
    if (const int rc = check_launch("w4_verify_drafts")) return rc;
  }
  return W4_OK;
}
