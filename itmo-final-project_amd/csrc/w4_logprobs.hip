// Log probabilities of given tokens, the entropy of their distributions and the most
// likely alternatives, from rows of logits (int4_hip/scoring.py).
#include <hip/hip_runtime.h>

#include "w4_common.hpp"

namespace w4 {

constexpr int kLogThreads = 256;
constexpr int kMaxTop = 64;
constexpr int kLogBlock = 8192;                 // logits a workgroup reads in a step: 32 a thread
constexpr int kLogGroups = kLogBlock / 128;     // groups of 128 logits in it, a quad of lanes each
constexpr int kLogMaxGroups = 192;              // groups that may hold alternatives: under 2 top + kLogGroups
constexpr int kLogNear = 1024;                  // groups whose maxima LDS holds, of a row in one part
constexpr int kLogSpare = 16;                   // groups too many, before the range of their maxima is narrowed again
constexpr int kLogList = 512;
constexpr int kLogRank = 128;                   // numbers ranked against each other
constexpr int kLogBins = 2048;
constexpr int64_t kLogMaxVocab = 1 << 22;
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kLogBufFlags = 0x00020000;        // raw buffer: the range is checked in bytes
constexpr int kLogCoherentAux = 16;             // sc1: the cache policy of agent-scope atomic loads and stores

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float *logprob, *entropy, *top_logprob;
  int64_t* top_token;
  unsigned* cnt;     // one arrival counter a row
  uint32_t* scratch; // of a row: (maximum, sum, weighted sum, -) of every part, then the keys of its groups' maxima
  int64_t stride;
  int vocab, top, parts, blocks, row_words;
};

template <int DT> struct Logits {  // 16 bytes of them
  static constexpr int N = 8;
  typedef uint16_t scalar;
  // (rows need not start on 16 bytes: a vocabulary may be odd)
  typedef u32x4 vec __attribute__((aligned(2)));
};
template <> struct Logits<W4_DTYPE_FP32> {
  static constexpr int N = 4;
  typedef float scalar;
  typedef u32x4 vec __attribute__((aligned(4)));
};

template <int DT>
__device__ __forceinline__ float logit_at(const void* x, int64_t i) {
  if constexpr (DT == W4_DTYPE_FP32) return static_cast<const float*>(x)[i];
  else return act_bits_to_float(static_cast<const uint16_t*>(x)[i], DT);
}

// Sums over some logits x of 2^y and 2^y y with y = x log2(e) - ref(m).  The reference m is their maximum; it starts at
// the lowest finite number, so that rows of -inf meet no difference of infinities.
struct LogSum {
  float m = -3.402823466e38f, s = 0.f, t = 0.f;
  static __device__ __forceinline__ bool plain(float m) { return __builtin_fabsf(m) < 1e38f; }  // m log2(e) is finite
  // ref(m) is m log2(e) rounded, which y's one fma subtracts exactly; what the rounding left out comes off the
  // logarithm at the end.
  static __device__ __forceinline__ float left(float m) {
    return plain(m) ? __builtin_fmaf(m, kLog2e, -(m * kLog2e)) : 0.f;
  }
  __device__ __forceinline__ void rebase(float to) {  // to >= m
#pragma clang fp contract(off)
    const float a = m * kLog2e, b = to * kLog2e;
    const float d = plain(m) && plain(to) ? a - b : (m - to) * kLog2e;
    const float f = __builtin_amdgcn_exp2f(d);
    // (a distance beyond all exponents: nothing is left of the sums, whatever the product)
    t = s == 0.f ? t * f : f * (fmaxf(d, -1e4f) * s + t);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float m1, float s1, float t1) {
    LogSum o;
    o.m = m1, o.s = s1, o.t = t1;
    const float to = fmaxf(m, m1);
    rebase(to), o.rebase(to);
    s += o.s, t += o.t;
  }
};

// Values of `each` between lo and hi (those above are kept, `wanted` of the `count` between are), narrowed eleven bits
// at a time until no more than `stop` are left or lo == hi; the number above grows with them.  hist is zero before and
// after.
template <typename Each>
__device__ __forceinline__ void narrow(const Each& each, uint64_t& lo, uint64_t& hi, int& wanted, int& above,
                                       int& count, int stop, int* hist, int* wave_s, int* found_s) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  constexpr int PER = kLogBins / kLogThreads;
  while (count > stop && lo < hi) {
    const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);
    each([&](uint64_t v) __attribute__((always_inline)) {
      if (v >= lo && v <= hi) atomicAdd(&hist[(int)((v - lo) >> shift)], 1);
    });
    __syncthreads();
    const int top = kLogBins - PER - PER * tid;  // from the top
    i32x4 bins[PER / 4];
    int mine = 0;
#pragma unroll
    for (int e = 0; e < PER / 4; ++e) {
      bins[e] = *reinterpret_cast<const i32x4*>(&hist[top + 4 * e]);
      *reinterpret_cast<i32x4*>(&hist[top + 4 * e]) = i32x4{0, 0, 0, 0};
      mine += bins[e][0] + bins[e][1] + bins[e][2] + bins[e][3];
    }
    const int upto = wave_scan(mine);
    if (lane == 63) wave_s[wv] = upto;
    __syncthreads();
    int over = upto - mine;
    for (int w = 0; w < wv; ++w) over += wave_s[w];
    if (over < wanted && over + mine >= wanted) {
      bool found = false;
#pragma unroll
      for (int e = PER - 1; e >= 0; --e) {
        const int in = bins[e / 4][e % 4];
        if (!found && over + in >= wanted) {
          found = true;
          found_s[0] = top + e;
          found_s[1] = over;
          found_s[2] = in;
        }
        over += in;
      }
    }
    __syncthreads();
    lo += (uint64_t)found_s[0] << shift;
    const uint64_t end = lo + ((1ull << shift) - 1ull);
    hi = end < hi ? end : hi;
    wanted -= found_s[1];
    above += found_s[1];
    count = found_s[2];
  }
}

// One workgroup = one row and part of its blocks.  Everything of a logit is done when it is read: the sums of the
// softmax and the entropy, relative to the lane's own maximum so far, and the maximum of its group of 128.  The last
// part of a row to arrive joins the sums, in their order, and finds the alternatives: as many groups reach the top-th
// largest of the groups' maxima as there are alternatives (or more, where they are equal), and no alternative lies
// outside of them, so only those groups' logits are read again.
//
// Bound by memory where there are many rows: 500 x 128256 bf16 with 20 alternatives in 31.5 us, 128 MB at 4.1 TB/s
// (five operations and an exponential a logit beside it), 1000 x 32001 fp32 without in 24.0, 128 MB at 5.3 TB/s.  A
// few rows are a chain of latencies, 8 with 5 alternatives 11.6 us; so are many short ones, a dozen barriers each and
// four workgroups on a CU: 2000 x 1000 fp32 with 20 in 30 us.
template <int DT>
__global__ __launch_bounds__(kLogThreads) void logprob_kernel(LogprobArgs a) {
  typedef Logits<DT> T;
  constexpr int NV = 32 / T::N, PIECE = 64 * T::N;  // loads of a thread in a block, logits of a wave's load
  __shared__ f32x4 sum_s[kLogThreads / 64];
  __shared__ __attribute__((aligned(16))) int hist[kLogBins];
  __shared__ uint32_t key_s[kLogNear];
  __shared__ __attribute__((aligned(16))) uint64_t list[kLogList];
  __shared__ int groups_s[kLogMaxGroups + kLogGroups];
  __shared__ int wave_s[kLogThreads / 64], found_s[3];
  __shared__ unsigned arrived_s;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int b0 = (int)((int64_t)part * a.blocks / a.parts), b1 = (int)((int64_t)(part + 1) * a.blocks / a.parts);
  const typename T::scalar* const x = static_cast<const typename T::scalar*>(a.x) + row * a.stride;
  uint32_t* const scratch = a.scratch + (int64_t)row * a.row_words;
  const __amdgpu_buffer_rsrc_t rp =
      __builtin_amdgcn_make_buffer_rsrc((void*)scratch, (short)0, a.row_words * 4, kLogBufFlags);

  // The N logits from i on; past the row: -inf.
  auto load_at = [&](int i) __attribute__((always_inline)) -> u32x4 {
    if (i + T::N <= a.vocab) return *reinterpret_cast<const typename T::vec*>(x + i);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == W4_DTYPE_FP32) {
        w[e] = i + e < a.vocab ? __builtin_bit_cast(uint32_t, x[i + e]) : 0xFF800000u;
      } else {
        const uint32_t none = DT == W4_DTYPE_BF16 ? 0xFF80u : 0xFC00u;
        const uint32_t l = i + 2 * e < a.vocab ? x[i + 2 * e] : none;
        const uint32_t h = i + 2 * e + 1 < a.vocab ? x[i + 2 * e + 1] : none;
        w[e] = l | h << 16;
      }
    }
    return u32x4{w[0], w[1], w[2], w[3]};
  };
  auto unpack = [&](const u32x4& r, float* v) __attribute__((always_inline)) {
    if constexpr (DT == W4_DTYPE_FP32) {
      const f32x4 f = __builtin_bit_cast(f32x4, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = f[e];
    } else {
      unpack8<DT>(r, v);
    }
  };
  u32x4 raw[NV];
  auto load = [&](int blk) __attribute__((always_inline)) {
    const int i0 = blk * kLogBlock + wv * 2048 + lane * T::N;
    if ((blk + 1) * kLogBlock <= a.vocab) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        raw[j] = __builtin_nontemporal_load(reinterpret_cast<const typename T::vec*>(x + i0 + j * PIECE));
    } else {  // the row's last block
#pragma unroll
      for (int j = 0; j < NV; ++j) raw[j] = load_at(i0 + j * PIECE);
    }
  };
  const int groups = a.blocks * kLogGroups;
  const bool near = a.parts == 1 && groups <= kLogNear;
  LogSum sum;
  load(b0);
  for (int i = tid; i < kLogBins; i += kLogThreads) hist[i] = 0;
  for (int blk = b0; blk < b1; ++blk) {
    float v[32];
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack(raw[j], v + T::N * j);
    if (blk + 1 < b1) load(blk + 1);  // on its way under this one's arithmetic
    float top = v[0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, v[e]);
    sum.rebase(fmaxf(sum.m, top));
    float s = 0.f, t = 0.f;
    const float ref = sum.m * kLog2e;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const float y = __builtin_fmaf(v[e], kLog2e, -ref), p = __builtin_amdgcn_exp2f(y);
      s += p;
      t = __builtin_fmaf(p, y, t);
      if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // (all at once would cost a wave a SIMD)
    }
    // -inf among them (0 * -inf; it counts nothing), numbers near the range's ends, infinities and NaN
    if (__ballot(t != t || !LogSum::plain(sum.m))) {
      s = t = 0.f;
      const bool plain = LogSum::plain(sum.m);
      float again = ref;
      asm volatile("" : "+v"(again));  // (else the exponents above would be kept in registers for here)
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float y = plain ? __builtin_fmaf(v[e], kLog2e, -again) : (v[e] - sum.m) * kLog2e;
        const float p = __builtin_amdgcn_exp2f(y);
        s += p;
        t = __builtin_fmaf(p, fmaxf(y, -1e4f), t);
        if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);
      }
    }
    sum.s += s;
    sum.t += t;
    if (a.top) {
      if (__ballot(s != s)) {  // a NaN (or a +inf) among them: NaN is above every number
#pragma unroll
        for (int e = 0; e < 32; ++e) top = v[e] != v[e] ? v[e] : top;
      }
      uint32_t key = order_key(top);
      key = max(key, dpp_mov<0xB1>(key));  // lane ^ 1
      key = max(key, dpp_mov<0x4E>(key));  // lane ^ 2
      const int g = blk * kLogGroups + wv * 16 + lane / 4;
      if ((lane & 3) == 0) {
        if (near) key_s[g] = key;
        else __builtin_amdgcn_raw_buffer_store_b32(key, rp, (uint32_t)(a.parts * 4 + g) * 4u, 0, kLogCoherentAux);
      }
    }
  }
  {
    LogSum w = sum;
    w.rebase(wave_max(sum.m));
    w.s = wave_sum(w.s), w.t = wave_sum(w.t);
    if (lane == 0) sum_s[wv] = f32x4{w.m, w.s, w.t, 0.f};
  }
  __syncthreads();
  sum = LogSum();
  for (int w = 0; w < kLogThreads / 64; ++w) sum.add(sum_s[w][0], sum_s[w][1], sum_s[w][2]);
  if (a.parts > 1) {
    if (tid == 0)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{sum.m, sum.s, sum.t, 0.f}), rp,
                                             (uint32_t)part * 16u, 0, kLogCoherentAux);
    __builtin_amdgcn_s_waitcnt(0);  // the stores have reached the level all XCDs share
    __syncthreads();
    if (tid == 0) arrived_s = __hip_atomic_fetch_add(a.cnt + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived_s != (unsigned)(a.parts - 1)) return;
    if (tid == 0) __hip_atomic_store(a.cnt + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
    if (!near) __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  auto group_key = [&](int g) __attribute__((always_inline)) {
    if (near) return key_s[g];
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rp, (uint32_t)(a.parts * 4 + g) * 4u, 0, kLogCoherentAux);
  };
  uint32_t gk[4];  // of the first 1024 groups, this thread's
  if (a.top) {
#pragma unroll
    for (int i = 0; i < 4; ++i) gk[i] = group_key(min(tid + i * kLogThreads, groups - 1));
  }
  if (a.parts > 1) {
    sum = LogSum();
    for (int p = lane; p < a.parts; p += 64) {
      const f32x4 o = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, (uint32_t)p * 16u, 0, kLogCoherentAux));
      sum.add(o[0], o[1], o[2]);
    }
    sum.rebase(wave_max(sum.m));
    sum.s = wave_sum(sum.s), sum.t = wave_sum(sum.t);
  }
  const float ln2 = 0.6931471805599453f, logs = logf(sum.s), logz = __builtin_fmaf(-LogSum::left(sum.m), ln2, logs);
  if (tid == 0) {
    a.entropy[row] = __builtin_fmaf(-ln2, sum.t / sum.s, logs);
    if (a.tokens) {
      const int64_t tok = a.tokens[row];
      a.logprob[row] =
          (uint64_t)tok < (uint64_t)a.vocab ? (logit_at<DT>(x, tok) - sum.m) - logz : __builtin_nanf("");
    }
  }
  if (a.top == 0) return;

  // The groups that may hold alternatives.
  auto each_group = [&](auto f) __attribute__((always_inline)) {  // f(group, key)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (tid + i * kLogThreads < groups) f(tid + i * kLogThreads, gk[i]);
    for (int g = tid + 4 * kLogThreads; g < groups; g += kLogThreads) f(g, group_key(g));
  };
  uint32_t low = 0xFFFFFFFFu, high = 0;
  each_group([&](int, uint32_t k) { low = min(low, k), high = max(high, k); });
  low = ~wave_umax(~low), high = wave_umax(high);
  if (lane == 0) wave_s[wv] = (int)low, groups_s[wv] = (int)high;
  if (tid == 0) found_s[0] = 0;
  __syncthreads();
  for (int w = 0; w < kLogThreads / 64; ++w)
    low = min(low, (uint32_t)wave_s[w]), high = max(high, (uint32_t)groups_s[w]);
  uint64_t lo = low, hi = high;
  int wanted = a.top, above = 0, count = groups;  // (there are at least 64)
  const int used = (a.vocab + 2047) / 2048 * 16;  // groups that hold any logits: the first ones
  __syncthreads();
  if (used > a.top)
    narrow([&](auto f) { each_group([&](int, uint32_t k) { f((uint64_t)k); }); }, lo, hi, wanted, above, count,
           kLogSpare, hist, wave_s, found_s);
  __syncthreads();
  int held = 0;
  if (used <= a.top) {  // all of them (no more than one block's; no alternative lies below the least maximum)
    if (tid < used) groups_s[tid] = tid;
    held = used;
  } else if (above + count <= kLogMaxGroups) {  // in any order
    if (tid == 0) found_s[0] = 0;
    __syncthreads();
    each_group([&](int g, uint32_t k) {
      if (k >= lo) groups_s[atomicAdd(&found_s[0], 1)] = g;
    });
    __syncthreads();
    held = found_s[0];
  } else {
    // More equal maxima than fit: those of the first blocks, until there is one for every alternative (a block is a
    // run of logits, so its equal logits come before all later ones).
    int equal = 0;
    for (int g0 = 0; g0 < groups; g0 += kLogThreads) {
      const int g = g0 + tid;
      const uint32_t k = g < groups ? group_key(g) : 0u;
      const bool same = g < groups && k == lo;
      const uint64_t m_same = __ballot(same);
      __syncthreads();
      if (lane == 0) wave_s[wv] = __popcll(m_same);
      __syncthreads();
      int before = equal;  // of the blocks in front (a wave has one block)
      for (int w = 0; w < kLogThreads / 64; ++w) {
        before += w < wv ? wave_s[w] : 0;
        equal += wave_s[w];
      }
      const bool take = g < groups && (k > lo || (same && before < a.top));
      const uint64_t m_take = __ballot(take);
      __syncthreads();
      if (lane == 0) wave_s[wv] = __popcll(m_take);
      __syncthreads();
      int at = held + __popcll(m_take & ((1ull << lane) - 1));
      for (int w = 0; w < kLogThreads / 64; ++w) {
        at += w < wv ? wave_s[w] : 0;
        held += wave_s[w];
      }
      if (take) groups_s[at] = g;
    }
  }
  __syncthreads();

  // Their logits: (key, lower index first) in one number.
  auto members = [&](auto f) __attribute__((always_inline)) {
    constexpr int VECS = 128 / T::N, STEP = kLogThreads / VECS, U = 4;  // loads of a group, groups of a step
    const int vec = tid % VECS;
    for (int i = tid / VECS; i < held; i += U * STEP) {
      int at[U];
      u32x4 r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = groups_s[min(i + u * STEP, held - 1)];
        at[u] = (g / kLogGroups) * kLogBlock + (g / 16 % 4) * 2048 + vec / 4 * PIECE + (g % 16 * 4 + vec % 4) * T::N;
        r[u] = load_at(at[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[T::N];
        unpack(r[u], v);
#pragma unroll
        for (int e = 0; e < T::N; ++e)
          if (i + u * STEP < held && at[u] + e < a.vocab) f((uint64_t)order_key(v[e]) << 32 | (uint32_t)~(at[u] + e));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  const uint64_t most = (uint64_t)high << 32 | 0xFFFFFFFFu;
  uint64_t from = lo << 32;
  int n = used <= a.top ? a.vocab : 0;  // as far as it is known
  for (;;) {
    if (n > kLogList) {
      // many equal or neighbouring logits: the threshold is sought among the members, which are all different
      uint64_t to = most;
      int want = a.top, over = 0;
      __syncthreads();
      narrow(members, from, to, want, over, n, kLogList - kMaxTop, hist, wave_s, found_s);
      __syncthreads();
    }
    if (tid == 0) found_s[0] = 0;
    __syncthreads();
    members([&](uint64_t v) __attribute__((always_inline)) {
      if (v >= from) {
        const int at = atomicAdd(&found_s[0], 1);
        if (at < kLogList) list[at] = v;
      }
    });
    __syncthreads();
    n = found_s[0];
    if (n <= kLogList) break;
  }
  // Ranked one against all; of many, those that come into question (2000 x 1000 with 20: 30 us, 51 without this and
  // the shorter ways above).
  const uint64_t* ranked = list;
  if (n > kLogRank) {
    uint64_t to = most;
    int want = a.top, over = 0, left = n;
    narrow([&](auto f) __attribute__((always_inline)) {
      for (int i = tid; i < n; i += kLogThreads) f(list[i]);
    }, from, to, want, over, left, kLogRank - kMaxTop, hist, wave_s, found_s);
    __syncthreads();
    if (tid == 0) found_s[0] = 0;
    __syncthreads();
    uint64_t* const some = reinterpret_cast<uint64_t*>(hist);
    for (int i = tid; i < n; i += kLogThreads)
      if (list[i] >= from) some[atomicAdd(&found_s[0], 1)] = list[i];
    __syncthreads();
    n = found_s[0];
    ranked = some;
  }
  for (int i = tid; i < n; i += kLogThreads) {
    const uint64_t v = ranked[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += ranked[j] > v;
    if (rank < a.top) {
      const uint32_t key = (uint32_t)(v >> 32);
      const float l = key == 0xFFFFFFFFu ? __builtin_nanf("")
                                         : __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
      a.top_token[(int64_t)row * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)v;
      a.top_logprob[(int64_t)row * a.top + rank] = (l - sum.m) - logz;
    }
  }
}

}  // namespace w4

// ---------------------------------------------------------------- host side
using namespace w4host;

namespace {

struct LogprobPlan {
  int blocks, parts;
  int64_t row_words, slice;  // words of scratch a row, rows of a launch
};

// A row is cut into parts of whole blocks while the launch has fewer than three workgroups a CU; more of them are no
// faster.
LogprobPlan logprob_plan(int64_t rows, int64_t vocab) {
  LogprobPlan p;
  p.blocks = (int)((vocab + w4::kLogBlock - 1) / w4::kLogBlock);
  const int64_t most = 3 * device_cu_count();
  p.parts = (int)(rows >= most ? 1 : most / rows < p.blocks ? most / rows : p.blocks);
  p.row_words = p.parts * 4 + (int64_t)p.blocks * w4::kLogGroups;
  // arrival counters, and no more than 64 MiB of scratch
  p.slice = W4_WORKSPACE_COUNTER_BYTES / 4;
  const int64_t fit = (64 << 20) / (p.row_words * 4);
  if (p.slice > fit) p.slice = fit;
  if (p.slice > rows) p.slice = rows;
  return p;
}

}  // namespace

extern "C" size_t w4_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  (void)top;
  if (rows < 1 || vocab < 1 || vocab > w4::kLogMaxVocab) return 0;
  const LogprobPlan p = logprob_plan(rows, vocab);
  return W4_WORKSPACE_COUNTER_BYTES + (size_t)(p.slice * p.row_words) * 4;
}

extern "C" int w4_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride,
                                 const int64_t* tokens, int64_t top, float* logprob, float* entropy,
                                 float* top_logprob, int64_t* top_token, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  clear_error();
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16 && dtype != W4_DTYPE_FP32)
    return fail(W4_ERR_INVALID, "w4_token_logprobs: dtype must be bf16, fp16 or fp32 (got code %d)", dtype);
  if (rows < 0 || vocab < 1 || vocab >= (1ll << 31) || stride < 0 || top < 0 || top > w4::kMaxTop || top > vocab)
    return fail(W4_ERR_INVALID, "w4_token_logprobs: %lld rows of %lld logits, the top %lld (at most %d)",
                (long long)rows, (long long)vocab, (long long)top, w4::kMaxTop);
  if (rows >= (1ll << 24) || vocab > w4::kLogMaxVocab)
    return fail(W4_ERR_UNSUPPORTED, "w4_token_logprobs: %lld rows of %lld logits", (long long)rows, (long long)vocab);
  if (rows == 0) return W4_OK;
  if (!logits || !entropy || (!tokens != !logprob) || (top && (!top_logprob || !top_token)))
    return fail(W4_ERR_INVALID, "w4_token_logprobs: null pointer");
  if ((uintptr_t)logits % (dtype == W4_DTYPE_FP32 ? 4 : 2))
    return fail(W4_ERR_INVALID, "w4_token_logprobs: logits must be aligned to their size");
  const size_t need = w4_token_logprobs_workspace_bytes(rows, vocab, top);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return fail(W4_ERR_WORKSPACE, "w4_token_logprobs: needs a 256-byte aligned workspace of %zu bytes (got %zu)", need,
                workspace_bytes);
  const LogprobPlan p = logprob_plan(rows, vocab);
  const int64_t bytes = dtype == W4_DTYPE_FP32 ? 4 : 2;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int64_t r = 0; r < rows; r += p.slice) {
    const int64_t n = rows - r < p.slice ? rows - r : p.slice;
    w4::LogprobArgs a{};
    a.x = static_cast<const char*>(logits) + r * stride * bytes;
    a.tokens = tokens ? tokens + r : nullptr;
    a.logprob = logprob ? logprob + r : nullptr;
    a.entropy = entropy + r;
    a.top_logprob = top_logprob ? top_logprob + r * top : nullptr;
    a.top_token = top_token ? top_token + r * top : nullptr;
    a.cnt = static_cast<unsigned*>(workspace);
    a.scratch = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + W4_WORKSPACE_COUNTER_BYTES);
    a.stride = stride;
    a.vocab = (int)vocab;
    a.top = (int)top;
    a.parts = p.parts;
    a.blocks = p.blocks;
    a.row_words = (int)p.row_words;
    const dim3 grid((unsigned)(n * p.parts));
    if (dtype == W4_DTYPE_BF16) w4::logprob_kernel<W4_DTYPE_BF16><<<grid, w4::kLogThreads, 0, st>>>(a);
    else if (dtype == W4_DTYPE_FP16) w4::logprob_kernel<W4_DTYPE_FP16><<<grid, w4::kLogThreads, 0, st>>>(a);
    else w4::logprob_kernel<W4_DTYPE_FP32><<<grid, w4::kLogThreads, 0, st>>>(a);
    if (const int rc = check_launch("w4_token_logprobs")) return rc;
  }
  return W4_OK;
}
