// Key-value cache in pages held in 8 bits (int4_hip/paged8.py): tokens quantised as
// they are written, read back, and the attention of a few new tokens of every row over
// them, of all that came before or of a sliding window and a few first tokens.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "w4_paged.hpp"

namespace w4 {

constexpr int kP8Threads = 256;

struct Paged8View {
  uint8_t* k;       // [pages, nkv, S, D] codes
  uint8_t* v;
  float* k_scale;   // [pages, nkv, S / block]
  float* v_scale;
  const int32_t* table;  // [rows, width]
  int64_t pages;
  int nkv, log2s, log2b, rows, width;

  __device__ __forceinline__ int64_t capacity() const { return (int64_t)width << log2s; }
  // The page of a slot; -1 where the table or the pool ends before.
  __device__ __forceinline__ int page(int row, int slot) const {
    const int at = slot >> log2s;
    if ((unsigned)at >= (unsigned)width) return -1;
    const int p = table[(int64_t)row * width + at];
    return (uint64_t)(int64_t)p < (uint64_t)pages ? p : -1;
  }
  // Index of a slot of a page among the pool's tokens, and of its block among the blocks, for one head.
  __device__ __forceinline__ int64_t token(int page, int head, int slot) const {
    return (((int64_t)page * nkv + head) << log2s) + (slot & ((1 << log2s) - 1));
  }
  __device__ __forceinline__ int64_t block(int page, int head, int slot) const { return token(page, head, slot) >> log2b; }
};

// The new tokens of every row: tokens offsets[b]..offsets[b + 1] go to slots lengths[b].. .
struct RowSpan {
  int len, o0, n;  // n = 0: nothing to do with this row; len < 0: idle, or refused: slots past the table, too many
};
constexpr int kP8Refused = -2;
__device__ __forceinline__ RowSpan row_span(const Paged8View& c, const int32_t* __restrict__ lengths,
                                            const int32_t* __restrict__ offsets, int tokens, int longest, int r) {
  RowSpan s{-1, 0, 0};
  if (r >= c.rows) return s;
  s.len = max(lengths[r], -1);
  s.o0 = min(max(offsets[r], 0), tokens);
  s.n = min(max(offsets[r + 1], s.o0), tokens) - s.o0;
  if ((int64_t)s.len + s.n > c.capacity() || s.n > longest) s.len = s.len < 0 ? -1 : kP8Refused;
  return s;
}

// ---------------------------------------------------------------- codes
template <int CT> struct Code;
template <> struct Code<W4_CODE_INT8> { static constexpr int most = 127; };
template <> struct Code<W4_CODE_E4M3> { static constexpr int most = 448; };

constexpr double kSmallestScale = 1.1754943508222875e-38;  // 2^-126: scales are normal numbers, or 0

__device__ __forceinline__ double two_to(int e) { return __builtin_bit_cast(double, (uint64_t)(1023 + e) << 52); }
__device__ __forceinline__ int exponent_of(double y) {  // of a normal number; -1023 of 0
  return (int)((__builtin_bit_cast(uint64_t, y) >> 52) & 0x7FF) - 1023;
}

// The code of x / s, to nearest, ties to even.  `inv` is 1 / s: the quotient is taken as x inv, an error of 2^-52, and
// divided out only where it lies within that of the middle between two codes (values with few bits, as projections
// are, do lie there).
template <int CT>
__device__ __forceinline__ uint32_t encode(double x, double s, double inv) {
  const double y = x * inv;
  double up = 1.0;
  int e = 0;
  if constexpr (CT == W4_CODE_E4M3) {  // a code is a multiple of 2^(e - 3), subnormal ones of 2^-9
    e = min(max(exponent_of(y), -6), 8);
    up = two_to(3 - e);
  }
  double t = y * up, n = __builtin_rint(t);
  if (__builtin_fabs(__builtin_fabs(t - n) - 0.5) < 1e-9) n = __builtin_rint(x / s * up);
  const int i = (int)n;
  if constexpr (CT == W4_CODE_INT8) return (uint32_t)min(max(i, -127), 127) & 0xFFu;
  // eight steps lead from one exponent to the next, so a step count and the exponent add up to the code
  const int c = min(((e + 7) << 3) + abs(i) - 8, 0x7E);
  return (uint32_t)c | (__builtin_bit_cast(uint64_t, x) >> 63 ? 0x80u : 0u);
}

template <int CT>
__device__ __forceinline__ double decode(uint32_t c) {
  if constexpr (CT == W4_CODE_INT8) return (double)(int8_t)c;
  const int e = (int)(c >> 3 & 15), m = (int)(c & 7);
  const double y = e ? (double)(8 + m) * two_to(e - 10) : (double)m * two_to(-9);
  return c & 0x80 ? -y : y;
}

// Eight codes of a block whose scale has grown by 2^m.  (Seldom: a loop, to be small.)
template <int CT>
__device__ __forceinline__ u32x2 shrink8(u32x2 w, int m) {
  const double f = two_to(-min(m, 200));
  uint64_t from = __builtin_bit_cast(uint64_t, w), r = 0;
#pragma unroll 1
  for (int e = 0; e < 64; e += 8) {
    const uint32_t c = (uint32_t)(from >> e) & 0xFFu;
    const uint32_t n = CT == W4_CODE_E4M3 && (c & 0x7F) == 0x7F ? c : encode<CT>(decode<CT>(c) * f, 1.0, 1.0);
    r |= (uint64_t)n << e;
  }
  return __builtin_bit_cast(u32x2, r);
}

// The scale of a block whose new values reach the magnitude x (of the bits of a double: an infinity or NaN among them
// is not less than one), with scale `old` (0: it begins), and by how many powers of two it has grown.
template <int CT>
__device__ __forceinline__ double block_scale(double x, double old, int* grow) {
  constexpr double Q = Code<CT>::most;
  *grow = 0;
  if (!(x < __builtin_inf()) || old != old) return __builtin_nan("");
  if (!(old > 0.0)) return x > 0.0 ? fmax((double)(float)(x / Q), kSmallestScale) : 0.0;
  if (x > Q * old) {  // the least power of two that will do
    const double r = x / (Q * old);
    const int e = exponent_of(r);
    *grow = r > two_to(e) ? e + 1 : e;
  }
  return old * two_to(*grow);
}

// Eight codes as bf16, exactly: int8 has 7 bits and a sign, e4m3 4 bits of bf16's exponents.
template <int CT>
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi) {
  u32x4 r;
  if constexpr (CT == W4_CODE_E4M3) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    auto two = [](bf16x2 v) { return __builtin_bit_cast(uint32_t, v); };
    r[0] = two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    r[1] = two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    r[2] = two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    r[3] = two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? lo : hi;
      const float a = (float)(int8_t)(w >> (16 * (i & 1))), b = (float)(int8_t)(w >> (16 * (i & 1) + 8));
      // (the upper halves of the fp32 numbers, which need no rounding)
      r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
    }
  }
  return __builtin_bit_cast(bf16x8, r);
}

// 1 in every byte that is the NaN of e4m3.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
}

// ---------------------------------------------------------------- append
struct Append8Args {
  Paged8View c;
  const uint16_t* k;  // [T, nkv * D], row strides below
  const uint16_t* v;
  int64_t stride_k, stride_v, angles;
  const int32_t *lengths, *offsets, *positions;
  const float *cos, *sin;  // [angles, D / 2]
  int tokens, longest, heads;  // heads of a workgroup
};

// Item -> a row and one of its blocks that get new tokens, counted over all rows.
__device__ __forceinline__ bool find_block(const Append8Args& a, int item, int* row, int* block, RowSpan* span) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int r = 0; r < a.c.rows; r += 64) {
    const RowSpan s = row_span(a.c, a.lengths, a.offsets, a.tokens, a.longest, r + lane);
    const int first = s.len >> a.c.log2b;
    const int blocks = s.len >= 0 && s.n > 0 ? ((s.len + s.n - 1) >> a.c.log2b) - first + 1 : 0;
    const int upto = base + wave_scan(blocks);
    const int end = __builtin_amdgcn_readlane(upto, 63);
    if (item < end) {
      const int i = __popcll(__ballot(item >= upto));
      *row = r + i;
      span->len = __builtin_amdgcn_readlane(s.len, i);
      span->o0 = __builtin_amdgcn_readlane(s.o0, i);
      span->n = __builtin_amdgcn_readlane(s.n, i);
      *block = (span->len >> a.c.log2b) + item - (__builtin_amdgcn_readlane(upto, i) - __builtin_amdgcn_readlane(blocks, i));
      return true;
    }
    base = end;
  }
  return false;
}

// The codes of a number that 32 bits hold to 2^-24, by quotients in 32 bits that are a little larger and smaller, by
// more than they may be off: in the lowest bytes of *c and of the result, which are equal but next to the middle of two.
template <int CT>
__device__ __forceinline__ uint32_t two_codes(float x, float more, float less, uint32_t* c) {
  if constexpr (CT == W4_CODE_INT8) {
    // a number this large has no bits below 1: its lowest eight are the rounded quotient's
    *c = __builtin_bit_cast(uint32_t, __builtin_fmaf(x, more, 12582912.f));
    return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, less, 12582912.f));
  } else {
    *c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x * more, x * less, 0, false);
    return *c >> 8;
  }
}
constexpr float kMore = 1.f + 0x1p-21f, kLess = 1.f - 0x1p-21f;
// Eight codes; *odd is set where one could be another.
template <int CT>
__device__ __forceinline__ u32x2 quick_codes(const float x[8], float inv, uint32_t* odd) {
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t other = two_codes<CT>(x[e], inv * kMore, inv * kLess, &c[e]);
    *odd |= (c[e] ^ other) & 0xFFu;
  }
  auto four = [&](int e) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[e + 3], c[e + 2], 0x0C0C0400u),
                                 __builtin_amdgcn_perm(c[e + 1], c[e], 0x0C0C0400u), 0x05040100u);
  };
  return u32x2{four(0), four(4)};
}
// Which of the eight.
template <int CT>
__device__ __forceinline__ unsigned odd_ones(const float x[8], float inv) {
  unsigned some = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t c;
    const uint32_t other = two_codes<CT>(x[e], inv * kMore, inv * kLess, &c);
    some |= (c ^ other) & 0xFFu ? 1u << e : 0u;
  }
  return some;
}

// One workgroup has one block of one row, for as many heads as its 256 threads hold: block * D / 16 threads a head
// (ITS = 2: twice over, of 512), eight rotary pairs of a key and the sixteen values beside them each.
//
// Keys are rotated in 64 bits, where the products of 16-bit numbers and 24-bit angles are exact, so a code is that of
// the rotated key and not of a rounding of it.  The quotients are taken in 32 bits, which finds nearly all codes; a
// thread with one that lies next to the middle between two codes takes its own again in 64.
//
// A block's scale is its largest magnitude over the largest code.  Tokens that come into a block that holds some
// already let its scale grow by a power of two, if they need it: e4m3 codes then stay as they are (but for the
// smallest), and int8 codes, each rounding at half the step of the next, are never off by more than one step in all.
//
// What bounds it: 7999 tokens of 8 x 128 (37 MB in, 16.5 out) take 18.9 us.  66 MB come in: a block's heads are eight
// workgroups, on eight XCDs, each of which fetches the angles (4.1 MB) into its own L2; so 83 MB pass at 4.4 TB/s.  Two
// thirds of a busy CU's cycles go to the vector instructions, the rotation in 64 bits and two quotients a code (50 us with
// every code in 64 bits, 31 where a thread with one doubtful code took all of its own again).  32 tokens take 6.2 us, a
// chain of dependent loads: lengths and offsets, page and position, angles and the block's scale.
template <int DT, int CT, int D, int ITS>
__global__ __launch_bounds__(kP8Threads, ITS > 1 ? 3 : 5) void paged8_append_kernel(Append8Args a) {
  constexpr int CH = D / 16;  // threads per token
  constexpr int UNITS = kP8Threads / 32;
  __shared__ unsigned long long top_s[2][UNITS];
  const int tid = threadIdx.x;
  int row, jb;
  RowSpan sp;
  const int groups = (a.c.nkv + a.heads - 1) / a.heads, go = blockIdx.x;
  if (!find_block(a, go / groups, &row, &jb, &sp)) return;
  const int slot0 = jb << a.c.log2b, per = CH << a.c.log2b;
  const int units = ITS > 1 ? 1 : kP8Threads / per, unit = ITS > 1 ? 0 : tid / per, r0 = tid - unit * per;
  const bool live = go % groups * units + unit < a.c.nkv;
  const int h = min(go % groups * units + unit, a.c.nkv - 1);
  const int page = a.c.page(row, slot0);
  if (page < 0) return;  // (uniform)
  if (tid < 2 * UNITS) (&top_s[0][0])[tid] = 0;
  const bool fresh = slot0 >= sp.len;
  const int64_t blk = a.c.block(page, h, slot0);
  float there[2] = {0.f, 0.f};  // (read before the barriers, written behind them)
  if (!fresh) there[0] = a.c.k_scale[blk], there[1] = a.c.v_scale[blk];
  __syncthreads();

  const int d = (r0 % CH) * 8;
  float x[ITS][4][8];  // the key's pairs, rotated, and the values beside them
  bool isnew[ITS];
  const uint16_t *kp[ITS], *vp[ITS];
  int64_t angle[ITS];  // of the position's row in the tables; -1: it has none
  // the largest magnitudes (as integers their order is that of the numbers, a NaN above an infinity above them all)
  uint64_t top = 0;
  uint32_t top_v = 0;
#pragma unroll
  for (int it = 0; it < ITS; ++it) {
    const int at = slot0 + (r0 + it * kP8Threads) / CH - sp.len;
    isnew[it] = live && at >= 0 && at < sp.n;
    if (!isnew[it]) continue;
    const int64_t t = sp.o0 + at;
    const int pos = a.positions[t];
    kp[it] = a.k + t * a.stride_k + h * D + d;
    vp[it] = a.v + t * a.stride_v + h * D + d;
    unpack8<DT>(*reinterpret_cast<const u32x4*>(kp[it]), x[it][0]);
    unpack8<DT>(*reinterpret_cast<const u32x4*>(kp[it] + D / 2), x[it][1]);
    unpack8<DT>(*reinterpret_cast<const u32x4*>(vp[it]), x[it][2]);
    unpack8<DT>(*reinterpret_cast<const u32x4*>(vp[it] + D / 2), x[it][3]);
    angle[it] = (uint64_t)(int64_t)pos < (uint64_t)a.angles ? (int64_t)pos * (D / 2) + d : -1;
    const f32x4* const cosp = reinterpret_cast<const f32x4*>(a.cos + max(angle[it], (int64_t)0));
    const f32x4* const sinp = reinterpret_cast<const f32x4*>(a.sin + max(angle[it], (int64_t)0));
    const f32x4 cs[2] = {cosp[0], cosp[1]}, sn[2] = {sinp[0], sinp[1]};
    double most = 0.0;
    float none = angle[it] < 0 ? __builtin_nanf("") : 0.f;  // NaN where a key is no number
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double c = (double)cs[j >> 2][j & 3], s = (double)sn[j >> 2][j & 3];
      const double x1 = (double)x[it][0][j], x2 = (double)x[it][1][j];
      const double y1 = x1 * c - x2 * s, y2 = x2 * c + x1 * s;
      most = fmax(most, fmax(__builtin_fabs(y1), __builtin_fabs(y2)));
      x[it][0][j] = (float)y1;
      x[it][1][j] = (float)y2;
      none = __builtin_fmaf(x[it][0][j], 0.f, none);
      none = __builtin_fmaf(x[it][1][j], 0.f, none);
    }
    // (a maximum leaves a NaN out; an infinity may be a number that 32 bits do not hold)
    if (none != 0.f) {
      bool wrong = angle[it] < 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        wrong = wrong || x[it][0][j] != x[it][0][j] || x[it][1][j] != x[it][1][j];
      if (wrong) most = __builtin_nan("");
    }
    const uint64_t bits = __builtin_bit_cast(uint64_t, most) & ~(1ull << 63);
    top = bits > top ? bits : top;
#pragma unroll
    for (int q = 2; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) top_v = max(top_v, __builtin_bit_cast(uint32_t, x[it][q][j]) & 0x7FFFFFFFu);
  }
  // Element j of a thread's sixteen of a key, in 64 bits.
  auto key = [&](int it, int j) {
    const int i = j & 7;
    const double x1 = act_bits_to_float(kp[it][i], DT), x2 = act_bits_to_float(kp[it][i + D / 2], DT);
    const double c = a.cos[angle[it] + i], s = a.sin[angle[it] + i];
    return j < 8 ? x1 * c - x2 * s : x2 * c + x1 * s;
  };
  if (top) atomicMax(&top_s[0][unit], (unsigned long long)top);
  if (top_v) atomicMax(&top_s[1][unit], (unsigned long long)top_v);
  __syncthreads();

  double scale[2], inv[2];
  int grow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double most = i ? (double)__builtin_bit_cast(float, (uint32_t)top_s[1][unit])
                          : __builtin_bit_cast(double, (uint64_t)top_s[0][unit]);
    scale[i] = block_scale<CT>(most, (double)there[i], &grow[i]);
    inv[i] = scale[i] > 0.0 ? 1.0 / scale[i] : 0.0;  // (also of NaN: its codes are 0)
  }
  if (!live) return;
  if (r0 == 0) {
    a.c.k_scale[blk] = (float)scale[0];
    a.c.v_scale[blk] = (float)scale[1];
  }
#pragma unroll
  for (int it = 0; it < ITS; ++it) {
    const int slot = slot0 + (r0 + it * kP8Threads) / CH;
    const int64_t at = a.c.token(page, h, slot) * D + d;
    if (isnew[it]) {
      uint32_t odd[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = q >> 1;
        u32x2 w = quick_codes<CT>(x[it][q], (float)inv[i], &odd[i]);
        if (!(inv[i] > 0.0)) w = u32x2{0u, 0u};
        *reinterpret_cast<u32x2*>((i ? a.c.v : a.c.k) + at + (q & 1) * (D / 2)) = w;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // (also where 32 bits are short of exponents)
        const double u = inv[i];
        const bool all = u > 0x1p100 || u < 0x1p-100;
        if (u > 0.0 && (odd[i] || all)) {
          unsigned some = all ? 0xFFFFu : odd_ones<CT>(x[it][2 * i], (float)u) | odd_ones<CT>(x[it][2 * i + 1], (float)u) << 8;
          for (; some; some &= some - 1) {
            const int j = __builtin_ctz(some), e = (j & 7) + (j >> 3) * (D / 2);
            const double y = i ? (double)act_bits_to_float(vp[it][e], DT) : key(it, j);
            (i ? a.c.v : a.c.k)[at + e] = (uint8_t)encode<CT>(y, scale[i], u);
          }
        }
      }
    } else {  // all codes of the block, also those behind the row's last token
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (grow[i] > 0) {
          for (int e = 0; e < 2; ++e) {
            u32x2* const p = reinterpret_cast<u32x2*>((i ? a.c.v : a.c.k) + at + e * (D / 2));
            *p = shrink8<CT>(*p, grow[i]);
          }
        }
    }
  }
}

// ---------------------------------------------------------------- read
struct Read8Args {
  Paged8View c;
  const int32_t *starts, *offsets;
  void *k, *v;  // [tokens, nkv * D]
  int tokens;
};

// Sixteen values of a key and of the value beside it a thread.  Bound by HBM: 60000 tokens of 8 x 128 to fp16 (369 MB)
// take 79 us, 4.7 TB/s (a large copy: 4.9); 300 tokens 3.5 us, a launch and three dependent loads.
template <int CT, int OUT, int D>
__global__ __launch_bounds__(kP8Threads) void paged8_read_kernel(Read8Args a) {
  constexpr int CH = D / 16;
  const int64_t i = (int64_t)blockIdx.x * kP8Threads + threadIdx.x;
  const int per = a.c.nkv * CH, lane = threadIdx.x & 63;
  const int64_t t0 = ((int64_t)blockIdx.x * kP8Threads + (threadIdx.x & ~63)) / per;  // the wave's first token
  int row = 0;
  for (int r = 0; r < a.c.rows; r += 64) {
    const int n = __popcll(__ballot(r + lane < a.c.rows && a.offsets[r + lane + 1] <= t0));
    row += n;
    if (n < 64) break;
  }
  const int64_t t = i / per;
  if (t >= a.tokens) return;
  while (row < a.c.rows && a.offsets[row + 1] <= t) ++row;
  const int r = (int)(i - t * per), h = r / CH, d = (r % CH) * 16;
  bool zero = row >= a.c.rows, bad = false;
  u32x4 kw = {0u, 0u, 0u, 0u}, vw = {0u, 0u, 0u, 0u};
  float ks = 0.f, vs = 0.f;
  if (!zero) {
    const int start = a.starts[row];
    const int64_t o0 = a.offsets[row], slot = start + t - o0;
    zero = start < 0 || t < o0;
    if (!zero) {
      const int page = slot < a.c.capacity() ? a.c.page(row, (int)slot) : -1;
      bad = page < 0;
      if (!bad) {
        const int64_t at = a.c.token(page, h, (int)slot) * D + d, blk = a.c.block(page, h, (int)slot);
        kw = *reinterpret_cast<const u32x4*>(a.c.k + at);
        vw = *reinterpret_cast<const u32x4*>(a.c.v + at);
        ks = a.c.k_scale[blk];
        vs = a.c.v_scale[blk];
      }
    }
  }
  if (bad) ks = vs = __builtin_nanf("");
  const int64_t out = t * ((int64_t)a.c.nkv * D) + h * D + d;
  auto put = [&](void* to, const u32x4& w, float s) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float x[8];
      unpack8<W4_DTYPE_BF16>(__builtin_bit_cast(u32x4, codes8<CT>(w[2 * g], w[2 * g + 1])), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = zero ? 0.f : x[e] * s;
      if constexpr (OUT == W4_DTYPE_FP32) {
        f32x4* const p = reinterpret_cast<f32x4*>(static_cast<float*>(to) + out + 8 * g);
        p[0] = f32x4{x[0], x[1], x[2], x[3]};
        p[1] = f32x4{x[4], x[5], x[6], x[7]};
      } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(to) + out + 8 * g) = pack8<OUT>(x);
      }
    }
  };
  put(a.k, kw, ks);
  put(a.v, vw, vs);
}

// ---------------------------------------------------------------- attention
struct Attend8Args {
  Paged8View c;
  const uint16_t* q;
  int64_t stride_q, angles;
  const int32_t *lengths, *offsets, *positions;
  const float *cos, *sin;
  uint16_t* out;  // [tokens, nkv * g * D]
  float* part;    // [split items, 16, D]: outputs of the parts of tiles whose slots are cut
  float* stats;   // [split items, 16, 2]: their references and sums
  unsigned* cnt;  // arrival counters of those tiles
  float scale;    // 1 / sqrt(D)
  const uint16_t *k, *v;  // PUT: the new tokens', which the attention writes itself
  int64_t stride_k, stride_v;
  int tokens, longest, g, window, sinks;  // window: 0 for none
  int many;  // rows of so many new tokens and more are paged8_prompt_kernel's
};

// The work of one workgroup: a tile of sixteen (new token, query head) columns of one row and key-value head, and a
// part of the slots that they see.
struct Item8 {
  int b, h, tile, part, parts;
  int len, o0, n;
  int first, counter;  // of a tile in several parts: the index of part 0 among such parts, and of the tile among such tiles
};

constexpr int kP8Unit = 32;  // slots that a wave takes at once
constexpr int kP8AtOnce = 8;  // parts that a thread of the joining reads together
constexpr int kP8Waves = 4, kP8MinUnits = 4;
// A part takes time with its units, the joining of a tile with its parts, eight at once: parts of sqrt(units / 2) units at
// least keep the two alike.  (Without: one row of 60000 slots of 20 / 2 heads of 128 84 us, with 39, one of 131000 of 6 / 1
// 89 and 41; 4000 of 8 / 2 of 64 10.2 and 11.0.  Of sqrt(units / 5): 46.5, 41, 10.8; sqrt(1.5 units): 40.5, 47.6, 12.3.)
constexpr float kP8Join = 0.5f;
// Three parts a CU with heads of 64, two with those of 128, as measured.  (512 and 768: 32 ragged rows of 64 26.0 and 24.8
// us; 131000 slots of 128 57 and 76, drafts 24 and 28.)
constexpr int p8_parts(int d) { return d == 64 ? 768 : 512; }

// Rows are cut into parts of about (all columns' tiles x units of slots) / PARTS, so that time follows the slots there
// are and not the table.  Those that are cut have at most 2 * PARTS parts in all: each has more units than `per`, and
// PARTS * per are at least all there are.
template <int UP, int PARTS>
__device__ __forceinline__ bool find_item8(const Attend8Args& a, int item, Item8* it, int* total) {
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](const RowSpan& s) { return s.n < a.many ? a.c.nkv * (int)(((int64_t)s.n * a.g + 15) / 16) : 0; };
  // units that one tile of a row reads at most, or nearly so
  auto units_of = [&](const RowSpan& s) {
    if (s.len < 0 || s.n == 0) return 1;
    const int all = (s.len + s.n - 1) / UP + 1;
    if (!a.window) return all;
    const int64_t span = (int64_t)a.window + min((16 + a.g - 2) / a.g, s.n - 1);
    return (int)min((int64_t)all, span / UP + 2 + (a.sinks + UP - 1) / UP);
  };
  auto span = [&](int r) { return row_span(a.c, a.lengths, a.offsets, a.tokens, a.longest, r + lane); };
  const RowSpan s0 = span(0);
  float all = (float)tiles_of(s0) * (float)units_of(s0), news = (float)s0.n;
  for (int r = 64; r < a.c.rows; r += 64) {
    const RowSpan s = span(r);
    all += (float)tiles_of(s) * (float)units_of(s);
    news += (float)s.n;
  }
  all = wave_sum(all);
  // Rows that overlap (offsets that decrease) may need more workgroups than there are: none of them is cut, or parts
  // would wait for others that never come, and their counter be left for the next call.
  const bool overlap = wave_sum(news) > (float)a.tokens;
  // (rounded up beyond what the sum's own rounding can have taken)
  const int per = overlap ? INT32_MAX : max((int)fminf(ceilf(all * (1.0001f / PARTS)), 1e9f), kP8MinUnits);
  int base = 0, split = 0, counters = 0;
  for (int r = 0; r < a.c.rows; r += 64) {
    const RowSpan s = r ? span(r) : s0;
    const int tiles = tiles_of(s), units = units_of(s);
    const int parts = 1 + (units - 1) / max(per, (int)__builtin_amdgcn_sqrtf((float)units * kP8Join));
    const int upto = base + wave_scan(parts * tiles);
    const int split_to = split + wave_scan(parts > 1 ? parts * tiles : 0);
    const int counters_to = counters + wave_scan(parts > 1 ? tiles : 0);
    const int end = __builtin_amdgcn_readlane(upto, 63);
    if (item < end) {
      const int i = __popcll(__ballot(item >= upto));
      auto at = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
      it->parts = at(parts);
      const int rem = item - (at(upto) - it->parts * at(tiles)), tile = rem / it->parts;
      it->b = r + i;
      it->part = rem - tile * it->parts;
      it->first = at(split_to) - (at(tiles) - tile) * it->parts;
      it->counter = at(counters_to) - (at(tiles) - tile);
      it->len = at(s.len), it->o0 = at(s.o0), it->n = at(s.n);
      it->tile = tile / a.c.nkv;
      it->h = tile - it->tile * a.c.nkv;
      return true;
    }
    base = end;
    split = __builtin_amdgcn_readlane(split_to, 63);
    counters = __builtin_amdgcn_readlane(counters_to, 63);
  }
  *total = base;
  return false;
}

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

typedef ShareOf<true> Share8;

// Eight codes, which fp16 holds exactly.
template <int CT>
__device__ __forceinline__ f16x8 codes8h(uint32_t lo, uint32_t hi) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 r[4];
  if constexpr (CT == W4_CODE_E4M3) {
    r[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    r[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    r[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    r[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  } else {
    // below the exponent of 1024 a byte is 1024 + the code + 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = (i < 2 ? lo : hi) ^ 0x80808080u;
      const uint32_t b = __builtin_amdgcn_perm(0x64646464u, w, i & 1 ? 0x04030402u : 0x04010400u);
      r[i] = __builtin_bit_cast(f16x2, b) - (f16x2){(_Float16)1152.f, (_Float16)1152.f};
    }
  }
  return __builtin_bit_cast(f16x8, (u32x4){__builtin_bit_cast(uint32_t, r[0]), __builtin_bit_cast(uint32_t, r[1]),
                                           __builtin_bit_cast(uint32_t, r[2]), __builtin_bit_cast(uint32_t, r[3])});
}

// Numbers below 2^16 as the sums of two of fp16, each with 11 bits and a sign of its own: three in four exactly, the others
// within 2^-23 of themselves (the last of 24 bits); to 2^-25 where they are so small that fp16 has no smaller step.
__device__ __forceinline__ void halves8(const float x[8], f16x8 out[2]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 h[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), f16x2);
    r[i] = __builtin_convertvector((f32x2{x[2 * i] - (float)h[i][0], x[2 * i + 1] - (float)h[i][1]}), f16x2);
  }
  __builtin_memcpy(&out[0], h, 16);
  __builtin_memcpy(&out[1], r, 16);
}

// The power of two (2^-115.. 2^126) that takes numbers up to `most` below 2^to and above 2^(to - 2).
__device__ __forceinline__ float raise_to(float most, int to) {
  const int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23 & 0xFF) - 127;  // most < 2^(e + 1)
  return __builtin_bit_cast(float, (uint32_t)(min(max(to - 1 - e, -115), 126) + 127) << 23);
}
__device__ __forceinline__ float inverse_power(float f) {  // of such a power
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, f));
}

// A column's rotated query, of which a lane has some elements, in two parts of fp16; the factor it is short of,
// times log2(e).  One that holds an infinity or NaN is NaN.
template <int NJ>
__device__ __forceinline__ float query_parts(const float (*x)[8], f16x8 (*qf)[2]) {
  float top = 0.f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, __builtin_fabsf(x[j][e]));
      odd |= !(__builtin_fabsf(x[j][e]) < __builtin_inff());
    }
  if (odd) top = __builtin_inff();
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const float f = raise_to(top, 15);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[j][e] * f;
    halves8(y, qf[j]);
  }
  return top < __builtin_inff() ? kLog2e * inverse_power(f) : __builtin_nanf("");
}

// Which of the slots from.. from + 7 the token of slot `mine` sees, a bit each.
__device__ __forceinline__ uint32_t seen8(int from, int mine, int window, int sinks) {
  auto below = [&](int slot) { return (1u << min(max(max(slot, 0) - from, 0), 8)) - 1u; };  // those before it
  uint32_t v = below(mine + 1);
  if (window) v &= ~below(mine - window + 1) | below(sinks);
  return v;
}

// A workgroup's four waves take units of 32 slots in turn, each its own.
//
// Both products are 16x16x32 fp16 matrix instructions, transposed, with the columns (new tokens x query heads of the
// group) as their columns: S^T = K Q^T, then O^T = V^T P^T.  Codes are fp16 numbers exactly; the scales stay outside: a
// slot's score is multiplied by its key's, its probability by its value's, which makes its weight.  Queries and weights
// enter as the sum of two fp16 numbers, so within 2^-23 of themselves, twice fp32's own rounding at most, as long as they
// are not far below the largest of their column: a power of two takes a column's queries and weights below 2^15, and what
// is far below is then off by 2^-38 of the largest query at most, by 2^-35 (2^-40 at best) of the largest weight.  The
// weights' power follows the largest so far: it changes with the softmax's reference, and when a weight passes 2^15.
// (Three bf16 numbers each hold any size and cost half as many matrix instructions again and twice the other ones: 32
// rows of up to 4000 slots 29.3 us instead of 26.8, 131000 slots 63 instead of 58, a window 25 instead of 21.)
//
// Keys come from memory straight into the first product's operand: its inner index may run over a head in any order,
// so a lane takes sixteen bytes in a row of a slot, four lanes 64.  A tile's row r is slot 8 (r / 4) + 4 t + r % 4 of its
// block of 32 (t: the first or second tile), so the scores that a lane holds of a column are those of eight slots in a
// row, its part of the second product's operand.  Values go through a wave's own LDS, which transposes them on reading.
//
// PUT: no row has more than one new token, a row's and head's columns are one tile, and a block lies in one unit: the
// wave that takes a row's last unit writes the token (and, where the block's scale grows, its other codes), as
// paged8_append_kernel does.  That saves a launch: 100 slots 9.0 us a call instead of 12.4, 32 rows of up to 4000 24.7
// instead of 28.3, one of 131000 56.8 instead of 58.9.
//
// What bounds it: one row of 131000 slots of 8 x 128 (268 MB) takes 56 us, 4.8 TB/s, HBM.  32 rows of up to 4000 slots of
// 8 x 64 (62 MB) take 24.2 us, 24 windows of 128-wide heads (49 MB) 20.4: of either, the vector instructions (conversion of
// codes, softmax, weights in two parts) take about half the cycles of a busy CU and the matrix instructions a twelfth, and
// 7 us go before the first and after the last unit.  Five drafts of four query heads are 20 columns, two tiles, each of
// which converts all codes: 16 rows of 3001 slots with one to five drafts 23.8 us.  100 slots: 7.9 us of dependent loads.
template <int DT, int CT, int D, int W, bool PUT>
__global__ __launch_bounds__(64 * W, D == 64 ? 4 : PUT ? 2 : 3) void paged8_attention_kernel(Attend8Args a) {
  constexpr int UP = kP8Unit, KB = UP / 32, NJ = D / 32, ND = D / 16;
  constexpr int KC = D / 64;               // 16-byte loads of a key a lane
  constexpr int VR = 1024 / D, VC = D / 16;  // rows of values in a load of the wave, 16-byte chunks of a row
  constexpr int NV = UP / VR;
  constexpr int OROW = D + 4;              // floats of an output row in LDS
  constexpr int WAVE_B = 16 * OROW * 4 > UP * D ? 16 * OROW * 4 : UP * D;
  constexpr int kThreads = 64 * W;
  typedef Mfma<W4_DTYPE_FP16> M;
  __shared__ __attribute__((aligned(16))) uint8_t v_s[W][WAVE_B];
  __shared__ float m_s[W][16], l_s[W][16];
  __shared__ __attribute__((aligned(16))) uint8_t new_s[2][D];
  __shared__ unsigned arrived_s;
  static_assert(!PUT || KB == 1, "a block lies in one unit");

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, c = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nh = a.c.nkv * a.g;
  Item8 it;
  int total;
  if (!find_item8<UP, p8_parts(D)>(a, blockIdx.x, &it, &total)) {
    // what is left over of the launch (one workgroup at least): tokens of no row
    const int before = a.c.rows ? min(max(a.offsets[0], 0), a.tokens) : 0;
    const int after = a.c.rows ? min(max(a.offsets[a.c.rows], before), a.tokens) : 0;
    const int pads = before + a.tokens - after;
    for (int64_t i = (int64_t)(blockIdx.x - total) * kThreads + tid; i < (int64_t)pads * (nh * D / 8);
         i += (int64_t)(gridDim.x - total) * kThreads) {
      const int64_t p = i / (nh * D / 8), t = p < before ? p : p - before + after;
      *reinterpret_cast<u32x4*>(a.out + t * (nh * D) + (i - p * (nh * D / 8)) * 8) = u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
  const int b = it.b, h = it.h, len = it.len;
  const int col0 = it.tile * 16, cols = min(it.n * a.g - col0, 16);
  // where column `col` of the tile goes
  auto out_at = [&](int col) {
    const int j = (col0 + col) / a.g;
    return a.out + ((int64_t)(it.o0 + j) * nh + h * a.g + (col0 + col - j * a.g)) * D;
  };
  if (len < 0) {
    const uint16_t fill = len == kP8Refused ? float_to_act_bits<DT>(__builtin_nanf("")) : 0;
    for (int i = tid; i < cols * D; i += kThreads) out_at(i / D)[i % D] = fill;
    return;
  }
  // The slots that the tile's columns see: lo..hi of the first's and the last's tokens, and the sinks before.
  const int first_slot = len + col0 / a.g, last_slot = len + (col0 + cols - 1) / a.g;
  const int lo = a.window ? max(first_slot - a.window + 1, 0) : 0;
  const int u_lo = lo / UP, sink_units = a.window ? min((a.sinks + UP - 1) / UP, u_lo) : 0;
  const int units = sink_units + last_slot / UP - u_lo + 1;
  auto base_of = [&](int u) { return (u < sink_units ? u : u_lo + u - sink_units) * UP; };
  const int u0 = (int)((int64_t)it.part * units / it.parts), u1 = (int)((int64_t)(it.part + 1) * units / it.parts);

  u32x4 kr[KB][2][KC], vr[NV];
  float ks[KB], vs[KB];
  int ids[KB], next_ids[KB];
  const int32_t* const table = a.c.table + (int64_t)b * a.c.width;
  // Lane: the pages of the groups of eight slots that its rows of keys are in, as the table has them.  (Looked at
  // before they are needed, they would make the wave wait for all the loads before them.)
  auto load_ids = [&](int u, int id[KB]) __attribute__((always_inline)) {
    const int base = base_of(u);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      id[kb] = table[min(base + kb * 32 + 8 * (l16 >> 2), last_slot) >> a.c.log2s];
  };
  auto load = [&](int u) __attribute__((always_inline)) {
    const int base = base_of(u);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      ids[kb] = base + kb * 32 + 8 * (l16 >> 2) <= last_slot && (uint64_t)(int64_t)ids[kb] < (uint64_t)a.c.pages ? ids[kb] : -1;
      const int64_t at = a.c.token(max(ids[kb], 0), h, base + kb * 32 + 8 * (l16 >> 2) + (l16 & 3));
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < KC; ++i)
          kr[kb][t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.k + (at + 4 * t) * D + 64 * i + 16 * c));
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {  // (the lane's scores are of group c)
      const int id = __shfl(ids[kb], 4 * c);
      const int64_t blk = a.c.block(max(id, 0), h, base + kb * 32 + 8 * c);
      const float k0 = a.c.k_scale[blk], v0 = a.c.v_scale[blk];
      ks[kb] = id < 0 ? __builtin_nanf("") : k0;
      vs[kb] = id < 0 ? __builtin_nanf("") : v0;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      int page;
      if constexpr (D == 128) {
        page = __builtin_amdgcn_readlane(ids[i >> 2], 4 * (i & 3));
      } else {
        const int p0 = __builtin_amdgcn_readlane(ids[i >> 1], 8 * (i & 1)),
                  p1 = __builtin_amdgcn_readlane(ids[i >> 1], 8 * (i & 1) + 4);
        page = lane < 32 ? p0 : p1;
      }
      const int64_t at = a.c.token(max(page, 0), h, base + i * VR + lane / VC);
      vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.v + at * D + (lane % VC) * 16));
    }
  };
  // The 16-byte chunk of a row of values lies where it shares no bank with those that are read beside it.
  // (The same for rows 8, D = 64: 16, apart, so loads and blocks of 32 slots are a constant apart.)
  auto swizzle = [&](int row) { return D == 128 ? row & 7 : (row >> 2) & 3; };
  uint8_t* const vw = v_s[wv];
  const int put_at = lane / VC * D + (((lane % VC) ^ swizzle(lane / VC)) << 4);
  const int get_row = 8 * c + (l16 >> 1), get_at = get_row * D + (swizzle(get_row) << 4) + 8 * (l16 & 1);

  int u = u0 + wv;
  if (u < u1) {  // on their way before the query is at hand
    load_ids(u, ids);
    load(u);
    load_ids(min(u + W, u1 - 1), next_ids);
  }

  // The query of this lane's column; columns past the last copy it and count for nothing.
  const int col = min(l16, cols - 1), tok = it.o0 + (col0 + col) / a.g;
  const int mine = len + (col0 + col) / a.g;  // its slot
  f16x8 qf[NJ][2];
  float q_short;
  {
    float xs[NJ][8];
    const int pos = a.positions[tok];
    const bool there = (uint64_t)(int64_t)pos < (uint64_t)a.angles;
    const uint16_t* const qp = a.q + tok * a.stride_q + (h * a.g + (col0 + col) % a.g) * D;
    const float* const cosr = a.cos + (there ? (int64_t)pos * (D / 2) : 0);
    const float* const sinr = a.sin + (there ? (int64_t)pos * (D / 2) : 0);
    const float scale = there ? a.scale : __builtin_nanf("");
    // chunk j: elements 64 (j / 2) + 16 c + 8 (j % 2).. ; those that they are rotated with are D / 2 from them, in another
    // chunk of the lane or (D = 64) another lane's
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float* const x = xs[j];
      const int d = 64 * (j >> 1) + 16 * c + 8 * (j & 1), da = d & (D / 2 - 1);
      const bool low = D == 128 ? j < 2 : c < 2;
      float y[8];
      unpack8<DT>(*reinterpret_cast<const u32x4*>(qp + d), x);
      unpack8<DT>(*reinterpret_cast<const u32x4*>(qp + (d ^ (D / 2))), y);
      const f32x4* const cp = reinterpret_cast<const f32x4*>(cosr + da);
      const f32x4* const sp = reinterpret_cast<const f32x4*>(sinr + da);
      const f32x4 cs[2] = {cp[0], cp[1]}, sn[2] = {sp[0], sp[1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float cc = cs[e >> 2][e & 3], ss = sn[e >> 2][e & 3];
        float r1, r2;
        if (low) rope_pair(x[e], y[e], cc, ss, &r1, &r2), x[e] = r1 * scale;
        else rope_pair(y[e], x[e], cc, ss, &r1, &r2), x[e] = r2 * scale;
      }
    }
    q_short = query_parts<NJ>(xs, qf);
  }

  // The new token, quantised (the wave that takes the last unit): its codes in LDS, its block's scales.
  uint32_t new_scale[2];
  int grow[2];
  if constexpr (PUT) {
    if (it.part == it.parts - 1 && wv == (units - 1 - u0) % W) {
      const int pos = a.positions[it.o0], lane2 = lane & (D / 2 - 1);
      const bool there = (uint64_t)(int64_t)pos < (uint64_t)a.angles;
      const uint16_t* const kp = a.k + it.o0 * a.stride_k + h * D;
      const uint16_t* const vp = a.v + it.o0 * a.stride_v + h * D;
      const int64_t at = there ? (int64_t)pos * (D / 2) + lane2 : 0;
      const double cc = there ? (double)a.cos[at] : (double)__builtin_nanf(""), ss = (double)a.sin[at];
      const double x1 = act_bits_to_float(kp[lane2], DT), x2 = act_bits_to_float(kp[lane2 + D / 2], DT);
      const double x[2][2] = {{x1 * cc - x2 * ss, x2 * cc + x1 * ss},
                              {act_bits_to_float(vp[lane2], DT), act_bits_to_float(vp[lane2 + D / 2], DT)}};
      const int page = a.c.page(b, len);
      const bool fresh = (len & ((1 << a.c.log2b) - 1)) == 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t y1 = __builtin_bit_cast(uint64_t, __builtin_fabs(x[i][0])),
                       y2 = __builtin_bit_cast(uint64_t, __builtin_fabs(x[i][1])), y = y1 > y2 ? y1 : y2;
        const uint32_t hi = wave_umax((uint32_t)(y >> 32));
        const uint32_t lo = wave_umax((uint32_t)(y >> 32) == hi ? (uint32_t)y : 0u);
        const double old = fresh || page < 0 ? 0.0 : (double)(i ? a.c.v_scale : a.c.k_scale)[a.c.block(page, h, len)];
        const double scale = block_scale<CT>(__builtin_bit_cast(double, (uint64_t)hi << 32 | lo), old, &grow[i]);
        const double inv = scale > 0.0 ? 1.0 / scale : 0.0;
        grow[i] = __builtin_amdgcn_readfirstlane(grow[i]);
        new_scale[i] = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, (float)scale));
#pragma unroll
        for (int e = 0; e < 2; ++e)
          new_s[i][lane2 + e * (D / 2)] = (uint8_t)(inv > 0.0 ? encode<CT>(x[i][e], scale, inv) : 0u);
      }
    }
  }

  float m = -__builtin_inff(), l = 0.f;  // the column's reference and this lane's share of its sum
  float heavy = 0.f, lift = 1.f;         // the largest of this lane's weights, what the column's are multiplied by
  f32x4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (; u < u1; u += W) {
    const int base = base_of(u);
    if constexpr (PUT) {
      const int page = u == units - 1 ? a.c.page(b, len) : -1;
      if (page >= 0) {
        const int slot0 = len & ~((1 << a.c.log2b) - 1);
        const int64_t tok0 = a.c.token(page, h, slot0), blk = a.c.block(page, h, len);
        if (grow[0] > 0 || grow[1] > 0) {
          for (int i = 0; i < 2; ++i) {
            if (grow[i] == 0) continue;
            uint8_t* const p = (i ? a.c.v : a.c.k) + tok0 * D;
            for (int j = lane * 8; j < D << a.c.log2b; j += 512)
              *reinterpret_cast<u32x2*>(p + j) = shrink8<CT>(*reinterpret_cast<const u32x2*>(p + j), grow[i]);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // other lanes load what a lane has stored
          load(u);
        }
        wave_lds_order();
        const int row = len - base;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const u32x4 n = *reinterpret_cast<const u32x4*>(&new_s[0][64 * i + 16 * c]);
            if (8 * (l16 >> 2) + 4 * t + (l16 & 3) == row) kr[0][t][i] = n;
          }
        const u32x4 n = *reinterpret_cast<const u32x4*>(&new_s[1][lane % VC * 16]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i * VR + lane / VC == row) vr[i] = n;
        if ((base + 8 * c) >> a.c.log2b == len >> a.c.log2b) {
          ks[0] = __builtin_bit_cast(float, new_scale[0]);
          vs[0] = __builtin_bit_cast(float, new_scale[1]);
        }
        if (lane < D / 16) {
          const int64_t at = a.c.token(page, h, len) * D + lane * 16;
          *reinterpret_cast<u32x4*>(a.c.k + at) = *reinterpret_cast<const u32x4*>(&new_s[0][lane * 16]);
          *reinterpret_cast<u32x4*>(a.c.v + at) = *reinterpret_cast<const u32x4*>(&new_s[1][lane * 16]);
        }
        if (lane == 0) {
          a.c.k_scale[blk] = __builtin_bit_cast(float, new_scale[0]);
          a.c.v_scale[blk] = __builtin_bit_cast(float, new_scale[1]);
        }
      }
    }
    f32x4 s[KB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f16x8 kf[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          uint32_t k0 = kr[kb][t][j >> 1][2 * (j & 1)], k1 = kr[kb][t][j >> 1][2 * (j & 1) + 1];
          // (hidden, or the compiler converts where the words are loaded and holds four times as many registers)
          asm("" : "+v"(k0), "+v"(k1));
          kf[j] = codes8h<CT>(k0, k1);
        }
        s[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 1; p >= 0; --p)  // the small parts first
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[kb][t] = M::m16(kf[j], qf[j][p], s[kb][t]);
      }
    // A slot that a column does not see has score -inf and, whatever is stored there, no share in the output.
    const bool whole = base + UP - 1 <= first_slot && (!a.window || base > last_slot - a.window || base + UP <= a.sinks);
    wave_lds_order();  // the unit before has been read
#pragma unroll
    for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4*>(vw + put_at + i * (VR * D)) = vr[i];
    wave_lds_order();
    if constexpr (CT == W4_CODE_E4M3) {
      // e4m3 has a NaN: what a program that is not this one left in the pages.  It must not meet the probability 0 of a
      // slot that is not seen, so it is taken out here, and what sees it is made NaN by itself.  (Where all is seen, it
      // does its work.)
      if (!whole) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) any |= nan_bytes(vr[i][e]);
        if (__ballot(any != 0)) {
          for (int row = 0; row < UP; ++row) {
            const bool see = seen8(base + row, mine, a.window, a.sinks) & 1;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(vw + row * D + ((d ^ swizzle(row)) << 4) + 4 * c);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (see && (w >> (8 * e) & 0x7F) == 0x7F) o[d][e] = __builtin_nanf("");
            }
          }
          wave_lds_order();
#pragma unroll
          for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[i][e] &= ~(nan_bytes(vr[i][e]) * 0xFFu);
            *reinterpret_cast<u32x4*>(vw + put_at + i * (VR * D)) = vr[i];
          }
          wave_lds_order();
        }
      }
    }
    float sk[KB], sv[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) sk[kb] = ks[kb] * q_short, sv[kb] = vs[kb];
    if (u + W < u1) {  // the next unit's loads travel under the rest
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) ids[kb] = next_ids[kb];
      load(u + W);
      load_ids(min(u + 2 * W, u1 - 1), next_ids);
    }

#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[kb][t] *= sk[kb];
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t sight = seen8(base + kb * 32 + 8 * c, mine, a.window, a.sinks);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[kb][e >> 2][e & 3] = sight >> e & 1 ? s[kb][e >> 2][e & 3] : -__builtin_inff();
        // (a scale that is NaN is no matter of a token that sees none of its slots)
        sv[kb] = sight ? sv[kb] : 0.f;
      }
    }
    float top = -__builtin_inff(), top_kb[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      top_kb[kb] = s[kb][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top_kb[kb] = fmaxf(top_kb[kb], s[kb][e >> 2][e & 3]);
      top = fmaxf(top, top_kb[kb]);
    }
    // Scores are exponents of 2.  A column's reference is raised, to 2 above its largest score so far, once a score passes
    // it by 6: probabilities are 2^6 at most.
    float al = 1.f;
    if (__ballot(top - m > 6.f)) {
      float mn = fmaxf(top, __shfl_xor(top, 16));
      mn = fmaxf(mn, __shfl_xor(mn, 32));
      mn = mn - m > 6.f ? mn + 2.f : m;
      al = __builtin_amdgcn_exp2f(m - finite_or_zero(mn));
      l *= al;
      heavy *= al;
      m = mn;
    }
    const float mz = finite_or_zero(m);
    auto prob = [&](float x) { return __builtin_amdgcn_exp2f(x - mz); };
    // The largest of eight slots' weights with one scale is that of their largest score.
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) heavy = fmaxf(heavy, prob(top_kb[kb]) * sv[kb]);
    if (__ballot(al < 1.f || heavy * lift > 0x1p15f)) {
      heavy = fmaxf(heavy, __shfl_xor(heavy, 16));
      heavy = fmaxf(heavy, __shfl_xor(heavy, 32));
      const float to = al < 1.f || heavy * lift > 0x1p15f ? raise_to(heavy, 12) : lift;
      const float by = al * fminf(to * inverse_power(lift), 0x1p127f);
      lift = to;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= by;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = prob(s[kb][e >> 2][e & 3]);
        l += p[e];
        p[e] = p[e] * sv[kb] * lift;
      }
      f16x8 pf[2];
      halves8(p, pf);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2)(vw + (get_at ^ (d << 4)) + kb * (32 * D)));
        const f16x8 vf = codes8h<CT>((uint32_t)w[0], (uint32_t)w[1]);
#pragma unroll
        for (int q = 1; q >= 0; --q) o[d] = M::m16(vf, pf[q], o[d]);
      }
    }
  }

  // The waves' outputs meet in LDS.
  wave_lds_order();
  float* const ow = reinterpret_cast<float*>(vw);
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int d = 0; d < ND; ++d)
    *reinterpret_cast<f32x4*>(ow + l16 * OROW + d * 16 + 4 * c) = o[d] * (0x1p-6f * inverse_power(lift));
  if (c == 0) m_s[wv][l16] = m, l_s[wv][l16] = 0x1p-6f * l;
  __syncthreads();
  constexpr int STRIDE = 16 * D;
  const int quads = cols * (D / 4);
  const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.part + (int64_t)it.first * STRIDE), (short)0, it.parts * STRIDE * 4, kPagedBufFlags);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.stats + (int64_t)it.first * 32), (short)0,
                                                                      it.parts * 128, kPagedBufFlags);
  for (int i = tid; i < quads; i += kThreads) {
    const int hd = i / (D / 4), d = i % (D / 4) * 4;
    Share8 x;
#pragma unroll
    for (int w = 0; w < W; ++w)
      x.add(m_s[w][hd], l_s[w][hd],
            *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(v_s[w]) + hd * OROW + d));
    if (it.parts == 1) {
      *reinterpret_cast<u32x2*>(out_at(hd) + d) = x.template out<DT>();
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x.t), rp,
                                             (uint32_t)(it.part * STRIDE + i * 4) * 4u, 0, kPagedCoherentAux);
      if (d == 0)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{x.M, x.L}), rs,
                                              (uint32_t)(it.part * 16 + hd) * 8u, 0, kPagedCoherentAux);
    }
  }
  if (it.parts == 1) return;

  // The last part of a tile to arrive joins them, in their order.
  __builtin_amdgcn_s_waitcnt(0);  // the stores have reached the level all XCDs share
  __syncthreads();
  unsigned* const cnt = a.cnt + it.counter;
  if (tid == 0) arrived_s = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived_s != (unsigned)(it.parts - 1)) return;
  if (tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int runs = max(1, kThreads / quads), run = min(tid / quads, runs);
  f32x4* const red = reinterpret_cast<f32x4*>(&v_s[0][0]);
  f32x2* const red_ml = reinterpret_cast<f32x2*>(red + kThreads);
  for (int i = tid - run * quads; i < quads; i += kThreads) {
    const int hd = i / (D / 4);
    Share8 x;
    if (run < runs) {
      for (int p0 = run; p0 < it.parts; p0 += runs * kP8AtOnce) {
        f32x4 t[kP8AtOnce];
        f32x2 ml[kP8AtOnce];
#pragma unroll
        for (int k = 0; k < kP8AtOnce; ++k) {
          const int p = min(p0 + k * runs, it.parts - 1);
          t[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rp, (uint32_t)(p * STRIDE + i * 4) * 4u, 0, kPagedCoherentAux));
          ml[k] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, (uint32_t)(p * 16 + hd) * 8u, 0,
                                                                                 kPagedCoherentAux));
        }
#pragma unroll
        for (int k = 0; k < kP8AtOnce; ++k)
          if (p0 + k * runs < it.parts) x.add(ml[k][0], ml[k][1], t[k]);
      }
    }
    if (runs > 1) {  // (then this is the only go, of all threads)
      if (run < runs) red[tid] = x.t, red_ml[tid] = f32x2{x.M, x.L};
      __syncthreads();
      if (run == 0)
        for (int r = 1; r < runs; ++r) x.add(red_ml[r * quads + i][0], red_ml[r * quads + i][1], red[r * quads + i]);
    }
    if (run == 0) *reinterpret_cast<u32x2*>(out_at(hd) + i % (D / 4) * 4) = x.template out<DT>();
  }
}

// ---------------------------------------------------------------- attention of rows with many new tokens
constexpr int kPromptCols = 64, kPromptUnit = 64;

// A workgroup has 64 columns of a row and key-value head, sixteen a wave, and all the slots that they see, 64 at once:
// the four waves turn the codes into fp16 in LDS together, once, and multiply from there.  Otherwise as
// paged8_attention_kernel, whose waves share their columns and not the slots: that spreads a few columns over the chip,
// but converts every code for sixteen columns alone.
//
// What bounds it: 2000 tokens of 32 / 8 x 64 (16.4 GFLOP) take 59 us, 0.28 PFLOP/s (in two parts each, 0.56; a large
// product reaches 1.18): of a busy CU's cycles the vector instructions take 0.7, the LDS 0.4 and the matrix
// instructions 0.3.  (Without LDS conversion, sixteen columns a workgroup: 110 us.  Masks tested slot by slot: 86
// instead of 79 at that time.  Two workgroups a CU instead of four: 95 against 86.  Every second unit in one half of eight
// waves: 64 against 60.  The order of tiles turned round in every second 256: 60.4 against 59.9.)
template <int DT, int CT, int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void paged8_prompt_kernel(Attend8Args a) {
  constexpr int UP = kPromptUnit, KB = UP / 32, NJ = D / 32, ND = D / 16;
  constexpr int KROW = D + 8;               // halfwords of a key row in LDS: sixteen rows on different banks
  constexpr int VROW = D == 64 ? 72 : 144;  // of a value row: four rows of 32 bytes on different banks
  constexpr int CH = D / 16, NC = UP * CH / 256;  // chunks of 16 codes of a slot, and of a thread
  typedef Mfma<W4_DTYPE_FP16> M;
  __shared__ __attribute__((aligned(16))) uint16_t k_s[2][UP * KROW], v_s[2][UP * VROW];
  __shared__ float ks_s[2][UP / 8], vs_s[2][UP / 8];
  __shared__ uint16_t nan_s[2][CT == W4_CODE_E4M3 ? UP * CH : 1];
  __shared__ int odd_s[2];  // the unit there, where it has codes of NaN

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, c = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nh = a.c.nkv * a.g;
  // The row and the tile of its columns, a head's tiles beside another head's; the last ones, which see most, first.
  RowSpan sp;
  int b = 0, tile = 0, h = 0;
  for (int r = 0, base = 0;; r += 64) {
    if (r >= a.c.rows) return;
    const RowSpan s = row_span(a.c, a.lengths, a.offsets, a.tokens, a.longest, r + lane);
    const int tiles = s.n >= a.many ? (int)(((int64_t)s.n * a.g + kPromptCols - 1) / kPromptCols) * a.c.nkv : 0;
    const int upto = base + wave_scan(tiles), item = blockIdx.x;
    const int end = __builtin_amdgcn_readlane(upto, 63);
    if (item < end) {
      const int i = __popcll(__ballot(item >= upto));
      b = r + i;
      sp.len = __builtin_amdgcn_readlane(s.len, i);
      sp.o0 = __builtin_amdgcn_readlane(s.o0, i);
      sp.n = __builtin_amdgcn_readlane(s.n, i);
      const int left = __builtin_amdgcn_readlane(upto, i) - 1 - item;
      tile = left / a.c.nkv;
      h = left - tile * a.c.nkv;
      break;
    }
    base = end;
  }
  const int len = sp.len, col0 = tile * kPromptCols, cols = min(sp.n * a.g - col0, kPromptCols);
  auto out_at = [&](int col) {
    const int j = (col0 + col) / a.g;
    return a.out + ((int64_t)(sp.o0 + j) * nh + h * a.g + (col0 + col - j * a.g)) * D;
  };
  if (len < 0) {
    const uint16_t fill = len == kP8Refused ? float_to_act_bits<DT>(__builtin_nanf("")) : 0;
    for (int i = tid; i < cols * D; i += 256) out_at(i / D)[i % D] = fill;
    return;
  }
  const int first_slot = len + col0 / a.g, last_slot = len + (col0 + cols - 1) / a.g;
  const int lo = a.window ? max(first_slot - a.window + 1, 0) : 0;
  const int u_lo = lo / UP, sink_units = a.window ? min((int)(((int64_t)a.sinks + UP - 1) / UP), u_lo) : 0;
  const int units = sink_units + last_slot / UP - u_lo + 1;
  auto base_of = [&](int u) { return (u < sink_units ? u : u_lo + u - sink_units) * UP; };
  // this wave's columns (past the tile's last: copies of it that count for nothing)
  const int wcol = min(wv * 16, cols - 1);
  const int w_first = len + (col0 + wcol) / a.g, w_last = len + (col0 + min(wv * 16 + 15, cols - 1)) / a.g;

  // A thread's chunks of a unit: chunk tid + 256 i is chunk % CH of slot / CH.
  const int32_t* const table = a.c.table + (int64_t)b * a.c.width;
  u32x4 kr[NC], vr[NC];
  float sr = 0.f;
  int ids[NC], sid = 0;
  auto load_ids = [&](int u) __attribute__((always_inline)) {
    const int base = base_of(u);
#pragma unroll
    for (int i = 0; i < NC; ++i) ids[i] = table[min(base + (tid + 256 * i) / CH, last_slot) >> a.c.log2s];
    sid = table[min(base + 8 * (tid & 7), last_slot) >> a.c.log2s];
  };
  // whether columns of these tokens, from the first to the last, all see a whole unit
  auto all_see = [&](int base, int first, int last) {
    return base + UP - 1 <= first && (!a.window || base > last - a.window || base + UP <= a.sinks);
  };
  auto valid = [&](int id, int slot) {
    return slot <= last_slot && (uint64_t)(int64_t)id < (uint64_t)a.c.pages ? id : -1;
  };
  auto load = [&](int u) __attribute__((always_inline)) {
    const int base = base_of(u);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int slot = base + (tid + 256 * i) / CH;
      const int64_t at = a.c.token(max(valid(ids[i], slot), 0), h, slot) * D + tid % CH * 16;
      kr[i] = *reinterpret_cast<const u32x4*>(a.c.k + at);
      vr[i] = *reinterpret_cast<const u32x4*>(a.c.v + at);
    }
    if (tid < 16) {  // keys' scales of the unit's groups of eight slots, then values'
      const int slot = base + 8 * (tid & 7), id = valid(sid, slot);
      const float x = (tid < 8 ? a.c.k_scale : a.c.v_scale)[a.c.block(max(id, 0), h, slot)];
      sr = id < 0 ? __builtin_nanf("") : x;
    }
  };
  auto stage = [&](int u) __attribute__((always_inline)) {
    const int buf = u & 1;
    bool some = false;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int slot = (tid + 256 * i) / CH, ch = tid % CH;
      const int row = (slot & 32) + ((slot >> 2) & 1) * 16 + ((slot >> 3) & 3) * 4 + (slot & 3);
      if (CT == W4_CODE_E4M3 && !all_see(base_of(u), first_slot, last_slot)) {
        // NaN of e4m3, what a program that is not this one left in the pages, must not meet the probability 0 of a slot
        // that is not seen: it is taken out, and what sees it is made NaN by itself.
        uint32_t bad[4], any = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= bad[e] = nan_bytes(vr[i][e]);
        uint32_t bits = 0;
        if (any) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            vr[i][e] &= ~(bad[e] * 0xFFu);
            bits |= (bad[e] & 1 | bad[e] >> 7 & 2 | bad[e] >> 14 & 4 | bad[e] >> 21 & 8) << (4 * e);
          }
          some = true;
        }
        nan_s[buf][tid + 256 * i] = (uint16_t)bits;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        *reinterpret_cast<f16x8*>(&k_s[buf][row * KROW + ch * 16 + 8 * g]) = codes8h<CT>(kr[i][2 * g], kr[i][2 * g + 1]);
        *reinterpret_cast<f16x8*>(&v_s[buf][slot * VROW + ch * 16 + 8 * g]) = codes8h<CT>(vr[i][2 * g], vr[i][2 * g + 1]);
      }
    }
    if (tid < 8) ks_s[buf][tid] = sr;
    else if (tid < 16) vs_s[buf][tid - 8] = sr;
    if (CT == W4_CODE_E4M3 && some) odd_s[buf] = u;
  };

  if (tid < 2) odd_s[tid] = -1;
  load_ids(0);
  load(0);
  load_ids(min(1, units - 1));

  const int col = min(wv * 16 + l16, cols - 1), tok = sp.o0 + (col0 + col) / a.g, mine = len + (col0 + col) / a.g;
  f16x8 qf[NJ][2];
  float q_short;
  {
    float xs[NJ][8];
    const int pos = a.positions[tok];
    const bool there = (uint64_t)(int64_t)pos < (uint64_t)a.angles;
    const uint16_t* const qp = a.q + tok * a.stride_q + (h * a.g + (col0 + col) % a.g) * D;
    const float* const cosr = a.cos + (there ? (int64_t)pos * (D / 2) : 0);
    const float* const sinr = a.sin + (there ? (int64_t)pos * (D / 2) : 0);
    const float scale = there ? a.scale : __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < NJ / 2; ++j) {
      const int d = 32 * j + 8 * c;
      float *const x = xs[j], *const y = xs[j + NJ / 2];
      unpack8<DT>(*reinterpret_cast<const u32x4*>(qp + d), x);
      unpack8<DT>(*reinterpret_cast<const u32x4*>(qp + d + D / 2), y);
      const f32x4* const cp = reinterpret_cast<const f32x4*>(cosr + d);
      const f32x4* const sp4 = reinterpret_cast<const f32x4*>(sinr + d);
      const f32x4 cs[2] = {cp[0], cp[1]}, sn[2] = {sp4[0], sp4[1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float r1, r2;
        rope_pair(x[e], y[e], cs[e >> 2][e & 3], sn[e >> 2][e & 3], &r1, &r2);
        x[e] = r1 * scale, y[e] = r2 * scale;
      }
    }
    q_short = query_parts<NJ>(xs, qf);
  }
  __syncthreads();
  stage(0);
  __syncthreads();

  float m = -__builtin_inff(), l = 0.f, heavy = 0.f, lift = 1.f;  // as there
  f32x4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int u = 0; u < units; ++u) {
    const int base = base_of(u), buf = u & 1;
    if (u + 1 < units) {  // the next unit's loads travel under this one's products
      load(u + 1);
      load_ids(min(u + 2, units - 1));
    }
    // (a wave none of whose columns sees any of it waits)
    if (base <= w_last && (!a.window || base + UP - 1 > w_first - a.window || base < a.sinks)) {
      const bool whole = all_see(base, w_first, w_last);
      f32x4 s[KB][2];
      float sv[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const float sk = ks_s[buf][4 * kb + c] * q_short;
        sv[kb] = vs_s[buf][4 * kb + c];
        f16x8 kf[2][NJ];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            kf[t][j] = *reinterpret_cast<const f16x8*>(&k_s[buf][(kb * 32 + t * 16 + l16) * KROW + 8 * c + 32 * j]);
          s[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int p = 1; p >= 0; --p)  // the small parts first
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[kb][t] = M::m16(kf[t][j], qf[j][p], s[kb][t]);
#pragma unroll
        for (int t = 0; t < 2; ++t) s[kb][t] *= sk;
      }
      if (!whole) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint32_t sight = seen8(base + kb * 32 + 8 * c, mine, a.window, a.sinks);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s[kb][e >> 2][e & 3] = sight >> e & 1 ? s[kb][e >> 2][e & 3] : -__builtin_inff();
          // (a scale that is NaN is no matter of a token that sees none of its slots)
          sv[kb] = sight ? sv[kb] : 0.f;
        }
      }
      float top = -__builtin_inff(), top_kb[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        top_kb[kb] = s[kb][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top_kb[kb] = fmaxf(top_kb[kb], s[kb][e >> 2][e & 3]);
        top = fmaxf(top, top_kb[kb]);
      }
      float al = 1.f;
      if (__ballot(top - m > 6.f)) {
        float mn = fmaxf(top, __shfl_xor(top, 16));
        mn = fmaxf(mn, __shfl_xor(mn, 32));
        mn = mn - m > 6.f ? mn + 2.f : m;
        al = __builtin_amdgcn_exp2f(m - finite_or_zero(mn));
        l *= al;
        heavy *= al;
        m = mn;
      }
      const float mz = finite_or_zero(m);
      auto prob = [&](float x) { return __builtin_amdgcn_exp2f(x - mz); };
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) heavy = fmaxf(heavy, prob(top_kb[kb]) * sv[kb]);
      if (__ballot(al < 1.f || heavy * lift > 0x1p15f)) {
        heavy = fmaxf(heavy, __shfl_xor(heavy, 16));
        heavy = fmaxf(heavy, __shfl_xor(heavy, 32));
        const float to = al < 1.f || heavy * lift > 0x1p15f ? raise_to(heavy, 12) : lift;
        const float by = al * fminf(to * inverse_power(lift), 0x1p127f);
        lift = to;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] *= by;
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = prob(s[kb][e >> 2][e & 3]);
          l += p[e];
          p[e] = p[e] * sv[kb] * lift;
        }
        f16x8 pf[2];
        halves8(p, pf);
        f16x8 vf[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const uint16_t* at = &v_s[buf][(kb * 32 + 8 * c + (l16 >> 2)) * VROW + d * 16 + 4 * (l16 & 3)];
          const s16x4 vl = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
          const s16x4 vh = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * VROW));
          const u32x2 lw = __builtin_bit_cast(u32x2, vl), hw = __builtin_bit_cast(u32x2, vh);
          vf[d] = __builtin_bit_cast(f16x8, u32x4{lw[0], lw[1], hw[0], hw[1]});
        }
#pragma unroll
        for (int q = 1; q >= 0; --q)
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] = M::m16(vf[d], pf[q], o[d]);
      }
      if (CT == W4_CODE_E4M3 && odd_s[buf] == u) {
        for (int row = 0; row < UP; ++row) {
          const bool see = seen8(base + row, mine, a.window, a.sinks) & 1;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const uint32_t bits = nan_s[buf][row * CH + d] >> (4 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (see && bits >> e & 1) o[d][e] = __builtin_nanf("");
          }
        }
      }
    }
    if (u + 1 < units) {
      stage(u + 1);  // (what was there was read before the last barrier)
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (wv * 16 + l16 < cols) {
    const float inv = 1.f / l, down = inverse_power(lift);
    uint16_t* const out = out_at(wv * 16 + l16) + 4 * c;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      u32x2 w;
      w[0] = (uint32_t)float_to_act_bits<DT>(o[d][0] * inv * down) | ((uint32_t)float_to_act_bits<DT>(o[d][1] * inv * down) << 16);
      w[1] = (uint32_t)float_to_act_bits<DT>(o[d][2] * inv * down) | ((uint32_t)float_to_act_bits<DT>(o[d][3] * inv * down) << 16);
      *reinterpret_cast<u32x2*>(out + 16 * d) = w;
    }
  }
}

}  // namespace w4

// ---------------------------------------------------------------- host side
using namespace w4host;

namespace {

int check_cache8(const w4_paged8_cache* c, const char* what) {
  if (!c) return fail(W4_ERR_INVALID, "%s: null cache", what);
  if (c->code != W4_CODE_INT8 && c->code != W4_CODE_E4M3)
    return fail(W4_ERR_INVALID, "%s: codes must be int8 or e4m3 (got code %d)", what, c->code);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(W4_ERR_UNSUPPORTED, "%s: heads of %lld (64 or 128)", what, (long long)c->head_dim);
  if (!is_pow2(c->page_size) || c->page_size < 8 || c->page_size > 1024)
    return fail(W4_ERR_UNSUPPORTED, "%s: pages of %lld tokens (a power of two from 8 to 1024)", what,
                (long long)c->page_size);
  if (!is_pow2(c->block) || c->block < 8 || c->block > 64 || c->block > c->page_size)
    return fail(W4_ERR_UNSUPPORTED, "%s: blocks of %lld tokens (a power of two from 8 to 64, at most a page)", what,
                (long long)c->block);
  if (c->pages < 1 || c->pages >= (1ll << 31) || c->kv_heads < 1 || c->kv_heads > 65535 || c->rows < 0 ||
      c->rows > 65535 || c->width < 1 || c->width > (1ll << 30) || c->width * c->page_size >= (1ll << 30))
    return fail(W4_ERR_INVALID, "%s: %lld pages, %lld heads, a table of %lld x %lld pages of %lld", what,
                (long long)c->pages, (long long)c->kv_heads, (long long)c->rows, (long long)c->width,
                (long long)c->page_size);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || (c->rows && !c->table))
    return fail(W4_ERR_INVALID, "%s: null pointer", what);
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4)
    return fail(W4_ERR_INVALID, "%s: pages must be 16-byte aligned, scales 4-byte", what);
  return W4_OK;
}

w4::Paged8View view_of(const w4_paged8_cache* c) {
  w4::Paged8View v{};
  v.k = static_cast<uint8_t*>(c->k);
  v.v = static_cast<uint8_t*>(c->v);
  v.k_scale = c->k_scale;
  v.v_scale = c->v_scale;
  v.table = c->table;
  v.pages = c->pages;
  v.nkv = (int)c->kv_heads;
  v.log2s = ilog2(c->page_size);
  v.log2b = ilog2(c->block);
  v.rows = (int)c->rows;
  v.width = (int)c->width;
  return v;
}

bool rows_ok(const void* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 8 == 0; }

constexpr int64_t kMostTokens = 1 << 24;

// `f(std::integral_constant)` of a runtime choice.
template <typename F> int by_code(int code, const F& f) {
  return code == W4_CODE_INT8 ? f(std::integral_constant<int, W4_CODE_INT8>{})
                              : f(std::integral_constant<int, W4_CODE_E4M3>{});
}
template <typename F> int by_head(int64_t d, const F& f) {
  return d == 64 ? f(std::integral_constant<int, 64>{}) : f(std::integral_constant<int, 128>{});
}
template <typename F> int by_dtype(int dtype, const F& f) {
  return dtype == W4_DTYPE_BF16 ? f(std::integral_constant<int, W4_DTYPE_BF16>{})
                                : f(std::integral_constant<int, W4_DTYPE_FP16>{});
}

int check_new(const w4_paged8_cache* c, int dtype, const void* k, const void* v, int64_t stride_k, int64_t stride_v,
              int64_t tokens, const int32_t* lengths, const int32_t* offsets, const int32_t* positions,
              const float* cos, const float* sin, int64_t angles, const char* what) {
  if (const int rc = check_cache8(c, what)) return rc;
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16)
    return fail(W4_ERR_INVALID, "%s: dtype must be bf16 or fp16 (got code %d)", what, dtype);
  if (tokens < 0 || angles < 1)
    return fail(W4_ERR_INVALID, "%s: %lld tokens, %lld angles", what, (long long)tokens, (long long)angles);
  if (tokens > kMostTokens) return fail(W4_ERR_UNSUPPORTED, "%s: %lld tokens in a call", what, (long long)tokens);
  if (tokens == 0) return W4_OK;
  if (!k || !v || !positions || !cos || !sin || (c->rows && (!lengths || !offsets)))
    return fail(W4_ERR_INVALID, "%s: null pointer", what);
  if (!rows_ok(k, stride_k) || !rows_ok(v, stride_v) || ((uintptr_t)cos | (uintptr_t)sin) % 16)
    return fail(W4_ERR_INVALID, "%s: operands must be 16-byte aligned, row strides multiples of 8", what);
  return W4_OK;
}

int launch_append8(w4::Append8Args a, int dtype, int code, int64_t head_dim, hipStream_t st, const char* what) {
  // blocks that get tokens: at most as many as tokens, and two a row more than whole ones
  const int64_t block = 1ll << a.c.log2b;
  const int64_t items = std::min<int64_t>(a.tokens, a.tokens / block + 2 * (int64_t)a.c.rows);
  if (items == 0) return W4_OK;
  const int64_t per = block * (head_dim / 16), units = std::max<int64_t>(w4::kP8Threads / per, 1);
  const int64_t groups = items * ((a.c.nkv + units - 1) / units);
  if (groups > 0xFFFFFFFFll / w4::kP8Threads)  // HIP refuses launches of 2^32 threads and more
    return fail(W4_ERR_UNSUPPORTED, "%s: %d tokens of %d heads", what, a.tokens, a.c.nkv);
  a.heads = (int)units;
  const dim3 grid((unsigned)groups);
  return by_dtype(dtype, [&](auto dt) {
    return by_code(code, [&](auto ct) {
      return by_head(head_dim, [&](auto d) {
        if (per <= w4::kP8Threads) w4::paged8_append_kernel<dt(), ct(), d(), 1><<<grid, w4::kP8Threads, 0, st>>>(a);
        else if constexpr (d() == 128) w4::paged8_append_kernel<dt(), ct(), d(), 2><<<grid, w4::kP8Threads, 0, st>>>(a);
        return check_launch(what);
      });
    });
  });
}

struct Attend8Plan {
  int64_t items;
  size_t stats, part, bytes;
};

// `tokens` new tokens of `rows` rows are at most this many tiles of sixteen columns; of those that are cut see
// find_item8.
Attend8Plan attend8_plan(int64_t rows, int64_t tokens, int64_t num_heads, int64_t kv_heads, int64_t head_dim) {
  const int64_t g = num_heads / kv_heads;
  const int64_t split = 2 * w4::p8_parts((int)head_dim);
  Attend8Plan p;
  p.items = kv_heads * ((tokens * g + 15 * std::min(rows, tokens)) / 16) + split + 1;
  p.stats = W4_WORKSPACE_COUNTER_BYTES;
  p.part = p.stats + split * 16 * 8;
  p.bytes = p.part + (size_t)split * 16 * head_dim * 4;
  return p;
}

}  // namespace

extern "C" int w4_paged8_append(const w4_paged8_cache* cache, int dtype, const void* k, const void* v, int64_t stride_k,
                                int64_t stride_v, int64_t tokens, const int32_t* lengths, const int32_t* offsets,
                                const int32_t* positions, const float* cos, const float* sin, int64_t angles,
                                void* stream) {
  clear_error();
  if (const int rc = check_new(cache, dtype, k, v, stride_k, stride_v, tokens, lengths, offsets, positions, cos, sin,
                               angles, "w4_paged8_append"))
    return rc;
  if (tokens == 0 || cache->rows == 0) return W4_OK;
  const w4::Append8Args a{view_of(cache), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), stride_k,
                          stride_v, angles, lengths, offsets, positions, cos, sin, (int)tokens, (int)tokens, 0};
  return launch_append8(a, dtype, cache->code, cache->head_dim, static_cast<hipStream_t>(stream), "w4_paged8_append");
}

extern "C" int w4_paged8_read(const w4_paged8_cache* cache, int dtype, const int32_t* starts, const int32_t* offsets,
                              int64_t tokens, void* k, void* v, void* stream) {
  clear_error();
  if (const int rc = check_cache8(cache, "w4_paged8_read")) return rc;
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16 && dtype != W4_DTYPE_FP32)
    return fail(W4_ERR_INVALID, "w4_paged8_read: dtype must be bf16, fp16 or fp32 (got code %d)", dtype);
  if (tokens < 0) return fail(W4_ERR_INVALID, "w4_paged8_read: %lld tokens", (long long)tokens);
  const int64_t per = cache->kv_heads * (cache->head_dim / 16);
  if (tokens > kMostTokens || tokens * per >= (1ll << 32) - w4::kP8Threads)  // HIP refuses launches of 2^32 threads
    return fail(W4_ERR_UNSUPPORTED, "w4_paged8_read: %lld tokens in a call", (long long)tokens);
  if (tokens == 0) return W4_OK;
  if (!k || !v || (cache->rows && (!starts || !offsets))) return fail(W4_ERR_INVALID, "w4_paged8_read: null pointer");
  if (((uintptr_t)k | (uintptr_t)v) % 16)
    return fail(W4_ERR_INVALID, "w4_paged8_read: outputs must be 16-byte aligned");
  const w4::Read8Args a{view_of(cache), starts, offsets, k, v, (int)tokens};
  const dim3 grid((unsigned)((tokens * per + w4::kP8Threads - 1) / w4::kP8Threads));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_code(cache->code, [&](auto ct) {
    return by_head(cache->head_dim, [&](auto d) {
      if (dtype == W4_DTYPE_FP32) w4::paged8_read_kernel<ct(), W4_DTYPE_FP32, d()><<<grid, w4::kP8Threads, 0, st>>>(a);
      else if (dtype == W4_DTYPE_FP16) w4::paged8_read_kernel<ct(), W4_DTYPE_FP16, d()><<<grid, w4::kP8Threads, 0, st>>>(a);
      else w4::paged8_read_kernel<ct(), W4_DTYPE_BF16, d()><<<grid, w4::kP8Threads, 0, st>>>(a);
      return check_launch("w4_paged8_read");
    });
  });
}

extern "C" size_t w4_paged8_attention_workspace_bytes(int64_t rows, int64_t tokens, int64_t num_heads, int64_t kv_heads,
                                                      int64_t head_dim) {
  if (rows < 0 || tokens < 1 || tokens > kMostTokens || num_heads < 1 || kv_heads < 1 || num_heads % kv_heads) return 0;
  return attend8_plan(rows, tokens, num_heads, kv_heads, head_dim).bytes;
}

extern "C" int w4_paged8_attention(const w4_paged8_cache* cache, int dtype, const void* q, const void* k, const void* v,
                                   int64_t stride_q, int64_t stride_k, int64_t stride_v, int64_t num_heads,
                                   int64_t tokens, int64_t longest, int64_t window, int64_t sinks,
                                   const int32_t* lengths, const int32_t* offsets, const int32_t* positions,
                                   const float* cos, const float* sin, int64_t angles, void* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = check_new(cache, dtype, k, v, stride_k, stride_v, tokens, lengths, offsets, positions, cos, sin,
                               angles, "w4_paged8_attention"))
    return rc;
  if (num_heads < 1 || num_heads % cache->kv_heads || num_heads / cache->kv_heads > 256)
    return fail(W4_ERR_INVALID, "w4_paged8_attention: %lld query heads on %lld key-value heads", (long long)num_heads,
                (long long)cache->kv_heads);
  if (window < 0 || sinks < 0 || longest < 0)
    return fail(W4_ERR_INVALID, "w4_paged8_attention: a window of %lld, %lld first tokens, at most %lld new ones a row",
                (long long)window, (long long)sinks, (long long)longest);
  if (tokens == 0) return W4_OK;
  if (tokens * num_heads >= (1ll << 27))
    return fail(W4_ERR_UNSUPPORTED, "w4_paged8_attention: %lld tokens of %lld heads", (long long)tokens,
                (long long)num_heads);
  if (!q || !out) return fail(W4_ERR_INVALID, "w4_paged8_attention: null pointer");
  if (!rows_ok(q, stride_q) || (uintptr_t)out % 16)
    return fail(W4_ERR_INVALID, "w4_paged8_attention: operands must be 16-byte aligned, row strides multiples of 8");
  const Attend8Plan p = attend8_plan(cache->rows, tokens, num_heads, cache->kv_heads, cache->head_dim);
  if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 256)
    return fail(W4_ERR_WORKSPACE, "w4_paged8_attention: needs a 256-byte aligned workspace of %zu bytes (got %zu)",
                p.bytes, workspace_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const w4::Paged8View view = view_of(cache);
  const int most_new = (int)(longest && longest < tokens ? longest : tokens);
  const bool put = most_new == 1 && num_heads / cache->kv_heads <= 16 && cache->block <= w4::kP8Unit;
  // Calls of so many columns fill the chip with tiles of 64 of them and all their slots.  Times of both ways, us, tiles of
  // 64 first, of one row of new tokens on an empty cache / after 2000 slots / after 8000:
  //   columns  32 / 8 x 64                32 / 8 x 128               24 / 1 x 64                20 / 2 x 128
  //   19200    31 25 / 77 63 / 231 169    36 32 / 103 85 / 321 243   33 26 / 75 60 / 224 158    45 39 / 109 91 / 327 252
  //   36864    43 40 / 99 97 / 285 269    55 60 / 173 156 / 533 487  51 48 / 99 103 / 288 279   76 83 / 199 190 / 557 536
  //   64000    65 83 / 145 178 / 386 482  106 135 / 249 321 / 676 932  80 100 / 155 196 / 399 492
  //   and of 20 / 2 x 128 146 193 / 295 391 / 712 993.
  // Four rows of 150 tokens of 64 heads after 100000 slots: 3191 and 3795 (heads of 64), 7270 and 8221 (of 128).  Rows of
  // fewer than 150 tokens of 64 heads are cut among them all the same.  One long row whose tokens are few and that passes
  // by the others' columns is slower for it: 150 tokens of 64 heads after 100000 slots beside 460 single ones 2242 and
  // 1137, after 2000 131 and 106; the lengths are on the GPU, so the rule cannot know.
  constexpr int64_t kAllColumns = 36864, kManyColumns = 9600;
  const int64_t many = (kManyColumns + num_heads - 1) / num_heads;
  // (Not where the attention writes: a single token of 9600 heads and more is a prompt by its columns, and nobody's to write.)
  const bool prompts = !put && tokens * num_heads >= kAllColumns && most_new >= many;
  const int64_t wide = tokens / many;  // such rows, at most
  // (and the others' tokens)
  const int64_t rest = prompts ? std::min(tokens, cache->rows * (many - 1)) : tokens;
  const int64_t items = attend8_plan(cache->rows, rest, num_heads, cache->kv_heads, cache->head_dim).items;
  const int64_t prompt_items =
      cache->kv_heads * ((tokens * (num_heads / cache->kv_heads) + (w4::kPromptCols - 1) * wide) / w4::kPromptCols);
  if (std::max(items, prompts ? prompt_items : 0) > 0xFFFFFFFFll / 256)  // HIP refuses launches of 2^32 threads and more
    return fail(W4_ERR_UNSUPPORTED, "w4_paged8_attention: %lld tokens of %lld heads", (long long)tokens,
                (long long)num_heads);
  static_assert(64 * w4::kP8Waves == 256, "threads of a workgroup");
  if (!put) {
    const w4::Append8Args p{view, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), stride_k, stride_v,
                            angles, lengths, offsets, positions, cos, sin, (int)tokens, most_new, 0};
    if (const int rc = launch_append8(p, dtype, cache->code, cache->head_dim, st, "w4_paged8_attention (append)"))
      return rc;
  }
  const int64_t most = 1 << 30;  // (of slots, which are fewer)
  char* const ws = static_cast<char*>(workspace);
  w4::Attend8Args a{};
  a.c = view;
  a.q = static_cast<const uint16_t*>(q);
  a.stride_q = stride_q;
  a.angles = angles;
  a.lengths = lengths;
  a.offsets = offsets;
  a.positions = positions;
  a.cos = cos;
  a.sin = sin;
  a.out = static_cast<uint16_t*>(out);
  a.stats = reinterpret_cast<float*>(ws + p.stats);
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.cnt = reinterpret_cast<unsigned*>(ws);
  a.scale = 1.f / sqrtf((float)cache->head_dim);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.stride_k = stride_k;
  a.stride_v = stride_v;
  a.tokens = (int)tokens;
  a.longest = most_new;
  a.g = (int)(num_heads / cache->kv_heads);
  a.window = window >= most ? 0 : (int)window;
  a.sinks = (int)std::min(sinks, most);
  a.many = prompts ? (int)many : INT32_MAX;
  const dim3 grid((unsigned)items), prompt((unsigned)prompt_items);
  return by_dtype(dtype, [&](auto dt) {
    return by_code(cache->code, [&](auto ct) {
      return by_head(cache->head_dim, [&](auto d) {
        if (prompts) {
          w4::paged8_prompt_kernel<dt(), ct(), d()><<<prompt, 256, 0, st>>>(a);
          if (const int rc = check_launch("w4_paged8_attention (prompts)")) return rc;
        }
        if (put) w4::paged8_attention_kernel<dt(), ct(), d(), w4::kP8Waves, true><<<grid, 64 * w4::kP8Waves, 0, st>>>(a);
        else w4::paged8_attention_kernel<dt(), ct(), d(), w4::kP8Waves, false><<<grid, 64 * w4::kP8Waves, 0, st>>>(a);
        return check_launch("w4_paged8_attention");
      });
    });
  });
}
