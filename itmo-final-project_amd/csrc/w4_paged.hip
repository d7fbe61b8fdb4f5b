// Key-value cache in pages for batches of sequences (int4_hip/paged.py): tokens
// written into the pages, the attention of one new token of every sequence over
// them, and eviction by accumulated attention weight.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "w4_common.hpp"

namespace w4 {

constexpr int kPagedThreads = 256;
constexpr int kPagedBufFlags = 0x00020000;  // raw buffer: the range is checked in bytes
constexpr int kPagedCoherentAux = 16;       // sc1: the cache policy of agent-scope atomic loads and stores

struct PagedView {
  uint16_t* k;     // [pages, nkv, S, D]
  uint16_t* v;
  float* weight;   // [pages, nkv, S] or null
  const int32_t* table;  // [rows, width]
  int64_t pages;
  int nkv, log2s, rows, width;

  __device__ __forceinline__ int capacity() const { return width << log2s; }
  // Index of a slot's token among all tokens of the pool, for one head; -1 outside the pool.
  __device__ __forceinline__ int64_t token(int row, int slot, int head) const {
    const int64_t page = table[(int64_t)row * width + (slot >> log2s)];
    if ((uint64_t)page >= (uint64_t)pages) return -1;
    return (((page * nkv + head) << log2s) + (slot & ((1 << log2s) - 1)));
  }
};

// ---------------------------------------------------------------- append
struct AppendArgs {
  PagedView c;
  const uint16_t* k;  // [T, nkv * D], row strides below
  const uint16_t* v;
  int64_t stride_k, stride_v, tokens, angles;
  const int32_t *rows, *slots, *positions;
  const float *cos, *sin;  // [angles, D / 2]
};

// Eight rotary pairs of key and the sixteen values beside them a thread: 16-byte loads and stores throughout, and the
// rotation needs no other thread.  Bound by memory: 7999 tokens of 8 heads of 128 in 12.7 us, 70.0 MB at 5.5 TB/s (a
// large copy: 5.1); 300 of 64 in 3.1 us, a launch's least.
template <int DT, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(AppendArgs a) {
  constexpr int CH = D / 16;  // threads per head
  const int64_t i = (int64_t)blockIdx.x * kPagedThreads + threadIdx.x;
  const int64_t t = i / (a.c.nkv * CH);
  if (t >= a.tokens) return;
  const int r = (int)(i - t * (a.c.nkv * CH)), h = r / CH, d = (r % CH) * 8;
  const int row = a.rows[t], slot = a.slots[t], pos = a.positions[t];
  if ((unsigned)row >= (unsigned)a.c.rows || (unsigned)slot >= (unsigned)a.c.capacity() ||
      (uint64_t)(int64_t)pos >= (uint64_t)a.angles)
    return;
  const int64_t at = a.c.token(row, slot, h);
  if (at < 0) return;
  const uint16_t* kp = a.k + t * a.stride_k + h * D + d;
  const uint16_t* vp = a.v + t * a.stride_v + h * D + d;
  float x1[8], x2[8];
  unpack8<DT>(*reinterpret_cast<const u32x4*>(kp), x1);
  unpack8<DT>(*reinterpret_cast<const u32x4*>(kp + D / 2), x2);
  const u32x4 v1 = *reinterpret_cast<const u32x4*>(vp), v2 = *reinterpret_cast<const u32x4*>(vp + D / 2);
  const float *cp = a.cos + (int64_t)pos * (D / 2) + d, *sp = a.sin + (int64_t)pos * (D / 2) + d;
#pragma unroll
  for (int j = 0; j < 8; ++j) rope_pair(x1[j], x2[j], cp[j], sp[j], &x1[j], &x2[j]);
  uint16_t* ko = a.c.k + at * D + d;
  uint16_t* vo = a.c.v + at * D + d;
  *reinterpret_cast<u32x4*>(ko) = pack8<DT>(x1);
  *reinterpret_cast<u32x4*>(ko + D / 2) = pack8<DT>(x2);
  *reinterpret_cast<u32x4*>(vo) = v1;
  *reinterpret_cast<u32x4*>(vo + D / 2) = v2;
  if (a.c.weight && d == 0) a.c.weight[at] = 0.f;
}

// ---------------------------------------------------------------- attention
struct PagedAttnArgs {
  PagedView c;
  const uint16_t *q, *k, *v;
  int64_t stride_q, stride_k, stride_v, angles;
  const int32_t *lengths, *positions;
  const float *cos, *sin;
  uint16_t* out;  // [rows, nkv * g * D]
  float* scores;  // [rows, nkv * g, width * page_size], of q K / sqrt(D); null without weights
  float* part;    // [items, min(g, tile), D]: outputs of a part, where a row's slots are cut
  float* stats;   // [items, tile, 2]: its heads' references and sums relative to them
  int* first;     // [rows, nkv * htiles, 2]: index of a row and tile's first part, and how many there are
  unsigned* cnt;  // one arrival counter per row and tile of heads
  float scale;    // 1 / sqrt(D)
  int g, tile, htiles;  // query heads a key-value head, of them in a tile, tiles
  int later;      // the parts are joined by a launch of its own
  int at_once;    // parts that the joining reads together
};

// The work of one workgroup: a part of the slots of one row and one tile of its heads.
struct AttnItem {
  int b, tile, part, parts, first;  // first: the index of part 0
  int len, pos;                     // of the row
};

// Workgroups of four waves, the tokens of a batch cut into about 256 parts; of one wave and 1024 parts where there are
// many rows of a bounded length (see paged_attn_plan).  Parts have four units of slots at least.
constexpr int kAttnWaves = 4, kAttnItems = 256, kAttnOneWaveItems = 1024;
constexpr int kAttnMinUnits = 4;
constexpr int kPagedCounters = W4_WORKSPACE_COUNTER_BYTES / 4;

// Which item this is, the same in every wave and launch.  The lengths lie on the GPU, so the split is made here:
// every row is cut into equal parts of at most `per` units of UP slots, per = all units / ITEMS, so that short
// rows stay whole and long ones spread over the chip, whatever else is in the batch.  Rows that need no
// attention (idle, refused) are one part.  `at_once`: the parts that the joining reads together; a row has more only if
// its parts would be longer than twice the least (4000 slots of 32 / 8 heads of 128: 16 parts 13.1 us, 32 14.6).
template <int UP, int ITEMS>
__device__ __forceinline__ bool find_item(const PagedView& c, const int32_t* __restrict__ lengths,
                                          const int32_t* __restrict__ positions, int tiles, int at_once, int item,
                                          AttnItem* it) {
  const int lane = threadIdx.x & 63;
  auto length = [&](int r) { return r + lane < c.rows ? lengths[r + lane] : -1; };
  auto position = [&](int r) { return r + lane < c.rows ? positions[r + lane] : 0; };
  auto units = [&](int r, int len) {
    return r + lane >= c.rows ? 0 : len >= 0 && len < c.capacity() ? len / UP + 1 : 1;
  };
  // the first 128 rows' stay in registers
  const int len0 = length(0), pos0 = position(0), len1 = length(64), pos1 = position(64);
  const float nu0 = (float)units(0, len0), nu1 = (float)units(64, len1);
  float all = nu0 + nu1;
  for (int r = 128; r < c.rows; r += 64) all += (float)units(r, length(r));
  all = wave_sum(all);
  int per = (int)fminf(ceilf(all * ((float)tiles / ITEMS)), 1e9f);
  per = max(per, kAttnMinUnits);
  if ((int64_t)c.rows * tiles > kPagedCounters) per = 1 << 30;  // no counters for parts to meet at
  int base = 0;
  // The rows r.. whose parts are of the size class asked for: whether the item is among them.
  auto among = [&](int r, int len, int pos, int size, float quarter) __attribute__((always_inline)) {
    const int nu = units(r, len);
    const int of = max(per, min((nu + at_once - 1) / at_once, 2 * kAttnMinUnits));
    int parts = (nu + of - 1) / of;
    if (quarter > 0.f && min((int)((float)nu / (float)max(parts, 1) * quarter), 3) != size) parts = 0;
    const int upto = base + wave_scan(parts * tiles);
    const int end = __builtin_amdgcn_readlane(upto, 63);
    if (item >= end) {
      base = end;
      return false;
    }
    const int i = __popcll(__ballot(item >= upto));
    it->parts = __builtin_amdgcn_readlane(parts, i);
    const int rem = item - (__builtin_amdgcn_readlane(upto, i) - it->parts * tiles);
    it->b = r + i;
    it->tile = rem / it->parts;
    it->part = rem - it->tile * it->parts;
    it->first = item - it->part;
    it->len = __builtin_amdgcn_readlane(len, i);
    it->pos = __builtin_amdgcn_readlane(pos, i);
    return true;
  };
  // Where the chip is full, the rows with the longest parts first, by quarters of the longest: the short ones fill the
  // gaps at the end (32 rows of up to 4000 slots 31.1 us instead of 32.6, 20 of up to 9000 40.4 instead of 43.1).
  const bool ordered = c.rows >= 8 && c.rows <= 128 && per > kAttnMinUnits;
  const float quarter = ordered ? 4.f / fminf(wave_max(fmaxf(nu0, nu1)), (float)per) : 0.f;
  for (int size = ordered ? 3 : 0; size >= 0; --size) {
    if (among(0, len0, pos0, size, quarter)) return true;
    if (c.rows > 64 && among(64, len1, pos1, size, quarter)) return true;
  }
  for (int r = 128; r < c.rows; r += 64)
    if (among(r, length(r), position(r), 0, 0.f)) return true;
  return false;
}

// How an fp32 operand enters 16-bit matrix instructions: as the sum of its roundings.
template <int DT> struct Split;
template <> struct Split<W4_DTYPE_BF16> { static constexpr int N = 3; };  // 8 significant bits each: all 24
template <> struct Split<W4_DTYPE_FP16> { static constexpr int N = 2; };  // 11 each: 22

// The range of the probabilities: a head's reference is a score, whose own probability is `first` = 2^above, and is
// raised to the largest one only once that passes it by 2^lag.  bf16 has fp32's exponents.  fp16 ends at 65504, so the
// largest probability is kept between 2^13 and 2^15: both parts of one 2^25 times smaller are then still numbers, and
// what is lost of any is 2^-38 of the largest.  (With the largest at 1, the tail of a row that one token dominates by
// e^17 would be lost, while its sum counts it.)
template <int DT> struct Probs;
template <> struct Probs<W4_DTYPE_BF16> { static constexpr float above = 0.f, first = 1.f, lag = 8.f; };
template <> struct Probs<W4_DTYPE_FP16> { static constexpr float above = 13.f, first = 8192.f, lag = 2.f; };

// What a head's query is multiplied by before it is split, a power of two.  Its scores carry it until they become
// exponents (or are stored).  bf16: nothing.  fp16: its largest element gets to 2^13 or more, so that the parts of one
// 2^38 times smaller are still numbers, whatever the scale of queries and keys.
template <int DT> struct QueryScale {
  __device__ __forceinline__ float set(float) { return 1.f; }
  __device__ __forceinline__ float back() const { return 1.f; }
};
template <> struct QueryScale<W4_DTYPE_FP16> {
  float b = 1.f;
  // The factor, from the largest magnitude of this lane's elements of the head (its four lanes take part).
  __device__ __forceinline__ float set(float largest) {
    largest = fmaxf(largest, __shfl_xor(largest, 16));
    largest = fmaxf(largest, __shfl_xor(largest, 32));
    // the exponent field; 2^13 / 2^e and back are numbers for any that fp16 elements and their rotations have
    const uint32_t e = max(__builtin_bit_cast(uint32_t, largest) >> 23, 64u);
    if (largest == 0.f || e == 255u) return 1.f;  // nothing to scale, or an infinity
    b = __builtin_bit_cast(float, (e - 13u) << 23);
    return __builtin_bit_cast(float, (267u - e) << 23);
  }
  __device__ __forceinline__ float back() const { return b; }
};

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

// Eight elements with zeros in the place of infinities and NaN.
template <int DT>
__device__ __forceinline__ typename Act<DT>::frag finite_part(const typename Act<DT>::frag& f) {
  constexpr uint32_t TOP = DT == W4_DTYPE_BF16 ? 0x7F80u : 0x7C00u;  // all ones: not finite
  u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((w[e] & TOP) == TOP) w[e] &= 0xFFFF0000u;
    if ((w[e] & (TOP << 16)) == (TOP << 16)) w[e] &= 0xFFFFu;
  }
  return __builtin_bit_cast(typename Act<DT>::frag, w);
}

// Lane group c holds D / 32 chunks of eight elements of a head's D (chunk j: elements 32 j + 8 c..).  Chunk j < D / 64
// and its partner D / 2 further on, rotated and multiplied by `scale`.
template <int DT, int D>
__device__ __forceinline__ void rope_chunk(const uint16_t* __restrict__ x, const float* __restrict__ cos,
                                           const float* __restrict__ sin, int j, int c, float scale, float lo[8],
                                           float hi[8]) {
  const int d = 32 * j + 8 * c;
  unpack8<DT>(*reinterpret_cast<const u32x4*>(x + d), lo);
  unpack8<DT>(*reinterpret_cast<const u32x4*>(x + d + D / 2), hi);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r1, r2;
    rope_pair(lo[e], hi[e], cos[d + e], sin[d + e], &r1, &r2);
    lo[e] = r1 * scale;
    hi[e] = r2 * scale;
  }
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -__builtin_inff() ? 0.f : m; }

// Softmax sums and a quad of outputs, relative to the score M.  (Scores are subtracted before they become exponents:
// past 2^24 the exponent's own rounding would be powers of two.)  A refused part's reference is NaN and stays.
struct Share {
  float M = -__builtin_inff(), L = 0.f;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m, float l, const f32x4& x) {
    const float mn = M != M || m != m ? __builtin_nanf("") : fmaxf(M, m), mz = finite_or_zero(mn);
    const float w0 = __builtin_amdgcn_exp2f((M - mz) * kLog2e), w1 = __builtin_amdgcn_exp2f((m - mz) * kLog2e);
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

// Between LDS accesses of one wave whose lanes write what others read: the LDS takes a wave's accesses in their order,
// and the compiler is to leave them in it.  No instruction.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// The probabilities of slots s.. s + 3 added to their weights (the new token's, slot `len`, set); head(g): the
// reference (not -inf) of a key-value head's query head, and its own probability.
template <typename Head>
__device__ __forceinline__ void add_weights(const PagedAttnArgs& a, int b, int h, int s, int len, const Head& head) {
  const int64_t cap = a.c.capacity();
  const float* const sp = a.scores + ((int64_t)b * a.c.nkv + h) * a.g * cap + s;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < a.g; ++g) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(sp + g * cap);
    const f32x2 ml = head(g);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += __builtin_amdgcn_exp2f((y[e] - ml[0]) * kLog2e) * ml[1];
  }
  float* const wp = a.c.weight + a.c.token(b, s, h);
  f32x4 w = *reinterpret_cast<const f32x4*>(wp);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = s + e < len ? w[e] + t[e] : s + e == len ? t[e] : w[e];
  *reinterpret_cast<f32x4*>(wp) = w;
}

// One workgroup = one part of one row's slots for up to 16 HT query heads of one key-value head; its waves take units
// of UP = 4096 / D slots in turn (16 KB of keys and values).
//
// Both products are 16x16x32 matrix instructions, transposed: scores S^T = K Q^T, slots by heads, then O^T = V^T P^T.
// A tile's row r of keys is slot 8 (r / 4) + 4 t + r % 4 of its block of 32 (t: the first or second tile), so the
// scores that a lane holds of one head are those of eight slots in a row: exactly its part of the second product's
// operand, which never leaves its registers.  Keys and values come in whole lines and go through a wave's own LDS,
// which puts the keys into the tiles' order and transposes the values on reading.  A head's reference follows the
// running maximum with a lag (Probs; its value cancels in the end), so that most units need no exchange between lanes.
//
// Bound by memory where there is enough of it: 131000 slots of 32 / 8 heads of 128 in 90.2 us, 537 MB at 5.9 TB/s; 16
// rows of 3001 with the weights' scores (203 MB) in 39.4; 32 rows of up to 4000 of 64 in 32.6, 123 MB at 3.8 TB/s,
// whose unequal parts leave CUs idle at the end.  A short row is a chain of latencies (lengths, page, tokens, sums,
// output): 100 slots 7.7 us.  bf16 probabilities in three parts instead of two cost 1 to 3% (6 rows of up to 117000
// slots of 24 / 1 heads of 64: 33.3 us instead of 31.3), scores subtracted before they are scaled up to 1%.
template <int DT, int D, int W, int HT>
__global__ __launch_bounds__(64 * W, 2) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr int KB = 128 / D, UP = 32 * KB, NJ = D / 32, ND = D / 16, VR = 512 / D, NP = Split<DT>::N;
  constexpr int KROW = D + 8;              // halfwords of a key row in LDS: sixteen rows on different banks
  constexpr int VROW = D == 64 ? 72 : 144; // of a value row: four rows of 32 bytes on different banks
  constexpr int OROW = D + 4;              // floats of an output row in LDS
  constexpr int WAVE_H = UP * (KROW + VROW), ITEMS = W == 1 ? kAttnOneWaveItems : kAttnItems, kThreads = 64 * W;
  constexpr int HEADS = 16 * HT;
  static_assert(HEADS * OROW * 2 <= WAVE_H, "a wave's outputs take its tokens' place");
  typedef typename Act<DT>::frag frag;
  typedef Probs<DT> P;
  __shared__ __attribute__((aligned(16))) uint16_t kv_s[W][WAVE_H];
  __shared__ __attribute__((aligned(16))) uint16_t new_s[2][D];
  __shared__ float m_s[W][HEADS], l_s[W][HEADS];
  __shared__ f32x2 head_s[HEADS];
  __shared__ int bad_s[W];
  __shared__ unsigned arrived_s;

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, c = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  AttnItem it;
  if (!find_item<UP, ITEMS>(a.c, a.lengths, a.positions, a.c.nkv * a.htiles, a.at_once, blockIdx.x, &it)) return;
  const int b = it.b, h = it.tile / a.htiles, ht = it.tile - h * a.htiles;
  const int h0 = h * a.g + ht * HEADS, gh = min(a.g - ht * HEADS, HEADS);  // query heads of the row
  const int nh = a.c.nkv * a.g;
  const int len = it.len, pos = it.pos;
  uint16_t* const out = a.out + ((int64_t)b * nh + h0) * D;
  if (len < 0 || len >= a.c.capacity() || (uint64_t)(int64_t)pos >= (uint64_t)a.angles) {
    const uint16_t fill = len < 0 ? 0 : float_to_act_bits<DT>(__builtin_nanf(""));
    for (int i = tid; i < gh * D; i += kThreads) out[i] = fill;
    if (a.later && tid == 0) a.first[(b * a.c.nkv * a.htiles + it.tile) * 2 + 1] = 1;
    return;
  }
  const int nu = len / UP + 1;
  const int u0 = (int)((int64_t)it.part * nu / it.parts), u1 = (int)((int64_t)(it.part + 1) * nu / it.parts);
  const float* const cosr = a.cos + (int64_t)pos * (D / 2);
  const float* const sinr = a.sin + (int64_t)pos * (D / 2);
  const int32_t* const table = a.c.table + (int64_t)b * a.c.width;
  const int smask = (1 << a.c.log2s) - 1;

  u32x4 kr[8], vr[8];
  bool bad = false;
  // Lane i: the page of the unit's slots 8 i.. (past the row's end, its last page).
  auto load_ids = [&](int u) {
    const int slot = min(u * UP + 8 * min(lane, UP / 8 - 1), len);
    return table[slot >> a.c.log2s];
  };
  auto load = [&](int u, int ids) {
    const bool out_of_pool = (unsigned)ids >= (unsigned)a.c.pages;
    bad = bad || __ballot(out_of_pool);
    ids = out_of_pool ? 0 : ids;
    const int base = u * UP;
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // eight (D = 64) or four rows
      const int page = __builtin_amdgcn_readlane(ids, i * VR / 8);
      const int64_t at = ((((int64_t)page * a.c.nkv + h) << a.c.log2s) + ((base + i * VR) & smask)) * D + lane * 8;
      kr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.k + at));
      vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.v + at));
    }
  };
  uint16_t* const kw = kv_s[wv];
  uint16_t* const vw = kw + UP * KROW;
  const int srow = lane * 8 / D, sd = lane * 8 % D;  // this lane's place in a load's rows
  // A key lies in LDS in the order of the tiles' rows: slot 8 g + 4 t + e of a block at row 16 t + 4 g + e.
  auto krow = [&](int i) {
    return D == 64 ? (i >> 2) * 32 + (srow >> 2) * 16 + (i & 3) * 4 + (srow & 3) : (i & 1) * 16 + (i >> 1) * 4 + srow;
  };
  int u = u0 + wv, ids = 0;
  if (u < u1) {  // on their way before the query is at hand
    load(u, load_ids(u));
    ids = load_ids(min(u + W, u1 - 1));
  }

  // the query: heads past gh copy another and count for nothing
  u32x4 qf[HT][NJ][NP];
  QueryScale<DT> qs[HT];
#pragma unroll
  for (int ht0 = 0; ht0 < HT; ++ht0) {
    const int hd = ht0 * 16 + l16;
    const uint16_t* const qp = a.q + b * a.stride_q + (int64_t)(h0 + min(hd, gh - 1)) * D;
    const float scale = hd < gh ? a.scale : 0.f;
    float lo[NJ / 2][8], hi[NJ / 2][8], largest = 0.f;
#pragma unroll
    for (int j = 0; j < NJ / 2; ++j) {
      rope_chunk<DT, D>(qp, cosr, sinr, j, c, scale, lo[j], hi[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fmaxf(__builtin_fabsf(lo[j][e]), __builtin_fabsf(hi[j][e])));
    }
    const float f = qs[ht0].set(largest);
#pragma unroll
    for (int j = 0; j < NJ / 2; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[j][e] *= f, hi[j][e] *= f;
      split8<DT, true>(lo[j], qf[ht0][j]);
      split8<DT, true>(hi[j], qf[ht0][j + NJ / 2]);
    }
  }
  // The wave that takes the row's last unit rotates the new key, keeps it and the value at hand and writes them to
  // the cache.
  if (it.part == it.parts - 1 && wv == (nu - 1 - u0) % W) {
    const uint16_t* const kin = a.k + b * a.stride_k + h * D;
    float x[8], y[8];
    unpack8<DT>(*reinterpret_cast<const u32x4*>(kin + sd), x);
    unpack8<DT>(*reinterpret_cast<const u32x4*>(kin + (sd ^ (D / 2))), y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float cc = cosr[(sd & (D / 2 - 1)) + e], ss = sinr[(sd & (D / 2 - 1)) + e];
      float r1, r2;
      if (sd < D / 2) rope_pair(x[e], y[e], cc, ss, &r1, &r2), x[e] = r1;
      else rope_pair(y[e], x[e], cc, ss, &r1, &r2), x[e] = r2;
    }
    const u32x4 kn = pack8<DT>(x), vn = *reinterpret_cast<const u32x4*>(a.v + b * a.stride_v + h * D + sd);
    const int page = table[len >> a.c.log2s];
    if (srow == 0) {
      *reinterpret_cast<u32x4*>(&new_s[0][sd]) = kn;
      *reinterpret_cast<u32x4*>(&new_s[1][sd]) = vn;
      if (ht == 0 && (unsigned)page < (unsigned)a.c.pages) {
        const int64_t tok = ((((int64_t)page * a.c.nkv + h) << a.c.log2s) + (len & smask)) * D + sd;
        *reinterpret_cast<u32x4*>(a.c.k + tok) = kn;
        *reinterpret_cast<u32x4*>(a.c.v + tok) = vn;
      }
    }
  }

  float m[HT], l[HT];  // of head l16 of a tile: the reference and this lane's share of the sum
  f32x4 o[HT][ND];
  // The part's units; careful: infinities and NaN are looked for.
  auto attend = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HT; ++i) {
      m[i] = -__builtin_inff(), l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (; u < u1; u += W) {
      const int base = u * UP;
      const bool last = base + UP > len;  // the new token is in this unit, and what lies past it
      wave_lds_order();  // the new token is there, the unit before has been read
      if (last) {
        const int at = len - base;
        const u32x4 kn = *reinterpret_cast<const u32x4*>(&new_s[0][sd]);
        const u32x4 vn = *reinterpret_cast<const u32x4*>(&new_s[1][sd]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * VR + srow;
          kr[i] = row == at ? kn : kr[i];
          vr[i] = row == at ? vn : row > at ? u32x4{0u, 0u, 0u, 0u} : vr[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        *reinterpret_cast<u32x4*>(kw + krow(i) * KROW + sd) = kr[i];
        *reinterpret_cast<u32x4*>(vw + (i * VR + srow) * VROW + sd) = vr[i];
      }
      wave_lds_order();
      if (u + W < u1) {  // the next unit's loads travel under the rest
        load(u + W, ids);
        ids = load_ids(min(u + 2 * W, u1 - 1));
      }
#pragma unroll
      for (int i = 0; i < HT; ++i) {
        if constexpr (HT > 1) wave_lds_order();  // (keys held for both tiles would be spilled)
        f32x4 s[KB][2];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint16_t* const at = kw + (kb * 32 + t * 16 + l16) * KROW + 8 * c;
            frag kf[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) kf[j] = *reinterpret_cast<const frag*>(at + 32 * j);
            s[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto small = [&](auto f) __attribute__((always_inline)) {  // the small parts first
#pragma unroll
              for (int p = NP - 1; p > 0; --p)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                  s[kb][t] = Mfma<DT>::m16(f(kf[j]), __builtin_bit_cast(frag, qf[i][j][p]), s[kb][t]);
            };
            if (careful) small(finite_part<DT>);
            else small([](const frag& k) { return k; });
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              s[kb][t] = Mfma<DT>::m16(kf[j], __builtin_bit_cast(frag, qf[i][j][0]), s[kb][t]);
          }
        if (last) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (base + kb * 32 + 8 * c + 4 * t + e > len) s[kb][t][e] = -__builtin_inff();
        }
        if (a.scores && i * 16 + l16 < gh) {
          float* sp = a.scores + ((int64_t)b * nh + h0 + i * 16 + l16) * a.c.capacity() + base + 8 * c;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (base + kb * 32 + 8 * c + 4 * t <= len)
                *reinterpret_cast<f32x4*>(sp + kb * 32 + 4 * t) = s[kb][t] * qs[i].back();
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, s[kb][t][e]);
        const float log2e = kLog2e * qs[i].back();
        if (__ballot((top - m[i]) * log2e > P::lag)) {
          float mn = fmaxf(top, m[i]);
          mn = fmaxf(mn, __shfl_xor(mn, 16));
          mn = fmaxf(mn, __shfl_xor(mn, 32));
          const float al = __builtin_amdgcn_exp2f((m[i] - finite_or_zero(mn)) * log2e);
          l[i] *= al;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][d][e] *= al;
          m[i] = mn;
        }
        const float mz = finite_or_zero(m[i]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e >> 2][e & 3] - mz, log2e, P::above));
            l[i] += p[e];
          }
          u32x4 pf[NP];
          split8<DT, false>(p, pf);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const uint16_t* at = vw + (kb * 32 + 8 * c + (l16 >> 2)) * VROW + d * 16 + 4 * (l16 & 3);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * VROW));
            const u32x2 lw = __builtin_bit_cast(u32x2, lo), hw = __builtin_bit_cast(u32x2, hi);
            const frag vf = __builtin_bit_cast(frag, u32x4{lw[0], lw[1], hw[0], hw[1]});
            const frag vs = careful ? finite_part<DT>(vf) : vf;
#pragma unroll
            for (int p = NP - 1; p > 0; --p) o[i][d] = Mfma<DT>::m16(vs, __builtin_bit_cast(frag, pf[p]), o[i][d]);
            o[i][d] = Mfma<DT>::m16(vf, __builtin_bit_cast(frag, pf[0]), o[i][d]);
          }
        }
      }
    }
  };
  auto all_finite = [&]() __attribute__((always_inline)) {
    bool yes = true;
#pragma unroll
    for (int i = 0; i < HT; ++i) {
      float sum = l[i];
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += __builtin_fabsf(o[i][d][e]);
      yes = yes && !__ballot(i * 16 + l16 < gh && !(sum < __builtin_inff()));
    }
    return yes;
  };
  auto rewind = [&]() __attribute__((always_inline)) {
    u = u0 + wv;
    load(u, load_ids(u));
    ids = load_ids(min(u + W, u1 - 1));
  };
  // An infinity would meet the small parts of the other operand as inf * 0 or with the wrong sign, so it is to meet the
  // leading one alone, whose zeros and signs are the operand's.  Where a head's sums are not finite the part is done
  // again with keys and values that are not finite left out of the products with the small parts (a query's own have
  // none, split8).  What is finite keeps its bits.
  attend(std::false_type{});
  if (!all_finite()) rewind(), attend(std::true_type{});

  // The waves' outputs meet in LDS.
  wave_lds_order();
  float* const ow = reinterpret_cast<float*>(kw);
#pragma unroll
  for (int i = 0; i < HT; ++i) {
    const int hd = i * 16 + l16;
    l[i] += __shfl_xor(l[i], 16);
    l[i] += __shfl_xor(l[i], 32);
    if (hd < gh) {
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(ow + hd * OROW + d * 16 + 4 * c) = o[i][d];
      if (c == 0) m_s[wv][hd] = m[i] * qs[i].back(), l_s[wv][hd] = l[i];
    }
  }
  if (lane == 0) bad_s[wv] = bad;
  __syncthreads();
  int refused = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) refused |= bad_s[w];
  const int quads = gh * (D / 4), stride = min(a.g, HEADS) * D;
  const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.part + (int64_t)it.first * stride), (short)0, it.parts * stride * 4, kPagedBufFlags);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.stats + (int64_t)it.first * (2 * HEADS)), (short)0, it.parts * HEADS * 8, kPagedBufFlags);
  if (a.later && it.part == 0 && tid == 0) {
    int* const f = a.first + (b * a.c.nkv * a.htiles + it.tile) * 2;
    f[0] = it.first;
    f[1] = it.parts;
  }
  for (int i = tid; i < quads; i += kThreads) {
    const int hd = i / (D / 4), d = i % (D / 4) * 4;
    Share x;
#pragma unroll
    for (int w = 0; w < W; ++w)
      x.add(m_s[w][hd], l_s[w][hd],
            *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(kv_s[w]) + hd * OROW + d));
    if (refused) x.M = x.L = __builtin_nanf("");
    if (d == 0) head_s[hd] = f32x2{finite_or_zero(x.M), P::first / x.L};
    if (it.parts == 1)
      *reinterpret_cast<u32x2*>(out + hd * D + d) = x.template out<DT>();
    else
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x.t), rp,
                                             (uint32_t)(it.part * stride + i * 4) * 4u, 0, kPagedCoherentAux);
    if (d == 0 && (it.parts > 1 || a.later))
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{x.M, x.L}), rs,
                                            (uint32_t)(it.part * HEADS + hd) * 8u, 0, kPagedCoherentAux);
  }
  if (a.later) return;
  if (it.parts == 1) {
    if (a.scores && !refused) {  // no row of the call has more parts, nor a head tiles
      __builtin_amdgcn_s_waitcnt(0);  // the scores have left this wave
      __syncthreads();
      for (int s = 4 * tid; s <= len; s += 4 * kThreads)
        add_weights(a, b, h, s, len, [&](int g) { return head_s[g]; });
    }
    return;
  }

  // The last part of a row and tile to arrive joins them, in their order.
  __builtin_amdgcn_s_waitcnt(0);  // the stores have reached the level all XCDs share
  __syncthreads();
  unsigned* const cnt = a.cnt + b * (a.c.nkv * a.htiles) + it.tile;
  if (tid == 0) arrived_s = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived_s != (unsigned)(it.parts - 1)) return;
  if (tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // Threads: the quads of the output, and several runs of parts beside each other (or several goes, of a single wave).
  // Maxima, sums and outputs of eight parts travel together.
  const int runs = max(1, kThreads / quads), run = min(tid / quads, runs);
  f32x4* const red = reinterpret_cast<f32x4*>(&kv_s[0][0]);
  f32x2* const red_ml = reinterpret_cast<f32x2*>(red + kThreads);
  for (int i = tid - run * quads; i < quads; i += kThreads) {
    const int hd = i / (D / 4);
    Share x;
    if (run < runs) {
      for (int p0 = run; p0 < it.parts; p0 += runs * 8) {
        f32x4 t[8];
        f32x2 ml[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int p = min(p0 + k * runs, it.parts - 1);
          t[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rp, (uint32_t)(p * stride + i * 4) * 4u, 0, kPagedCoherentAux));
          ml[k] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, (uint32_t)(p * HEADS + hd) * 8u, 0,
                                                                                 kPagedCoherentAux));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (p0 + k * runs < it.parts) x.add(ml[k][0], ml[k][1], t[k]);
      }
    }
    if (runs > 1) {  // (then this is the only go, of all threads)
      if (run < runs) red[tid] = x.t, red_ml[tid] = f32x2{x.M, x.L};
      __syncthreads();
      if (run == 0)
        for (int r = 1; r < runs; ++r) x.add(red_ml[r * quads + i][0], red_ml[r * quads + i][1], red[r * quads + i]);
    }
    if (run == 0) *reinterpret_cast<u32x2*>(out + i * 4) = x.template out<DT>();
  }
}

// What the attention leaves to a second launch.  Workgroups [0, rows * heads): the parts of one row and query head
// joined (a wide group's by the last part alone would be one CU's traffic with memory).  The others add every
// slot's probabilities to its weight, from the scores, maxima and sums: the parts of the rows again, four slots
// a thread.  (In the attention itself the sums are not at hand until all parts are through.)  A chain of latencies, of
// the parts, their sums, the scores: 6.0 us for 16 rows of 3001 slots of 32 / 8 heads, 9.2 MB; 7.0 for 3 of up to 20000
// of 20 / 2 heads.
template <int DT, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_finish_kernel(PagedAttnArgs a) {
  constexpr int UP = 4096 / D, QUADS = D / 4, RUNS = kPagedThreads / QUADS;
  __shared__ f32x4 red[kPagedThreads];
  __shared__ f32x2 red_ml[kPagedThreads];
  const int tid = threadIdx.x, nh = a.c.nkv * a.g;
  auto parts_of = [&](int b, int h, int g) { return a.first + ((b * a.c.nkv + h) * a.htiles + g / a.tile) * 2; };
  if (blockIdx.x < (unsigned)(a.c.rows * nh)) {
    const int b = blockIdx.x / nh, head = blockIdx.x - b * nh, h = head / a.g, g = head - h * a.g;
    const int* const f = parts_of(b, h, g);
    const int first = f[0], parts = f[1];
    if (parts == 1) return;
    const int stride = min(a.g, a.tile) * D, run = tid / QUADS, i = tid % QUADS;
    const float* const part = a.part + (int64_t)first * stride + g % a.tile * D + i * 4;
    const float* const st = a.stats + ((int64_t)first * a.tile + g % a.tile) * 2;
    Share x;
    for (int p0 = run; p0 < parts; p0 += RUNS * 8) {
      f32x4 t[8];
      f32x2 ml[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t p = min(p0 + k * RUNS, parts - 1);
        t[k] = *reinterpret_cast<const f32x4*>(part + p * stride);
        ml[k] = *reinterpret_cast<const f32x2*>(st + p * (2 * a.tile));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (p0 + k * RUNS < parts) x.add(ml[k][0], ml[k][1], t[k]);
    }
    red[tid] = x.t;
    red_ml[tid] = f32x2{x.M, x.L};
    __syncthreads();
    if (run > 0) return;
    for (int r = 1; r < min(RUNS, parts); ++r)
      x.add(red_ml[r * QUADS + i][0], red_ml[r * QUADS + i][1], red[r * QUADS + i]);
    *reinterpret_cast<u32x2*>(a.out + ((int64_t)b * nh + head) * D + i * 4) = x.template out<DT>();
    return;
  }
  AttnItem it;
  const int item = blockIdx.x - a.c.rows * nh;
  if (!find_item<UP, kAttnItems>(a.c, a.lengths, a.positions, a.c.nkv, a.at_once, item, &it)) return;
  const int b = it.b, h = it.tile, len = it.len, pos = it.pos;
  if (len < 0 || len >= a.c.capacity() || (uint64_t)(int64_t)pos >= (uint64_t)a.angles) return;
  const int nu = len / UP + 1;
  const int s0 = (int)((int64_t)it.part * nu / it.parts) * UP;
  const int s1 = min((int)((int64_t)(it.part + 1) * nu / it.parts) * UP, len + 1);
  // the heads' maxima and sums: several threads a head, each some of its parts
  const int runs = kPagedThreads / a.g, run = tid / a.g, g = tid - run * a.g;
  const int* const f = parts_of(b, h, g);
  const int parts = f[1];  // (the same for all tiles of a row)
  Share x;
  if (run < runs) {
    const float* const st = a.stats + ((int64_t)f[0] * a.tile + g % a.tile) * 2;
    for (int p = run; p < parts; p += runs) {
      const float* const sp = st + p * (2 * a.tile);
      x.add(sp[0], sp[1], f32x4{0.f, 0.f, 0.f, 0.f});
    }
    red_ml[tid] = f32x2{x.M, x.L};
  }
  __syncthreads();
  if (run == 0) {
    for (int r = 1; r < min(runs, parts); ++r)
      x.add(red_ml[r * a.g + g][0], red_ml[r * a.g + g][1], f32x4{0.f, 0.f, 0.f, 0.f});
    red[g] = f32x4{finite_or_zero(x.M), Probs<DT>::first / x.L, 0.f, 0.f};
  }
  __syncthreads();
  if (red[0][0] != red[0][0]) return;  // a page outside the pool (in all heads alike)
  for (int s = s0 + 4 * tid; s < s1; s += 4 * kPagedThreads)
    add_weights(a, b, h, s, len, [&](int e0) { return f32x2{red[e0][0], red[e0][1]}; });
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
  PagedView c;
  const int32_t* lengths;
  const int32_t* new_table;  // [rows, new_width]
  int32_t* scratch;          // of a row and head: select_words(), see below
  int32_t* new_lengths;
  int new_width, keep, recent;
};

// What the selection leaves of a row and head: the key of the last kept token, how many equal keys are kept, and of
// every 256 slots the number of larger (low half) and of equal keys; then the kept slots.
constexpr int kSelectBlock = 256;
__host__ __device__ constexpr int64_t select_words(int64_t capacity, int64_t keep) {
  return 2 + (capacity + kSelectBlock - 1) / kSelectBlock + keep;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectBins = 4096;
constexpr int kSelectList = 2048;  // keys few enough to be put aside
constexpr int kSelectRank = 256;   // and to be ranked against each other

constexpr int kSelectRun = 32768;  // keys that LDS holds
constexpr int kSelectPlace = 16384;  // early slots that the selection lists itself

// One workgroup per row and key-value head finds the slots to keep.  The key of the last one (its weight's place in
// the order of all weights) lies in a range that a histogram of 4096 bins narrows twelve bits at a time; once no more
// than 2048 keys are in it they are put aside and narrowed alone, and the last 256 are ranked one against all.  The
// larger and equal keys of every 256 slots are counted, from which a launch that has all of the chip finds the slots'
// places.
//
// What bounds it is the latency of its steps on the one CU that has the row and head, so the keys are read from memory
// once and stay in LDS (of more than 32768 early slots, a run at a time in every step).  32768 slots: 20.1 us, of them
// 4.1 for the keys, 4.0 for the first histogram, 3.3 for the list, 2.8 for the counts; 100000 slots 55.1.  Equal
// weights are the slowest: all keys fall into one bin, an atomic on one address each, in every histogram (an eviction
// of 4 x 32768 slots 127 us instead of 54, of 576 slots 13.7 instead of 11.5, of 100000 328 instead of 91).
//
// ONCE: no row is longer than LDS holds (a kernel that may have to load again is slower for the others: 32768 slots
// 21.8 us instead of 20.2, 576 slots 6.2 instead of 5.7).  PLACE: the rows are short enough that the kept slots are
// best listed here (576 slots 6.5 us instead of 5.7 and 3.4 for a launch that places them, 16000 16.6 instead of 13.4
// and 5.0, 32768 26.0 instead of 20.2 and 5.1).
template <bool ONCE, bool PLACE>
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(EvictArgs a) {
  constexpr int WAVES = kSelectThreads / 64, RUN = kSelectRun, Q = RUN / (4 * kSelectThreads);
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x, b = blockIdx.y;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ __attribute__((aligned(16))) uint32_t key_s[RUN];
  __shared__ int hist[kSelectBins];
  __shared__ __attribute__((aligned(16))) uint32_t list[kSelectList];
  __shared__ uint16_t from_s[kSelectList];  // the 256 slots that a key of the list is from
  __shared__ int wave_s[2][WAVES], found_s[3];
  __shared__ __attribute__((aligned(16))) uint32_t rank_s[kSelectRank];
  __shared__ uint32_t edge_s;
  __shared__ int ties_s;
  const int n = a.lengths[b];
  if (n <= a.keep || n > a.c.capacity()) return;  // idle, or all of it kept
  const int early = n - a.recent;
  const int want = a.keep - a.recent;
  if (want == 0) return;  // the last ones alone
  int32_t* const scratch = a.scratch + ((int64_t)b * a.c.nkv + h) * select_words(a.c.capacity(), a.keep);

  // Quad q of a thread: four slots of a run from at(q) on; a wave's quads are `quads` * 256 slots in a row.
  const int quads = min(Q, (early + 4 * kSelectThreads - 1) / (4 * kSelectThreads));
  auto at = [&](int q) { return (wv * quads + q) * 256 + 4 * lane; };
  auto load = [&](int run) __attribute__((always_inline)) {
    int64_t tok[Q];
    f32x4 w[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) tok[q] = q < quads && run + at(q) < early ? a.c.token(b, run + at(q), h) : -1;
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (tok[q] >= 0) w[q] = *reinterpret_cast<const f32x4*>(a.c.weight + tok[q]);
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (q < quads) {
        u32x4 x = {0u, 0u, 0u, 0u};  // on a page outside the pool: below all
        if (tok[q] >= 0) x = u32x4{order_key(w[q][0]), order_key(w[q][1]), order_key(w[q][2]), order_key(w[q][3])};
        *reinterpret_cast<u32x4*>(&key_s[at(q)]) = x;
      }
  };
  const bool once = ONCE || early <= RUN;
  if (once) load(0);  // (a wave reads back what it wrote itself)
  auto quad = [&](int q) { return *reinterpret_cast<const u32x4*>(&key_s[at(q)]); };
  // f(s0, keys, valid) for every 256 early slots from s0 on, a quad of keys a lane, the first `valid` of them early.
  auto each_quad = [&](auto f) __attribute__((always_inline)) {
    for (int run = 0; run < early; run += RUN) {
      if (!once) load(run);
      for (int q = 0; q < quads; ++q) {
        const int s0 = run + (wv * quads + q) * 256;
        if (s0 >= early) break;
        f(s0, quad(q), early - s0 - 4 * lane);
      }
    }
  };
  auto each = [&](auto f) __attribute__((always_inline)) {  // f(key)
    each_quad([&](int s0, const u32x4& k, int valid) __attribute__((always_inline)) {
      if (s0 + 256 <= early) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f((uint32_t)k[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < valid) f((uint32_t)k[e]);
      }
    });
  };

  uint32_t lo = 0, hi = 0xFFFFFFFFu;
  int count = early, wanted = want;  // keys in the range, and how many of them are kept
  auto narrow = [&](auto keys, int stop) __attribute__((always_inline)) {
    while (count > stop && lo < hi) {
      const int shift = max(0, 32 - __builtin_clz(hi - lo) - 12);
      for (int i = tid; i < kSelectBins; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      keys([&](uint32_t key) __attribute__((always_inline)) {
        if (key >= lo && key <= hi) atomicAdd(&hist[(key - lo) >> shift], 1);
      });
      __syncthreads();
      // from the top: thread t has the bins 4 (1023 - t)..
      const int top = kSelectBins - 4 - 4 * tid;
      const int mine = hist[top] + hist[top + 1] + hist[top + 2] + hist[top + 3];
      const int upto = wave_scan(mine);
      if (lane == 63) wave_s[0][wv] = upto;
      __syncthreads();
      int above = upto - mine;
      for (int w = 0; w < wv; ++w) above += wave_s[0][w];
      if (above < wanted && above + mine >= wanted) {
        int e = 3;
        while (above + hist[top + e] < wanted) above += hist[top + e--];
        found_s[0] = top + e;
        found_s[1] = above;
        found_s[2] = hist[top + e];
      }
      __syncthreads();
      lo += (uint32_t)found_s[0] << shift;
      hi = min(hi, lo + ((1u << shift) - 1u));
      wanted -= found_s[1];
      count = found_s[2];
    }
  };
  narrow(each, kSelectList);
  uint32_t edge = lo;
  int ties = wanted;  // keys equal to the edge that are kept
  // Where a look at the keys is a pass over memory, the larger ones are counted while the list is made (100000 slots
  // 55.1 us instead of 65.5; 32768 in LDS gain nothing by it).
  const bool count_here = !once && lo < hi && early <= kSelectBlock << 16;
  int held = 0;  // keys put aside
  if (lo < hi) {
    __syncthreads();
    if (tid == 0) found_s[0] = 0;
    __syncthreads();
    each_quad([&](int s0, const u32x4& k, int valid) __attribute__((always_inline)) {
      int larger = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (count_here) larger += __popcll(__ballot(e < valid && k[e] > hi));
        if (e < valid && k[e] >= lo && k[e] <= hi) {
          const int to = atomicAdd(&found_s[0], 1);
          if (to < kSelectList)  // (weights that change under the call stay in bounds)
            list[to] = k[e], from_s[to] = (uint16_t)(s0 / kSelectBlock);
        }
      }
      if (count_here && lane == 0) scratch[2 + s0 / kSelectBlock] = larger;
    });
    __builtin_amdgcn_s_waitcnt(0);  // the counts are where others will add to them
    __syncthreads();
    held = min(found_s[0], kSelectList);
    narrow([&](auto f) __attribute__((always_inline)) {
      for (int i = tid; i < held; i += kSelectThreads) f(list[i]);
    }, kSelectRank);
    if (lo < hi) {
      // of the keys in the range (a thread has at most two): how many are larger, how many equal
      __syncthreads();
      if (tid < kSelectRank) rank_s[tid] = 0;
      if (tid == 0) found_s[0] = 0;
      __syncthreads();
      for (int i = tid; i < held; i += kSelectThreads)
        if (list[i] >= lo && list[i] <= hi) rank_s[min(atomicAdd(&found_s[0], 1), kSelectRank - 1)] = list[i];
      __syncthreads();
      if (tid < count) {
        const uint32_t key = rank_s[tid];
        int more = 0, same = 0;
#pragma unroll 4
        for (int i = 0; i < count; i += 4) {  // (what lies past them is zero; its count is taken off below)
          const u32x4 x = *reinterpret_cast<const u32x4*>(&rank_s[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) more += x[e] > key, same += x[e] == key;
        }
        if (key == 0) same -= (-count) & 3;
        // (all equal keys say the same)
        if (more < wanted && more + same >= wanted) edge_s = key, ties_s = wanted - more;
      }
      __syncthreads();
      edge = edge_s;
      ties = ties_s;
    } else {
      edge = lo;
      ties = wanted;
    }
  }

  if constexpr (PLACE) {
    int32_t* const kept = scratch + (select_words(a.c.capacity(), a.keep) - a.keep);
    // 1 for a larger key, 1 << 16 for an equal one
    auto weigh = [&](uint32_t key, bool valid) { return !valid ? 0 : key > edge ? 1 : key == edge ? 1 << 16 : 0; };
    int mine = 0;
    each_quad([&](int, const u32x4& k, int valid) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += weigh(k[e], e < valid);
    });
    mine = __builtin_amdgcn_readlane(wave_scan(mine), 63);
    if (lane == 0) wave_s[1][wv] = mine;
    __syncthreads();
    int front = 0;
    for (int w = 0; w < wv; ++w) front += wave_s[1][w];
    each_quad([&](int s0, const u32x4& k, int valid) __attribute__((always_inline)) {
      int x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x += weigh(k[e], e < valid);
      const int upto = front + wave_scan(x);
      x = upto - x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int y = weigh(k[e], e < valid), to = (x & 0xFFFF) + min(x >> 16, ties);
        if ((y == 1 || (y && x >> 16 < ties)) && (unsigned)to < (unsigned)want) kept[to] = s0 + 4 * lane + e;
        x += y;
      }
      front = __builtin_amdgcn_readlane(upto, 63);
    });
    for (int i = tid; i < a.recent; i += kSelectThreads) kept[want + i] = early + i;
    return;
  }
  if (tid == 0) scratch[0] = (int)edge, scratch[1] = ties;
  if (count_here) {
    for (int i = tid; i < held; i += kSelectThreads)
      if (list[i] >= edge) atomicAdd(&scratch[2 + from_s[i]], list[i] > edge ? 1 : 1 << 16);
    return;
  }
  each_quad([&](int s0, const u32x4& k, int valid) __attribute__((always_inline)) {
    int x = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) x += k[e] > edge ? 1 : k[e] == edge ? 1 << 16 : 0;
    x = __builtin_amdgcn_readlane(wave_scan(x), 63);
    if (lane == 0) scratch[2 + s0 / kSelectBlock] = x;
  });
}

// One workgroup per 1024 slots of a row and head: the kept slots in their order.  A slot's place is the number of
// larger keys in front of it, and of equal ones as far as they are kept; the last `recent` come behind all.  Latency
// again (counts, page, weight, two sums over lanes): 5.0 us for 4 x 8 x 32768 slots.
constexpr int kPlaceSlots = 4 * kPagedThreads;

__global__ __launch_bounds__(kPagedThreads) void paged_place_kernel(EvictArgs a) {
  constexpr int WAVES = kPagedThreads / 64;
  __shared__ int front_s[2][WAVES], own_s[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = blockIdx.y, b = blockIdx.z;
  const int s0 = blockIdx.x * kPlaceSlots, s = s0 + 4 * tid, n = a.lengths[b];
  if (n <= a.keep || n > a.c.capacity() || s0 >= n) return;  // idle, or all of it kept: no list
  const int early = n - a.recent, want = a.keep - a.recent;
  const int32_t* const scratch = a.scratch + ((int64_t)b * a.c.nkv + h) * select_words(a.c.capacity(), a.keep);
  int32_t* const kept =
      a.scratch + ((int64_t)b * a.c.nkv + h + 1) * select_words(a.c.capacity(), a.keep) - a.keep;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (s + e >= early && s + e < n) kept[want + s + e - early] = s + e;
  if (want == 0 || s0 >= early) return;
  const uint32_t edge = (uint32_t)scratch[0];
  const int ties = scratch[1];
  int larger = 0, equal = 0;  // in front of this workgroup
  for (int i = tid; i < s0 / kSelectBlock; i += kPagedThreads) {
    const int x = scratch[2 + i];
    larger += x & 0xFFFF, equal += x >> 16;
  }
  uint32_t key[4] = {0u, 0u, 0u, 0u};
  const int64_t at = s < early ? a.c.token(b, s, h) : -1;
  if (at >= 0) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(a.c.weight + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) key[e] = order_key(w[e]);
  }
  int x = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (s + e < early) x += key[e] > edge ? 1 : key[e] == edge ? 1 << 16 : 0;
  const int upto = wave_scan(x);
  larger = wave_scan(larger), equal = wave_scan(equal);
  if (lane == 63) front_s[0][wv] = larger, front_s[1][wv] = equal, own_s[wv] = upto;
  __syncthreads();
  int l = (upto - x) & 0xFFFF, t = (upto - x) >> 16;
  for (int w = 0; w < WAVES; ++w) l += front_s[0][w], t += front_s[1][w];
  for (int w = 0; w < wv; ++w) l += own_s[w] & 0xFFFF, t += own_s[w] >> 16;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool g = s + e < early && key[e] > edge, q = s + e < early && key[e] == edge;
    const int to = l + min(t, ties);
    if ((g || (q && t < ties)) && (unsigned)to < (unsigned)want) kept[to] = s + e;  // (whatever the scratch holds)
    l += g, t += q;
  }
}

// Sixteen bytes of a kept token's key and value a thread, of four tokens at a time: the chain from place to slot to
// page to token is four loads long, and four of them hide each other.  Bound by memory: 4 x 8 x 4096 tokens of 128 in
// 28.1 us, 135 MB at 4.8 TB/s, read in pieces of 256 bytes.
template <int D>
__global__ __launch_bounds__(kPagedThreads) void paged_copy_kernel(EvictArgs a) {
  constexpr int CH = D / 8, TOK = kPagedThreads / CH, PER = 4;
  const int h = blockIdx.y, b = blockIdx.z, c = threadIdx.x % CH;
  const int len = a.lengths[b], n = len > a.c.capacity() ? -1 : min(len, a.keep);
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.new_lengths[b] = n < 0 ? -1 : n;
  const int j0 = blockIdx.x * (TOK * PER) + threadIdx.x / CH;
  if (j0 >= n) return;
  const int32_t* const kept =
      a.scratch + ((int64_t)b * a.c.nkv + h + 1) * select_words(a.c.capacity(), a.keep) - a.keep;
  const bool all = len <= a.keep;
  int64_t src[PER], dst[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = min(j0 + i * TOK, n - 1);
    src[i] = all ? j : min((unsigned)kept[j], (unsigned)len - 1u);
    dst[i] = a.new_table[(int64_t)b * a.new_width + (j >> a.c.log2s)];
  }
  u32x4 k[PER], v[PER];
  float w[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = min(j0 + i * TOK, n - 1);
    const int64_t page = dst[i];
    src[i] = a.c.token(b, (int)src[i], h);
    const bool ok = src[i] >= 0 && (uint64_t)page < (uint64_t)a.c.pages && j0 + i * TOK < n;
    dst[i] = ok ? ((page * a.c.nkv + h) << a.c.log2s) + (j & ((1 << a.c.log2s) - 1)) : -1;
    if (ok) {
      k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.k + src[i] * D + c * 8));
      v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.c.v + src[i] * D + c * 8));
      w[i] = a.c.weight[src[i]];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (dst[i] >= 0) {
      *reinterpret_cast<u32x4*>(a.c.k + dst[i] * D + c * 8) = k[i];
      *reinterpret_cast<u32x4*>(a.c.v + dst[i] * D + c * 8) = v[i];
      if (c == 0) a.c.weight[dst[i]] = w[i];
    }
}

}  // namespace w4

// ---------------------------------------------------------------- host side
using namespace w4host;

namespace {

// The checks every entry point makes of a cache; 0 or the error code.
int check_cache(const w4_paged_cache* c, int dtype, const char* what) {
  if (!c) return fail(W4_ERR_INVALID, "%s: null cache", what);
  if (dtype != W4_DTYPE_BF16 && dtype != W4_DTYPE_FP16)
    return fail(W4_ERR_INVALID, "%s: dtype must be bf16 or fp16 (got code %d)", what, dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(W4_ERR_UNSUPPORTED, "%s: heads of %lld (64 or 128)", what, (long long)c->head_dim);
  if (!is_pow2(c->page_size) || c->page_size < 8 || c->page_size > 1024)
    return fail(W4_ERR_UNSUPPORTED, "%s: pages of %lld tokens (a power of two from 8 to 1024)", what,
                (long long)c->page_size);
  if (c->pages < 1 || c->pages >= (1ll << 31) || c->kv_heads < 1 || c->kv_heads > 65535 || c->rows < 0 ||
      c->rows > 65535 || c->width < 1 || c->width > (1ll << 30) || c->width * c->page_size >= (1ll << 30))
    return fail(W4_ERR_INVALID, "%s: %lld pages, %lld heads, a table of %lld x %lld pages of %lld", what,
                (long long)c->pages, (long long)c->kv_heads, (long long)c->rows, (long long)c->width,
                (long long)c->page_size);
  if (!c->k || !c->v || (c->rows && !c->table)) return fail(W4_ERR_INVALID, "%s: null pointer", what);
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16)
    return fail(W4_ERR_INVALID, "%s: pages must be 16-byte aligned", what);
  return W4_OK;
}

w4::PagedView view_of(const w4_paged_cache* c) {
  w4::PagedView v{};
  v.k = static_cast<uint16_t*>(c->k);
  v.v = static_cast<uint16_t*>(c->v);
  v.weight = c->weight;
  v.table = c->table;
  v.pages = c->pages;
  v.nkv = (int)c->kv_heads;
  v.log2s = ilog2(c->page_size);
  v.rows = (int)c->rows;
  v.width = (int)c->width;
  return v;
}

bool rows_ok(const void* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 8 == 0; }

}  // namespace

extern "C" int w4_paged_append(const w4_paged_cache* cache, int dtype, const void* k, const void* v, int64_t stride_k,
                               int64_t stride_v, int64_t tokens, const int32_t* rows, const int32_t* slots,
                               const int32_t* positions, const float* cos, const float* sin, int64_t angles,
                               void* stream) {
  clear_error();
  if (const int rc = check_cache(cache, dtype, "w4_paged_append")) return rc;
  if (tokens < 0 || angles < 1)
    return fail(W4_ERR_INVALID, "w4_paged_append: %lld tokens, %lld angles", (long long)tokens, (long long)angles);
  if (tokens == 0 || cache->rows == 0) return W4_OK;
  if (!k || !v || !rows || !slots || !positions || !cos || !sin)
    return fail(W4_ERR_INVALID, "w4_paged_append: null pointer");
  if (!rows_ok(k, stride_k) || !rows_ok(v, stride_v) || ((uintptr_t)cos | (uintptr_t)sin) % 16)
    return fail(W4_ERR_INVALID, "w4_paged_append: operands must be 16-byte aligned, row strides multiples of 8");
  w4::AppendArgs a{view_of(cache), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), stride_k,
                   stride_v, tokens, angles, rows, slots, positions, cos, sin};
  const int64_t per = cache->kv_heads * (cache->head_dim / 16);
  const int64_t most = 0xFFFFFFFFll / w4::kPagedThreads;  // HIP refuses launches of 2^32 threads and more
  if (tokens > most * w4::kPagedThreads / per)
    return fail(W4_ERR_UNSUPPORTED, "w4_paged_append: %lld tokens in a call", (long long)tokens);
  const dim3 grid((unsigned)((tokens * per + w4::kPagedThreads - 1) / w4::kPagedThreads));
  hipStream_t st = static_cast<hipStream_t>(stream);
#define W4_APPEND(DT, D) w4::paged_append_kernel<DT, D><<<grid, w4::kPagedThreads, 0, st>>>(a)
  if (dtype == W4_DTYPE_BF16) {
    if (cache->head_dim == 64) W4_APPEND(W4_DTYPE_BF16, 64);
    else W4_APPEND(W4_DTYPE_BF16, 128);
  } else {
    if (cache->head_dim == 64) W4_APPEND(W4_DTYPE_FP16, 64);
    else W4_APPEND(W4_DTYPE_FP16, 128);
  }
#undef W4_APPEND
  return check_launch("w4_paged_append");
}

namespace {

struct PagedAttnPlan {
  int64_t tile, tiles, items;   // query heads of a tile, tiles a row, workgroups
  bool one_wave;                // those of one wave each
  size_t part, first, bytes;    // offsets of PagedAttnArgs' part and first in the workspace, and all of it
};

// `units` of slots that a row has at most.  More rows and tiles than the chip holds workgroups of four waves (two a CU:
// LDS) are faster a wave each, four or eight to a CU: of 32 / 8 heads of 64, 500 rows of up to 100 slots 29.9 us
// instead of 73.2, 96 of them 9.9 instead of 14.5, 200 of up to 1000 46.6 instead of 51.0.  Long rows are not:
// their units follow each other in one wave (64 of 4000 87.8 instead of 82.7; one of 131000 among 31 short ones 69
// instead of 49).
//
// More than sixteen query heads a key-value head of 64 share their slots' loads in tiles of 32, where the parts are
// long enough for it: 24 / 1 heads, 10 rows of 107000 slots with weights 109 us instead of 170, 6 of up to 117000 26.7
// instead of 49.1; 16 of up to 2000 would take 14.2 instead of 11.1.  So they do where the weights then need no second
// launch (7 of 15 11.8 us instead of 8.4 and 5.8, 300 of 120 17.7 instead of 15.9 and 12.7).  (Heads of 128 have no
// registers for two tiles.)  (Both sides of each with bf16 probabilities in two parts, 1 to 3% faster than three.)
bool paged_attn_plan(int64_t rows, int64_t num_heads, int64_t kv_heads, int64_t head_dim, int64_t units, bool weights,
                     PagedAttnPlan* p) {
  if (rows < 0 || num_heads < 1 || kv_heads < 1 || num_heads % kv_heads) return false;
  const int64_t g = num_heads / kv_heads;
  const bool alone = weights && units <= w4::kAttnMinUnits && g <= 32;
  p->tile = g > 16 && head_dim == 64 && (alone || rows * kv_heads * units >= 8 * w4::kAttnItems) ? 32 : 16;
  p->tiles = kv_heads * ((g + p->tile - 1) / p->tile);
  p->one_wave = rows * p->tiles > 2 * device_cu_count() && units <= 128;
  p->items = (p->one_wave ? w4::kAttnOneWaveItems : w4::kAttnItems) + rows * p->tiles + 1;
  if (p->items >= (1 << 22)) return false;
  p->part = W4_WORKSPACE_COUNTER_BYTES + (size_t)(p->items * p->tile) * 8;
  p->first = p->part;
  if (rows * p->tiles <= w4::kPagedCounters) p->first += (size_t)(p->items * std::min(g, p->tile) * head_dim) * 4;
  p->bytes = p->first + (size_t)(rows * p->tiles) * 8;
  return true;
}

template <int DT, int D>
int launch_paged_attention(const w4::PagedAttnArgs& a, const PagedAttnPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.items), threads(p.one_wave ? 64 : 64 * w4::kAttnWaves);
  auto run = [&](auto kernel) { kernel<<<grid, threads, 0, st>>>(a); };
  if (p.tile == 16) {
    if (p.one_wave) run(w4::paged_attention_kernel<DT, D, 1, 1>);
    else run(w4::paged_attention_kernel<DT, D, w4::kAttnWaves, 1>);
  } else if constexpr (D == 64) {
    if (p.one_wave) run(w4::paged_attention_kernel<DT, D, 1, 2>);
    else run(w4::paged_attention_kernel<DT, D, w4::kAttnWaves, 2>);
  }
  if (const int rc = check_launch("w4_paged_attention")) return rc;
  if (!a.later) return W4_OK;
  const int64_t more = a.scores ? w4::kAttnItems + (int64_t)a.c.rows * a.c.nkv + 1 : 0;
  const dim3 finish((unsigned)((int64_t)a.c.rows * a.c.nkv * a.g + more));
  w4::paged_finish_kernel<DT, D><<<finish, w4::kPagedThreads, 0, st>>>(a);
  return check_launch("w4_paged_attention (finish)");
}

}  // namespace

extern "C" size_t w4_paged_attention_workspace_bytes(int64_t rows, int64_t num_heads, int64_t kv_heads,
                                                     int64_t head_dim) {
  size_t bytes = 0;  // of tables of any width
  for (const int64_t units : {1, 128, 129, 1 << 30})
    for (const bool weights : {false, true}) {
      PagedAttnPlan p;
      if (rows > 0 && paged_attn_plan(rows, num_heads, kv_heads, head_dim, units, weights, &p))
        bytes = std::max(bytes, p.bytes);
    }
  return bytes;
}

extern "C" int w4_paged_attention(const w4_paged_cache* cache, int dtype, const void* q, const void* k, const void* v,
                                  int64_t stride_q, int64_t stride_k, int64_t stride_v, int64_t num_heads,
                                  const int32_t* lengths, const int32_t* positions, const float* cos,
                                  const float* sin, int64_t angles, void* out, float* scores, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = check_cache(cache, dtype, "w4_paged_attention")) return rc;
  if (num_heads < 1 || num_heads % cache->kv_heads || num_heads / cache->kv_heads > 256 || angles < 1)
    return fail(W4_ERR_INVALID, "w4_paged_attention: %lld query heads on %lld key-value heads, %lld angles",
                (long long)num_heads, (long long)cache->kv_heads, (long long)angles);
  if (cache->rows == 0) return W4_OK;
  const int64_t units = (cache->width * cache->page_size * cache->head_dim + 4095) / 4096;
  PagedAttnPlan p;
  if (!paged_attn_plan(cache->rows, num_heads, cache->kv_heads, cache->head_dim, units, cache->weight, &p) ||
      cache->rows * num_heads >= (1 << 23))
    return fail(W4_ERR_UNSUPPORTED, "w4_paged_attention: %lld rows of %lld heads", (long long)cache->rows,
                (long long)num_heads);
  if (!q || !k || !v || !lengths || !positions || !cos || !sin || !out || (cache->weight && !scores))
    return fail(W4_ERR_INVALID, "w4_paged_attention: null pointer");
  if (!rows_ok(q, stride_q) || !rows_ok(k, stride_k) || !rows_ok(v, stride_v) ||
      ((uintptr_t)cos | (uintptr_t)sin | (uintptr_t)out | (uintptr_t)scores | (uintptr_t)cache->weight) % 16)
    return fail(W4_ERR_INVALID, "w4_paged_attention: operands must be 16-byte aligned, row strides multiples of 8");
  if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 256)
    return fail(W4_ERR_WORKSPACE, "w4_paged_attention: needs a 256-byte aligned workspace of %zu bytes (got %zu)",
                p.bytes, workspace_bytes);
  w4::PagedAttnArgs a{};
  a.c = view_of(cache);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.stride_q = stride_q, a.stride_k = stride_k, a.stride_v = stride_v, a.angles = angles;
  a.lengths = lengths, a.positions = positions, a.cos = cos, a.sin = sin;
  a.out = static_cast<uint16_t*>(out);
  a.scores = cache->weight ? scores : nullptr;
  char* const ws = static_cast<char*>(workspace);
  a.cnt = reinterpret_cast<unsigned*>(ws);
  a.stats = reinterpret_cast<float*>(ws + W4_WORKSPACE_COUNTER_BYTES);
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.first = reinterpret_cast<int*>(ws + p.first);
  a.scale = 1.f / sqrtf((float)cache->head_dim);
  a.g = (int)(num_heads / cache->kv_heads);
  a.htiles = (int)(p.tiles / cache->kv_heads);
  // The weights need a launch behind the attention, but where every row is a workgroup's alone (1 row of 100 slots of
  // 32 / 8 heads of 128 9.2 us instead of 8.2 and 4.6, 250 of them 31.5 instead of 30.0 and 15.8).  Without them the
  // last part joins, unless a tile's outputs are more than two quads a thread (four of a lone wave, whose rows have few
  // parts), or its parts may be more than the joining reads in two goes (24 heads of 64 on one key-value head, 131000
  // slots in 128 parts: 36 us, with a launch of its own 20).
  a.tile = (int)p.tile;
  const int quads = std::min(a.g, a.tile) * (int)cache->head_dim / 4, threads = p.one_wave ? 64 : 64 * w4::kAttnWaves;
  a.at_once = 8 * std::max(threads / quads, 1);
  const int64_t parts = std::min(p.items / (cache->rows * p.tiles), units / w4::kAttnMinUnits + 1);
  const bool whole = units <= w4::kAttnMinUnits;  // no row of the table has a second part
  a.later = a.scores ? !whole || a.htiles > 1
                     : !whole && (quads > (p.one_wave ? 4 : 2) * threads || parts > 2 * a.at_once + 1);
  if (a.later) a.at_once = 1 << 20;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == W4_DTYPE_BF16)
    return cache->head_dim == 64 ? launch_paged_attention<W4_DTYPE_BF16, 64>(a, p, st)
                                 : launch_paged_attention<W4_DTYPE_BF16, 128>(a, p, st);
  return cache->head_dim == 64 ? launch_paged_attention<W4_DTYPE_FP16, 64>(a, p, st)
                               : launch_paged_attention<W4_DTYPE_FP16, 128>(a, p, st);
}

extern "C" size_t w4_paged_evict_scratch_words(const w4_paged_cache* cache, int64_t keep) {
  if (!cache || cache->rows < 1 || cache->kv_heads < 1 || cache->width < 1 || cache->page_size < 1 || keep < 1)
    return 0;
  return (size_t)(cache->rows * cache->kv_heads * w4::select_words(cache->width * cache->page_size, keep));
}

extern "C" int w4_paged_evict(const w4_paged_cache* cache, int dtype, const int32_t* lengths,
                              const int32_t* new_table, int64_t new_width, int64_t keep, int64_t recent,
                              int32_t* scratch, int32_t* new_lengths, void* stream) {
  clear_error();
  if (const int rc = check_cache(cache, dtype, "w4_paged_evict")) return rc;
  if (keep < 1 || recent < 0 || recent > keep || new_width < 1 || new_width > (1ll << 30) ||
      new_width * cache->page_size >= (1ll << 30) || keep > new_width * cache->page_size)
    return fail(W4_ERR_INVALID, "w4_paged_evict: keep %lld with the last %lld in %lld pages of %lld", (long long)keep,
                (long long)recent, (long long)new_width, (long long)cache->page_size);
  if (cache->rows == 0) return W4_OK;
  if (!cache->weight || !lengths || !new_table || !scratch || !new_lengths)
    return fail(W4_ERR_INVALID, "w4_paged_evict: null pointer");
  if ((uintptr_t)cache->weight % 16) return fail(W4_ERR_INVALID, "w4_paged_evict: weight must be 16-byte aligned");
  w4::EvictArgs a{view_of(cache), lengths, new_table, scratch, new_lengths, (int)new_width, (int)keep, (int)recent};
  const int64_t slots = cache->width * cache->page_size;
  const unsigned heads = (unsigned)cache->kv_heads, rows = (unsigned)cache->rows;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (slots > keep) {  // (else no row has more than it keeps)
    const bool place = recent < keep && slots - recent <= w4::kSelectPlace;
    if (recent < keep) {
      const dim3 grid(heads, rows);
      if (place) w4::paged_select_kernel<true, true><<<grid, w4::kSelectThreads, 0, st>>>(a);
      else if (slots - recent <= w4::kSelectRun)
        w4::paged_select_kernel<true, false><<<grid, w4::kSelectThreads, 0, st>>>(a);
      else w4::paged_select_kernel<false, false><<<grid, w4::kSelectThreads, 0, st>>>(a);
      if (const int rc = check_launch("w4_paged_evict (select)")) return rc;
    }
    if (!place) {
      const dim3 grid((unsigned)((slots + w4::kPlaceSlots - 1) / w4::kPlaceSlots), heads, rows);
      w4::paged_place_kernel<<<grid, w4::kPagedThreads, 0, st>>>(a);
      if (const int rc = check_launch("w4_paged_evict (place)")) return rc;
    }
  }
  const int64_t tok = 4 * w4::kPagedThreads / (cache->head_dim / 8);
  const dim3 grid((unsigned)((keep + tok - 1) / tok), heads, rows);
  if (cache->head_dim == 64) w4::paged_copy_kernel<64><<<grid, w4::kPagedThreads, 0, st>>>(a);
  else w4::paged_copy_kernel<128><<<grid, w4::kPagedThreads, 0, st>>>(a);
  return check_launch("w4_paged_evict (copy)");
}
