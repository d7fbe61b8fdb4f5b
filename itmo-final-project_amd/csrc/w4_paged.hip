// Key-value cache in pages for batches of sequences (int4_hip/paged.py): tokens
// written into the pages, the attention of one new token of every sequence over
// them, and eviction by accumulated attention weight.
#include <hip/hip_runtime.h>

#include "w4_common.hpp"

namespace w4 {

constexpr int kPagedThreads = 256;

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

// Eight rotary pairs of key (or the sixteen values beside them) a thread.
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
  float scale;    // 1 / sqrt(D)
  int g;
};

// One workgroup per row and key-value head, its query heads one after the other;
// a thread holds the running maximum, sum and output of every 256th slot, joined at
// the end of a head.  The weights' pass computes the scores again.
template <int DT, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_attention_kernel(PagedAttnArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y;
  __shared__ __attribute__((aligned(16))) float q_s[D];
  __shared__ float red[4], o_s[4][D];
  __shared__ int bad_s;
  const int len = a.lengths[b], pos = a.positions[b];
  uint16_t* const out = a.out + ((int64_t)b * a.c.nkv + h) * a.g * D;
  const int n = len + 1;
  if (tid == 0) bad_s = 0;
  __syncthreads();
  bool bad = len >= a.c.capacity() || (uint64_t)(int64_t)pos >= (uint64_t)a.angles;
  if (len >= 0 && !bad) {
    for (int p = tid; p <= (len >> a.c.log2s); p += kPagedThreads)
      if (a.c.token(b, p << a.c.log2s, h) < 0) bad_s = 1;
    const int64_t at = a.c.token(b, len, h);
    if (at >= 0) {
      if (tid < D / 2) {
        const uint16_t* kp = a.k + b * a.stride_k + h * D + tid;
        float r1, r2;
        rope_pair(act_bits_to_float(kp[0], DT), act_bits_to_float(kp[D / 2], DT), a.cos[(int64_t)pos * (D / 2) + tid],
                  a.sin[(int64_t)pos * (D / 2) + tid], &r1, &r2);
        a.c.k[at * D + tid] = float_to_act_bits<DT>(r1);
        a.c.k[at * D + tid + D / 2] = float_to_act_bits<DT>(r2);
      } else if (tid >= 128 && tid < 128 + D) {
        a.c.v[at * D + tid - 128] = a.v[b * a.stride_v + h * D + tid - 128];
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  bad = bad || bad_s;
  if (len < 0 || bad) {
    const uint16_t fill = len < 0 ? 0 : float_to_act_bits<DT>(__builtin_nanf(""));
    for (int i = tid; i < a.g * D; i += kPagedThreads) out[i] = fill;
    return;
  }
  auto score = [&](int j) {
    const uint16_t* kp = a.c.k + a.c.token(b, j, h) * D;
    float s = 0.f;
    for (int d = 0; d < D; d += 8) {
      float x[8];
      unpack8<DT>(*reinterpret_cast<const u32x4*>(kp + d), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(q_s[d + e], x[e], s);
    }
    return s;
  };
  for (int hq = 0; hq < a.g; ++hq) {
    __syncthreads();
    if (tid < D / 2) {
      const uint16_t* qp = a.q + b * a.stride_q + (int64_t)(h * a.g + hq) * D + tid;
      float r1, r2;
      rope_pair(act_bits_to_float(qp[0], DT), act_bits_to_float(qp[D / 2], DT), a.cos[(int64_t)pos * (D / 2) + tid],
                a.sin[(int64_t)pos * (D / 2) + tid], &r1, &r2);
      q_s[tid] = r1 * a.scale;
      q_s[tid + D / 2] = r2 * a.scale;
    }
    __syncthreads();
    float m = -__builtin_inff(), l = 0.f, o[D];
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = 0.f;
    for (int j = tid; j < n; j += kPagedThreads) {
      const float s = score(j);
      const float mn = fmaxf(m, s), base = mn == -__builtin_inff() ? 0.f : mn;
      const float al = expf(m - base), p = expf(s - base);
      const uint16_t* vp = a.c.v + a.c.token(b, j, h) * D;
      l = l * al + p;
#pragma unroll
      for (int d = 0; d < D; d += 8) {
        float x[8];
        unpack8<DT>(*reinterpret_cast<const u32x4*>(vp + d), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[d + e] = __builtin_fmaf(p, x[e], o[d + e] * al);
      }
      m = mn;
    }
    const float wm = wave_max(m);
    if (lane == 0) red[wv] = wm;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), base = M == -__builtin_inff() ? 0.f : M;
    const float al = expf(m - base);
    __syncthreads();
    const float wl = wave_sum(l * al);
    if (lane == 0) red[wv] = wl;
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const float t = wave_sum(l == 0.f ? 0.f : o[d] * al);
      if (lane == 0) o_s[wv][d] = t;
    }
    __syncthreads();
    const float L = (red[0] + red[1]) + (red[2] + red[3]);
    if (tid < D)
      out[hq * D + tid] = float_to_act_bits<DT>(((o_s[0][tid] + o_s[1][tid]) + (o_s[2][tid] + o_s[3][tid])) / L);
    if (a.c.weight)
      for (int j = tid; j < n; j += kPagedThreads) {
        float* w = a.c.weight + a.c.token(b, j, h);
        const float p = expf(score(j) - base) / L;
        *w = j == len && hq == 0 ? p : *w + p;
      }
  }
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
  PagedView c;
  const int32_t* lengths;
  const int32_t* new_table;  // [rows, new_width]
  int32_t* kept;             // [rows, nkv, keep]
  int32_t* new_lengths;
  int new_width, keep, recent;
};

// One workgroup per row and key-value head finds the slots to keep: the key of the
// last one by bisection, then its equals counted from the front.
__global__ __launch_bounds__(kPagedThreads) void paged_select_kernel(EvictArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = blockIdx.x, b = blockIdx.y;
  __shared__ int red[4];
  int n = a.lengths[b];
  if (n > a.c.capacity()) n = -1;
  if (h == 0 && tid == 0) a.new_lengths[b] = n < 0 ? -1 : min(n, a.keep);
  if (n < 0) return;
  int32_t* const kept = a.kept + ((int64_t)b * a.c.nkv + h) * a.keep;
  if (n <= a.keep) {
    for (int j = tid; j < n; j += kPagedThreads) kept[j] = j;
    return;
  }
  const int early = n - a.recent, want = a.keep - a.recent;
  auto key = [&](int j) {
    const int64_t at = a.c.token(b, j, h);
    return at < 0 ? 0u : order_key(a.c.weight[at]);
  };
  auto total = [&](int x) {  // of the workgroup
    for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s);
    __syncthreads();
    if (lane == 0) red[wv] = x;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
  };
  uint32_t edge = 0;  // the largest key that at least `want` slots reach
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = edge | (1u << bit);
    int x = 0;
    for (int j = tid; j < early; j += kPagedThreads) x += key(j) >= t;
    if (total(x) >= want) edge = t;
  }
  int above = 0;
  for (int j = tid; j < early; j += kPagedThreads) above += key(j) > edge;
  const int ties = want - total(above);
  int done = 0, equal = 0;
  for (int j0 = 0; j0 < early; j0 += kPagedThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < early ? key(j) : 0u;
    auto before = [&](bool f, int* all) {  // of the threads in front of this one
      const uint64_t m = __ballot(f);
      __syncthreads();
      if (lane == 0) red[wv] = __popcll(m);
      __syncthreads();
      int x = __popcll(m & ((1ull << lane) - 1));
      for (int w = 0; w < wv; ++w) x += red[w];
      *all = red[0] + red[1] + red[2] + red[3];
      return x;
    };
    int all;
    const bool tie = j < early && k == edge;
    const int rank = equal + before(tie, &all);
    equal += all;
    const bool take = j < early && (k > edge || (tie && rank < ties));
    const int at = done + before(take, &all);
    done += all;
    if (take) kept[at] = j;
  }
  for (int j = tid; j < a.recent; j += kPagedThreads) kept[want + j] = early + j;
}

// Sixteen bytes of a kept token's key and value a thread.
template <int D>
__global__ __launch_bounds__(kPagedThreads) void paged_copy_kernel(EvictArgs a) {
  constexpr int CH = D / 8, TOK = kPagedThreads / CH;
  const int h = blockIdx.y, b = blockIdx.z, c = threadIdx.x % CH;
  const int j = blockIdx.x * TOK + threadIdx.x / CH, n = a.new_lengths[b];
  if (j >= n) return;
  const int64_t src = a.c.token(b, a.kept[((int64_t)b * a.c.nkv + h) * a.keep + j], h);
  const int64_t page = a.new_table[(int64_t)b * a.new_width + (j >> a.c.log2s)];
  if (src < 0 || (uint64_t)page >= (uint64_t)a.c.pages) return;
  const int64_t dst = ((page * a.c.nkv + h) << a.c.log2s) + (j & ((1 << a.c.log2s) - 1));
  *reinterpret_cast<u32x4*>(a.c.k + dst * D + c * 8) = *reinterpret_cast<const u32x4*>(a.c.k + src * D + c * 8);
  *reinterpret_cast<u32x4*>(a.c.v + dst * D + c * 8) = *reinterpret_cast<const u32x4*>(a.c.v + src * D + c * 8);
  if (c == 0) a.c.weight[dst] = a.c.weight[src];
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

extern "C" size_t w4_paged_attention_workspace_bytes(int64_t rows, int64_t num_heads, int64_t kv_heads,
                                                     int64_t head_dim) {
  (void)rows, (void)num_heads, (void)kv_heads, (void)head_dim;
  return 0;
}

extern "C" int w4_paged_attention(const w4_paged_cache* cache, int dtype, const void* q, const void* k, const void* v,
                                  int64_t stride_q, int64_t stride_k, int64_t stride_v, int64_t num_heads,
                                  const int32_t* lengths, const int32_t* positions, const float* cos,
                                  const float* sin, int64_t angles, void* out, float* scores, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  (void)workspace, (void)workspace_bytes;
  if (const int rc = check_cache(cache, dtype, "w4_paged_attention")) return rc;
  if (num_heads < 1 || num_heads % cache->kv_heads || num_heads / cache->kv_heads > 1024 || angles < 1)
    return fail(W4_ERR_INVALID, "w4_paged_attention: %lld query heads on %lld key-value heads, %lld angles",
                (long long)num_heads, (long long)cache->kv_heads, (long long)angles);
  if (cache->rows == 0) return W4_OK;
  if (!q || !k || !v || !lengths || !positions || !cos || !sin || !out || (cache->weight && !scores))
    return fail(W4_ERR_INVALID, "w4_paged_attention: null pointer");
  if (!rows_ok(q, stride_q) || !rows_ok(k, stride_k) || !rows_ok(v, stride_v) ||
      ((uintptr_t)cos | (uintptr_t)sin | (uintptr_t)out | (uintptr_t)scores) % 16)
    return fail(W4_ERR_INVALID, "w4_paged_attention: operands must be 16-byte aligned, row strides multiples of 8");
  w4::PagedAttnArgs a{};
  a.c = view_of(cache);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.stride_q = stride_q, a.stride_k = stride_k, a.stride_v = stride_v, a.angles = angles;
  a.lengths = lengths, a.positions = positions, a.cos = cos, a.sin = sin;
  a.out = static_cast<uint16_t*>(out);
  a.scale = 1.f / sqrtf((float)cache->head_dim);
  a.g = (int)(num_heads / cache->kv_heads);
  const dim3 grid((unsigned)cache->kv_heads, (unsigned)cache->rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define W4_ATTN(DT, D) w4::paged_attention_kernel<DT, D><<<grid, w4::kPagedThreads, 0, st>>>(a)
  if (dtype == W4_DTYPE_BF16) {
    if (cache->head_dim == 64) W4_ATTN(W4_DTYPE_BF16, 64);
    else W4_ATTN(W4_DTYPE_BF16, 128);
  } else {
    if (cache->head_dim == 64) W4_ATTN(W4_DTYPE_FP16, 64);
    else W4_ATTN(W4_DTYPE_FP16, 128);
  }
#undef W4_ATTN
  return check_launch("w4_paged_attention");
}

extern "C" int w4_paged_evict(const w4_paged_cache* cache, int dtype, const int32_t* lengths,
                              const int32_t* new_table, int64_t new_width, int64_t keep, int64_t recent,
                              int32_t* kept, int32_t* new_lengths, void* stream) {
  clear_error();
  if (const int rc = check_cache(cache, dtype, "w4_paged_evict")) return rc;
  if (keep < 1 || recent < 0 || recent > keep || new_width < 1 || new_width > (1ll << 30) ||
      new_width * cache->page_size >= (1ll << 30) || keep > new_width * cache->page_size)
    return fail(W4_ERR_INVALID, "w4_paged_evict: keep %lld with the last %lld in %lld pages of %lld", (long long)keep,
                (long long)recent, (long long)new_width, (long long)cache->page_size);
  if (cache->rows == 0) return W4_OK;
  if (!cache->weight || !lengths || !new_table || !kept || !new_lengths)
    return fail(W4_ERR_INVALID, "w4_paged_evict: null pointer");
  w4::EvictArgs a{view_of(cache), lengths, new_table, kept, new_lengths, (int)new_width, (int)keep, (int)recent};
  hipStream_t st = static_cast<hipStream_t>(stream);
  w4::paged_select_kernel<<<dim3((unsigned)cache->kv_heads, (unsigned)cache->rows), w4::kPagedThreads, 0, st>>>(a);
  if (const int rc = check_launch("w4_paged_evict (select)")) return rc;
  const int tok = w4::kPagedThreads / (int)(cache->head_dim / 8);
  const dim3 grid((unsigned)((keep + tok - 1) / tok), (unsigned)cache->kv_heads, (unsigned)cache->rows);
  if (cache->head_dim == 64) w4::paged_copy_kernel<64><<<grid, w4::kPagedThreads, 0, st>>>(a);
  else w4::paged_copy_kernel<128><<<grid, w4::kPagedThreads, 0, st>>>(a);
  return check_launch("w4_paged_evict (copy)");
}
