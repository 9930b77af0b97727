// Paged key-value cache (gfx950): attention of one new token a sequence over its pages, and the
// write of new tokens into pages (q/k RMSNorm, RoPE, the stored element type).
#include "mtl_common.h"
#include "mtl_paged.h"

namespace mtl {

// One layer's pages as the kernels take them (strides in elements).
struct PagePool {
  void* k;
  void* v;
  int64_t k_page, k_head, k_token, v_page, v_head, v_token;
  const float* k_scale;
  const float* v_scale;
  int pages, kv_heads, page_size;
};

template <int TYPE>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if (TYPE == MTL_T_E4M3) {
    const uint32_t b = static_cast<const uint8_t*>(p)[i];
    const bf16x2_t v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
    return (float)v.x;
  }
  const uint32_t b = static_cast<const uint16_t*>(p)[i];
  return TYPE == MTL_T_BF16 ? bf16_to_f32(b) : f16_to_f32(b);
}

// float32 -> one stored element, to nearest even; e4m3 limited to +-448 (a NaN stays one).
template <int TYPE>
__device__ __forceinline__ uint32_t to_elem(float x) {
  if (TYPE == MTL_T_E4M3) {
    x = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xffu;
  }
  return TYPE == MTL_T_BF16 ? f32_to_bf16(x)
                            : (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)x);
}

template <int TYPE>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float x) {
  if (TYPE == MTL_T_E4M3)
    static_cast<uint8_t*>(p)[i] = (uint8_t)to_elem<TYPE>(x);
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)to_elem<TYPE>(x);
}

// ----------------------------------------------------------------------------------
// Attention: one wave per (sequence, query head), one position after the other with the
// running maximum m and sum l of the softmax: acc = acc * exp(m - m') + exp(s - m') v.
// ----------------------------------------------------------------------------------
template <int QT, int KT, int D>
__global__ void __launch_bounds__(64) paged_attention_kernel(
    const void* __restrict__ q, int64_t ldq, int64_t ldh, PagePool pool,
    const int32_t* __restrict__ table, int64_t ldt, int64_t width,
    const int32_t* __restrict__ lens, int n_heads, float scale, void* __restrict__ out,
    float* __restrict__ lse) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x, h = blockIdx.x;
  const int64_t b = blockIdx.y;
  const int kvh = h / (n_heads / pool.kv_heads);
  const float ks = pool.k_scale ? pool.k_scale[kvh] : 1.f;
  const float vs = pool.v_scale ? pool.v_scale[kvh] : 1.f;
  const int64_t cap = width * pool.page_size;
  const int64_t len = lens[b] < cap ? lens[b] : cap;
  float qv[E], acc[E], m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = load_elem<QT>(q, b * ldq + h * ldh + lane * E + e);
    acc[e] = 0.f;
  }
  for (int64_t p = 0; p < len; ++p) {
    const int32_t page = table[b * ldt + p / pool.page_size];
    if ((uint32_t)page >= (uint32_t)pool.pages) continue;
    const int64_t row = p % pool.page_size;
    const int64_t ko = page * pool.k_page + kvh * pool.k_head + row * pool.k_token + lane * E;
    const int64_t vo = page * pool.v_page + kvh * pool.v_head + row * pool.v_token + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], load_elem<KT>(pool.k, ko + e), s);
    s = wave_sum(s) * (scale * ks);
    const float mn = fmaxf(m, s);
    const float mu = mn == -__builtin_inff() ? 0.f : mn;
    const float a = expf(m - mu), w = expf(s - mu);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, load_elem<KT>(pool.v, vo + e), acc[e] * a);
    m = mn;
  }
  const float r = l == 0.f ? 0.f : vs / l;
#pragma unroll
  for (int e = 0; e < E; ++e)
    store_elem<QT>(out, (b * n_heads + h) * (int64_t)D + lane * E + e, acc[e] * r);
  if (lse && lane == 0)
    lse[b * n_heads + h] = l == 0.f ? -__builtin_inff()
                                    : (m == -__builtin_inff() ? 0.f : m) + logf(l);
}

// ----------------------------------------------------------------------------------
// Write: one wave per (row, head of q | k | v); a lane holds the pair of dims that RoPE
// rotates (t, t + D/2).  fp32 until the store.
// ----------------------------------------------------------------------------------
template <int T, int KT, int D>
__global__ void __launch_bounds__(64) paged_write_kernel(
    const void* __restrict__ qkv, int64_t ldq, PagePool pool, const int32_t* __restrict__ table,
    int64_t ldt, int64_t width, int64_t seqs, const int64_t* __restrict__ positions,
    const int32_t* __restrict__ row_seq, const void* __restrict__ q_norm,
    const void* __restrict__ k_norm, const void* __restrict__ cos_tab,
    const void* __restrict__ sin_tab, int rope_f32, int64_t rope_rows, float eps, int n_heads,
    void* __restrict__ q_out) {
  constexpr int HALF = D / 2;
  const int h = blockIdx.x, t = threadIdx.x & (HALF - 1);
  const int64_t r = blockIdx.y;
  const int64_t pos = positions[r];
  const bool rows_ok = pos >= 0 && (!cos_tab || pos < rope_rows);
  const int which = h < n_heads ? 0 : h < n_heads + pool.kv_heads ? 1 : 2;   // q, k, v
  float x0 = load_elem<T>(qkv, r * ldq + (int64_t)h * D + t);
  float x1 = load_elem<T>(qkv, r * ldq + (int64_t)h * D + t + HALF);
  if (which < 2) {
    const void* w = which == 0 ? q_norm : k_norm;
    if (w) {
      float ss = threadIdx.x < HALF ? fmaf(x0, x0, x1 * x1) : 0.f;
      ss = wave_sum(ss);
      const float rr = rsqrtf(ss / (float)D + eps);
      x0 *= rr * load_elem<T>(w, t);
      x1 *= rr * load_elem<T>(w, t + HALF);
    }
    if (cos_tab && rows_ok) {
      float c[2], s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t at = pos * D + t + i * HALF;
        c[i] = rope_f32 ? static_cast<const float*>(cos_tab)[at] : load_elem<T>(cos_tab, at);
        s[i] = rope_f32 ? static_cast<const float*>(sin_tab)[at] : load_elem<T>(sin_tab, at);
      }
      const float y0 = x0 * c[0] - x1 * s[0];
      x1 = x1 * c[1] + x0 * s[1];
      x0 = y0;
    }
  }
  if (threadIdx.x >= HALF) return;
  if (which == 0) {
    const int64_t o = (r * n_heads + h) * (int64_t)D + t;
    store_elem<T>(q_out, o, rows_ok ? x0 : 0.f);
    store_elem<T>(q_out, o + HALF, rows_ok ? x1 : 0.f);
    return;
  }
  const int64_t s = row_seq ? row_seq[r] : r;
  if (!rows_ok || s < 0 || s >= seqs || pos >= width * pool.page_size) return;
  const int32_t page = table[s * ldt + pos / pool.page_size];
  if ((uint32_t)page >= (uint32_t)pool.pages) return;
  const int64_t row = pos % pool.page_size;
  if (which == 1) {
    const int kvh = h - n_heads;
    if (pool.k_scale) { x0 /= pool.k_scale[kvh]; x1 /= pool.k_scale[kvh]; }
    const int64_t o = page * pool.k_page + kvh * pool.k_head + row * pool.k_token + t;
    store_elem<KT>(pool.k, o, x0);
    store_elem<KT>(pool.k, o + HALF, x1);
  } else {
    const int kvh = h - n_heads - pool.kv_heads;
    if (pool.v_scale) { x0 /= pool.v_scale[kvh]; x1 /= pool.v_scale[kvh]; }
    const int64_t o = page * pool.v_page + kvh * pool.v_head + row * pool.v_token + t;
    store_elem<KT>(pool.v, o, x0);
    store_elem<KT>(pool.v, o + HALF, x1);
  }
}

// ----------------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------------
inline bool page_size_ok(int32_t ps) {
  return ps == 16 || ps == 32 || ps == 64 || ps == 128 || ps == 256;
}

// The argument rules both entries share; fills the kernels' form of the pool.
static int check_pool(const mtl_page_pool* p, const mtl_page_table* t, int32_t type, PagePool& o) {
  if (!p || !t || !p->k || !p->v || p->pages < 1 || p->pages > INT32_MAX || p->kv_heads < 1 ||
      t->seqs < 0 || t->width < 0 || (t->seqs > 0 && t->width > 0 && !t->table) ||
      t->ld < t->width)
    return MTL_ERR_INVALID_ARG;
  if (type != MTL_T_BF16 && type != MTL_T_F16) return MTL_ERR_UNSUPPORTED;
  if (p->type != type && p->type != MTL_T_E4M3) return MTL_ERR_UNSUPPORTED;
  if (p->type != MTL_T_E4M3 && (p->k_scale || p->v_scale)) return MTL_ERR_UNSUPPORTED;
  if ((p->head_dim != 64 && p->head_dim != 128) || !page_size_ok(p->page_size))
    return MTL_ERR_SHAPE;
  const int64_t piece = p->type == MTL_T_E4M3 ? 16 : 8;   // elements in 16 bytes
  const int64_t st[6] = {p->k_page, p->k_head, p->k_token, p->v_page, p->v_head, p->v_token};
  for (int64_t s : st)
    if (s < 0 || s % piece) return MTL_ERR_ALIGN;
  if (!aligned16(p->k) || !aligned16(p->v)) return MTL_ERR_ALIGN;
  o = PagePool{p->k, p->v, p->k_page, p->k_head, p->k_token, p->v_page, p->v_head, p->v_token,
               p->k_scale, p->v_scale, (int)p->pages, p->kv_heads, p->page_size};
  return MTL_OK;
}

// Calls F<type, page type, head_dim>.
#define MTL_PAGED_CASES(F, type, kt, d)                                                   \
  do {                                                                                    \
    const int key_ = (type) * 4 + ((kt) == MTL_T_E4M3 ? 2 : 0) + ((d) == 128 ? 1 : 0);    \
    if (key_ == 0) F(MTL_T_BF16, MTL_T_BF16, 64);                                         \
    if (key_ == 1) F(MTL_T_BF16, MTL_T_BF16, 128);                                        \
    if (key_ == 2) F(MTL_T_BF16, MTL_T_E4M3, 64);                                         \
    if (key_ == 3) F(MTL_T_BF16, MTL_T_E4M3, 128);                                        \
    if (key_ == 4) F(MTL_T_F16, MTL_T_F16, 64);                                           \
    if (key_ == 5) F(MTL_T_F16, MTL_T_F16, 128);                                          \
    if (key_ == 6) F(MTL_T_F16, MTL_T_E4M3, 64);                                          \
    if (key_ == 7) F(MTL_T_F16, MTL_T_E4M3, 128);                                         \
  } while (0)

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_paged_attention_workspace_bytes(int64_t seqs, int32_t n_heads,
                                                       int32_t kv_heads, int32_t head_dim,
                                                       int64_t width, int32_t page_size) {
  (void)seqs; (void)n_heads; (void)kv_heads; (void)head_dim; (void)width; (void)page_size;
  return 0;
}

extern "C" int mtl_paged_attention(const void* q, int64_t ldq, int64_t ldh,
                                   const mtl_page_pool* pool, const mtl_page_table* table,
                                   const int32_t* lens, int32_t n_heads, int32_t q_type,
                                   float scale, void* out, float* lse, void* workspace,
                                   int64_t ws_bytes, void* stream) {
  (void)workspace; (void)ws_bytes;
  PagePool p;
  const int st = check_pool(pool, table, q_type, p);
  if (st != MTL_OK) return st;
  if (n_heads < 1 || n_heads % pool->kv_heads) return MTL_ERR_SHAPE;
  if (table->seqs == 0) return MTL_OK;
  if (!q || !lens || !out) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || ldh % 8 || !aligned16(q)) return MTL_ERR_ALIGN;
  if (table->seqs > 65535) return MTL_ERR_SHAPE;
  const dim3 grid(n_heads, (unsigned)table->seqs);
#define MTL_RUN(T, KT, D)                                                                       \
  paged_attention_kernel<T, KT, D><<<grid, 64, 0, (hipStream_t)stream>>>(                       \
      q, ldq, ldh, p, table->table, table->ld, table->width, lens, n_heads, scale, out, lse)
  MTL_PAGED_CASES(MTL_RUN, q_type, pool->type, pool->head_dim);
#undef MTL_RUN
  return launch_status();
}

extern "C" int mtl_paged_write(const void* qkv, int64_t ldq, int64_t rows,
                               const mtl_page_pool* pool, const mtl_page_table* table,
                               const int64_t* positions, const int32_t* row_seq,
                               const void* q_norm, const void* k_norm, const void* cos_tab,
                               const void* sin_tab, int32_t rope_f32, int64_t rope_rows, float eps,
                               int32_t n_heads, int32_t type, void* q_out, void* stream) {
  PagePool p;
  const int st = check_pool(pool, table, type, p);
  if (st != MTL_OK) return st;
  if (rows < 0 || n_heads < 1 || !q_norm != !k_norm || !cos_tab != !sin_tab ||
      (cos_tab && rope_rows < 0))
    return MTL_ERR_INVALID_ARG;
  const int64_t heads = (int64_t)n_heads + 2 * pool->kv_heads;
  if (ldq < heads * pool->head_dim || rows > 65535) return MTL_ERR_SHAPE;
  if (rows == 0) return MTL_OK;
  if (!qkv || !positions || !q_out) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || !aligned16(qkv)) return MTL_ERR_ALIGN;
  const dim3 grid((unsigned)heads, (unsigned)rows);
#define MTL_RUN(T, KT, D)                                                                    \
  paged_write_kernel<T, KT, D><<<grid, 64, 0, (hipStream_t)stream>>>(                        \
      qkv, ldq, p, table->table, table->ld, table->width, table->seqs, positions, row_seq,   \
      q_norm, k_norm, cos_tab, sin_tab, rope_f32, rope_rows, eps, n_heads, q_out)
  MTL_PAGED_CASES(MTL_RUN, type, pool->type, pool->head_dim);
#undef MTL_RUN
  return launch_status();
}
