// The write of new tokens into the pages of a key-value cache (gfx950): q/k RMSNorm, RoPE and the
// stored element type.
#include "mtl_paged_pool.h"

namespace mtl {

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

}  // namespace mtl

using namespace mtl;

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
