// The write of new tokens into the pages of a key-value cache (gfx950): q/k RMSNorm, RoPE and the
// stored element type.
#include "mtl_paged_pool.h"

namespace mtl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight elements of 2 bytes, as float32.
template <int T>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&x)[8]) {
  const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = T == MTL_T_BF16 ? lo_bf(v[j]) : f16_to_f32(v[j] & 0xffffu);
    x[2 * j + 1] = T == MTL_T_BF16 ? hi_bf(v[j]) : f16_to_f32(v[j] >> 16);
  }
}

template <int T>
__device__ __forceinline__ void load8_table(const void* p, int f32, int64_t i, float (&x)[8]) {
  if (!f32) return load8<T>(p, i, x);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4 * j);
    x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
  }
}

template <int T>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&x)[8]) {
  uint32_t e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = to_elem<T>(x[j]);
  if (T == MTL_T_E4M3)
    *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p) + i) =
        u32x2{e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24, e[4] | e[5] << 8 | e[6] << 16 | e[7] << 24};
  else
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) =
        u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
}

// ----------------------------------------------------------------------------------
// Write: y = w x / sqrt(mean x^2 + eps), r = y cos + rotate_half(y) sin, in fp32 until the
// store.  A workgroup takes a row, a group of D / 8 lanes a head of q | k | v, 8 dims a lane;
// the dims that RoPE pairs, t and t + D/2, lie half a group apart.  A lane meets the same dims
// in every head, so it reads the row's cos and sin once.  Bound by memory: 3300 rows of 48
// heads of 128 into 8-bit pages (75 MB) 16.8 us, 4.5 TB/s (a lane with one pair of dims 45;
// all heads' rows loaded ahead 20; workgroups of 128 or 512 threads 19.6, 20.4).
// ----------------------------------------------------------------------------------
template <int T, int KT, int D>
__global__ void __launch_bounds__(256) paged_write_kernel(
    const void* __restrict__ qkv, int64_t ldq, PagePool pool, const int32_t* __restrict__ table,
    int64_t ldt, int64_t width, int64_t seqs, const int64_t* __restrict__ positions,
    const int32_t* __restrict__ row_seq, const void* __restrict__ q_norm,
    const void* __restrict__ k_norm, const void* __restrict__ cos_tab,
    const void* __restrict__ sin_tab, int rope_f32, int64_t rope_rows, float eps, int n_heads,
    void* __restrict__ q_out) {
  constexpr int LANES = D / 8, HEADS = 256 / LANES;
  const int lane = threadIdx.x % LANES, d = 8 * lane;
  const int64_t r = blockIdx.x, pos = positions[r];
  const bool there = pos >= 0 && (!cos_tab || pos < rope_rows);
  const int64_t s = row_seq ? row_seq[r] : r;
  int32_t page = -1;
  if (there && s >= 0 && s < seqs && pos < width * pool.page_size)
    page = table[s * ldt + pos / pool.page_size];
  const bool write = (uint32_t)page < (uint32_t)pool.pages;
  const int64_t in_page = pos & (pool.page_size - 1);
  float c[8], sn[8];
  if (cos_tab && there) {
    load8_table<T>(cos_tab, rope_f32, pos * D + d, c);
    load8_table<T>(sin_tab, rope_f32, pos * D + d, sn);
  }
  const int heads = n_heads + 2 * pool.kv_heads;
  for (int h = blockIdx.y * HEADS + threadIdx.x / LANES; h < heads; h += gridDim.y * HEADS) {
    const bool is_q = h < n_heads, is_v = h >= n_heads + pool.kv_heads;
    const int kvh = is_v ? h - n_heads - pool.kv_heads : h - n_heads;
    if (!is_q && !write) continue;
    float x[8];
    load8<T>(qkv, r * ldq + (int64_t)h * D + d, x);
    if (!is_v) {
      const void* w = is_q ? q_norm : k_norm;
      if (w) {
        float ss = 0.f, g[8];
        load8<T>(w, d, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
        ss = group_sum_valu<LANES>(ss);          // whole groups are here, or not
        const float rr = rsqrtf(ss / (float)D + eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= rr * g[j];
      }
      if (cos_tab && there) {
        const float sign = lane < LANES / 2 ? -1.f : 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = LANES == 16 ? dpp_f32<kDppRor8>(x[j]) : __shfl_xor(x[j], LANES / 2);
          x[j] = x[j] * c[j] + sign * y * sn[j];
        }
      }
    }
    if (is_q) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = there ? x[j] : 0.f;
      store8<T>(q_out, (r * n_heads + h) * (int64_t)D + d, x);
      continue;
    }
    const float* scale = is_v ? pool.v_scale : pool.k_scale;
    if (KT == MTL_T_E4M3 && scale) {
      // x / by rounded once: the product with the rounded reciprocal, corrected by the remainder
      // (a quotient past 1e30, an infinity or a NaN is stored as 448 or NaN without it).  The
      // reciprocal and the remainder need a scale far from float32's ends; others are divided by.
      const float by = scale[kvh], inv = 1.f / by;
      if (fabsf(by) > 0x1p-100f && fabsf(by) < 0x1p100f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float q = x[j] * inv;
          x[j] = fabsf(q) < 1e30f ? fmaf(fmaf(-q, by, x[j]), inv, q) : q;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] /= by;
      }
    }
    if (is_v)
      store8<KT>(pool.v, page * pool.v_page + kvh * pool.v_head + in_page * pool.v_token + d, x);
    else
      store8<KT>(pool.k, page * pool.k_page + kvh * pool.k_head + in_page * pool.k_token + d, x);
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
  const int64_t heads = (int64_t)n_heads + 2 * (int64_t)pool->kv_heads;
  if (heads > 65535 || ldq < heads * pool->head_dim || rows > UINT32_MAX / 256)
    return MTL_ERR_SHAPE;                // the launch's threads, within 32 bits
  if (rows == 0) return MTL_OK;
  if (!qkv || !positions || !q_out) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || !aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm) ||
      !aligned16(k_norm) || !aligned16(cos_tab) || !aligned16(sin_tab))
    return MTL_ERR_ALIGN;
  // Few rows: a workgroup for each 256 lanes' heads, so that a step's rows reach more CUs; many:
  // one for all heads of a row, which reads cos and sin once.  Rows of 48 heads of 128 split over
  // the heads and whole, in us: 16 rows 2.8 and 4.0, 512 rows 5.4 and 5.8, 1000 rows 8.4 and 8.3,
  // 3300 rows 18.3 and 16.9.  Where the rule changes sides, 512 rows split and 513 whole: 12 heads
  // 3.2 and 3.3, 80 heads 6.9 and 7.7, 128 heads 9.2 and 11.3, 44 heads of 64 4.1 and 4.3.
  const int64_t passes = (heads * (pool->head_dim / 8) + 255) / 256;
  const dim3 grid((unsigned)rows, rows <= 512 ? (unsigned)passes : 1);
#define MTL_RUN(T, KT, D)                                                                    \
  paged_write_kernel<T, KT, D><<<grid, 256, 0, (hipStream_t)stream>>>(                        \
      qkv, ldq, p, table->table, table->ld, table->width, table->seqs, positions, row_seq,   \
      q_norm, k_norm, cos_tab, sin_tab, rope_f32, rope_rows, eps, n_heads, q_out)
  MTL_PAGED_CASES(MTL_RUN, type, pool->type, pool->head_dim);
#undef MTL_RUN
  return launch_status();
}
