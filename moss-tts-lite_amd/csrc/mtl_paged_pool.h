// What the kernels over a paged key-value cache share: the pool's form, element conversions and
// the argument rules.
#pragma once

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

// Inclusive sum over the lanes of a wave (all active).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

inline bool page_size_ok(int32_t ps) {
  return ps == 16 || ps == 32 || ps == 64 || ps == 128 || ps == 256;
}

// The argument rules both entries share; fills the kernels' form of the pool.
inline int check_pool(const mtl_page_pool* p, const mtl_page_table* t, int32_t type, PagePool& o) {
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
  // rows of a head must not overlap: a token's stride holds a row
  if (p->k_token < p->head_dim || p->v_token < p->head_dim) return MTL_ERR_SHAPE;
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
