/*
 * mtl_rotary.h -- C ABI of the rotation of queries and keys by their positions (MI355X /
 * gfx950), with the RMSNorm of each head in the same pass.  Same conventions as mtl_gptq.h:
 * 0 = MTL_OK, negative = MTL_ERR_*, raw device pointers, a hipStream_t, no allocation or host
 * synchronisation, capturable into a hipGraph.  The structures below are host memory, read
 * during the call.
 *
 * The reference rotates half of a whole head's dims against the other half out of bf16 tables
 * (moss_tts_lite/model.py:34-44,115-124), which mtl_decode.h does; these entries are for other
 * layouts, parts of a head, scaled frequencies and positions too far for a table.
 */
#ifndef MTL_ROTARY_H
#define MTL_ROTARY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The heads of q or of k: [rows, heads, head_dim], strides in elements.  The elements of a head
 * are adjacent; bases are 16-byte aligned, strides multiples of 8. */
typedef struct mtl_rotary_heads {
  const void* x;
  int64_t x_row, x_head;
  void* out;                          /* may be x, with the same strides: in place */
  int64_t out_row, out_head;
  const void* norm;                   /* [head_dim] of type, 16-byte aligned; NULL: no norm */
  int32_t heads;                      /* 0: there are none */
} mtl_rotary_heads;

/*
 * Row r, each head x of it:  y = norm x / sqrt(mean x^2 + eps) (y = x without norm), and with
 * a_t = positions[r] * freqs[t], t < turned / 2, each pair of dims (u, v) of y becomes
 *   (amplitude (u cos a_t - v sin a_t), amplitude (v cos a_t + u sin a_t)).
 * The pairs are dims (t, t + turned / 2), or (2t, 2t + 1) with interleaved.  Dims from turned on
 * are y as it is.  fp32 (angles: the product in 64 bits, reduced to a part of a turn there), one
 * rounding to type.
 *   positions  int64 [rows] (device), below 2^53.  A negative one is padding: out 0, or in
 *              place x as it is
 *   freqs      float64 [turned / 2] (device), radians a position
 *   head_dim   a multiple of 8, 8 .. 512; turned even, 0 .. head_dim
 *   type       MTL_T_BF16 or MTL_T_F16 (mtl_paged.h)
 * out of q and of k share no memory with each other or, but in place, with x.
 */
int mtl_qk_rotary(const mtl_rotary_heads* q, const mtl_rotary_heads* k, int64_t rows,
                  int32_t head_dim, const int64_t* positions, const double* freqs, int32_t turned,
                  int32_t interleaved, float amplitude, float eps, int32_t type, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MTL_ROTARY_H */
