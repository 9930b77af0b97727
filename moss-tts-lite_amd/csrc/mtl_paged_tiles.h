// What the kernels that attend over pages share: loads of tiles through buffer descriptors, matrix
// products, weights in two terms, and the store of an output.
#pragma once

#include "mtl_paged_pool.h"

namespace mtl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;               // positions a wave takes at a time
constexpr int64_t kMaxPositions = 1 << 30;      // of one sequence: they fit an int with room
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A lane's 16, 8 or 4 bytes of 16 rows that begin at a base, through a buffer descriptor: the
// descriptor's length lets rows that are not there be read as 0, whatever lies behind them, so
// every load of a tile can be issued without a condition (under a condition the compiler waits
// for all loads in flight where its paths join).
// K and V are read once: loads that leave no trace in the caches read 7.1 TB/s here, others 6.4.
// With more than 16 query heads to a kv head its rows are read again, and the loads leave a trace.
typedef __amdgpu_buffer_rsrc_t Rsrc;

__device__ __forceinline__ Rsrc rows_at(const char* base, int bytes) {
  // the same in all lanes, which the compiler does not see everywhere
  const uint64_t b = reinterpret_cast<uintptr_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0,
      __builtin_amdgcn_readfirstlane(bytes), 0x00027000);
}

template <bool ONCE>
__device__ __forceinline__ void load_row(Rsrc rows, int offset, uint32_t (&x)[4]) {
  const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, ONCE ? 2 : 0);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <bool ONCE>
__device__ __forceinline__ void load_row(Rsrc rows, int offset, uint32_t (&x)[2]) {
  const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, ONCE ? 2 : 0);
  x[0] = v.x; x[1] = v.y;
}
template <bool ONCE>
__device__ __forceinline__ void load_row(Rsrc rows, int offset, uint32_t (&x)[1]) {
  x[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, ONCE ? 2 : 0);
}

// x as a value that the compiler forms anew from here on, and does not keep over a loop before.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// p[i] for an i that is the same in all lanes, as a scalar load: a vector load would have the
// wave wait for the K and V in flight before it.
template <class T>
__device__ __forceinline__ T uniform_load(const T* p, int64_t i) {
  typedef const T __attribute__((address_space(4)))* Constant;
  return ((Constant)(uintptr_t)p)[i];
}

template <int QT>
__device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) {
  if (QT == MTL_T_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Two e4m3 elements of x (the upper half's with HI) as two of the rows' type; exact.
template <int QT, bool HI>
__device__ __forceinline__ uint32_t widen(uint32_t x) {
  if (QT == MTL_T_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, HI));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HI));
}

// Two weights in the rows' type, and what is left of them.
template <int QT>
__device__ __forceinline__ void two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
  if (QT == MTL_T_BF16) {
    hi = cvt_pk_bf16(a, b);
    lo = cvt_pk_bf16(a - lo_bf(hi), b - hi_bf(hi));
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    const auto r = __builtin_amdgcn_cvt_pkrtz(a - (float)h.x, b - (float)h.y);
    lo = __builtin_bit_cast(uint32_t, r);
  }
}

template <int QT>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  return to_elem<QT>(a) | to_elem<QT>(b) << 16;
}

__device__ __forceinline__ int clamp_len(int32_t len, int64_t cap) {
  return len < 0 ? 0 : (int)(len < cap ? len : cap);
}

// What weights are multiplied with as they enter the product, whose sums carry it to the output: in
// f16 2^15 (the largest weight is 1, f16 ends at 65504 and 2^-24).  As they are, weights more than
// 16.6 nats below the largest would be 0 in both terms and the others lose up to 2^-24, while
// their sum counts them in full.
template <int QT>
constexpr float kLift = QT == MTL_T_F16 ? 32768.f : 1.f;

// The output of one query head of one sequence from its sum o (4 dims), base-2 maximum and
// weights' sum.
template <int QT, int D>
__device__ __forceinline__ void write_out(uint16_t* __restrict__ out, float* __restrict__ lse,
                                          int64_t head, int d, floatx4 o, float top, float sum,
                                          float vs) {
  const float f = sum == 0.f ? 0.f : vs / sum * (1.f / kLift<QT>);
  *reinterpret_cast<u32x2*>(out + head * D + d) =
      u32x2{pack_out<QT>(o[0] * f, o[1] * f), pack_out<QT>(o[2] * f, o[3] * f)};
  if (lse && d == 0)
    lse[head] = sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace mtl
