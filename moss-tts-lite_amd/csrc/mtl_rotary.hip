// RMSNorm of each head of q and k and their rotation by position, in one pass (gfx950).
//
// Memory bounds it: q and k are read and written once.  A row's angles are worth about 30 fp32 and
// 10 fp64 operations each, more than all else that is done to a head, and all heads of a row share
// them: a wave takes a row, computes each cosine and sine once (a lane an angle), and passes them
// on through LDS; then groups of G lanes take heads, 8 dims a lane.
//
// The angle: the frequency in turns as two doubles, times the position, less its whole turns; the
// product's rounding comes back from an fma.  What is left is exact to 2^-50 of a turn for any
// position below 2^53, and float32 from there on.
//
// Measured (a copy moves 4.9 TB/s): 16 000 rows of 32 + 8 heads of 128 in bf16, 328 MB in and out,
// 72 us, 4.5 TB/s; 3300 rows, 68 MB, which stays in the last cache, 13 us, 5.1 TB/s; 18 rows 4 us,
// where a launch and two trips to the memory (position and frequencies, heads) are all there is.
#include "mtl_common.h"
#include "mtl_paged.h"
#include "mtl_rotary.h"

namespace mtl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRotaryWaves = 4;
constexpr int kMaxHeadDim = 512;
// Up to so many rows every wave's worth of heads gets a wave of its own, which makes the angles anew.
// Both sides measured in us, 32 + 8 heads of 128 (of 256): 1 row 3.3 (8.0 by one wave a row), 256
// 4.6 (9.5), 1024 8.7 (10.7), 2048 14.0 (13.9); of 256 15.8 (21.4) at 1024, 26.9 (24.6) at 2048.
constexpr int kFewRows = 1024;

struct RotaryHeads {
  const uint16_t* x;
  int64_t x_row, x_head;
  uint16_t* out;
  int64_t out_row, out_head;
  const uint16_t* norm;
  int heads;
};

template <int T>
__device__ __forceinline__ void unpack8(u32x4 v, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = T == MTL_T_BF16 ? lo_bf(v[j]) : f16_to_f32(v[j] & 0xffffu);
    x[2 * j + 1] = T == MTL_T_BF16 ? hi_bf(v[j]) : f16_to_f32(v[j] >> 16);
  }
}

template <int T>
__device__ __forceinline__ uint32_t round16(float x) {
  return T == MTL_T_BF16 ? f32_to_bf16(x)
                         : (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)x);
}

template <int T>
__device__ __forceinline__ float element(const uint16_t* p) {
  return T == MTL_T_BF16 ? bf16_to_f32(*p) : f16_to_f32(*p);
}

__device__ __forceinline__ u32x4 load16(const uint16_t* p) {
  return *reinterpret_cast<const u32x4*>(p);
}

// cos and sin of pos * f radians, times amplitude.
__device__ __forceinline__ float2 turn(double pos, double f, float amplitude) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;   // 1 / (2 pi)
  const double t = f * kHi, t_lo = fma(f, kHi, -t) + f * kLo;
  const double p = pos * t, p_lo = fma(pos, t, -p) + pos * t_lo;
  const float part = (float)((p - rint(p)) + p_lo);
  float s, c;
  sincospif(2.f * part, &s, &c);
  return make_float2(amplitude * c, amplitude * s);
}

// MODE 0: pairs (2t, 2t + 1); 1: pairs half a rotated part apart, whole lanes; 2: the same where
// half the rotated part is no multiple of 8, and a lane reads its partners by themselves.
template <int T, int G, int MODE>
__global__ void __launch_bounds__(kRotaryWaves * 64) qk_rotary_kernel(
    RotaryHeads q, RotaryHeads k, int64_t rows, int dim, const int64_t* __restrict__ positions,
    const double* __restrict__ freqs, int half, float amplitude, float eps) {
  extern __shared__ float2 turns[];               // [kRotaryWaves][half]
  constexpr int GROUPS = 64 / G;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = (int64_t)blockIdx.x * kRotaryWaves + wave;
  const int64_t pos = row < rows ? positions[row] : -1;
  float2* mine = turns + wave * half;
  if (pos >= 0)
    for (int t = lane; t < half; t += 64) mine[t] = turn((double)pos, freqs[t], amplitude);
  __syncthreads();
  if (row >= rows) return;
  const int l = lane % G, d = 8 * l;
  const bool in = d < dim;
  float c[8], s[8];                               // s carries the sign of the pair's first dim
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int at = d + j;
    const int t = MODE == 0 ? at >> 1 : at < half ? at : at - half;
    const bool first = MODE == 0 ? !(at & 1) : at < half;
    c[j] = 1.f;
    s[j] = 0.f;
    if (at < 2 * half && pos >= 0) {
      const float2 cs = mine[t];
      c[j] = cs.x;
      s[j] = first ? -cs.y : cs.y;
    }
  }
  const int heads = q.heads + k.heads, each = (heads + gridDim.y - 1) / gridDim.y;
  const int begin = blockIdx.y * each, end = min(heads, begin + each);
  for (int h0 = begin; h0 < end; h0 += GROUPS) {
    const int h = h0 + lane / G;
    const bool there = h < end && in, is_q = h < q.heads;
    const uint16_t* x = is_q ? q.x + row * q.x_row + h * q.x_head
                             : k.x + row * k.x_row + (h - q.heads) * k.x_head;
    uint16_t* out = is_q ? q.out + row * q.out_row + h * q.out_head
                         : k.out + row * k.out_row + (h - q.heads) * k.out_head;
    const uint16_t* norm = is_q ? q.norm : k.norm;
    if (pos < 0) {
      if (there && out != x) *reinterpret_cast<u32x4*>(out + d) = u32x4{0, 0, 0, 0};
      continue;
    }
    float y[8] = {}, w[8], pair[8];
    if (there) unpack8<T>(load16(x + d), y);
    if (MODE == 2 && there) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = d + j;
        pair[j] = at < 2 * half ? element<T>(x + (at < half ? at + half : at - half)) : 0.f;
      }
    }
    // all lanes of a wave take part in the sum
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
    ss = group_sum_valu<G>(ss);
    if (norm && there) {
      const float r = rsqrtf(ss / (float)dim + eps);
      unpack8<T>(load16(norm + d), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= r * w[j];
      if (MODE == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = d + j;
          if (at < 2 * half)
            pair[j] *= r * element<T>(norm + (at < half ? at + half : at - half));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (MODE == 0) pair[j] = y[j ^ 1];
      if (MODE == 1) {
        const int other = d < half ? l + half / 8 : l - half / 8;
        pair[j] = __shfl(y[j], (lane & ~(G - 1)) + (other & (G - 1)));
      }
    }
    if (!there) continue;
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      e[j] = round16<T>(d + j < 2 * half ? y[j] * c[j] + pair[j] * s[j] : y[j]);
    *reinterpret_cast<u32x4*>(out + d) = u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16,
                                               e[4] | e[5] << 16, e[6] | e[7] << 16};
  }
}

static bool heads_aligned(const mtl_rotary_heads& h) {
  return h.x_row % 8 == 0 && h.x_head % 8 == 0 && h.out_row % 8 == 0 && h.out_head % 8 == 0 &&
         aligned16(h.x) && aligned16(h.out) && aligned16(h.norm);
}

static RotaryHeads kernel_heads(const mtl_rotary_heads& h) {
  return RotaryHeads{static_cast<const uint16_t*>(h.x), h.x_row, h.x_head,
                     static_cast<uint16_t*>(h.out), h.out_row, h.out_head,
                     static_cast<const uint16_t*>(h.norm), h.heads};
}

template <int T, int G>
static void launch_rotary(const RotaryHeads& q, const RotaryHeads& k, int64_t rows, int dim,
                          const int64_t* positions, const double* freqs, int half,
                          bool interleaved, float amplitude, float eps, hipStream_t stream) {
  const int heads = q.heads + k.heads;
  const dim3 grid((unsigned)((rows + kRotaryWaves - 1) / kRotaryWaves),
                  rows <= kFewRows ? min(1024, (heads + 64 / G - 1) / (64 / G)) : 1);
  const size_t lds = (size_t)kRotaryWaves * half * sizeof(float2);
#define MTL_RUN(MODE)                                                                          \
  qk_rotary_kernel<T, G, MODE><<<grid, kRotaryWaves * 64, lds, stream>>>(                      \
      q, k, rows, dim, positions, freqs, half, amplitude, eps)
  if (interleaved)
    MTL_RUN(0);
  else if (half % 8 == 0)
    MTL_RUN(1);
  else
    MTL_RUN(2);
#undef MTL_RUN
}

}  // namespace mtl

using namespace mtl;

extern "C" int mtl_qk_rotary(const mtl_rotary_heads* q, const mtl_rotary_heads* k, int64_t rows,
                             int32_t head_dim, const int64_t* positions, const double* freqs,
                             int32_t turned, int32_t interleaved, float amplitude, float eps,
                             int32_t type, void* stream) {
  if (!q || !k || rows < 0 || q->heads < 0 || k->heads < 0) return MTL_ERR_INVALID_ARG;
  if (type != MTL_T_BF16 && type != MTL_T_F16) return MTL_ERR_UNSUPPORTED;
  if (head_dim < 8 || head_dim > kMaxHeadDim || head_dim % 8 || turned < 0 || turned % 2 ||
      turned > head_dim)
    return MTL_ERR_SHAPE;
  // the launch's threads, within 32 bits
  if (rows > (int64_t)1 << 25 || q->heads > 65535 || k->heads > 65535) return MTL_ERR_SHAPE;
  if (rows == 0 || q->heads + k->heads == 0) return MTL_OK;
  if (!positions || (turned && !freqs) || (q->heads && (!q->x || !q->out)) ||
      (k->heads && (!k->x || !k->out)))
    return MTL_ERR_INVALID_ARG;
  for (const mtl_rotary_heads* h : {q, k}) {
    if (h->heads == 0) continue;
    if (!heads_aligned(*h)) return MTL_ERR_ALIGN;
    if (h->x == h->out && (h->x_row != h->out_row || h->x_head != h->out_head))
      return MTL_ERR_INVALID_ARG;
  }
  const RotaryHeads a = kernel_heads(*q), b = kernel_heads(*k);
#define MTL_ROTARY(T, G)                                                                      \
  launch_rotary<T, G>(a, b, rows, head_dim, positions, freqs, turned / 2, interleaved != 0,    \
                      amplitude, eps, (hipStream_t)stream)
#define MTL_ROTARY_TYPES(G)                                                                   \
  do {                                                                                        \
    if (type == MTL_T_BF16) MTL_ROTARY(MTL_T_BF16, G);                                        \
    else MTL_ROTARY(MTL_T_F16, G);                                                            \
  } while (0)
  if (head_dim <= 64) MTL_ROTARY_TYPES(8);
  else if (head_dim <= 128) MTL_ROTARY_TYPES(16);
  else if (head_dim <= 256) MTL_ROTARY_TYPES(32);
  else MTL_ROTARY_TYPES(64);
#undef MTL_ROTARY_TYPES
#undef MTL_ROTARY
  return launch_status();
}
