// Attention of one new token of each sequence over a paged key-value cache (gfx950).
//
// The work is reading K and V once (2 * len * kv_heads * head_dim elements; 4 operations per
// element and query head of the group), so HBM bounds it, and what the kernel does about that:
//
// * A wave takes 32 positions at a time and holds K and V of them in registers, loaded 16 bytes
//   a lane straight from the pages; no tile passes through LDS.
// * Both products run on 16x16x32 MFMA with the positions along the product's other axis:
//   S^T[position][head] = K Q^T and O^T[dim][head] = V^T P^T, at most 16 query heads of one kv
//   head as columns.  S^T comes out with 4 positions of one head in a lane, which is the form
//   that P^T goes in with, once the 32 positions are counted in the order the lanes hold them:
//   the weights never move between lanes.  V^T needs 8 positions of one dim in a lane: a lane
//   loads 16 bytes of dims for each of its 8 positions and transposes them with v_perm.
// * The maximum and sum of the softmax run along (fp32); accumulators are rescaled only when a
//   maximum grew.  Weights enter the product as two rows-type numbers, the rounded weight and
//   what the rounding left: the output is then off by its own rounding alone (with one, by
//   1.4 times that).
// * Sequences are cut into chunks of equal length, chosen on the device from the lengths so that
//   all chunks together fill the chip; chunks of one sequence are joined by a second launch in
//   chunk order.  Short tables (at most kDirectPositions) need neither.
#include "mtl_paged_pool.h"

namespace mtl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;               // positions a wave takes at a time
constexpr int kSplitWaves = 4;
constexpr int kBlock = kTile * kSplitWaves;   // chunks are multiples of this
constexpr int kTargetChunks = 2048;     // chunks of all heads together, at most this many ...
constexpr int kDirectPositions = 1024;
constexpr int kDirectWaves = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The workspace: [groups][heads][head_dim] sums and [groups][heads][2] (maximum, sum) in fp32,
// then int2 [seqs] (first chunk, chunks), for `groups` workgroups of up to 16 query heads.
struct Split {
  int64_t groups;
  int head_tiles, tile_heads;
};

__host__ __device__ inline Split split_of(int64_t seqs, int n_heads, int kv_heads) {
  Split s;
  const int g = n_heads / kv_heads;
  s.tile_heads = g < 16 ? g : 16;
  s.head_tiles = (g + 15) / 16;
  const int64_t units = (int64_t)kv_heads * s.head_tiles;
  s.groups = (kTargetChunks / units + seqs) * units;
  return s;
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

// One chunk of one sequence for up to 16 query heads of one kv head.
template <int QT, int KT, int D, int WAVES>
struct Attend {
  static constexpr int E = KT == MTL_T_E4M3 ? 1 : 2;    // bytes of a stored element
  static constexpr int KL = D * E / 64;                 // 16-byte loads of a lane's K row
  static constexpr int QS = D / 32;                     // MFMA steps over the dims
  static constexpr int VD = D / 16;                     // dims of a lane's V pieces
  static constexpr int VW = VD * E / 4;                 // ... in dwords
  u32x4 qf[QS];
  u32x4 kf[2][KL];
  uint32_t vf[8][VW];
  floatx4 acc[VD];
  float m, l, c;                                        // c: scale to base 2
  int lane, r, g, k_lane, v_lane, k_row, v_row;

  // The pages of the tile's two halves of 16 positions; -1: none.
  struct Tile {
    int page[2];
  };

  __device__ __forceinline__ Tile pages(const int32_t* __restrict__ row, int shift, int p0, int end,
                                        int n_pages) const {
    Tile t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = p0 + 16 * h;
      int id = -1;
      if (p < end) id = row[p >> shift];
      t.page[h] = (uint32_t)id < (uint32_t)n_pages ? id : -1;
    }
    return t;
  }

  // A half without a page reads page 0 (any rows do: they are masked).  All 16 rows of a half
  // lie in its page, those past the sequence's end too.
  __device__ __forceinline__ void load_k(const PagePool& pool, const char* base, const Tile& t,
                                         int p0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int id = t.page[h] < 0 ? 0 : t.page[h];
      const char* p = base + (id * pool.k_page + ((p0 + 16 * h) & (pool.page_size - 1)) *
                                                     pool.k_token) * E;
#pragma unroll
      for (int s = 0; s < KL; ++s)
        kf[h][s] = *reinterpret_cast<const u32x4*>(p + (uint32_t)(k_lane + 64 * s));
    }
  }

  __device__ __forceinline__ void load_v(const PagePool& pool, const char* base, const Tile& t,
                                         int p0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int id = t.page[h] < 0 ? 0 : t.page[h];
      const char* p = base + (id * pool.v_page + ((p0 + 16 * h) & (pool.page_size - 1)) *
                                                     pool.v_token) * E;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* q = p + (uint32_t)(v_lane + j * v_row);
        if (VW == 4) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(q);
          vf[4 * h + j][0] = x.x; vf[4 * h + j][1 % VW] = x.y;
          vf[4 * h + j][2 % VW] = x.z; vf[4 * h + j][3 % VW] = x.w;
        } else if (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(q);
          vf[4 * h + j][0] = x.x; vf[4 * h + j][1 % VW] = x.y;
        } else {
          vf[4 * h + j][0] = *reinterpret_cast<const uint32_t*>(q);
        }
      }
    }
  }

  __device__ __forceinline__ void scores(float (&s)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      floatx4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const u32x4 x = kf[h][i];
        if (E == 2) {
          a = mfma<QT>(x, qf[i], a);
        } else {
          a = mfma<QT>(u32x4{widen<QT, false>(x.x), widen<QT, true>(x.x), widen<QT, false>(x.y),
                             widen<QT, true>(x.y)}, qf[(2 * i) % QS], a);
          a = mfma<QT>(u32x4{widen<QT, false>(x.z), widen<QT, true>(x.z), widen<QT, false>(x.w),
                             widen<QT, true>(x.w)}, qf[(2 * i + 1) % QS], a);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * h + i] = a[i] * c;
    }
  }

  // Positions past the end and without a page: score -inf, value 0 (what is stored there may
  // be anything).
  __device__ __forceinline__ void mask(float (&s)[8], const Tile& t, int p0, int end) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int h = j >> 2;
      const bool in = t.page[h] >= 0 && p0 + 16 * h + 4 * g + (j & 3) < end;
      s[j] = in ? s[j] : -__builtin_inff();
#pragma unroll
      for (int w = 0; w < VW; ++w) vf[j][w] = in ? vf[j][w] : 0u;
    }
  }

  // Running softmax; s becomes the weights.
  __device__ __forceinline__ void weights(float (&s)[8]) {
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                      fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    top = xor32_max(xor16_max(top));
    if (__any(top > m)) {
      const float mn = fmaxf(m, top);
      const float a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= a;
#pragma unroll
      for (int d = 0; d < VD; ++d) acc[d] *= a;
      m = mn;
    }
    const float mu = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(s[j] - mu);
    l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  }

  __device__ __forceinline__ void values(const float (&s)[8]) {
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a, b;
      two_terms<QT>(s[2 * j], s[2 * j + 1], a, b);
      hi[j] = a;
      lo[j] = b;
    }
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = vf[2 * j][d * E / 4], b = vf[2 * j + 1][d * E / 4];
        if (E == 2) {
          v[j] = __builtin_amdgcn_perm(b, a, (d & 1) ? 0x07060302u : 0x05040100u);
        } else {
          // bytes (a0 b0 a1 b1) or (a2 b2 a3 b3): two dims' pairs of positions
          const uint32_t x = __builtin_amdgcn_perm(b, a, (d & 2) ? 0x07030602u : 0x05010400u);
          v[j] = (d & 1) ? widen<QT, true>(x) : widen<QT, false>(x);
        }
      }
      acc[d] = mfma<QT>(v, hi, acc[d]);
      acc[d] = mfma<QT>(v, lo, acc[d]);
    }
  }

  __device__ __forceinline__ void load_q(const uint16_t* __restrict__ q, int64_t ldh, int heads) {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int d = E == 2 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      qf[s] = r < heads ? *reinterpret_cast<const u32x4*>(q + r * ldh + d) : u32x4{0, 0, 0, 0};
    }
  }

  // Positions [begin, end) of one sequence, this wave's tiles of them.
  __device__ __forceinline__ void run(const PagePool& pool, const int32_t* __restrict__ row,
                                      int kvh, int begin, int end, int wave) {
    const int shift = __builtin_ctz(pool.page_size);
    const char* kb = static_cast<const char*>(pool.k) + kvh * pool.k_head * E;
    const char* vb = static_cast<const char*>(pool.v) + kvh * pool.v_head * E;
    k_lane = r * (int)pool.k_token * E + 16 * g;
    v_row = (int)pool.v_token * E;
    v_lane = 4 * g * v_row + r * VD * E;
    int p0 = begin + wave * kTile;
    if (p0 >= end) return;
    Tile t = pages(row, shift, p0, end, pool.pages);
    load_k(pool, kb, t, p0);
    load_v(pool, vb, t, p0);
    int p1 = p0 + WAVES * kTile;
    Tile next = pages(row, shift, p1, end, pool.pages);
    while (true) {
      float s[8];
      scores(s);
      const bool more = p1 < end;
      if (more) load_k(pool, kb, next, p1);
      if (p0 + kTile > end || t.page[0] < 0 || t.page[1] < 0) mask(s, t, p0, end);
      weights(s);
      values(s);
      if (!more) break;
      load_v(pool, vb, next, p1);
      t = next;
      p0 = p1;
      p1 += WAVES * kTile;
      next = pages(row, shift, p1, end, pool.pages);
    }
  }
};

// Chunk of a workgroup: the sequence, its positions and how many chunks it has.
struct Chunk {
  int seq, begin, end, count;
};

// Where group `slot` of the launch belongs.  Every wave finds it by itself: a lane counts the
// blocks of a run of sequences, the sum over the wave gives the chunks' length, a scan over the
// lanes' chunks the place.  Returns false past the last chunk.
__device__ __forceinline__ bool find_chunk(const int32_t* __restrict__ lens, int64_t seqs,
                                           int64_t cap, int units, int slot, Chunk& c) {
  const int lane = threadIdx.x & 63;
  const int per = (int)((seqs + 63) / 64);
  const int64_t s0 = (int64_t)lane * per;
  int blocks = 0;
  for (int i = 0; i < per; ++i)
    if (s0 + i < seqs) blocks += (clamp_len(lens[s0 + i], cap) + kBlock - 1) / kBlock;
  int total = blocks;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  const int64_t work = (int64_t)total * units;
  int len = (int)((work + kTargetChunks - 1) / kTargetChunks);     // blocks of a chunk
  len = len < 1 ? 1 : len;
  int chunks = 0;
  for (int i = 0; i < per; ++i)
    if (s0 + i < seqs) {
      const int n = ((clamp_len(lens[s0 + i], cap) + kBlock - 1) / kBlock + len - 1) / len;
      chunks += n < 1 ? 1 : n;
    }
  int upto = chunks;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(upto, o);
    if (lane >= o) upto += y;
  }
  const uint64_t past = __ballot(slot < upto);
  if (past == 0) return false;
  const int at = __builtin_ctzll(past);
  int first = __builtin_amdgcn_readlane(upto - chunks, at);
  for (int64_t s = (int64_t)at * per;; ++s) {
    const int n_pos = clamp_len(lens[s], cap);
    int n = ((n_pos + kBlock - 1) / kBlock + len - 1) / len;
    n = n < 1 ? 1 : n;
    if (slot < first + n) {
      const int64_t begin = (int64_t)(slot - first) * len * kBlock;
      const int64_t end = begin + (int64_t)len * kBlock;
      c.seq = (int)s;
      c.begin = (int)begin;
      c.end = end < n_pos ? (int)end : n_pos;
      c.count = n;
      return true;
    }
    first += n;
  }
}

// DIRECT: workgroup (unit, sequence) takes the whole sequence.
template <int QT, int KT, int D, int WAVES, bool DIRECT>
__global__ void __launch_bounds__(WAVES * 64) paged_attention_kernel(
    const uint16_t* __restrict__ q, int64_t ldq, int64_t ldh, PagePool pool,
    const int32_t* __restrict__ table, int64_t ldt, int64_t cap, int64_t seqs,
    const int32_t* __restrict__ lens, int n_heads, int head_tiles, int tile_heads, float scale,
    uint16_t* __restrict__ out, float* __restrict__ lse, float* __restrict__ part,
    float* __restrict__ part_ml, int2* __restrict__ plan) {
  extern __shared__ float lds[];
  constexpr int LD = D + 4;
  const int units = pool.kv_heads * head_tiles;
  Chunk ch;
  int unit;
  if (DIRECT) {
    unit = blockIdx.x % units;
    ch.seq = blockIdx.x / units;
    ch.begin = 0;
    ch.end = clamp_len(lens[ch.seq], cap);
    ch.count = 1;
  } else {
    unit = blockIdx.x % units;
    const int slot = blockIdx.x / units;
    if (!find_chunk(lens, seqs, cap, units, slot, ch)) return;
    if (unit == 0 && ch.begin == 0 && threadIdx.x == 0) plan[ch.seq] = make_int2(slot, ch.count);
  }
  ch.seq = __builtin_amdgcn_readfirstlane(ch.seq);
  ch.begin = __builtin_amdgcn_readfirstlane(ch.begin);
  ch.end = __builtin_amdgcn_readfirstlane(ch.end);
  ch.count = __builtin_amdgcn_readfirstlane(ch.count);
  const int kvh = unit / head_tiles, group = n_heads / pool.kv_heads;
  const int h0 = kvh * group + (unit % head_tiles) * 16;
  const int heads = min(16, (kvh + 1) * group - h0);
  const int wave = wave_id();

  Attend<QT, KT, D, WAVES> a;
  a.lane = threadIdx.x & 63;
  a.r = a.lane & 15;
  a.g = a.lane >> 4;
  a.m = -__builtin_inff();
  a.l = 0.f;
  a.c = scale * (pool.k_scale ? pool.k_scale[kvh] : 1.f) * kLog2e;
#pragma unroll
  for (int d = 0; d < a.VD; ++d) a.acc[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  a.load_q(q + ch.seq * ldq + h0 * ldh, ldh, heads);
  a.run(pool, table + ch.seq * ldt, kvh, ch.begin, ch.end, wave);

  // join the waves
  float* ml = lds + WAVES * tile_heads * LD;
  a.l = xor32_add(xor16_add(a.l));
  if (a.r < heads) {
    float* o = lds + (wave * tile_heads + a.r) * LD + a.VD * 4 * a.g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < a.VD; d += 4)
        *reinterpret_cast<floatx4*>(o + i * a.VD + d) =
            floatx4{a.acc[d][i], a.acc[d + 1][i], a.acc[d + 2][i], a.acc[d + 3][i]};
    if (a.g == 0) {
      ml[2 * (wave * 16 + a.r)] = a.m;
      ml[2 * (wave * 16 + a.r) + 1] = a.l;
    }
  }
  __syncthreads();
  const float vs = pool.v_scale ? pool.v_scale[kvh] : 1.f;
  for (int i = threadIdx.x; i < heads * (D / 4); i += WAVES * 64) {
    const int h = i / (D / 4), d = 4 * (i % (D / 4));
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml[2 * (w * 16 + h)]);
    const float mu = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float e = __builtin_amdgcn_exp2f(ml[2 * (w * 16 + h)] - mu);
      sum = fmaf(ml[2 * (w * 16 + h) + 1], e, sum);
      o += e * *reinterpret_cast<const floatx4*>(lds + (w * tile_heads + h) * LD + d);
    }
    if (ch.count == 1) {
      const float f = sum == 0.f ? 0.f : vs / sum;
      *reinterpret_cast<u32x2*>(out + ((int64_t)ch.seq * n_heads + h0 + h) * D + d) =
          u32x2{pack_out<QT>(o[0] * f, o[1] * f), pack_out<QT>(o[2] * f, o[3] * f)};
      if (lse && d == 0)
        lse[(int64_t)ch.seq * n_heads + h0 + h] =
            sum == 0.f ? -__builtin_inff() : (mu + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
      const int64_t at = (int64_t)blockIdx.x * tile_heads + h;
      *reinterpret_cast<floatx4*>(part + at * D + d) = o;
      if (d == 0) {
        part_ml[2 * at] = top;
        part_ml[2 * at + 1] = sum;
      }
    }
  }
}

// Joins the chunks of one query head of one sequence, in chunk order.
template <int QT, int D>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(
    const float* __restrict__ part, const float* __restrict__ part_ml,
    const int2* __restrict__ plan, int kv_heads, int head_tiles, int tile_heads, int n_heads,
    const float* __restrict__ v_scale, uint16_t* __restrict__ out, float* __restrict__ lse) {
  constexpr int LANES = D / 4, SETS = 256 / LANES;
  __shared__ floatx4 sums[SETS][LANES];
  __shared__ float tops[4], totals[SETS];
  const int64_t seq = blockIdx.y;
  const int h = blockIdx.x, group = n_heads / kv_heads, kvh = h / group;
  const int2 p = plan[seq];
  if (p.y == 1) return;
  const int units = kv_heads * head_tiles, unit = kvh * head_tiles + h % group / 16;
  const int64_t first = ((int64_t)p.x * units + unit) * tile_heads + h % group % 16;
  const int64_t step = (int64_t)units * tile_heads;        // from one chunk's row to the next's
  float top = -__builtin_inff();
  for (int i = threadIdx.x; i < p.y; i += 256) top = fmaxf(top, part_ml[2 * (first + i * step)]);
  top = wave_max_valu(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float mu = top == -__builtin_inff() ? 0.f : top;
  const int set = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
#pragma unroll 4
  for (int i = set; i < p.y; i += SETS) {
    const int64_t at = first + i * step;
    const float e = __builtin_amdgcn_exp2f(part_ml[2 * at] - mu);
    total = fmaf(part_ml[2 * at + 1], e, total);
    o += e * *reinterpret_cast<const floatx4*>(part + at * D + 4 * lane);
  }
  sums[set][lane] = o;
  if (lane == 0) totals[set] = total;
  __syncthreads();
  if (threadIdx.x >= LANES) return;
  total = 0.f;
  o = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    total += totals[s];
    o += sums[s][lane];
  }
  const float f = total == 0.f ? 0.f : (v_scale ? v_scale[kvh] : 1.f) / total;
  *reinterpret_cast<u32x2*>(out + (seq * n_heads + h) * D + 4 * lane) =
      u32x2{pack_out<QT>(o[0] * f, o[1] * f), pack_out<QT>(o[2] * f, o[3] * f)};
  if (lse && lane == 0)
    lse[seq * n_heads + h] = total == 0.f ? -__builtin_inff()
                                          : (mu + __builtin_amdgcn_logf(total)) * kLn2;
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_paged_attention_workspace_bytes(int64_t seqs, int32_t n_heads,
                                                       int32_t kv_heads, int32_t head_dim,
                                                       int64_t width, int32_t page_size) {
  if (seqs < 1 || kv_heads < 1 || n_heads < kv_heads || n_heads % kv_heads || head_dim < 1 ||
      page_size < 1 || width < 0 || width * page_size <= kDirectPositions)
    return 0;
  const Split s = split_of(seqs, n_heads, kv_heads);
  return s.groups * s.tile_heads * (head_dim + 2) * 4 + 8 * seqs;
}

extern "C" int mtl_paged_attention(const void* q, int64_t ldq, int64_t ldh,
                                   const mtl_page_pool* pool, const mtl_page_table* table,
                                   const int32_t* lens, int32_t n_heads, int32_t q_type,
                                   float scale, void* out, float* lse, void* workspace,
                                   int64_t ws_bytes, void* stream) {
  PagePool p;
  const int st = check_pool(pool, table, q_type, p);
  if (st != MTL_OK) return st;
  if (n_heads < 1 || n_heads % pool->kv_heads) return MTL_ERR_SHAPE;
  if (table->seqs == 0) return MTL_OK;
  if (!q || !lens || !out) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || ldh % 8 || !aligned16(q) || !aligned16(out)) return MTL_ERR_ALIGN;
  // rows of a page within 31 bits of a lane's offset; blocks of all sequences within 31 bits
  const int64_t most = INT32_MAX / 64;
  if (p.k_token > most || p.v_token > most || table->seqs > 65535) return MTL_ERR_SHAPE;
  int64_t cap = table->width > INT32_MAX / p.page_size ? INT32_MAX / p.page_size * p.page_size
                                                       : table->width * p.page_size;
  if (table->seqs * ((cap + kBlock - 1) / kBlock) > INT32_MAX) return MTL_ERR_SHAPE;
  const Split s = split_of(table->seqs, n_heads, pool->kv_heads);
  const int units = pool->kv_heads * s.head_tiles, d = pool->head_dim;
  const int64_t need = mtl_paged_attention_workspace_bytes(table->seqs, n_heads, pool->kv_heads, d,
                                                           table->width, p.page_size);
  const bool direct = need == 0;
  const int64_t groups = direct ? table->seqs * units : s.groups;
  if (groups > INT32_MAX) return MTL_ERR_SHAPE;
  if (!direct && (!workspace || ws_bytes < need)) return MTL_ERR_WORKSPACE;
  if (!direct && !aligned16(workspace)) return MTL_ERR_ALIGN;
  float* part = static_cast<float*>(workspace);
  float* part_ml = direct ? nullptr : part + s.groups * s.tile_heads * d;
  int2* plan = direct ? nullptr
                      : reinterpret_cast<int2*>(part_ml + s.groups * s.tile_heads * 2);
  const int waves = direct ? kDirectWaves : kSplitWaves;
  const size_t shared = (size_t)waves * (s.tile_heads * (d + 4) + 32) * 4;
  hipStream_t hs = (hipStream_t)stream;
#define MTL_RUN(T, KT, D)                                                                       \
  do {                                                                                          \
    if (direct)                                                                                 \
      paged_attention_kernel<T, KT, D, kDirectWaves, true>                                      \
          <<<(unsigned)groups, kDirectWaves * 64, shared, hs>>>(                                \
              (const uint16_t*)q, ldq, ldh, p, table->table, table->ld, cap, table->seqs, lens, \
              n_heads, s.head_tiles, s.tile_heads, scale, (uint16_t*)out, lse, part, part_ml,   \
              plan);                                                                            \
    else                                                                                        \
      paged_attention_kernel<T, KT, D, kSplitWaves, false>                                      \
          <<<(unsigned)groups, kSplitWaves * 64, shared, hs>>>(                                 \
              (const uint16_t*)q, ldq, ldh, p, table->table, table->ld, cap, table->seqs, lens, \
              n_heads, s.head_tiles, s.tile_heads, scale, (uint16_t*)out, lse, part, part_ml,   \
              plan);                                                                            \
  } while (0)
  MTL_PAGED_CASES(MTL_RUN, q_type, pool->type, d);
#undef MTL_RUN
  if (!direct) {
    const dim3 grid(n_heads, (unsigned)table->seqs);
#define MTL_JOIN(T, D)                                                                       \
  paged_attention_join_kernel<T, D><<<grid, 256, 0, hs>>>(part, part_ml, plan, p.kv_heads,   \
                                                          s.head_tiles, s.tile_heads, n_heads, \
                                                          p.v_scale, (uint16_t*)out, lse)
    if (q_type == MTL_T_BF16) { if (d == 128) MTL_JOIN(MTL_T_BF16, 128); else MTL_JOIN(MTL_T_BF16, 64); }
    else { if (d == 128) MTL_JOIN(MTL_T_F16, 128); else MTL_JOIN(MTL_T_F16, 64); }
#undef MTL_JOIN
  }
  return launch_status();
}
