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
// * A launch of kWorkgroups workgroups, all on the chip at once, shares the blocks of 128
//   positions of all sequences evenly: the blocks stand in one row, sequence after sequence, and
//   each workgroup of a kv head finds its piece of that row on the device from the lengths.  A
//   sequence that several workgroups have pieces of is joined by a second launch, piece after
//   piece.  Short tables (at most kDirectPositions) need neither: a workgroup a sequence and
//   kv head.
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
constexpr int kBlock = kTile * kSplitWaves;
constexpr int kWorkgroups = 512;        // 2 of 4 waves on each of 256 CUs
constexpr int kDirectPositions = 512;
constexpr int kDirectWaves = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How the launch is shared: `pieces` workgroups for each unit (up to 16 query heads of a kv
// head).  The workspace holds two rows of sums a workgroup, its first piece's and its last's
// (fp32 [pieces * units][2][tile_heads][head_dim], then (maximum, sum) for each), and int4
// [seqs] with what the second launch needs.
struct Split {
  int units, head_tiles, tile_heads, pieces;
  int64_t rows;
};

__host__ __device__ inline Split split_of(int n_heads, int kv_heads) {
  Split s;
  const int g = n_heads / kv_heads;
  s.tile_heads = g < 16 ? g : 16;
  s.head_tiles = (g + 15) / 16;
  s.units = kv_heads * s.head_tiles;
  s.pieces = s.units < kWorkgroups ? kWorkgroups / s.units : 1;
  s.rows = (int64_t)s.pieces * s.units * 2 * s.tile_heads;
  return s;
}

// K and V are read once: loads that leave no trace in the caches read 7.1 TB/s here, others 6.4.
// With more than 16 query heads to a kv head its rows are read again, from the caches.
template <bool ONCE, class T>
__device__ __forceinline__ T load(const char* p) {
  const T* q = reinterpret_cast<const T*>(p);
  return ONCE ? __builtin_nontemporal_load(q) : *q;
}

// A lane's 32-bit offset, formed where it is used: the load then takes base and offset as they
// are.  Without this the compiler keeps every offset as a 64-bit pair (24 registers).
__device__ __forceinline__ uint32_t fresh(int offset) {
  uint32_t o = (uint32_t)offset;
  asm volatile("" : "+v"(o));
  return o;
}

// table[i] for an i that is the same in all lanes, as a scalar load: a vector load would have
// the wave wait for the K and V in flight before it.
__device__ __forceinline__ int uniform_load(const int32_t* p, int64_t i) {
  typedef const int32_t __attribute__((address_space(4)))* Constant;
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

// One chunk of one sequence for up to 16 query heads of one kv head.
template <int QT, int KT, int D, int WAVES, bool ONCE>
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
  int r, g, k_lane, v_lane, v_row;

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
      if (p < end) id = uniform_load(row, p >> shift);
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
      const uint32_t o = fresh(k_lane);
#pragma unroll
      for (int s = 0; s < KL; ++s) kf[h][s] = load<ONCE, u32x4>(p + o + 64 * s);
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
        const char* q = p + fresh(v_lane + j * v_row);
        if (VW == 4) {
          const u32x4 x = load<ONCE, u32x4>(q);
          vf[4 * h + j][0] = x.x; vf[4 * h + j][1 % VW] = x.y;
          vf[4 * h + j][2 % VW] = x.z; vf[4 * h + j][3 % VW] = x.w;
        } else if (VW == 2) {
          const u32x2 x = load<ONCE, u32x2>(q);
          vf[4 * h + j][0] = x.x; vf[4 * h + j][1 % VW] = x.y;
        } else {
          vf[4 * h + j][0] = load<ONCE, uint32_t>(q);
        }
      }
    }
  }

  __device__ __forceinline__ void scores(float (&s)[8]) const {
    floatx4 a[2] = {};                    // two chains of products, in turn
#pragma unroll
    for (int i = 0; i < KL; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 x = kf[h][i];
        if (E == 2)
          a[h] = mfma<QT>(x, qf[i], a[h]);
        else
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x.x), widen<QT, true>(x.x),
                                widen<QT, false>(x.y), widen<QT, true>(x.y)},
                          qf[(2 * i) % QS], a[h]);
      }
      if (E == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 x = kf[h][i];
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x.z), widen<QT, true>(x.z),
                                widen<QT, false>(x.w), widen<QT, true>(x.w)},
                          qf[(2 * i + 1) % QS], a[h]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = a[j >> 2][j & 3] * c;
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
    for (int d0 = 0; d0 < VD; d0 += 2) {  // two accumulators in turn
      u32x4 v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = d0 + e;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a = vf[2 * j][d * E / 4], b = vf[2 * j + 1][d * E / 4];
          if (E == 2) {
            v[e][j] = __builtin_amdgcn_perm(b, a, e ? 0x07060302u : 0x05040100u);
          } else {
            // bytes (a0 b0 a1 b1) or (a2 b2 a3 b3): two dims' pairs of positions
            const uint32_t x = __builtin_amdgcn_perm(b, a, (d & 2) ? 0x07030602u : 0x05010400u);
            v[e][j] = e ? widen<QT, true>(x) : widen<QT, false>(x);
          }
        }
      }
      acc[d0] = mfma<QT>(v[0], hi, acc[d0]);
      acc[d0 + 1] = mfma<QT>(v[1], hi, acc[d0 + 1]);
      acc[d0] = mfma<QT>(v[0], lo, acc[d0]);
      acc[d0 + 1] = mfma<QT>(v[1], lo, acc[d0 + 1]);
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
    float s[8];
    // The next tile's K is loaded once this one's scores are formed, its V once this one's values
    // are summed.  The last tile stands apart: a load under a condition would have the compiler
    // wait for all loads wherever it joins.
    while (p1 < end) {
      scores(s);
      load_k(pool, kb, next, p1);
      if (t.page[0] < 0 || t.page[1] < 0) mask(s, t, p0, end);
      weights(s);
      values(s);
      load_v(pool, vb, next, p1);
      t = next;
      p0 = p1;
      p1 += WAVES * kTile;
      next = pages(row, shift, p1, end, pool.pages);
    }
    scores(s);
    if (p0 + kTile > end || t.page[0] < 0 || t.page[1] < 0) mask(s, t, p0, end);
    weights(s);
    values(s);
  }
};

// The blocks of all sequences in one row, cut into `pieces` parts that differ by one block at
// most.
struct Cuts {
  int each, extra;
  __device__ __forceinline__ Cuts(int total, int pieces) : each(total / pieces),
                                                           extra(total % pieces) {}
  __device__ __forceinline__ int start(int piece) const {
    return piece * each + min(piece, extra);
  }
  __device__ __forceinline__ int piece_of(int block) const {
    const int longer = extra * (each + 1);
    return block < longer ? block / (each + 1) : extra + (block - longer) / each;
  }
};

__device__ __forceinline__ int blocks_of(int len) { return (len + kBlock - 1) / kBlock; }

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

// Every wave finds its place by itself: a lane counts the blocks of a run of `per` sequences.
struct Scan {
  int per, len, upto, total;
  __device__ __forceinline__ Scan(const int32_t* __restrict__ lens, int seqs, int64_t cap) {
    const int lane = threadIdx.x & 63;
    per = (seqs + 63) / 64;
    const int64_t s0 = (int64_t)lane * per;
    int blocks = 0;
    for (int i = 0; i < per; ++i) {
      len = s0 + i < seqs ? clamp_len(lens[s0 + i], cap) : 0;
      blocks += blocks_of(len);
    }
    upto = wave_scan(blocks);
    total = __builtin_amdgcn_readlane(upto, 63);
  }
};

// The output of one query head of one sequence from its sum o (4 dims), base-2 maximum and
// weights' sum.
template <int QT, int D>
__device__ __forceinline__ void write_out(uint16_t* __restrict__ out, float* __restrict__ lse,
                                          int64_t head, int d, floatx4 o, float top, float sum,
                                          float vs) {
  const float f = sum == 0.f ? 0.f : vs / sum;
  *reinterpret_cast<u32x2*>(out + head * D + d) =
      u32x2{pack_out<QT>(o[0] * f, o[1] * f), pack_out<QT>(o[2] * f, o[3] * f)};
  if (lse && d == 0)
    lse[head] = sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

struct Rows {
  const uint16_t* q;
  int64_t ldq, ldh;
  const int32_t* table;
  int64_t ldt, cap;
  const int32_t* lens;
  int seqs, n_heads, head_tiles, tile_heads, pieces;
  float scale;
  uint16_t* out;
  float* lse;
  float* part;
  float* part_ml;
  int4* plan;
};

// Positions [begin, end) of a sequence for one unit; the waves' results are joined through LDS
// into out (row < 0) or into a row of the workspace.
template <int QT, int KT, int D, int WAVES, bool ONCE>
__device__ __forceinline__ void attend_piece(const Rows& a, const PagePool& pool, int unit, int seq,
                                             int begin, int end, int64_t row, float* lds) {
  constexpr int LD = D + 4;
  const int kvh = unit / a.head_tiles, group = a.n_heads / pool.kv_heads;
  const int h0 = kvh * group + (unit % a.head_tiles) * 16;
  const int heads = min(16, (kvh + 1) * group - h0);
  const int wave = wave_id();

  Attend<QT, KT, D, WAVES, ONCE> w;
  // what depends on the thread is formed anew for each piece, before and after the loop over
  // its tiles: kept over the loop it costs 30 registers
  int thread = (int)fresh(threadIdx.x);
  w.r = thread & 15;
  w.g = (thread & 63) >> 4;
  w.m = -__builtin_inff();
  w.l = 0.f;
  w.c = a.scale * (pool.k_scale ? pool.k_scale[kvh] : 1.f) * kLog2e;
#pragma unroll
  for (int d = 0; d < w.VD; ++d) w.acc[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  w.load_q(a.q + seq * a.ldq + h0 * a.ldh, a.ldh, heads);
  w.run(pool, a.table + seq * a.ldt, kvh, begin, end, wave);

  float* ml = lds + WAVES * a.tile_heads * LD;
  w.l = xor32_add(xor16_add(w.l));
  thread = (int)fresh(threadIdx.x);
  const int r = thread & 15, g = (thread & 63) >> 4;
  if (r < heads) {
    float* o = lds + (wave * a.tile_heads + r) * LD + w.VD * 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < w.VD; d += 4)
        *reinterpret_cast<floatx4*>(o + i * w.VD + d) =
            floatx4{w.acc[d][i], w.acc[d + 1][i], w.acc[d + 2][i], w.acc[d + 3][i]};
    if (g == 0) {
      ml[2 * (wave * 16 + r)] = w.m;
      ml[2 * (wave * 16 + r) + 1] = w.l;
    }
  }
  __syncthreads();
  for (int i = thread; i < heads * (D / 4); i += WAVES * 64) {
    const int h = i / (D / 4), d = 4 * (i % (D / 4));
    float top = -__builtin_inff();
#pragma unroll
    for (int x = 0; x < WAVES; ++x) top = fmaxf(top, ml[2 * (x * 16 + h)]);
    const float mu = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < WAVES; ++x) {
      const float e = __builtin_amdgcn_exp2f(ml[2 * (x * 16 + h)] - mu);
      sum = fmaf(ml[2 * (x * 16 + h) + 1], e, sum);
      o += e * *reinterpret_cast<const floatx4*>(lds + (x * a.tile_heads + h) * LD + d);
    }
    if (row < 0) {
      write_out<QT, D>(a.out, a.lse, (int64_t)seq * a.n_heads + h0 + h, d, o, mu, sum,
                       pool.v_scale ? pool.v_scale[kvh] : 1.f);
    } else {
      *reinterpret_cast<floatx4*>(a.part + (row + h) * D + d) = o;
      if (d == 0) {
        a.part_ml[2 * (row + h)] = top;
        a.part_ml[2 * (row + h) + 1] = sum;
      }
    }
  }
}

// Workgroup (unit, sequence) takes the whole sequence.
template <int QT, int KT, int D, bool ONCE>
__global__ void __launch_bounds__(kDirectWaves * 64) paged_attention_direct_kernel(Rows a,
                                                                                   PagePool pool) {
  extern __shared__ float lds[];
  const int units = pool.kv_heads * a.head_tiles;
  const int seq = blockIdx.x / units;
  attend_piece<QT, KT, D, kDirectWaves, ONCE>(a, pool, blockIdx.x % units, seq, 0,
                                              clamp_len(uniform_load(a.lens, seq), a.cap), -1, lds);
}

// Workgroup (unit, piece) takes its piece of the row of blocks; the one past them all writes
// down for each sequence which pieces it has (first piece, pieces, the first one's row).
template <int QT, int KT, int D, bool ONCE>
__global__ void __launch_bounds__(kSplitWaves * 64, 2) paged_attention_kernel(Rows a,
                                                                              PagePool pool) {
  extern __shared__ float lds[];
  const int units = pool.kv_heads * a.head_tiles;
  const int unit = blockIdx.x % units, piece = blockIdx.x / units;
  const Scan scan(a.lens, a.seqs, a.cap);
  const Cuts cuts(scan.total, a.pieces);
  const int lane = threadIdx.x & 63;
  if (piece == a.pieces) {
    if (threadIdx.x >= 64) return;
    int base = __builtin_amdgcn_update_dpp(0, scan.upto, 0x138, 0xf, 0xf, false);   // wave_shr:1
    for (int i = 0; i < scan.per; ++i) {
      const int64_t s = (int64_t)lane * scan.per + i;
      if (s >= a.seqs) break;
      const int n = blocks_of(clamp_len(a.lens[s], a.cap));
      int4 p = make_int4(0, 0, 0, 0);
      if (n > 0) {
        p.x = cuts.piece_of(base);
        p.y = cuts.piece_of(base + n - 1) - p.x + 1;
        p.z = cuts.start(p.x) < base;
      }
      a.plan[s] = p;
      base += n;
    }
    return;
  }
  int at = cuts.start(piece);
  const int stop = cuts.start(piece + 1);
  if (at == stop) return;
  const int from = __builtin_ctzll(__ballot(at < scan.upto));
  int base = from ? __builtin_amdgcn_readlane(scan.upto, from - 1) : 0;
  int seq = from * scan.per;
  int len = scan.per == 1 ? __builtin_amdgcn_readlane(scan.len, from) : clamp_len(uniform_load(a.lens, seq), a.cap);
  while (true) {
    const int n = blocks_of(len);
    if (at < base + n) {
      const int first = at - base, last = min(stop - base, n);
      const int64_t row = first == 0 && last == n ? -1
          : ((int64_t)blockIdx.x * 2 + (at > cuts.start(piece))) * a.tile_heads;
      attend_piece<QT, KT, D, kSplitWaves, ONCE>(a, pool, unit, seq, first * kBlock,
                                                 min(last * kBlock, len), row, lds);
      at = base + last;
      if (at == stop) return;
      __syncthreads();                 // the next piece uses the same LDS
    }
    base += n;
    if (++seq >= a.seqs) return;       // lengths that changed under the launch
    len = clamp_len(uniform_load(a.lens, seq), a.cap);
  }
}

// Joins the pieces of one query head of one sequence, in their order: each set of lanes takes
// every SETS-th piece with a running maximum of its own, the sets are joined through LDS.
template <int QT, int D>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(Rows a, int kv_heads,
                                                                   const float* __restrict__ v_scale) {
  constexpr int LANES = D / 4, SETS = 256 / LANES;
  __shared__ floatx4 sums[SETS][LANES];
  __shared__ float tops[SETS], totals[SETS];
  const int64_t seq = blockIdx.y;
  const int h = blockIdx.x, group = a.n_heads / kv_heads, kvh = h / group;
  const int4 p = a.plan[seq];
  if (p.y == 1) return;
  const int units = kv_heads * a.head_tiles, unit = kvh * a.head_tiles + h % group / 16;
  const int set = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), total = 0.f;
#pragma unroll 4
  for (int i = set; i < p.y; i += SETS) {
    const int64_t at = (((int64_t)(p.x + i) * units + unit) * 2 + (i == 0 ? p.z : 0)) *
                           a.tile_heads + h % group % 16;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
    const floatx4 x = *reinterpret_cast<const floatx4*>(a.part + at * D + 4 * lane);
    const float t = fmaxf(top, ml.x), mu = t == -__builtin_inff() ? 0.f : t;
    const float e0 = __builtin_amdgcn_exp2f(top - mu), e1 = __builtin_amdgcn_exp2f(ml.x - mu);
    total = total * e0 + ml.y * e1;
    o = o * e0 + x * e1;
    top = t;
  }
  sums[set][lane] = o;
  if (lane == 0) {
    tops[set] = top;
    totals[set] = total;
  }
  __syncthreads();
  if (threadIdx.x >= LANES) return;
  top = tops[0];
#pragma unroll
  for (int s = 1; s < SETS; ++s) top = fmaxf(top, tops[s]);
  const float mu = top == -__builtin_inff() ? 0.f : top;
  total = 0.f;
  o = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    const float e = __builtin_amdgcn_exp2f(tops[s] - mu);
    total = fmaf(totals[s], e, total);
    o += e * sums[s][lane];
  }
  write_out<QT, D>(a.out, a.lse, seq * a.n_heads + h, 4 * lane, o, mu, total,
                   v_scale ? v_scale[kvh] : 1.f);
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_paged_attention_workspace_bytes(int64_t seqs, int32_t n_heads,
                                                       int32_t kv_heads, int32_t head_dim,
                                                       int64_t width, int32_t page_size) {
  if (seqs < 1 || kv_heads < 1 || n_heads < kv_heads || n_heads % kv_heads || head_dim < 1 ||
      page_size < 1 || width < 0 || width <= kDirectPositions / page_size)
    return 0;
  return split_of(n_heads, kv_heads).rows * (head_dim + 2) * 4 + 16 * seqs;
}

namespace mtl {

template <int QT, int KT, int D, bool ONCE>
static void launch_attention(const Rows& a, const PagePool& p, bool direct, const Split& s,
                             hipStream_t stream) {
  const size_t wave = (size_t)(s.tile_heads * (D + 4) + 32) * 4;
  if (direct) {
    paged_attention_direct_kernel<QT, KT, D, ONCE>
        <<<(unsigned)(a.seqs * s.units), kDirectWaves * 64, kDirectWaves * wave, stream>>>(a, p);
    return;
  }
  paged_attention_kernel<QT, KT, D, ONCE>
      <<<(unsigned)(s.pieces * s.units + 1), kSplitWaves * 64, kSplitWaves * wave, stream>>>(a, p);
  paged_attention_join_kernel<QT, D><<<dim3(a.n_heads, a.seqs), 256, 0, stream>>>(a, p.kv_heads,
                                                                                  p.v_scale);
}

}  // namespace mtl

extern "C" int mtl_paged_attention(const void* q, int64_t ldq, int64_t ldh,
                                   const mtl_page_pool* pool, const mtl_page_table* table,
                                   const int32_t* lens, int32_t n_heads, int32_t q_type,
                                   float scale, void* out, float* lse, void* workspace,
                                   int64_t ws_bytes, void* stream) {
  PagePool p;
  const int st = check_pool(pool, table, q_type, p);
  if (st != MTL_OK) return st;
  if (n_heads < 1 || n_heads % pool->kv_heads || n_heads > 65535) return MTL_ERR_SHAPE;
  if (table->seqs == 0) return MTL_OK;
  if (!q || !lens || !out) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || ldh % 8 || !aligned16(q) || !aligned16(out)) return MTL_ERR_ALIGN;
  // a lane's offset within a page, and the row of all sequences' blocks, within 31 bits
  const int64_t most = INT32_MAX / 64;
  if (p.k_token > most || p.v_token > most || table->seqs > 65535) return MTL_ERR_SHAPE;
  const int64_t wide = INT32_MAX / p.page_size;
  const int64_t cap = (table->width < wide ? table->width : wide) * p.page_size;
  if (table->seqs * ((cap + kBlock - 1) / kBlock) > INT32_MAX) return MTL_ERR_SHAPE;
  const Split s = split_of(n_heads, pool->kv_heads);
  const int d = pool->head_dim;
  const int64_t need = mtl_paged_attention_workspace_bytes(table->seqs, n_heads, pool->kv_heads, d,
                                                           table->width, p.page_size);
  const bool direct = need == 0;
  if (table->seqs * s.units > INT32_MAX) return MTL_ERR_SHAPE;
  if (!direct && (!workspace || ws_bytes < need)) return MTL_ERR_WORKSPACE;
  if (!direct && !aligned16(workspace)) return MTL_ERR_ALIGN;
  char* ws = static_cast<char*>(workspace);
  const Rows a{static_cast<const uint16_t*>(q), ldq, ldh, table->table, table->ld, cap, lens,
               (int)table->seqs, n_heads, s.head_tiles, s.tile_heads, s.pieces, scale,
               static_cast<uint16_t*>(out), lse, reinterpret_cast<float*>(ws + 16 * table->seqs),
               reinterpret_cast<float*>(ws + 16 * table->seqs + s.rows * d * 4),
               reinterpret_cast<int4*>(ws)};
#define MTL_RUN(T, KT, D)                                                        \
  do {                                                                           \
    if (s.head_tiles == 1)                                                       \
      launch_attention<T, KT, D, true>(a, p, direct, s, (hipStream_t)stream);    \
    else                                                                         \
      launch_attention<T, KT, D, false>(a, p, direct, s, (hipStream_t)stream);   \
  } while (0)
  MTL_PAGED_CASES(MTL_RUN, q_type, pool->type, d);
#undef MTL_RUN
  return launch_status();
}
