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
//   what the rounding left: a weight is off by 2^-16 of itself in bf16, by 2^-20 of itself and
//   2^-39 of the largest in f16, far below the output's own rounding (with one number the output
//   is off by 1.4 times as much).  f16 ends at 2^-24, so its weights enter 2^15 larger.
// * A launch of kWorkgroups workgroups, all on the chip at once, shares the blocks of 128
//   positions of all sequences evenly: the blocks stand in one row, sequence after sequence, and
//   each workgroup of a kv head finds its piece of that row on the device from the lengths.  A
//   sequence that several workgroups have pieces of is joined by a second launch, piece after
//   piece.  Short tables (at most kDirectPositions) need neither: a workgroup a sequence and
//   kv head.
//
// Measured, head_dim 128, bf16, a memory rate of 7.1 TB/s for such reads: one sequence of 131 000
// positions and 4 kv heads (537 MB) 81 + 5 us in the two launches, 6.6 TB/s in the first; 128
// ragged sequences (594 MB) 97 + 5 us, 6.1 TB/s; ragged sequences in e4m3 (322 MB) 55 + 5 us, 5.8
// TB/s.  About 10 us of that do not grow with the bytes (two launches; lengths, page ids and the
// first tile, which wait for one another; the join), the rest streams at 7 TB/s: 307 MB take 53
// to 56 us in bf16 and 55 to 58 in e4m3, as one sequence or as 64 equal ones, in pages of 16, 64
// or 256.  A short table (300 positions) takes 6 us, which is a launch and three trips to the
// memory (length and page ids, tile, output).  The counters show no byte of the cache read twice
// with up to 16 query heads to a kv head.  Past that K and V are read for each 16 of them, by
// workgroups that share no L2: 300 MB take 55 to 60 us with 32 heads over 2 (L2 misses 303 MB) and
// 89 to 93 with 34 to 64 over 2 (602 MB).
//
// Tried and slower: 3 or 4 waves on each of a CU's four parts (their registers spill), the next
// sequence's first tile loaded ahead (even), 6, 8 or 12 waves in 256 workgroups, shares in tiles
// of 32 positions, 64 positions of e4m3 to a wave (60 against 58 us for 300 MB), and joining in
// the first launch by whoever comes last, which needs counters to be cleared beforehand and
// signals past the chip's separate caches that cost what the second launch costs (3 to 5 us).
#include "mtl_paged_pool.h"

namespace mtl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;               // positions a wave takes at a time
constexpr int kSplitWaves = 4;
constexpr int kBlock = kTile * kSplitWaves;
// 2 workgroups of 4 waves on each of 256 CUs: all their registers' room.  768 and 1024 (which
// then come in turns) were not faster at any of 16 shapes, and have more to join.
constexpr int kWorkgroups = 512;
// The longest table for which every sequence gets a workgroup of its own.  Both sides measured,
// one against the other in us: 1 sequence of 250 positions 5.3 (7.1 shared out), of 500 7.9 (7.1),
// of 700 9.5 (7.2); 32 of 500 13.0 (16.4).  Past it the uneven ends of long sequences lose more:
// 512 of mixed lengths up to 1024 100 (78).
constexpr int kDirectPositions = 512;
constexpr int kDirectWaves = 8;
constexpr int64_t kMaxPositions = 1 << 30;      // of one sequence: they fit an int with room
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How the launch is shared: `pieces` workgroups for each unit (up to 16 query heads of a kv
// head).  The workspace holds two rows of sums a workgroup, its first piece's and its last's
// (fp32 [pieces * units][2][tile_heads][head_dim], then (maximum, sum) for each), and int4
// [min(seqs, pieces)] with what the second launch joins.
struct Split {
  int units, head_tiles, tile_heads, pieces;
  int64_t rows;
  // sequences that lie in several pieces, at most
  int64_t joined(int64_t seqs) const { return seqs < pieces ? seqs : pieces; }
};

inline Split split_of(int n_heads, int kv_heads) {
  Split s;
  const int g = n_heads / kv_heads;
  s.tile_heads = g < 16 ? g : 16;
  s.head_tiles = (g + 15) / 16;
  s.units = kv_heads * s.head_tiles;
  s.pieces = s.units < kWorkgroups ? kWorkgroups / s.units : 1;
  s.rows = (int64_t)s.pieces * s.units * 2 * s.tile_heads;
  return s;
}

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

// A wave's part of one piece of one sequence, for up to 16 query heads of one kv head.
template <int QT, int KT, int D, int WAVES, bool ONCE>
struct Attend {
  static constexpr int E = KT == MTL_T_E4M3 ? 1 : 2;    // bytes of a stored element
  static constexpr int KL = D * E / 64;                 // 16-byte loads of a lane's K row
  static constexpr int QS = D / 32;                     // MFMA steps over the dims
  static constexpr int VD = D / 16;                     // dims of a lane's V pieces
  static constexpr int VW = VD * E / 4;                 // ... in dwords
  u32x4 qf[QS];
  uint32_t kf[2][KL][4];
  uint32_t vf[8][VW];
  floatx4 acc[VD];
  float m, l, c;                                        // c: scale to base 2
  int r, g, k_lane, v_lane, v_row;

  // A tile's two halves of 16 positions: each one's page and how many of its rows count (0: none).
  struct Tile {
    int page[2], rows[2];
  };
  Tile t;                                               // of the tile in kf and vf

  // One kv head's ends of the pages.
  struct Ends {
    const char* k;
    const char* v;
    int shift;
  };

  // The page ids of the tile at p0, where the table has them (`limit`).
  __device__ __forceinline__ void ids(const int32_t* __restrict__ row, int shift, int p0, int limit,
                                      Tile& t) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = p0 + 16 * h;
      t.page[h] = p < limit ? uniform_load(row, p >> shift) : -1;
    }
  }

  __device__ __forceinline__ void count(int p0, int end, int n_pages, Tile& t) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool there = (uint32_t)t.page[h] < (uint32_t)n_pages;
      t.rows[h] = there ? min(max(end - (p0 + 16 * h), 0), 16) : 0;
      t.page[h] = there ? t.page[h] : 0;
    }
  }

  __device__ __forceinline__ void load_k(const PagePool& pool, const Ends& e, const Tile& t,
                                         int p0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Rsrc rows = rows_at(e.k + (t.page[h] * pool.k_page +
                                       ((p0 + 16 * h) & (pool.page_size - 1)) * pool.k_token) * E,
                                t.rows[h] * (int)pool.k_token * E);
#pragma unroll
      for (int s = 0; s < KL; ++s) load_row<ONCE>(rows, k_lane + 64 * s, kf[h][s]);
    }
  }

  __device__ __forceinline__ void load_v(const PagePool& pool, const Ends& e, const Tile& t,
                                         int p0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Rsrc rows = rows_at(e.v + (t.page[h] * pool.v_page +
                                       ((p0 + 16 * h) & (pool.page_size - 1)) * pool.v_token) * E,
                                t.rows[h] * (int)pool.v_token * E);
#pragma unroll
      for (int j = 0; j < 4; ++j) load_row<ONCE>(rows, v_lane + j * v_row, vf[4 * h + j]);
    }
  }

  __device__ __forceinline__ void scores(float (&s)[8]) const {
    floatx4 a[2] = {};                    // two chains of products, in turn
#pragma unroll
    for (int i = 0; i < KL; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t(&x)[4] = kf[h][i];
        if (E == 2)
          a[h] = mfma<QT>(u32x4{x[0], x[1], x[2], x[3]}, qf[i], a[h]);
        else
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x[0]), widen<QT, true>(x[0]),
                                widen<QT, false>(x[1]), widen<QT, true>(x[1])},
                          qf[(2 * i) % QS], a[h]);
      }
      if (E == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t(&x)[4] = kf[h][i];
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x[2]), widen<QT, true>(x[2]),
                                widen<QT, false>(x[3]), widen<QT, true>(x[3])},
                          qf[(2 * i + 1) % QS], a[h]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = a[j >> 2][j & 3] * c;
  }

  // Rows that do not count: score -inf (their K and V are 0).
  __device__ __forceinline__ void mask(float (&s)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s[j] = 4 * g + (j & 3) < t.rows[j >> 2] ? s[j] : -__builtin_inff();
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
      two_terms<QT>(s[2 * j] * kLift<QT>, s[2 * j + 1] * kLift<QT>, a, b);
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

  __device__ __forceinline__ void load_q(const uint16_t* __restrict__ q, int64_t ldh, int heads,
                                         u32x4 (&f)[QS]) const {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int d = E == 2 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      f[s] = r < heads ? *reinterpret_cast<const u32x4*>(q + r * ldh + d) : u32x4{0, 0, 0, 0};
    }
  }

  // This wave's tiles of positions [begin, end); the page ids of a tile are read while the one
  // before is worked on, up to position `limit` >= end.
  __device__ __forceinline__ void run(const PagePool& pool, const Ends& e,
                                      const int32_t* __restrict__ row, int begin, int end,
                                      int limit) {
    constexpr int kStep = WAVES * kTile;
    int p0 = begin + wave_id() * kTile;
    Tile next;
    ids(row, e.shift, p0, limit, next);
    while (p0 < end) {
      t = next;
      count(p0, end, pool.pages, t);
      load_k(pool, e, t, p0);
      load_v(pool, e, t, p0);
      ids(row, e.shift, p0 + kStep, limit, next);
      float s[8];
      scores(s);
      if (t.rows[0] + t.rows[1] < kTile) mask(s);
      weights(s);
      values(s);
      p0 += kStep;
    }
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

// The end of `blocks` blocks of a sequence of len positions.
__device__ __forceinline__ int blocks_end(int blocks, int len) {
  const int64_t end = (int64_t)blocks * kBlock;
  return end < len ? (int)end : len;
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
  const float f = sum == 0.f ? 0.f : vs / sum * (1.f / kLift<QT>);
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

// What a workgroup of one unit works with.
template <int QT, int KT, int D, int WAVES, bool ONCE>
struct Unit {
  using Wave = Attend<QT, KT, D, WAVES, ONCE>;
  static constexpr int LD = D + 4;
  const Rows& a;
  const PagePool& pool;
  float* lds;
  int kvh, h0, heads;
  float v_scale;
  typename Wave::Ends ends;
  Wave w;

  __device__ __forceinline__ Unit(const Rows& a, const PagePool& pool, int unit, float* lds)
      : a(a), pool(pool), lds(lds) {
    kvh = unit / a.head_tiles;
    const int group = a.n_heads / pool.kv_heads;
    h0 = kvh * group + (unit % a.head_tiles) * 16;
    heads = min(16, (kvh + 1) * group - h0);
    ends.shift = __builtin_ctz(pool.page_size);
    ends.k = static_cast<const char*>(pool.k) + kvh * pool.k_head * w.E;
    ends.v = static_cast<const char*>(pool.v) + kvh * pool.v_head * w.E;
    w.c = a.scale * (pool.k_scale ? uniform_load(pool.k_scale, kvh) : 1.f) * kLog2e;
    v_scale = pool.v_scale ? uniform_load(pool.v_scale, kvh) : 1.f;
  }

  // What depends on the lane is formed anew for each piece: kept from one to the next, with what
  // the compiler derives from it, it costs 30 registers.
  __device__ __forceinline__ void lane() {
    const int thread = fresh(threadIdx.x);
    w.r = thread & 15;
    w.g = (thread & 63) >> 4;
    w.k_lane = w.r * (int)pool.k_token * w.E + 16 * w.g;
    w.v_row = (int)pool.v_token * w.E;
    w.v_lane = 4 * w.g * w.v_row + w.r * w.VD * w.E;
  }

  __device__ __forceinline__ const int32_t* row(int seq) const { return a.table + seq * a.ldt; }

  __device__ __forceinline__ void query(int seq, u32x4 (&f)[Wave::QS]) const {
    w.load_q(a.q + seq * a.ldq + h0 * a.ldh, a.ldh, heads, f);
  }

  __device__ __forceinline__ void clear() {
    w.m = -__builtin_inff();
    w.l = 0.f;
#pragma unroll
    for (int d = 0; d < w.VD; ++d) w.acc[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  // Joins the waves through LDS, into out (dst < 0) or into rows of the workspace from dst on.
  __device__ __forceinline__ void join(int seq, int64_t dst) {
    float* ml = lds + WAVES * a.tile_heads * LD;
    const int thread = fresh(threadIdx.x), wave = wave_id();
    const int r = thread & 15, g = (thread & 63) >> 4;
    w.l = xor32_add(xor16_add(w.l));
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
      if (dst < 0) {
        write_out<QT, D>(a.out, a.lse, (int64_t)seq * a.n_heads + h0 + h, d, o, mu, sum, v_scale);
      } else {
        *reinterpret_cast<floatx4*>(a.part + (dst + h) * D + d) = o;
        if (d == 0) {
          a.part_ml[2 * (dst + h)] = top;
          a.part_ml[2 * (dst + h) + 1] = sum;
        }
      }
    }
  }
};

// Workgroup (unit, sequence) takes the whole sequence; page ids and length are read at once.
template <int QT, int KT, int D, bool ONCE>
__global__ void __launch_bounds__(kDirectWaves * 64) paged_attention_direct_kernel(Rows a,
                                                                                   PagePool pool) {
  extern __shared__ float lds[];
  const int units = pool.kv_heads * a.head_tiles;
  const int seq = blockIdx.x / units;
  Unit<QT, KT, D, kDirectWaves, ONCE> u(a, pool, blockIdx.x % units, lds);
  u.lane();
  u.query(seq, u.w.qf);
  u.clear();
  u.w.run(pool, u.ends, u.row(seq), 0, clamp_len(uniform_load(a.lens, seq), a.cap), (int)a.cap);
  u.join(seq, -1);
}

// What the second launch joins: sequences with several pieces, (sequence, first piece, pieces,
// the first piece's row), at most one for each cut; (., ., 0, .) behind them.
__device__ __forceinline__ void write_plan(const Rows& a, const Scan& scan, const Cuts& cuts) {
  const int lane = threadIdx.x & 63;
  const int most = min(a.seqs, a.pieces);
  const int before = __builtin_amdgcn_update_dpp(0, scan.upto, 0x138, 0xf, 0xf, false);  // lane - 1
  for (int pass = 0, slot = 0, listed = 0; pass < 2; ++pass) {
    int base = before, mine = 0;
    for (int i = 0; i < scan.per; ++i) {
      const int64_t s = (int64_t)lane * scan.per + i;
      const int n = s < a.seqs ? blocks_of(clamp_len(a.lens[s], a.cap)) : 0;
      if (n > 1) {
        const int p = cuts.piece_of(base), count = cuts.piece_of(base + n - 1) - p + 1;
        if (count > 1) {
          if (pass == 1) a.plan[slot + mine] = make_int4((int)s, p, count, cuts.start(p) < base);
          ++mine;
        }
      }
      base += n;
    }
    if (pass == 0) {
      const int upto = wave_scan(mine);
      slot = upto - mine;
      listed = __builtin_amdgcn_readlane(upto, 63);
    } else {
      for (int k = listed + lane; k < most; k += 64) a.plan[k] = make_int4(0, 0, 0, 0);
    }
  }
}

// Sequences without positions: 0 and -inf, shared among the workgroup's waves.
template <int D>
__device__ __forceinline__ void write_empty(const Rows& a, const Scan& scan, int h0, int heads) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  for (int i = 0; i < scan.per; ++i) {
    const int64_t s = (int64_t)lane * scan.per + i;
    uint64_t empty = __ballot(s < a.seqs && clamp_len(s < a.seqs ? a.lens[s] : 1, a.cap) == 0);
    for (int k = 0; empty; ++k, empty &= empty - 1) {
      if (k % kSplitWaves != wave) continue;
      const int64_t head = ((int64_t)__builtin_ctzll(empty) * scan.per + i) * a.n_heads + h0;
      for (int j = lane; j < heads * (D / 8); j += 64)
        *reinterpret_cast<u32x4*>(a.out + head * D + 8 * j) = u32x4{0, 0, 0, 0};
      if (a.lse && lane < heads) a.lse[head + lane] = -__builtin_inff();
    }
  }
}

// Workgroup (unit, piece) takes its piece of the row of blocks, sequence after sequence.  The
// workgroups past the pieces write down what needs joining, and the empty sequences' outputs.
template <int QT, int KT, int D, bool ONCE>
__global__ void __launch_bounds__(kSplitWaves * 64, 2) paged_attention_kernel(Rows a,
                                                                              PagePool pool) {
  extern __shared__ float lds[];
  const int units = pool.kv_heads * a.head_tiles;
  const int unit = blockIdx.x % units, piece = blockIdx.x / units;
  const Scan scan(a.lens, a.seqs, a.cap);
  const Cuts cuts(scan.total, a.pieces);
  Unit<QT, KT, D, kSplitWaves, ONCE> u(a, pool, unit, lds);
  if (piece == a.pieces) {
    if (unit == 0 && a.pieces > 1 && wave_id() == 0) write_plan(a, scan, cuts);
    write_empty<D>(a, scan, u.h0, u.heads);
    return;
  }
  const int start = cuts.start(piece), stop = cuts.start(piece + 1);
  if (start == stop) return;
  const int from = __builtin_ctzll(__ballot(start < scan.upto));
  int base = from ? __builtin_amdgcn_readlane(scan.upto, from - 1) : 0;
  int seq = from * scan.per;
  int at = start, len = scan.per == 1 ? __builtin_amdgcn_readlane(scan.len, from)
                          : clamp_len(uniform_load(a.lens, seq), a.cap);
  while (true) {
    const int n = blocks_of(len);
    if (at < base + n) {
      const int first = at - base, end = blocks_end(stop - base, len);
      u.lane();
      u.query(seq, u.w.qf);
      u.clear();
      u.w.run(pool, u.ends, u.row(seq), first * kBlock, end, end);
      u.join(seq, first == 0 && end == len
                      ? -1 : ((int64_t)blockIdx.x * 2 + (at > start)) * a.tile_heads);
      at = min(base + n, stop);
      if (at == stop) return;
      __syncthreads();                 // the next sequence uses the same LDS
    }
    base += n;
    if (++seq >= a.seqs) return;       // lengths that changed under the launch
    len = clamp_len(uniform_load(a.lens, seq), a.cap);
  }
}

// Joins the pieces of one query head of one sequence, in their order: each set of lanes takes
// every SETS-th piece with a running maximum of its own, the sets are joined through LDS.
// 4 to 5 us, nearly all of it the launch and two dependent loads; 64, 128 or 512 threads were not
// faster.
template <int QT, int D>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(Rows a, int kv_heads,
                                                                   const float* __restrict__ v_scale) {
  constexpr int LANES = D / 4, SETS = 256 / LANES;
  __shared__ floatx4 sums[SETS][LANES];
  __shared__ float tops[SETS], totals[SETS];
  const int h = blockIdx.x, group = a.n_heads / kv_heads, kvh = h / group;
  const int4 p = a.plan[blockIdx.y];
  if (p.z == 0) return;
  const int units = kv_heads * a.head_tiles, unit = kvh * a.head_tiles + h % group / 16;
  const int set = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), total = 0.f;
#pragma unroll 4
  for (int i = set; i < p.z; i += SETS) {
    const int64_t at = (((int64_t)(p.y + i) * units + unit) * 2 + (i == 0 ? p.w : 0)) *
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
  write_out<QT, D>(a.out, a.lse, (int64_t)p.x * a.n_heads + h, 4 * lane, o, mu, total,
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
  const Split s = split_of(n_heads, kv_heads);
  return s.rows * (head_dim + 2) * 4 + 16 * s.joined(seqs);
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
      <<<(unsigned)((s.pieces + 1) * s.units), kSplitWaves * 64, kSplitWaves * wave, stream>>>(a, p);
  if (s.pieces == 1) return;           // no sequence is cut
  paged_attention_join_kernel<QT, D>
      <<<dim3(a.n_heads, (unsigned)s.joined(a.seqs)), 256, 0, stream>>>(a, p.kv_heads, p.v_scale);
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
  if (table->width > kMaxPositions / p.page_size) return MTL_ERR_SHAPE;
  const int64_t cap = table->width * p.page_size;
  if (table->seqs * ((cap + kBlock - 1) / kBlock) > INT32_MAX) return MTL_ERR_SHAPE;
  const Split s = split_of(n_heads, pool->kv_heads);
  const int d = pool->head_dim;
  const int64_t need = mtl_paged_attention_workspace_bytes(table->seqs, n_heads, pool->kv_heads, d,
                                                           table->width, p.page_size);
  const bool direct = need == 0;
  // the launch's threads, within 32 bits
  if (direct && table->seqs * s.units > UINT32_MAX / (kDirectWaves * 64)) return MTL_ERR_SHAPE;
  if (!direct && (!workspace || ws_bytes < need)) return MTL_ERR_WORKSPACE;
  if (!direct && !aligned16(workspace)) return MTL_ERR_ALIGN;
  char* ws = static_cast<char*>(workspace);
  const int64_t lists = 16 * s.joined(table->seqs);
  const Rows a{static_cast<const uint16_t*>(q), ldq, ldh, table->table, table->ld, cap, lens,
               (int)table->seqs, n_heads, s.head_tiles, s.tile_heads, s.pieces, scale,
               static_cast<uint16_t*>(out), lse, reinterpret_cast<float*>(ws + lists),
               reinterpret_cast<float*>(ws + lists + s.rows * d * 4),
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
