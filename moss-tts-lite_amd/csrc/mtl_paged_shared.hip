// Attention of one new token of each sequence over a paged key-value cache, where consecutive
// sequences form groups that hold their first positions in the same pages (gfx950).
//
// A group's shared positions are attended once for all of its queries: the query heads of one kv
// head, of all its sequences, are the columns of the matrix products, kWide of them at a time, and
// K and V of a tile of 32 positions stay in a wave's registers for all of these columns.  What a
// sequence holds by itself follows in the same launch, and a second launch joins the parts of each
// query head.
//
// * Items: (group, up to kWide columns, its shared positions) and (sequence, up to kWide query
//   heads of a kv head, its own positions), cut into blocks of 128 positions, each with a cost by
//   its columns.  They stand in one row, which the workgroups of a kv head share evenly; each
//   finds its piece on the device from lengths and groups.
// * A wave takes every fourth tile of a piece, with running maxima and sums of its own, joined
//   through LDS at a piece's end.  As soon as a product has used up K (or V) in the registers, the
//   next tile's is on its way there.
// * Groups that overlap or leave the batch give undefined results, but every index is bounded.
// * Shared positions count in multiples of 16, so that tiles begin at whole halves; the rest of a
//   shared prefix is read as the sequences' own.
#include "mtl_paged_tiles.h"

namespace mtl {

constexpr int kSharedWaves = 4;
constexpr int kSharedBlock = kTile * kSharedWaves;
constexpr int kStash = 1024;            // sequences whose lengths a workgroup keeps in LDS

// What a block costs, by its sets of 16 columns.
__host__ __device__ constexpr int block_cost(int sets) {
  return sets <= 1 ? 4 : sets <= 2 ? 6 : 10;
}

struct SharedCall {
  const uint16_t* q;
  int64_t ldq, ldh;
  const int32_t* table;
  int64_t ldt, cap;
  const int32_t* lens;
  const int32_t* groups;                // [n_groups + 1]
  const int32_t* shared;                // [n_groups]
  int seqs, n_groups, n_heads, per_kv, own_tiles, pieces, tiles;
  float scale;
  uint16_t* out;
  float* lse;
  float* whole;                         // [2][seqs * n_heads][D]: shared, own parts of whole items
  float* whole_ml;                      // (maximum, sum)
  float* cut;                           // [workgroups][2][wide][D]: first and last items of pieces
  float* cut_ml;
  int2* item_tiles;                     // first and last piece of a group's set of columns
  int2* item_own;                       // ... of a sequence's own part; (0, -1): there is none
  int2* seq_items;                      // its group's first set of columns or -1, its first column
};

struct Group {
  int begin, end, shared;               // shared: 0 where nothing is attended together
};

__device__ __forceinline__ Group group_at(const SharedCall& a, int i) {
  Group g;
  g.begin = min(max(a.groups[i], 0), a.seqs);
  g.end = min(max(a.groups[i + 1], g.begin), a.seqs);
  g.shared = g.end - g.begin > 1 ? clamp_len(a.shared[i], a.cap) & ~15 : 0;
  return g;
}

// The group of a sequence: -1 for none.
__device__ __forceinline__ int group_of(const SharedCall& a, int seq, Group& g) {
  int lo = 0, hi = a.n_groups;          // groups below lo begin at or before seq
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.groups[mid] <= seq) lo = mid + 1;
    else hi = mid;
  }
  g = Group{seq, seq + 1, 0};
  if (lo == 0) return -1;
  const Group x = group_at(a, lo - 1);
  if (seq < x.begin || seq >= x.end) return -1;
  g = x;
  return lo - 1;
}

__device__ __forceinline__ int blocks_in(int positions) {
  return (positions + kSharedBlock - 1) / kSharedBlock;
}

// The cost of `columns` columns over `blocks` blocks.
template <int WIDE>
__device__ __forceinline__ int cost_of(int columns, int blocks) {
  const int rest = columns % WIDE;
  return blocks * (columns / WIDE * block_cost(WIDE / 16) +
                   (rest ? block_cost((rest + 15) / 16) : 0));
}

// Where the items lie in the row, as every wave finds it: a lane adds up a run of groups and a run
// of sequences.
template <int WIDE>
struct Row {
  int per_group, per_seq, groups_upto, seqs_upto, shared_cost, total, pieces;

  __device__ __forceinline__ Row(const SharedCall& a, int2* stash) {
    const int lane = threadIdx.x & 63;
    per_group = (a.n_groups + 63) / 64;
    per_seq = (a.seqs + 63) / 64;
    int cost = 0;
    for (int i = 0; i < per_group; ++i) {
      const int64_t at = (int64_t)lane * per_group + i;
      if (at >= a.n_groups) break;
      const Group g = group_at(a, (int)at);
      cost += cost_of<WIDE>((g.end - g.begin) * a.per_kv, blocks_in(g.shared));
    }
    groups_upto = wave_scan(cost);
    shared_cost = __builtin_amdgcn_readlane(groups_upto, 63);
    cost = 0;
    for (int i = 0; i < per_seq; ++i) {
      const int64_t at = (int64_t)lane * per_seq + i;
      if (at >= a.seqs) break;
      const int2 own = own_of(a, (int)at);
      if (stash && at < kStash) stash[at] = own;
      cost += cost_of<WIDE>(a.per_kv, blocks_in(own.y - own.x));
    }
    seqs_upto = wave_scan(cost);
    total = shared_cost + __builtin_amdgcn_readlane(seqs_upto, 63);
    // no piece is shorter than a block
    pieces = max(1, min(a.pieces, total / block_cost(WIDE / 16)));
  }

  // A sequence's own positions [x, y).
  static __device__ __forceinline__ int2 own_of(const SharedCall& a, int seq) {
    Group g;
    group_of(a, seq, g);
    const int len = clamp_len(a.lens[seq], a.cap);
    return make_int2(min(g.shared, len), len);
  }

  __device__ __forceinline__ int start(int piece) const {
    return (int)((int64_t)piece * total / pieces);
  }
  __device__ __forceinline__ int piece_of(int at) const {
    return (int)((((int64_t)at + 1) * pieces - 1) / max(total, 1));
  }
  // The pieces that an item of `blocks` blocks of cost `each` from `base` on lies in.
  __device__ __forceinline__ int2 pieces_of(int base, int blocks, int each) const {
    return blocks ? make_int2(piece_of(base), piece_of(base + (blocks - 1) * each))
                  : make_int2(0, -1);
  }
};

// ------------------------------------------------------------------------------ a wave's work
// Up to 16 N columns over positions of one table row.
template <int QT, int KT, int D, int N>
struct Columns {
  static constexpr int E = KT == MTL_T_E4M3 ? 1 : 2;    // bytes of a stored element
  static constexpr int KL = D * E / 64;                 // 16-byte loads of a lane's K row
  static constexpr int QS = D / 32;                     // MFMA steps over the dims
  static constexpr int VD = D / 16;                     // dims of a lane's V pieces
  static constexpr int VW = VD * E / 4;                 // ... in dwords
  u32x4 qf[N][QS];
  uint32_t kf[2][KL][4];
  uint32_t vf[8][VW];
  floatx4 acc[N][VD];
  float m[N], l[N], c;                                  // c: scale to base 2
  int seen[N];                                          // positions that a lane's column attends to
  int r, g, k_lane, v_lane, v_row;

  struct Tile {                                         // two halves of 16 positions
    int page[2], rows[2];
  };
  struct Ends {
    const char* k;
    const char* v;
    int shift;
  };

  __device__ __forceinline__ void lane(const PagePool& pool) {
    const int thread = fresh(threadIdx.x);
    r = thread & 15;
    g = (thread & 63) >> 4;
    k_lane = r * (int)pool.k_token * E + 16 * g;
    v_row = (int)pool.v_token * E;
    v_lane = 4 * g * v_row + r * VD * E;
  }

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
      for (int s = 0; s < KL; ++s) load_row<false>(rows, k_lane + 64 * s, kf[h][s]);
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
      for (int j = 0; j < 4; ++j) load_row<false>(rows, v_lane + j * v_row, vf[4 * h + j]);
    }
  }

  __device__ __forceinline__ void scores(const u32x4 (&q)[QS], float (&s)[8]) const {
    floatx4 a[2] = {};
#pragma unroll
    for (int i = 0; i < KL; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t(&x)[4] = kf[h][i];
        if (E == 2)
          a[h] = mfma<QT>(u32x4{x[0], x[1], x[2], x[3]}, q[i], a[h]);
        else
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x[0]), widen<QT, true>(x[0]),
                                widen<QT, false>(x[1]), widen<QT, true>(x[1])},
                          q[(2 * i) % QS], a[h]);
      }
      if (E == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t(&x)[4] = kf[h][i];
          a[h] = mfma<QT>(u32x4{widen<QT, false>(x[2]), widen<QT, true>(x[2]),
                                widen<QT, false>(x[3]), widen<QT, true>(x[3])},
                          q[(2 * i + 1) % QS], a[h]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = a[j >> 2][j & 3] * c;
  }

  // Rows that do not count, and positions past a column's end: score -inf.
  __device__ __forceinline__ void mask(const Tile& t, int p0, int n, float (&s)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = 4 * g + (j & 3);
      s[j] = at < t.rows[j >> 2] && p0 + 16 * (j >> 2) + at < seen[n] ? s[j] : -__builtin_inff();
    }
  }

  // Running softmax of one set of columns; s becomes the weights.
  __device__ __forceinline__ void weights(int n, float (&s)[8]) {
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                      fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    top = xor32_max(xor16_max(top));
    if (__any(top > m[n])) {
      const float mn = fmaxf(m[n], top);
      const float a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
      l[n] *= a;
#pragma unroll
      for (int d = 0; d < VD; ++d) acc[n][d] *= a;
      m[n] = mn;
    }
    const float mu = m[n] == -__builtin_inff() ? 0.f : m[n];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(s[j] - mu);
    l[n] += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  }

  // V of one dim of a lane's pieces, 8 positions.
  __device__ __forceinline__ u32x4 value(int d) const {
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
    return v;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      m[n] = -__builtin_inff();
      l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < VD; ++d) acc[n][d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // This wave's tiles of positions [begin, end) for the first M sets of columns.  least: the
  // smallest `seen` of all columns.
  template <int M>
  __device__ __forceinline__ void run(const PagePool& pool, const Ends& e,
                                      const int32_t* __restrict__ row, int begin, int end,
                                      int least) {
    constexpr int kStep = kSharedWaves * kTile;
    int p0 = begin + wave_id() * kTile;
    if (p0 >= end) return;
    Tile t, next;
    ids(row, e.shift, p0, end, t);
    count(p0, end, pool.pages, t);
    load_k(pool, e, t, p0);
    load_v(pool, e, t, p0);
    while (true) {
      const int p1 = p0 + kStep;
      const bool more = p1 < end;
      ids(row, e.shift, p1, end, next);
      count(p1, end, pool.pages, next);
      float s[M][8];
#pragma unroll
      for (int n = 0; n < M; ++n) scores(qf[n], s[n]);
      if (more) load_k(pool, e, next, p1);
      if (t.rows[0] + t.rows[1] < kTile || p0 + kTile > least) {
#pragma unroll
        for (int n = 0; n < M; ++n) mask(t, p0, n, s[n]);
      }
#pragma unroll
      for (int n = 0; n < M; ++n) weights(n, s[n]);
      u32x4 hi[M], lo[M];
#pragma unroll
      for (int n = 0; n < M; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t x, y;
          two_terms<QT>(s[n][2 * j] * kLift<QT>, s[n][2 * j + 1] * kLift<QT>, x, y);
          hi[n][j] = x;
          lo[n][j] = y;
        }
#pragma unroll
      for (int d = 0; d < VD; ++d) {
        const u32x4 v = value(d);
#pragma unroll
        for (int n = 0; n < M; ++n) acc[n][d] = mfma<QT>(v, hi[n], acc[n][d]);
#pragma unroll
        for (int n = 0; n < M; ++n) acc[n][d] = mfma<QT>(v, lo[n], acc[n][d]);
      }
      if (!more) return;
      load_v(pool, e, next, p1);
      t = next;
      p0 = p1;
    }
  }
};

// ------------------------------------------------------------------------------ a workgroup
template <int QT, int KT, int D, int N>
struct Piece {
  using Wave = Columns<QT, KT, D, N>;
  static constexpr int WIDE = 16 * N, LD = D + 4;
  const SharedCall& a;
  const PagePool& pool;
  float* lds;
  int kvh;
  typename Wave::Ends ends;
  Wave w;

  __device__ __forceinline__ Piece(const SharedCall& a, const PagePool& pool, int kvh, float* lds)
      : a(a), pool(pool), lds(lds), kvh(kvh) {
    ends.shift = __builtin_ctz(pool.page_size);
    ends.k = static_cast<const char*>(pool.k) + kvh * pool.k_head * w.E;
    ends.v = static_cast<const char*>(pool.v) + kvh * pool.v_head * w.E;
    w.c = a.scale * (pool.k_scale ? uniform_load(pool.k_scale, kvh) : 1.f) * kLog2e;
  }

  // Columns c0 .. c0 + columns - 1 of the sequences from `first` on, over positions [begin, end) of
  // the row of `leader`.  whole: where the parts of an uncut item lie; cut: a cut one's.
  __device__ __forceinline__ void attend(int first, int c0, int columns, int leader, int begin,
                                         int end, float* whole, float* whole_ml, int64_t cut) {
    w.lane(pool);
    int least = INT_MAX;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = 16 * n + w.r;
      const bool there = at < columns;
      const int c = c0 + at, seq = first + (there ? c / a.per_kv : 0);
      const uint16_t* q = a.q + seq * a.ldq + (kvh * a.per_kv + c % a.per_kv) * a.ldh;
#pragma unroll
      for (int s = 0; s < w.QS; ++s) {
        const int d = w.E == 2 ? 32 * s + 8 * w.g : 64 * (s >> 1) + 16 * w.g + 8 * (s & 1);
        w.qf[n][s] = there ? *reinterpret_cast<const u32x4*>(q + d) : u32x4{0, 0, 0, 0};
      }
      w.seen[n] = there ? clamp_len(a.lens[seq], a.cap) : INT_MAX;
      least = min(least, w.seen[n]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o));
    least = __builtin_amdgcn_readfirstlane(least);
    w.clear();
    const int32_t* row = a.table + leader * a.ldt;
    const int sets = (columns + 15) / 16;
    if (N == 1 || sets == 1) w.template run<1>(pool, ends, row, begin, end, least);
    else if (N == 2 || sets == 2) w.template run<(N < 2 ? N : 2)>(pool, ends, row, begin, end, least);
    else w.template run<N>(pool, ends, row, begin, end, least);
    join(first, c0, columns, sets, whole, whole_ml, cut);
  }

  // Joins the waves through LDS, a set of columns at a time.
  __device__ __forceinline__ void join(int first, int c0, int columns, int sets, float* whole,
                                       float* whole_ml, int64_t cut) {
    float* ml = lds + kSharedWaves * 16 * LD;
    const int thread = fresh(threadIdx.x), wave = wave_id();
    const int r = thread & 15, g = (thread & 63) >> 4;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (n >= sets) break;
      const float l = xor32_add(xor16_add(w.l[n]));
      __syncthreads();                 // what was read there before
      float* o = lds + (wave * 16 + r) * LD + w.VD * 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < w.VD; d += 4)
          *reinterpret_cast<floatx4*>(o + i * w.VD + d) = floatx4{
              w.acc[n][d][i], w.acc[n][d + 1][i], w.acc[n][d + 2][i], w.acc[n][d + 3][i]};
      if (g == 0) {
        ml[2 * (wave * 16 + r)] = w.m[n];
        ml[2 * (wave * 16 + r) + 1] = l;
      }
      __syncthreads();
      const int there = min(16, columns - 16 * n);
      for (int i = thread; i < there * (D / 4); i += kSharedWaves * 64) {
        const int h = i / (D / 4), d = 4 * (i % (D / 4));
        float top = -__builtin_inff();
#pragma unroll
        for (int x = 0; x < kSharedWaves; ++x) top = fmaxf(top, ml[2 * (x * 16 + h)]);
        const float mu = top == -__builtin_inff() ? 0.f : top;
        float sum = 0.f;
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < kSharedWaves; ++x) {
          const float e = __builtin_amdgcn_exp2f(ml[2 * (x * 16 + h)] - mu);
          sum = fmaf(ml[2 * (x * 16 + h) + 1], e, sum);
          s += e * *reinterpret_cast<const floatx4*>(lds + (x * 16 + h) * LD + d);
        }
        const int at = 16 * n + h, c = c0 + at;
        const int64_t head = (int64_t)(first + c / a.per_kv) * a.n_heads + kvh * a.per_kv +
                             c % a.per_kv;
        float* to = cut < 0 ? whole + head * D : a.cut + (cut + at) * D;
        float* to_ml = cut < 0 ? whole_ml + 2 * head : a.cut_ml + 2 * (cut + at);
        *reinterpret_cast<floatx4*>(to + d) = s;
        if (d == 0) {
          to_ml[0] = top;
          to_ml[1] = sum;
        }
      }
    }
    __syncthreads();
  }

  // The table row that a group's shared positions are read through, and how many of them any of its
  // sequences reaches: the first sequence that reaches all, or else the longest.
  __device__ __forceinline__ int2 leader(const Group& g) const {
    const int lane = threadIdx.x & 63;
    int best = -1, at = g.begin;
    for (int s0 = g.begin; s0 < g.end; s0 += 64) {
      const int s = s0 + lane;
      const int len = s < g.end ? min(clamp_len(a.lens[s], a.cap), g.shared) : -1;
      int most = len;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
      most = __builtin_amdgcn_readfirstlane(most);
      if (most > best) {
        best = most;
        at = s0 + __builtin_ctzll(__ballot(len == most));
      }
      if (best == g.shared) break;
    }
    return make_int2(at, max(best, 0));
  }
};

// The blocks [x, y) of an item that fall into a piece: blocks that begin within [lo, hi).
__device__ __forceinline__ int2 blocks_within(int base, int blocks, int each, int lo, int hi) {
  const int x = lo <= base ? 0 : (lo - base + each - 1) / each;
  const int y = hi <= base ? 0 : (hi - base + each - 1) / each;
  return make_int2(min(max(x, 0), blocks), min(max(y, 0), blocks));
}

// What the second launch goes by.
template <int WIDE>
__device__ __forceinline__ void write_items(const SharedCall& a, const Row<WIDE>& row) {
  const int lane = threadIdx.x & 63;
  const int before_groups = __builtin_amdgcn_update_dpp(0, row.groups_upto, 0x138, 0xf, 0xf, false);
  const int before_seqs = __builtin_amdgcn_update_dpp(0, row.seqs_upto, 0x138, 0xf, 0xf, false);
  if (wave_id() == 0) {
    int base = before_groups;
    for (int i = 0; i < row.per_group; ++i) {
      const int64_t at = (int64_t)lane * row.per_group + i;
      if (at >= a.n_groups) break;
      const Group g = group_at(a, (int)at);
      const int blocks = blocks_in(g.shared), columns = (g.end - g.begin) * a.per_kv;
      if (!blocks) continue;
      const int id = g.begin * a.per_kv / WIDE + (int)at;
      for (int c = 0, t = 0; c < columns; c += WIDE, ++t) {
        const int each = block_cost((min(WIDE, columns - c) + 15) / 16);
        if (id + t < a.tiles) a.item_tiles[id + t] = row.pieces_of(base, blocks, each);
        base += blocks * each;
      }
    }
  } else if (wave_id() == 1) {
    int base = row.shared_cost + before_seqs;
    for (int i = 0; i < row.per_seq; ++i) {
      const int64_t at = (int64_t)lane * row.per_seq + i;
      if (at >= a.seqs) break;
      const int s = (int)at;
      Group g;
      const int group = group_of(a, s, g);
      const int len = clamp_len(a.lens[s], a.cap), blocks = blocks_in(len - min(g.shared, len));
      a.seq_items[s] = g.shared ? make_int2(g.begin * a.per_kv / WIDE + group,
                                            (s - g.begin) * a.per_kv)
                                : make_int2(-1, 0);
      for (int c = 0, t = 0; c < a.per_kv; c += WIDE, ++t) {
        const int each = block_cost((min(WIDE, a.per_kv - c) + 15) / 16);
        a.item_own[at * a.own_tiles + t] = row.pieces_of(base, blocks, each);
        base += blocks * each;
      }
    }
  }
}

template <int QT, int KT, int D, int N>
__global__ void __launch_bounds__(kSharedWaves * 64, N == 1 ? 2 : 1) paged_shared_kernel(
    SharedCall a, PagePool pool) {
  constexpr int WIDE = 16 * N;
  __shared__ float lds[kSharedWaves * 16 * (D + 4) + 2 * kSharedWaves * 16];
  __shared__ int2 stash[kStash];
  const int units = pool.kv_heads;
  const int kvh = blockIdx.x % units, piece = blockIdx.x / units;
  const Row<WIDE> row(a, wave_id() == 0 ? stash : nullptr);
  if (piece == a.pieces) {
    if (kvh == 0) write_items<WIDE>(a, row);
    return;
  }
  if (piece >= row.pieces || row.total <= 0) return;
  __syncthreads();
  const int lo = row.start(piece), hi = row.start(piece + 1);
  if (lo >= hi) return;
  Piece<QT, KT, D, N> p(a, pool, kvh, lds);
  const int64_t slot = (int64_t)blockIdx.x * 2 * WIDE;
  const int64_t heads = (int64_t)a.seqs * a.n_heads;
  if (lo < row.shared_cost) {
    const int from = __builtin_ctzll(__ballot(lo < row.groups_upto));
    int base = from ? __builtin_amdgcn_readlane(row.groups_upto, from - 1) : 0;
    for (int64_t i = (int64_t)from * row.per_group; i < a.n_groups && base < hi; ++i) {
      const Group g = group_at(a, (int)i);
      const int blocks = blocks_in(g.shared), columns = (g.end - g.begin) * a.per_kv;
      const int cost = cost_of<WIDE>(columns, blocks);
      if (base + cost > lo) {
        const int2 lead = p.leader(g);
        const int full = blocks * block_cost(N);
        const int skip = lo > base ? max(min((lo - base) / full, columns / WIDE), 0) : 0;
        int at = base + skip * full;
        for (int c = skip * WIDE; c < columns && at < hi; c += WIDE) {
          const int n = min(WIDE, columns - c), each = block_cost((n + 15) / 16);
          const int2 b = blocks_within(at, blocks, each, lo, hi);
          if (b.x < b.y)
            p.attend(g.begin, c, n, lead.x, b.x * kSharedBlock,
                     min(b.y * kSharedBlock, lead.y), a.whole, a.whole_ml,
                     b.x == 0 && b.y == blocks ? -1 : slot + (b.x == 0) * WIDE);
          at += blocks * each;
        }
      }
      base += cost;
    }
  }
  if (hi > row.shared_cost) {
    const int from = lo <= row.shared_cost
                         ? 0 : __builtin_ctzll(__ballot(lo < row.shared_cost + row.seqs_upto));
    int base = row.shared_cost +
               (from ? __builtin_amdgcn_readlane(row.seqs_upto, from - 1) : 0);
    for (int64_t s = (int64_t)from * row.per_seq; s < a.seqs && base < hi; ++s) {
      int2 own = s < kStash ? stash[s] : Row<WIDE>::own_of(a, (int)s);
      own.x = __builtin_amdgcn_readfirstlane(own.x);
      own.y = __builtin_amdgcn_readfirstlane(own.y);
      const int blocks = blocks_in(own.y - own.x);
      for (int c = 0; c < a.per_kv; c += WIDE) {
        const int n = min(WIDE, a.per_kv - c), each = block_cost((n + 15) / 16);
        const int2 b = blocks_within(base, blocks, each, lo, hi);
        if (b.x < b.y)
          p.attend((int)s, c, n, (int)s, own.x + b.x * kSharedBlock,
                   min(own.x + b.y * kSharedBlock, own.y), a.whole + heads * D,
                   a.whole_ml + 2 * heads,
                   b.x == 0 && b.y == blocks ? -1 : slot + (b.x == 0) * WIDE);
        base += blocks * each;
      }
    }
  }
}

// Joins the parts of each query head: LANES lanes a head, the shared part's pieces in their order,
// then its own.
template <int QT, int D, int WIDE>
__global__ void __launch_bounds__(256) paged_shared_join_kernel(SharedCall a, int kv_heads,
                                                                const float* __restrict__ v_scale) {
  constexpr int LANES = D / 4, HEADS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t heads = (int64_t)a.seqs * a.n_heads;
  const int64_t head = (int64_t)blockIdx.x * HEADS + threadIdx.x / LANES;
  if (head >= heads) return;
  const int seq = (int)(head / a.n_heads), h = (int)(head % a.n_heads);
  const int kvh = h / a.per_kv, hc = h % a.per_kv;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), total = 0.f;
  auto add = [&](const float* part, const float* ml) {
    const float2 x = *reinterpret_cast<const float2*>(ml);
    const floatx4 y = *reinterpret_cast<const floatx4*>(part + 4 * lane);
    const float t = fmaxf(top, x.x), mu = t == -__builtin_inff() ? 0.f : t;
    const float e0 = __builtin_amdgcn_exp2f(top - mu), e1 = __builtin_amdgcn_exp2f(x.x - mu);
    total = total * e0 + x.y * e1;
    o = o * e0 + y * e1;
    top = t;
  };
  auto item = [&](int2 pieces, int64_t whole, int column) {
    if (pieces.x == pieces.y) {
      add(a.whole + whole * D, a.whole_ml + 2 * whole);
      return;
    }
    const int last = min(pieces.y, a.pieces - 1);
#pragma unroll 4
    for (int p = max(pieces.x, 0); p <= last; ++p) {
      const int64_t at = (((int64_t)p * kv_heads + kvh) * 2 + (p == pieces.x)) * WIDE + column;
      add(a.cut + at * D, a.cut_ml + 2 * at);
    }
  };
  const int2 own = a.item_own[(int64_t)seq * a.own_tiles + hc / WIDE], in = a.seq_items[seq];
  if (in.x >= 0) {
    const int c = in.y + hc, id = in.x + c / WIDE;
    if (id < a.tiles) item(a.item_tiles[id], head, c % WIDE);
  }
  if (own.y >= own.x) item(own, heads + head, hc % WIDE);
  write_out<QT, D>(a.out, a.lse, head, 4 * lane, o, top == -__builtin_inff() ? 0.f : top, total,
                   v_scale ? v_scale[kvh] : 1.f);
}

// How a call is laid out.
struct SharedPlan {
  int sets, wide, own_tiles, pieces;
  int64_t tiles, rows;                   // rows: of parts
};

static SharedPlan shared_plan(int64_t seqs, int64_t groups, int n_heads, int kv_heads) {
  SharedPlan p;
  const int64_t per_kv = n_heads / kv_heads, columns = seqs * per_kv;
  p.sets = columns <= 16 ? 1 : columns <= 32 ? 2 : 4;
  p.wide = 16 * p.sets;
  p.own_tiles = (int)((per_kv + p.wide - 1) / p.wide);
  const int workgroups = p.sets == 1 ? 512 : 256;
  p.pieces = kv_heads < workgroups ? workgroups / kv_heads : 1;
  p.tiles = columns / p.wide + groups + 1;
  p.rows = 2 * seqs * n_heads + (int64_t)p.pieces * kv_heads * 2 * p.wide;
  return p;
}

template <int QT, int KT, int D>
static void launch_shared(const SharedCall& a, const PagePool& p, const SharedPlan& s,
                          hipStream_t stream) {
  const unsigned grid = (unsigned)((s.pieces + 1) * p.kv_heads);
  const unsigned joins = (unsigned)(((int64_t)a.seqs * a.n_heads * (D / 4) + 255) / 256);
#define MTL_RUN(N)                                                                          \
  do {                                                                                      \
    paged_shared_kernel<QT, KT, D, N><<<grid, kSharedWaves * 64, 0, stream>>>(a, p);        \
    paged_shared_join_kernel<QT, D, 16 * N><<<joins, 256, 0, stream>>>(a, p.kv_heads,       \
                                                                       p.v_scale);          \
  } while (0)
  if (s.sets == 1) MTL_RUN(1);
  else if (s.sets == 2) MTL_RUN(2);
  else MTL_RUN(4);
#undef MTL_RUN
}

}  // namespace mtl

using namespace mtl;

static bool shared_sizes_ok(int64_t seqs, int64_t groups, int32_t n_heads, int32_t kv_heads,
                            int64_t width, int32_t page_size) {
  if (seqs < 0 || groups < 0 || groups > 65535 || seqs > 65535 || kv_heads < 1 || n_heads < 1 ||
      n_heads % kv_heads || n_heads > 65535 || width < 0 || page_size < 1 ||
      width > kMaxPositions / page_size)
    return false;
  if (seqs == 0) return true;
  const SharedPlan p = shared_plan(seqs, groups, n_heads, kv_heads);
  // the row of all items' blocks, and the launches' threads, within 32 bits
  const int64_t blocks = (width * page_size + kSharedBlock - 1) / kSharedBlock;
  const int64_t items = p.tiles + seqs * p.own_tiles;
  return items <= INT32_MAX / block_cost(4) / (blocks + 1) &&
         seqs * n_heads <= (int64_t)UINT32_MAX / 64 && (int64_t)(p.pieces + 1) * kv_heads <= 1 << 23;
}

extern "C" int64_t mtl_paged_attention_shared_workspace_bytes(int64_t seqs, int64_t groups,
                                                              int32_t n_heads, int32_t kv_heads,
                                                              int32_t head_dim, int64_t width,
                                                              int32_t page_size) {
  if (seqs < 1 || head_dim < 1 ||
      !shared_sizes_ok(seqs, groups, n_heads, kv_heads, width, page_size))
    return 0;
  const SharedPlan p = shared_plan(seqs, groups, n_heads, kv_heads);
  return p.rows * (head_dim + 2) * 4 + 8 * (p.tiles + seqs * (p.own_tiles + 1));
}

extern "C" int mtl_paged_attention_shared(const void* q, int64_t ldq, int64_t ldh,
                                          const mtl_page_pool* pool, const mtl_page_table* table,
                                          const int32_t* lens, const int32_t* groups,
                                          const int32_t* shared, int64_t n_groups, int32_t n_heads,
                                          int32_t q_type, float scale, void* out, float* lse,
                                          void* workspace, int64_t ws_bytes, void* stream) {
  PagePool p;
  const int st = check_pool(pool, table, q_type, p);
  if (st != MTL_OK) return st;
  if (!shared_sizes_ok(table->seqs, n_groups, n_heads, pool->kv_heads, table->width, p.page_size))
    return MTL_ERR_SHAPE;
  if (table->seqs == 0) return MTL_OK;
  if (!q || !lens || !out || !groups || (n_groups > 0 && !shared)) return MTL_ERR_INVALID_ARG;
  if (ldq % 8 || ldh % 8 || !aligned16(q) || !aligned16(out)) return MTL_ERR_ALIGN;
  const int64_t most = INT32_MAX / 64;   // a lane's offset within a page, within 31 bits
  if (p.k_token > most || p.v_token > most) return MTL_ERR_SHAPE;
  const int d = pool->head_dim;
  const int64_t seqs = table->seqs, heads = seqs * n_heads;
  if (!workspace || ws_bytes < mtl_paged_attention_shared_workspace_bytes(
                                   seqs, n_groups, n_heads, pool->kv_heads, d, table->width,
                                   p.page_size))
    return MTL_ERR_WORKSPACE;
  if (!aligned16(workspace)) return MTL_ERR_ALIGN;
  const SharedPlan s = shared_plan(seqs, n_groups, n_heads, pool->kv_heads);
  float* parts = static_cast<float*>(workspace);
  float* ml = parts + s.rows * d;
  int2* items = reinterpret_cast<int2*>(ml + 2 * s.rows);
  const SharedCall a{static_cast<const uint16_t*>(q), ldq, ldh, table->table, table->ld,
                     table->width * p.page_size, lens, groups, shared, (int)seqs, (int)n_groups,
                     n_heads, n_heads / pool->kv_heads, s.own_tiles, s.pieces, (int)s.tiles, scale,
                     static_cast<uint16_t*>(out), lse, parts, ml, parts + 2 * heads * d,
                     ml + 4 * heads, items, items + s.tiles, items + s.tiles + seqs * s.own_tiles};
#define MTL_RUN(T, KT, D) launch_shared<T, KT, D>(a, p, s, (hipStream_t)stream)
  MTL_PAGED_CASES(MTL_RUN, q_type, pool->type, d);
#undef MTL_RUN
  return launch_status();
}
