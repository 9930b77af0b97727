// Attention of one new token of each sequence over a paged key-value cache, where consecutive
// sequences form groups that hold their first positions in the same pages (gfx950).
//
// A group's shared positions are attended for all of its queries together: the query heads of one
// kv head, of all its sequences, are the columns of the matrix products, up to kWide at a time, and
// each kWide columns read the K and V once (with kWide query heads to a kv head a sequence fills
// them, and nothing is read together).  What a sequence holds by itself follows in the same launch,
// and a second launch joins the parts of each query head.  Products, softmax and the two-term
// weights are those of mtl_paged_attention.
//
// * Items: (group, up to kWide columns, its shared positions) and (sequence, up to kWide query
//   heads of a kv head, its own positions), cut into blocks of 128 positions, each with a cost by
//   its columns.  They stand in one row, which the workgroups of a kv head share evenly; each
//   finds its piece on the device from lengths and groups, which it keeps in LDS where there is
//   room.
// * Up to kNarrow columns: a wave takes every fourth tile of 32 positions, K and V in registers, with
//   running maxima and sums of its own, joined through LDS at a piece's end.  As soon as a product
//   has used up K (or V) in the registers, the next tile's is on its way there.  More columns would
//   spill, or read every tile for each 32 of them.
// * Up to kWide columns: tiles of kStage positions pass through LDS; two waves take half of the
//   columns each, two the other half of the positions.
// * Groups whose numbers do not ascend are not there, and numbers past the batch count as its end: so
//   groups never overlap, which the sum of all costs needs to stay within 32 bits.
// * Shared positions count in multiples of 16, so that tiles begin at whole halves; the rest of a
//   shared prefix is read as the sequences' own.
// * A short prefix of few sequences stays with the sequences (Batch::group): an item of its own
//   costs more than what is read again from the L2 (13 us by themselves, 20 shared).
//
// Measured, head_dim 128, bf16, 32 heads over 8 kv heads, the two launches in a kernel trace: 192
// sequences on a prefix of 6001 positions and up to 700 of their own (121 MB of K and V once; 19
// GFLOP) 83 + 6 us (77 for a whole call outside of the trace), where the matrix rate would take 16
// and memory 17; 16 sentences with up to 6 candidates (67 MB) 24 + 5; prefixes in e4m3 (51 MB)
// 25 + 4; head_dim 64 in f16, 3 groups, 19 + 5; two sequences of 700 positions 9 + 4.
// * A tile of 64 positions by 64 columns takes some 3600 cycles, of which vector instructions are
//   issued in 85 of 100 and the matrix units work in 25 to 40.  A wave has 48 matrix and some 250
//   vector instructions for it, with 16 scores a lane: 95 for maxima, exponentials and sums, 48 for
//   the weights' two terms, 32 for V's bytes, 75 for pages, addresses and staging; and 41 more for
//   each 16 columns whose sums are brought to a new maximum.
// * By the items' costs the sequences' own parts are 41 of 100 of all work of the 192 sequences, 74
//   of the candidates, 53 of the e4m3 case and 50 of the two sequences, and some 70 of 100 of that
//   is what an item costs by itself: a workgroup takes 1 or 2 blocks by 4 columns, clears four waves'
//   sums and joins them twice through LDS.
// * About 18 000 cycles of a piece do not grow with it (lists, queries, first tile; joining).
// * Past 512 sequences or groups the lists do not fit LDS and every workgroup looks for each
//   sequence's group in memory.  By groups of 16 on 600 positions and up to 200 of their own, 1024
//   sequences take 218 us; of 16 on 300 and up to 100, 4096 sequences 797.
// mtl_paged_attention on the same inputs, a call: 500 us for the 192 sequences (77 here), 32 for
// the candidates (27), 55 in e4m3 (27), 19.5 for head_dim 64 (23.2), 7.9 for the two sequences
// (12.1), 418 and 965 for the 1024 and 4096 (218, 797).
//
// Tried and slower: 64 columns a wave with K and V straight from the caches (222 us for the 192
// sequences), 128-column tiles of 4 waves (ahead past some 20 000 positions only, 154 against 160 us,
// and behind below), page ids by scalar loads, 384, 768 and 1024 workgroups (768 takes many
// small groups at head_dim 64 from 89 to 70 us and others from 23 to 30).
#include "mtl_paged_items.h"
#include "mtl_paged_tiles.h"

namespace mtl {

constexpr int kSharedWaves = 4;
static_assert(kSharedBlock == kTile * kSharedWaves, "a tile of each wave");
constexpr int kStage = 64;              // positions of a tile in LDS
constexpr int kSharedWorkgroups = 512;  // 2 on each of 256 CUs: all their registers' room
// Tables up to which, and sequences times kv heads (and 16 query heads) up to which a sequence by
// itself is faster: one launch instead of two, and what is read again comes from the L2s.  Both
// sides measured in us, head_dim 128, bf16, 300 shared of 400 positions in one group: 2 sequences of
// 80 positions 9.9 (12.5 shared), 16 of 32 heads over 8 10.0 (15.3), 64 13.4 (19.5); 400 of 450
// positions in groups of 4, 64 sequences 17.1 (20.1), 128 32.8 (28.5), 256 63.4 (55.6).
constexpr int kShortTable = 512;
constexpr int kShortUnits = 512;
constexpr int kStash = 512;             // sequences and groups that a workgroup keeps in LDS

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

// Lengths and groups: in LDS where there is room, since everything that is decided from them waits
// for one entry after the other.
struct Lists {
  int lens[kStash], groups[kStash + 1], shared[kStash];
  int2 own[kStash];                     // a sequence's own positions [x, y)
  int falls[kSharedWaves];              // of each wave: whether a group begins behind its end
};

struct Batch {
  const SharedCall& a;
  Lists& l;
  int wide;                             // columns of an item, at most
  bool near;
  int n_groups;                         // 0 where they do not ascend

  __device__ __forceinline__ Batch(const SharedCall& a, Lists& l, int wide)
      : a(a), l(l), wide(wide), near(a.seqs <= kStash && a.n_groups <= kStash) {
    bool falls = false;
    const int entries = near ? max(a.seqs, a.n_groups + 1) : a.n_groups;
    for (int i = threadIdx.x; i < entries; i += kSharedWaves * 64) {
      if (i < a.n_groups) falls |= a.groups[i] > a.groups[i + 1];
      if (!near) continue;
      if (i < a.seqs) l.lens[i] = clamp_len(a.lens[i], a.cap);
      if (i <= a.n_groups) l.groups[i] = a.groups[i];
      if (i < a.n_groups) l.shared[i] = a.shared[i];
    }
    const bool any = __any(falls);
    if ((threadIdx.x & 63) == 0) l.falls[wave_id()] = any;
    __syncthreads();
    int found = 0;
#pragma unroll
    for (int i = 0; i < kSharedWaves; ++i) found |= l.falls[i];
    n_groups = __builtin_amdgcn_readfirstlane(found) ? 0 : a.n_groups;
    if (!near) return;
    for (int i = threadIdx.x; i < a.seqs; i += kSharedWaves * 64) l.own[i] = find_own(i);
    __syncthreads();
  }

  __device__ __forceinline__ int len(int s) const {
    return near ? l.lens[s] : clamp_len(a.lens[s], a.cap);
  }
  __device__ __forceinline__ int start(int i) const { return near ? l.groups[i] : a.groups[i]; }

  __device__ __forceinline__ Group group(int i) const {
    Group g;
    g.begin = min(max(start(i), 0), a.seqs);
    g.end = min(max(start(i + 1), g.begin), a.seqs);
    g.shared = clamp_len(near ? l.shared[i] : a.shared[i], a.cap) & ~15;
    // Few sequences with a short prefix read it for themselves, where that costs no more.
    const int n = g.end - g.begin, blocks = blocks_in(g.shared);
    if (cost_of(n * a.per_kv, blocks, wide) >= n * blocks * block_cost(min(a.per_kv, wide)))
      g.shared = 0;
    return g;
  }

  // The group of a sequence: -1 for none.
  __device__ __forceinline__ int group_of(int seq, Group& g) const {
    int lo = 0, hi = n_groups;          // groups below lo begin at or before seq
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= seq) lo = mid + 1;
      else hi = mid;
    }
    g = Group{seq, seq + 1, 0};
    if (lo == 0) return -1;
    const Group x = group(lo - 1);
    if (seq < x.begin || seq >= x.end) return -1;
    g = x;
    return lo - 1;
  }

  __device__ __forceinline__ int2 find_own(int seq) const {
    Group g;
    group_of(seq, g);
    const int n = len(seq);
    return make_int2(min(g.shared, n), n);
  }
  __device__ __forceinline__ int2 own_of(int seq) const {
    return near ? l.own[seq] : find_own(seq);
  }
};

// Where the items lie in the row, as every wave finds it: a lane adds up a run of groups and a run
// of sequences.
template <int WIDE>
struct Row {
  int per_group, per_seq, groups_upto, seqs_upto, shared_cost, total, pieces;
  Pieces cut;

  __device__ __forceinline__ Row(const SharedCall& a, const Batch& batch) {
    const int lane = threadIdx.x & 63;
    per_group = (batch.n_groups + 63) / 64;
    per_seq = (a.seqs + 63) / 64;
    int cost = 0, widest = min(a.per_kv, WIDE);
    for (int i = 0; i < per_group; ++i) {
      const int64_t at = (int64_t)lane * per_group + i;
      if (at >= batch.n_groups) break;
      const Group g = batch.group((int)at);
      const int columns = (g.end - g.begin) * a.per_kv;
      cost += cost_of(columns, blocks_in(g.shared), WIDE);
      if (g.shared) widest = max(widest, min(columns, WIDE));
    }
    const int most = block_cost(__builtin_amdgcn_readfirstlane((int)wave_max_valu((float)widest)));
    groups_upto = wave_scan(cost);
    shared_cost = __builtin_amdgcn_readlane(groups_upto, 63);
    cost = 0;
    for (int i = 0; i < per_seq; ++i) {
      const int64_t at = (int64_t)lane * per_seq + i;
      if (at >= a.seqs) break;
      const int2 own = batch.own_of((int)at);
      cost += cost_of(a.per_kv, blocks_in(own.y - own.x), WIDE);
    }
    seqs_upto = wave_scan(cost);
    total = shared_cost + __builtin_amdgcn_readlane(seqs_upto, 63);
    // no piece is shorter than a block
    pieces = max(1, min(a.pieces, total / most));
    cut.each = total / pieces;
    cut.longer = total - cut.each * pieces;
  }

  __device__ __forceinline__ int2 pieces_of(int base, int blocks, int columns) const {
    const Span x = cut.pieces_of(base, blocks, columns);
    return make_int2(x.x, x.y);
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
  int k_place, v_place;                                 // of a lane's first pieces in LDS
  int at_run, token_bytes;                              // of the run that a lane finds
  uint64_t base, page_bytes;

  // Where the rows of a tile lie.  A tile is up to four runs of 16 positions, each in one page; lane
  // i finds run i % 4 in K (i / 4 even) or in V, in vector registers: for each run anew in scalar
  // ones it is 130 instructions a tile, a third of all the wave's.
  struct Where {
    uint32_t lo, hi;
    int bytes, rows;
  };

  __device__ __forceinline__ void lane(const PagePool& pool, const char* k, const char* v) {
    const int thread = fresh(threadIdx.x);
    r = thread & 15;
    g = (thread & 63) >> 4;
    k_lane = r * (int)pool.k_token * E + 16 * g;
    v_row = (int)pool.v_token * E;
    v_lane = 4 * g * v_row + r * VD * E;
    k_place = r * RB + ((g ^ swap(r)) << 4);
    const int bytes = r * VD * E;
    v_place = 4 * g * RB + (((bytes >> 4) ^ swap(4 * g)) << 4) + (bytes & 15);
    const bool of_v = thread & 4;
    at_run = (thread & 3) * 16;
    base = reinterpret_cast<uintptr_t>(of_v ? v : k);
    page_bytes = (of_v ? pool.v_page : pool.k_page) * E;
    token_bytes = (int)(of_v ? pool.v_token : pool.k_token) * E;
  }

  // The page of the lane's run of the tile at p0 < end.
  __device__ __forceinline__ int page_id(const int32_t* __restrict__ row, int shift, int p0,
                                         int end) const {
    return row[max(min(p0 + at_run, end - 1), 0) >> shift];
  }

  __device__ __forceinline__ Where where(const PagePool& pool, int page, int p0, int end) const {
    const int p = p0 + at_run;
    Where x;
    x.rows = (uint32_t)page < (uint32_t)pool.pages ? min(max(end - p, 0), 16) : 0;
    const uint64_t at = base + (uint64_t)(uint32_t)(x.rows ? page : 0) * page_bytes +
                        (uint64_t)(p & (pool.page_size - 1)) * (uint32_t)token_bytes;
    x.lo = (uint32_t)at;
    x.hi = (uint32_t)(at >> 32) & 0xffffu;
    x.bytes = x.rows * token_bytes;
    return x;
  }

  static __device__ __forceinline__ Rsrc rows_of(const Where& x, int i) {
    const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(x.hi, i) << 32 |
                        (uint32_t)__builtin_amdgcn_readlane(x.lo, i);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(at), 0,
                                             __builtin_amdgcn_readlane(x.bytes, i), 0x00027000);
  }

  __device__ __forceinline__ void load_k(const Where& x) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Rsrc rows = rows_of(x, h);
#pragma unroll
      for (int s = 0; s < KL; ++s) load_row<false>(rows, k_lane + 64 * s, kf[h][s]);
    }
  }

  __device__ __forceinline__ void load_v(const Where& x) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Rsrc rows = rows_of(x, 4 + h);
#pragma unroll
      for (int j = 0; j < 4; ++j) load_row<false>(rows, v_lane + j * v_row, vf[4 * h + j]);
    }
  }

  // Two chains of products a set, all in turn.
  template <int M>
  __device__ __forceinline__ void scores(float (&s)[M][8]) const {
    floatx4 a[M][2] = {};
#pragma unroll
    for (int i = 0; i < KL; ++i) {
#pragma unroll
      for (int part = 0; part < (E == 2 ? 1 : 2); ++part) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t(&x)[4] = kf[h][i];
          const uint32_t x0 = x[2 * part], x1 = x[2 * part + 1];
          const u32x4 k = E == 2 ? u32x4{x[0], x[1], x[2], x[3]}
                                 : u32x4{widen<QT, false>(x0), widen<QT, true>(x0),
                                         widen<QT, false>(x1), widen<QT, true>(x1)};
#pragma unroll
          for (int n = 0; n < M; ++n)
            a[n][h] = mfma<QT>(k, qf[n][E == 2 ? i : (2 * i + part) % QS], a[n][h]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < M; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[n][j] = a[n][j >> 2][j & 3];
  }

  // Rows that do not count, and positions past a column's end: score -inf.
  __device__ __forceinline__ void mask(int rows0, int rows1, int p0, int n, float (&s)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = 4 * g + (j & 3);
      s[j] = at < (j < 4 ? rows0 : rows1) && p0 + 16 * (j >> 2) + at < seen[n] ? s[j]
                                                                               : -__builtin_inff();
    }
  }

  // Running softmax of one set of columns; s, products of q and k, become the weights.  The factor c
  // is above 0, so the largest product is the largest score.
  __device__ __forceinline__ void weights(int n, float (&s)[8]) {
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), s[2]), fmaxf(fmaxf(s[3], s[4]), s[5]));
    top = fmaxf(fmaxf(top, s[6]), s[7]);
    top = xor32_max(xor16_max(top)) * c;
    // in bf16 weights may grow to 2^8 before all sums are brought to the new maximum (f16 has no
    // room above 1): pieces are short, and the maximum grows in nearly every tile of one
    if (__any(top > m[n] + (QT == MTL_T_BF16 ? 8.f : 0.f))) {
      const float mn = fmaxf(m[n], top);
      const float a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
      l[n] *= a;
#pragma unroll
      for (int d = 0; d < VD; ++d) acc[n][d] *= a;
      m[n] = mn;
    }
    const float mu = m[n] == -__builtin_inff() ? 0.f : m[n];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c, -mu));
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

  // 32 positions from p0 on, in kf and vf, for M sets of columns.  rows0, rows1: how many of each 16
  // count; least: the smallest `seen` of all columns; k_done is called when kf is used up.
  template <int M, class F>
  __device__ __forceinline__ void tile(int rows0, int rows1, int p0, int least, F&& k_done) {
    float s[M][8];
    scores<M>(s);
    k_done();
    if (rows0 + rows1 < kTile || p0 + kTile > least) {
#pragma unroll
      for (int n = 0; n < M; ++n) mask(rows0, rows1, p0, n, s[n]);
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
    for (int d = 0; d < VD; d += 2) {     // no product waits for the one before
      const u32x4 v0 = value(d), v1 = value(d + 1);
#pragma unroll
      for (int n = 0; n < M; ++n) {
        acc[n][d] = mfma<QT>(v0, hi[n], acc[n][d]);
        acc[n][d + 1] = mfma<QT>(v1, hi[n], acc[n][d + 1]);
      }
#pragma unroll
      for (int n = 0; n < M; ++n) {
        acc[n][d] = mfma<QT>(v0, lo[n], acc[n][d]);
        acc[n][d + 1] = mfma<QT>(v1, lo[n], acc[n][d + 1]);
      }
    }
  }

  // This wave's tiles from p0 to `end`, every fourth, for M sets of columns.  page0, page: of the
  // first two.
  template <int M>
  __device__ __forceinline__ void run(const PagePool& pool, const int32_t* __restrict__ row,
                                      int shift, int p0, int end, int least, int page0, int page) {
    constexpr int kStep = kSharedWaves * kTile;
    if (p0 >= end) return;
    Where x = where(pool, page0, p0, end);
    load_k(x);
    load_v(x);
    while (true) {
      const int p1 = p0 + kStep;
      const int rows0 = __builtin_amdgcn_readlane(x.rows, 0);
      const int rows1 = __builtin_amdgcn_readlane(x.rows, 1);
      if (p1 < end) {
        x = where(pool, page, p1, end);
        page = page_id(row, shift, p1 + kStep, end);
      }
      tile<M>(rows0, rows1, p0, least, [&] { if (p1 < end) load_k(x); });
      if (p1 >= end) return;
      load_v(x);
      p0 = p1;
    }
  }

  // --- tiles of kStage positions in LDS, which all waves of the workgroup go through, each with
  // columns of its own.  Pieces of 16 bytes of a row lie in an order that goes by the row, so that
  // 16 lanes that read one piece of 16 rows (K), or one row (V), meet all banks once.
  static constexpr int RB = D * E, PIECES = RB / 16, LOADS = kStage * PIECES / 256;
  static constexpr int kStageBytes = kStage * RB;       // of K, and again of V

  // What a row's pieces are exchanged by; rows 16 apart have the same.
  static __device__ __forceinline__ int swap(int row) { return row / (256 / RB) & (PIECES - 1); }

  // A wave brings one run of 16 rows of K (or V), 1 KB at a time; x[i] goes to LDS in its place.
  __device__ __forceinline__ void fetch(const Where& t, int run, int token, uint32_t (&x)[LOADS][4])
      const {
    const int lane = fresh(threadIdx.x) & 63, row = lane / PIECES;
    const Rsrc rows = rows_of(t, run);
    const int at = row * token * E, piece = ((lane % PIECES) ^ swap(row)) << 4;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)     // rows 64 / PIECES apart exchange by 4 more
      load_row<false>(rows, at + (piece ^ (i << 6)) + i * (64 / PIECES) * token * E, x[i]);
  }

  __device__ __forceinline__ void put(char* to, const uint32_t (&x)[LOADS][4]) const {
    char* mine = to + wave_id() * 16 * RB + (fresh(threadIdx.x) & 63) * 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *reinterpret_cast<u32x4*>(mine + i * 1024) = u32x4{x[i][0], x[i][1], x[i][2], x[i][3]};
  }

  // kf (vf) of 32 positions from row `first` of the tile on.  Addresses are formed anew from two
  // that a lane keeps: all of them, kept over the loop, do not fit the registers.
  __device__ __forceinline__ void take_k(const char* k, int first) {
    const int at = fresh(k_place);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < KL; ++s) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(k + (at ^ s << 6) + (first + 16 * h) * RB);
        kf[h][s][0] = x.x; kf[h][s][1] = x.y; kf[h][s][2] = x.z; kf[h][s][3] = x.w;
      }
  }

  __device__ __forceinline__ void take_v(const char* v, int first) {
    const int at = fresh(v_place);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = j & 3, other = PIECES == 16 ? row : PIECES == 8 ? row >> 1 : 0;
      const char* from = v + (at ^ other << 4) + (first + 16 * (j >> 2) + row) * RB;
      if (VW == 4) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = x[w];
      } else if (VW == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(from);
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = x[w];
      } else {
        vf[j][0] = *reinterpret_cast<const uint32_t*>(from);
      }
    }
  }

  // Positions [begin, end): of each tile in LDS this wave takes the first or second 32.
  __device__ __forceinline__ void run_wide(const PagePool& pool, const int32_t* __restrict__ row,
                                           int shift, int begin, int end, int least, int half,
                                           char* lds, int page0, int page) {
    if (begin >= end) return;
    uint32_t kx[LOADS][4], vx[LOADS][4];
    Where x = where(pool, page0, begin, end);
    fetch(x, wave_id(), (int)pool.k_token, kx);
    fetch(x, 4 + wave_id(), (int)pool.v_token, vx);
    __syncthreads();                    // what was read there before
    put(lds, kx);
    put(lds + kStageBytes, vx);
    __syncthreads();
    int buffer = 0;
    for (int p0 = begin; p0 < end; p0 += kStage) {
      const int p1 = p0 + kStage;
      const bool more = p1 < end;
      const int rows0 = __builtin_amdgcn_readlane(x.rows, 2 * half);
      const int rows1 = __builtin_amdgcn_readlane(x.rows, 2 * half + 1);
      if (more) {
        x = where(pool, page, p1, end);
        page = page_id(row, shift, p1 + kStage, end);
        fetch(x, wave_id(), (int)pool.k_token, kx);
        fetch(x, 4 + wave_id(), (int)pool.v_token, vx);
      }
      const char* k = lds + buffer * 2 * kStageBytes;
      take_k(k, 32 * half);
      tile<N>(rows0, rows1, p0 + 32 * half, least, [&] { take_v(k + kStageBytes, 32 * half); });
      buffer ^= 1;
      if (more) {
        put(lds + buffer * 2 * kStageBytes, kx);
        put(lds + buffer * 2 * kStageBytes + kStageBytes, vx);
      }
      __syncthreads();
    }
  }
};

// ------------------------------------------------------------------------------ a workgroup
template <int QT, int KT, int D, int N>
struct Piece {
  using Wave = Columns<QT, KT, D, N>;
  // LDS of two waves' sums, or of two tiles of K and V
  static constexpr int kSumBytes = N * 64 * (Wave::VD * 16 + 8);
  static constexpr int kJoinBytes = 2 * kSumBytes;
  static constexpr int kBytes = N > 1 && 4 * Wave::kStageBytes > kJoinBytes ? 4 * Wave::kStageBytes
                                                                            : kJoinBytes;
  const SharedCall& a;
  const Batch& batch;
  const PagePool& pool;
  char* lds;
  int kvh;
  float by;                             // 1 / per_kv
  const char* k_end;                    // the kv head's K and V in the first page
  const char* v_end;
  int shift;
  uint32_t sign;
  Wave w;

  __device__ __forceinline__ Piece(const Batch& batch, const PagePool& pool, int kvh, char* lds)
      : a(batch.a), batch(batch), pool(pool), lds(lds), kvh(kvh), by(1.f / batch.a.per_kv) {
    shift = __builtin_ctz(pool.page_size);
    k_end = static_cast<const char*>(pool.k) + kvh * pool.k_head * w.E;
    v_end = static_cast<const char*>(pool.v) + kvh * pool.v_head * w.E;
    // a factor below 0 is the queries' sign; 0 is as good as the smallest number, beside which a
    // masked -infinity stays one
    const float c = a.scale * (pool.k_scale ? uniform_load(pool.k_scale, kvh) : 1.f) * kLog2e;
    sign = c < 0.f ? 0x80008000u : 0u;
    w.c = fmaxf(fabsf(c), 0x1p-126f);
  }

  // n / per_kv for n < 2^20: (n + 1/2) / per_kv lies further from a whole number than float32 is off.
  __device__ __forceinline__ int sequences_in(int n) const { return (int)((n + 0.5f) * by); }

  // Columns c0 .. c0 + columns - 1 of the sequences from `first` on, over positions [begin, end) of
  // the row of `leader`; columns that are not there go along as the first one, and no further.  whole: where the parts of an uncut item lie; cut: a cut one's.
  __device__ __forceinline__ void attend(int first, int c0, int columns, int leader, int begin,
                                         int end, float* whole, float* whole_ml, int64_t cut) {
    // wide: two waves beside each other take the columns, two take the positions
    const bool wide = N > 1 && columns > kNarrow;
    const int sets = (columns + 15) / 16;
    const int from = wide ? (wave_id() & 1) * 32 : 0;
    w.lane(pool, k_end, v_end);
    const int32_t* row = a.table + leader * a.ldt;
    const int p0 = wide ? begin : begin + wave_id() * kTile;
    const int page0 = w.page_id(row, shift, p0, end);
    const int page1 = w.page_id(row, shift, p0 + (wide ? kStage : kSharedBlock), end);
    const int seq0 = first + c0 / a.per_kv, skip = c0 % a.per_kv;
    int least = INT_MAX;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = from + 16 * n + w.r;
      const bool there = at < columns;
      const int on = there ? sequences_in(skip + at) : 0, seq = seq0 + on;
      const int head = kvh * a.per_kv + (there ? skip + at - on * a.per_kv : 0);
      const uint16_t* q = a.q + seq * a.ldq + head * a.ldh;
#pragma unroll
      for (int s = 0; s < w.QS; ++s) {
        const int d = w.E == 2 ? 32 * s + 8 * w.g : 64 * (s >> 1) + 16 * w.g + 8 * (s & 1);
        w.qf[n][s] = *reinterpret_cast<const u32x4*>(q + d) ^ sign;
      }
      const int len = batch.len(seq);
      w.seen[n] = there ? len : INT_MAX;
      least = min(least, w.seen[n]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o));
    least = __builtin_amdgcn_readfirstlane(least);
    w.clear();
    if (wide) w.run_wide(pool, row, shift, p0, end, least, wave_id() >> 1, lds, page0, page1);
    else if (sets == 1) w.template run<1>(pool, row, shift, p0, end, least, page0, page1);
    else w.template run<N>(pool, row, shift, p0, end, least, page0, page1);
    take_in(2, sets);
    if (!wide) take_in(1, sets);
    if (wave_id() >= (wide ? 2 : 1)) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = from + 16 * n + w.r;
      const float l = xor32_add(xor16_add(w.l[n]));
      if (at >= columns) continue;
      const int on = sequences_in(skip + at);
      const int64_t head = (int64_t)(seq0 + on) * a.n_heads + kvh * a.per_kv + skip + at -
                           on * a.per_kv;
      float* to = (cut < 0 ? whole + head * D : a.cut + (cut + at) * D) + w.VD * 4 * w.g;
      float* to_ml = cut < 0 ? whole_ml + 2 * head : a.cut_ml + 2 * (cut + at);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < w.VD; d += 4)
          *reinterpret_cast<floatx4*>(to + i * w.VD + d) = floatx4{
              w.acc[n][d][i], w.acc[n][d + 1][i], w.acc[n][d + 2][i], w.acc[n][d + 3][i]};
      if (w.g == 0) *reinterpret_cast<float2*>(to_ml) = make_float2(w.m[n], l);
    }
  }

  // Waves `half` .. 2 half - 1 hand their sums to waves 0 .. half - 1, through LDS as the lanes have
  // them.
  __device__ __forceinline__ void take_in(int half, int sets) {
    const int lane = fresh(threadIdx.x) & 63, wave = wave_id();
    __syncthreads();                    // what was read there before
    if (wave >= half && wave < 2 * half) {
      char* to = lds + (wave - half) * kSumBytes + lane * 16;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n >= sets) break;
#pragma unroll
        for (int d = 0; d < w.VD; ++d)
          *reinterpret_cast<floatx4*>(to + (n * w.VD + d) * 1024) = w.acc[n][d];
        *reinterpret_cast<float2*>(to + N * w.VD * 1024 + n * 512 - lane * 8) =
            make_float2(w.m[n], w.l[n]);
      }
    }
    __syncthreads();
    if (wave >= half) return;
    const char* from = lds + wave * kSumBytes + lane * 16;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (n >= sets) break;
      const float2 ml = *reinterpret_cast<const float2*>(from + N * w.VD * 1024 + n * 512 - lane * 8);
      const float top = fmaxf(w.m[n], ml.x), mu = top == -__builtin_inff() ? 0.f : top;
      const float e0 = __builtin_amdgcn_exp2f(w.m[n] - mu), e1 = __builtin_amdgcn_exp2f(ml.x - mu);
      w.m[n] = top;
      w.l[n] = w.l[n] * e0 + ml.y * e1;
#pragma unroll
      for (int d = 0; d < w.VD; ++d)
        w.acc[n][d] = w.acc[n][d] * e0 +
                      *reinterpret_cast<const floatx4*>(from + (n * w.VD + d) * 1024) * e1;
    }
  }

  // The table row that a group's shared positions are read through, and how many of them any of its
  // sequences reaches: the first sequence that reaches all, or else the longest.
  __device__ __forceinline__ int2 leader(const Group& g) const {
    const int lane = threadIdx.x & 63;
    int best = -1, at = g.begin;
    for (int s0 = g.begin; s0 < g.end; s0 += 64) {
      const int s = s0 + lane;
      const int len = s < g.end ? min(batch.len(s), g.shared) : -1;
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

// What the second launch goes by.
template <int WIDE>
__device__ __forceinline__ void write_items(const Batch& batch, const Row<WIDE>& row) {
  const SharedCall& a = batch.a;
  const int lane = threadIdx.x & 63;
  const int before_groups = __builtin_amdgcn_update_dpp(0, row.groups_upto, 0x138, 0xf, 0xf, false);
  const int before_seqs = __builtin_amdgcn_update_dpp(0, row.seqs_upto, 0x138, 0xf, 0xf, false);
  if (wave_id() == 0) {
    int base = before_groups;
    for (int i = 0; i < row.per_group; ++i) {
      const int64_t at = (int64_t)lane * row.per_group + i;
      if (at >= batch.n_groups) break;
      const Group g = batch.group((int)at);
      const int blocks = blocks_in(g.shared), columns = (g.end - g.begin) * a.per_kv;
      if (!blocks) continue;
      const int id = g.begin * a.per_kv / WIDE + (int)at;
      for (int c = 0, t = 0; c < columns; c += WIDE, ++t) {
        const int n = min(WIDE, columns - c);
        if (id + t < a.tiles) a.item_tiles[id + t] = row.pieces_of(base, blocks, n);
        base += item_cost(n, blocks);
      }
    }
  } else if (wave_id() == 1) {
    int base = row.shared_cost + before_seqs;
    for (int i = 0; i < row.per_seq; ++i) {
      const int64_t at = (int64_t)lane * row.per_seq + i;
      if (at >= a.seqs) break;
      const int s = (int)at;
      Group g;
      const int group = batch.group_of(s, g);
      const int len = batch.len(s), blocks = blocks_in(len - min(g.shared, len));
      a.seq_items[s] = g.shared ? make_int2(g.begin * a.per_kv / WIDE + group,
                                            (s - g.begin) * a.per_kv)
                                : make_int2(-1, 0);
      for (int c = 0, t = 0; c < a.per_kv; c += WIDE, ++t) {
        const int n = min(WIDE, a.per_kv - c);
        a.item_own[at * a.own_tiles + t] = row.pieces_of(base, blocks, n);
        base += item_cost(n, blocks);
      }
    }
  }
}

template <int QT, int KT, int D, int N>
__global__ void __launch_bounds__(kSharedWaves * 64, 2) paged_shared_kernel(SharedCall a,
                                                                            PagePool pool) {
  constexpr int WIDE = N == 1 ? 16 : kWide;
  __shared__ __align__(16) char lds[Piece<QT, KT, D, N>::kBytes];
  __shared__ Lists lists;
  const int units = pool.kv_heads;
  const int kvh = blockIdx.x % units, piece = blockIdx.x / units;
  const Batch batch(a, lists, WIDE);
  const Row<WIDE> row(a, batch);
  if (piece == a.pieces) {
    if (kvh == 0) write_items<WIDE>(batch, row);
    return;
  }
  if (piece >= row.pieces || row.total <= 0) return;
  const int lo = row.cut.start(piece), hi = row.cut.start(piece + 1);
  if (lo >= hi) return;
  Piece<QT, KT, D, N> p(batch, pool, kvh, lds);
  const int64_t slot = (int64_t)blockIdx.x * 2 * WIDE;
  const int64_t heads = (int64_t)a.seqs * a.n_heads;
  // Items from the first that reaches into the piece on: groups, then sequences.  One place in the
  // code attends to both, which keeps the code within the instruction cache.
  bool own = lo >= row.shared_cost;
  int from = __builtin_ctzll(__ballot(own ? lo < row.shared_cost + row.seqs_upto
                                          : lo < row.groups_upto));
  int base = own ? row.shared_cost : 0;
  if (from) base += __builtin_amdgcn_readlane(own ? row.seqs_upto : row.groups_upto, from - 1);
  int64_t i = (int64_t)from * (own ? row.per_seq : row.per_group);
  while (base < hi) {
    int first, columns, leader, begin, end, blocks;
    if (!own) {
      if (i >= batch.n_groups) {
        own = true;
        i = 0;
        base = row.shared_cost;
        continue;
      }
      Group g = batch.group((int)i++);  // out of LDS: the same in all lanes
      g.begin = __builtin_amdgcn_readfirstlane(g.begin);
      g.end = __builtin_amdgcn_readfirstlane(g.end);
      g.shared = __builtin_amdgcn_readfirstlane(g.shared);
      first = g.begin;
      columns = (g.end - g.begin) * a.per_kv;
      blocks = blocks_in(g.shared);
      const int cost = cost_of(columns, blocks, WIDE);
      if (base + cost <= lo) {
        base += cost;
        continue;
      }
      const int2 lead = p.leader(g);
      leader = __builtin_amdgcn_readfirstlane(lead.x);
      begin = 0;
      end = __builtin_amdgcn_readfirstlane(lead.y);
    } else {
      if (i >= a.seqs) break;
      const int2 at = batch.own_of((int)i);
      leader = first = (int)i++;
      columns = a.per_kv;
      begin = __builtin_amdgcn_readfirstlane(at.x);
      end = __builtin_amdgcn_readfirstlane(at.y);
      blocks = blocks_in(end - begin);
    }
    items_within<WIDE>(base, columns, blocks, lo, hi, [&](int c, int n, Span b) {
      p.attend(first, c, n, leader, begin + b.x * kSharedBlock,
               min(begin + b.y * kSharedBlock, end), a.whole + (own ? heads * D : 0),
               a.whole_ml + (own ? 2 * heads : 0),
               b.x == 0 && b.y == blocks ? -1 : slot + (b.x == 0) * WIDE);
    });
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
  // Parts at(0) .. at(n - 1), several on their way at a time.
  auto add = [&](int n, auto&& at) {
    constexpr int kAhead = 8;
    for (int i = 0; i < n; i += kAhead) {
      float2 ml[kAhead];
      floatx4 y[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        ml[j] = make_float2(-__builtin_inff(), 0.f);
        y[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (i + j < n) at(i + j, ml[j], y[j]);
      }
      float t = top;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) t = fmaxf(t, ml[j].x);
      const float mu = t == -__builtin_inff() ? 0.f : t;
      const float e0 = __builtin_amdgcn_exp2f(top - mu);
      total *= e0;
      o *= e0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float e = __builtin_amdgcn_exp2f(ml[j].x - mu);
        total = fmaf(ml[j].y, e, total);
        o += y[j] * e;
      }
      top = t;
    }
  };
  auto item = [&](int2 pieces, int64_t whole, int column) {
    const int last = min(pieces.y, a.pieces - 1), begin = max(pieces.x, 0);
    add(last - begin + 1, [&](int i, float2& ml, floatx4& y) {
      const int64_t cut = (((int64_t)(begin + i) * kv_heads + kvh) * 2 + (i == 0)) * WIDE + column;
      const bool is_whole = pieces.x == pieces.y;
      ml = *reinterpret_cast<const float2*>(is_whole ? a.whole_ml + 2 * whole : a.cut_ml + 2 * cut);
      y = *reinterpret_cast<const floatx4*>((is_whole ? a.whole + whole * D : a.cut + cut * D) +
                                            4 * lane);
    });
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
  p.sets = columns <= 16 ? 1 : 2;
  p.wide = columns <= 16 ? 16 : kWide;
  p.own_tiles = (int)((per_kv + p.wide - 1) / p.wide);
  p.pieces = kv_heads < kSharedWorkgroups ? kSharedWorkgroups / kv_heads : 1;
  p.tiles = columns / p.wide + groups + 1;
  p.rows = 2 * seqs * n_heads + (int64_t)p.pieces * kv_heads * 2 * p.wide;
  return p;
}

template <int QT, int KT, int D>
static void launch_shared(const SharedCall& a, const PagePool& p, const SharedPlan& s,
                          hipStream_t stream) {
  const unsigned grid = (unsigned)((s.pieces + 1) * p.kv_heads);
  const unsigned joins = (unsigned)(((int64_t)a.seqs * a.n_heads * (D / 4) + 255) / 256);
#define MTL_RUN(N, WIDE)                                                                    \
  do {                                                                                      \
    paged_shared_kernel<QT, KT, D, N><<<grid, kSharedWaves * 64, 0, stream>>>(a, p);        \
    paged_shared_join_kernel<QT, D, WIDE><<<joins, 256, 0, stream>>>(a, p.kv_heads,         \
                                                                     p.v_scale);            \
  } while (0)
  if (s.sets == 1) MTL_RUN(1, 16);
  else MTL_RUN(2, kWide);
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
  return items <= INT32_MAX / kItemCost / (blocks + 1) &&
         seqs * n_heads <= (int64_t)UINT32_MAX / 64 && (int64_t)(p.pieces + 1) * kv_heads <= 1 << 23;
}

// Few sequences with short tables: one launch that takes each by itself (mtl_paged_attention without
// a workspace) instead of two.
static bool alone_is_faster(int64_t seqs, int32_t n_heads, int32_t kv_heads, int64_t width,
                            int32_t page_size) {
  const int64_t units = (int64_t)kv_heads * ((n_heads / kv_heads + 15) / 16);
  return width * page_size <= kShortTable && seqs * units <= kShortUnits;
}

extern "C" int64_t mtl_paged_attention_shared_workspace_bytes(int64_t seqs, int64_t groups,
                                                              int32_t n_heads, int32_t kv_heads,
                                                              int32_t head_dim, int64_t width,
                                                              int32_t page_size) {
  if (seqs < 1 || head_dim < 1 ||
      !shared_sizes_ok(seqs, groups, n_heads, kv_heads, width, page_size))
    return 0;
  if (alone_is_faster(seqs, n_heads, kv_heads, width, page_size)) return 16;   // not used
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
  if (alone_is_faster(seqs, n_heads, pool->kv_heads, table->width, p.page_size))
    return mtl_paged_attention(q, ldq, ldh, pool, table, lens, n_heads, q_type, scale, out, lse,
                               nullptr, 0, stream);
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
