// Drawing tokens from logits: temperature, top-k, top-p and min-p (gfx950).
//
// Everything is decided by sums of weights, and a row has as many borders as tokens: with float32
// sums (2^-24 of the whole) one row in some thousands would draw another token than the definition.
// Weights are of 64 bits and their sums whole numbers of 2^-51 up to 4096 tokens, of twice that for
// each doubling (2^-45 up to 2^18 tokens, 2^-43 at 2^20: a row of the largest weights is 2^63 then),
// whose order changes nothing.  A border may be off by half a unit for each token before it.
//
// The work is one read of the logits; no row is ever sorted:
// * A first launch cuts rows into slices of 32 tokens (128 past 262 144) and keeps the largest logit
//   of each (rows of up to kMaxSlices tokens need none: they fit LDS).
// * Rows that need the sum of all weights (top-p without top-k; no filter) are weighed in a second
//   launch: a sum for each kChunk tokens, and for top-p by the logits' distance to the largest, in
//   steps of 1/128 octave.
// * In the last launch a workgroup takes a row.  The slices' largest logits, counted by steps, give a
//   step that top-k's tokens lie within (as many slices' largest do); min-p's border is a step known
//   beforehand.  The slices that reach it are read again: up to kCandidates tokens are sorted in
//   registers, by the order for the borders and by index for the draw.  More of them are kept in LDS,
//   and borders found among them by digits of their ordered keys.
// * Where a list of kFewer cannot settle a row that top-p alone cuts, its border lies in one step,
//   whose tokens are gathered; the draw then falls into one chunk, which is read again.
// * What none of these settles (over kHeld tokens within the step; thousands of equal logits; top-p
//   without top-k past a list in rows that need no slices) takes passes over the whole row: 290 us
//   for 151 000 tokens, where kept tokens take 46; 22 for 31 rows of 1025 by top-p 0.8 alone, 37 for
//   rows of 8192, though they lie in LDS.
//
// What bounds it: a chain of dependent steps in one workgroup (barriers, 3 to 5 trips to memory), not
// the bytes.  Measured: one row of 151 936 bf16 logits, top-k 50, 2.5 + 12 us; 31 rows of 1025,
// top-k 25 and top-p, 10 us in one launch (min-p alone 10, no filter 9); 24 rows of 151 936 by top-p
// 4 + 12 + 16 us, whose steps (8 KB a chunk, written once and read twice) are as many bytes as bf16
// logits; 96 float32 rows with a setting each (58 MB) 10 + 11 + 16 us, and 60 in the last where a row's
// top-p border is past its list: that row's workgroup reads its 600 KB alone.  The first
// launch reads 5.6 TB/s there.  Tried and slower: 1024 threads a row, ranks by comparing all pairs of
// a list, more kept tokens (96 KB of LDS: even, and 287 -> 354 us for 500 rows).
#include "mtl_common.h"
#include "mtl_paged.h"
#include "mtl_sample.h"

namespace mtl {

typedef unsigned long long u64;

constexpr int kThreads = 512;          // of a row
constexpr int kWaves = kThreads / 64;
// Tokens of a workgroup of the first two launches (8192 tokens and 256 threads: one row by top-p 26 us
// for 22, no filter 24 for 20, 24 rows by top-p 29.6 for 28.6).
constexpr int kChunk = 4096;
constexpr int kChunkThreads = 512;
constexpr int kCandidates = kThreads;
// Tokens that a weighed row's list is made for: 24 rows of top-p 0.95 28.6 us, with 32 51 (rows whose
// border is past their list), with 128 32.6 (a longer sort for all).
constexpr int kFewer = 64;
constexpr int kBins = 2048;
constexpr int kMaxSlices = 8192;
constexpr int kHeld = kMaxSlices / 2;   // tokens kept, in the room of the slices' largest logits
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxChunks = kMaxVocab / kChunk;
constexpr int kMaxRows = 65535;
constexpr int kMostUnit = 51;           // a weight beside 2^52, which rounds it, stays below 2^53

constexpr int kSteps = 1024;

struct SampleCall {
  const void* x;
  int64_t ld;
  int vocab, slice_shift, slices, unit; // slices of 2^slice_shift; weights are counted in 2^-unit
  int chunks;                           // 0: one launch does it all
  int weighed;                          // rows that need the sum of their weights have it
  const float* u;
  mtl_sample_settings s;
  int64_t* token;
  float* logprob;
  float* tops;                          // [rows][slices]
  float* chunk_tops;                    // [rows][chunks]
  u64* sums;                            // [rows][chunks]
  u64* steps;                           // [rows][chunks][kSteps]; null: no row can need them
};

// A row's settings.
struct Settings {
  float temperature, p, m;
  int k;

  __device__ __forceinline__ Settings(const SampleCall& c, int64_t r) {
    const mtl_sample_settings& s = c.s;
    temperature = s.temperature ? s.temperature[r] : s.temperature_all;
    k = s.top_k ? s.top_k[r] : s.top_k_all;
    p = s.top_p ? s.top_p[r] : s.top_p_all;
    m = s.min_p ? s.min_p[r] : s.min_p_all;
    k = k <= 0 || k > c.vocab ? c.vocab : k;
  }
  // The first of the order is all that stays.
  __device__ __forceinline__ bool greedy() const {
    return !(temperature > 0.f) || k == 1 || !(p > 0.f) || !(m <= 1.f);
  }
  __device__ __forceinline__ bool by_steps(int vocab) const { return k == vocab && p < 1.f; }
  __device__ __forceinline__ bool weighed(int vocab) const {
    return !greedy() && k == vocab && (p < 1.f || !(m > 0.f));
  }
};

// ------------------------------------------------------------------------------ logits
template <int T>
struct Logits {
  static constexpr int kDrop = T == MTL_T_BF16 ? 16 : T == MTL_T_F16 ? 13 : 0;
  const char* p;
  int n;

  __device__ __forceinline__ Logits(const SampleCall& c, int64_t row)
      : p(static_cast<const char*>(c.x) + row * c.ld * (T == MTL_T_F32 ? 4 : 2)), n(c.vocab) {}

  // NaN counts as -infinity, -0 as 0.
  static __device__ __forceinline__ float clean(float x) {
    return x == x ? x + 0.f : -__builtin_inff();
  }

  __device__ __forceinline__ float at(int i) const {
    if (T == MTL_T_F32) return clean(reinterpret_cast<const float*>(p)[i]);
    const uint32_t e = reinterpret_cast<const uint16_t*>(p)[i];
    return clean(T == MTL_T_BF16 ? bf16_to_f32(e) : f16_to_f32(e));
  }

  // Logits i .. i + 7, all there.
  __device__ __forceinline__ void load_whole(int i, float (&x)[8]) const {
    if (T == MTL_T_F32) {
      float v[8];
      __builtin_memcpy(v, p + (int64_t)i * 4, 32);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = clean(v[j]);
    } else {
      uint32_t v[4];
      __builtin_memcpy(v, p + (int64_t)i * 2, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t e = j & 1 ? v[j / 2] >> 16 : v[j / 2] & 0xffffu;
        x[j] = clean(T == MTL_T_BF16 ? bf16_to_f32(e) : f16_to_f32(e));
      }
    }
  }

  // Logits i .. i + 7, -infinity past the end.
  __device__ __forceinline__ void load(int i, float (&x)[8]) const {
    if (i + 8 <= n) return load_whole(i, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < n ? at(i + j) : -__builtin_inff();
  }

  // Whole numbers in the logits' order; key: without the bits that the type does not have.
  static __device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ uint32_t key(float x) {
    return order(x) >> kDrop;
  }
  static __device__ __forceinline__ float of_order(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    k = k << kDrop;
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k & ~((1u << kDrop) - 1));
  }
};

// 2^t for t <= 0, to some 2^-50 of itself (0 far below): the whole part into the exponent, 2^f =
// e^(f ln 2) for the rest, |f| <= 1/2, by its series (the 14th term is below 2^-54).  The library's
// function takes four times as long, which is what weighing a row costs.
__device__ __forceinline__ double power_of_two(double t) {
  const double n = rint(t), r = (t - n) * 0x1.62e42fefa39efp-1;
  double e = 1.0 / 6227020800.0;
  constexpr double kTerms[13] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720,
                                 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800,
                                 1.0 / 39916800, 1.0 / 479001600};
#pragma unroll
  for (int i = 12; i >= 0; --i) e = fma(e, r, kTerms[i]);
  const int whole = (int)fmax(n, -1000.0);
  return __longlong_as_double(__double_as_longlong(e) + ((long long)whole << 52));
}

struct Weight {
  float top;
  double by;                            // log2(e) / temperature
  __device__ __forceinline__ Weight(float top, float temperature)
      : top(top),
        by(0x1.71547652b82fep+0 / (double)fminf(temperature, 3.4028234663852886e38f)) {}
  __device__ __forceinline__ double operator()(float x) const {
    const double w = power_of_two(fmax(((double)x - (double)top) * by, -2000.0));
    return x == top ? 1.0 : w;
  }
};

// A weight (at most 1) in whole units of 2^-unit, unit <= kMostUnit: the sum with 2^52 rounds to them.
__device__ __forceinline__ u64 whole_units(double w, int unit) {
  const double one = __longlong_as_double((u64)(1023 + unit) << 52);
  return (u64)__double_as_longlong(fma(w, one, 0x1p52)) - (u64)__double_as_longlong(0x1p52);
}

// Steps of the distance to the largest logit, 128 to an octave from 1/4 to 64: the same or a later
// one for a smaller logit.
constexpr int kFirstStep = 125 * 128 - 1;
__device__ __forceinline__ int step_at(float distance) {
  const int s = (int)(__float_as_uint(distance) >> 16) - kFirstStep;
  return min(max(s, 0), kSteps - 1);
}
__device__ __forceinline__ int step_of(float top, float x) { return x == top ? 0 : step_at(top - x); }

// ------------------------------------------------------------------------------ workgroup steps
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 scan_step(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((u64)hi << 32 | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}

// Inclusive sums over a wave (all lanes active), and over the workgroup in thread order with their
// total.
template <class V>
__device__ __forceinline__ V lanes_upto(V v) {
  v = scan_step<0x111, 0xf>(v);         // row_shr:1, 2, 4, 8; row_bcast:15, 31
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);
  return scan_step<0x143, 0xc>(v);
}

template <int WAVES, class V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
  v = lanes_upto(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[wave_id()] = v;
  __syncthreads();
  V before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i == wave_id()) before = sum;
    sum += part[i];
  }
  total = sum;
  return before + v;
}

template <int WAVES>
__device__ __forceinline__ float block_max(float v, float* part) {
  v = wave_max_valu(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[wave_id()] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) v = fmaxf(v, part[i]);
  return v;
}

struct Shared {
  union {
    float top[kMaxSlices];              // each slice's largest logit
    u64 held[kHeld];                    // tokens of one step: (logit, index)
  };
  union {
    u64 sums[kBins];
    int active[kHeld];
    struct {
      uint32_t steps[kSteps];
      int active[kCandidates];
      u64 order[kCandidates];           // (the logit's key, the index from above)
      u64 w[kCandidates];               // by rank
      u64 swap[kCandidates];
    } list;
  };
  union {
    u64 u[kWaves];
    int i[kWaves];
    float f[kWaves];
  } part;
  u64 chunk[kMaxChunks];                // what stays of each chunk
  int ties[kMaxChunks];
  int n, m, first;
  u64 above;
};

// ------------------------------------------------------------------------------ a row
template <int T>
struct Draw {
  static constexpr int THREADS = kThreads, WAVES = kWaves;
  const SampleCall& c;
  const int64_t row;
  Shared& sh;
  const Logits<T> x;
  Weight weight;
  int k;
  double p, m, u;
  bool weighed;
  // What is left to draw from once the borders are known: tokens down to `key`, the first `ties` of
  // its own; `mine` of their weight lies in chunk threadIdx.x, and sh.ties[chunk] tokens of the key
  // in earlier chunks.
  u64 mine;
  uint32_t key;
  int ties, held_step = -1;             // of a long list

  __device__ __forceinline__ Draw(const SampleCall& c, int64_t row, Shared& sh, float top, const Settings& s,
                  float u)
      : c(c), row(row), sh(sh), x(c, row), weight(top, s.temperature), k(s.k), p(s.p), m(s.m),
        u(u >= 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0),
        weighed(c.weighed && s.weighed(c.vocab)) {}

  __device__ __forceinline__ void result(int token, double logprob) {
    c.token[row] = token;
    if (c.logprob) c.logprob[row] = (float)logprob;
  }

  // The lowest index of the largest logit.
  __device__ __forceinline__ void greedy() {
    if (threadIdx.x == 0) sh.first = c.vocab;
    __syncthreads();
    for (int s = threadIdx.x; s < c.slices; s += THREADS) {
      if (sh.top[s] != weight.top) continue;
      for (int i = s << c.slice_shift; i < min(c.vocab, (s + 1) << c.slice_shift); ++i)
        if (x.at(i) == weight.top) {
          atomicMin(&sh.first, i);
          break;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) result(sh.first, 0.0);
  }

  // Calls f(index, logit) for all tokens of the row.
  template <class F>
  __device__ __forceinline__ void all(F&& f) const {
    for (int i = threadIdx.x * 8; i < c.vocab; i += THREADS * 8) {
      float v[8];
      x.load(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f(i + j, v[j]);
    }
  }

  // The sum of all weights.
  __device__ __forceinline__ u64 total() {
    u64 sum = 0, whole;
    if (weighed) {
      for (int i = threadIdx.x; i < c.chunks; i += THREADS) sum += c.sums[row * c.chunks + i];
    } else {
      all([&](int, float v) { sum += whole_units(weight(v), c.unit); });
    }
    block_scan<WAVES>(sum, sh.part.u, whole);
    return whole;
  }

  // Calls f(slice, its largest logit) for all slices with a number.
  template <class F>
  __device__ __forceinline__ void tops(F&& f) const {
    constexpr int AHEAD = 4;
    for (int s0 = threadIdx.x; s0 < c.slices; s0 += AHEAD * THREADS) {
      float v[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        v[a] = s0 + a * THREADS < c.slices ? sh.top[min(s0 + a * THREADS, kMaxSlices - 1)]
                                           : -__builtin_inff();
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (v[a] != -__builtin_inff()) f(s0 + a * THREADS, v[a]);
    }
  }

  // One exchange of a sort between lanes `BY` apart: v and the other's in any order.
  template <int BY>
  static __device__ __forceinline__ void lanes_apart(u64 v, u64& a, u64& b) {
    uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32), lo2 = lo, hi2 = hi;
    if (BY == 32) {
      permlane_swap32(lo, lo2);
      permlane_swap32(hi, hi2);
    } else if (BY == 16) {
      permlane_swap16(lo, lo2);
      permlane_swap16(hi, hi2);
    } else {
      constexpr int kCtrl = BY == 8 ? kDppRor8 : BY == 4 ? kDppHalfMirror : BY == 2 ? kDppXor2
                                                                                    : kDppXor1;
      lo2 = __builtin_amdgcn_update_dpp(0, lo, kCtrl, 0xf, 0xf, false);
      hi2 = __builtin_amdgcn_update_dpp(0, hi, kCtrl, 0xf, 0xf, false);
      if (BY == 4) {                    // the mirror of 8 and that of 4: 4 apart
        lo2 = __builtin_amdgcn_update_dpp(0, lo2, 0x1b, 0xf, 0xf, false);
        hi2 = __builtin_amdgcn_update_dpp(0, hi2, 0x1b, 0xf, 0xf, false);
      }
    }
    a = (u64)hi << 32 | lo;
    b = (u64)hi2 << 32 | lo2;
  }

  template <int BY>
  static __device__ __forceinline__ u64 exchanged(u64 v, bool down) {
    u64 a, b;
    lanes_apart<BY>(v, a, b);
    const bool larger = !(threadIdx.x & BY) == down;
    return (a > b) == larger ? a : b;
  }

  // Sorts the values of threads 0 .. m - 1 (a power of two, at least 64), the largest first.
  __device__ __forceinline__ u64 sorted(u64 v, int m) {
    for (int size = 2; size <= m; size <<= 1) {
      const bool down = !(threadIdx.x & size);
      for (int by = size >> 1; by > 32; by >>= 1) {
        __syncthreads();
        sh.list.swap[threadIdx.x] = v;
        __syncthreads();
        const u64 other = sh.list.swap[threadIdx.x ^ by];
        v = (v > other) == (!(threadIdx.x & by) == down) ? v : other;
      }
      if ((int)threadIdx.x >= m) continue;            // whole waves
      if (size > 32) v = exchanged<32>(v, down);
      if (size > 16) v = exchanged<16>(v, down);
      if (size > 8) v = exchanged<8>(v, down);
      if (size > 4) v = exchanged<4>(v, down);
      if (size > 2) v = exchanged<2>(v, down);
      v = exchanged<1>(v, down);
    }
    return v;
  }

  // Draws from a list of candidates; false where a list cannot settle the row.
  __device__ __forceinline__ bool by_list() {
    auto& l = sh.list;
    const int t = threadIdx.x;
    const bool k_set = k < c.vocab;
    // The step that min-p's border lies in (a little further, for rounding): no token past it stays,
    // nor is one looked at unless the mass that top-k leaves is asked for.
    int cut = kSteps;
    if (m > 0 && (p >= 1 || !k_set))
      cut = step_at((float)((double)(0.f - log2f((float)m)) / weight.by) * 1.0001f);
    // a weighed row has another way where its list is too short
    const int want = k_set ? k : weighed ? kFewer : c.vocab + 1;
    for (int i = t; i < kSteps; i += THREADS) l.steps[i] = 0;
    if (t == 0) {
      sh.n = sh.m = 0;
      sh.first = min(kSteps - 1, cut);
    }
    __syncthreads();
    tops([&](int, float v) { atomicAdd(&l.steps[step_of(weight.top, v)], 1u); });
    __syncthreads();
    // the first step that `want` slices reach, or the last
    constexpr int EACH = kSteps / THREADS;
    int mine = 0, all_of;
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine += (int)l.steps[t * EACH + i];
    int upto = block_scan<WAVES>(mine, sh.part.i, all_of) - mine;
    if (upto < want && upto + mine >= want) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        upto += (int)l.steps[t * EACH + i];
        if (upto >= want) {
          sh.first = min(t * EACH + i, cut);
          break;
        }
      }
    }
    __syncthreads();
    const int last = sh.first;
    // where the list has no room
    if (k_set || cut < kSteps - 1) held_step = k_set ? last : cut;
    if (k_set && k > kCandidates && cut == kSteps) return false;
    tops([&](int s, float v) {
      if (step_of(weight.top, v) > last) return;
      const int at = atomicAdd(&sh.m, 1);
      if (at < kCandidates) l.active[at] = s;
    });
    __syncthreads();
    const int active = sh.m;
    if (active > kCandidates) return false;
    for (int i = t; i < active << c.slice_shift; i += THREADS) {
      const int e = (l.active[i >> c.slice_shift] << c.slice_shift) + (i & ((1 << c.slice_shift) - 1));
      const float v = c.slice_shift == 0 ? sh.top[e] : e < c.vocab ? x.at(e) : -__builtin_inff();
      if (v != -__builtin_inff() && step_of(weight.top, v) <= last) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kCandidates) l.order[at] = (u64)x.order(v) << 32 | (uint32_t)~e;
      }
    }
    __syncthreads();
    const int n = sh.n;
    if (n > kCandidates) return false;
    int m_sort = 64;
    while (m_sort < n) m_sort <<= 1;
    // sorted by the order, and then what stays by index, each token with its rank
    u64 by_index = t < n ? l.order[t] : 0, mass, whole;
    for (int pass = 0; pass < 2; ++pass) {            // one copy of the code
      by_index = sorted(by_index, m_sort);
      if (pass) break;
      const u64 mine_is = by_index;
      const double w = t < n ? weight(x.of_order((uint32_t)(mine_is >> 32))) : 0.0;
      const u64 units = whole_units(w, c.unit);
      const u64 before = block_scan<WAVES>(units, sh.part.u, whole) - units;
      // the weight of those that top-k left
      if (t == 0) sh.above = whole;
      __syncthreads();
      if (t == k) sh.above = before;
      __syncthreads();
      mass = sh.above;
      if (last < kSteps - 1 && !(k_set && k <= n)) {  // tokens outside the list may count
        const bool enough = last >= cut;              // ... or not, by min-p
        if (!enough && (k_set || p >= 1)) return false;
        if (p < 1) mass = total();
        if (!enough && !(whole > (u64)(p * (double)mass))) return false;
      }
      const bool keep = t < n && t < k && (p >= 1 || before <= (u64)(p * (double)mass)) &&
                        (w >= m || t == 0) && units > 0;
      l.w[t] = units;
      by_index = keep ? (u64)(kMaxVocab - (int)~(uint32_t)mine_is) << 16 | (uint32_t)t : 0;
    }
    __syncthreads();
    const int rank = (int)(by_index & 0xffff);
    const u64 here = by_index ? l.w[rank] : 0;
    const u64 upto_w = block_scan<WAVES>(t < m_sort ? here : 0, sh.part.u, whole);
    const u64 goal = (u64)(u * (double)whole);
    // by_index is above 0 wherever something stays
    if (mine_is_it(t < m_sort && here > 0, upto_w > goal)) {
      const int token = kMaxVocab - (int)(by_index >> 16);
      result(token, log(weight(x.at(token)) / ldexp((double)whole, -c.unit)));
    }
    return true;
  }

  // The first thread that passes the goal, or, where rounding leaves none, the last with something.
  __device__ __forceinline__ bool mine_is_it(bool some, bool passes) {
    if (threadIdx.x == 0) {
      sh.first = THREADS;
      sh.m = -1;
    }
    __syncthreads();
    const u64 has = __ballot(some), over = __ballot(some && passes);
    if ((threadIdx.x & 63) == 0) {
      const int at = threadIdx.x;
      if (has) atomicMax(&sh.m, at + 63 - __builtin_clzll(has));
      if (over) atomicMin(&sh.first, at + __builtin_ctzll(over));
    }
    __syncthreads();
    return (int)threadIdx.x == min(sh.first, sh.m);
  }

  // A border in the order of keys from `lo` to `hi`: the key at which `limit` is passed, going down,
  // and what lies above it (`above` at first lies above hi).  each(f) calls f(logit) for all tokens
  // in question.  WEIGH: weights in units of 2^-unit, else tokens.
  template <bool WEIGH, class Each>
  __device__ __forceinline__ void border(Each&& each, uint32_t lo, uint32_t hi, u64 limit, uint32_t& key,
                         u64& above) {
    constexpr int EACH = kBins / THREADS;
    while (true) {
      const uint32_t range = hi - lo;
      const int shift = range < kBins ? 0 : 21 - __builtin_clz(range);
      const int bins = (int)(range >> shift) + 1;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += THREADS) sh.sums[i] = 0;
      if (threadIdx.x == 0) {
        sh.first = kBins;
        sh.m = -1;
      }
      __syncthreads();
      each([&](float v) {
        const uint32_t b = x.key(v);
        if (v != -__builtin_inff() && b >= lo && b <= hi)
          atomicAdd(&sh.sums[(b - lo) >> shift], WEIGH ? whole_units(weight(v), c.unit) : (u64)1);
      });
      __syncthreads();
      const int j0 = EACH * threadIdx.x;              // bins from the largest key down
      u64 mine = 0, all_of;
#pragma unroll
      for (int i = 0; i < EACH; ++i) mine += j0 + i < bins ? sh.sums[bins - 1 - j0 - i] : 0;
      u64 ahead = above + block_scan<WAVES>(mine, sh.part.u, all_of) - mine;
      bool found = false;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const u64 here = j0 + i < bins ? sh.sums[bins - 1 - j0 - i] : 0;
        if (here) atomicMax(&sh.m, j0 + i);
        if (!found && (WEIGH ? ahead + here > limit : ahead + here >= limit)) {
          found = true;
          atomicMin(&sh.first, j0 + i);
        }
        ahead += here;
      }
      __syncthreads();
      const int pick = min(sh.first, max(sh.m, 0));
      ahead -= mine;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        if (pick == j0 + i) sh.above = ahead;
        ahead += j0 + i < bins ? sh.sums[bins - 1 - j0 - i] : 0;
      }
      __syncthreads();
      above = sh.above;
      lo += (uint32_t)(bins - 1 - pick) << shift;
      if (shift == 0) break;
      hi = min(hi, lo + ((1u << shift) - 1));
    }
    key = lo;
  }

  // How many tokens of weight w stay behind a weight of `above` under `limit`.
  __device__ __forceinline__ int that_stay(double limit, u64 above, double w) const {
    const double room = (limit - ldexp((double)above, -c.unit)) / w;
    return room < (double)c.vocab ? max((int)floor(room) + 1, 1) : c.vocab;
  }

  // Draws by passes over the row.
  __device__ __forceinline__ void by_passes() {
    auto row_of = [&](auto&& f) { all([&](int, float v) { f(v); }); };
    const uint32_t low = x.key(-__builtin_inff()) + 1, high = x.key(weight.top);
    uint32_t key = low, at;
    int ties = c.vocab;                               // of that key, how many stay
    if (k < c.vocab) {
      u64 above = 0;
      border<false>(row_of, low, high, (u64)k, at, above);
      key = at;
      ties = k - (int)above;
    }
    if (p < 1) {
      // the weight of what top-k left
      u64 sum = 0, whole, above = 0;
      int same = 0, all_same;
      all([&](int, float v) {
        if (v == -__builtin_inff()) return;
        if (x.key(v) > key) sum += whole_units(weight(v), c.unit);
        same += x.key(v) == key;
      });
      block_scan<WAVES>(sum, sh.part.u, whole);
      block_scan<WAVES>(same, sh.part.i, all_same);
      const double limit = p * (ldexp((double)whole, -c.unit) +
                                (double)min(ties, all_same) * weight(x.of_key(key)));
      border<true>(row_of, low, high, (u64)ldexp(limit, c.unit), at, above);
      const int stay = that_stay(limit, above, weight(x.of_key(at)));
      ties = at == key ? min(ties, stay) : stay;
      key = at;
    }
    // by index: each thread a run of tokens
    const int per = ((c.vocab + THREADS - 1) / THREADS + 7) & ~7;
    const int begin = min(c.vocab, (int)threadIdx.x * per), end = min(c.vocab, begin + per);
    const u64 tie = stays(x.of_key(key));
    u64 sum = 0, whole;
    int same = 0, all_same;
    for (int i = begin; i < end; i += 8) {
      float v[8];
      x.load(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j >= end || v[j] == -__builtin_inff()) continue;
        const uint32_t b = x.key(v[j]);
        same += b == key;
        if (b > key) sum += stays(v[j]);
      }
    }
    const int had = block_scan<WAVES>(same, sh.part.i, all_same) - same;
    sum += (u64)min(max(ties - had, 0), same) * tie;
    const u64 upto = block_scan<WAVES>(sum, sh.part.u, whole);
    const u64 goal = (u64)(u * (double)whole);
    if (!mine_is_it(sum > 0, upto > goal)) return;
    // within the run that the draw falls into
    u64 run = upto - sum;
    int last = -1, seen = had;
    for (int i = begin; i < end && run <= goal; ++i) {
      const float v = x.at(i);
      if (v == -__builtin_inff()) continue;
      const uint32_t b = x.key(v);
      if (b < key || (b == key && seen++ >= ties)) continue;
      const u64 w = b == key ? tie : stays(v);
      if (w == 0) continue;
      run += w;
      last = i;
    }
    result(last, log(weight(x.at(last)) / ldexp((double)whole, -c.unit)));
  }

  // A token's weight in whole units, 0 where min-p drops it.
  __device__ __forceinline__ u64 stays(float v) const {
    const double w = weight(v);
    return w >= m || v == weight.top ? whole_units(w, c.unit) : 0;
  }

  // The draw among what is left.
  __device__ __forceinline__ void in_chunk() {
    u64 whole, upto = block_scan<WAVES>(mine, sh.part.u, whole);
    const u64 goal = (u64)(u * (double)whole);
    if (mine_is_it(mine > 0, upto > goal)) {
      sh.n = threadIdx.x;
      sh.above = upto - mine;
    }
    __syncthreads();
    // the draw falls into chunk sh.n, a thread 8 tokens of it
    static_assert(kChunk % (8 * kThreads) == 0 && kChunk <= 32 * kThreads, "a thread's tokens");
    constexpr int EACH = kChunk / THREADS;
    const int chunk = sh.n, begin = chunk * kChunk + threadIdx.x * EACH;
    u64 w[EACH], sum = 0;
    int tied = 0, same = 0;
#pragma unroll
    for (int i = 0; i < EACH; i += 8) {
      float v[8];
      x.load(min(begin + i, c.vocab), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool there = begin + i + j < c.vocab && v[j] != -__builtin_inff();
        const uint32_t b = x.key(v[j]);
        w[i + j] = there && b >= key ? stays(v[j]) : 0;
        if (there && b == key) {
          tied |= 1 << (i + j);
          ++same;
        }
      }
    }
    int all_same;
    int left = ties - sh.ties[chunk] - (block_scan<WAVES>(same, sh.part.i, all_same) - same);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (tied >> i & 1 && left-- <= 0) w[i] = 0;
      sum += w[i];
    }
    const u64 before = sh.above;
    u64 chunk_whole;
    upto = before + block_scan<WAVES>(sum, sh.part.u, chunk_whole);
    if (!mine_is_it(sum > 0, upto > goal)) return;
    u64 run = upto - sum;
    int last = -1;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (w[i] && run <= goal) {
        run += w[i];
        last = begin + i;
      }
    // the weight itself, not in whole units: it may be small
    result(last, log(weight(x.at(last)) / ldexp((double)whole, -c.unit)));
  }

  // Tokens kept where the slices' largest logits were, each with its index.
  struct Held {
    const u64* of;
    int n;
    template <class F>
    __device__ __forceinline__ void operator()(F&& f) const {
      for (int i = threadIdx.x; i < n; i += THREADS)
        f((int)(uint32_t)of[i], __uint_as_float((uint32_t)(of[i] >> 32)));
    }
  };

  // `mine` of these tokens; `earlier(chunk)` is what the chunk has besides, a wave at a time.
  template <class Earlier>
  __device__ __forceinline__ void of_chunks(const Held& tokens, Earlier&& earlier) {
    const int chunks = (c.vocab + kChunk - 1) / kChunk;
    __syncthreads();
    for (int i = threadIdx.x; i < chunks; i += THREADS) {
      sh.chunk[i] = 0;
      sh.ties[i] = 0;
    }
    __syncthreads();
    tokens([&](int i, float v) {
      if (v == -__builtin_inff()) return;
      const uint32_t b = x.key(v);
      if (b > key) atomicAdd(&sh.chunk[i / kChunk], stays(v));
      if (b == key) atomicAdd(&sh.ties[i / kChunk], 1);
    });
    for (int i = wave_id(); i < chunks; i += WAVES) {
      const u64 v = earlier(i);
      if (v && (threadIdx.x & 63) == 0) atomicAdd(&sh.chunk[i], v);
    }
    __syncthreads();
    int has = (int)threadIdx.x < chunks ? sh.ties[threadIdx.x] : 0, all_has;
    const int had = block_scan<WAVES>(has, sh.part.i, all_has) - has;
    mine = 0;
    if ((int)threadIdx.x < chunks) {
      sh.ties[threadIdx.x] = had;
      mine = sh.chunk[threadIdx.x] + (u64)min(max(ties - had, 0), has) * stays(x.of_key(key));
    }
  }

  // The borders where top-k or min-p keeps more tokens than a list has room for, all of them in steps
  // up to `last`: these are kept, and borders looked for among them.
  __device__ __forceinline__ bool by_held(int last) {
    if (last == kSteps - 1) return false;
    if (threadIdx.x == 0) sh.n = sh.m = 0;
    __syncthreads();
    tops([&](int s, float v) {
      if (step_of(weight.top, v) > last) return;
      const int at = atomicAdd(&sh.m, 1);
      if (at < kHeld) sh.active[at] = s;
    });
    __syncthreads();
    const int active = sh.m;
    if (active > kHeld) return false;
    // 8 tokens at a time, or one
    const int parts = c.slice_shift == 0 ? 0 : c.slice_shift - 3;
    for (int i = threadIdx.x; i < active << parts; i += THREADS) {
      const int from = (sh.active[i >> parts] << c.slice_shift) + (i & ((1 << parts) - 1)) * 8;
      float v[8];
      x.load(min(from, c.vocab), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c.slice_shift == 0 && j > 0) break;
        if (v[j] == -__builtin_inff() || step_of(weight.top, v[j]) > last) continue;
        const int to = atomicAdd(&sh.n, 1);
        if (to < kHeld) sh.held[to] = (u64)__float_as_uint(v[j]) << 32 | (uint32_t)(from + j);
      }
    }
    __syncthreads();
    const Held tokens{sh.held, sh.n};
    if (tokens.n > kHeld) return false;
    auto logits = [&](auto&& f) { tokens([&](int, float v) { f(v); }); };
    const uint32_t low = x.key(-__builtin_inff()) + 1, high = x.key(weight.top);
    const bool k_set = k < c.vocab;
    uint32_t at;
    u64 above = 0;
    key = low;
    ties = c.vocab;
    if (k_set) {
      border<false>(logits, low, high, (u64)k, at, above);
      key = at;
      ties = k - (int)above;
    }
    if (p < 1) {
      u64 sum = 0, whole;
      int same = 0, all_same = 0;
      above = 0;
      if (k_set) {
        tokens([&](int, float v) {
          if (x.key(v) > key) sum += whole_units(weight(v), c.unit);
          same += x.key(v) == key;
        });
        block_scan<WAVES>(sum, sh.part.u, whole);
        block_scan<WAVES>(same, sh.part.i, all_same);
      } else {
        whole = total();
      }
      const double limit = p * (ldexp((double)whole, -c.unit) +
                                (double)min(ties, all_same) * weight(x.of_key(key)));
      border<true>(logits, low, high, (u64)ldexp(limit, c.unit), at, above);
      const int stay = that_stay(limit, above, weight(x.of_key(at)));
      ties = at == key ? min(ties, stay) : stay;
      key = at;
    }
    of_chunks(tokens, [](int) { return (u64)0; });
    return true;
  }

  // The border of a weighed row: top-p alone, or no filter.  False where min-p cuts deeper.
  __device__ __forceinline__ bool by_chunks() {
    key = x.key(-__builtin_inff()) + 1;
    ties = c.vocab;
    const u64* sums = c.sums + row * c.chunks;
    u64 whole;
    mine = (int)threadIdx.x < c.chunks ? sums[threadIdx.x] : 0;
    block_scan<WAVES>(mine, sh.part.u, whole);
    if (p < 1) {
      // the step of the border, of all chunks together
      static_assert(kSteps % THREADS == 0, "a thread's steps");
      constexpr int EACH = kSteps / THREADS;
      const u64* steps = c.steps + row * c.chunks * kSteps;
      const double limit = p * ldexp((double)whole, -c.unit);
      const u64 limit_units = (u64)ldexp(limit, c.unit);
      u64 of[EACH] = {}, sum = 0, total;
#pragma unroll 8
      for (int i = 0; i < c.chunks; ++i)
#pragma unroll
        for (int e = 0; e < EACH; ++e) of[e] += steps[i * kSteps + threadIdx.x * EACH + e];
#pragma unroll
      for (int e = 0; e < EACH; ++e) sum += of[e];
      u64 ahead = block_scan<WAVES>(sum, sh.part.u, total) - sum;
      if (threadIdx.x == 0) {
        sh.first = kSteps - 1;
        sh.above = 0;
      }
      __syncthreads();
      bool found = false;
      const u64 ahead0 = ahead;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (!found && ahead + of[e] > limit_units) {
          found = true;
          atomicMin(&sh.first, (int)threadIdx.x * EACH + e);
        }
        ahead += of[e];
      }
      __syncthreads();
      const int step = sh.first;
      ahead = ahead0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (step == (int)threadIdx.x * EACH + e) sh.above = ahead;
        ahead += of[e];
      }
      __syncthreads();
      u64 above = sh.above;
      // A few in a hundred tokens are in the step: lanes first note which of theirs are, and then
      // each keeps its next one, as often as the fullest lane has some.  They are kept where the
      // slices' largest logits were.
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      constexpr int AHEAD = 4;                        // pieces of 8 tokens on their way at a time
      for (int i0 = threadIdx.x; i0 * 8 < c.vocab; i0 += AHEAD * THREADS) {
        float v[AHEAD][8];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)               // the last one begins earlier
          x.load_whole(min((i0 + a * THREADS) * 8, c.vocab - 8), v[a]);
        uint32_t hits = 0;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int i = (i0 + a * THREADS) * 8, from = min(i, c.vocab - 8);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (from + j >= i && step_of(weight.top, v[a][j]) == step) hits |= 1u << (8 * a + j);
        }
        for (; hits; hits &= hits - 1) {
          const int bit = __builtin_ctz(hits);
          const int i = min((i0 + (bit >> 3) * THREADS) * 8, c.vocab - 8) + (bit & 7);
          const int to = atomicAdd(&sh.n, 1);
          if (to < kHeld) sh.held[to] = (uint32_t)i;
        }
      }
      __syncthreads();
      const int held = sh.n;
      if (held > kHeld) return false;
      // their logits, all on their way at once (read again where they were noted, they would wait for
      // one another)
      constexpr int ALL = kHeld / THREADS;
      uint32_t at[ALL];
      float logit[ALL];
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const int to = (int)threadIdx.x + i * THREADS;
        at[i] = to < held ? (uint32_t)sh.held[to] : 0;
        logit[i] = x.at((int)at[i]);
      }
#pragma unroll
      for (int i = 0; i < ALL; ++i)
        if ((int)threadIdx.x + i * THREADS < held)
          sh.held[threadIdx.x + i * THREADS] = (u64)__float_as_uint(logit[i]) << 32 | at[i];
      __syncthreads();
      const Held tokens{sh.held, held};
      // The step's tokens lie between two keys: distances are off by 2^-24 of themselves, which are many
      // keys where the logit is near 0, and the bounds' own rounding is within two.
      const float far = step == kSteps - 1 ? __builtin_inff()
                                           : __uint_as_float((uint32_t)(step + 1 + kFirstStep) << 16);
      const float near = step == 0 ? 0.f : __uint_as_float((uint32_t)(step + kFirstStep) << 16);
      const uint32_t low = key, high = x.key(weight.top);
      const uint32_t lo = max(x.key(weight.top - far * 1.000001f), low + 2) - 2;
      border<true>([&](auto&& f) { tokens([&](int, float v) { f(v); }); }, lo,
                   min(x.key(weight.top - near * 0.999999f) + 2, high), limit_units, key, above);
      const double wk = weight(x.of_key(key));
      if (!(wk >= m)) return false;
      ties = that_stay(limit, above, wk);
      of_chunks(tokens, [&](int i) {                            // its earlier steps
        u64 v = 0;
        const int e0 = 2 * (threadIdx.x & 63);
        u64 two[kSteps / 128][2];                     // all on their way at once
#pragma unroll
        for (int j = 0; j < kSteps / 128; ++j)
          __builtin_memcpy(two[j], steps + i * kSteps + e0 + 128 * j, 16);
#pragma unroll
        for (int j = 0; j < kSteps / 128; ++j)
          v += (e0 + 128 * j < step ? two[j][0] : 0) + (e0 + 1 + 128 * j < step ? two[j][1] : 0);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
        return v;
      });
    } else if ((int)threadIdx.x < c.chunks) {
      sh.ties[threadIdx.x] = 0;
    }
    return true;
  }
};

// The largest logit of each slice.
template <int T>
__global__ void __launch_bounds__(kChunkThreads) sample_tops_kernel(SampleCall c) {
  const int64_t row = blockIdx.y;
  const Logits<T> x(c, row);
  const int lanes = 1 << (c.slice_shift - 3);         // of a slice: 4 or 16
  __shared__ float part[kChunkThreads / 64];
  float top = -__builtin_inff();
  float v[kChunk / kChunkThreads / 8][8];
#pragma unroll
  for (int i = 0; i < kChunk / kChunkThreads / 8; ++i) {
    const int at = blockIdx.x * kChunk + (i * kChunkThreads + (int)threadIdx.x) * 8;
    x.load(min(at, c.vocab), v[i]);
  }
#pragma unroll
  for (int i = 0; i < kChunk / kChunkThreads / 8; ++i) {
    const int at = blockIdx.x * kChunk + (i * kChunkThreads + (int)threadIdx.x) * 8;
    float best = v[i][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) best = fmaxf(best, v[i][j]);
    top = fmaxf(top, best);
    best = fmaxf(best, dpp_f32<kDppXor1>(best));
    best = fmaxf(best, dpp_f32<kDppXor2>(best));
    if (lanes == 16) {
      best = fmaxf(best, dpp_f32<kDppHalfMirror>(best));
      best = fmaxf(best, dpp_f32<kDppMirror>(best));
    }
    if (at < c.vocab && (threadIdx.x & (lanes - 1)) == 0)
      c.tops[row * c.slices + (at >> c.slice_shift)] = best;
  }
  if (!c.weighed) return;
  top = block_max<kChunkThreads / 64>(top, part);
  if (threadIdx.x == 0) c.chunk_tops[row * c.chunks + blockIdx.x] = top;
}

// Each chunk's weights, and by steps, of rows that need them.
template <int T>
__global__ void __launch_bounds__(kChunkThreads) sample_weights_kernel(SampleCall c) {
  constexpr int WAVES = kChunkThreads / 64;
  __shared__ u64 steps[kSteps];
  __shared__ union {
    float f[WAVES];
    u64 u[WAVES];
  } part;
  const int64_t row = blockIdx.y;
  const Settings s(c, row);
  if (!s.weighed(c.vocab)) return;
  const bool by_steps = s.by_steps(c.vocab);
  const Logits<T> x(c, row);
  float v[kChunk / kChunkThreads / 8][8];
#pragma unroll
  for (int i = 0; i < kChunk / kChunkThreads / 8; ++i) {
    const int at = blockIdx.x * kChunk + (i * kChunkThreads + (int)threadIdx.x) * 8;
    x.load(min(at, c.vocab), v[i]);
  }
  float top = -__builtin_inff();
  if ((int)threadIdx.x < c.chunks) top = c.chunk_tops[row * c.chunks + threadIdx.x];
  top = block_max<WAVES>(top, part.f);
  if (by_steps)
    for (int i = threadIdx.x; i < kSteps; i += kChunkThreads) steps[i] = 0;
  __syncthreads();
  const Weight weight(top, s.temperature);
  // Less than this part of the whole lies behind the border whatever the rest is: all such tokens
  // together weigh less than half of 1 - p, and the whole at least 1.
  const u64 least = (u64)ldexp(fmax(1.0 - (double)s.p, 0.0) / (2.0 * c.vocab), c.unit);
  u64 sum = 0;
#pragma unroll
  for (int i = 0; i < kChunk / kChunkThreads / 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u64 w = whole_units(weight(v[i][j]), c.unit);
      sum += w;
      if (by_steps && w > least) atomicAdd(&steps[step_of(top, v[i][j])], w);
    }
  u64 whole;
  block_scan<WAVES>(sum, part.u, whole);
  if (threadIdx.x == 0) c.sums[row * c.chunks + blockIdx.x] = whole;
  if (!by_steps) return;
  __syncthreads();
  u64* to = c.steps + (row * c.chunks + blockIdx.x) * kSteps;
  for (int i = threadIdx.x; i < kSteps; i += kChunkThreads) to[i] = steps[i];
}

template <int T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleCall c) {
  constexpr int THREADS = kThreads;
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const Settings s(c, row);
  const float u = c.u[row];
  const Logits<T> x(c, row);
  float top = -__builtin_inff();
  constexpr int kAhead = 5;
  const float* tops = c.tops + row * c.slices;
  for (int i0 = threadIdx.x; i0 < c.slices; i0 += kAhead * THREADS) {
    float v[kAhead];                    // several on their way at a time
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = min(i0 + j * THREADS, c.slices - 1);
      v[j] = c.slice_shift == 0 ? x.at(i) : tops[i];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      top = fmaxf(top, v[j]);
      if (i0 + j * THREADS < c.slices) sh.top[i0 + j * THREADS] = v[j];
    }
  }
  top = block_max<kWaves>(top, sh.part.f);
  Draw<T> d(c, row, sh, top, s, u);
  if (top == -__builtin_inff()) {
    if (threadIdx.x == 0) d.result(-1, -__builtin_inff());
    return;
  }
  if (s.greedy()) return d.greedy();
  if ((s.k < c.vocab || s.p < 1.f || s.m > 0.f) && d.by_list()) return;
  __syncthreads();
  bool found = d.held_step >= 0 && d.by_held(d.held_step);
  __syncthreads();
  if (!found) found = d.weighed && d.by_chunks();
  if (found) return d.in_chunk();
  __syncthreads();
  d.by_passes();
}

// What a call needs besides the last launch.
struct SamplePlan {
  int slice, chunks;
  bool weighed, steps;
  int64_t slices, steps_bytes, sums_bytes, bytes;
};

static SamplePlan sample_plan(int64_t rows, int64_t vocab, const mtl_sample_settings& s) {
  SamplePlan p{};
  p.slice = vocab <= kMaxSlices ? 1 : vocab <= 32 * kMaxSlices ? 32 : 128;
  p.slices = (vocab + p.slice - 1) / p.slice;
  if (p.slice == 1) return p;
  p.chunks = (int)((vocab + kChunk - 1) / kChunk);
  const bool k_open = s.top_k || s.top_k_all <= 0 || s.top_k_all >= vocab;
  const bool draws = s.temperature || s.temperature_all > 0.f;
  p.steps = k_open && draws && (s.top_p || (s.top_p_all < 1.f && s.top_p_all > 0.f));
  p.weighed = p.steps || (k_open && draws && (s.min_p || !(s.min_p_all > 0.f)));
  p.steps_bytes = p.steps ? rows * p.chunks * kSteps * 8 : 0;
  p.sums_bytes = p.weighed ? rows * p.chunks * 8 : 0;
  p.bytes = p.steps_bytes + p.sums_bytes + rows * (p.slices + p.chunks) * 4;
  return p;
}

template <int T>
static void launch_sample(const SampleCall& c, int64_t rows, hipStream_t stream) {
  const dim3 grid(c.chunks, (unsigned)rows);
  if (c.chunks) sample_tops_kernel<T><<<grid, kChunkThreads, 0, stream>>>(c);
  if (c.weighed) sample_weights_kernel<T><<<grid, kChunkThreads, 0, stream>>>(c);
  sample_kernel<T><<<(unsigned)rows, kThreads, 0, stream>>>(c);
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_sample_workspace_bytes(int64_t rows, int64_t vocab, int32_t type,
                                              const mtl_sample_settings* settings) {
  (void)type;
  if (!settings || rows < 1 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return 0;
  return sample_plan(rows, vocab, *settings).bytes;
}

extern "C" int mtl_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t type,
                          const float* u, const mtl_sample_settings* settings, int64_t* token,
                          float* logprob, void* workspace, int64_t ws_bytes, void* stream) {
  if (!settings || rows < 0 || vocab < 1 || ld < 0) return MTL_ERR_INVALID_ARG;
  if (type != MTL_T_BF16 && type != MTL_T_F16 && type != MTL_T_F32) return MTL_ERR_UNSUPPORTED;
  if (vocab > kMaxVocab || rows > kMaxRows) return MTL_ERR_SHAPE;
  if (rows == 0) return MTL_OK;
  if (!logits || !u || !token) return MTL_ERR_INVALID_ARG;
  const int size = type == MTL_T_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return MTL_ERR_ALIGN;
  const SamplePlan p = sample_plan(rows, vocab, *settings);
  if (p.bytes > 0 && (!workspace || ws_bytes < p.bytes)) return MTL_ERR_WORKSPACE;
  if (p.bytes > 0 && !aligned16(workspace)) return MTL_ERR_ALIGN;
  int unit = kMostUnit;
  while (vocab > (int64_t)1 << (63 - unit)) --unit;
  char* ws = static_cast<char*>(workspace);
  float* tops = reinterpret_cast<float*>(ws + p.steps_bytes + p.sums_bytes);
  const SampleCall c{logits, ld, (int)vocab, __builtin_ctz(p.slice), (int)p.slices, unit, p.chunks,
                     p.weighed, u, *settings, token, logprob, tops, tops + rows * p.slices,
                     reinterpret_cast<u64*>(ws + p.steps_bytes),
                     p.steps ? reinterpret_cast<u64*>(ws) : nullptr};
  hipStream_t st = (hipStream_t)stream;
  if (type == MTL_T_BF16) launch_sample<MTL_T_BF16>(c, rows, st);
  else if (type == MTL_T_F16) launch_sample<MTL_T_F16>(c, rows, st);
  else launch_sample<MTL_T_F32>(c, rows, st);
  return launch_status();
}
