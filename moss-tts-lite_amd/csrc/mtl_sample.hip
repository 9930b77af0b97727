// Drawing tokens from logits: temperature, top-k, top-p and min-p (gfx950).
//
// Everything is decided by sums of weights, and a row has as many borders as tokens: with float32
// sums (2^-24 of the whole) one row in some thousands would draw another token than the definition,
// so weights and sums are of 64 bits.  Sums that come together by atomics are whole numbers
// (weights in units of 2^-44), whose order changes nothing.
//
// A workgroup takes a row.  It never sorts the row:
// * The row is cut into slices; the largest logit of each gives a bound that at least n tokens
//   reach (n slices' largest do).  Only slices that reach it are read again, and give a short list
//   of candidates, in which every token counts those ahead of it and their weight.
// * Where a list of at most kCandidates cannot settle the row (a wide top-p, many equal logits),
//   the border token is found by counting or weighing the row by digits of its logits' ordered
//   keys, kBins at a time, and the draw follows in a last pass by index.
#include "mtl_common.h"
#include "mtl_paged.h"
#include "mtl_sample.h"

namespace mtl {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kCandidates = 512;
constexpr int kFew = 256;               // tokens that a list is made for
constexpr int kBins = 2048;
constexpr int kMaxSlices = 8192;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxRows = 65535;

struct SampleCall {
  const void* x;
  int64_t ld;
  int vocab, slice, slices, unit;       // unit: weights are counted in 2^-unit
  const float* u;
  mtl_sample_settings s;
  int64_t* token;
  float* logprob;
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

  // Logits i .. i + 7, -infinity past the end.
  __device__ __forceinline__ void load(int i, float (&x)[8]) const {
    if (i + 8 > n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = i + j < n ? at(i + j) : -__builtin_inff();
      return;
    }
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

  // Whole numbers in the logits' order, without the bits that the type does not have.
  static __device__ __forceinline__ uint32_t key(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kDrop;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    k = k << kDrop;
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k & ~((1u << kDrop) - 1));
  }
};

struct Weight {
  float top;
  double by;                            // 1 / temperature
  __device__ __forceinline__ double operator()(float x) const {
    return x == top ? 1.0 : x == -__builtin_inff() ? 0.0 : exp(((double)x - (double)top) * by);
  }
};

// Steps of the distance to the largest logit, 32 to an octave: the same or a later one for a
// smaller logit.
constexpr int kSteps = 1024;
__device__ __forceinline__ int step_of(float top, float x) {
  if (x == top) return 0;
  const int s = (int)(__float_as_uint(top - x) >> 18) - (117 * 32 - 1);
  return min(max(s, 0), kSteps - 1);
}

// ------------------------------------------------------------------------------ workgroup steps
// Inclusive sums over the workgroup in thread order, and their total; every thread takes part.
template <class V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
  const int lane = threadIdx.x & 63, wave = wave_id();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  V before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) before = sum;
    sum += part[i];
  }
  total = sum;
  return before + v;
}

__device__ __forceinline__ float block_max(float v, float* part) {
  v = wave_max_valu(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[wave_id()] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) v = fmaxf(v, part[i]);
  return v;
}

struct Shared {
  float top[kMaxSlices];                // each slice's largest logit
  union {
    u64 sums[kBins];
    struct {
      uint32_t steps[kSteps];
      int active[kCandidates];
      float x[2][kCandidates];
      int at[2][kCandidates];
      double w[kCandidates];
    } list;
  };
  union {
    double d[kWaves];
    u64 u[kWaves];
    int i[kWaves];
    float f[kWaves];
  } part;
  int n, m, first;
  u64 above;
};

// ------------------------------------------------------------------------------ a row
template <int T>
struct Draw {
  const SampleCall& c;
  const int64_t row;
  Shared& sh;
  const Logits<T> x;
  Weight weight;
  int k;
  double p, m, u;

  __device__ Draw(const SampleCall& c, int64_t row, Shared& sh) : c(c), row(row), sh(sh), x(c, row) {}

  __device__ void result(int token, double logprob) {
    c.token[row] = token;
    if (c.logprob) c.logprob[row] = (float)logprob;
  }

  // The lowest index of the largest logit.
  __device__ void greedy() {
    if (threadIdx.x == 0) sh.first = c.vocab;
    __syncthreads();
    for (int s = threadIdx.x; s < c.slices; s += kThreads) {
      if (sh.top[s] != weight.top) continue;
      for (int i = s * c.slice; i < min(c.vocab, (s + 1) * c.slice); ++i)
        if (x.at(i) == weight.top) {
          atomicMin(&sh.first, i);
          break;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) result(sh.first, 0.0);
  }

  // Calls f(index, logit) for all tokens of the row, a thread's slices one after the other.
  template <class F>
  __device__ __forceinline__ void all(F&& f) const {
    for (int s = threadIdx.x; s < c.slices; s += kThreads)
      for (int i = s * c.slice; i < (s + 1) * c.slice; i += 8) {
        float v[8];
        x.load(i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f(i + j, v[j]);
      }
  }

  // The sum of all weights.
  __device__ double total() {
    double sum = 0, whole;
    all([&](int, float v) { sum += weight(v); });
    block_scan(sum, sh.part.d, whole);
    return whole;
  }

  // Draws from a list of candidates; false where a list cannot settle the row.
  __device__ bool by_list() {
    auto& l = sh.list;
    const int t = threadIdx.x;
    const bool k_set = k < c.vocab;
    const int want = k_set ? min(k, kFew) : kFew;
    for (int i = t; i < kSteps; i += kThreads) l.steps[i] = 0;
    if (t == 0) sh.n = sh.m = 0;
    __syncthreads();
    int finite = 0;
    for (int s = t; s < c.slices; s += kThreads)
      if (sh.top[s] != -__builtin_inff()) {
        atomicAdd(&l.steps[step_of(weight.top, sh.top[s])], 1u);
        ++finite;
      }
    __syncthreads();
    // the first step that `want` slices reach, or the last
    int slices;
    const int upto = block_scan((int)l.steps[t], sh.part.i, slices);
    if (t == 0) sh.first = kSteps - 1;
    __syncthreads();
    if (upto >= want) atomicMin(&sh.first, t);
    __syncthreads();
    const int last = sh.first;
    for (int s = t; s < c.slices; s += kThreads)
      if (sh.top[s] != -__builtin_inff() && step_of(weight.top, sh.top[s]) <= last) {
        const int at = atomicAdd(&sh.m, 1);
        if (at < kCandidates) l.active[at] = s;
      }
    __syncthreads();
    const int active = sh.m;
    if (active > kCandidates) return false;
    for (int i = t; i < active * c.slice; i += kThreads) {
      const int e = l.active[i / c.slice] * c.slice + i % c.slice;
      const float v = e < c.vocab ? x.at(e) : -__builtin_inff();
      if (v != -__builtin_inff() && step_of(weight.top, v) <= last) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kCandidates) {
          l.x[0][at] = v;
          l.at[0][at] = e;
        }
      }
    }
    __syncthreads();
    const int n = sh.n;
    if (n > kCandidates) return false;
    // by index, so that sums have one order
    if (t < n) {
      int to = 0;
      const int mine = l.at[0][t];
      for (int j = 0; j < n; ++j) to += l.at[0][j] < mine;
      l.x[1][to] = l.x[0][t];
      l.at[1][to] = mine;
      l.w[to] = weight(l.x[0][t]);
    }
    __syncthreads();
    int rank = 0;
    double before = 0, w = 0;
    float v = 0;
    if (t < n) {
      v = l.x[1][t];
      w = l.w[t];
      for (int j = 0; j < n; ++j) {
        const float y = l.x[1][j];
        if (y > v || (y == v && j < t)) {
          ++rank;
          before += l.w[j];
        }
      }
    }
    double mass;
    const bool in_k = t < n && rank < k;
    block_scan(in_k ? w : 0.0, sh.part.d, mass);
    if (last < kSteps - 1 && !(k_set && k <= n)) {    // tokens outside the list may count
      if (k_set) return false;
      int low;
      block_scan((int)(t < n && !(w >= m)), sh.part.i, low);
      if (!low && p >= 1) return false;
      const double whole = p < 1 ? total() : 0.0;
      if (!low && !(mass > p * whole)) return false;
      mass = whole;
    }
    const bool keep = in_k && (p >= 1 || before <= p * mass) && (w >= m || rank == 0);
    double whole;
    const double upto_w = block_scan(keep ? w : 0.0, sh.part.d, whole);
    if (t == 0) {
      sh.first = kCandidates;
      sh.m = -1;
    }
    __syncthreads();
    if (keep && w > 0) {
      atomicMax(&sh.m, t);                            // the last one, where rounding leaves none
      if (upto_w > u * whole) atomicMin(&sh.first, t);
    }
    __syncthreads();
    if (t == min(sh.first, sh.m)) result(l.at[1][t], log(w / whole));
    return true;
  }

  // A border in the order of keys: the key at which `limit` is passed, going down from the largest,
  // and what lies above it.  WEIGH: weights in units of 2^-unit, else tokens.
  template <bool WEIGH>
  __device__ void border(uint32_t lo, u64 limit, uint32_t& key, u64& above) {
    uint32_t hi = x.key(weight.top);
    above = 0;
    while (true) {
      const uint32_t range = hi - lo;
      const int shift = range < kBins ? 0 : 21 - __builtin_clz(range);
      const int bins = (int)(range >> shift) + 1;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += kThreads) sh.sums[i] = 0;
      if (threadIdx.x == 0) {
        sh.first = kBins;
        sh.m = -1;
      }
      __syncthreads();
      all([&](int, float v) {
        const uint32_t b = x.key(v);
        if (v != -__builtin_inff() && b >= lo && b <= hi)
          atomicAdd(&sh.sums[(b - lo) >> shift],
                    WEIGH ? (u64)rint(ldexp(weight(v), c.unit)) : (u64)1);
      });
      __syncthreads();
      const int j = 2 * threadIdx.x;                  // bins from the largest key down
      const u64 a = j < bins ? sh.sums[bins - 1 - j] : 0;
      const u64 b = j + 1 < bins ? sh.sums[bins - 2 - j] : 0;
      u64 all_of;
      const u64 upto = block_scan(a + b, sh.part.u, all_of), ahead = above + upto - a - b;
      const bool at_a = WEIGH ? ahead + a > limit : ahead + a >= limit;
      const bool at_b = WEIGH ? ahead + a + b > limit : ahead + a + b >= limit;
      if (at_a || at_b) atomicMin(&sh.first, at_a ? j : j + 1);
      if (a || b) atomicMax(&sh.m, b ? j + 1 : j);
      __syncthreads();
      const int pick = min(sh.first, max(sh.m, 0));
      if (pick == j || pick == j + 1) sh.above = pick == j ? ahead : ahead + a;
      __syncthreads();
      above = sh.above;
      lo += (uint32_t)(bins - 1 - pick) << shift;
      if (shift == 0) break;
      hi = min(hi, lo + ((1u << shift) - 1));
    }
    key = lo;
  }

  // Draws by passes over the row.
  __device__ void by_passes() {
    uint32_t key = x.key(-__builtin_inff()) + 1, at;
    int ties = c.vocab;                               // of that key, how many stay
    u64 above;
    if (k < c.vocab) {
      border<false>(key, (u64)k, at, above);
      key = at;
      ties = k - (int)above;
    }
    if (p < 1) {
      // the weight of what top-k left
      double sum = 0, mass;
      int same = 0, all_same;
      all([&](int, float v) {
        if (x.key(v) > key) sum += weight(v);
        same += x.key(v) == key && v != -__builtin_inff();
      });
      block_scan(sum, sh.part.d, mass);
      block_scan(same, sh.part.i, all_same);
      mass += (double)min(ties, all_same) * weight(x.of_key(key));
      border<true>(key, (u64)ldexp(p * mass, c.unit), at, above);
      const double w = weight(x.of_key(at));
      const double room = (p * mass - ldexp((double)above, -c.unit)) / w;
      const int stay = room < (double)c.vocab ? max((int)floor(room) + 1, 1) : c.vocab;
      ties = at == key ? min(ties, stay) : stay;
      key = at;
    }
    // by index: each thread a run of slices
    const int per = (c.slices + kThreads - 1) / kThreads;
    const int begin = min(c.vocab, (int)threadIdx.x * per * c.slice);
    const int end = min(c.vocab, begin + per * c.slice);
    const double wk = weight(x.of_key(key));
    double sum = 0;
    int same = 0;
    for (int i = begin; i < end; i += 8) {
      float v[8];
      x.load(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j >= end || v[j] == -__builtin_inff()) continue;
        const uint32_t b = x.key(v[j]);
        same += b == key;
        if (b > key) {
          const double w = weight(v[j]);
          if (w >= m || v[j] == weight.top) sum += w;
        }
      }
    }
    int all_same;
    const int had = block_scan(same, sh.part.i, all_same) - same;
    const bool tie_stays = wk >= m || x.of_key(key) == weight.top;
    if (tie_stays) sum += (double)min(max(ties - had, 0), same) * wk;
    double whole;
    const double upto = block_scan(sum, sh.part.d, whole);
    const double goal = u * whole;
    if (threadIdx.x == 0) {
      sh.first = kThreads;
      sh.m = -1;
    }
    __syncthreads();
    if (sum > 0) {
      atomicMax(&sh.m, (int)threadIdx.x);
      if (upto > goal) atomicMin(&sh.first, (int)threadIdx.x);
    }
    __syncthreads();
    if ((int)threadIdx.x != min(sh.first, sh.m)) return;
    // within the run that the draw falls into
    double run = upto - sum, w_last = 0;
    int last = -1, seen = had;
    for (int i = begin; i < end; ++i) {
      const float v = x.at(i);
      if (v == -__builtin_inff()) continue;
      const uint32_t b = x.key(v);
      if (b < key || (b == key && seen++ >= ties)) continue;
      const double w = weight(v);
      if (!(w >= m || v == weight.top) || !(w > 0)) continue;
      run += w;
      last = i;
      w_last = w;
      if (run > goal) break;
    }
    result(last, log(w_last / whole));
  }
};

template <int T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleCall c) {
  __shared__ Shared sh;
  Draw<T> d(c, blockIdx.x, sh);
  const mtl_sample_settings& s = c.s;
  const int64_t r = d.row;
  const float temperature = s.temperature ? s.temperature[r] : s.temperature_all;
  const int k = s.top_k ? s.top_k[r] : s.top_k_all;
  const float p = s.top_p ? s.top_p[r] : s.top_p_all, m = s.min_p ? s.min_p[r] : s.min_p_all;
  const float u = c.u[r];
  float top = -__builtin_inff();
  for (int i = threadIdx.x; i < c.slices; i += kThreads) {
    float best = -__builtin_inff();
    for (int e = i * c.slice; e < (i + 1) * c.slice; e += 8) {
      float v[8];
      d.x.load(e, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) best = fmaxf(best, v[j]);
    }
    sh.top[i] = best;
    top = fmaxf(top, best);
  }
  top = block_max(top, sh.part.f);
  d.weight.top = top;
  d.weight.by = 1.0 / (double)fminf(temperature, 3.4028234663852886e38f);
  d.k = k <= 0 || k > c.vocab ? c.vocab : k;
  d.p = p;
  d.m = m;
  d.u = u >= 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
  if (top == -__builtin_inff()) {
    if (threadIdx.x == 0) d.result(-1, -__builtin_inff());
    return;
  }
  // settings that leave the first of the order alone
  if (!(temperature > 0.f) || k == 1 || !(p > 0.f) || !(m <= 1.f)) return d.greedy();
  if ((d.k < c.vocab || p < 1.f || m > 0.f) && d.by_list()) return;
  __syncthreads();
  d.by_passes();
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_sample_workspace_bytes(int64_t rows, int64_t vocab, int32_t type,
                                              const mtl_sample_settings* settings) {
  (void)rows, (void)vocab, (void)type, (void)settings;
  return 0;
}

extern "C" int mtl_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t type,
                          const float* u, const mtl_sample_settings* settings, int64_t* token,
                          float* logprob, void* workspace, int64_t ws_bytes, void* stream) {
  (void)workspace, (void)ws_bytes;
  if (!settings || rows < 0 || vocab < 1 || ld < 0) return MTL_ERR_INVALID_ARG;
  if (type != MTL_T_BF16 && type != MTL_T_F16 && type != MTL_T_F32) return MTL_ERR_UNSUPPORTED;
  if (vocab > kMaxVocab || rows > kMaxRows) return MTL_ERR_SHAPE;
  if (rows == 0) return MTL_OK;
  if (!logits || !u || !token) return MTL_ERR_INVALID_ARG;
  const int size = type == MTL_T_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return MTL_ERR_ALIGN;
  int unit = 44;
  while (unit > 0 && (vocab >> (62 - unit)) > 0) --unit;
  const int slice = vocab <= 8 * kThreads ? 8 : vocab <= 32 * kMaxSlices ? 32 : 128;
  const SampleCall c{logits, ld, (int)vocab, slice, (int)((vocab + slice - 1) / slice), unit, u,
                     *settings, token, logprob};
  hipStream_t st = (hipStream_t)stream;
  if (type == MTL_T_BF16) sample_kernel<MTL_T_BF16><<<(unsigned)rows, kThreads, 0, st>>>(c);
  else if (type == MTL_T_F16) sample_kernel<MTL_T_F16><<<(unsigned)rows, kThreads, 0, st>>>(c);
  else sample_kernel<MTL_T_F32><<<(unsigned)rows, kThreads, 0, st>>>(c);
  return launch_status();
}
