// Bookkeeping of a paged key-value cache on the device (gfx950): extending, forking and
// truncating sequences, compaction of the pool, and the copies of whole pages these need.
//
// A call decides in one workgroup (its checks, the order of its entries and the choice of the
// lowest free pages are global), then, where work grows with the sequences' lengths, a second
// launch carries it out.  Every result is a function of the arguments alone: pages are taken in
// ascending order by ranks from prefix sums, and the atomics only add integers.
#include "mtl_common.h"
#include "mtl_paged.h"

namespace mtl {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxCall = MTL_PAGES_MAX_CALL;
constexpr int kMaxSeqs = MTL_PAGES_MAX_SEQS;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Exclusive prefix sum over the workgroup's threads; total receives the sum.  All threads.
template <class I>
__device__ __forceinline__ I block_scan(I v, I* waves, I& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  I x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const I y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                       // the sums of an earlier call have been read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  I before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const I s = waves[w];
    before += w < wave ? s : 0;
    sum += s;
  }
  total = sum;
  return before + x - v;
}

// Marks s; true when it was marked before.
__device__ __forceinline__ bool mark(uint32_t* bits, int s) {
  const uint32_t b = 1u << (s & 31);
  return atomicOr(&bits[s >> 5], b) & b;
}

__device__ __forceinline__ int pages_of(int64_t len, int page_size) {
  return (int)((len + page_size - 1) / page_size);
}

__global__ void __launch_bounds__(kThreads) pages_extend_kernel(
    mtl_page_state st, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int n,
    int32_t* __restrict__ copy_src, int32_t* __restrict__ copy_dst, int32_t* __restrict__ status,
    int32_t* __restrict__ list) {
  __shared__ uint32_t seen[kMaxSeqs / 32];
  __shared__ int last[kMaxCall], off[kMaxCall], first[kMaxCall], seq[kMaxCall];
  __shared__ int64_t waves64[kWaves];
  __shared__ int waves[kWaves];
  __shared__ int bad, shared_pages;
  const int t = threadIdx.x;
  for (int i = t; i < kMaxSeqs / 32; i += kThreads) seen[i] = 0;
  if (t == 0) bad = shared_pages = 0;
  __syncthreads();
  const int64_t cap = st.width * st.page_size;
  int s = 0, c = 0, held = 0, page = -1, page_refs = 0;
  int64_t len = 0;
  bool wrong = false;
  if (t < n) {
    s = seqs[t];
    c = counts[t];
    wrong = s < 0 || s >= st.seqs || c < 0;
    if (!wrong) {
      len = st.lens[s];
      wrong = mark(seen, s) || len < 0 || len + c > cap || len + c > INT32_MAX;
    }
    if (!wrong) {
      held = pages_of(len, st.page_size);
      if (c > 0 && len % st.page_size) {
        const int p = st.table[s * st.ld + len / st.page_size];
        if (p >= 0 && p < st.pages && (page_refs = st.refs[p]) > 1) page = p;
      }
    }
    if (wrong) bad = 1;
    last[t] = page;
    if (page >= 0) shared_pages = 1;
  }
  __syncthreads();
  // Of the sequences that share a partly filled page, each of a call's in turn takes a copy
  // while others hold it still; the last holder keeps it.
  bool copy = false;
  if (shared_pages && page >= 0) {
    int earlier = 0;
    for (int i = 0; i < t; ++i) earlier += last[i] == page;
    copy = page_refs - earlier > 1;
  }
  int64_t need = 0, total;
  if (t < n && !wrong) need = pages_of(len + c, st.page_size) - held + (copy ? 1 : 0);
  const int64_t at = block_scan<int64_t>(need, waves64, total);
  int64_t found = 0;
  if (!bad && total <= st.pages) {
    for (int64_t p0 = 0; p0 < st.pages && found < total; p0 += kThreads) {
      const int64_t p = p0 + t;
      const int free_page = p < st.pages && st.refs[p] == 0;
      int here;
      const int64_t rank = found + block_scan<int>(free_page, waves, here);
      if (free_page && rank < total) list[rank] = (int)p;
      found += here;
    }
  }
  const bool ok = !bad && total <= found;
  if (t == 0) status[0] = bad ? 2 : ok ? 0 : 1;
  if (t < n) {
    off[t] = (int)at;
    first[t] = copy ? (int)(len / st.page_size) : held;    // a copied page is the one before
    seq[t] = s;
  }
  __syncthreads();                                         // the list and the entries' places
  if (t < n) {
    copy_src[t] = ok && copy ? page : -1;
    copy_dst[t] = ok && copy ? list[at] : -1;
    if (ok) {
      st.lens[s] = (int)(len + c);
      if (copy) atomicSub(&st.refs[page], 1);
    }
  }
  if (!ok) return;
  for (int r = t; r < total; r += kThreads) {
    int lo = 0, hi = n - 1;                                // the last entry with off <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (off[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int p = list[r];
    st.table[seq[lo] * st.ld + first[lo] + (r - off[lo])] = p;
    st.refs[p] = 1;
  }
}

__global__ void __launch_bounds__(kThreads) pages_fork_check_kernel(
    mtl_page_state st, const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
    int n, int32_t* __restrict__ status, int32_t* __restrict__ held) {
  __shared__ uint32_t seen[kMaxSeqs / 32];
  __shared__ int bad;
  const int t = threadIdx.x;
  for (int i = t; i < kMaxSeqs / 32; i += kThreads) seen[i] = 0;
  if (t == 0) bad = 0;
  __syncthreads();
  int p = 0, c = 0;
  int64_t len = 0;
  bool wrong = false;
  if (t < n) {
    p = parents[t];
    c = children[t];
    wrong = p < 0 || p >= st.seqs || c < 0 || c >= st.seqs;
    if (!wrong) {
      len = st.lens[p];
      wrong = mark(seen, c) || st.lens[c] != 0 || len < 0 || len > st.width * st.page_size;
    }
  }
  __syncthreads();
  if (t < n && !wrong) wrong = seen[p >> 5] >> (p & 31) & 1;
  if (wrong) bad = 1;
  __syncthreads();
  if (t == 0) status[0] = bad ? 2 : 0;
  if (t < n) {
    held[t] = bad ? 0 : pages_of(len, st.page_size);
    if (!bad) st.lens[c] = (int)len;
  }
}

__global__ void __launch_bounds__(256) pages_fork_kernel(
    mtl_page_state st, const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
    const int32_t* __restrict__ held) {
  const int i = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= held[i]) return;
  const int p = st.table[parents[i] * st.ld + j];
  st.table[children[i] * st.ld + j] = p;
  if (p >= 0 && p < st.pages) atomicAdd(&st.refs[p], 1);
}

__global__ void __launch_bounds__(kThreads) pages_truncate_check_kernel(
    mtl_page_state st, const int32_t* __restrict__ seqs, const int32_t* __restrict__ new_lens,
    int n, int32_t* __restrict__ status, int32_t* __restrict__ held) {
  __shared__ uint32_t seen[kMaxSeqs / 32];
  __shared__ int bad;
  const int t = threadIdx.x;
  for (int i = t; i < kMaxSeqs / 32; i += kThreads) seen[i] = 0;
  if (t == 0) bad = 0;
  __syncthreads();
  int s = 0, keep = 0;
  int64_t len = 0;
  bool wrong = false;
  if (t < n) {
    s = seqs[t];
    keep = new_lens[t];
    wrong = s < 0 || s >= st.seqs || keep < 0;
    if (!wrong) {
      len = st.lens[s];
      wrong = mark(seen, s) || keep > len || len > st.width * st.page_size;
    }
    if (wrong) bad = 1;
  }
  __syncthreads();
  if (t == 0) status[0] = bad ? 2 : 0;
  if (t < n) {
    held[t] = bad ? 0 : pages_of(len, st.page_size);
    if (!bad) st.lens[s] = keep;
  }
}

__global__ void __launch_bounds__(256) pages_truncate_kernel(
    mtl_page_state st, const int32_t* __restrict__ seqs, const int32_t* __restrict__ new_lens,
    const int32_t* __restrict__ held) {
  const int i = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= held[i] || j < pages_of(new_lens[i], st.page_size)) return;
  int32_t* e = st.table + seqs[i] * st.ld + j;
  const int p = *e;
  *e = -1;
  if (p >= 0 && p < st.pages) atomicSub(&st.refs[p], 1);
}

__global__ void __launch_bounds__(kThreads) pages_compact_plan_kernel(
    const int32_t* refs, int64_t pages, int32_t* refs_out, int32_t* __restrict__ live_out,
    int32_t* __restrict__ moves_out, int32_t* __restrict__ src, int32_t* __restrict__ dst,
    int32_t* __restrict__ goes) {
  __shared__ int waves[kWaves];
  const int t = threadIdx.x;
  int held = 0, live;
  for (int64_t p = t; p < pages; p += kThreads) held += refs[p] > 0;
  block_scan<int>(held, waves, live);
  int movers = 0, holes = 0;
  for (int64_t p0 = 0; p0 < pages; p0 += kThreads) {
    const int64_t p = p0 + t;
    const bool in = p < pages, used = in && refs[p] > 0;
    const int mover = used && p >= live, hole = in && !used && p < live;
    int sum;                                   // both counts stay below 2^16 in a strip
    const int ranks = block_scan<int>(mover | hole << 16, waves, sum);
    if (mover) src[movers + (ranks & 0xffff)] = (int)p;
    if (hole) dst[holes + (ranks >> 16)] = (int)p;
    if (in && p >= live && !mover) goes[p] = (int)p;
    movers += sum & 0xffff;
    holes += sum >> 16;
  }
  __syncthreads();
  // refs_out may be refs: the moved counts first, read past live and written below it
  for (int k = t; k < movers; k += kThreads) {
    goes[src[k]] = dst[k];
    refs_out[dst[k]] = refs[src[k]];
  }
  __syncthreads();
  for (int64_t p = t; p < pages; p += kThreads) {
    if (p >= live) refs_out[p] = 0;
    else if (refs[p] > 0) refs_out[p] = refs[p];
  }
  if (t == 0) {
    live_out[0] = live;
    moves_out[0] = movers;
  }
}

__global__ void __launch_bounds__(256) pages_compact_table_kernel(
    const int32_t* table, int64_t ld, int64_t width, int32_t* table_out, int64_t ld_out,
    int64_t pages, const int32_t* __restrict__ live, const int32_t* __restrict__ goes) {
  const int64_t j = blockIdx.x * (int64_t)256 + threadIdx.x, s = blockIdx.y;
  if (j >= width) return;
  const int p = table[s * ld + j];
  table_out[s * ld_out + j] = p >= live[0] && p < pages ? goes[p] : p;
}

__global__ void __launch_bounds__(256) pages_copy_kernel(
    char* __restrict__ k, char* __restrict__ v, int64_t k_layer, int64_t v_layer, int64_t k_page,
    int64_t v_page, int64_t page_bytes, int64_t pages, const int32_t* __restrict__ src,
    const int32_t* __restrict__ dst, const int32_t* __restrict__ count) {
  const int i = blockIdx.x;
  if (count && i >= count[0]) return;
  const int64_t a = src[i], b = dst[i], l = blockIdx.y;
  if (a < 0 || a >= pages || b < 0 || b >= pages) return;
  const char* from = blockIdx.z ? v + l * v_layer + a * v_page : k + l * k_layer + a * k_page;
  char* to = blockIdx.z ? v + l * v_layer + b * v_page : k + l * k_layer + b * k_page;
  for (int64_t o = 16 * threadIdx.x; o < page_bytes; o += 16 * 256)
    *reinterpret_cast<u32x4*>(to + o) = *reinterpret_cast<const u32x4*>(from + o);
}

// Arguments every bookkeeping entry shares.
static int check_state(const mtl_page_state* st, int64_t n, const void* status, const void* ws,
                       int64_t ws_bytes, bool lens = true) {
  if (!st || n < 0 || st->seqs < 0 || st->width < 0 || st->ld < st->width || st->pages < 0 ||
      st->pages > INT32_MAX || !status)
    return MTL_ERR_INVALID_ARG;
  if (n > kMaxCall || st->seqs > kMaxSeqs) return MTL_ERR_SHAPE;
  if (st->page_size < 1 || (st->page_size & (st->page_size - 1))) return MTL_ERR_SHAPE;
  if (st->width > INT32_MAX / st->page_size) return MTL_ERR_SHAPE;
  if ((st->seqs > 0 && ((lens && !st->lens) || (st->width > 0 && !st->table))) ||
      (st->pages > 0 && !st->refs))
    return MTL_ERR_INVALID_ARG;
  if (!ws || ws_bytes < mtl_pages_workspace_bytes(n, st->pages)) return MTL_ERR_WORKSPACE;
  return MTL_OK;
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_pages_workspace_bytes(int64_t n, int64_t pages) {
  if (n < 0 || pages < 0) return 0;
  return 4 * (n + pages + 16);
}

extern "C" int mtl_pages_extend(const mtl_page_state* st, const int32_t* seqs,
                                const int32_t* counts, int64_t n, int32_t* copy_src,
                                int32_t* copy_dst, int32_t* status, void* workspace,
                                int64_t ws_bytes, void* stream) {
  const int e = check_state(st, n, status, workspace, ws_bytes);
  if (e != MTL_OK) return e;
  if (n > 0 && (!seqs || !counts || !copy_src || !copy_dst)) return MTL_ERR_INVALID_ARG;
  pages_extend_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(
      *st, seqs, counts, (int)n, copy_src, copy_dst, status, static_cast<int32_t*>(workspace));
  return launch_status();
}

extern "C" int mtl_pages_fork(const mtl_page_state* st, const int32_t* parents,
                              const int32_t* children, int64_t n, int32_t* status,
                              void* workspace, int64_t ws_bytes, void* stream) {
  const int e = check_state(st, n, status, workspace, ws_bytes);
  if (e != MTL_OK) return e;
  if (n > 0 && (!parents || !children)) return MTL_ERR_INVALID_ARG;
  int32_t* held = static_cast<int32_t*>(workspace);
  pages_fork_check_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(*st, parents, children, (int)n,
                                                                   status, held);
  if (n > 0 && st->width > 0) {
    const dim3 grid((unsigned)((st->width + 255) / 256), (unsigned)n);
    pages_fork_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(*st, parents, children, held);
  }
  return launch_status();
}

extern "C" int mtl_pages_truncate(const mtl_page_state* st, const int32_t* seqs,
                                  const int32_t* new_lens, int64_t n, int32_t* status,
                                  void* workspace, int64_t ws_bytes, void* stream) {
  const int e = check_state(st, n, status, workspace, ws_bytes);
  if (e != MTL_OK) return e;
  if (n > 0 && (!seqs || !new_lens)) return MTL_ERR_INVALID_ARG;
  int32_t* held = static_cast<int32_t*>(workspace);
  pages_truncate_check_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(*st, seqs, new_lens, (int)n,
                                                                       status, held);
  if (n > 0 && st->width > 0) {
    const dim3 grid((unsigned)((st->width + 255) / 256), (unsigned)n);
    pages_truncate_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(*st, seqs, new_lens, held);
  }
  return launch_status();
}

extern "C" int mtl_pages_compact(const mtl_page_state* st, int32_t* table_out, int64_t ld_out,
                                 int32_t* refs_out, int32_t* live, int32_t* moves,
                                 int32_t* move_src, int32_t* move_dst, void* workspace,
                                 int64_t ws_bytes, void* stream) {
  const int e = check_state(st, 0, live, workspace, ws_bytes, false);
  if (e != MTL_OK) return e;
  if (!moves || ld_out < st->width || (st->pages > 0 && !refs_out) ||
      (st->pages > 1 && (!move_src || !move_dst)) ||
      (st->seqs > 0 && st->width > 0 && !table_out))
    return MTL_ERR_INVALID_ARG;
  int32_t* goes = static_cast<int32_t*>(workspace);
  pages_compact_plan_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(
      st->refs, st->pages, refs_out, live, moves, move_src, move_dst, goes);
  if (st->seqs > 0 && st->width > 0) {
    const dim3 grid((unsigned)((st->width + 255) / 256), (unsigned)st->seqs);
    pages_compact_table_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(
        st->table, st->ld, st->width, table_out, ld_out, st->pages, live, goes);
  }
  return launch_status();
}

extern "C" int mtl_pages_copy(void* k, void* v, int64_t layers, int64_t k_layer, int64_t v_layer,
                              int64_t k_page, int64_t v_page, int64_t page_bytes, int64_t pages,
                              const int32_t* src, const int32_t* dst, int64_t n,
                              const int32_t* count, void* stream) {
  if (layers < 0 || k_layer < 0 || v_layer < 0 || page_bytes < 0 || pages < 0 || n < 0 ||
      k_page < page_bytes || v_page < page_bytes)
    return MTL_ERR_INVALID_ARG;
  if (layers == 0 || page_bytes == 0 || pages == 0 || n == 0) return MTL_OK;
  if (!k || !v || !src || !dst) return MTL_ERR_INVALID_ARG;
  if (!aligned16(k) || !aligned16(v) || k_layer % 16 || v_layer % 16 || k_page % 16 ||
      v_page % 16 || page_bytes % 16)
    return MTL_ERR_ALIGN;
  if (layers > 65535 || n > INT32_MAX) return MTL_ERR_SHAPE;
  const dim3 grid((unsigned)n, (unsigned)layers, 2);
  pages_copy_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(
      static_cast<char*>(k), static_cast<char*>(v), k_layer, v_layer, k_page, v_page, page_bytes,
      pages, src, dst, count);
  return launch_status();
}
