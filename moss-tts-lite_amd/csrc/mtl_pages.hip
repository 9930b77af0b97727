// Bookkeeping of a paged key-value cache on the device (gfx950): extending, forking and
// truncating sequences, compaction of the pool, and the copies of whole pages these need.
//
// A call decides in one workgroup (its checks, the order of its entries and the choice of the
// lowest free pages are global), then, where work grows with the sequences' lengths, a second
// launch carries it out.  Every result is a function of the arguments alone: pages are taken in
// ascending order by ranks from prefix sums, and the atomics only add integers.
#include "mtl_paged_pool.h"

namespace mtl {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxCall = MTL_PAGES_MAX_CALL;
constexpr int kMaxSeqs = MTL_PAGES_MAX_SEQS;
constexpr int kStrip = 16 * kThreads;    // pages the workgroup looks at in one turn
// Table entries up to which the deciding workgroup does the work itself, and a second launch
// costs more than it saves.  Forking and freeing 16 sequences of 30 pages 6.3 us in one launch
// each, 8.1 in two; 64 of 16 pages 10.4 and 8.0.  Planning a compaction with 3000 entries 5.8 and
// 7.2, with 10000 10.8 and 9.0.
constexpr int64_t kMoveHere = kThreads;
constexpr int64_t kTableHere = 4 * kThreads;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Exclusive prefix sum over the workgroup's threads; total receives the sum.  All threads.
__device__ __forceinline__ int block_scan(int v, int* waves, int& total) {
  const int wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();                       // the sums of an earlier call have been read
  if ((threadIdx.x & 63) == 63) waves[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int s = waves[w];
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

__device__ __forceinline__ void clear_marks(uint32_t* bits, int64_t seqs) {
  for (int i = threadIdx.x; i < (seqs + 31) / 32; i += kThreads) bits[i] = 0;
}

__device__ __forceinline__ int pages_of(int64_t len, int page_size) {
  return (int)((len + page_size - 1) / page_size);
}

// The counts of pages p0 .. p0 + 15, on their way; pages past the pool count as held.
struct Counts {
  int4 v[4];
  __device__ __forceinline__ void load(const int32_t* refs, int64_t p0, int64_t pages) {
    if (p0 + 16 <= pages && (reinterpret_cast<uintptr_t>(refs) & 15u) == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const int4*>(refs + p0 + 4 * i);
    } else {
      auto at = [&](int64_t p) { return p < pages ? refs[p] : 1; };
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = make_int4(at(p0 + 4 * i), at(p0 + 4 * i + 1), at(p0 + 4 * i + 2),
                         at(p0 + 4 * i + 3));
    }
  }
  // bit i: page p0 + i is held
  __device__ __forceinline__ uint32_t held() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m |= ((v[i].x > 0) | (v[i].y > 0) << 1 | (v[i].z > 0) << 2 | (v[i].w > 0) << 3) << 4 * i;
    return m;
  }
};

__device__ __forceinline__ uint32_t held_mask(const int32_t* refs, int64_t p0, int64_t pages) {
  Counts c;
  c.load(refs, p0, pages);
  return c.held();
}

// What an entry of a call to fork or truncate moves: pages first .. held - 1, none where held is
// not past first (a refused call's spans are empty: row and from may lie outside the table).
struct Span {
  int row, from, first, held;            // row: the table row written; from: the one read
};

// Forks (FORK) or truncates one page.
template <bool FORK>
__device__ __forceinline__ void move_page(const mtl_page_state& st, const Span& s, int j) {
  if (j >= s.held) return;
  const int p = st.table[s.from * st.ld + j];
  st.table[s.row * st.ld + j] = FORK ? p : -1;
  if (p >= 0 && p < st.pages) atomicAdd(&st.refs[p], FORK ? 1 : -1);
}

// A lane an entry: checks, the pages each needs (prefix sum), then the lowest free pages in strips
// of kStrip counts until there are enough (the next strip on its way meanwhile), then the writes.
// Bound by the trips to the memory that wait for one another (entry, length, table, count; counts;
// the writes): 5.2 us for 2 entries, 7.6 for 64.  Entries that share a partly filled page count
// their forerunners one by one: a call of 64 such entries takes 5 us longer, of 256 10, of 1024 35,
// the copies included.
__global__ void __launch_bounds__(kThreads) pages_extend_kernel(
    mtl_page_state st, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int n,
    int32_t* __restrict__ copy_src, int32_t* __restrict__ copy_dst, int32_t* __restrict__ copies,
    int32_t* __restrict__ status, int32_t* __restrict__ list) {
  __shared__ uint32_t seen[kMaxSeqs / 32];
  __shared__ int last[kMaxCall], off[kMaxCall], first[kMaxCall], seq[kMaxCall];
  __shared__ int waves[kWaves];
  __shared__ int bad, shared_pages;
  const int t = threadIdx.x;
  Counts strip;                          // of the search for free pages, always one ahead
  strip.load(st.refs, 16 * t, st.pages);
  clear_marks(seen, st.seqs);
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
      wrong = mark(seen, s) || len < 0 || len + c > cap;
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
  int need = 0, total, all_copies;
  if (t < n && !wrong) need = pages_of(len + c, st.page_size) - held + copy;
  const int at = block_scan(need, waves, total);
  const int place = block_scan(copy, waves, all_copies);
  int found = 0;
  if (!bad) {
    for (int64_t p0 = 0; p0 < st.pages && found < total; p0 += kStrip) {
      const int64_t p = p0 + 16 * t;
      uint32_t free_pages = ~strip.held() & 0xffffu;
      if (p0 + kStrip < st.pages) strip.load(st.refs, p + kStrip, st.pages);
      int here;
      int rank = found + block_scan(__popc(free_pages), waves, here);
      for (; free_pages && rank < total; free_pages &= free_pages - 1)
        list[rank++] = (int)p + __ffs(free_pages) - 1;
      found += here;
    }
  }
  const bool ok = !bad && total <= found;
  if (t == 0) {
    status[0] = bad ? 2 : ok ? 0 : 1;
    copies[0] = ok ? all_copies : 0;
  }
  if (t < n) {
    off[t] = at;
    first[t] = copy ? (int)(len / st.page_size) : held;    // a copied page is the one before
    seq[t] = s;
  }
  __syncthreads();                                         // the list and the entries' places
  if (!ok) return;
  if (t < n) {
    st.lens[s] = (int)(len + c);
    if (copy) {
      copy_src[place] = page;
      copy_dst[place] = list[at];
      atomicSub(&st.refs[page], 1);
    }
  }
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

// Checks a call to fork or truncate and moves its pages, or leaves that to the next launch
// (spans).  a, b: parents and children, or sequences and new lengths.
template <bool FORK, bool ALL>
__global__ void __launch_bounds__(kThreads) pages_move_kernel(
    mtl_page_state st, const int32_t* __restrict__ a, const int32_t* __restrict__ b, int n,
    int32_t* __restrict__ status, Span* __restrict__ spans_out) {
  __shared__ uint32_t seen[kMaxSeqs / 32];
  __shared__ Span spans[kMaxCall];
  __shared__ int bad, widest;
  const int t = threadIdx.x;
  clear_marks(seen, st.seqs);
  if (t == 0) bad = widest = 0;
  __syncthreads();
  const int64_t cap = st.width * st.page_size;
  int x = 0, y = 0;
  int64_t len = 0;
  bool wrong = false;
  if (t < n) {
    x = a[t];
    y = b[t];
    wrong = x < 0 || x >= st.seqs || y < 0 || (FORK && y >= st.seqs);
    if (!wrong) {
      len = st.lens[x];
      wrong = mark(seen, FORK ? y : x) || len < 0 || len > cap ||
              (FORK ? st.lens[y] != 0 : y > len);
    }
  }
  if (FORK) {                                              // no parent is a child
    __syncthreads();
    if (t < n && !wrong) wrong = seen[x >> 5] >> (x & 31) & 1;
  }
  if (wrong) bad = 1;
  __syncthreads();
  const bool ok = !bad;
  if (t == 0) status[0] = ok ? 0 : 2;
  if (t < n) {
    Span s{FORK ? y : x, x, 0, 0};
    if (ok) {
      if (!FORK) s.first = pages_of(y, st.page_size);
      s.held = pages_of(len, st.page_size);
      st.lens[s.row] = FORK ? (int)len : y;
    }
    if (ALL) {
      spans[t] = s;
      if (s.held > s.first) atomicMax(&widest, s.held - s.first);
    } else {
      spans_out[t] = s;
    }
  }
  if (ALL) {
    __syncthreads();
    for (int e = t; e < n * widest; e += kThreads) {       // at most kMoveHere
      const Span& s = spans[e / widest];
      move_page<FORK>(st, s, s.first + e % widest);
    }
  }
}

template <bool FORK>
__global__ void __launch_bounds__(256) pages_move_wide_kernel(mtl_page_state st,
                                                              const Span* __restrict__ spans) {
  const Span s = spans[blockIdx.y];
  move_page<FORK>(st, s, s.first + blockIdx.x * 256 + threadIdx.x);
}

__device__ __forceinline__ int moved(int p, int live, int64_t pages, const int32_t* goes) {
  return p >= live && p < pages ? goes[p] : p;
}

// Plans the moves: one pass over the counts for L, one that ranks movers and free pages below L by
// prefix sums in strips of kStrip; with ALL it rewrites the table too.  Bound by the trips to the
// memory one workgroup makes: 7 us for 900 pages, 48 for 70 000, 191 for 300 000.  That is a small
// part of what the copies take where a large part of such a pool moves, and the most of the call
// where little does.
template <bool ALL>
__global__ void __launch_bounds__(kThreads) pages_compact_plan_kernel(
    const int32_t* refs, int64_t pages, int32_t* refs_out, int32_t* __restrict__ live_out,
    int32_t* __restrict__ moves_out, int32_t* __restrict__ src, int32_t* __restrict__ dst,
    int32_t* __restrict__ goes, const int32_t* table, int64_t ld, int64_t width, int64_t seqs,
    int32_t* table_out, int64_t ld_out) {
  __shared__ int waves[kWaves];
  const int t = threadIdx.x;
  const int all = (int)(seqs * width), w = (int)width;   // with ALL at most kTableHere
  int page[kTableHere / kThreads];           // the table, on its way
#pragma unroll
  for (int k = 0; k < kTableHere / kThreads; ++k) {
    const int e = t + k * kThreads;
    page[k] = ALL && e < all ? table[e / w * ld + e % w] : 0;
  }
  int held = 0, live;
  uint32_t strip0 = 0;
  for (int64_t p = 16 * t; p < pages; p += kStrip) {
    const uint32_t in = pages - p < 16 ? (1u << (pages - p)) - 1 : 0xffffu;
    const uint32_t used = held_mask(refs, p, pages) & in;
    if (p < kStrip) strip0 = used;
    held += __popc(used);
  }
  block_scan(held, waves, live);
  int movers = 0, holes = 0;
  for (int64_t p0 = 0; p0 < pages; p0 += kStrip) {
    const int64_t p = p0 + 16 * t;
    uint32_t mover = 0, hole = 0, rest = 0;
    if (p < pages) {
      const uint32_t in = pages - p < 16 ? (1u << (pages - p)) - 1 : 0xffffu;
      const uint32_t used = p0 == 0 ? strip0 : held_mask(refs, p, pages) & in;
      const uint32_t low = live <= p ? 0u : live - p < 16 ? (1u << (live - p)) - 1 : 0xffffu;
      mover = used & ~low;
      hole = ~used & low & in;
      rest = ~used & ~low & in;
    }
    int sum;                                   // at most 2^14 of each in a strip
    const int ranks = block_scan(__popc(mover) | __popc(hole) << 16, waves, sum);
    int k = movers + (ranks & 0xffff);
    for (; mover; mover &= mover - 1) src[k++] = (int)p + __ffs(mover) - 1;
    k = holes + (ranks >> 16);
    for (; hole; hole &= hole - 1) dst[k++] = (int)p + __ffs(hole) - 1;
    for (; rest; rest &= rest - 1) {
      const int q = (int)p + __ffs(rest) - 1;
      goes[q] = q;
    }
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
  if (!ALL) return;
#pragma unroll
  for (int k = 0; k < kTableHere / kThreads; ++k) page[k] = moved(page[k], live, pages, goes);
#pragma unroll
  for (int k = 0; k < kTableHere / kThreads; ++k) {
    const int e = t + k * kThreads;
    if (e < all) table_out[e / w * ld_out + e % w] = page[k];
  }
}

__global__ void __launch_bounds__(256) pages_compact_table_kernel(
    const int32_t* table, int64_t ld, int64_t width, int32_t* table_out, int64_t ld_out,
    int64_t pages, const int32_t* __restrict__ live, const int32_t* __restrict__ goes) {
  const int64_t j = blockIdx.x * (int64_t)256 + threadIdx.x, s = blockIdx.y;
  if (j >= width) return;
  table_out[s * ld_out + j] = moved(table[s * ld + j], live[0], pages, goes);
}

// A workgroup takes pieces of kPiece bytes of (pair, layer, K or V), as many pairs as there are,
// all of a pair's before the next one's.  Bound by memory.  Loads may stay in the caches (forks
// of one sequence copy the same page), stores leave no trace there: 16 pages four times each in
// 36 layers (302 MB) 32 us, with loads that leave none either 49, layer by layer 40.  A pool's
// 2.1 GB take 427 us that way, 411 with both.
constexpr int kPiece = 16384;
constexpr int kCopyGroups = 4096;

__global__ void __launch_bounds__(256) pages_copy_kernel(
    char* k, char* v, int64_t layers, int64_t k_layer, int64_t v_layer, int64_t k_page,
    int64_t v_page, int64_t page_bytes, int64_t pages, const int32_t* __restrict__ src,
    const int32_t* __restrict__ dst, int64_t n, const int32_t* __restrict__ count) {
  const int64_t pairs = count && count[0] < n ? count[0] : n;
  const int64_t pieces = (page_bytes + kPiece - 1) / kPiece;
  const int64_t all = pairs * layers * 2 * pieces;
  for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const int64_t piece = i % pieces, j = i / pieces % (2 * layers), l = j / 2,
                  pair = i / pieces / (2 * layers);
    const int64_t a = src[pair], b = dst[pair];
    if (a < 0 || a >= pages || b < 0 || b >= pages) continue;
    const char* from = j & 1 ? v + l * v_layer + a * v_page : k + l * k_layer + a * k_page;
    char* to = j & 1 ? v + l * v_layer + b * v_page : k + l * k_layer + b * k_page;
    const int64_t o = piece * kPiece + 16 * threadIdx.x;
    u32x4 x[4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (o + 4096 * m < page_bytes)
        x[m] = *reinterpret_cast<const u32x4*>(from + o + 4096 * m);
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (o + 4096 * m < page_bytes)
        __builtin_nontemporal_store(x[m], reinterpret_cast<u32x4*>(to + o + 4096 * m));
  }
}

// Arguments every bookkeeping entry shares.
static int check_state(const mtl_page_state* st, int64_t n, const void* status, const void* ws,
                       int64_t ws_bytes, bool lens = true) {
  if (!st || n < 0 || st->seqs < 0 || st->width < 0 || st->ld < st->width || st->pages < 0 ||
      st->pages > INT32_MAX - kStrip || !status)
    return MTL_ERR_INVALID_ARG;
  if (n > kMaxCall || st->seqs > kMaxSeqs || st->width > MTL_PAGES_MAX_WIDTH)
    return MTL_ERR_SHAPE;
  if (!page_size_ok(st->page_size)) return MTL_ERR_SHAPE;
  if ((st->seqs > 0 && ((lens && !st->lens) || (st->width > 0 && !st->table))) ||
      (st->pages > 0 && !st->refs))
    return MTL_ERR_INVALID_ARG;
  if (!ws || ws_bytes < mtl_pages_workspace_bytes(n, st->pages)) return MTL_ERR_WORKSPACE;
  return aligned16(ws) ? MTL_OK : MTL_ERR_ALIGN;
}

template <bool FORK>
static int move_call(const mtl_page_state* st, const int32_t* a, const int32_t* b, int64_t n,
                     int32_t* status, void* workspace, int64_t ws_bytes, hipStream_t stream) {
  const int e = check_state(st, n, status, workspace, ws_bytes);
  if (e != MTL_OK) return e;
  if (n > 0 && (!a || !b)) return MTL_ERR_INVALID_ARG;
  Span* spans = static_cast<Span*>(workspace);
  if (n * st->width <= kMoveHere) {
    pages_move_kernel<FORK, true><<<1, kThreads, 0, stream>>>(*st, a, b, (int)n, status, spans);
  } else {
    pages_move_kernel<FORK, false><<<1, kThreads, 0, stream>>>(*st, a, b, (int)n, status, spans);
    const dim3 grid((unsigned)((st->width + 255) / 256), (unsigned)n);
    pages_move_wide_kernel<FORK><<<grid, 256, 0, stream>>>(*st, spans);
  }
  return launch_status();
}

}  // namespace mtl

using namespace mtl;

extern "C" int64_t mtl_pages_workspace_bytes(int64_t n, int64_t pages) {
  if (n < 0 || pages < 0) return 0;
  return 16 * (n + 1) + 4 * pages;
}

extern "C" int mtl_pages_extend(const mtl_page_state* st, const int32_t* seqs,
                                const int32_t* counts, int64_t n, int32_t* copy_src,
                                int32_t* copy_dst, int32_t* copies, int32_t* status,
                                void* workspace, int64_t ws_bytes, void* stream) {
  const int e = check_state(st, n, status, workspace, ws_bytes);
  if (e != MTL_OK) return e;
  if (!copies || (n > 0 && (!seqs || !counts || !copy_src || !copy_dst)))
    return MTL_ERR_INVALID_ARG;
  pages_extend_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(
      *st, seqs, counts, (int)n, copy_src, copy_dst, copies, status,
      static_cast<int32_t*>(workspace));
  return launch_status();
}

extern "C" int mtl_pages_fork(const mtl_page_state* st, const int32_t* parents,
                              const int32_t* children, int64_t n, int32_t* status,
                              void* workspace, int64_t ws_bytes, void* stream) {
  return move_call<true>(st, parents, children, n, status, workspace, ws_bytes,
                         (hipStream_t)stream);
}

extern "C" int mtl_pages_truncate(const mtl_page_state* st, const int32_t* seqs,
                                  const int32_t* new_lens, int64_t n, int32_t* status,
                                  void* workspace, int64_t ws_bytes, void* stream) {
  return move_call<false>(st, seqs, new_lens, n, status, workspace, ws_bytes, (hipStream_t)stream);
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
  hipStream_t hs = (hipStream_t)stream;
  if (st->seqs * st->width <= kTableHere) {
    pages_compact_plan_kernel<true><<<1, kThreads, 0, hs>>>(
        st->refs, st->pages, refs_out, live, moves, move_src, move_dst, goes, st->table, st->ld,
        st->width, st->seqs, table_out, ld_out);
  } else {
    pages_compact_plan_kernel<false><<<1, kThreads, 0, hs>>>(
        st->refs, st->pages, refs_out, live, moves, move_src, move_dst, goes, st->table, st->ld,
        st->width, st->seqs, table_out, ld_out);
    const dim3 grid((unsigned)((st->width + 255) / 256), (unsigned)st->seqs);
    pages_compact_table_kernel<<<grid, 256, 0, hs>>>(st->table, st->ld, st->width, table_out,
                                                     ld_out, st->pages, live, goes);
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
  const int64_t most = n * layers * 2 * ((page_bytes + kPiece - 1) / kPiece);
  pages_copy_kernel<<<(unsigned)(most < kCopyGroups ? most : kCopyGroups), 256, 0,
                      (hipStream_t)stream>>>(
      static_cast<char*>(k), static_cast<char*>(v), layers, k_layer, v_layer, k_page, v_page,
      page_bytes, pages, src, dst, n, count);
  return launch_status();
}
