/*
 * mtl_paged.h -- C ABI of the paged key-value cache (MI355X / gfx950): several sequences in
 * one pool of pages, the attention of one new token a sequence over them, the write of new
 * tokens, and the bookkeeping of pages (reference counts, forks, freeing, compaction).
 * Same conventions as mtl_gptq.h: 0 = MTL_OK, negative = MTL_ERR_*, raw device pointers, a
 * hipStream_t, no allocation or host synchronisation, capturable into a hipGraph.  The
 * structures below are host memory, read during the call.
 *
 * The reference holds one dense cache of one sequence (moss_tts_lite/model.py:110-112);
 * these entries have no counterpart there.
 *
 * A page holds page_size consecutive tokens of one sequence, all kv heads, one layer.
 * Position p of sequence s lies in page table[s][p / page_size], row p % page_size.  A table
 * entry outside [0, pages) is a hole: its positions take no part in the attention and are
 * not written.
 */
#ifndef MTL_PAGED_H
#define MTL_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types.  E4M3 (float8, no infinities) is a page type only: a stored element times
 * its kv head's scale is the value. */
#define MTL_T_BF16 0
#define MTL_T_F16 1
#define MTL_T_E4M3 2

/* One layer's pages.  Strides in elements; the head_dim elements of a row are adjacent, and
 * k_token, v_token >= head_dim; bases and strides are multiples of 16 bytes. */
typedef struct mtl_page_pool {
  void* k;
  void* v;
  int64_t pages;                      /* 1 .. 2^31 - 1 */
  int64_t k_page, k_head, k_token;
  int64_t v_page, v_head, v_token;
  int32_t kv_heads;
  int32_t page_size;                  /* 16, 32, 64, 128 or 256 */
  int32_t head_dim;                   /* 64 or 128 */
  int32_t type;                       /* MTL_T_* */
  const float* k_scale;               /* device [kv_heads]; NULL: 1.  E4M3 only */
  const float* v_scale;
} mtl_page_pool;

/* Which pages a batch of sequences has: row i of table (int32, ld entries apart) holds the
 * pages of sequence i, width of them at most. */
typedef struct mtl_page_table {
  const int32_t* table;
  int64_t ld;
  int64_t width;
  int64_t seqs;
} mtl_page_table;

/*
 * Attention of one query token of each sequence over its pages (the SDPA call of a decode
 * step, moss_tts_lite/fast.py:149-162, over pages): for sequence b and query head h, with
 * kv head h / (n_heads / kv_heads),
 *   s_j = scale * k_scale * (q . k_j),  j in [0, lens[b]);  out = v_scale * sum softmax(s)_j v_j
 * fp32 softmax and sums; a weight enters the product with v to 2^-16 of itself (bf16) or to
 * 2^-20 of itself and 2^-39 of the largest (f16).  Lengths past width * page_size (at most 2^30)
 * count as that, negative ones as 0.
 *   q    [seqs, n_heads, head_dim] of q_type (bf16 or f16), rows ldq and heads ldh elements
 *        apart (multiples of 8, base 16-byte aligned)
 *   out  [seqs, n_heads, head_dim] of q_type, contiguous, 16-byte aligned; a sequence without
 *        positions: 0
 *   lse  NULL, or fp32 [seqs, n_heads]: the natural logarithm of sum_j exp(s_j) (-inf for a
 *        sequence without positions)
 *   workspace  mtl_paged_attention_workspace_bytes(...) bytes, 16-byte aligned, any content,
 *        one launch at a time
 * The pages have q_type's type or E4M3.  n_heads % kv_heads == 0, n_heads and seqs at most
 * 65535, and with width * page_size <= 512 seqs * kv heads * (query heads of one / 16, rounded
 * up) at most 2^23 - 1.  The same call gives the same bits; the order of a sequence's sums goes by
 * all lengths.  Nothing in a hole or past a length has an effect, NaN included; K and V of the
 * positions attended to are finite (an infinity or NaN there gives NaN where it enters).
 */
int64_t mtl_paged_attention_workspace_bytes(int64_t seqs, int32_t n_heads, int32_t kv_heads,
                                            int32_t head_dim, int64_t width, int32_t page_size);
int mtl_paged_attention(const void* q, int64_t ldq, int64_t ldh, const mtl_page_pool* pool,
                        const mtl_page_table* table, const int32_t* lens, int32_t n_heads,
                        int32_t q_type, float scale, void* out, float* lse, void* workspace,
                        int64_t ws_bytes, void* stream);

/*
 * q/k RMSNorm, RoPE and the page write of new tokens, each row at its own position of its own
 * sequence (mtl_qk_norm_rope_kv_rows over pages; moss_tts_lite/fast.py:226-237).
 *   qkv        [rows, ldq] of type (bf16 or f16), each row q | k | v
 *              ((n_heads + 2 kv_heads) * head_dim); ldq a multiple of 8, 16-byte aligned
 *   positions  int64 [rows] (device).  A negative position (or one past the RoPE tables) is
 *              padding: its q row is 0 and no page is written
 *   row_seq    int32 [rows] (device), the sequence of each row; NULL: row r is sequence r
 *   q_norm, k_norm  [head_dim] of type; both NULL: no norm
 *   cos_tab, sin_tab  [rope_rows, head_dim], fp32 (rope_f32 = 1) or of type; both NULL: no RoPE
 *   q_out      [rows, n_heads, head_dim] of type, contiguous
 * q_out, norms and tables are 16-byte aligned.
 * The arithmetic is fp32 throughout with one rounding where q, k and v are stored (the dense
 * entries round after every step as the reference does).  E4M3 pages store x / scale,
 * limited to +-448, rounded to nearest even.  Rows whose page is a hole, whose position lies
 * past the table or whose sequence is outside it write no page.  No two rows may name the
 * same position of the same sequence, and no two places of k and v are the same memory.
 */
int mtl_paged_write(const void* qkv, int64_t ldq, int64_t rows, const mtl_page_pool* pool,
                    const mtl_page_table* table, const int64_t* positions, const int32_t* row_seq,
                    const void* q_norm, const void* k_norm, const void* cos_tab,
                    const void* sin_tab, int32_t rope_f32, int64_t rope_rows, float eps,
                    int32_t n_heads, int32_t type, void* q_out, void* stream);

/*
 * Bookkeeping, all on the device.  A page is free when refs[page] == 0; a sequence of length
 * len holds ceil(len / page_size) pages, the first entries of its table row, the others -1.
 * Each call does all of its work or, on a bad argument, none, and writes status[0]:
 *   0  done
 *   1  not enough free pages (extend)
 *   2  a sequence outside [0, seqs), the same one twice, or a length out of range
 * n <= MTL_PAGES_MAX_CALL sequences a call, seqs <= MTL_PAGES_MAX_SEQS, width <=
 * MTL_PAGES_MAX_WIDTH, page_size as in mtl_page_pool.  workspace: mtl_pages_workspace_bytes(n,
 * pages) bytes (n = 0 for compaction), 16-byte aligned, any content, one launch at a time.
 */
#define MTL_PAGES_MAX_CALL 1024
#define MTL_PAGES_MAX_SEQS 32768
#define MTL_PAGES_MAX_WIDTH (1 << 20)

typedef struct mtl_page_state {
  int32_t* table;                     /* [seqs][ld], width entries used */
  int64_t ld, width, seqs;
  int32_t* lens;                      /* [seqs]; not read by mtl_pages_compact */
  int32_t* refs;                      /* [pages] */
  int64_t pages;
  int32_t page_size;
} mtl_page_state;

int64_t mtl_pages_workspace_bytes(int64_t n, int64_t pages);

/*
 * Room for counts[i] more tokens of sequence seqs[i], in call order: a partly filled last
 * page that others hold too is replaced by a copy, then each further page is taken; every
 * page taken is the lowest free one.  Adds counts to lens.  copies[0] pairs copy_src[i],
 * copy_dst[i] (up to n) say which pages' contents the caller has to copy (mtl_pages_copy).
 */
int mtl_pages_extend(const mtl_page_state* st, const int32_t* seqs, const int32_t* counts,
                     int64_t n, int32_t* copy_src, int32_t* copy_dst, int32_t* copies,
                     int32_t* status, void* workspace, int64_t ws_bytes, void* stream);

/*
 * Sequence children[i] becomes parents[i]: the same pages (their counts rise) and length.
 * Children are distinct, empty, and no parents; a parent may be forked several times.
 */
int mtl_pages_fork(const mtl_page_state* st, const int32_t* parents, const int32_t* children,
                   int64_t n, int32_t* status, void* workspace, int64_t ws_bytes, void* stream);

/*
 * Sequence seqs[i] keeps its first new_lens[i] tokens (0: it is freed); pages past them are
 * given back, and are free once no sequence holds them.
 */
int mtl_pages_truncate(const mtl_page_state* st, const int32_t* seqs, const int32_t* new_lens,
                       int64_t n, int32_t* status, void* workspace, int64_t ws_bytes,
                       void* stream);

/*
 * Compaction: with L the number of pages held, the k-th held page at or past L moves to the
 * k-th free page below L, both ascending.  Writes table_out (rows ld_out apart; may be
 * st->table) and refs_out (may be st->refs), live[0] = L, moves[0] = the number of moves and
 * move_src / move_dst (pages / 2 entries each), whose contents the caller has to copy.
 */
int mtl_pages_compact(const mtl_page_state* st, int32_t* table_out, int64_t ld_out,
                      int32_t* refs_out, int32_t* live, int32_t* moves, int32_t* move_src,
                      int32_t* move_dst, void* workspace, int64_t ws_bytes, void* stream);

/*
 * Copies whole pages in every layer, K and V: page dst[i] = page src[i], i < n and, with
 * count (device, may be NULL), i < count[0].  Entries outside [0, pages) are skipped.  No
 * page is dst twice, or both src and dst.  Page p of layer l lies page_bytes long at
 * base + l * layer stride + p * page stride (strides in bytes, everything in multiples of 16).
 */
int mtl_pages_copy(void* k, void* v, int64_t layers, int64_t k_layer, int64_t v_layer,
                   int64_t k_page, int64_t v_page, int64_t page_bytes, int64_t pages,
                   const int32_t* src, const int32_t* dst, int64_t n, const int32_t* count,
                   void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MTL_PAGED_H */
