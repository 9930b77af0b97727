/*
 * mtl_sample.h -- C ABI of drawing tokens from logits (MI355X / gfx950): temperature, top-k, top-p
 * and min-p, from given random numbers.  Same conventions as mtl_gptq.h: 0 = MTL_OK, negative =
 * MTL_ERR_*, raw device pointers, a hipStream_t, no allocation or host synchronisation,
 * capturable into a hipGraph.  The structure below is host memory, read during the call.
 *
 * The reference filters and draws with torch operations, one sentence at a time
 * (moss_tts_lite/sampling.py:9-126).
 */
#ifndef MTL_SAMPLE_H
#define MTL_SAMPLE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the logits: MTL_T_BF16 and MTL_T_F16 (mtl_paged.h), and float32. */
#define MTL_T_F32 3

/* How the rows draw: where a pointer (device, [rows]) is given it holds each row's setting,
 * otherwise the number beside it is every row's. */
typedef struct mtl_sample_settings {
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int32_t top_k_all;
  float top_p_all, min_p_all;
} mtl_sample_settings;

/*
 * Row r of logits x: its tokens stand in an order, the larger logit first, of equal ones the lower
 * index.  With w_i = exp((x_i - max x) / temperature), in 64 bits:
 *   1. the first top_k of the order stay (top_k <= 0: all),
 *   2. of these, those stay before which weights of at most top_p times these' sum lie (top_p >= 1:
 *      all),
 *   3. of these, those of w_i >= min_p stay.
 * The first of the order always stays.  token is the lowest index i that stays and before and at
 * which the weights of those that stay, summed by index, exceed u[r] times their whole sum; logprob
 * the logarithm of w_i over that sum.  A temperature that is not above 0 gives the first of the
 * order, logprob 0.  A NaN counts as -infinity, which has weight 0; beside +infinity everything
 * finite has weight 0.  A row of -infinity only: -1, logprob -infinity.
 * Sums are whole numbers of 64 bits, so that their order changes nothing: a weight counts as a
 * multiple of 2^-n, with the largest n up to 51 for which vocab 2^n is at most 2^63 (51 up to 4096
 * tokens, 45 up to 2^18, 43 at 2^20).  So borders are right to half of 2^-n a token, and a token of
 * less weight than that is not drawn, unless it is the first of the order.
 *   logits   [rows, vocab] of type, ld elements apart (0: every row draws from the same ones)
 *   u        fp32 [rows] in [0, 1) (others count as the nearest of these, NaN as 0)
 *   token    int64 [rows];  logprob  NULL, or fp32 [rows]
 *   workspace  mtl_sample_workspace_bytes(...) bytes, 16-byte aligned, any content, one launch at a
 *              time.  Past 8192 tokens a row takes 2 bytes or so for each token where top_p may cut
 *              it without top_k (a pointer may hold any setting), an eighth of one otherwise
 * vocab at most 2^20, rows at most 65535.
 */
int64_t mtl_sample_workspace_bytes(int64_t rows, int64_t vocab, int32_t type,
                                   const mtl_sample_settings* settings);
int mtl_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t type,
               const float* u, const mtl_sample_settings* settings, int64_t* token,
               float* logprob, void* workspace, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MTL_SAMPLE_H */
