/*
 * czg_ops.h -- operators on device buffers, beside the whole-model engine of czg.h
 * and exported by the same library: the int8 product with a scale for each token
 * and each channel, attention over a key/value cache held in 4 bits, and eviction
 * from that cache by accumulated attention weight.  (No counterpart in the
 * reference: its products have one multiplier and shift for a whole matrix,
 * rust/src/model.rs:280-300, and its cache holds 8 bits and ends with the context,
 * rust/src/attention.rs:112-160.)
 *
 * Conventions: as czg_encode_intervals_static.  Every buffer is device memory of the
 * current device and belongs to the caller; no entry point allocates, copies to the
 * host or waits.  Work is queued on `stream` (a cudaStream_t of the current device;
 * NULL is the legacy default stream) and may be captured into a graph.  Arguments that the
 * host can see are checked before anything is queued (CZG_E_ARG, CZG_E_LIMIT,
 * CZG_E_UNSUPPORTED; czg_ops_last_error holds the reason); what only the device can
 * see (slots and lengths) is checked there: what is out of range is neither read nor
 * written, and a bit of czg_kv4.status says so.  n = 0 rows or sequences: CZG_OK, nothing queued.
 *
 * A row of a product, and a sequence of a cache call, depends on its own operands alone:
 * not on how many others are in the call, on its place among them, its slot, or the
 * grid, to the bit.  No result comes out of an atomic whose order could change it.  A
 * sequence's operands are all its rows and entries of the call: attention of the same row
 * over the same entries may differ in its last bits between calls of one row (t = 1) and of
 * several, and between calls that hold more or fewer entries behind those it sees.
 */
#ifndef CZG_OPS_H
#define CZG_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "czg.h"

#ifdef __cplusplus
extern "C" {
#endif

enum czg_dtype { CZG_F32 = 0, CZG_BF16 = 1, CZG_F16 = 2 };

/* Why the last call of this thread that returned another status than CZG_OK did so. */
const char *czg_ops_last_error(void);

/* Waits for the current device.  CZG_E_TIMEOUT if a kernel of an operator gave up a
 * bounded wait on it since the last such answer (its results are incomplete). */
int czg_ops_check(void);

/* ---- int8 product ------------------------------------------------------------- */

/* Rows of x ([m][k] of `dtype`, ld_x elements apart) as int8 codes and one scale each:
 *   scale = max |x| / 127,  code = round-half-even(127 x / max |x|)
 * (the code exact for 16-bit x; for fp32 x its product and quotient round to fp32)
 * (a row of zeros: scale 0, codes 0; a row with a NaN or an infinity: scale NaN,
 * codes 0).  codes: rows ld_codes bytes apart, 16-byte aligned, ld_codes a multiple
 * of 16; the bytes from k to the next multiple of 16 are set to 0. */
int czg_quantize_rows(const void *x, int dtype, int64_t ld_x, int64_t m, int64_t k, int8_t *codes,
                      int64_t ld_codes, float *scales, void *stream);

/* out[i][j] = (sum over k of x[i][k] w[j][k]) * x_scale[i] * w_scale[j] + bias[j]:
 * the sum exact in int32, the rest in fp32 in this order, one rounding to out_dtype.
 * x: m rows, w: n rows of k codes, ld_x and ld_w bytes apart (16-byte aligned, a
 * multiple of 16; bytes from k on are ignored).  bias may be NULL.  out: rows ld_out
 * elements apart, not over x or w.  k <= CZG_LINEAR_MAX_K (the int32 sum), m, n <= 2^31 - 512. */
#define CZG_LINEAR_MAX_K 131071
int czg_linear_i8(const int8_t *x, int64_t ld_x, const float *x_scale, const int8_t *w, int64_t ld_w,
                  const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k, void *out,
                  int out_dtype, int64_t ld_out, void *stream);

/* czg_quantize_rows and then czg_linear_i8, with the same bits.  ws: 16-byte aligned,
 * czg_linear_i8_workspace(m, k) bytes (0, and NULL will do, for a few short rows, which
 * one kernel takes), free again when the queued work is done.  With
 * czg_linear_i8_dynamic_workspace(m, n, k) bytes, which are never fewer, a few short rows on
 * so many channels that two kernels are faster take two. */
uint64_t czg_linear_i8_workspace(int64_t m, int64_t k);
uint64_t czg_linear_i8_dynamic_workspace(int64_t m, int64_t n, int64_t k);
int czg_linear_i8_dynamic(const void *x, int dtype, int64_t ld_x, const int8_t *w, int64_t ld_w,
                          const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k, void *out,
                          int out_dtype, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream);

/* ---- key/value cache in 4 bits -------------------------------------------------- */

/* n_slots slots of `capacity` entries for each of n_heads key heads.  A head's key of
 * an entry, and its value, are head_dim (64 or 128) codes of 4 bits, byte i holding
 * dimension 2i in its low half, and two bf16 numbers:
 *   lo = min x rounded down, step = (max x - lo) / 15 rounded up,
 *   code = round-half-even((x - lo) / step)   (step 0: code 0), held value lo + step * code
 * so that no value is off by more than step / 2, but for the difference and the quotient,
 * which round to fp32 before the code does (30 * 2^-24 of a step next to a half).  A row with a
 * NaN or an infinity, or whose range overflows fp32, holds NaN in every place.
 *   k, v     [n_slots][n_heads][capacity][head_dim / 2] bytes, 16-byte aligned
 *   scales   [n_slots][n_heads][capacity][4] bf16: k step, k lo, v step, v lo; 8-byte aligned
 *   weights  NULL, or [n_slots][n_heads][capacity] sums of attention weights
 *   status   one int32 that the caller zeroes: CZG_KV4_* bits of what calls left out */
typedef struct {
    uint8_t *k, *v;
    void *scales;
    float *weights;
    int32_t *status;
    int32_t n_slots, n_heads, capacity, head_dim;
} czg_kv4;

#define CZG_KV4_BAD_SLOT 1    /* a slot >= n_slots: its sequence is treated as padding         */
#define CZG_KV4_BAD_LENGTH 2  /* a length < 0, > capacity or > max_len: cut to the range; append
                               * leaves out rows that lie outside the slot                    */
#define CZG_KV4_TWICE 4       /* a slot named twice in a call that writes slots: what that slot
                               * then holds is unspecified                                    */

/* Sequences of a call: slots[b] names the slot of sequence b, a negative one a padded
 * place of the batch (nothing is read or written for it, its outputs are 0).
 * lengths[b] counts its entries, the t rows of this call among them.  At most 65,535
 * sequences a call (evict: 65,534). */

/* Row i of sequence b (k, v: [b][t][n_heads][head_dim] of `dtype`, strides in elements,
 * the last one 1) becomes entry lengths[b] - t + i; rows before entry 0 are padding and
 * left out.  The weights of the entries written are set to 0. */
int czg_kv4_append(const czg_kv4 *cache, const void *k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void *v,
                   int64_t v_sb, int64_t v_st, int64_t v_sh, int dtype, const int32_t *slots,
                   const int32_t *lengths, int32_t b, int32_t t, void *stream);

/* Entries starts[b] .. starts[b] + count - 1 as values, k_out and v_out
 * [b][count][n_heads][head_dim] of `dtype`, 16-byte aligned; 0 for what lies outside
 * the slot (and CZG_KV4_BAD_LENGTH).  Either output may be NULL. */
int czg_kv4_read(const czg_kv4 *cache, const int32_t *slots, const int32_t *starts, int32_t b, int32_t count,
                 void *k_out, void *v_out, int dtype, void *stream);

/* Attention of t rows a sequence over its entries: row i sees the first
 * lengths[b] - (t - 1 - i) of them (0 where that leaves none: the row's output is 0).
 * q, out: [b][t][hq][head_dim] of `dtype` (bf16 or fp16), strides in elements, the last one 1;
 * hq a multiple of n_heads, query heads of a key head adjacent.  out may be q itself, and
 * lies over no other part of it.
 *   out = sum_j p_j v_j, p = softmax_j(scale q.k_j)
 * Scores, p and the sums are fp32; p below 2^-126 of a row's largest counts as 0.  p_j step_j is
 * rounded to 11 bits (fp16: 22), and to 2^-25 of the largest p times the largest step of those
 * that are alike within 2^6, or of the row's largest p_j step_j, so what other entries hold,
 * seen or not, costs a row nothing.  Values may be as large as bf16 goes (beside one of 2^87
 * and more, in the same 512 entries or unit, those below 2^-90 lose bits).
 * cache->weights != NULL: every entry's weight grows by its p, summed over the rows
 * and query heads of its key head.  max_len: no length of the call is above it.
 * The rows of each key head make blocks of 16 (of 8 where there are no more); all key heads'
 * blocks of a sequence, about t * hq / 16, are at most 65,535 (CZG_E_LIMIT).
 * ws: 16-byte aligned, czg_kv4_attend_workspace bytes (may be 0): for calls of more than 512
 * entries or, with weights, of several blocks of rows, a partial result of each row and unit (at
 * most 128 units a sequence), and with weights 4 bytes a row, query head and entry of max_len. */
uint64_t czg_kv4_attend_workspace(const czg_kv4 *cache, int32_t b, int32_t t, int32_t hq, int32_t max_len);
int czg_kv4_attend(const czg_kv4 *cache, const void *q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype,
                   const int32_t *slots, const int32_t *lengths, int32_t b, int32_t t, int32_t hq,
                   int32_t max_len, float scale, void *out, int64_t o_sb, int64_t o_st, int64_t o_sh, void *ws,
                   uint64_t ws_bytes, void *stream);

/* Sequences longer than `budget` are cut to it: of each head the last `recent` entries
 * stay and, of those before them, the budget - recent with the largest weights (a NaN
 * counts as the largest; of equal ones the first), in their order, moved with their
 * weights to the front of the slot.  What lies behind entry budget - 1 is left as it
 * was.  kept (may be NULL): [b][n_heads][budget], the entries' places before the call,
 * -1 behind a shorter sequence's end; new_lengths (may be NULL; not the same array as
 * lengths): min(length, budget).  1 <= budget, 0 <= recent <= budget; max_len: no
 * length of the call is above it, at most CZG_KV4_EVICT_MAX. */
#define CZG_KV4_EVICT_MAX 1048576
int czg_kv4_evict(const czg_kv4 *cache, const int32_t *slots, const int32_t *lengths, int32_t b, int32_t max_len,
                  int32_t budget, int32_t recent, int32_t *kept, int32_t *new_lengths, void *stream);

#ifdef __cplusplus
}
#endif
#endif
