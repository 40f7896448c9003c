/*
 * paged_ops.h — a paged KV cache on the GPU: the pages of a step, the write into them, and
 * attention of new tokens over them.  None of these operators has a counterpart in the
 * reference, whose cache is one (B, max_seq, H_kv, d) tensor per layer.
 *
 * The cache of a layer is num_pages pages of page_size positions: K and V pages
 * (num_pages, page_size, H_kv, d).  Position p of sequence b is on page
 * block_table[b * max_pages + p / page_size], at row p % page_size; its slot is
 * page * page_size + p % page_size.  A contiguous cache of MHA_Decode whose max_seq is a
 * multiple of page_size is such a cache as it is: page b * (max_seq / page_size) + j.
 *
 * A step of a batch is one kv_page_map (pages and slots for the new tokens) and then, per
 * layer, one kv_page_store (new K and V rows to their slots, Q and K rotated) and one
 * mha_paged_attn (every new token over its sequence).  The tokens of a step are the rows of
 * one (T, ., d) tensor, sequence after sequence: rows q_start[b] .. q_start[b + 1] - 1 are
 * sequence b's.  Lengths, offsets, tables and slots stay on the device, so a captured step
 * replays at every length; what they hold cannot be checked on the host, and a value out
 * of range is never followed: a page outside [0, num_pages) holds no position (nothing is
 * stored there, nothing of it is attended), a slot outside [0, num_pages * page_size)
 * stores nothing, lengths and offsets are clamped to the table and to the rows.
 *
 * Operator signature and return codes as in mha_ops.h: 0; -1 invalid arguments or workspace
 * failure; a hipError_t value if a launch failed.  All integers on the device are int32.
 */
#ifndef CF_PAGED_OPS_H_
#define CF_PAGED_OPS_H_

#include <stdint.h>
#include "operator.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the pages of a step ---- */

typedef struct {
    int64_t batch_size;   /* B >= 1 */
    int64_t num_tokens;   /* T: entries of positions and slots, at least the step's tokens */
    int64_t page_size;    /* positions per page */
    int64_t num_pages;    /* pages of the cache; num_pages * page_size < 2^31 */
    int64_t max_pages;    /* entries of one row of the block table; max_pages * page_size < 2^31 */
    int64_t ring_size;    /* R: entries of the ring of free pages; num_pages hold every page */
} kv_page_map_params_t;

/* Gives each request the pages its new tokens need, and takes back those of ended ones.
 * inputs  [cache_lens (B): positions each sequence holds,
 *          new_lens (B): tokens it adds, or a negative number: the sequence has ended,
 *          counters (3): place of the ring's first free page, number of free pages, (unused)]
 * outputs [block_table (B, max_pages), updated in place: entries of new pages,
 *          ring (R), updated in place: pages of ended sequences behind the free ones,
 *          seq_lens (B): cache_lens + new_lens, 0 for an ended one,
 *          q_start (B + 1): first row of each sequence, and the number of rows,
 *          positions (T) and slots (T) of the rows; -1 in rows behind the last,
 *          counters (3): the same after the step, and how many sequences were not served]
 * seq_lens may be cache_lens, and the counters one array, so that a captured step advances.
 * Pages are taken from the ring's front in the order of the sequences.  A sequence is not
 * served when the pages asked for up to and with it outnumber the free ones (pages that
 * this call takes back count from the next call on), or when its length passes the table:
 * it then takes none, its table entries from the first new page on (to the end of the row
 * where the length passes it) and its slots are -1.  The others are not affected.  A later
 * call with the same cache_len tries again (new_lens 0 for those that were served).
 * seq_lens counts the tokens of a sequence that is not served too.  Where it is cache_lens,
 * the entry is therefore no longer what the sequence holds; the caller sets it back before
 * it tries again.  Until then the sequence is known by what it lacks (the entry of its last
 * position is negative, or its length passes the table): each call counts it as not served,
 * asks no page for it and leaves its length.  In either state it can be ended: an ended
 * sequence gives back those of its ceil(cache_len / page_size) entries that are pages, as
 * far as the ring has places.  No other sequence may hold them. */
int kv_page_map_i32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

/* ---- new rows into the pages ---- */

typedef struct {
    int64_t num_tokens;    /* T */
    int64_t num_heads;     /* H_q (read with a Q only) */
    int64_t num_kv_heads;  /* H_kv */
    int64_t head_dim;      /* d; with RoPE even and at most 256; H_kv d at most 2^29 */
    int64_t page_size;
    int64_t num_pages;
    float   rope_base;     /* > 0: Q and K are rotated; 0: rows are stored as they are */
    /* Elements from one row to the next; 0: rows follow each other.  The inputs can be the
     * parts of one (T, (H_q + 2 H_kv) d) projection. */
    int64_t q_stride;      /* Q */
    int64_t kv_stride;     /* K_new and V_new */
    int64_t q_out_stride;  /* the rotated Q */
    /* Elements from page to page, position to position and head to head of the cache; 0: the
     * (num_pages, page_size, H_kv, d) layout's. */
    int64_t page_stride, row_stride, head_stride;
} kv_page_store_params_t;

/* inputs  [K_new (T, H_kv, d), V_new (T, H_kv, d), slots (T), positions (T) (RoPE), Q (T, H_q, d) (RoPE)]
 * outputs [K_pages, V_pages, Q_rotated (T, H_q, d), may be Q (with one stride, else -1)]
 * With rope_base = 0 the last two inputs and the last output are not looked at (the arrays may
 * end before them); with RoPE either Q and Q_rotated are both given or both NULL.  Pairs
 * (2i, 2i + 1) turn by position * base^(-2i / d), the angle reduced in 64 bits and the
 * rotation in FP32 with one rounding to the type (rope_ops.h's operators round the angle to
 * FP32, as the reference does, which at position 100000 is off by up to 4e-3).  A row with
 * an invalid slot is not stored; a row with a negative position leaves its Q_rotated row
 * alone.  Each slot may be given once per call: of two rows for one slot, parts of either
 * may be stored. */
int kv_page_store_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
int kv_page_store_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

/* ---- attention of new tokens over the pages ---- */

typedef struct {
    int64_t batch_size;    /* B */
    int64_t num_tokens;    /* T: rows of Q and O */
    int64_t num_heads;     /* H_q */
    int64_t num_kv_heads;  /* H_kv (<= 0 means H_q) */
    int64_t head_dim;      /* d, at most 512 */
    float   scale;         /* usually 1/sqrt(d) */
    int64_t page_size;
    int64_t num_pages;
    int64_t max_pages;     /* entries of one row of the block table */
    /* Most rows and most positions a sequence has in this call, 0 = unknown (the table's
     * length).  They choose the kernels only: more than that is computed all the same.
     * Without max_new a batch of decode rows takes the chunks' kernel (16 rows of 32 heads of 128
     * over 8, up to 4096 positions: 46 us, without 57); without max_len, where the table is
     * long, short contexts take the long ones' (the same over 512: 10 us, without 13.5). */
    int64_t max_new, max_len;
    int64_t q_stride;      /* elements from row to row of Q; 0 = H_q d */
    int64_t page_stride, row_stride, head_stride;   /* of the cache, as in kv_page_store_params_t */
} mha_paged_params_t;

/* inputs  [Q (T, H_q, d), K_pages, V_pages, block_table (B, max_pages), seq_lens (B), q_start (B + 1)]
 * outputs [O (T, H_q, d)]
 * seq_lens counts the new tokens, whose K and V are in their pages already: row i of n of
 * sequence b is position p = seq_lens[b] - n + i and attends positions 0 .. p (query head h
 * reads KV head h / (H_q / H_kv)).  A row that sees no position (no page of it is valid, or
 * p < 0) gives 0.  Rows of O outside q_start[0] .. q_start[B] are left as they are; what
 * pages hold past seq_lens[b] is not looked at, and what a row does not see does not touch it,
 * infinite or NaN either.  Such V cost time: a tile that holds them reads its V a second time, and
 * rows that do not see them, though a later token of the same call does, are computed again by a
 * slow loop.  Tables may name a page twice and share pages; O must not overlap an input (-1 where
 * it is Q or a cache).  d = 64 and 128 with pages of a multiple of 16 positions, 16-byte
 * aligned pointers and strides, scale > 0 and at most 32768 sequences run on the matrix cores,
 * every other call on a plain kernel.
 * Scores, maxima and sums are FP32.  fp16 weights of the matrix cores' products with V: tiles
 * of up to 16 rows (n G of a sequence, or what is left of a chunk) hold each as the sum of two
 * fp16 numbers, tiles of more rows round it to fp16, by at most 2^-11 of itself; over thousands
 * of positions results are then off by 2.9e-4 of their size in the root mean square, by 2.1e-4 of
 * it from their own rounding alone.  Which tiles a chunk is cut into depends on the whole batch. */
int mha_paged_attn_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
int mha_paged_attn_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

/* ---- the same cache in 8 bits ----
 *
 * A number of the cache is an e4m3 byte (one sign, four exponent and three mantissa bits, bias 7, at
 * most 448; 0x7f and 0xff are NaN, infinity there is none) times the power of two of its block:
 * positions s B .. s B + B - 1 of a page, of one KV head, share a byte e that stands for 2^(e - 127)
 * (255: NaN).  Layouts: K and V pages (num_pages, page_size, H_kv, d) bytes, K and V powers
 * (num_pages, page_size / B, H_kv) bytes; 1 + 1 / (B d) bytes a value.  The steps, tables, slots
 * and lengths are those above; kv_page_map serves both.  A power of two instead of any scale: taking
 * a larger one later leaves the numbers' mantissas alone, and fp16 and bf16 hold the values exactly. */

typedef struct {
    int64_t num_tokens;    /* T */
    int64_t num_kv_heads;  /* H_kv */
    int64_t head_dim;      /* d; H_kv d at most 2^29 */
    int64_t page_size;
    int64_t num_pages;
    int64_t block_size;    /* B: at most 64, divides page_size; 0: 16 */
    int64_t kv_stride;     /* elements from row to row of K_new and V_new; 0: H_kv d */
    int64_t page_stride, row_stride, head_stride;   /* bytes of the cache; 0: the dense layout's */
} kv_page_store_q8_params_t;

/* inputs  [K_new (T, H_kv, d), V_new (T, H_kv, d), slots (T)]
 * outputs [K_pages, V_pages, K_powers, V_powers], in place
 * The power of a block's new rows is the least whose 448 fold no finite value of theirs exceeds (0 where
 * there is none).  A block whose first position is among them begins with it; else the block takes
 * the larger of it and the one that it has, and where that grows what the block holds (all its
 * positions but the new ones) is divided by as much: exact but for numbers that come below 2^-6 of
 * the power.  Values are rounded to nearest, ties to even; infinite and NaN ones become NaN.  Where a
 * rounding would pass the type's largest number, as 65504 to 65536, the one below is stored, so that
 * what is read back stays finite.  A row with an invalid slot is not stored.  Rows for one block stand
 * together, as kv_page_map gives them: in any order, the first and the last of them less than 64 rows apart, and
 * between them no other row but such as are not stored; and each slot may be given once per
 * call: otherwise that block's numbers and powers mean nothing.  Seven arrays of their own (-1 where
 * an output is another array). */
int kv_page_store_q8_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
int kv_page_store_q8_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

typedef struct {
    int64_t batch_size, num_tokens, num_heads, num_kv_heads, head_dim;   /* as in mha_paged_params_t */
    float   scale;
    int64_t page_size, num_pages, max_pages;
    int64_t block_size;    /* as in kv_page_store_q8_params_t */
    int64_t max_new, max_len;
    int64_t q_stride;      /* elements from row to row of Q; 0 = H_q d */
    int64_t page_stride, row_stride, head_stride;   /* bytes of the cache; 0: the dense layout's */
} mha_paged_q8_params_t;

/* inputs  [Q (T, H_q, d), K_pages, V_pages, block_table (B, max_pages), seq_lens (B), q_start (B + 1),
 *          K_powers, V_powers]
 * outputs [O (T, H_q, d)]
 * mha_paged_attn's rules, on the values that the bytes stand for; Q and O are of the operator's type.
 * f16: values are taken as fp16, which is exact for what kv_page_store_q8_f16 stores; past fp16's range
 * they may count as infinite.  The weights of V are sums of two fp16 numbers each, in every tile (other than
 * mha_paged_attn's, whose tiles of more than 16 rows round them to one).  f32: as bf16, exact but for
 * values below 2^-126, with Q and the weights as sums of three bf16 numbers each, which are FP32's 24 bits (Q
 * below 3.38e38).  A NaN V touches the rows
 * that see it; rows that do not, though a later token of the same call does, are computed again by a slow
 * loop.  d = 64 and 128 with blocks of a multiple of 16 positions, 16-byte aligned pointers (the powers'
 * apart) and strides, scale > 0 and at most 32768 sequences run on the matrix cores, every other
 * call on a plain kernel. */
int mha_paged_attn_q8_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
int mha_paged_attn_q8_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

int register_kv_page_map_i32_cuda(void);
int register_kv_page_store_f32_cuda(void);
int register_kv_page_store_f16_cuda(void);
int register_mha_paged_attn_f32_cuda(void);
int register_mha_paged_attn_f16_cuda(void);
int register_kv_page_store_q8_f32_cuda(void);
int register_kv_page_store_q8_f16_cuda(void);
int register_mha_paged_attn_q8_f32_cuda(void);
int register_mha_paged_attn_q8_f16_cuda(void);

#ifdef __cplusplus
}
#endif

#endif /* CF_PAGED_OPS_H_ */
