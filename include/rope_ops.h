/*
 * rope_ops.h — rotary position encoding on the GPU: the reference's RoPE operator and a
 * decode operator with RoPE applied to the new token's Q and K.
 *
 * Angles follow rope.c:38-45 exactly: angle = pos / powf(base, 2i/d), with (cos, sin)
 * from glibc on the host, kept per device in a table of (n_pos, d/2) float pairs that
 * grows on demand (a synchronous upload the first time a (base, d) pair or a longer
 * range is used) and is freed by gpu_platform_finalize.  Pairs (2i, 2i+1) of each head
 * are rotated: x'[2i] = x[2i]·cos − x[2i+1]·sin, x'[2i+1] = x[2i]·sin + x[2i+1]·cos, in
 * fp32 without contraction (fp16 I/O rounds once).  Return codes as in mha_ops.h.
 */
#ifndef CF_ROPE_OPS_H_
#define CF_ROPE_OPS_H_

#include "operator.h"
#include "rope_int.h"
#include "mha_decode_int.h"

#ifdef __cplusplus
extern "C" {
#endif

/* RoPE, FP32.  Replaces rope_f32_cuda (src/operator/nn/rope_cuda.cu:35-51).
 * inputs [x (S, H, d)], outputs [y (S, H, d)], y may alias x (in place, OP_FLAG_IN_PLACE);
 * row pos is rotated by position pos.  Like the reference, one sequence (B = 1): a batch
 * is S·B rows only if positions restart per sequence, which they do not here. */
int rope_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
/* RoPE with FP16 I/O (new; the graph dispatches "<base>_f16_cuda" for an F16 output). */
int rope_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

/* MHA_Decode with RoPE (new; the reference runs RoPE as a separate op on the
 * projections, which its fused decode op cannot do).  Same slots, validation and
 * results as mha_decode_{f32,f16}_cuda, except that Q and K_new are rotated at the
 * token's position (cache_len, or seq_lens[b] in ragged mode) after the projection,
 * before K_new is stored and before the scores.  V is not rotated. */
typedef struct {
    mha_decode_params_t decode;
    float               rope_base;   /* > 0 */
    int32_t             reserved;    /* 0 */
} mha_decode_rope_params_t;

int mha_decode_rope_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params,
                             stream_t* stream);
int mha_decode_rope_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params,
                             stream_t* stream);

/* Norms of Q and K, each head by itself, and their rotation by position, in one pass (new): what
 * stands between a layer's projection and a cache.  x is a head's d values, in FP32:
 *   norm 1  y = x / sqrt(mean(x^2) + eps) * gain
 *   norm 2  y = (x - mean(x)) / sqrt(var(x) + eps) * gain + bias   (var: the mean square around it)
 *   norm 0  y = x
 * then the first rotary_dim values of y are turned and the rest stay as they are; the result is
 * rounded to the type once.  Pair i < r / 2 of r = rotary_dim values is (2i, 2i + 1), or with
 * `halves` (i, i + r / 2); it turns by position * f_i with f_i = base^(-2i / r), or for contexts
 * longer than the trained one (`original_len` = L positions, `factor` = s)
 *   scaling 1  f_i / s
 *   scaling 2  by the turns t_i = L f_i / (2 pi) that the pair makes in L: f_i / s where t_i < low, f_i
 *              where t_i > high, in between f_i (w + (1 - w) / s) with w = (t_i - low) / (high - low)
 *   scaling 3  by the pair's index: f_i (1 - g + g / s), g = (i - lo) / max(hi - lo, 0.001) held in
 *              [0, 1], with lo = max(floor(c(high)), 0), hi = min(ceil(c(low)), r - 1) and
 *              c(t) = r ln(L / (2 pi t)) / (2 ln base)
 * and cos and sin are multiplied by `amplitude`.  Frequencies and angles are worked out in 64 bits, so
 * far positions lose nothing. */
#define QK_ROPE_MAX_DIM 256
#define QK_HEAD_MAX_DIM 1024
typedef struct {
    int64_t num_tokens;     /* T: rows */
    int64_t num_heads;      /* H_q, 0: no Q */
    int64_t num_kv_heads;   /* H_kv, 0: no K */
    int64_t head_dim;       /* d, at most QK_HEAD_MAX_DIM */
    int64_t rotary_dim;     /* r: even, at most d and QK_ROPE_MAX_DIM; 0: d */
    int32_t halves;         /* 0 or 1 */
    int32_t norm;           /* 0, 1, 2 */
    float   eps;            /* >= 0 */
    float   rope_base;      /* > 0 (scaling 3: > 1); 0: no rotation, positions are not looked at */
    int32_t scaling;        /* 0, 1, 2, 3 */
    float   factor;         /* scaling 1, 2, 3: > 0 */
    float   original_len;   /* scaling 2, 3: > 0 */
    float   low, high;      /* scaling 2, 3: 0 < low < high */
    float   amplitude;      /* 0: 1 */
    /* Elements from one row to the next; 0: rows follow each other.  The inputs can be the parts of
     * one (T, (H_q + 2 H_kv) d) projection. */
    int64_t q_stride, k_stride, q_out_stride, k_out_stride;
} qk_norm_rope_params_t;

/* inputs  [Q (T, H_q, d), K (T, H_kv, d), positions (T, int32), gain of Q (d), gain of K (d),
 *          bias of Q (d), bias of K (d)]
 * outputs [Q' (T, H_q, d), K' (T, H_kv, d)]
 * Without rotation positions may be NULL; with it a row of a negative position is left alone in both
 * outputs.  Gains are read with norm 1 and 2 and biases with norm 2 only; NULL stands for ones and
 * zeros (the slots have to be there).  An output may be its input (with one stride, else -1); other
 * overlaps are not allowed (-1 where the other's input or output is named).  Where every pointer and
 * stride is a multiple of 16 bytes, d one of 32 and at most 2048 bytes, and what turns together (r
 * values, half of them with `halves`) one of 16 bytes, a row's pieces of 16 bytes go at once; other calls take a
 * plain kernel. */
int qk_norm_rope_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);
int qk_norm_rope_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream);

int register_rope_f32_cuda(void);
int register_rope_f16_cuda(void);
int register_qk_norm_rope_f32_cuda(void);
int register_qk_norm_rope_f16_cuda(void);
int register_mha_decode_rope_f32_cuda(void);
int register_mha_decode_rope_f16_cuda(void);

/* Device (cos, sin) table for (base, d) covering positions 0 .. n_pos-1 on the current
 * device (NULL on failure).  Owned by the library. */
const float* rope_table_device(float base, int64_t d, int64_t n_pos);

#ifdef __cplusplus
}
#endif

#endif /* CF_ROPE_OPS_H_ */
