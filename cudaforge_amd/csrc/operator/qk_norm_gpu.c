/*
 * qk_norm_gpu.c — host side of the norms and rotation of Q and K (rope_ops.h): argument checks,
 * the pairs' frequencies and the launch.
 */
#include "rope_ops.h"
#include "op_common.h"
#include "../kernels/kernels.h"

#include <math.h>
#include <string.h>

#define TWO_PI 6.283185307179586476925286766559L

static int positive(float x) { return x > 0.0f && !isinf(x); }

/* Turns per position of each of the r / 2 pairs.  In turns, so that the kernel reduces an angle by
 * dropping whole numbers; one power and products of 64 bits of mantissa, as a power per pair would
 * take longer than the launch.  -1: parameters that give no frequency. */
static int fill_turns(const qk_norm_rope_params_t* p, int64_t r, double* turns) {
    const long double base = p->rope_base, factor = p->factor, L = p->original_len;
    long double low = p->low, high = p->high;
    if (p->scaling < 0 || p->scaling > 3) return -1;
    if (p->scaling >= 1 && !positive(p->factor)) return -1;
    if (p->scaling >= 2 && (!positive(p->original_len) || !positive(p->low) || !positive(p->high) || !(p->low < p->high))) return -1;
    if (p->scaling == 3) {
        if (!(p->rope_base > 1.0f)) return -1;
        /* low and high become the indexes between which the division sets in. */
        const long double per = (long double)r / (2.0L * logl(base));
        const long double lo = floorl(per * logl(L / (TWO_PI * high))), hi = ceill(per * logl(L / (TWO_PI * low)));
        low = lo > 0.0L ? lo : 0.0L;
        high = hi < (long double)(r - 1) ? hi : (long double)(r - 1);
    }
    const long double step = powl(base, -2.0L / (long double)r), divided = p->scaling ? 1.0L / factor : 1.0L;
    const long double range = p->scaling < 2 ? 0.0L : 1.0L / (p->scaling == 2 || high - low > 0.001L ? high - low : 0.001L);
    long double f = 1.0L / TWO_PI;
    for (int64_t i = 0; i < r / 2; i++, f *= step) {
        long double keep = p->scaling == 1 ? 0.0L : 1.0L;      /* share of f that is not divided */
        if (p->scaling == 2) keep = (L * f - low) * range;
        if (p->scaling == 3) keep = 1.0L - ((long double)i - low) * range;
        keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
        turns[i] = (double)(p->scaling == 0 ? f : f * (keep + (1.0L - keep) * divided));
    }
    return 0;
}

static int qk_norm_rope_op(int elem, const void* inputs[], void* outputs[], const operator_params_t* params,
                           stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    const qk_norm_rope_params_t* p = (const qk_norm_rope_params_t*)params;
    const int64_t d = p->head_dim, r = p->rotary_dim > 0 ? p->rotary_dim : d;
    if (p->num_tokens < 0 || p->num_tokens > INT32_MAX || d <= 0 || d > QK_HEAD_MAX_DIM || p->rotary_dim < 0) return -1;
    if (p->num_heads < 0 || p->num_kv_heads < 0 || p->num_heads > 65535 || p->num_kv_heads > 65535) return -1;
    if (p->num_heads + p->num_kv_heads == 0) return -1;
    if (p->norm < 0 || p->norm > 2 || (p->halves != 0 && p->halves != 1)) return -1;
    if (p->norm != 0 && (!(p->eps >= 0.0f) || isinf(p->eps))) return -1;
    if (!(p->rope_base >= 0.0f) || isinf(p->rope_base) || isnan(p->amplitude) || isinf(p->amplitude)) return -1;
    cf_qk_norm_args_t a;
    memset(&a, 0, sizeof(a));
    a.T = p->num_tokens;
    a.d = (int32_t)d;
    a.halves = p->halves;
    a.norm = p->norm;
    a.eps = p->eps;
    a.elem = elem;
    a.amplitude = p->amplitude != 0.0f ? p->amplitude : 1.0f;
    const int64_t heads[2] = {p->num_heads, p->num_kv_heads};
    const int64_t in[2] = {p->q_stride, p->k_stride}, out[2] = {p->q_out_stride, p->k_out_stride};
    for (int i = 0; i < 2; i++) {
        if (in[i] < 0 || out[i] < 0) return -1;
        if (heads[i] == 0) continue;
        if (!inputs[i] || !outputs[i]) return -1;
        cf_qk_rows_t* const x = &a.rows[i];
        x->x = inputs[i];
        x->y = outputs[i];
        x->heads = (int32_t)heads[i];
        x->stride = in[i] > 0 ? in[i] : heads[i] * d;
        x->out_stride = out[i] > 0 ? out[i] : heads[i] * d;
        if (x->x == x->y && x->stride != x->out_stride) return -1;
        if (p->norm >= 1) x->gain = inputs[3 + i];
        if (p->norm == 2) x->bias = inputs[5 + i];
    }
    /* Rows of Q and of K are written while others of both are still to be read. */
    if (heads[0] && heads[1] && (outputs[0] == outputs[1] || outputs[0] == inputs[1] || outputs[1] == inputs[0])) return -1;
    if (p->rope_base > 0.0f) {
        if ((r & 1) || r > d || r > QK_ROPE_MAX_DIM || !inputs[2]) return -1;
        if (fill_turns(p, r, a.turns) != 0) return -1;
        a.positions = (const int32_t*)inputs[2];
        a.r = (int32_t)r;
    }
    if (p->num_tokens == 0) return 0;
    return cf_launch_qk_norm(&a, cf_stream_of(stream));
}

int qk_norm_rope_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return qk_norm_rope_op(CF_ELEM_F32, inputs, outputs, params, stream);
}

int qk_norm_rope_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return qk_norm_rope_op(CF_ELEM_F16, inputs, outputs, params, stream);
}

int register_qk_norm_rope_f32_cuda(void) {
    static const operator_registry_t reg = {"qk_norm_rope_f32_cuda", "f32", qk_norm_rope_f32_cuda, 1, OP_FLAG_IN_PLACE};
    return operator_register(&reg);
}

int register_qk_norm_rope_f16_cuda(void) {
    static const operator_registry_t reg = {"qk_norm_rope_f16_cuda", "f16", qk_norm_rope_f16_cuda, 1, OP_FLAG_IN_PLACE};
    return operator_register(&reg);
}
