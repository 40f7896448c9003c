/*
 * paged_gpu.c — host side of the paged KV cache's operators (paged_ops.h): argument checks,
 * layout defaults and launches.  Nothing here reads device memory: lengths, tables and slots
 * are checked where the kernels use them.
 */
#include "paged_ops.h"
#include "gpu_ops.h"
#include "op_common.h"
#include "../kernels/kernels.h"

#include <math.h>
#include <stdint.h>
#include <string.h>

/* num_pages pages of page_size positions, counted in 32 bits. */
static int pages_ok(int64_t page_size, int64_t num_pages) {
    return page_size > 0 && num_pages > 0 && num_pages <= INT32_MAX / page_size;
}

/* The cache's strides, the dense (num_pages, page_size, H_kv, d) ones where 0 is given. */
typedef struct { int64_t page, row, head; } cache_strides_t;

static int cache_strides(int64_t page, int64_t row, int64_t head, int64_t page_size, int64_t H_kv, int64_t d,
                         cache_strides_t* s) {
    if (page < 0 || row < 0 || head < 0) return -1;
    s->head = head > 0 ? head : d;
    s->row = row > 0 ? row : H_kv * d;
    s->page = page > 0 ? page : page_size * H_kv * d;
    return 0;
}

/* ------------------------------------------------------------------ the map --- */

int kv_page_map_i32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    for (int i = 0; i < 3; i++) if (!inputs[i]) return -1;
    for (int i = 0; i < 7; i++) if (!outputs[i]) return -1;
    const kv_page_map_params_t* p = (const kv_page_map_params_t*)params;
    if (p->batch_size <= 0 || p->num_tokens < 0 || p->max_pages <= 0 || p->ring_size <= 0) return -1;
    if (p->batch_size > INT32_MAX - 1 || p->num_tokens > INT32_MAX || p->ring_size > (1 << 30)) return -1;
    if (!pages_ok(p->page_size, p->num_pages) || !pages_ok(p->page_size, p->max_pages)) return -1;
    /* The running count of new pages stays within 32 bits. */
    if (p->max_pages > INT32_MAX / p->batch_size) return -1;
    cf_page_map_args_t a;
    memset(&a, 0, sizeof(a));
    a.cache_lens = (const int32_t*)inputs[0];
    a.new_lens = (const int32_t*)inputs[1];
    a.counters = (const int32_t*)inputs[2];
    a.table = (int32_t*)outputs[0];
    a.ring = (int32_t*)outputs[1];
    a.seq_lens = (int32_t*)outputs[2];
    a.q_start = (int32_t*)outputs[3];
    a.positions = (int32_t*)outputs[4];
    a.slots = (int32_t*)outputs[5];
    a.counters_out = (int32_t*)outputs[6];
    a.B = (int32_t)p->batch_size;
    a.T = (int32_t)p->num_tokens;
    a.page_size = (int32_t)p->page_size;
    a.num_pages = (int32_t)p->num_pages;
    a.max_pages = (int32_t)p->max_pages;
    a.ring_size = (int32_t)p->ring_size;
    void* st = cf_stream_of(stream);
    const size_t ints = cf_page_map_info_ints(a.B, a.T);
    if (ints > 0 && !(a.info = (int32_t*)gpu_workspace_get_stream(st, ints * sizeof(int32_t)))) return -1;
    return cf_launch_page_map(&a, st);
}

/* ------------------------------------------------------------------ the store --- */

static int page_store_op(int elem, const void* inputs[], void* outputs[], const operator_params_t* params,
                         stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    for (int i = 0; i < 3; i++) if (!inputs[i]) return -1;
    if (!outputs[0] || !outputs[1]) return -1;
    const kv_page_store_params_t* p = (const kv_page_store_params_t*)params;
    if (p->num_tokens < 0 || p->num_kv_heads <= 0 || p->head_dim <= 0 || !pages_ok(p->page_size, p->num_pages)) return -1;
    if (p->num_tokens > INT32_MAX || p->num_kv_heads > 65535 || p->head_dim > 65535) return -1;
    /* The kernel counts the pieces of a K and a V row together in 32 bits. */
    if (p->num_kv_heads * p->head_dim > (1 << 29)) return -1;
    if (!(p->rope_base >= 0.0f) || isinf(p->rope_base)) return -1;
    if (p->q_stride < 0 || p->kv_stride < 0 || p->q_out_stride < 0) return -1;
    cf_page_store_args_t a;
    memset(&a, 0, sizeof(a));
    a.d = (int32_t)p->head_dim;
    a.H_kv = (int32_t)p->num_kv_heads;
    const int64_t kvd = p->num_kv_heads * p->head_dim;
    a.kv_stride = p->kv_stride > 0 ? p->kv_stride : kvd;
    if (p->rope_base > 0.0f) {
        if ((p->head_dim & 1) || p->head_dim > CF_PAGE_ROPE_MAX_DIM || !inputs[3]) return -1;
        if (!inputs[4] != !outputs[2]) return -1;
        a.rope = 1;
        a.positions = (const int32_t*)inputs[3];
        if (inputs[4]) {
            if (p->num_heads <= 0 || p->num_heads > 65535) return -1;
            a.q = inputs[4];
            a.q_out = outputs[2];
            a.H_q = (int32_t)p->num_heads;
            a.q_stride = p->q_stride > 0 ? p->q_stride : p->num_heads * p->head_dim;
            a.q_out_stride = p->q_out_stride > 0 ? p->q_out_stride : p->num_heads * p->head_dim;
            if (a.q_out == a.q && a.q_out_stride != a.q_stride) return -1;
        }
        /* In turns, so that the kernel reduces an angle by dropping whole numbers; one power and
         * products of 64 bits of mantissa (128 of them are off by 2^-57), as a power per pair
         * would take longer than the launch. */
        const long double step = powl((long double)p->rope_base, -2.0L / (long double)a.d);
        long double turns = 1.0L / 6.283185307179586476925286766559L;
        for (int i = 0; i < a.d / 2; i++, turns *= step) a.turns[i] = (double)turns;
    }
    cache_strides_t cs;
    if (cache_strides(p->page_stride, p->row_stride, p->head_stride, p->page_size, p->num_kv_heads, p->head_dim, &cs) != 0)
        return -1;
    if (p->num_tokens == 0) return 0;
    a.k = inputs[0];
    a.v = inputs[1];
    a.slots = (const int32_t*)inputs[2];
    a.k_pages = outputs[0];
    a.v_pages = outputs[1];
    a.T = p->num_tokens;
    a.page_stride = cs.page;
    a.row_stride = cs.row;
    a.head_stride = cs.head;
    a.page_size = (int32_t)p->page_size;
    a.num_slots = (int32_t)(p->num_pages * p->page_size);
    a.elem = elem;
    return cf_launch_page_store(&a, cf_stream_of(stream));
}

int kv_page_store_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return page_store_op(CF_ELEM_F32, inputs, outputs, params, stream);
}

int kv_page_store_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return page_store_op(CF_ELEM_F16, inputs, outputs, params, stream);
}

/* ------------------------------------------------------------------ attention --- */

/* 1: `a` (all zeros before) holds the call; 0: there is nothing to do; -1: refused. */
static int paged_attn_args(const mha_paged_params_t* p, int elem, const void* inputs[], void* outputs[],
                           cf_paged_attn_args_t* to) {
    for (int i = 0; i < 6; i++) if (!inputs[i]) return -1;
    if (!outputs[0]) return -1;
    const int64_t H = p->num_heads, H_kv = p->num_kv_heads > 0 ? p->num_kv_heads : H, d = p->head_dim;
    if (p->batch_size < 0 || p->num_tokens < 0 || H <= 0 || d <= 0 || H % H_kv != 0) return -1;
    if (p->batch_size > INT32_MAX - 1 || p->num_tokens > INT32_MAX || H > 65535 || d > 512) return -1;
    if (!pages_ok(p->page_size, p->num_pages) || p->max_pages <= 0 || !pages_ok(p->page_size, p->max_pages)) return -1;
    if (p->max_new < 0 || p->max_len < 0 || p->q_stride < 0) return -1;
    cache_strides_t cs;
    if (cache_strides(p->page_stride, p->row_stride, p->head_stride, p->page_size, H_kv, d, &cs) != 0) return -1;
    if (p->batch_size == 0 || p->num_tokens == 0) return 0;
    /* A row's tile may be read after another's rows are written. */
    for (int i = 0; i < 3; i++) if (outputs[0] == inputs[i]) return -1;
    cf_paged_attn_args_t a = *to;
    a.q = inputs[0];
    a.k = inputs[1];
    a.v = inputs[2];
    a.table = (const int32_t*)inputs[3];
    a.seq_lens = (const int32_t*)inputs[4];
    a.q_start = (const int32_t*)inputs[5];
    a.o = outputs[0];
    a.q_stride = p->q_stride > 0 ? p->q_stride : H * d;
    a.page_stride = cs.page;
    a.row_stride = cs.row;
    a.head_stride = cs.head;
    a.B = (int32_t)p->batch_size;
    a.T = (int32_t)p->num_tokens;
    a.H_q = (int32_t)H;
    a.H_kv = (int32_t)H_kv;
    a.d = (int32_t)d;
    a.page_size = (int32_t)p->page_size;
    a.num_pages = (int32_t)p->num_pages;
    a.max_pages = (int32_t)p->max_pages;
    a.max_new = p->max_new > 0 && p->max_new < p->num_tokens ? (int32_t)p->max_new : a.T;
    const int64_t table_len = p->max_pages * p->page_size;
    a.max_len = (int32_t)(p->max_len > 0 && p->max_len < table_len ? p->max_len : table_len);
    a.scale = p->scale;
    a.elem = elem;
    *to = a;
    return 1;
}

/* Without a buffer (no memory, or a recording on a stream that has none of that size) no tile
 * is cut. */
static void paged_attn_workspace(cf_paged_attn_args_t* a, size_t bytes, void* st) {
    if (bytes > 0 && !(a->workspace = gpu_workspace_try_stream(st, bytes)) &&
        !(a->workspace = gpu_workspace_get_stream(st, bytes)))
        a->uncut = 1;
}

static int paged_attn_op(int elem, const void* inputs[], void* outputs[], const operator_params_t* params,
                         stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    cf_paged_attn_args_t a;
    memset(&a, 0, sizeof(a));
    const int rc = paged_attn_args((const mha_paged_params_t*)params, elem, inputs, outputs, &a);
    if (rc != 1) return rc;
    void* st = cf_stream_of(stream);
    paged_attn_workspace(&a, cf_paged_attn_bytes(&a), st);
    return cf_launch_paged_attn(&a, st);
}

int mha_paged_attn_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return paged_attn_op(CF_ELEM_F32, inputs, outputs, params, stream);
}

int mha_paged_attn_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return paged_attn_op(CF_ELEM_F16, inputs, outputs, params, stream);
}

/* ------------------------------------------------------------------ the same in 8 bits --- */

/* Positions of a block, 0 where they are not allowed. */
static int64_t block_of(int64_t block, int64_t page_size) {
    if (block == 0) block = 16;
    return block > 0 && block <= CF_Q8_MAX_BLOCK && page_size % block == 0 ? block : 0;
}

static int page_store_q8_op(int elem, const void* inputs[], void* outputs[], const operator_params_t* params,
                            stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    for (int i = 0; i < 3; i++) if (!inputs[i]) return -1;
    for (int i = 0; i < 4; i++) if (!outputs[i]) return -1;
    const kv_page_store_q8_params_t* p = (const kv_page_store_q8_params_t*)params;
    if (p->num_tokens < 0 || p->num_kv_heads <= 0 || p->head_dim <= 0 || !pages_ok(p->page_size, p->num_pages)) return -1;
    if (p->num_tokens > INT32_MAX || p->num_kv_heads > 65535 || p->head_dim > 65535) return -1;
    if (p->num_kv_heads * p->head_dim > (1 << 29) || p->kv_stride < 0) return -1;
    const int64_t block = block_of(p->block_size, p->page_size);
    if (block == 0) return -1;
    cache_strides_t cs;
    if (cache_strides(p->page_stride, p->row_stride, p->head_stride, p->page_size, p->num_kv_heads, p->head_dim, &cs) != 0)
        return -1;
    if (p->num_tokens == 0) return 0;
    /* Each array is written by waves of its own. */
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < i; j++) if (outputs[i] == outputs[j]) return -1;
        for (int j = 0; j < 3; j++) if (outputs[i] == inputs[j]) return -1;
    }
    cf_page_store_q8_args_t a;
    memset(&a, 0, sizeof(a));
    a.k = inputs[0];
    a.v = inputs[1];
    a.slots = (const int32_t*)inputs[2];
    a.k_pages = (uint8_t*)outputs[0];
    a.v_pages = (uint8_t*)outputs[1];
    a.k_scales = (uint8_t*)outputs[2];
    a.v_scales = (uint8_t*)outputs[3];
    a.T = p->num_tokens;
    a.kv_stride = p->kv_stride > 0 ? p->kv_stride : p->num_kv_heads * p->head_dim;
    a.page_stride = cs.page;
    a.row_stride = cs.row;
    a.head_stride = cs.head;
    a.H_kv = (int32_t)p->num_kv_heads;
    a.d = (int32_t)p->head_dim;
    a.page_size = (int32_t)p->page_size;
    a.block = (int32_t)block;
    a.num_slots = (int32_t)(p->num_pages * p->page_size);
    a.elem = elem;
    return cf_launch_page_store_q8(&a, cf_stream_of(stream));
}

int kv_page_store_q8_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return page_store_q8_op(CF_ELEM_F32, inputs, outputs, params, stream);
}

int kv_page_store_q8_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return page_store_q8_op(CF_ELEM_F16, inputs, outputs, params, stream);
}

static int paged_attn_q8_op(int elem, const void* inputs[], void* outputs[], const operator_params_t* params,
                            stream_t* stream) {
    if (!inputs || !outputs || !params) return -1;
    for (int i = 0; i < 8; i++) if (!inputs[i]) return -1;
    const mha_paged_q8_params_t* p = (const mha_paged_q8_params_t*)params;
    const mha_paged_params_t same = {
        .batch_size = p->batch_size, .num_tokens = p->num_tokens, .num_heads = p->num_heads, .num_kv_heads = p->num_kv_heads,
        .head_dim = p->head_dim, .scale = p->scale, .page_size = p->page_size, .num_pages = p->num_pages,
        .max_pages = p->max_pages, .max_new = p->max_new, .max_len = p->max_len, .q_stride = p->q_stride,
        .page_stride = p->page_stride, .row_stride = p->row_stride, .head_stride = p->head_stride};
    cf_paged_q8_args_t a;
    memset(&a, 0, sizeof(a));
    const int rc = paged_attn_args(&same, elem, inputs, outputs, &a.at);
    if (rc < 0 || (a.block = (int32_t)block_of(p->block_size, p->page_size)) == 0) return -1;
    if (rc == 0) return 0;
    for (int i = 6; i < 8; i++) if (outputs[0] == inputs[i]) return -1;
    a.k_scales = (const uint8_t*)inputs[6];
    a.v_scales = (const uint8_t*)inputs[7];
    void* st = cf_stream_of(stream);
    paged_attn_workspace(&a.at, cf_paged_attn_q8_bytes(&a), st);
    return cf_launch_paged_attn_q8(&a, st);
}

int mha_paged_attn_q8_f32_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return paged_attn_q8_op(CF_ELEM_F32, inputs, outputs, params, stream);
}

int mha_paged_attn_q8_f16_cuda(const void* inputs[], void* outputs[], const operator_params_t* params, stream_t* stream) {
    return paged_attn_q8_op(CF_ELEM_F16, inputs, outputs, params, stream);
}

/* ------------------------------------------------------------------ registrations --- */

int register_kv_page_map_i32_cuda(void) {
    static const operator_registry_t reg = {"kv_page_map_i32_cuda", "i32", kv_page_map_i32_cuda, 1, OP_FLAG_ALLOW_ALIAS};
    return operator_register(&reg);
}

int register_kv_page_store_f32_cuda(void) {
    static const operator_registry_t reg = {"kv_page_store_f32_cuda", "f32", kv_page_store_f32_cuda, 1, OP_FLAG_ALLOW_ALIAS};
    return operator_register(&reg);
}

int register_kv_page_store_f16_cuda(void) {
    static const operator_registry_t reg = {"kv_page_store_f16_cuda", "f16", kv_page_store_f16_cuda, 1, OP_FLAG_ALLOW_ALIAS};
    return operator_register(&reg);
}

int register_mha_paged_attn_f32_cuda(void) {
    static const operator_registry_t reg = {"mha_paged_attn_f32_cuda", "f32", mha_paged_attn_f32_cuda, 1, OP_FLAG_NONE};
    return operator_register(&reg);
}

int register_mha_paged_attn_f16_cuda(void) {
    static const operator_registry_t reg = {"mha_paged_attn_f16_cuda", "f16", mha_paged_attn_f16_cuda, 1, OP_FLAG_NONE};
    return operator_register(&reg);
}

int register_kv_page_store_q8_f32_cuda(void) {
    static const operator_registry_t reg = {"kv_page_store_q8_f32_cuda", "f32", kv_page_store_q8_f32_cuda, 1, OP_FLAG_ALLOW_ALIAS};
    return operator_register(&reg);
}

int register_kv_page_store_q8_f16_cuda(void) {
    static const operator_registry_t reg = {"kv_page_store_q8_f16_cuda", "f16", kv_page_store_q8_f16_cuda, 1, OP_FLAG_ALLOW_ALIAS};
    return operator_register(&reg);
}

int register_mha_paged_attn_q8_f32_cuda(void) {
    static const operator_registry_t reg = {"mha_paged_attn_q8_f32_cuda", "f32", mha_paged_attn_q8_f32_cuda, 1, OP_FLAG_NONE};
    return operator_register(&reg);
}

int register_mha_paged_attn_q8_f16_cuda(void) {
    static const operator_registry_t reg = {"mha_paged_attn_q8_f16_cuda", "f16", mha_paged_attn_q8_f16_cuda, 1, OP_FLAG_NONE};
    return operator_register(&reg);
}
