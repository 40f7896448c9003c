// paged_attn_q8.hip — attention of chunks of new tokens over a paged KV cache of 8-bit numbers
// (gfx950).  The sums, rows and positions are those of paged_attn.hip; K and V are codes times the
// power of two of their block.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_tiles.h"
#include "e4m3.h"

namespace {

// What the kernels go by beside PagedPlan.
struct Q8Divs { FastDiv page, block; };

// A position's place in the cache (bytes) and its block's in the powers, of KV head 0; at < 0: none.
struct Cell { int64_t at, power; };
__device__ __forceinline__ Cell cell_of(const cf_paged_q8_args_t& a, const Q8Divs& dv, const int32_t* table, int key) {
    const int idx = fastdiv(key, dv.page), page = table[idx], in = key - idx * a.at.page_size;
    if ((unsigned)page >= (unsigned)a.at.num_pages) return {-1, 0};
    return {(int64_t)page * a.at.page_stride + (int64_t)in * a.at.row_stride,
            ((int64_t)page * (a.at.page_size / a.block) + fastdiv(in, dv.block)) * a.at.H_kv};
}

// ---- One row of one head by a wave, 64 positions at a time: lanes are positions for the scores
// and dims (at most 64 DIMS) for the sum over V.  Of positions [key0, key1); into O, or into a
// record whose m, l and sum for this row start at rec, rec + tm and rec_sum. ----
template <typename T, int DIMS>
__device__ __forceinline__ void plain_row_q8(const cf_paged_q8_args_t& a, const Q8Divs& dv, const SeqRows& s, int b, int tok,
                                             int h, int d, int key0 = 0, int key1 = INT32_MAX, float* rec = nullptr,
                                             int tm = 0, float* rec_sum = nullptr) {
    const int lane = threadIdx.x & 63;
    const int seen = min(min(s.len - s.n + tok + 1, s.len), key1);
    const int kvh = h / (a.at.H_q / a.at.H_kv);
    const int32_t* const table = a.at.table + (size_t)b * a.at.max_pages;
    const T* const q = (const T*)a.at.q + (int64_t)(s.row0 + tok) * a.at.q_stride + (int64_t)h * d;
    const uint8_t* const k = (const uint8_t*)a.at.k + (int64_t)kvh * a.at.head_stride;
    const uint8_t* const v = (const uint8_t*)a.at.v + (int64_t)kvh * a.at.head_stride;
    const float c = a.at.scale * kLog2e;
    float m = -INFINITY, l = 0.0f, acc[DIMS];
#pragma unroll
    for (int i = 0; i < DIMS; i++) acc[i] = 0.0f;
#pragma clang loop unroll(disable)
    for (uint32_t at0 = (uint32_t)key0; at0 < (uint32_t)max(seen, 0); at0 += 64) {    // unsigned: up to 2^31 positions
        const int k0 = (int)at0, key = k0 + lane;
        int64_t at = 0;
        int vpower = 0;
        float x = -INFINITY;
        if (key < seen) {
            const Cell cell = cell_of(a, dv, table, key);
            if (cell.at >= 0) {
                at = cell.at;
                vpower = a.v_scales[cell.power + kvh];
                const float kpower = power_bits(a.k_scales[cell.power + kvh]);
                float dot = 0.0f;
#pragma clang loop unroll(disable)
                for (int e = 0; e < d; e++) dot = __builtin_fmaf((float)q[e], codes_f32<false>(k[at + e], kpower)[0], dot);
                x = dot * c;
            }
        }
        const float m_new = fmaxf(m, wave_max(x));
        if (m_new == -INFINITY && !__builtin_amdgcn_ballot_w64(x != x)) continue;
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2f(m - m_use), p = exp2f(x - m_use);
        m = m_new;
        l = l * alpha + wave_sum(p);
#pragma unroll
        for (int i = 0; i < DIMS; i++) acc[i] *= alpha;
#pragma clang loop unroll(disable)
        for (int j = 0; j < min(64, seen - k0); j++) {
            const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
            if (pj == 0.0f) continue;          // not attended: its V may hold anything
            const int64_t row = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32) |
                                          (uint32_t)__builtin_amdgcn_readlane((int)at, j));
            const float power = power_bits(__builtin_amdgcn_readlane(vpower, j));
#pragma unroll
            for (int i = 0; i < DIMS; i++)
                if (lane + 64 * i < d)
                    acc[i] = __builtin_fmaf(pj, codes_f32<false>(v[row + lane + 64 * i], power)[0], acc[i]);
        }
    }
    if (rec) {
        if (lane == 0) {
            rec[0] = m;
            rec[tm] = l;
        }
#pragma unroll
        for (int i = 0; i < DIMS; i++)
            if (lane + 64 * i < d) rec_sum[lane + 64 * i] = acc[i];
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* const o = (T*)a.at.o + ((int64_t)(s.row0 + tok) * a.at.H_q + h) * d;
#pragma unroll
    for (int i = 0; i < DIMS; i++)
        if (lane + 64 * i < d) o[lane + 64 * i] = (T)(acc[i] * inv);
}

// ---- Every shape: a wave per row and head. ----
constexpr int kAnyDims = 512 / 64;             // dims per lane
template <typename T>
__global__ __launch_bounds__(256)
void paged_any_q8(cf_paged_q8_args_t a, Q8Divs dv) {
    for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < (int64_t)a.at.T * a.at.H_q;
         unit += 4 * (int64_t)gridDim.x) {
        const int t = (int)(unit / a.at.H_q), h = (int)(unit - (int64_t)t * a.at.H_q);
        int lo = 0, hi = a.at.B;               // the last sequence that does not start behind t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.at.q_start[mid] <= t) lo = mid; else hi = mid;
        }
        const SeqRows s = seq_rows(a.at, lo);
        if (t >= s.row0 && t < s.row0 + s.n) plain_row_q8<T, kAnyDims>(a, dv, s, lo, t - s.row0, h, a.at.d);
    }
}

}  // namespace

extern "C" size_t cf_paged_attn_q8_bytes(const cf_paged_q8_args_t*) { return 0; }

extern "C" int cf_launch_paged_attn_q8(const cf_paged_q8_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    const cf_paged_attn_args_t& t = a->at;
    if (t.B <= 0 || t.T <= 0 || t.d <= 0 || t.d > 64 * kAnyDims || t.H_kv <= 0 || t.H_q % t.H_kv != 0 || a->block <= 0 ||
        t.page_size % a->block != 0)
        return (int)hipErrorInvalidValue;
    const Q8Divs dv = {fastdiv_make(t.page_size), fastdiv_make(a->block)};
    int64_t wgs = ((int64_t)t.T * t.H_q + 3) / 4;
    if (wgs > (1 << 22)) wgs = 1 << 22;        // a grid has less than 2^32 threads
    if (t.elem == CF_ELEM_F16) hipLaunchKernelGGL(paged_any_q8<_Float16>, dim3((unsigned)wgs), dim3(256), 0, st, *a, dv);
    else hipLaunchKernelGGL(paged_any_q8<float>, dim3((unsigned)wgs), dim3(256), 0, st, *a, dv);
    return (int)hipGetLastError();
}
