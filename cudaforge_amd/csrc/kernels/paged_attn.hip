// paged_attn.hip — attention of chunks of new tokens over a paged KV cache (gfx950).
//
// Row i of the n_b new rows of sequence b is position p = L_b - n_b + i of its L_b, and
//   O = sum_{j <= p} softmax_j(scale * q . k_j) v_j
// over the positions of valid pages (position j: page table[b][j / P], row j % P).  Softmax
// in one pass: running maximum m and sum l in FP32, everything rescaled by 2^(m_old - m)
// when the maximum moves; scores are kept in the log2 domain.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "cdna4.h"

namespace {

using namespace cdna4;

constexpr float kLog2e = 1.4426950408889634f;

// The rows of sequence b: q_start and seq_lens hold anything, rows stay within 0 .. T and
// the length within the table.
struct SeqRows {
    int row0;   // first row
    int n;      // rows
    int len;    // positions, the new ones included
};
__device__ __forceinline__ SeqRows seq_rows(const cf_paged_attn_args_t& a, int b) {
    SeqRows s;
    s.row0 = min(max(a.q_start[b], 0), a.T);
    s.n = min(max(a.q_start[b + 1], s.row0), a.T) - s.row0;
    s.len = min(max(a.seq_lens[b], 0), a.max_pages * a.page_size);
    return s;
}

// ---- Every shape: one wave per row and head, 64 positions at a time.  Lanes are positions
// for the scores and dims for the sum over V. ----
constexpr int kAnyDims = 512 / 64;             // dims per lane
template <typename T>
__global__ __launch_bounds__(256)
void paged_any(cf_paged_attn_args_t a, FastDiv by_page) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(unit / a.H_q), h = (int)(unit - (int64_t)t * a.H_q);
    if (t >= a.T) return;
    int lo = 0, hi = a.B;                      // the last sequence that does not start behind t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const SeqRows s = seq_rows(a, lo);
    if (t < s.row0 || t >= s.row0 + s.n) return;
    const int seen = min(s.len - s.n + (t - s.row0) + 1, s.len);
    const int32_t* const table = a.table + (size_t)lo * a.max_pages;
    const T* const q = (const T*)a.q + (int64_t)t * a.q_stride + (int64_t)h * a.d;
    const T* const k = (const T*)a.k + (int64_t)(h / (a.H_q / a.H_kv)) * a.head_stride;
    const T* const v = (const T*)a.v + (int64_t)(h / (a.H_q / a.H_kv)) * a.head_stride;
    const float c = a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f, acc[kAnyDims];
#pragma unroll
    for (int i = 0; i < kAnyDims; i++) acc[i] = 0.0f;
    for (int k0 = 0; k0 < seen; k0 += 64) {
        const int key = k0 + lane;
        int64_t at = 0;
        float x = -INFINITY;
        if (key < seen) {
            const int idx = fastdiv(key, by_page);
            const int page = table[idx];
            if ((unsigned)page < (unsigned)a.num_pages) {
                at = (int64_t)page * a.page_stride + (int64_t)(key - idx * a.page_size) * a.row_stride;
                float dot = 0.0f;
                for (int e = 0; e < a.d; e++) dot = __builtin_fmaf((float)q[e], (float)k[at + e], dot);
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
        for (int i = 0; i < kAnyDims; i++) acc[i] *= alpha;
        for (int j = 0; j < min(64, seen - k0); j++) {
            const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
            if (pj == 0.0f) continue;          // not attended: its V may hold anything
            const int64_t row = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32) |
                                          (uint32_t)__builtin_amdgcn_readlane((int)at, j));
#pragma unroll
            for (int i = 0; i < kAnyDims; i++)
                if (lane + 64 * i < a.d) acc[i] = __builtin_fmaf(pj, (float)v[row + lane + 64 * i], acc[i]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* const o = (T*)a.o + ((int64_t)t * a.H_q + h) * a.d;
#pragma unroll
    for (int i = 0; i < kAnyDims; i++)
        if (lane + 64 * i < a.d) o[lane + 64 * i] = (T)(acc[i] * inv);
}

}  // namespace

extern "C" int cf_launch_paged_attn(const cf_paged_attn_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    if (a->B <= 0 || a->T <= 0 || a->d <= 0 || a->d > 64 * kAnyDims || a->H_kv <= 0 || a->H_q % a->H_kv != 0)
        return (int)hipErrorInvalidValue;
    const FastDiv by_page = fastdiv_make(a->page_size);
    const int64_t wgs = ((int64_t)a->T * a->H_q + 3) / 4;
    if (wgs > 0x7fffffff) return (int)hipErrorInvalidValue;
    if (a->elem == CF_ELEM_F16) hipLaunchKernelGGL(paged_any<_Float16>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    else hipLaunchKernelGGL(paged_any<float>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    return (int)hipGetLastError();
}
