// qk_norm.hip — norms of Q and K, each head by itself, and their rotation by position (gfx950).
//
// Per head of d values: m = mean(x) (norm 2, else 0), s = 1 / sqrt(mean((x - m)^2) + eps),
// y = (x - m) s gain + bias, all in FP32; then pairs (u, v) of the first r values become
// (u c - v s, u s + v c) with the cosine and sine of position * turns_i * 2 pi, the whole turns of
// which are dropped in 64 bits.  One rounding, of the result.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "cdna4.h"

namespace {

using namespace cdna4;

// (cos, sin) of pair i at a position.
__device__ __forceinline__ float2 turn_of(const cf_qk_norm_args_t& a, int pos, int i) {
    double w = (double)pos * a.turns[i];
    w -= rint(w);
    float s, c;
    sincospif(2.0f * (float)w, &s, &c);
    return float2{a.amplitude * c, a.amplitude * s};
}

// ---- Every shape: a wave per head, its lanes over the pairs and then over what is not turned. ----
constexpr int kAnyThreads = 256, kAnyWaves = kAnyThreads / 64;
template <typename T>
__global__ __launch_bounds__(kAnyThreads)
void qk_norm_any(cf_qk_norm_args_t a) {
    const int lane = threadIdx.x & 63, heads = a.rows[0].heads + a.rows[1].heads;
    const int64_t units = a.T * heads;
    for (int64_t unit = (int64_t)blockIdx.x * kAnyWaves + (threadIdx.x >> 6); unit < units; unit += (int64_t)gridDim.x * kAnyWaves) {
        const int64_t t = unit / heads;
        const int head = (int)(unit - t * heads), which = head >= a.rows[0].heads;
        const cf_qk_rows_t& rows = a.rows[which];
        const int h = head - (which ? a.rows[0].heads : 0);
        const int pos = a.positions ? a.positions[t] : 0;
        if (pos < 0) continue;
        const T* const x = (const T*)rows.x + t * rows.stride + (int64_t)h * a.d;
        T* const y = (T*)rows.y + t * rows.out_stride + (int64_t)h * a.d;
        const T* const gain = (const T*)rows.gain;
        const T* const bias = (const T*)rows.bias;
        float mean = 0.0f, scale = 1.0f;
        if (a.norm == 2) {
            float sum = 0.0f;
            for (int e = lane; e < a.d; e += 64) sum += (float)x[e];
            mean = wave_sum(sum) / (float)a.d;
        }
        if (a.norm) {
            float sum = 0.0f;
            for (int e = lane; e < a.d; e += 64) {
                const float u = (float)x[e] - mean;
                sum = __builtin_fmaf(u, u, sum);
            }
            scale = 1.0f / sqrtf(wave_sum(sum) / (float)a.d + a.eps);
        }
        auto normed = [&](int e) {
            float u = ((float)x[e] - mean) * scale;
            if (gain) u *= (float)gain[e];
            if (bias) u += (float)bias[e];
            return u;
        };
        // A lane reads a pair before it writes it, and no other lane's pair: x may be y.
        for (int i = lane; i < a.r / 2; i += 64) {
            const int e0 = a.halves ? i : 2 * i, e1 = a.halves ? i + a.r / 2 : 2 * i + 1;
            const float u = normed(e0), v = normed(e1);
            const float2 cs = turn_of(a, pos, i);
            y[e0] = (T)(u * cs.x - v * cs.y);
            y[e1] = (T)(u * cs.y + v * cs.x);
        }
        for (int e = a.r + lane; e < a.d; e += 64) y[e] = (T)normed(e);
    }
}

template <typename T>
int launch_qk(const cf_qk_norm_args_t& a, hipStream_t st) {
    const int heads = a.rows[0].heads + a.rows[1].heads;
    int64_t wgs = (a.T * heads + kAnyWaves - 1) / kAnyWaves;
    if (wgs > (1 << 22)) wgs = 1 << 22;            // a grid has less than 2^32 threads
    hipLaunchKernelGGL(qk_norm_any<T>, dim3((unsigned)wgs), dim3(kAnyThreads), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int cf_launch_qk_norm(const cf_qk_norm_args_t* a, void* stream) {
    if (a->T <= 0 || a->d <= 0 || a->r < 0 || a->r > a->d || a->r > CF_QK_ROPE_MAX_DIM || a->rows[0].heads + a->rows[1].heads <= 0)
        return (int)hipErrorInvalidValue;
    return a->elem == CF_ELEM_F16 ? launch_qk<_Float16>(*a, (hipStream_t)stream) : launch_qk<float>(*a, (hipStream_t)stream);
}
