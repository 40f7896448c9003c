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

// ---- Rows of 16-byte pieces: two of them per lane, the next power of two of d / 2 pieces lanes a
// head.  A lane's pieces hold both values of its pairs: with `halves` pieces j and j + r / 2 values,
// else neighbours; lane j has pairs VEC j .. + VEC - 1 either way.  It stays on one row and goes over
// its heads, so that it keeps their cosines and sines, which the workgroup works out once per row.
// HBM bounds it: 8192 rows of 40 heads of 128 fp16, 168 MB, 28.2 us (5.9 TB/s), of 1001 FP32 rows of 24
// heads of 64 7.0 us; 16 rows take 7.1 us, 4.3 of them the kernel's. ----
constexpr int kThreads = 256;
template <typename T> struct alignas(16) Piece { T e[16 / sizeof(T)]; };

struct WideQk {
    int lanes;             // a head's, a power of two
    int rows;              // of a workgroup
    int at_once;           // heads of a row: rows * at_once * lanes = kThreads
};

// Sum over the lanes of a head.
__device__ __forceinline__ float head_sum(float x, int lanes) {
    if (lanes > 1) x += dpp_f<kDppXor1>(x);
    if (lanes > 2) x += dpp_f<kDppXor2>(x);
    if (lanes > 4) x += dpp_f<kDppHalfMirror>(x);
    if (lanes > 8) x += dpp_f<kDppMirror>(x);
    if (lanes > 16) x = add_xor16(x);
    if (lanes > 32) x = add_xor32(x);
    return x;
}

constexpr int kRows = 4;
template <typename T, int NORM, bool PAST>
__global__ __launch_bounds__(kThreads)
void qk_norm_wide(cf_qk_norm_args_t a, WideQk p, int64_t row0) {
    constexpr int VEC = 16 / sizeof(T);
    typedef Piece<T> piece_t;
    // Two pairs' (cos, sin) together, those of neighbouring lanes beside each other.
    __shared__ f4_t turns[kRows][VEC / 2][CF_QK_ROPE_MAX_DIM / 2 / VEC + 1];
    const int tid = threadIdx.x, slot = tid / p.lanes, row = slot / p.at_once;
    const int64_t t0 = row0 + (int64_t)blockIdx.x * p.rows, t = t0 + row;
    const int n_rows = (int)min((int64_t)p.rows, a.T - t0);
    const int n_q = a.rows[0].heads, heads = n_q + a.rows[1].heads;
    // This lane's pieces.
    const int j = tid & (p.lanes - 1), half = a.r / (2 * VEC);
    const bool real = 2 * VEC * j < a.d, halves = a.halves && a.r > 0;
    const int e0 = halves ? (j < half ? VEC * j : 2 * VEC * j) : 2 * VEC * j;
    const int e1 = halves && j < half ? e0 + a.r / 2 : e0 + VEC;
    const bool turned0 = e0 < a.r, turned1 = halves ? turned0 : e1 < a.r;
    const int step = p.at_once * (int)gridDim.y;
    int head = slot % p.at_once + p.at_once * (int)blockIdx.y;
    const int pos = a.positions && row < n_rows ? a.positions[t] : 0;
    const bool skip = row >= n_rows || pos < 0;
    auto load = [&](int h, piece_t (&x)[2]) {
        if (h >= heads || skip || !real) return;
        const cf_qk_rows_t& rows = a.rows[h >= n_q];
        const T* const from = (const T*)rows.x + t * rows.stride + (int64_t)(h >= n_q ? h - n_q : h) * a.d;
        x[0] = *(const piece_t*)(from + e0);
        x[1] = *(const piece_t*)(from + e1);
    };
    piece_t next[2] = {};
    load(head, next);
    // Gains and biases of Q and K.
    piece_t gain[NORM > 0 ? 2 : 1][2], bias[NORM == 2 ? 2 : 1][2];
    auto of_head = [&](piece_t (&to)[2], const void* from, float without) {
        if (from && real) {
            to[0] = *(const piece_t*)((const T*)from + e0);
            to[1] = *(const piece_t*)((const T*)from + e1);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) to[0].e[e] = to[1].e[e] = (T)without;
        }
    };
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if constexpr (NORM > 0) of_head(gain[i], a.rows[i].gain, 1.0f);
        if constexpr (NORM == 2) of_head(bias[i], a.rows[i].bias, 0.0f);
    }
    float2 cs[VEC];
    if (a.positions) {
        for (int i = tid; i < n_rows * (a.r / 2); i += kThreads) {
            const int of = i / (a.r / 2), pair = i - of * (a.r / 2);
            ((float2*)&turns[of][pair % VEC / 2][pair / VEC])[pair & 1] = turn_of(a, a.positions[t0 + of], pair);
        }
        __syncthreads();
        if (turned0 && !skip)
#pragma unroll
            for (int q = 0; q < VEC / 2; q++) {
                const f4_t x = turns[row][q][j];
                cs[2 * q] = float2{x[0], x[1]};
                cs[2 * q + 1] = float2{x[2], x[3]};
            }
    }
    if (skip) return;
    for (; head < heads; head += step) {
        const bool is_k = head >= n_q;
        float u[2][VEC];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) u[k][e] = (float)next[k].e[e];       // zeros where there is no piece
        load(head + step, next);
        if constexpr (NORM > 0) {
            if constexpr (NORM == 2) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; e++) sum += u[0][e] + u[1][e];
                sum = head_sum(sum, p.lanes);                  // by all lanes
                const float mean = real ? sum / (float)a.d : 0.0f;
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) u[k][e] -= mean;
            }
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; e++) sum = __builtin_fmaf(u[0][e], u[0][e], __builtin_fmaf(u[1][e], u[1][e], sum));
            const float scale = 1.0f / sqrtf(head_sum(sum, p.lanes) / (float)a.d + a.eps);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    u[k][e] = u[k][e] * scale * (float)(is_k ? gain[1][k].e[e] : gain[0][k].e[e]);
                    if constexpr (NORM == 2) u[k][e] += (float)(is_k ? bias[1][k].e[e] : bias[0][k].e[e]);
                }
        }
        if (a.positions && turned0) {
            auto turn = [](float& x, float& y, float2 c) {
                const float v = x;
                x = v * c.x - y * c.y;
                y = v * c.y + y * c.x;
            };
            if (halves) {
#pragma unroll
                for (int e = 0; e < VEC; e++) turn(u[0][e], u[1][e], cs[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) turn(u[0][e], u[0][e + 1], cs[e / 2]);
                if (turned1)
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) turn(u[1][e], u[1][e + 1], cs[VEC / 2 + e / 2]);
            }
        }
        if (!real) continue;
        const cf_qk_rows_t& rows = a.rows[is_k];
        T* const y = (T*)rows.y + t * rows.out_stride + (int64_t)(is_k ? head - n_q : head) * a.d;
        piece_t out[2];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) out[k].e[e] = (T)u[k][e];
        auto put = [](T* to, const piece_t& x) {
            typedef uint32_t words_t __attribute__((ext_vector_type(4)));
            if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(words_t, x), (words_t*)to);
            else *(piece_t*)to = x;
        };
        put(y + e0, out[0]);
        put(y + e1, out[1]);
    }
}

// Results of more bytes than this are stored past the caches, which they would only sweep (rows of 40
// heads of 128 fp16, us by themselves and with a copy of Q behind them that reads it: 4096 rows, 42 MB,
// 16.0 and 33.0, through the caches 20.0 and 30.7; 8192 rows 29.7 and 63.3, and 40.8 and 65.5; 16384
// rows 73 and 126, and 76 and 134).
constexpr int64_t kPastBytes = 64 << 20;

template <typename T>
bool wide_ok(const cf_qk_norm_args_t& a) {
    constexpr int VEC = 16 / sizeof(T);
    uint64_t all = 0;
    for (int i = 0; i < 2; i++) {
        const cf_qk_rows_t& r = a.rows[i];
        if (r.heads == 0) continue;
        all |= (uint64_t)(uintptr_t)r.x | (uint64_t)(uintptr_t)r.y | (uint64_t)(uintptr_t)r.gain | (uint64_t)(uintptr_t)r.bias |
               (uint64_t)r.stride * sizeof(T) | (uint64_t)r.out_stride * sizeof(T);
    }
    return all % 16 == 0 && a.d % (2 * VEC) == 0 && a.d <= 64 * 2 * VEC && (a.halves ? a.r / 2 : a.r) % VEC == 0;
}

template <typename T>
int launch_qk_wide(const cf_qk_norm_args_t& a, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    WideQk p;
    p.lanes = 1;
    while (2 * VEC * p.lanes < a.d) p.lanes *= 2;
    const int heads = a.rows[0].heads + a.rows[1].heads;
    // Few rows: a workgroup for every 256 lanes' worth of heads, else one for four rows (us with the former and
    // with the latter: 40 heads of 128 fp16, 512 rows 7.1 and 7.8, 1001 9.6 and 9.2, 2048 16.3 and 11.8; 24 of 64
    // fp16 or FP32, up to 1500 rows 7.0 and 7.1, 4096 FP32 ones 11.2 and 10.1.  40 of 128 FP32, which the
    // rule does not go by, are faster with the former throughout: 512 rows 7.0 and 12.0, 4096 27.3 and 31.0).
    const bool few = a.T < 1024;
    p.rows = few ? 1 : kRows;
    p.at_once = kThreads / p.lanes / p.rows;
    const int parts = few ? (heads + p.at_once - 1) / p.at_once : 1;
    const bool past = a.T * heads * a.d * (int64_t)sizeof(T) > kPastBytes;
    constexpr int64_t kMost = 1 << 22;             // workgroups of a launch: a grid has less than 2^32 threads
    for (int64_t t0 = 0; t0 < a.T; t0 += kMost * p.rows) {
        const int64_t n = (a.T - t0 + p.rows - 1) / p.rows;
        const dim3 grid((unsigned)(n < kMost ? n : kMost), (unsigned)parts), block(kThreads);
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a, p, t0); };
        if (a.norm == 0) past ? go(qk_norm_wide<T, 0, true>) : go(qk_norm_wide<T, 0, false>);
        else if (a.norm == 1) past ? go(qk_norm_wide<T, 1, true>) : go(qk_norm_wide<T, 1, false>);
        else past ? go(qk_norm_wide<T, 2, true>) : go(qk_norm_wide<T, 2, false>);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return 0;
}

template <typename T>
int launch_qk(const cf_qk_norm_args_t& a, hipStream_t st) {
    if (wide_ok<T>(a)) return launch_qk_wide<T>(a, st);
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
