// paged_kv_q8.hip — the write of new K and V rows into pages of 8-bit numbers (gfx950).
//
// Rows of one block (block positions of a page, one KV head) stand together in a call, within 64 rows and with
// nothing between them but rows that are not stored: a run.  A wave takes a run of one head of K or V: the largest finite size A of it, the power p = the least
// with A <= 448 * 2^(p - 127), or the block's own where that is larger and the block was begun by an
// earlier call, then code = x * 2^(127 - p) to the nearest.  Where the power of a begun block grows,
// its other codes are rounded to the new one: a division by a power of two, so no mantissa changes
// but of numbers that leave the normal range.
//
// HBM bounds it: 8192 rows of 8 heads of 128 fp16, 50 MB, 11.9 us (4.2 TB/s); launch and latency few
// rows: 16 rows 6.4 us a call, 3.8 of them the kernel's, 840 FP32 rows of 12 heads of 64 6.4 and 5.6.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "cdna4.h"
#include "e4m3.h"

namespace {

using namespace cdna4;

struct StoreDivs { FastDiv block, blocks; };       // positions of a block, blocks of a page

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T e[N]; };

// The largest number that the type's own values can be read back as (fp16 61440: 65504 would be
// rounded to 65536).
template <typename T> constexpr float kMostStored = sizeof(T) == 2 ? 61440.0f : 0x1.ep127f;

// The largest size among a piece's values, by their bits: n of them, and whether all are finite.
template <int N> __device__ __forceinline__ float largest(const Pack<_Float16, N>& x, bool& finite) {
    typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
    us2_t m = {0, 0};
    if constexpr (N > 1) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const us2_t b = __builtin_bit_cast(us2_t, h2_t{x.e[i], x.e[i + 1]}) & us2_t{0x7fff, 0x7fff};
            m = __builtin_elementwise_max(m, b);
        }
    } else {
        m[0] = __builtin_bit_cast(unsigned short, x.e[0]) & 0x7fff;
    }
    const unsigned short most = m[0] > m[1] ? m[0] : m[1];
    finite &= most < 0x7c00;
    return (float)__builtin_bit_cast(_Float16, most);
}
template <int N> __device__ __forceinline__ float largest(const Pack<float, N>& x, bool& finite) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; i++) m = max(m, __float_as_uint(x.e[i]) & 0x7fffffffu);
    finite &= m < 0x7f800000u;
    return __uint_as_float(m);
}

// x at its power, in reach of the codes.
__device__ __forceinline__ float to_code(float x, int shift, float most) {
    const float y = __builtin_amdgcn_fmed3f(ldexpf(x, shift), -most, most);
    return __builtin_fabsf(x) < INFINITY ? y : NAN;
}
__device__ __forceinline__ float finite_size(float x) {
    const float s = __builtin_fabsf(x);
    return s < INFINITY ? s : 0.0f;
}

// A wave's run of len rows, whose slots the lanes 0 .. len - 1 hold: rows t .. t + len - 1, or with HOLES
// t + `off` of those lanes.
struct Run {
    int64_t t;
    int len;
    int off;
    uint8_t* cells;        // the block's first position
    int slot0;             // ... and its slot
};

// VEC elements of 16 bytes a lane, d / VEC = 2^k lanes a row, KEEP steps of rows in registers; VEC = 1:
// any shape, all lanes on one row.
template <typename T, int VEC, int KEEP, bool HOLES>
__device__ __forceinline__ void store_run(const cf_page_store_q8_args_t& a, const Run& run, int slot, const T* rows,
                                          uint8_t* power) {
    constexpr bool WIDE = VEC > 1;
    const int lane = threadIdx.x & 63;
    const int per_row = WIDE ? a.d / VEC : 64, at_once = 64 / per_row;
    const int sub = WIDE ? lane / per_row : 0, e0 = (lane % per_row) * VEC, step_e = WIDE ? a.d : 64;
    typedef Pack<T, VEC> pack_t;
    const int old = *power;
    auto row_at = [&](int r) {                     // (by all lanes)
        const int i = min(r, run.len - 1);
        return rows + (run.t + (HOLES ? __shfl(run.off, i) : i)) * a.kv_stride;
    };
    auto load = [&](const T* row, int e) { return *(const pack_t*)(row + e); };
    pack_t kept[KEEP];
    float most = 0.0f;
    bool finite = true;
    if constexpr (WIDE) {
#pragma unroll
        for (int s = 0; s < KEEP; s++)
            if (s * at_once < run.len) kept[s] = load(row_at(s * at_once + sub), e0);
#pragma unroll
        for (int s = 0; s < KEEP; s++)
            if (s * at_once < run.len) most = fmaxf(most, largest(kept[s], finite));
    }
    for (int r = WIDE ? KEEP * at_once : 0; r < run.len; r += at_once) {
        const T* const row = row_at(r + sub);
        for (int e = e0; e < a.d; e += step_e) most = fmaxf(most, largest(load(row, e), finite));
    }
    finite = !__builtin_amdgcn_ballot_w64(!finite);
    if (!finite) {                                 // once more, without what is infinite or NaN
        most = 0.0f;
        for (int r = 0; r < run.len; r += at_once) {
            const T* const row = row_at(r + sub);
            for (int e = e0; e < a.d; e += step_e) {
                const pack_t x = load(row, e);
#pragma unroll
                for (int i = 0; i < VEC; i++) most = fmaxf(most, finite_size((float)x.e[i]));
            }
        }
    }
    const int need = power_for(wave_max(most));
    const bool mine = lane < run.len;
    const bool begun = __builtin_amdgcn_ballot_w64(mine && slot == run.slot0) != 0;
    const int now = begun ? need : max(old, need);
    if (lane == 0) *power = (uint8_t)now;
    if (now > old && !begun) {
        // Positions that the run writes: a bit each.
        uint32_t lo = mine && slot - run.slot0 < 32 ? 1u << (slot - run.slot0) : 0u;
        uint32_t hi = mine && slot - run.slot0 >= 32 ? 1u << (slot - run.slot0 - 32) : 0u;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            lo |= __shfl_xor(lo, m);
            hi |= __shfl_xor(hi, m);
        }
        const uint64_t written = (uint64_t)hi << 32 | lo;
        const float by = power_bits(max(127 + old - now, 1));     // 448 * 2^-126 is no code any more
        for (int r = sub; r < a.block; r += at_once) {
            if ((written >> r) & 1) continue;
            for (int e = e0; e < a.d; e += step_e) {
                uint8_t* const cell = run.cells + (int64_t)r * a.row_stride + e;
                if constexpr (WIDE) {
                    Pack<uint32_t, VEC / 4> c = *(const Pack<uint32_t, VEC / 4>*)cell;
#pragma unroll
                    for (int i = 0; i < VEC / 4; i++) {
                        const f2_t x = codes_f32<false>(c.e[i], by), y = codes_f32<true>(c.e[i], by);
                        c.e[i] = codes_of<true>(codes_of<false>(0, x[0], x[1]), y[0], y[1]);
                    }
                    *(Pack<uint32_t, VEC / 4>*)cell = c;
                } else {
                    *cell = (uint8_t)codes_of<false>(0, codes_f32<false>(*cell, by)[0], 0.0f);
                }
            }
        }
    }
    // Where no code can pass 448 or the type's largest number, as almost always, one instruction does.
    const float limit = fminf(448.0f, ldexpf(kMostStored<T>, 127 - now)), over = power_bits(now);
    auto place = [&](int r) { return run.cells + (int64_t)(__shfl(slot, min(r, run.len - 1)) - run.slot0) * a.row_stride; };
    auto put = [&](int r, uint8_t* cell, const pack_t& x) {
        if (r >= run.len) return;
        if constexpr (WIDE) {
            Pack<uint32_t, VEC / 4> c;
#pragma unroll
            for (int i = 0; i < VEC / 4; i++) {
                if (limit == 448.0f) {
                    typedef T two_t __attribute__((ext_vector_type(2)));
                    const s2_t w = codes_over<false>(s2_t{0, 0}, two_t{x.e[4 * i], x.e[4 * i + 1]}, over);
                    c.e[i] = __builtin_bit_cast(uint32_t, codes_over<true>(w, two_t{x.e[4 * i + 2], x.e[4 * i + 3]}, over));
                } else {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = to_code((float)x.e[4 * i + j], 127 - now, limit);
                    c.e[i] = codes_of<true>(codes_of<false>(0, y[0], y[1]), y[2], y[3]);
                }
            }
            *(Pack<uint32_t, VEC / 4>*)cell = c;
        } else {
            *cell = (uint8_t)codes_of<false>(0, to_code((float)x.e[0], 127 - now, limit), 0.0f);
        }
    };
    if constexpr (WIDE)
#pragma unroll
        for (int s = 0; s < KEEP; s++)
            if (s * at_once < run.len) put(s * at_once + sub, place(s * at_once + sub) + e0, kept[s]);
    for (int r = WIDE ? KEEP * at_once : 0; r < run.len; r += at_once) {
        uint8_t* const cell = place(r + sub);      // (by all lanes)
        const T* const row = row_at(r + sub);
        for (int e = e0; e < a.d; e += step_e) put(r + sub, cell + e, load(row, e));
    }
}

// Workgroup (x, y): of the runs that begin in its 64 rows every 2^log_per-th, of heads 4 y .. 4 y + 3 of
// K's and V's, a wave each.  Which workgroup takes the first goes round with the rows: workgroups at a
// distance of a power of two share an XCD, or a part of one, and so would a long sequence's runs (8192 rows
// of 4, blocks of 64: 15.2 us, 29 without; 2048 of one 9.2 and 16.6).
constexpr int kStoreWaves = 4, kStoreRows = 64;
template <typename T, int VEC, int KEEP>
__global__ __launch_bounds__(64 * kStoreWaves)
void page_store_q8(cf_page_store_q8_args_t a, StoreDivs dv, int log_per, int64_t row0) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int unit = (int)blockIdx.y * kStoreWaves + wave;
    if (unit >= 2 * a.H_kv) return;
    const int which = unit >= a.H_kv, h = unit - (which ? a.H_kv : 0);
    const int part = (int)blockIdx.x >> log_per, sub = (int)blockIdx.x & ((1 << log_per) - 1);
    const int64_t t0 = row0 + (int64_t)part * kStoreRows;
    auto slot_at = [&](int64_t t) { return t >= 0 && t < a.T ? a.slots[t] : -1; };
    const int slot = slot_at(t0 + lane), next = slot_at(t0 + kStoreRows + lane), last = slot_at(t0 - kStoreRows + lane);
    auto block_of = [&](int s) { return (unsigned)s < (unsigned)a.num_slots ? fastdiv(s, dv.block) : -1; };
    const int block = block_of(slot), last_block = block_of(last);
    // The block of the stored row before this one, of those less than 64 rows before it.
    const uint64_t lower = (1ull << lane) - 1, stored = __builtin_amdgcn_ballot_w64(block >= 0) & lower;
    const uint64_t last_stored = __builtin_amdgcn_ballot_w64(last_block >= 0);
    const int last_lane = last_stored ? 63 - __builtin_clzll(last_stored) : 0;
    const int up = __shfl(block, stored ? 63 - __builtin_clzll(stored) : 0);
    const int before = stored ? up : last_lane > lane ? __builtin_amdgcn_readlane(last_block, last_lane) : -1;
    const uint64_t all = __builtin_amdgcn_ballot_w64(block >= 0 && block != before);
    const int rank = __builtin_popcountll(all & lower);
    uint64_t heads = __builtin_amdgcn_ballot_w64((all >> lane & 1) && ((rank + part + (part >> 2) - sub) & ((1 << log_per) - 1)) == 0);
    const T* const rows = (const T*)(which ? a.v : a.k) + (int64_t)h * a.d;
    uint8_t* const pages = which ? a.v_pages : a.k_pages;
    uint8_t* const powers = which ? a.v_scales : a.k_scales;
    // The run that begins at lane `first`: its rows, a bit each of the 64 from there, and this lane's slot among them.
    auto find = [&](int first, Run& run, int& its_slot, uint8_t*& power) {
        const int b = __builtin_amdgcn_readlane(block, first);
        const int here = __shfl(slot, (first + lane) & 63), behind = __shfl(next, (first + lane) & 63);
        its_slot = first + lane < 64 ? here : behind;
        const int its_block = block_of(its_slot);
        const uint64_t others = __builtin_amdgcn_ballot_w64(its_block >= 0 && its_block != b);
        const uint64_t its_rows = __builtin_amdgcn_ballot_w64(its_block == b) & ((others & -others) - 1);   // before another block's
        run.t = t0 + first;
        run.len = __builtin_popcountll(its_rows);
        run.slot0 = b * a.block;
        const int page = fastdiv(b, dv.blocks);
        run.cells = pages + (int64_t)page * a.page_stride + (int64_t)(run.slot0 - page * a.page_size) * a.row_stride +
                    (int64_t)h * a.head_stride;
        power = powers + (int64_t)b * a.H_kv + h;
        return its_rows;
    };
    uint64_t with_holes = 0;
    for (; heads; heads &= heads - 1) {
        Run run;
        int its_slot;
        uint8_t* power;
        const uint64_t its_rows = find(__builtin_ctzll(heads), run, its_slot, power);
        if (its_rows & (its_rows + 1)) with_holes |= heads & -heads;
        else store_run<T, VEC, KEEP, false>(a, run, its_slot, rows, power);
    }
    for (; with_holes; with_holes &= with_holes - 1) {        // rare: few registers
        Run run;
        int its_slot;
        uint8_t* power;
        const uint64_t its_rows = find(__builtin_ctzll(with_holes), run, its_slot, power);
        // Its rows to the lanes 0 .. len - 1, the others behind them.
        const int among = __builtin_popcountll(its_rows & lower);
        const int to = its_rows >> lane & 1 ? among : run.len + lane - among;
        run.off = __builtin_amdgcn_ds_permute(4 * to, lane);
        store_run<T, VEC, 1, true>(a, run, __shfl(its_slot, run.off), rows, power);
    }
}

template <typename T>
int launch_store(const cf_page_store_q8_args_t& a, hipStream_t st) {
    constexpr int kWide = 16 / sizeof(T);
    const uint64_t in = (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)a.kv_stride * sizeof(T);
    const uint64_t out = (uint64_t)(uintptr_t)a.k_pages | (uint64_t)(uintptr_t)a.v_pages | (uint64_t)a.page_stride |
                         (uint64_t)a.row_stride | (uint64_t)a.head_stride;
    const int per_row = a.d / kWide;
    const bool wide = in % 16 == 0 && out % kWide == 0 && a.d % kWide == 0 && per_row <= 64 && (per_row & (per_row - 1)) == 0;
    const StoreDivs dv = {fastdiv_make(a.block), fastdiv_make(a.page_size / a.block)};
    const unsigned parts = (unsigned)((2 * (int64_t)a.H_kv + kStoreWaves - 1) / kStoreWaves);
    // Each run that a wave takes costs it 1 us, one after the other, and workgroups that find none a little
    // too: for few rows a workgroup for each, for more as few as keep a thousand, at least two (8 heads of 128
    // fp16, us of the kernel with at most 640, 1024 and 1536: 1024 sequences of one row 12.2, 9.8, 9.8; 1000
    // rows of 2 sequences 5.0, 5.8, 5.8; 300 rows of one 4.9, 5.0, 5.5.  8192 rows of 4 with two 11.7, with
    // four 13.0).
    int log_per = 6;
    while (log_per > 1 && ((int64_t)a.T * parts << log_per) > kStoreRows * 1024) log_per--;
    constexpr int64_t kMost = 1 << 17;             // parts of 64 rows of a launch: a grid has less than 2^32 threads
    for (int64_t t0 = 0; t0 < a.T; t0 += kMost * kStoreRows) {
        const int64_t n = (a.T - t0 + kStoreRows - 1) / kStoreRows;
        const dim3 grid((unsigned)((n < kMost ? n : kMost) << log_per), parts), block(64 * kStoreWaves);
        if (wide && a.block * per_row <= 8 * 64) hipLaunchKernelGGL((page_store_q8<T, kWide, 8>), grid, block, 0, st, a, dv, log_per, t0);
        else if (wide) hipLaunchKernelGGL((page_store_q8<T, kWide, 16>), grid, block, 0, st, a, dv, log_per, t0);
        else hipLaunchKernelGGL((page_store_q8<T, 1, 1>), grid, block, 0, st, a, dv, log_per, t0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return 0;
}

}  // namespace

extern "C" int cf_launch_page_store_q8(const cf_page_store_q8_args_t* a, void* stream) {
    if (a->T <= 0 || a->d <= 0 || a->H_kv <= 0 || a->block <= 0 || a->block > CF_Q8_MAX_BLOCK || a->page_size % a->block != 0)
        return (int)hipErrorInvalidValue;
    return a->elem == CF_ELEM_F16 ? launch_store<_Float16>(*a, (hipStream_t)stream)
                                  : launch_store<float>(*a, (hipStream_t)stream);
}
