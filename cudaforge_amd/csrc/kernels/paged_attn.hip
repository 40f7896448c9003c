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

// ---- On the matrix cores: d = 64 or 128, pages of a multiple of 16 positions ----
//
// The n rows of a sequence times the G query heads of a KV head are one list of n G rows
// (row R: token R / G, head R % G), cut into tiles; a tile reads each K and V row once for
// all its rows.  A unit of work is (tile, range of key blocks, KV head).  Lengths are known
// to the device only, so every wave works out the units from them: with `ranges` the ranges
// that fill the chip, C = ceil(sum_b tiles_b blocks_b / ranges) is the most blocks of one
// range and sequence b's tiles are cut into ns_b = ceil(blocks_b / C) ranges each.  A tile
// in one range is finished by its unit; else the units leave m, l and the unnormalised sum
// per row, and paged_merge joins them.  More than one range needs blocks_b > C, so
// ns_b < 2 blocks_b / C and there are at most 2 ranges + 1 such units per KV head.

struct PagedPlan {
    float*  records;       // of the units of cut tiles
    int32_t max_records;   // per KV head
    int32_t ranges;        // key ranges (per KV head) that fill the chip
    int32_t min_blocks;    // no range is cut shorter
    int32_t waves;         // units in flight: the step of the unit loop
    int32_t merge_groups;  // workgroups that share the rows of a tile's merge
    FastDiv by_page, by_group;
};

// A unit's tile and range, or the tile to merge.
struct Unit {
    SeqRows s;
    int b, tile, range, n_ranges, record;   // record: of its first range (cut tiles)
};

// The tiles' geometry, one sequence per lane and 64 at a time.  TM rows per tile, BK
// positions per key block.
template <int TM, int BK>
struct Geometry {
    const cf_paged_attn_args_t& a;
    const PagedPlan& pl;
    int G, lane, C;
    SeqRows first;                       // lane: sequence `lane`, kept for the second pass

    __device__ __forceinline__ SeqRows rows(int b) const { return b < a.B ? seq_rows(a, b) : SeqRows{0, 0, 0}; }
    __device__ __forceinline__ int tiles(const SeqRows& s) const { return (int)(((int64_t)s.n * G + TM - 1) / TM); }
    __device__ __forceinline__ int blocks(const SeqRows& s) const { return (s.len + BK - 1) / BK; }

    __device__ __forceinline__ Geometry(const cf_paged_attn_args_t& a_, const PagedPlan& pl_) : a(a_), pl(pl_) {
        lane = threadIdx.x & 63;
        G = a.H_q / a.H_kv;
        first = rows(lane);
        float w = (float)tiles(first) * (float)blocks(first);
        for (int b = 64; b < a.B; b += 64) {
            const SeqRows s = rows(b + lane);
            w += (float)tiles(s) * (float)blocks(s);
        }
        w = ceilf(wave_sum(w) / (float)pl.ranges);
        C = __builtin_amdgcn_readfirstlane((int)fminf(fmaxf(w, (float)pl.min_blocks), 1e9f));
    }
    // Item u of all units (MERGE: of all cut tiles); false where there is none.
    template <bool MERGE>
    __device__ __forceinline__ bool find(int u, Unit& out) const {
        int items0 = 0, records0 = 0;
        SeqRows s = first;
        for (int base = 0; base < a.B; base += 64) {
            if (base > 0) s = rows(base + lane);
            const int t = tiles(s), ns = max((blocks(s) + C - 1) / C, 1);
            const int items = MERGE ? (ns > 1 ? t : 0) : t * ns;
            const int before = items0 + wave_excl_sum(items, lane);
            const int rec = ns > 1 ? t * ns : 0;
            const int rec_before = records0 + wave_excl_sum(rec, lane);
            const unsigned long long hit = __ballot(before <= u && u < before + items);
            if (hit) {
                const int src = __builtin_ctzll(hit);
                const int at = u - __builtin_amdgcn_readlane(before, src);
                out.n_ranges = __builtin_amdgcn_readlane(ns, src);
                const int nt = __builtin_amdgcn_readlane(t, src);
                const int i = MERGE ? at : at / out.n_ranges;
                out.range = MERGE ? 0 : at - i * out.n_ranges;
                out.tile = nt - 1 - i;                         // the longest first
                out.record = __builtin_amdgcn_readlane(rec_before, src) + out.tile * out.n_ranges;
                out.b = base + src;
                out.s.row0 = __builtin_amdgcn_readlane(s.row0, src);
                out.s.n = __builtin_amdgcn_readlane(s.n, src);
                out.s.len = __builtin_amdgcn_readlane(s.len, src);
                return out.n_ranges == 1 || out.record + out.n_ranges <= pl.max_records;
            }
            items0 = __builtin_amdgcn_readlane(before + items, 63);
            records0 = __builtin_amdgcn_readlane(rec_before + rec, 63);
        }
        return false;
    }
};

// Record of one unit: [m (TM)] [l (TM)] [sum (TM, D)], m in the log2 domain.
template <int TM, int D> constexpr size_t record_floats() { return (size_t)TM * (D + 2); }

// LDS rows are swizzled in 16-byte chunks: K (and Q) rows are read 16 rows at one chunk, V
// rows transposed (fp16, ds_read_b64_tr_b16) or 4 rows of 16 floats (fp32).
template <typename T, int D> __device__ __forceinline__ int kswz(int row) {
    return sizeof(T) == 4 || D == 128 ? row & 15 : (row >> 1) & 7;
}
template <typename T, int D> __device__ __forceinline__ int vswz(int row) {
    return sizeof(T) == 4 ? row & 15 : D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

// SHARED: a workgroup of 4 waves, 16 NJ rows each, through one ring of 64-position blocks
// (wave w loads positions 16 w .. 16 w + 15 of each).  Else a wave per unit, up to 16 rows,
// with a ring of its own and no barrier: the units of neighbouring KV heads in one workgroup,
// which read the same cache rows at about the same time.
template <typename T, int D, int NJ, bool SHARED> struct Shape {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int WAVES = 4;
    static constexpr int TM = SHARED ? 64 * NJ : 16;
    static constexpr int BK = SHARED ? 64 : F16 ? 32 : 16;
    static constexpr int NG = BK / 16;                        // 16-position groups of a block
    static constexpr int TILE = BK * D;                       // elements of K (or V) per stage
    static constexpr int NS = SHARED && F16 && D == 64 ? 3 : 2;
    static constexpr int RINGS = SHARED ? 1 : WAVES;
    static constexpr int LDS_ELEMS = RINGS * NS * 2 * TILE;
    // Workgroups per CU by LDS (160 KB), which is waves per SIMD.
    static constexpr int PER_CU = 160 * 1024 / (LDS_ELEMS * (int)sizeof(T)) > 2 && NJ == 2 ? 2
                                : 160 * 1024 / (LDS_ELEMS * (int)sizeof(T));
};

template <typename T, int D, int NJ, bool SHARED>
__global__ __launch_bounds__(256, (Shape<T, D, NJ, SHARED>::PER_CU))
void paged_tiles(cf_paged_attn_args_t a, PagedPlan pl) {
    using S = Shape<T, D, NJ, SHARED>;
    constexpr bool F16 = S::F16;
    constexpr int TM = S::TM, BK = S::BK, NG = S::NG, TILE = S::TILE, NS = S::NS;
    constexpr int CE = 16 / sizeof(T);            // elements per 16-byte chunk
    constexpr int CPR = D / CE;                   // chunks per row
    constexpr int RPI = 64 / CPR;                 // rows per DMA instruction (1 KB)
    constexpr int NI = 16 / RPI;                  // DMA instructions per 16 rows
    constexpr int MYG = SHARED ? 1 : NG;          // groups this wave loads
    constexpr int NL = 2 * MYG * NI;              // DMA instructions per wave and block
    constexpr int NF = F16 ? D / 32 : D / 16;     // chunks of a K row a lane takes
    constexpr int UT = D / 16;                    // 16-dim tiles of O^T
    constexpr uint64_t FULL = BK == 64 ? ~0ull : (1ull << (BK & 63)) - 1;
    static_assert((NS - 1) * NL < 64, "vmcnt range");
    __shared__ __attribute__((aligned(16))) T ring_all[S::LDS_ELEMS];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 15, lq = lane >> 4;
    T* const ring = ring_all + (SHARED ? 0 : wave * NS * 2 * TILE);
    const int G = a.H_q / a.H_kv;
    const Geometry<TM, BK> geo(a, pl);
    const float c = a.scale * kLog2e;

    // DMA offsets: lane L of instruction u writes physical chunk L % CPR of row RPI u + L / CPR
    // of a 16-row group, which holds logical chunk (L % CPR) ^ swizzle.
    const int drow = lane / CPR, dch = lane % CPR;
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int u = 0; u < NI; u++) {
        const int row = RPI * u + drow;
        koff[u] = (uint32_t)(row * (uint32_t)a.row_stride + CE * (dch ^ kswz<T, D>(row))) * (uint32_t)sizeof(T);
        voff[u] = (uint32_t)(row * (uint32_t)a.row_stride + CE * (dch ^ vswz<T, D>(row))) * (uint32_t)sizeof(T);
    }
    const uint32_t ring_base = __builtin_amdgcn_readfirstlane(lds_offset(ring));
    // LDS read offsets (elements) inside a stage.
    int k_rd[NF];                                 // + 16 t D for key tile t
#pragma unroll
    for (int f = 0; f < NF; f++) k_rd[f] = lr * D + CE * ((F16 ? 4 * f + lq : NF * lq + f) ^ kswz<T, D>(lr));
    int v_rd[F16 ? UT : 4];
    if constexpr (F16) {
        // ds_read_tr4: lane addresses key 4 lq + lr / 4, dims 16 u + 4 (lr % 4) .. + 3.
#pragma unroll
        for (int u = 0; u < UT; u++) {
            const int row = 4 * lq + (lr >> 2), col = 16 * u + 4 * (lr & 3);
            v_rd[u] = TILE + row * D + 8 * ((col >> 3) ^ vswz<T, D>(row)) + (col & 7);
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < 4; kk++) v_rd[kk] = TILE + (4 * lq + kk) * D + (lr & 3);
    }

    for (int unit = SHARED ? (int)blockIdx.x : (int)blockIdx.x * S::WAVES + wave;; unit += pl.waves) {
        const int range_id = unit / a.H_kv, kvh = unit - range_id * a.H_kv;
        Unit un;
        if (!geo.template find<false>(range_id, un)) break;
        const int n_rows = min(un.s.n * G - un.tile * TM, TM);
        const int R0 = un.tile * TM;
        // Row R sees positions below base + R / G; the tile's last row the most.
        const int base = un.s.len - un.s.n + 1;
        const int limit = min(max(base + fastdiv(R0 + n_rows - 1, pl.by_group), 0), un.s.len);
        const int all_blocks = (limit + BK - 1) / BK;
        const int per = (all_blocks + un.n_ranges - 1) / un.n_ranges;
        const int kb0 = min(un.range * per, all_blocks), nblk = min(kb0 + per, all_blocks) - kb0;

        const int wrow = SHARED ? 16 * NJ * wave : 0;             // this wave's first row of the tile
        const bool active = wrow < n_rows;
        int seen[NJ];                                             // positions the lane's row sees
#pragma unroll
        for (int j = 0; j < NJ; j++)
            seen[j] = min(base + fastdiv(R0 + min(wrow + 16 * j + lr, n_rows - 1), pl.by_group), un.s.len);
        const int seen_all = min(base + fastdiv(R0 + wrow, pl.by_group), un.s.len);   // every row of the wave

        typedef const int32_t __attribute__((address_space(4)))* const_i32;
        const const_i32 table = (const_i32)(uintptr_t)(a.table + (size_t)un.b * a.max_pages);
        const T* const kp = (const T*)a.k + (int64_t)kvh * a.head_stride;
        const T* const vp = (const T*)a.v + (int64_t)kvh * a.head_stride;
        int pages[NG];                                            // of the next block to issue
        auto fetch = [&](int blk) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const int key = (kb0 + blk) * BK + 16 * g;
                pages[g] = table[min(fastdiv(key, pl.by_page), a.max_pages - 1)];
            }
        };
        uint64_t mask[NS];                                        // per stage: positions that count
        auto issue = [&](int blk, auto stage_c) {
            constexpr int stage = decltype(stage_c)::value;
            uint64_t mk = 0;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const int key = (kb0 + blk) * BK + 16 * g;
                const bool valid = (unsigned)pages[g] < (unsigned)a.num_pages;
                const int count = valid ? min(max(limit - key, 0), 16) : 0;
                mk |= (uint64_t)((1u << count) - 1u) << (16 * g);
                if (!SHARED || g == wave) {
                    const int in_page = key - fastdiv(key, pl.by_page) * a.page_size;
                    const int64_t at = (int64_t)(valid ? pages[g] : 0) * a.page_stride + (int64_t)in_page * a.row_stride;
                    const uint32_t lds = ring_base + (uint32_t)((stage * 2 * TILE + 16 * g * D) * sizeof(T));
#pragma unroll
                    for (int u = 0; u < NI; u++) {
                        lds_dma16_s(koff[u], kp + at, lds + u * 1024u);
                        lds_dma16_s(voff[u], vp + at, lds + (uint32_t)(TILE * sizeof(T)) + u * 1024u);
                    }
                }
            }
            mask[stage] = mk;
        };

        f4_t acc[NJ][UT];
        float m_run[NJ], l_run[NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            m_run[j] = -INFINITY;
            l_run[j] = 0.0f;
#pragma unroll
            for (int u = 0; u < UT; u++) acc[j][u] = f4_t{0.f, 0.f, 0.f, 0.f};
        }

        if (nblk > 0) {
            // Q rows by DMA into the last stage, which the first blocks leave free.
            fetch(0);
            {
                constexpr int QI = (SHARED ? 16 * NJ : 16) / RPI;
                const uint32_t qlds = ring_base + (uint32_t)(((NS - 1) * 2 * TILE + wrow * D) * sizeof(T));
#pragma unroll
                for (int u = 0; u < QI; u++) {
                    const int row = min(wrow + RPI * u + drow, n_rows - 1);
                    const int tok = fastdiv(R0 + row, pl.by_group), h = kvh * G + (R0 + row - tok * G);
                    lds_dma16((const T*)a.q + (int64_t)(un.s.row0 + tok) * a.q_stride + h * D +
                                  CE * (dch ^ kswz<T, D>(RPI * u + drow)),
                              __builtin_amdgcn_readfirstlane(qlds + u * 1024u));
                }
            }
            issue(0, std::integral_constant<int, 0>{});
            if constexpr (NS > 2)
                if (1 < nblk) {
                    fetch(1);
                    issue(1, std::integral_constant<int, 1>{});
                }
            if (nblk >= NS) fetch(NS - 1);
            if (NS > 2 && nblk >= 2) wait_vm<(NS - 1) * NL>();
            else wait_vm<NL>();
            // B operand Q^T: fp16 lane (lr, lq) holds Q[row][32 f + 8 lq .. + 7]; fp32 lane holds
            // Q[row][D / 4 lq + 4 f .. + 3], k-slot lq of step s being dim D / 4 lq + s.
            typedef T chunk_t __attribute__((ext_vector_type(CE)));
            chunk_t qf[NJ][NF];
            const T* const qs = ring + (NS - 1) * 2 * TILE + wrow * D;
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int f = 0; f < NF; f++) qf[j][f] = *(const chunk_t*)(qs + 16 * j * D + k_rd[f]);
            wait_lds_reads();

            auto step = [&](int bi, auto stage_c) {
                constexpr int stage = decltype(stage_c)::value;
                constexpr int next = (stage + NS - 1) % NS;
                if constexpr (!SHARED) {
                    if (bi + NS - 1 < nblk) {
                        wait_lds_reads();                         // the last reads of that stage
                        issue(bi + NS - 1, std::integral_constant<int, next>{});
                        if (bi + NS < nblk) fetch(bi + NS);
                    }
                    wait_ahead<NL, NS - 1>(min(NS - 1, nblk - 1 - bi));
                } else {
                    wait_ahead<NL, NS - 2>(nblk - 1 - bi);
                }
                const uint64_t mk = mask[stage];
                const T* const st = ring + stage * 2 * TILE;
                if (mk != FULL) {
                    // V where nothing counts: 0, as p = 0 times whatever it holds need not be.
#pragma unroll
                    for (int g = 0; g < NG; g++)
                        if (!SHARED || g == wave)
#pragma unroll
                            for (int u = 0; u < NI; u++) {
                                const int row = 16 * g + RPI * u + drow;
                                if (!((mk >> row) & 1)) *(uint4*)(ring + stage * 2 * TILE + TILE + row * D + CE * dch) = uint4{};
                            }
                    wait_lds_reads();
                }
                if constexpr (SHARED) {
                    ring_barrier();
                    if (bi + NS - 1 < nblk) {
                        issue(bi + NS - 1, std::integral_constant<int, next>{});
                        if (bi + NS < nblk) fetch(bi + NS);
                    }
                }
                if (!active) return;
                const int k0 = (kb0 + bi) * BK;
                // S^T: sc[j][t][i] = score(key k0 + 16 t + 4 lq + i, row j).
                f4_t sc[NJ][NG];
#pragma unroll
                for (int t = 0; t < NG; t++) {
#pragma unroll
                    for (int j = 0; j < NJ; j++) sc[j][t] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int f = 0; f < NF; f++) {
                        const chunk_t kf = *(const chunk_t*)(st + 16 * t * D + k_rd[f]);
#pragma unroll
                        for (int j = 0; j < NJ; j++) {
                            if constexpr (F16) {
                                sc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[j][f], sc[j][t], 0, 0, 0);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    sc[j][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[j][f][e], sc[j][t], 0, 0, 0);
                            }
                        }
                    }
                }
                const bool edge = mk != FULL || k0 + BK > seen_all;
                _Float16 ph[NJ][4 * NG], pl16[SHARED ? 1 : NJ][4 * NG];
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    if (edge) {
#pragma unroll
                        for (int t = 0; t < NG; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int key = 16 * t + 4 * lq + i;
                                if (!((mk >> key) & 1) || k0 + key >= seen[j]) sc[j][t][i] = -INFINITY;
                            }
                    }
                    float mloc = fmaxf(fmaxf(sc[j][0][0], sc[j][0][1]), fmaxf(sc[j][0][2], sc[j][0][3]));
#pragma unroll
                    for (int t = 1; t < NG; t++)
                        mloc = fmaxf(mloc, fmaxf(fmaxf(sc[j][t][0], sc[j][t][1]), fmaxf(sc[j][t][2], sc[j][t][3])));
                    mloc = max_xor32(max_xor16(mloc)) * c;        // -inf if the row sees nothing here
                    // The maximum moves only when a block exceeds it by more than 2^kLazy.
                    constexpr float kLazy = 8.0f;
                    if (__builtin_amdgcn_ballot_w64(mloc > m_run[j] + kLazy)) {
                        const float m_new = mloc > m_run[j] + kLazy ? mloc : m_run[j];
                        const float alpha = __builtin_amdgcn_exp2f(m_run[j] - (m_new == -INFINITY ? 0.0f : m_new));
                        m_run[j] = m_new;
                        l_run[j] *= alpha;
#pragma unroll
                        for (int u = 0; u < UT; u++) acc[j][u] *= alpha;
                    }
                    const float m_use = m_run[j] == -INFINITY ? 0.0f : m_run[j];
                    float psum = 0.0f;
#pragma unroll
                    for (int t = 0; t < NG; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][t][i], c, -m_use));
                            psum += p;
                            if constexpr (F16) {
                                ph[j][4 * t + i] = (_Float16)p;
                                if constexpr (!SHARED) pl16[j][4 * t + i] = (_Float16)(p - (float)ph[j][4 * t + i]);
                            } else {
                                sc[j][t][i] = p;
                            }
                        }
                    l_run[j] += psum;
                }
                // O^T += V^T P^T.  fp16: in 32-key step s, k-slot e of lane group lq is key
                // 32 s + 16 (e / 4) + 4 lq + e % 4; fp32: in step kk of key tile t, key 16 t + 4 lq + kk:
                // the lane's own scores either way.
                if constexpr (F16) {
#pragma unroll
                    for (int s2 = 0; s2 < NG / 2; s2++) {
                        h8_t pf[NJ], pr[SHARED ? 1 : NJ];
#pragma unroll
                        for (int j = 0; j < NJ; j++)
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                pf[j][e] = ph[j][8 * s2 + e];
                                if constexpr (!SHARED) pr[j][e] = pl16[j][8 * s2 + e];
                            }
#pragma unroll
                        for (int u = 0; u < UT; u++) {
                            const h8_t vf = cat8(ds_read_tr4((const _Float16*)st + v_rd[u] + 32 * s2 * D),
                                                 ds_read_tr4((const _Float16*)st + v_rd[u] + (32 * s2 + 16) * D));
#pragma unroll
                            for (int j = 0; j < NJ; j++) {
                                // A wave of its own waits on memory, not on products: p as two fp16 numbers.
                                if constexpr (!SHARED)
                                    acc[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pr[j], acc[j][u], 0, 0, 0);
                                acc[j][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[j], acc[j][u], 0, 0, 0);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NG; t++)
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
#pragma unroll
                            for (int u = 0; u < UT; u++) {
                                const float vf = st[v_rd[kk] + 16 * t * D + 4 * ((4 * u + (lr >> 2)) ^ vswz<T, D>(4 * lq + kk))];
#pragma unroll
                                for (int j = 0; j < NJ; j++)
                                    acc[j][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, sc[j][t][kk], acc[j][u], 0, 0, 0);
                            }
                }
            };
            for_each_stage<NS>(nblk, step);
        }

        // Lane (lr, lq) holds dims 16 u + 4 lq .. + 3 of row lr.
        if (active) {
            float* const rec = un.n_ranges > 1
                ? pl.records + ((size_t)(un.record + un.range) * a.H_kv + kvh) * record_floats<TM, D>() : nullptr;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int row = wrow + 16 * j + lr;
                const float l = add_xor32(add_xor16(l_run[j]));
                if (row >= n_rows) continue;
                if (rec) {
#pragma unroll
                    for (int u = 0; u < UT; u++) *(f4_t*)(rec + 2 * TM + row * D + 16 * u + 4 * lq) = acc[j][u];
                    if (lq == 0) {
                        rec[row] = m_run[j];
                        rec[TM + row] = l;
                    }
                    continue;
                }
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int tok = fastdiv(R0 + row, pl.by_group), h = kvh * G + (R0 + row - tok * G);
                T* const o = (T*)a.o + ((int64_t)(un.s.row0 + tok) * a.H_q + h) * D + 4 * lq;
#pragma unroll
                for (int u = 0; u < UT; u++) {
                    typedef T four_t __attribute__((ext_vector_type(4)));
                    *(four_t*)(o + 16 * u) = four_t{(T)(acc[j][u][0] * inv), (T)(acc[j][u][1] * inv), (T)(acc[j][u][2] * inv),
                                                    (T)(acc[j][u][3] * inv)};
                }
            }
        }
        if constexpr (SHARED) ring_barrier();                     // the ring's reads, before the next unit's Q
    }
}

// Joins the ranges of cut tiles: O = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.  A
// workgroup per (tile, KV head) and ROWS rows: 256 / ROWS threads per row, D / 4 of them side
// by side over the dims, the rest sharing the ranges.
template <typename T, int D, int TM, int BK, int ROWS>
__global__ __launch_bounds__(256)
void paged_merge(cf_paged_attn_args_t a, PagedPlan pl) {
    constexpr int DL = D / 4, SUBS = 256 / ROWS / DL;      // lanes over the dims, shares of the ranges
    static_assert(SUBS >= 1, "rows per workgroup");
    __shared__ float ml[2][ROWS][SUBS];
    __shared__ f4_t part[SUBS > 1 ? SUBS * ROWS * DL : 1];
    const Geometry<TM, BK> geo(a, pl);
    const int G = a.H_q / a.H_kv;
    const int d4 = threadIdx.x % DL, sub = threadIdx.x / DL % SUBS, r = threadIdx.x / (DL * SUBS);
    for (int unit = blockIdx.x;; unit += gridDim.x) {
        const int th = unit / pl.merge_groups, group = unit - th * pl.merge_groups;
        const int tile_id = th / a.H_kv, kvh = th - tile_id * a.H_kv;
        Unit un;
        if (!geo.template find<true>(tile_id, un)) break;
        const int n_rows = min(un.s.n * G - un.tile * TM, TM);
        const float* const rec = pl.records + ((size_t)un.record * a.H_kv + kvh) * record_floats<TM, D>();
        const size_t step = (size_t)a.H_kv * record_floats<TM, D>();
        for (int row0 = group * ROWS; row0 < n_rows; row0 += pl.merge_groups * ROWS) {   // uniform
            const int row = row0 + r;
            float m = -INFINITY, l = 0.0f;
            f4_t acc = f4_t{0.f, 0.f, 0.f, 0.f};
            if (row < n_rows)
                for (int s = sub; s < un.n_ranges; s += SUBS) {
                    const float ms = rec[s * step + row], ls = rec[s * step + TM + row];
                    const f4_t as = *(const f4_t*)(rec + s * step + 2 * TM + row * D + 4 * d4);
                    const float m_new = fmaxf(m, ms), m_use = m_new == -INFINITY ? 0.0f : m_new;
                    const float wa = __builtin_amdgcn_exp2f(m - m_use), wb = __builtin_amdgcn_exp2f(ms - m_use);
                    m = m_new;
                    l = l * wa + ls * wb;
                    acc = acc * wa + as * wb;
                }
            if constexpr (SUBS > 1) {
                part[threadIdx.x] = acc;
                if (d4 == 0) {
                    ml[0][r][sub] = m;
                    ml[1][r][sub] = l;
                }
                __syncthreads();
                if (sub == 0) {
                    float M = m;
                    for (int k = 1; k < SUBS; k++) M = fmaxf(M, ml[0][r][k]);
                    const float m_use = M == -INFINITY ? 0.0f : M;
                    const float w0 = __builtin_amdgcn_exp2f(m - m_use);
                    l *= w0;
                    acc *= w0;
                    for (int k = 1; k < SUBS; k++) {
                        const float w = __builtin_amdgcn_exp2f(ml[0][r][k] - m_use);
                        l += ml[1][r][k] * w;
                        acc += part[threadIdx.x + k * DL] * w;
                    }
                }
                __syncthreads();
            }
            if (sub == 0 && row < n_rows) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int R = un.tile * TM + row, tok = fastdiv(R, pl.by_group), h = kvh * G + (R - tok * G);
                typedef T four_t __attribute__((ext_vector_type(4)));
                *(four_t*)((T*)a.o + ((int64_t)(un.s.row0 + tok) * a.H_q + h) * D + 4 * d4) =
                    four_t{(T)(acc[0] * inv), (T)(acc[1] * inv), (T)(acc[2] * inv), (T)(acc[3] * inv)};
            }
        }
    }
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

// The plan of a call on the matrix cores: the kernel's form and how its work is cut.
struct Plan {
    PagedPlan pl;
    int  nj;              // 0: a wave per unit (16-row tiles), 1 or 2: workgroups of 64 or 128 rows
    int  wgs, merge_wgs;
    size_t bytes;         // workspace
};

bool fast_ok(const cf_paged_attn_args_t& a) {
    const uint64_t ptrs = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)(uintptr_t)a.o;
    const uint64_t steps = (uint64_t)a.q_stride | (uint64_t)a.page_stride | (uint64_t)a.row_stride | (uint64_t)a.head_stride;
    const uint64_t es = a.elem == CF_ELEM_F16 ? 2 : 4;
    // Row numbers times the group stay in 31 bits, offsets inside a group of rows in 32.
    return (a.d == 64 || a.d == 128) && a.page_size % 16 == 0 && ptrs % 16 == 0 && steps * es % 16 == 0 && a.scale > 0.0f &&
           (int64_t)a.T * (a.H_q / a.H_kv) <= (1 << 30) && (uint64_t)a.row_stride * es * 16 < (1ull << 32);
}

Plan make_plan(const cf_paged_attn_args_t& a) {
    Plan p;
    const int64_t G = a.H_q / a.H_kv, cus = cu_count();
    const bool f16 = a.elem == CF_ELEM_F16;
    if ((int64_t)a.max_new * G <= 16) p.nj = 0;
    else p.nj = f16 && ((int64_t)a.T * G + 127) / 128 * a.H_kv >= 2 * cus ? 2 : 1;
    const int64_t TM = p.nj == 0 ? 16 : 64 * p.nj, BK = p.nj > 0 ? 64 : f16 ? 32 : 16;
    // Units in flight: a workgroup of four waves takes 128 KB (d = 128) or 64 KB of LDS without
    // shared tiles; with them 64 KB, 48 KB or (fp32, d = 128) 128 KB.
    const int64_t per_cu = p.nj == 0 ? (a.d == 128 ? 4 : 8) : (!f16 && a.d == 128) ? 1 : 2;
    const int64_t slots = cus * per_cu;
    const int64_t fill = slots / a.H_kv > 0 ? slots / a.H_kv : 1;
    // Tiles of the call, at most (where max_new holds).
    int64_t tiles = (int64_t)a.T * G / TM + (a.B < a.T ? a.B : a.T);
    if ((int64_t)a.max_new * G <= TM && tiles > a.B) tiles = a.B;
    int64_t ranges = fill;
    if (p.nj == 0) ranges = tiles <= fill / 2 ? fill - tiles : tiles <= fill ? 2 * fill - tiles : 2 * fill;
    p.pl.ranges = (int32_t)(ranges > 0 ? ranges : 1);
    p.pl.min_blocks = (int32_t)(256 / BK);
    p.pl.max_records = 2 * p.pl.ranges + 8;
    const int64_t most_blocks = ((int64_t)a.max_pages * a.page_size + BK - 1) / BK;
    const bool cut = most_blocks > p.pl.min_blocks;
    p.bytes = cut ? (size_t)p.pl.max_records * a.H_kv * (TM * (a.d + 2)) * sizeof(float) : 0;
    int64_t units = (tiles + (cut ? ranges : 0)) * a.H_kv;
    if (units > (1 << 24)) units = 1 << 24;
    p.wgs = (int)(p.nj == 0 ? (units + 3) / 4 : units);
    p.pl.waves = p.nj == 0 ? 4 * p.wgs : p.wgs;
    const int64_t cut_tiles = tiles < ranges + 4 ? tiles : ranges + 4;
    const int64_t most_rows = (int64_t)a.max_new * G < TM ? (int64_t)a.max_new * G : TM;
    p.pl.merge_groups = (int32_t)(p.nj == 0 ? most_rows : (most_rows + 3) / 4);
    const int64_t merge_wgs = cut_tiles * a.H_kv * p.pl.merge_groups;
    p.merge_wgs = !cut ? 0 : merge_wgs > (1 << 20) ? 1 << 20 : (int)merge_wgs;
    p.pl.by_page = fastdiv_make(a.page_size);
    p.pl.by_group = fastdiv_make((int)G);
    p.pl.records = nullptr;
    return p;
}

template <typename T, int D>
int launch_tiles(const cf_paged_attn_args_t& a, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)p.wgs), block(256);
    if (p.nj == 0) hipLaunchKernelGGL((paged_tiles<T, D, 1, false>), grid, block, 0, st, a, p.pl);
    else if (p.nj == 1) hipLaunchKernelGGL((paged_tiles<T, D, 1, true>), grid, block, 0, st, a, p.pl);
    // fp32 products take 16 times as long as fp16's: 16 rows a wave keep the matrix cores busy.
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((paged_tiles<T, D, 2, true>), grid, block, 0, st, a, p.pl);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.merge_wgs == 0) return (int)e;
    const dim3 mgrid((unsigned)p.merge_wgs);
    constexpr int BK0 = Shape<T, D, 1, false>::BK;
    if (p.nj == 0) hipLaunchKernelGGL((paged_merge<T, D, 16, BK0, 1>), mgrid, block, 0, st, a, p.pl);
    else if (p.nj == 1) hipLaunchKernelGGL((paged_merge<T, D, 64, 64, 4>), mgrid, block, 0, st, a, p.pl);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((paged_merge<T, D, 128, 64, 4>), mgrid, block, 0, st, a, p.pl);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" size_t cf_paged_attn_bytes(const cf_paged_attn_args_t* a) { return fast_ok(*a) ? make_plan(*a).bytes : 0; }

extern "C" int cf_launch_paged_attn(const cf_paged_attn_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    if (a->B <= 0 || a->T <= 0 || a->d <= 0 || a->d > 64 * kAnyDims || a->H_kv <= 0 || a->H_q % a->H_kv != 0)
        return (int)hipErrorInvalidValue;
    if (fast_ok(*a)) {
        Plan p = make_plan(*a);
        if (p.bytes > 0 && !a->records) return (int)hipErrorInvalidValue;
        p.pl.records = a->records;
        if (a->elem == CF_ELEM_F16)
            return a->d == 64 ? launch_tiles<_Float16, 64>(*a, p, st) : launch_tiles<_Float16, 128>(*a, p, st);
        return a->d == 64 ? launch_tiles<float, 64>(*a, p, st) : launch_tiles<float, 128>(*a, p, st);
    }
    const FastDiv by_page = fastdiv_make(a->page_size);
    const int64_t wgs = ((int64_t)a->T * a->H_q + 3) / 4;
    if (wgs > 0x7fffffff) return (int)hipErrorInvalidValue;
    if (a->elem == CF_ELEM_F16) hipLaunchKernelGGL(paged_any<_Float16>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    else hipLaunchKernelGGL(paged_any<float>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    return (int)hipGetLastError();
}
