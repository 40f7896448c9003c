// paged_attn.hip — attention of chunks of new tokens over a paged KV cache (gfx950).
//
// Row i of the n_b new rows of sequence b is position p = L_b - n_b + i of its L_b, and
//   O = sum_{j <= p} softmax_j(scale * q . k_j) v_j
// over the positions of valid pages (position j: page table[b][j / P], row j % P).  Softmax
// in one pass: running maximum m and sum l in FP32, everything rescaled by 2^(m_old - m)
// when the maximum moves; scores are kept in the log2 domain.
//
// Times below are of one call among others on one MI355X; "n rows over m" is n new tokens of
// a sequence of m positions in all, and heads are 32 of 128 over 8 KV heads where none are named.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_tiles.h"

namespace {

// ---- One row of one head by a wave, 64 positions at a time: lanes are positions for the
// scores and dims (at most 64 DIMS) for the sum over V.  Of positions [key0, key1); into O, or into a
// record whose m, l and sum for this row start at rec, rec + tm and rec_sum. ----
template <typename T, int DIMS>
__device__ __forceinline__ void plain_row(const cf_paged_attn_args_t& a, FastDiv by_page, const SeqRows& s, int b, int tok,
                                          int h, int d, int key0 = 0, int key1 = INT32_MAX, float* rec = nullptr, int tm = 0,
                                          float* rec_sum = nullptr) {
    const int lane = threadIdx.x & 63;
    const int seen = min(min(s.len - s.n + tok + 1, s.len), key1);
    const int32_t* const table = a.table + (size_t)b * a.max_pages;
    const T* const q = (const T*)a.q + (int64_t)(s.row0 + tok) * a.q_stride + (int64_t)h * d;
    const T* const k = (const T*)a.k + (int64_t)(h / (a.H_q / a.H_kv)) * a.head_stride;
    const T* const v = (const T*)a.v + (int64_t)(h / (a.H_q / a.H_kv)) * a.head_stride;
    const float c = a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f, acc[DIMS];
#pragma unroll
    for (int i = 0; i < DIMS; i++) acc[i] = 0.0f;
#pragma clang loop unroll(disable)
    for (uint32_t at0 = (uint32_t)key0; at0 < (uint32_t)max(seen, 0); at0 += 64) {    // unsigned: up to 2^31 positions
        const int k0 = (int)at0, key = k0 + lane;
        int64_t at = 0;
        float x = -INFINITY;
        if (key < seen) {
            const int idx = fastdiv(key, by_page);
            const int page = table[idx];
            if ((unsigned)page < (unsigned)a.num_pages) {
                at = (int64_t)page * a.page_stride + (int64_t)(key - idx * a.page_size) * a.row_stride;
                float dot = 0.0f;
#pragma clang loop unroll(disable)
                for (int e = 0; e < d; e++) dot = __builtin_fmaf((float)q[e], (float)k[at + e], dot);
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
#pragma unroll
            for (int i = 0; i < DIMS; i++)
                if (lane + 64 * i < d) acc[i] = __builtin_fmaf(pj, (float)v[row + lane + 64 * i], acc[i]);
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
    T* const o = (T*)a.o + ((int64_t)(s.row0 + tok) * a.H_q + h) * d;
#pragma unroll
    for (int i = 0; i < DIMS; i++)
        if (lane + 64 * i < d) o[lane + 64 * i] = (T)(acc[i] * inv);
}

// Which of some V are infinite (up, down) or NaN: a bit for each element of the lane's chunk.
struct Odd {
    uint32_t up = 0, down = 0, nan = 0;
    __device__ __forceinline__ uint32_t any() const { return up | down | nan; }
};
template <typename T, int D>
__device__ __forceinline__ void find_odd(const cf_paged_attn_args_t& a, FastDiv by_page, int b, int kvh, int from, int to, Odd& odd) {
    using R = Rows<T, D>;
    constexpr int U = 8;                                     // rows under way per lane
    constexpr uint32_t kExp = R::F16 ? 0x7c007c00u : 0x7f800000u, kOne = R::F16 ? 0x04000400u : 0x00800000u;
    constexpr uint32_t kCarry = R::F16 ? 0x80008000u : 0x80000000u;      // an exponent of ones carries into the sign
    const int lane = threadIdx.x & 63, sub = lane / R::CPR;
    const int32_t* const table = a.table + (size_t)b * a.max_pages;
    const T* const v = (const T*)a.v + (int64_t)kvh * a.head_stride + R::CE * (lane % R::CPR);
    Odd mine;
#pragma clang loop unroll(disable)
    for (int p0 = from; p0 < to; p0 += 64) {
        const int key = min(p0 + lane, to - 1), idx = fastdiv(key, by_page), page = table[idx];
        const bool valid = (unsigned)page < (unsigned)a.num_pages;
        const int64_t at = valid ? (int64_t)page * a.page_stride + (int64_t)(key - idx * a.page_size) * a.row_stride : -1;
        auto chunk = [&](int r) {
            const int64_t row = (int64_t)((uint64_t)(uint32_t)__shfl((int)(at >> 32), r) << 32 | (uint32_t)__shfl((int)at, r));
            return row < 0 ? uint4{} : *(const uint4*)(v + row);
        };
#pragma clang loop unroll(disable)
        for (int r0 = sub; r0 < 64; r0 += U * R::RPI) {
            uint4 x[U];
#pragma unroll
            for (int u = 0; u < U; u++) x[u] = chunk(r0 + u * R::RPI);
            uint32_t hit = 0;
#pragma unroll
            for (int u = 0; u < U; u++)
                hit |= ((x[u].x & kExp) + kOne) | ((x[u].y & kExp) + kOne) | ((x[u].z & kExp) + kOne) | ((x[u].w & kExp) + kOne);
            if (!__builtin_amdgcn_ballot_w64((hit & kCarry) != 0)) continue;
#pragma clang loop unroll(disable)
            for (int u = 0; u < U; u++) {
                const typename R::chunk_t c = __builtin_bit_cast(typename R::chunk_t, chunk(r0 + u * R::RPI));
#pragma unroll
                for (int e = 0; e < R::CE; e++) {
                    const float f = (float)c[e];
                    mine.nan |= f != f ? 1u << e : 0u;
                    mine.up |= f == INFINITY ? 1u << e : 0u;
                    mine.down |= f == -INFINITY ? 1u << e : 0u;
                }
            }
        }
    }
#pragma unroll
    for (int step = R::CPR; step < 64; step *= 2) {
        mine.up |= __shfl_xor(mine.up, step);
        mine.down |= __shfl_xor(mine.down, step);
        mine.nan |= __shfl_xor(mine.nan, step);
    }
    odd.up |= mine.up;
    odd.down |= mine.down;
    odd.nan |= mine.nan;
}

// Rows row0 + bit of a unit (a bit of `rows` each), computed and stored by this wave, where they are
// spoilt.  An element is what the V that its row sees make of it: infinite or NaN.  Where these are
// finite and only a hidden one is not, the row is computed again by the plain loop; hidden positions
// are a tile's own tokens, so that ends with the call that brings such V.  The V are read once for all
// rows, but for the tile's tokens (512 rows over 2048, a NaN among the cached V: 225 us, without it 51,
// with every such row by the plain loop 20000; 16 decode rows over 4000 each 105, 50 and 2070).
template <typename T, int D, int TM>
__device__ __forceinline__ void mend_rows(const cf_paged_attn_args_t& a, const PagedPlan& pl, const Unit& un, int kvh,
                                          const Work& w, int row0, uint32_t rows) {
    using R = Rows<T, D>;
    const int lane = threadIdx.x & 63;
    wait_vm<0>();                                             // what it stored is stored
    Odd seen;
    int upto = w.key0;
    for (; rows; rows &= rows - 1) {
        const int row = row0 + __builtin_ctz(rows);
        const RowAt at = row_at(pl, pl.G, kvh, w.R0 + row);
        const int sees = max(min(min(w.base + at.tok, un.s.len), w.key1), upto);     // rises with the rows
        find_odd<T, D>(a, pl.by_page, un.b, kvh, upto, sees, seen);
        upto = sees;
        Odd hidden;
        find_odd<T, D>(a, pl.by_page, un.b, kvh, sees, w.key1, hidden);
        float* const rec = un.n_ranges > 1 ? record_of<TM, D>(a, pl, un, kvh) : nullptr;
        T* const o = (T*)a.o + ((int64_t)(un.s.row0 + at.tok) * a.H_q + at.h) * D;
        if (__builtin_amdgcn_ballot_w64((hidden.any() & ~seen.any()) != 0)) {
            plain_row<T, D / 64>(a, pl.by_page, un.s, un.b, at.tok, at.h, D, w.key0, w.key1, rec ? rec + row : nullptr, TM,
                                 rec + 2 * TM + row * D);
            continue;
        }
        if (lane >= R::CPR) continue;
#pragma unroll
        for (int e = 0; e < R::CE; e++) {
            if (!((seen.any() >> e) & 1)) continue;
            const bool up = (seen.up >> e) & 1, down = (seen.down >> e) & 1;
            const float x = ((seen.nan >> e) & 1) || (up && down) ? NAN : up ? INFINITY : -INFINITY;
            if (rec) rec[2 * TM + row * D + R::CE * lane + e] = x;
            else o[R::CE * lane + e] = (T)x;
        }
    }
}

// ---- Up to 16 rows, one wave with a ring of its own: no barrier. ----
template <typename T, int D, int BK_> struct Narrow {
    static constexpr int BK = BK_, NS = 2;
    static constexpr int TILE = BK * D;
    static constexpr int RING = NS * 2 * TILE;               // elements
};

// Positions [key0, key1) (key0 a multiple of 16) of (b, kvh) for the unit's rows: leaves m and
// the lane's share of l, and lane (lr, lq) with dims 16 u + 4 lq .. + 3 of row lr.
template <typename T, int D, int BK>
__device__ __forceinline__ void narrow_range(const cf_paged_attn_args_t& a, const PagedPlan& pl, T* ring, const SeqRows& s,
                                             int b, int kvh, const Work& w, int key0, int key1,
                                             f4_t (&acc)[D / 16], float& m_run, float& l_run) {
    using R = Rows<T, D>;
    using N = Narrow<T, D, BK>;
    typedef typename R::chunk_t chunk_t;
    constexpr bool F16 = R::F16;
    constexpr int NG = BK / 16, NS = N::NS, TILE = N::TILE, NI = R::NI, NL = 2 * NG * NI, UT = R::UT, CE = R::CE;
    constexpr uint64_t FULL = (1ull << BK) - 1;
    static_assert(NS * NL < 64, "vmcnt range");
    const int lane = unit_lane(), lr = lane & 15;
    const int G = pl.G;
    const int drow = R::drow(lane), dch = R::dch(lane);
#pragma unroll
    for (int u = 0; u < UT; u++) acc[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = 0.0f;
    LongSum l;
    const int nblk = key1 > key0 ? (key1 - key0 + BK - 1) / BK : 0;
    if (nblk == 0) return;
    const float c = a.scale * kLog2e;
    const int seen = min(w.base + fastdiv(w.R0 + min(lr, w.n_rows - 1), pl.by_group), s.len);
    const int seen_all = min(w.base + fastdiv(w.R0, pl.by_group), s.len);

    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int u = 0; u < NI; u++) {
        const int row = R::RPI * u + drow;
        koff[u] = ((uint32_t)row * (uint32_t)a.row_stride + CE * (dch ^ kswz<T, D>(row))) * (uint32_t)sizeof(T);
        voff[u] = ((uint32_t)row * (uint32_t)a.row_stride + CE * (dch ^ vswz<T, D>(row))) * (uint32_t)sizeof(T);
    }
    int k_rd[R::NF], v_rd[R::VR];
    R::k_offsets(k_rd, lane);
    R::v_offsets(v_rd, lane);
    const uint32_t ring_base = __builtin_amdgcn_readfirstlane(lds_offset(ring));
    const T* const kp = (const T*)a.k + (int64_t)kvh * a.head_stride;
    const T* const vp = (const T*)a.v + (int64_t)kvh * a.head_stride;
    Groups groups = {a.table + (size_t)b * a.max_pages, 0, 0, 0, 0};
    groups.load(a, pl, 0, key0, key1);

    uint64_t mask[NS];                                        // per stage: positions that count
    auto issue = [&](int blk, auto stage_c) {
        constexpr int stage = decltype(stage_c)::value;
        if (blk > 0 && blk % (64 / NG) == 0) groups.load(a, pl, blk * NG, key0, key1);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int64_t at = groups.at(blk * NG + g);
            const uint32_t lds = ring_base + (uint32_t)((stage * 2 * TILE + 16 * g * D) * sizeof(T));
#pragma unroll
            for (int u = 0; u < NI; u++) {
                lds_dma16_s(koff[u], kp + at, lds + u * 1024u);
                lds_dma16_s(voff[u], vp + at, lds + (uint32_t)(TILE * sizeof(T)) + u * 1024u);
            }
        }
        mask[stage] = groups.template masks<NG>(blk * NG);
    };

    wait_lds_reads();                                         // what the ring held before
    // Q rows by DMA into the last stage, which the first blocks leave free.
    {
        const uint32_t qlds = ring_base + (uint32_t)((NS - 1) * 2 * TILE * sizeof(T));
#pragma unroll
        for (int u = 0; u < NI; u++) {
            const int row = R::RPI * u + drow;
            const RowAt at = row_at(pl, G, kvh, w.R0 + min(row, w.n_rows - 1));
            lds_dma16((const T*)a.q + (int64_t)(s.row0 + at.tok) * a.q_stride + at.h * D + CE * (dch ^ kswz<T, D>(row)),
                      __builtin_amdgcn_readfirstlane(qlds + u * 1024u));
        }
    }
    issue(0, std::integral_constant<int, 0>{});
    wait_vm<NL>();
    chunk_t qf[R::NF];                                        // B operand Q^T
#pragma unroll
    for (int f = 0; f < R::NF; f++) qf[f] = *(const chunk_t*)(ring + (NS - 1) * 2 * TILE + k_rd[f]);
    wait_lds_reads();

    auto step = [&](int bi, auto stage_c) {
        constexpr int stage = decltype(stage_c)::value;
        if (bi + NS - 1 < nblk) {
            wait_lds_reads();                                 // the last reads of that stage
            issue(bi + NS - 1, std::integral_constant<int, (stage + NS - 1) % NS>{});
        }
        wait_ahead<NL, NS - 1>(min(NS - 1, nblk - 1 - bi));
        const uint64_t mk = mask[stage];
        T* const st = ring + stage * 2 * TILE;
        if (mk != FULL) {
            // V where nothing counts: 0, as p = 0 times whatever it holds need not be.
#pragma unroll
            for (int u = 0; u < NG * NI; u++) {
                const int row = R::RPI * u + drow;
                if (!((mk >> row) & 1)) *(uint4*)(st + TILE + row * D + CE * dch) = uint4{};
            }
            wait_lds_reads();
        }
        const int k0 = key0 + bi * BK;
        // S^T: sc[t][i] = score(key k0 + 16 t + 4 lq + i, row lr).
        f4_t sc[NG];
#pragma unroll
        for (int t = 0; t < NG; t++) {
            sc[t] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < R::NF; f++) {
                const chunk_t kf = *(const chunk_t*)(st + 16 * t * D + k_rd[f]);
                if constexpr (F16) {
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[f], sc[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[f][e], sc[t], 0, 0, 0);
                }
            }
        }
        if (mk != FULL || k0 + BK > seen_all) {
            hide(sc, mk, seen - k0, lane);
        }
        float mloc = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
        for (int t = 1; t < NG; t++) mloc = fmaxf(mloc, fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])));
        mloc = low_max<T>(max_xor32(max_xor16(mloc)), c);         // -inf if the row sees nothing here
        float alpha;
        if (move_max<T>(mloc, m_run, alpha)) {
            l.scale(alpha);
#pragma unroll
            for (int u = 0; u < UT; u++) acc[u] *= alpha;
        }
        const float m_use = m_run == -INFINITY ? 0.0f : m_run;
        _Float16 hi[F16 ? 4 * NG : 1], lo[F16 ? 4 * NG : 1];
        float l_blk = 0.0f;
#pragma unroll
        for (int t = 0; t < NG; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], c, -m_use));
                l_blk += p;
                if constexpr (F16) {
                    hi[4 * t + i] = (_Float16)p;
                    lo[4 * t + i] = (_Float16)(p - (float)hi[4 * t + i]);
                } else {
                    sc[t][i] = p;
                }
            }
        l.add(l_blk);
        // O^T += V^T P^T, the lane's own scores being its B operand.  This wave waits on memory,
        // not on products: p as the sum of two fp16 numbers, so that its rounding (2^-11 of it,
        // otherwise as large as the result's own) leaves the result.
        if constexpr (F16 && NG == 2) {
            const h8_t pf = {hi[0], hi[1], hi[2], hi[3], hi[4], hi[5], hi[6], hi[7]};
            const h8_t pr = {lo[0], lo[1], lo[2], lo[3], lo[4], lo[5], lo[6], lo[7]};
#pragma unroll
            for (int u = 0; u < UT; u++) {
                const _Float16* const v = (const _Float16*)st + TILE + v_rd[u];
                const h8_t vf = cat8(ds_read_tr4(v), ds_read_tr4(v + 16 * D));
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pr, acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf, acc[u], 0, 0, 0);
            }
        } else if constexpr (F16) {
            // Both parts of 16 positions in one 32-k MFMA, V twice.
            const h8_t pf = {hi[0], hi[1], hi[2], hi[3], lo[0], lo[1], lo[2], lo[3]};
#pragma unroll
            for (int u = 0; u < UT; u++) {
                const h4_t v = ds_read_tr4((const _Float16*)st + TILE + v_rd[u]);
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cat8(v, v), pf, acc[u], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int t = 0; t < NG; t++)
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
#pragma unroll
                    for (int u = 0; u < UT; u++)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(R::v_at((const float*)st + TILE, v_rd, lane, t, kk, u),
                                                                      sc[t][kk], acc[u], 0, 0, 0);
        }
    };
    for_each_stage<NS>(nblk, step);
    l_run = l.sum();
}

// A wave per unit, the units of neighbouring KV heads in one workgroup: they read the same
// cache rows at about the same time.  HBM bounds it: with two blocks of 16 KB under way per
// wave and four waves a CU it streams 5.7 TB/s over long caches (64 rows over 8192 each, 2.15 GB:
// 380 us), and 16 sequences of 1778 to 4096 positions (227 MB) take 46 us, 42 of them here, the
// rest the merge.
template <typename T, int D> struct Heads {
    static constexpr int WAVES = 4, BK = sizeof(T) == 2 ? 32 : 16;
    static constexpr int RING = Narrow<T, D, BK>::RING;
    static constexpr int PER_CU = 160 * 1024 / (WAVES * RING * (int)sizeof(T));
};
template <typename T, int D>
__global__ __launch_bounds__(256, (Heads<T, D>::PER_CU))
void paged_heads(cf_paged_attn_args_t a, PagedPlan pl) {
    using H = Heads<T, D>;
    __shared__ __attribute__((aligned(16))) T ring_all[H::WAVES * H::RING];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int G = pl.G;
    const Geometry<16, H::BK, 1> geo(a, pl);
    if (geo.lists_cut_tiles()) return;
    for (int unit = (int)blockIdx.x * H::WAVES + wave;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        const Work w = unit_work<16, H::BK>(a, pl, un);
        const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
        f4_t acc[D / 16];
        float m, l;
        narrow_range<T, D, H::BK>(a, pl, ring_all + wave * H::RING, un.s, un.b, kvh, w, w.key0, w.key1, acc, m, l);
        l = add_xor32(add_xor16(l));
        const uint32_t again = rows_of_16(lr < w.n_rows && spoilt(acc, l));
        if (lr < w.n_rows) {
            if (un.n_ranges > 1) {
                float* const rec = record_of<16, D>(a, pl, un, kvh);
#pragma unroll
                for (int u = 0; u < D / 16; u++) *(f4_t*)(rec + 2 * 16 + lr * D + 16 * u + 4 * lq) = acc[u];
                if (lq == 0) {
                    rec[lr] = m;
                    rec[16 + lr] = l;
                }
            } else {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const RowAt at = row_at(pl, G, kvh, w.R0 + lr);
                T* const o = (T*)a.o + ((int64_t)(un.s.row0 + at.tok) * a.H_q + at.h) * D + 4 * lq;
#pragma unroll
                for (int u = 0; u < D / 16; u++) store4(o + 16 * u, acc[u] * inv);
            }
        }
        if (again) mend_rows<T, D, 16>(a, pl, un, kvh, w, 0, again);
    }
}

// Up to 16 rows by all waves of a workgroup (latency bounds it: fp32, a row of 12 heads of 64 over
// 257, 8.6 us; fp16, 16 rows over 512 each 10.1): each takes a share of the unit's positions, and
// they join their m, l and sums in LDS (WAVES rings at `lds`, one each).  True where rows that
// this wave stored are spoilt.
template <typename T, int D, int TM, int WAVES, int ALL = WAVES>
__device__ __forceinline__ bool narrow_unit(const cf_paged_attn_args_t& a, const PagedPlan& pl, T* lds, const Unit& un,
                                            int kvh, const Work& w) {
    constexpr int RING = Narrow<T, D, 16>::RING, LD = D + 4;
    static_assert(16 * (LD + 2) * 4 <= RING * (int)sizeof(T), "a wave's rows fit its ring");
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (ALL > WAVES && wave >= WAVES) {                       // whose rings the LDS has no room for
        __syncthreads();
        __syncthreads();
        return false;
    }
    T* const ring = lds + wave * RING;
    const int groups = w.key1 > w.key0 ? (w.key1 - w.key0 + 15) / 16 : 0;
    const int per = (groups + WAVES - 1) / WAVES * 16;
    const int k0 = min(w.key0 + wave * per, w.key1), k1 = min(k0 + per, w.key1);
    f4_t acc[D / 16];
    float m, l;
    narrow_range<T, D, 16>(a, pl, ring, un.s, un.b, kvh, w, k0, k1, acc, m, l);
    l = add_xor32(add_xor16(l));
    float* const mine = (float*)ring;                         // [16][LD], m [16], l [16]
    wait_lds_reads();
#pragma unroll
    for (int u = 0; u < D / 16; u++) *(f4_t*)(mine + lr * LD + 16 * u + 4 * lq) = acc[u];
    if (lq == 0) {
        mine[16 * LD + lr] = m;
        mine[16 * LD + 16 + lr] = l;
    }
    __syncthreads();
    bool again = false;
    for (int i = threadIdx.x; i < w.n_rows * (D / 4); i += 64 * WAVES) {
        const int row = i / (D / 4), d4 = i % (D / 4);
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < WAVES; v++) M = fmaxf(M, ((const float*)(lds + v * RING))[16 * LD + row]);
        const float m_use = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        f4_t sum = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < WAVES; v++) {
            const float* const p = (const float*)(lds + v * RING);
            const float x = __builtin_amdgcn_exp2f(p[16 * LD + row] - m_use);
            L += p[16 * LD + 16 + row] * x;
            sum += *(const f4_t*)(p + row * LD + 4 * d4) * x;
        }
        const f4_t one[1] = {sum};
        again |= spoilt(one, L);
        if (un.n_ranges > 1) {
            float* const rec = record_of<TM, D>(a, pl, un, kvh);
            *(f4_t*)(rec + 2 * TM + row * D + 4 * d4) = sum;
            if (d4 == 0) {
                rec[row] = M;
                rec[TM + row] = L;
            }
        } else {
            const RowAt at = row_at(pl, pl.G, kvh, w.R0 + row);
            store4((T*)a.o + ((int64_t)(un.s.row0 + at.tok) * a.H_q + at.h) * D + 4 * d4,
                   sum * (L == 0.0f ? 0.0f : 1.0f / L));
        }
    }
    __syncthreads();                                          // the rings, before the next unit
    return __builtin_amdgcn_ballot_w64(again) != 0;
}

// The rows that the wave stored there.
template <typename T, int D, int TM, int WAVES>
__device__ __forceinline__ void mend_narrow(const cf_paged_attn_args_t& a, const PagedPlan& pl, const Unit& un, int kvh,
                                            const Work& w) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t rows = 0;
    for (int r = 0; r < w.n_rows; r++)
        if (r / (256 / D) % WAVES == wave) rows |= 1u << r;
    mend_rows<T, D, TM>(a, pl, un, kvh, w, 0, rows);
}

template <typename T, int D> struct Split {
    static constexpr int WAVES = sizeof(T) * D > 256 ? 4 : 8;   // 16 or (fp32, d = 128) 32 KB of LDS each
};
template <typename T, int D>
__global__ __launch_bounds__(64 * (Split<T, D>::WAVES), (Split<T, D>::WAVES) / 4)
void paged_split(cf_paged_attn_args_t a, PagedPlan pl) {
    constexpr int WAVES = Split<T, D>::WAVES;
    __shared__ __attribute__((aligned(16))) T lds[WAVES * Narrow<T, D, 16>::RING];
    const Geometry<16, 64, 1, false> geo(a, pl);
    for (int unit = (int)blockIdx.x;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        const Work w = unit_work<16, 64>(a, pl, un);
        if (narrow_unit<T, D, 16, WAVES>(a, pl, lds, un, kvh, w)) mend_narrow<T, D, 16, WAVES>(a, pl, un, kvh, w);
    }
}

// ---- fp16, wide tiles: 8 waves of 16 NJ rows through one ring of 64-position blocks. ----
// Scores and sums cost the matrix cores about what softmax costs the vector unit (d = 128, 32
// rows, 64 positions: 64 MFMAs of 16 clk against ~190 vector instructions of 4 clk and 32
// exponentials of 16), and a wave does one after the other.  So the two waves of a SIMD, w and
// w + 4, take turns: with phases cut by barriers, waves 0 .. 3 run products while waves 4 .. 7
// run softmax, then the other way round.  Products of turn i are S(i) = K_i Q^T and
// O += V_{i-1} P(i-1), so a stage of the ring is K_i with V_{i-1}; with NS stages, NS - 2 of
// them are still under way when one is needed.
// NJ = 2: the matrix cores bound it, at what clock they leave (about 2.1 GHz): 2048 rows over 8192,
// 241 GFLOP in 240 to 260 us (925 to 1000 TFLOP/s; a large library product makes 1097).  NJ = 1
// halves the tile, and a turn takes two thirds of the time (a tile on every CU, over 8192 positions:
// 1.52 us a block for 2.23): each fragment read from LDS feeds one product, so the LDS bounds it with
// the turn's latencies.  Waves of 32 rows that share the positions instead take a fifth longer.
template <int D, int NJ> struct Wide16 {
    static constexpr int TM = 128 * NJ, BK = 64, NS = 4;
    static constexpr int TILE = BK * D;
    static constexpr int STAGE = 2 * TILE;
    static constexpr int LDS = NS * STAGE;                   // 128 KB (d = 128), 64 KB
    static constexpr int MASKS = 2 * NS;                     // blocks whose masks are kept
    static_assert(TM * D <= 2 * STAGE, "Q fits the last two stages");
    static_assert(8 * Narrow<_Float16, D, 16>::RING <= LDS, "the rings of narrow tiles fit");
};

// Returns the wave's rows that are spoilt, a bit each.
template <int D, int NJ>
__device__ __forceinline__ uint32_t wide16_unit(const cf_paged_attn_args_t& a, const PagedPlan& pl, _Float16* lds,
                                            uint64_t* masks, const Unit& un, int kvh, const Work& w) {
    using T = _Float16;
    using R = Rows<T, D>;
    using W = Wide16<D, NJ>;
    constexpr int BK = W::BK, NS = W::NS, TILE = W::TILE, STAGE = W::STAGE, UT = R::UT, NF = R::NF;
    constexpr int HI = R::NI / 2;                            // DMA instructions per 8 rows
    constexpr int NL = 2 * HI;                               // ... of a wave per stage
    static_assert(R::RPI <= 8 && (NS - 1) * NL < 64, "eight rows per wave");
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int G = pl.G, drow = R::drow(lane), dch = R::dch(lane);
    const float c = a.scale * kLog2e;
    const int wrow = 16 * NJ * wave;
    const bool active = wrow < w.n_rows;
    const int n = w.key1 > w.key0 ? (w.key1 - w.key0 + BK - 1) / BK : 0;
    f4_t acc[NJ][UT], lsum[NJ];
    float m_run[NJ];
    int seen[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        m_run[j] = -INFINITY;
        lsum[j] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < UT; u++) acc[j][u] = f4_t{0.f, 0.f, 0.f, 0.f};
        seen[j] = min(w.base + fastdiv(w.R0 + min(wrow + 16 * j + lr, w.n_rows - 1), pl.by_group), un.s.len);
    }
    const int seen_all = min(w.base + fastdiv(w.R0 + min(wrow, w.n_rows - 1), pl.by_group), un.s.len);

    if (n > 0) {
        // This wave's rows of a block: 8 half + 0 .. 7 of group `grp`.
        const int grp = wave >> 1, half = wave & 1;
        uint32_t koff[HI], voff[HI];
#pragma unroll
        for (int u = 0; u < HI; u++) {
            const int row = 8 * half + R::RPI * u + drow;
            koff[u] = ((uint32_t)row * (uint32_t)a.row_stride + 8 * (dch ^ kswz<T, D>(row))) * 2u;
            voff[u] = ((uint32_t)row * (uint32_t)a.row_stride + 8 * (dch ^ vswz<T, D>(row))) * 2u;
        }
        int k_rd[NF], v_rd[UT];
        R::k_offsets(k_rd, lane);
        R::v_offsets(v_rd, lane);
        const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_offset(lds));
        const uint32_t my_lds = lds_base + (uint32_t)((16 * grp + 8 * half) * D * 2);
        const table_t table = table_of(a, un.b);
        const T* const kp = (const T*)a.k + (int64_t)kvh * a.head_stride;
        const T* const vp = (const T*)a.v + (int64_t)kvh * a.head_stride;

        // Stage i of the ring is issued with the page of block i (K) and what is kept of block i - 1
        // (V).  Blocks outside 0 .. n - 1 load the nearest one, so every stage is NL loads.  A wave
        // looks up its own group's page only; which positions of it count goes to the others
        // through LDS.
        int page;
        int64_t v_at = 0;
        auto key_of = [&](int i) { return w.key0 + min(i, n - 1) * BK + 16 * grp; };
        auto fetch = [&](int i) { page = page_of(a, pl, table, key_of(i)); };
        auto issue = [&](int i, int to_slot) {
            const Group gr = group_of(a, pl, page, key_of(i), w.key1);
            if (lane == 0) ((uint16_t*)masks)[4 * (i % W::MASKS) + grp] = (uint16_t)gr.mask;
            if (i == 0) v_at = gr.at;
            const uint32_t to = my_lds + (uint32_t)(to_slot * STAGE * 2);
#pragma unroll
            for (int u = 0; u < HI; u++) {
                lds_dma16_s(koff[u], kp + gr.at, to + u * 1024u);
                lds_dma16_s(voff[u], vp + v_at, to + (uint32_t)(TILE * 2) + u * 1024u);
            }
            v_at = gr.at;
        };

        fetch(0);
        {
            const uint32_t qlds = lds_base + (uint32_t)((2 * STAGE + wrow * D) * 2);
#pragma unroll
            for (int u = 0; u < 16 * NJ / R::RPI; u++) {
                const int row = R::RPI * u + drow;
                const RowAt at = row_at(pl, G, kvh, w.R0 + min(wrow + row, w.n_rows - 1));
                lds_dma16((const T*)a.q + (int64_t)(un.s.row0 + at.tok) * a.q_stride + at.h * D + 8 * (dch ^ kswz<T, D>(row)),
                          __builtin_amdgcn_readfirstlane(qlds + u * 1024u));
            }
        }
        issue(0, 0);
        fetch(1);
        issue(1, 1);                                          // n >= 1: stages 0 and 1 exist
        fetch(2);
        wait_vm<2 * NL>();
        h8_t qf[NJ][NF];
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int f = 0; f < NF; f++) qf[j][f] = *(const h8_t*)(lds + 2 * STAGE + (wrow + 16 * j) * D + k_rd[f]);
        wait_lds_reads();

        f4_t sc[NJ][4];
        h8_t pf[NJ][2];
        h8_t ones = {1, 1, 1, 1, 1, 1, 1, 1};
        asm volatile("" : "+v"(ones));                        // kept in registers for the whole loop
        uint64_t mk = ~0ull;                                  // positions of this turn's block that count
        int slot = 0;                                         // of this turn's stage

        // Before the barrier that starts turn i: its stage has landed, this wave's share of it, and
        // its V (of block i - 1) is 0 where nothing counts (p = 0 times whatever it holds need not be).
        auto landed = [&](int i) {
            wait_ahead<NL, NS - 2>(min(i == 0 ? 1 : NS - 2, n - i));
            if (i > 0 && mk != ~0ull) {
#pragma unroll
                for (int u = 0; u < HI; u++) {
                    const int row = 16 * grp + 8 * half + R::RPI * u + drow;
                    if (!((mk >> row) & 1)) *(uint4*)(lds + slot * STAGE + TILE + row * D + 8 * dch) = uint4{};
                }
            }
            wait_lds_reads();
        };
        // After it: the stage of turn i - 1 is free.
        auto refill = [&](int i) {
            if (i + NS - 1 <= n) issue(i + NS - 1, slot == 0 ? NS - 1 : slot - 1);
        };
        // Fragment x of a turn: x < 2 UT is V^T (32-key step x / UT, dims 16 (x % UT)), the rest K
        // (key tile, then chunk).  They are read kAhead fragments before their products, in
        // exactly this order: left to itself the compiler reads them all first and spills (so does
        // 10 ahead: 252 us for 239).
        constexpr int kAhead = 8, kV = 2 * UT, kAll = kV + 4 * NF;
        auto products = [&](int i, auto first_c, auto last_c) {   // fragments first .. last - 1
            constexpr int first = decltype(first_c)::value, last = decltype(last_c)::value;
            if constexpr (last == kAll) mk = masks[i % W::MASKS];
            if (!active) return;
            const T* const st = lds + slot * STAGE;
            h8_t frag[kAhead];
            auto read = [&](auto x_c) {
                constexpr int x = decltype(x_c)::value;
                if constexpr (x < kV) {
                    const T* const v = st + TILE + v_rd[x % UT] + 32 * (x / UT) * D;
                    frag[x % kAhead] = cat8(ds_read_tr4(v), ds_read_tr4(v + 16 * D));
                } else if constexpr (x < kAll) {
                    frag[x % kAhead] = *(const h8_t*)(st + 16 * ((x - kV) % 4) * D + k_rd[(x - kV) / 4]);
                }
            };
            auto use = [&](auto x_c) {
                constexpr int x = decltype(x_c)::value;
                const h8_t f = frag[x % kAhead];
                // O^T += V^T P^T: in 32-key step s2, k-slot e of lane group lq is key
                // 32 s2 + 16 (e / 4) + 4 lq + e % 4, the lane's own scores.  p is rounded to fp16, the
                // type of V and of the product: 2^-11 of each weight, over thousands of positions together
                // about as much as the result's own rounding (2.9e-4 rms of the values, else 2.1e-4;
                // narrow tiles' second product would be half of all products again).  l comes out of
                // the matrix cores too, from the same rounded p that weights V.
                if constexpr (x < kV) {
                    if constexpr (x % UT == 0)
#pragma unroll
                        for (int j = 0; j < NJ; j++)
                            lsum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[j][x / UT], lsum[j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < NJ; j++)
                        acc[j][x % UT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, pf[j][x / UT], acc[j][x % UT], 0, 0, 0);
                } else {
                    // S^T: sc[j][t][e] = score(key 16 t + 4 lq + e of block i, row j).
                    constexpr int t = (x - kV) % 4, c0 = (x - kV) / 4;
#pragma unroll
                    for (int j = 0; j < NJ; j++)
                        sc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, qf[j][c0], c0 == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : sc[j][t],
                                                                          0, 0, 0);
                }
            };
            __builtin_amdgcn_s_setprio(1);
            static_for<kAhead - 1>([&](auto k) {
                constexpr int x = first + decltype(k)::value;
                if constexpr (x < last) read(std::integral_constant<int, x>{});
            });
            __builtin_amdgcn_sched_barrier(0);
            static_for<last - first>([&](auto k) {
                constexpr int x = first + decltype(k)::value;
                if constexpr (x + kAhead - 1 < last) read(std::integral_constant<int, x + kAhead - 1>{});
                use(std::integral_constant<int, x>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            __builtin_amdgcn_s_setprio(0);
        };
        const std::integral_constant<int, 0> from_v;
        const std::integral_constant<int, kV> to_v;
        const std::integral_constant<int, kAll> to_k;
        auto softmax = [&](int i) {
            if (!active) return;
            const int k0 = w.key0 + i * BK;
            const bool edge = mk != ~0ull || k0 + BK > seen_all;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                if (edge) hide(sc[j], mk, seen[j] - k0, lane);
                // Chains of three-input maxima.
                float mloc = fmaxf(fmaxf(sc[j][0][0], sc[j][0][1]), sc[j][0][2]);
#pragma unroll
                for (int e = 3; e < 15; e += 2)
                    mloc = fmaxf(fmaxf(mloc, sc[j][e >> 2][e & 3]), sc[j][(e + 1) >> 2][(e + 1) & 3]);
                mloc = fmaxf(mloc, sc[j][3][3]);
                mloc = low_max<T>(max_xor32(max_xor16(mloc)), c);  // -inf if the row sees nothing here
                float alpha;
                if (move_max<T>(mloc, m_run[j], alpha)) {
                    lsum[j] *= alpha;
#pragma unroll
                    for (int u = 0; u < UT; u++) acc[j][u] *= alpha;
                }
                const float m_use = m_run[j] == -INFINITY ? 0.0f : m_run[j];
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        pf[j][t >> 1][(t & 1) * 4 + e] =
                            (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][t][e], c, -m_use));
            }
        };
        auto next_turn = [&]() { slot = slot == NS - 1 ? 0 : slot + 1; };
        auto uniform = [](uint64_t x) {
            return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
        };

        // Turn i of waves 0 .. 3 takes phases 2 i (products) and 2 i + 1, of the others 2 i + 1 and
        // 2 i + 2; everybody meets at every barrier, 2 n + 2 of them.  A stage's page is looked up
        // during the softmax before its issue: a load through the scalar cache makes the waits for
        // LDS reads in order wait for everything.
        auto first_half = [&](int i) {
            mk = uniform(mk);
            ring_barrier();
            fetch(i + NS);
            softmax(i);
            next_turn();
            landed(i + 1);
            ring_barrier();
            refill(i + 1);
        };
        auto second_half = [&](int i) {
            mk = uniform(mk);
            next_turn();
            landed(i + 1);
            ring_barrier();
            refill(i + 1);
            fetch(i + NS + 1);
            softmax(i);
            ring_barrier();
        };
        landed(0);
        ring_barrier();
        if (2 <= n) issue(2, 2);
        fetch(3);
        if (3 <= n) issue(3, 3);
        fetch(4);
        if (wave < 4) {
            products(0, to_v, to_k);
            first_half(0);
#pragma clang loop unroll(disable)
            for (int i = 1; i < n; i++) {
                products(i, from_v, to_k);
                first_half(i);
            }
            products(n, from_v, to_v);
            ring_barrier();
        } else {
            ring_barrier();
            products(0, to_v, to_k);
            second_half(0);
#pragma clang loop unroll(disable)
            for (int i = 1; i < n; i++) {
                products(i, from_v, to_k);
                second_half(i);
            }
            products(n, from_v, to_v);
        }
    }
    uint32_t again_all = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int row = wrow + 16 * j + lr;
        const uint32_t again = rows_of_16(row < w.n_rows && spoilt(acc[j], lsum[j][0]));
        if (row < w.n_rows) {
            const RowOut out = row_out<T, D, W::TM>(a, pl, un, kvh, w, row, m_run[j], lsum[j][0], lq == 0);
#pragma unroll
            for (int u = 0; u < UT; u++) put4<T>(out, 16 * u + 4 * lq, acc[j][u]);
        }
        again_all |= again << (16 * j);
    }
    ring_barrier();                                           // the ring's reads, before the next unit
    return again_all;
}

// Blocks of tiles of up to 16 rows that cost a wide tile's one (31 decode rows beside a chunk of 20
// rows: 59 us; with 3 or 6: 62 and 65).
constexpr int kNarrowCost = 4;
template <int D, int NJ>
__global__ __launch_bounds__(512, 2)
void paged_wide16(cf_paged_attn_args_t a, PagedPlan pl) {
    using W = Wide16<D, NJ>;
    __shared__ __attribute__((aligned(1024))) _Float16 lds[W::LDS];
    __shared__ uint64_t masks[W::MASKS];
    __shared__ int kept[3 * 64];
    const Geometry<W::TM, 64, kNarrowCost> geo(a, pl, kept);
    if (geo.lists_cut_tiles()) return;
    for (int unit = (int)blockIdx.x;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        Work w = unit_work<W::TM, 64>(a, pl, un);
        const bool narrow = w.n_rows <= 16;
        const uint32_t again = narrow ? narrow_unit<_Float16, D, W::TM, 8>(a, pl, lds, un, kvh, w)
                                      : wide16_unit<D, NJ>(a, pl, lds, masks, un, kvh, w);
        if (!again) continue;
        if (!geo.find(id, un)) break;         // found anew: nothing is kept for this
        w = unit_work<W::TM, 64>(a, pl, un);
        if (narrow) mend_narrow<_Float16, D, W::TM, 8>(a, pl, un, kvh, w);
        else mend_rows<_Float16, D, W::TM>(a, pl, un, kvh, w, 16 * NJ * __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), again);
    }
}

// ---- fp32, wide tiles: 4 waves of 16 rows, or (d = 128) 8, which share the positions too. ----
// The fp32 MFMA (32 clk, 128 or 256 of them per 64 positions and 16 rows) bounds it; the rest of
// a block (its loads, 64 KB through the L1 in 1000 clk with d = 128, and softmax) has to run
// beside another wave's products.  d = 64: that of a second workgroup of the CU.  d = 128, whose
// ring takes the LDS: waves w and w + 4 of a SIMD have the same rows and half of every block's
// positions each, and join their sums in LDS at the end; w goes first, so that one is in its
// softmax while the other is in its products (200 rows of 32 heads over 1200: 58 us, with 4
// waves 63; d = 64 with 8 waves: 1 us more a unit, and no faster a block).
template <int D> struct Wide32 {
    static constexpr int TM = 64, BK = 64, NS = 2, TILE = BK * D, LDS = NS * 2 * TILE;   // 64 or 128 KB
    static constexpr int KS = D == 128 ? 2 : 1;              // waves that share a row's positions
    static constexpr int WAVES = 4 * KS, PER_CU = D == 64 ? 2 : 1;
};
template <int D>
__device__ __forceinline__ void wide32_unit(const cf_paged_attn_args_t& a, const PagedPlan& pl, float* ring, const Unit& un,
                                            int kvh, const Work& w) {
    using T = float;
    using R = Rows<T, D>;
    using W = Wide32<D>;
    constexpr int BK = W::BK, NS = W::NS, TILE = W::TILE, NI = R::NI, HI = NI / W::KS, NL = 2 * HI, UT = R::UT, NF = R::NF;
    constexpr int NT = 4 / W::KS;                            // tiles of 16 positions of a wave
    static_assert(NS * NL < 64, "vmcnt range");
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), share = wave >> 2;
    const int G = pl.G, drow = R::drow(lane), dch = R::dch(lane);
    const float c = a.scale * kLog2e;
    const int wrow = 16 * (wave & 3);
    const bool active = wrow < w.n_rows;
    const int n = w.key1 > w.key0 ? (w.key1 - w.key0 + BK - 1) / BK : 0;
    const int seen = min(w.base + fastdiv(w.R0 + min(wrow + lr, w.n_rows - 1), pl.by_group), un.s.len);
    const int seen_all = min(w.base + fastdiv(w.R0 + min(wrow, w.n_rows - 1), pl.by_group), un.s.len);
    f4_t acc[UT];
    float m_run = -INFINITY;
    LongSum l_run;
#pragma unroll
    for (int u = 0; u < UT; u++) acc[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
        // This wave loads 16 / KS rows of a block: `first` and on of group `grp`.
        const int grp = wave / W::KS, first = 16 / W::KS * (wave % W::KS);
        uint32_t koff[HI], voff[HI];
#pragma unroll
        for (int u = 0; u < HI; u++) {
            const int row = first + R::RPI * u + drow;
            koff[u] = ((uint32_t)row * (uint32_t)a.row_stride + 4 * (dch ^ kswz<T, D>(row))) * 4u;
            voff[u] = ((uint32_t)row * (uint32_t)a.row_stride + 4 * (dch ^ vswz<T, D>(row))) * 4u;
        }
        int k_rd[NF], v_rd[R::VR];
        R::k_offsets(k_rd, lane);
        R::v_offsets(v_rd, lane);
        const uint32_t ring_base = __builtin_amdgcn_readfirstlane(lds_offset(ring));
        const T* const kp = (const T*)a.k + (int64_t)kvh * a.head_stride;
        const T* const vp = (const T*)a.v + (int64_t)kvh * a.head_stride;
        Groups groups = {a.table + (size_t)un.b * a.max_pages, 0, 0, 0, 0};
        groups.load(a, pl, 0, w.key0, w.key1);
        uint64_t mask[NS];
        auto issue = [&](int i, auto stage_c) {
            constexpr int stage = decltype(stage_c)::value;
            if (i > 0 && i % 16 == 0) groups.load(a, pl, 4 * i, w.key0, w.key1);
            const int64_t at = groups.at(4 * i + grp);
            const uint32_t to = ring_base + (uint32_t)((stage * 2 * TILE + (16 * grp + first) * D) * 4);
#pragma unroll
            for (int u = 0; u < HI; u++) {
                lds_dma16_s(koff[u], kp + at, to + u * 1024u);
                lds_dma16_s(voff[u], vp + at, to + (uint32_t)(TILE * 4) + u * 1024u);
            }
            mask[stage] = groups.template masks<4>(4 * i);
        };
        {
            // (Waves that share rows bring them to the same place.)
            const uint32_t qlds = ring_base + (uint32_t)(((NS - 1) * 2 * TILE + wrow * D) * 4);
#pragma unroll
            for (int u = 0; u < NI; u++) {
                const int row = R::RPI * u + drow;
                const RowAt at = row_at(pl, G, kvh, w.R0 + min(wrow + row, w.n_rows - 1));
                lds_dma16((const T*)a.q + (int64_t)(un.s.row0 + at.tok) * a.q_stride + at.h * D + 4 * (dch ^ kswz<T, D>(row)),
                          __builtin_amdgcn_readfirstlane(qlds + u * 1024u));
            }
        }
        issue(0, std::integral_constant<int, 0>{});
        wait_vm<NL>();
        f4_t qf[NF];
#pragma unroll
        for (int f = 0; f < NF; f++) qf[f] = *(const f4_t*)(ring + (NS - 1) * 2 * TILE + wrow * D + k_rd[f]);
        wait_lds_reads();
        if (W::KS > 1 && share == 0) __builtin_amdgcn_s_setprio(1);
        auto step = [&](int i, auto stage_c) {
            constexpr int stage = decltype(stage_c)::value;
            wait_vm<0>();
            const uint64_t mk = mask[stage];
            if (mk != ~0ull) {
#pragma unroll
                for (int u = 0; u < HI; u++) {
                    const int row = 16 * grp + first + R::RPI * u + drow;
                    if (!((mk >> row) & 1)) *(uint4*)(ring + stage * 2 * TILE + TILE + row * D + 4 * dch) = uint4{};
                }
                wait_lds_reads();
            }
            ring_barrier();
            if (i + 1 < n) issue(i + 1, std::integral_constant<int, (stage + 1) % NS>{});
            if (!active) return;
            const int k0 = w.key0 + i * BK + 16 * NT * share;
            const T* const st = ring + stage * 2 * TILE + 16 * NT * share * D;
            // A dim chunk's fragments are read one or two chunks before their products, in this order;
            // the tiles' chains of sums go side by side (an MFMA that waits for the one before takes 44).
            constexpr int kAhead = 1 + 4 / NT;
            f4_t sc[NT], kf[kAhead][NT];
            auto read_k = [&](auto f_c) {
                constexpr int f = decltype(f_c)::value;
#pragma unroll
                for (int t = 0; t < NT; t++) kf[f % kAhead][t] = *(const f4_t*)(st + 16 * t * D + k_rd[f]);
            };
            static_for<kAhead - 1>(read_k);
            static_for<NF>([&](auto f_c) {
                constexpr int f = decltype(f_c)::value;
                if constexpr (f + kAhead - 1 < NF) read_k(std::integral_constant<int, f + kAhead - 1>{});
                if constexpr (f == 0)
#pragma unroll
                    for (int t = 0; t < NT; t++) sc[t] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[f % kAhead][t][e], qf[f][e], sc[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            });
            if (mk != ~0ull || k0 + 16 * NT > seen_all) hide(sc, mk >> (W::KS > 1 ? 32 * share : 0), seen - k0, lane);
            float mloc = fmaxf(fmaxf(sc[0][0], sc[0][1]), sc[0][2]);
#pragma unroll
            for (int e = 3; e < 4 * NT - 1; e += 2)
                mloc = fmaxf(fmaxf(mloc, sc[e >> 2][e & 3]), sc[(e + 1) >> 2][(e + 1) & 3]);
            mloc = fmaxf(mloc, sc[NT - 1][3]);
            mloc = low_max<T>(max_xor32(max_xor16(mloc)), c);
            float alpha;
            if (move_max<T>(mloc, m_run, alpha)) {
                l_run.scale(alpha);
#pragma unroll
                for (int u = 0; u < UT; u++) acc[u] *= alpha;
            }
            const float m_use = m_run == -INFINITY ? 0.0f : m_run;
            float l_blk = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    sc[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], c, -m_use));
                    l_blk += sc[t][e];
                }
            l_run.add(l_blk);
            // In step kk of key tile t, k-slot lq is key 16 t + 4 lq + kk: the lane's own score.
            float vf[2][UT];
            auto read_v = [&](auto g_c) {
                constexpr int g = decltype(g_c)::value;
#pragma unroll
                for (int u = 0; u < UT; u++) vf[g % 2][u] = R::v_at(st + TILE, v_rd, lane, g / 4, g % 4, u);
            };
            read_v(std::integral_constant<int, 0>{});
            static_for<4 * NT>([&](auto g_c) {
                constexpr int g = decltype(g_c)::value;
                if constexpr (g + 1 < 4 * NT) read_v(std::integral_constant<int, g + 1>{});
#pragma unroll
                for (int u = 0; u < UT; u++)
                    acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[g % 2][u], sc[g / 4][g % 4], acc[u], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        for_each_stage<NS>(n, step);
        if (W::KS > 1) __builtin_amdgcn_s_setprio(0);
    }
    float l = add_xor32(add_xor16(l_run.sum()));
    ring_barrier();                                           // the ring's reads
    if constexpr (W::KS > 1) {
        // The second waves' m, l and sums, through the ring.
        f4_t* const other = (f4_t*)ring + (wave & 3) * (UT + 1) * 64 + lane;
        static_assert(4 * (UT + 1) * 64 * 4 <= W::LDS, "they fit");
        if (share == 1) {
#pragma unroll
            for (int u = 0; u < UT; u++) other[64 * u] = acc[u];
            other[64 * UT] = f4_t{m_run, l, 0.f, 0.f};
            wait_lds_reads();
        }
        ring_barrier();
        if (share == 0) {
            const f4_t ml = other[64 * UT];
            const float M = fmaxf(m_run, ml[0]), m_use = M == -INFINITY ? 0.0f : M;
            const float x0 = __builtin_amdgcn_exp2f(m_run - m_use), x1 = __builtin_amdgcn_exp2f(ml[0] - m_use);
            m_run = M;
            l = l * x0 + ml[1] * x1;
#pragma unroll
            for (int u = 0; u < UT; u++) acc[u] = acc[u] * x0 + other[64 * u] * x1;
        }
        wait_lds_reads();
        ring_barrier();                                       // ... before the next unit
    }
    if (share == 0) {
        const uint32_t again = rows_of_16(wrow + lr < w.n_rows && spoilt(acc, l));
        if (wrow + lr < w.n_rows) {
            const RowOut out = row_out<T, D, W::TM>(a, pl, un, kvh, w, wrow + lr, m_run, l, lq == 0);
#pragma unroll
            for (int u = 0; u < UT; u++) put4<T>(out, 16 * u + 4 * lq, acc[u]);
        }
        if (again) mend_rows<T, D, W::TM>(a, pl, un, kvh, w, wrow, again);
    }
}

template <int D>
__global__ __launch_bounds__(64 * (Wide32<D>::WAVES), (Wide32<D>::PER_CU) * (Wide32<D>::KS))
void paged_wide32(cf_paged_attn_args_t a, PagedPlan pl) {
    using W = Wide32<D>;
    __shared__ __attribute__((aligned(16))) float lds[W::LDS];
    __shared__ int kept[3 * 64];
    const Geometry<W::TM, 64, kNarrowCost> geo(a, pl, kept);
    if (geo.lists_cut_tiles()) return;
    for (int unit = (int)blockIdx.x;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        const Work w = unit_work<W::TM, 64>(a, pl, un);
        if (w.n_rows > 16) wide32_unit<D>(a, pl, lds, un, kvh, w);
        else if (narrow_unit<float, D, W::TM, 4, W::WAVES>(a, pl, lds, un, kvh, w)) mend_narrow<float, D, W::TM, 4>(a, pl, un, kvh, w);
    }
}

// ---- Every shape: a wave per row and head. ----
constexpr int kAnyDims = 512 / 64;             // dims per lane
template <typename T>
__global__ __launch_bounds__(256)
void paged_any(cf_paged_attn_args_t a, FastDiv by_page) {
    for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < (int64_t)a.T * a.H_q; unit += 4 * (int64_t)gridDim.x) {
        const int t = (int)(unit / a.H_q), h = (int)(unit - (int64_t)t * a.H_q);
        int lo = 0, hi = a.B;                  // the last sequence that does not start behind t
        while (hi - lo > 1) {
            const int mid = lo + ((hi - lo) >> 1);
            if (a.q_start[mid] <= t) lo = mid; else hi = mid;
        }
        const SeqRows s = seq_rows(a, lo);
        if (t >= s.row0 && t < s.row0 + s.n) plain_row<T, kAnyDims>(a, by_page, s, lo, t - s.row0, h, a.d);
    }
}

// The plan of a call on the matrix cores: the kernel and how its work is cut.
enum Form { kHeads, kSplit, kWide1, kWide2 };   // kWide2: fp16 tiles of 256 rows
struct Plan {
    PagedPlan pl;
    Form form;
    int  wgs, merge_wgs;
    size_t bytes;         // workspace
};

// paged_split for sequences of up to 1024 positions, which it finishes in one range, as long as
// its units, a workgroup each, go in one round: fp16, 32 heads of 128 over 8, us with paged_split
// and paged_heads: 1 x 512 8.3 and 11.8, 16 x 512 10.3 and 14.6, 32 x 1024 28.0 and 31.8, 64 x 512
// both 31.3; longer ones need ranges and a merge in both: 8 x 2048 19.8 and 18.2, 16 x 8192 117
// and 98, 2 x 30000 52.9 and 51.4.
constexpr int64_t kSplitLen = 1024;
// Tiles of 256 rows read a block's K and V once for twice the rows, but are twice as long a
// piece of work.  They pay where they fill three quarters of the chip by themselves (4 x 517 rows
// over 517: 34.8 us, with 128 rows 38.0; 4 x 1024 over 2048: 139 and 160; 1024 over 1024: 40.1 and
// 28.7), and where long ranges of one or two long sequences can be cut evenly (517 over 8517: 93 and
// 115; 330 over 2530: 37.7 and 37.9; 230 over 2430, 28 units: 31.5 and 30.8; 4 x 230: 77 and 58.5).
constexpr int64_t kLongLen = 2048;


bool fast_ok(const cf_paged_attn_args_t& a) {
    const uint64_t ptrs = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)(uintptr_t)a.o;
    const uint64_t steps = (uint64_t)a.q_stride | (uint64_t)a.page_stride | (uint64_t)a.row_stride | (uint64_t)a.head_stride;
    const uint64_t es = a.elem == CF_ELEM_F16 ? 2 : 4;
    // Row numbers times the group and positions (with what is read ahead) stay in 31 bits, offsets
    // inside a group of rows in 32.
    return (a.d == 64 || a.d == 128) && a.page_size % 16 == 0 && ptrs % 16 == 0 && steps * es % 16 == 0 && a.scale > 0.0f &&
           a.B <= kMostSeqs && (int64_t)a.T * (a.H_q / a.H_kv) <= (1 << 30) && (int64_t)a.max_pages * a.page_size <= (1 << 30) &&
           (uint64_t)a.row_stride * es * 16 < (1ull << 32);
}

// max_new and max_len only choose: the kernels' loops run until no unit is left, whatever the
// grid, and a sequence that is longer is computed all the same.
Plan make_plan(const cf_paged_attn_args_t& a) {
    Plan p;
    const int64_t G = a.H_q / a.H_kv, cus = cu_count();
    const bool f16 = a.elem == CF_ELEM_F16;
    const int64_t rows = (int64_t)a.max_new * G;              // of a sequence, at most
    const int64_t seqs = a.B < a.T ? a.B : a.T;
    auto tiles_of = [&](int64_t TM) {                         // tiles of the call, at most
        const int64_t t = ((int64_t)a.T * G + seqs * (TM - 1)) / TM;
        return rows <= TM && t > seqs ? seqs : t;
    };
    if (rows <= 16) {
        const int64_t units = tiles_of(16) * a.H_kv;
        p.form = units <= cus && a.max_len <= kSplitLen ? kSplit : kHeads;
    } else {
        const int64_t units = (int64_t)a.T * G / 256 * a.H_kv;
        const bool few_long = a.max_len > kLongLen && 2 * (int64_t)a.max_new >= a.T && units >= cus / 8;
        p.form = f16 && (4 * units >= 3 * cus || few_long) ? kWide2 : kWide1;
    }
    const int64_t TM = p.form <= kSplit ? 16 : !f16 ? 64 : p.form == kWide2 ? 256 : 128;
    const int64_t BK = p.form != kHeads ? 64 : f16 ? 32 : 16;
    const int64_t tiles = tiles_of(TM);
    // Units in flight, by the LDS a workgroup takes.
    const int64_t per_cu = p.form == kHeads ? (a.d == 128 ? 4 : 8) : f16 || a.d == 128 ? 1 : 2;
    const int64_t fill = cus * per_cu > a.H_kv ? cus * per_cu / a.H_kv : 1;
    p.pl.fill = (int32_t)fill;
    // What is not worth cutting: a merge and the records cost paged_heads 5 us and a wide tile 10
    // to 12 (517 rows over 1029: 28.5 us, cut from 8 blocks on into ranges of 4: 35.1; fp32, 200 rows
    // over 1200: 57.5 us, from 24 blocks on into ranges of 12: 90).
    const bool wide16 = f16 && p.form > kSplit;
    p.pl.min_blocks = (int32_t)(p.form == kHeads ? 64 / BK : wide16 ? 12 : 4);
    p.pl.one_blocks = (int32_t)((p.form == kHeads ? 128 : wide16 ? 1536 : 512) / BK);
    p.pl.max_records = (int32_t)(4 * fill + 8);
    const bool cut = !a.uncut && p.form != kSplit && (a.max_len + BK - 1) / BK > (wide16 ? kFewOne / BK : p.pl.one_blocks);
    if (!cut) p.pl.one_blocks = INT32_MAX;                    // nor is what is longer than max_len
    p.bytes = cut ? header_bytes(p.pl.max_records) + (size_t)p.pl.max_records * a.H_kv * (TM * (a.d + 2)) * sizeof(float) : 0;
    int64_t units = (tiles + (cut ? 2 * fill : 0)) * a.H_kv;
    if (units > (1 << 22)) units = 1 << 22;
    p.wgs = (int)(p.form == kHeads ? (units + 3) / 4 : units);
    p.pl.step = p.form == kHeads ? 4 * p.wgs : p.wgs;
    p.pl.unit_wgs = p.wgs;
    if (cut) p.wgs++;                                         // lists the cut tiles
    const int64_t most_rows = rows < TM ? rows : TM;
    const int64_t merge_rows = p.form == kHeads ? 1 : 1024 / a.d;   // of a workgroup
    p.pl.merge_groups = (int32_t)((most_rows + merge_rows - 1) / merge_rows);
    const int64_t merge_wgs = (tiles < 2 * fill ? tiles : 2 * fill) * a.H_kv * p.pl.merge_groups;
    p.merge_wgs = !cut ? 0 : merge_wgs > 4096 ? 4096 : (int)merge_wgs;
    p.pl.by_page = fastdiv_make(a.page_size);
    p.pl.G = (int32_t)G;
    p.pl.by_group = fastdiv_make((int)G);
    p.pl.by_kv = fastdiv_make(a.H_kv);
    p.pl.by_groups = fastdiv_make(p.pl.merge_groups);
    p.pl.cut_count = nullptr;
    p.pl.cut_tiles = nullptr;
    p.pl.records = nullptr;
    return p;
}

template <typename T, int D>
int launch_tiles(const cf_paged_attn_args_t& a, const Plan& p, hipStream_t st) {
    constexpr bool F16 = sizeof(T) == 2;
    const dim3 grid((unsigned)p.wgs), mgrid((unsigned)p.merge_wgs);
    auto go = [&](auto tiles, int threads, auto merge) {
        hipLaunchKernelGGL(tiles, grid, dim3(threads), 0, st, a, p.pl);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.merge_wgs == 0) return (int)e;
        hipLaunchKernelGGL(merge, mgrid, dim3(256), 0, st, a, p.pl);
        return (int)hipGetLastError();
    };
    if (p.form == kHeads) return go(paged_heads<T, D>, 256, paged_merge<T, D, 16, 1>);
    if (p.form == kSplit) {                                   // nothing is cut
        hipLaunchKernelGGL((paged_split<T, D>), grid, dim3(64 * Split<T, D>::WAVES), 0, st, a, p.pl);
        return (int)hipGetLastError();
    }
    if constexpr (F16) {
        if (p.form == kWide2) return go(paged_wide16<D, 2>, 512, paged_merge<T, D, 256, 1024 / D>);
        return go(paged_wide16<D, 1>, 512, paged_merge<T, D, 128, 1024 / D>);
    } else {
        return go(paged_wide32<D>, 64 * Wide32<D>::WAVES, paged_merge<T, D, 64, 1024 / D>);
    }
}

}  // namespace

extern "C" size_t cf_paged_attn_bytes(const cf_paged_attn_args_t* a) { return fast_ok(*a) ? make_plan(*a).bytes : 0; }

extern "C" int cf_launch_paged_attn(const cf_paged_attn_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    if (a->B <= 0 || a->T <= 0 || a->d <= 0 || a->d > 64 * kAnyDims || a->H_kv <= 0 || a->H_q % a->H_kv != 0)
        return (int)hipErrorInvalidValue;
    if (fast_ok(*a)) {
        Plan p = make_plan(*a);
        if (p.bytes > 0 && !a->workspace) return (int)hipErrorInvalidValue;
        if (p.bytes > 0) {
            p.pl.cut_count = (int*)a->workspace;
            p.pl.cut_tiles = (CutTile*)((char*)a->workspace + 256);
            p.pl.records = (float*)((char*)a->workspace + header_bytes(p.pl.max_records));
        }
        if (a->elem == CF_ELEM_F16)
            return a->d == 64 ? launch_tiles<_Float16, 64>(*a, p, st) : launch_tiles<_Float16, 128>(*a, p, st);
        return a->d == 64 ? launch_tiles<float, 64>(*a, p, st) : launch_tiles<float, 128>(*a, p, st);
    }
    const FastDiv by_page = fastdiv_make(a->page_size);
    int64_t wgs = ((int64_t)a->T * a->H_q + 3) / 4;
    if (wgs > (1 << 22)) wgs = 1 << 22;        // a grid has less than 2^32 threads
    if (a->elem == CF_ELEM_F16) hipLaunchKernelGGL(paged_any<_Float16>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    else hipLaunchKernelGGL(paged_any<float>, dim3((unsigned)wgs), dim3(256), 0, st, *a, by_page);
    return (int)hipGetLastError();
}
