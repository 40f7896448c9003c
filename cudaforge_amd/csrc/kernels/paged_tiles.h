// paged_tiles.h — what the kernels of attention over a paged cache share, whatever its numbers are:
// the geometry of tiles and ranges, a unit's rows and their places, the softmax's state, and the
// merge of cut tiles.
#ifndef CF_PAGED_TILES_H_
#define CF_PAGED_TILES_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "cdna4.h"

namespace {

using namespace cdna4;

constexpr float kLog2e = 1.4426950408889634f;

// f(std::integral_constant<int, i>) for i = 0 .. N - 1, unrolled.
template <typename F, int... S>
__device__ __forceinline__ void static_for_seq(F& f, std::integer_sequence<int, S...>) {
    (f(std::integral_constant<int, S>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    static_for_seq(f, std::make_integer_sequence<int, N>{});
}

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
// to the device only, so every wave works out the units from them: with R the ranges that
// fill the chip, C = ceil(sum_b tiles_b blocks_b / R) is the most blocks of one range and
// sequence b's tiles are cut into ns_b = ceil(blocks_b / C) ranges each.  A tile in one range
// is finished by its unit; else the units leave m, l and the unnormalised sum per row, and
// paged_merge joins them.  More than one range needs blocks_b > C, so ns_b < 2 blocks_b / C
// and there are at most 2 R + 1 such units per KV head; R is at most 2 `fill`.
//
// The kernels that share this:
//   paged_heads   up to 16 rows per tile, a wave per unit (decode steps);
//   paged_split   up to 16 rows of short sequences, the waves of a workgroup share the positions;
//   paged_wide16, paged_wide32   fp16 and fp32 tiles of 64 to 256 rows; tiles of up to 16 rows go
//                 as in paged_split there, so a batch may mix prompt chunks and decode steps.

// A cut tile, for the merge, which then has no geometry to work out.
struct CutTile {
    SeqRows s;
    int b, tile, n_ranges, record;          // record: of its first range
    int pad;                                // 32 bytes
};
struct PagedPlan {
    int*     cut_count;    // cut tiles (per KV head) and the list of them, which the workgroup
    CutTile* cut_tiles;    // behind the units' leaves
    float*   records;      // of the units of cut tiles
    int32_t max_records;   // per KV head
    int32_t unit_wgs;      // workgroups of units
    int32_t fill;          // units (per KV head) that fill the chip
    int32_t min_blocks;    // no range is cut shorter
    int32_t one_blocks;    // tiles of up to this many blocks are not cut
    int32_t step;          // of the unit loop
    int32_t merge_groups;  // workgroups that share the rows of a tile's merge
    int32_t G;             // query heads per KV head
    FastDiv by_page, by_group, by_kv, by_groups;
};

constexpr int kFewOne = 512, kFewMin = 4;    // positions of tiles that are not cut; blocks of a range

// A unit's tile and range.
struct Unit {
    SeqRows s;
    int b, tile, range, n_ranges, record;   // record: of the tile's first range (cut tiles)
};

// The tiles' geometry, one sequence per lane and 64 at a time.  TM rows per tile, BK
// positions per key block; a tile of up to 16 rows costs 1 / NARROW of a full one's block.
// CUTS: tiles may be cut.  COUNTS: ranges of few sequences are counted, so that they go
// in one round, and where that can't be those of wide tiles are ordered.
template <int TM, int BK, int NARROW, bool CUTS = true, bool COUNTS = false>
struct Geometry {
    const cf_paged_attn_args_t& a;
    const PagedPlan& pl;
    int lane, one;                       // tiles of up to `one` blocks are not cut
    float C, inv_C;                      // most blocks of a range
    SeqRows first;                       // lane: sequence `lane`, kept for the second pass,
    int* kept;                           // by wide tiles in LDS: their registers are all taken

    __device__ __forceinline__ SeqRows rows(int b) const {
        SeqRows s = seq_rows(a, min(b, a.B - 1));
        if (b >= a.B) s.n = s.len = 0;
        return s;
    }
    // Sequences base + lane, base + 64 + lane, ..: the loads of four wait together (1024 sequences
    // of 128 positions: 154 us, one at a time 192).
    static constexpr int kAtOnce = 4;
    static constexpr bool ORDERS = COUNTS && NARROW > 1;
    __device__ __forceinline__ void next_rows(int base, SeqRows (&s)[kAtOnce]) const {
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) s[j] = rows(base + 64 * j + lane);
    }
    __device__ __forceinline__ int tiles(const SeqRows& s) const { return (int)(((int64_t)s.n * pl.G + TM - 1) / TM); }
    __device__ __forceinline__ int blocks(const SeqRows& s) const { return (s.len + BK - 1) / BK; }
    __device__ __forceinline__ bool narrow(const SeqRows& s) const { return NARROW > 1 && s.n * pl.G <= 16; }
    __device__ __forceinline__ float cost(const SeqRows& s) const {
        const float w = (float)tiles(s) * (float)blocks(s);
        return narrow(s) ? w * (1.0f / NARROW) : w;
    }
    __device__ __forceinline__ int ranges(const SeqRows& s) const {
        const int n = blocks(s);
        return !CUTS || n <= one ? 1 : (int)((float)(n - 1) * (narrow(s) ? inv_C * (1.0f / NARROW) : inv_C)) + 1;
    }

    __device__ __forceinline__ Geometry(const cf_paged_attn_args_t& a_, const PagedPlan& pl_, int* kept_ = nullptr)
        : a(a_), pl(pl_), kept(kept_) {
        lane = threadIdx.x & 63;
        first = lane < a.B ? seq_rows(a, lane) : SeqRows{0, 0, 0};
        if constexpr (NARROW > 1) {          // every wave writes the same
            kept[lane] = first.row0;
            kept[64 + lane] = first.n;
            kept[128 + lane] = first.len;
        }
        if constexpr (!CUTS) return;
        float w = cost(first), t = (float)tiles(first);
        // (Without cuts and kinds of tiles there is nothing to plan.)
        const bool plans = NARROW > 1 || pl.one_blocks != INT32_MAX;
        for (int base = 64; plans && base < a.B; base += 64 * kAtOnce) {
            SeqRows s[kAtOnce];
            next_rows(base, s);
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                w += cost(s[j]);
                t += (float)tiles(s[j]);
            }
        }
        w = wave_sum(w);
        t = wave_sum(t);
        // As many ranges as make, with the tiles' last ones, one or two rounds of units.
        const float fill = (float)pl.fill;
        const float n = t <= 0.5f * fill ? fill - t : t <= fill ? 2.0f * fill - t : NARROW > 1 ? fill : 2.0f * fill;
        w = ceilf(w / fmaxf(n, 1.0f));
        // With less than a quarter of the chip busy, fp16 wide tiles are cut sooner than else (150 rows
        // of 12 heads over 3050: 18.3 us, else 19.8).
        const bool few = NARROW > 1 && t <= 0.25f * fill;
        one = __builtin_amdgcn_readfirstlane(few ? min(pl.one_blocks, kFewOne / BK) : pl.one_blocks);
        C = fmaxf(w, (float)(few ? kFewMin : pl.min_blocks));
        inv_C = 1.0f / C;
        if (pl.one_blocks == INT32_MAX) one = INT32_MAX;
        if constexpr (COUNTS) {
            int one_round = 0;
            if (plans && a.B <= 64 && t <= fill) one_round = count_ranges(few);
            if constexpr (ORDERS) {
                one_round &= __builtin_amdgcn_ballot_w64(narrow(first)) == 0;
                int before = -1;
                if (a.B <= 64 && !__builtin_amdgcn_readfirstlane(one_round)) before = in_order();
                kept[192 + lane] = before;       // once: other waves, with the same values, may be ahead
            }
        }
    }
    // COUNTS: the shortest ranges that go in one round of `fill` units (narrow ones as parts of one), if they
    // are not much longer than an equal share: else a few long sequences would wait for ranges
    // of their own.  For up to 64 sequences, one per lane (64 decode rows over 2000 in 8 bits 55 us,
    // uncounted 69, 65 uncounted 63; 64 over 500, one of them over 32000, 34 and 41, 65 37).
    __device__ __forceinline__ bool count_ranges(bool few) {
        const float fill = (float)pl.fill;
        const float least = (float)(few ? kFewMin : pl.min_blocks), by_fill = 1.0f / fill, was = C;
        const float share = fmaxf(wave_sum(cost(first)) * by_fill, least);
        C = ceilf(share);
        for (int i = 0; i < 3 && C <= 1.5f * share + 1.0f; i++) {
            inv_C = __builtin_amdgcn_rcpf(C);
            const float own = (float)(tiles(first) * ranges(first));
            const float units = wave_sum(narrow(first) ? fminf(cost(first) * inv_C, own) : own);
            if (units <= fill) return true;
            C = fmaxf(C + 1.0f, ceilf(C * units * by_fill));
        }
        C = was;
        inv_C = 1.0f / C;
        return false;
    }
    // ORDERS: what goes before each sequence's units, the longest ranges first.  Narrow tiles as if they took
    // longer than they do, so that they are spread: all of them at once wait for memory, between wide
    // ones they wait beside products (us of 31 decode rows with 4 chunks, of 56 with 8, and of the 4 chunks
    // alone: 106, 126, 87; with a quarter 108, 126, 87, with half 109, 127, 87; in the order of the
    // sequences, what is less than half of C last, 111, 133, 95).
    static constexpr float kNarrowFirst = 1.0f / 3.0f;
    __device__ __forceinline__ int in_order() const {
        const int items = tiles(first) * ranges(first);
        const float x = narrow(first) ? (float)blocks(first) * kNarrowFirst : (float)blocks(first);
        const int key = (__float_as_int(x * __builtin_amdgcn_rcpf((float)ranges(first))) & ~63) | (63 - lane);
        int before = 0;
#pragma clang loop unroll(disable)
        for (int j = 0; j < min(a.B, 64); j++) {
            const int n = __builtin_amdgcn_readlane(items, j);
            before += __builtin_amdgcn_readlane(key, j) > key ? n : 0;
        }
        return before;
    }
    // True for the workgroup behind the units', which lists the cut tiles.
    __device__ __forceinline__ bool lists_cut_tiles() const {
        if ((int)blockIdx.x != pl.unit_wgs) return false;
        if (threadIdx.x >= 64) return true;
        int count = 0, records = 0;
        for (int base = 0; base < a.B; base += 64) {
            const SeqRows s = rows(base + lane);
            const int ns = ranges(s), t = ns > 1 ? tiles(s) : 0;
            const int at = count + wave_excl_sum(t, lane), rec = records + wave_excl_sum(t * ns, lane);
            for (int i = 0; i < t && rec + (i + 1) * ns <= pl.max_records; i++)
                pl.cut_tiles[at + i] = CutTile{s, base + lane, i, ns, rec + i * ns, 0};
            count = __builtin_amdgcn_readlane(at + t, 63);
            records = __builtin_amdgcn_readlane(rec + t * ns, 63);
        }
        if (lane == 0) *pl.cut_count = min(count, pl.max_records / 2);
        return true;
    }
    // Unit u; false where there is none.
    __device__ __forceinline__ bool find(int u, Unit& out) const {
        int items0 = 0;
        const int first_unit = ORDERS ? kept[192 + lane] : -1;
        const bool ordered = ORDERS && __builtin_amdgcn_readfirstlane(first_unit) >= 0;
        // Wide tiles: the sequences with the long ranges first, so that short pieces fill the end
        // (35 sequences, 4 of them chunks: 108 us, in the order of the sequences 131).
        constexpr int CLASSES = NARROW > 1 ? 2 : 1;
        for (int cls = 0; cls < (ordered ? 1 : CLASSES); cls++) {
            int records0 = 0;
            auto scan = [&](const SeqRows& s, int base) {
                const int t = tiles(s), ns = ranges(s), rec = ns > 1 ? t * ns : 0;
                const bool cut = __builtin_amdgcn_ballot_w64(ns > 1) != 0;
                int items = t * ns;
                if (CLASSES > 1 && !ordered && (2.0f * (float)blocks(s) > C * (float)ns ? 0 : 1) != cls) items = 0;
                const int before = ordered ? first_unit : items0 + wave_excl_sum(items, lane);
                const int rec_before = records0 + (cut ? wave_excl_sum(rec, lane) : 0);
                const unsigned long long hit = __ballot(before <= u && u < before + items);
                if (!hit) {
                    items0 = __builtin_amdgcn_readlane(before + items, 63);
                    records0 = __builtin_amdgcn_readlane(rec_before + rec, 63);
                    return false;
                }
                const int src = __builtin_ctzll(hit);
                const int at = u - __builtin_amdgcn_readlane(before, src);
                out.n_ranges = __builtin_amdgcn_readlane(ns, src);
                const int nt = __builtin_amdgcn_readlane(t, src);
                const int i = out.n_ranges == 1 ? at : at / out.n_ranges;
                out.range = at - i * out.n_ranges;
                out.tile = nt - 1 - i;                         // the longest first
                out.record = __builtin_amdgcn_readlane(rec_before, src) + out.tile * out.n_ranges;
                out.b = base + src;
                out.s.row0 = __builtin_amdgcn_readlane(s.row0, src);
                out.s.n = __builtin_amdgcn_readlane(s.n, src);
                out.s.len = __builtin_amdgcn_readlane(s.len, src);
                return true;
            };
            bool found = scan(NARROW > 1 ? SeqRows{kept[lane], kept[64 + lane], kept[128 + lane]} : first, 0);
            for (int base = 64; !found && base < a.B; base += 64 * kAtOnce) {
                SeqRows s[kAtOnce];
                next_rows(base, s);
#pragma unroll
                for (int j = 0; j < kAtOnce; j++)
                    if (!found && base + 64 * j < a.B) found = scan(s[j], base + 64 * j);
            }
            if (found) return out.n_ranges == 1 || out.record + out.n_ranges <= pl.max_records;
        }
        return false;
    }
};

// What a unit computes: rows R0 .. R0 + n_rows - 1 of the sequence's list over positions
// [key0, key1).  Row R sees positions below base + R / G.
struct Work {
    int R0, n_rows, base, key0, key1;
};
template <int TM, int BK>
__device__ __forceinline__ Work unit_work(const cf_paged_attn_args_t& a, const PagedPlan& pl, const Unit& un) {
    Work w;
    w.R0 = un.tile * TM;
    w.n_rows = min(un.s.n * pl.G - w.R0, TM);
    w.base = un.s.len - un.s.n + 1;
    const int limit = min(max(w.base + fastdiv(w.R0 + w.n_rows - 1, pl.by_group), 0), un.s.len);
    const int blocks = (limit + BK - 1) / BK;
    const int per = un.n_ranges == 1 ? blocks : (blocks + un.n_ranges - 1) / un.n_ranges;
    const int b0 = min(un.range * per, blocks), b1 = min(b0 + per, blocks);
    w.key0 = b0 * BK;
    w.key1 = min(b1 * BK, limit);
    return w;
}

// Record of one unit: [m (TM)] [l (TM)] [sum (TM, D)], m in the log2 domain.
template <int TM, int D> constexpr size_t record_floats() { return (size_t)TM * (D + 2); }
template <int TM, int D>
__device__ __forceinline__ float* record_of(const cf_paged_attn_args_t& a, const PagedPlan& pl, const Unit& un, int kvh) {
    return pl.records + ((size_t)(un.record + un.range) * a.H_kv + kvh) * record_floats<TM, D>();
}

// Row R of a sequence's list for KV head kvh: its place in Q or O, in rows of heads.
struct RowAt { int tok, h; };
__device__ __forceinline__ RowAt row_at(const PagedPlan& pl, int G, int kvh, int R) {
    const int tok = fastdiv(R, pl.by_group);
    return {tok, kvh * G + (R - tok * G)};
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f4_t x) {
    typedef T four_t __attribute__((ext_vector_type(4)));
    *(four_t*)p = four_t{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
}

// One entry through the scalar cache.
typedef const int32_t __attribute__((address_space(4)))* table_t;
__device__ __forceinline__ table_t table_of(const cf_paged_attn_args_t& a, int b) {
    return (table_t)(uintptr_t)(a.table + (size_t)b * a.max_pages);
}
__device__ __forceinline__ int page_of(const cf_paged_attn_args_t& a, const PagedPlan& pl, table_t table, int key) {
    return table[min(fastdiv(key, pl.by_page), a.max_pages - 1)];
}
// The group of 16 positions from `key` on `page`: where it starts in the cache (elements; page
// 0 stands in for one that is none), and which of its positions count (below key1, a real page).
struct Group { int64_t at; uint32_t mask; };
__device__ __forceinline__ Group group_of(const cf_paged_attn_args_t& a, const PagedPlan& pl, int page, int key, int key1) {
    const bool valid = (unsigned)page < (unsigned)a.num_pages;
    const int count = valid ? min(max(key1 - key, 0), 16) : 0;
    const int in_page = key - fastdiv(key, pl.by_page) * a.page_size;
    return {(int64_t)(valid ? page : 0) * a.page_stride + (int64_t)in_page * a.row_stride, (1u << count) - 1u};
}

// The next 64 groups of a range, one per lane.  A load of a table entry per group would be in
// the way: an ordinary one's wait drains the ring, and one through the scalar cache makes the
// waits for LDS reads wait for it; and a group's place takes some 40 scalar instructions.
// load() drains the ring once per 64 groups.
struct Groups {
    const int32_t* table;
    int lo, hi, mask;        // lane: Group of base + lane
    uint64_t whole;          // bit: all 16 positions of it count
    __device__ __forceinline__ void load(const cf_paged_attn_args_t& a, const PagedPlan& pl, int base, int key0, int key1) {
        const int key = key0 + (base + (int)(threadIdx.x & 63)) * 16;
        const Group g = group_of(a, pl, table[fastdiv(min(key, a.max_pages * a.page_size - 1), pl.by_page)], key, key1);
        lo = (int)g.at;
        hi = (int)(g.at >> 32);
        mask = (int)g.mask;
        asm volatile("" : "+v"(lo), "+v"(hi), "+v"(mask));    // they have arrived
        whole = __builtin_amdgcn_ballot_w64(mask == 0xffff);
    }
    __device__ __forceinline__ int64_t at(int i) const {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i & 63) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane(lo, i & 63));
    }
    // Positions of groups i .. i + N - 1 that count (i a multiple of N).
    template <int N>
    __device__ __forceinline__ uint64_t masks(int i) const {
        constexpr uint64_t all = N == 4 ? ~0ull : (1ull << (16 * N & 63)) - 1;
        if ((~(whole >> (i & 63)) & ((1u << N) - 1)) == 0) return all;
        uint64_t mk = 0;
#pragma unroll
        for (int g = 0; g < N; g++)
            mk |= (uint64_t)(uint32_t)__builtin_amdgcn_readlane(mask, (i + g) & 63) << (16 * g);
        return mk;
    }
};

// LDS rows are swizzled in 16-byte chunks: K (and Q) rows are read 16 rows at one chunk, V
// rows transposed (fp16, ds_read_b64_tr_b16) or 4 rows of 16 floats (fp32).
template <typename T, int D> __device__ __forceinline__ int kswz(int row) {
    return sizeof(T) == 4 || D == 128 ? row & 15 : (row >> 1) & 7;
}
template <typename T, int D> __device__ __forceinline__ int vswz(int row) {
    return sizeof(T) == 4 ? row & 15 : D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

// On the matrix cores a position that another row of the tile sees counts as 0 times its V, which is
// no 0 where V is infinite or NaN; and one that the row sees as a weight in two parts, whose products
// with an infinite V add up to NaN.  Where a sum is NaN while l is a number, mend_rows looks.
template <int N>
__device__ __forceinline__ bool spoilt(const f4_t (&acc)[N], float l) {
    f4_t x = acc[0];
#pragma unroll
    for (int u = 1; u < N; u++) x += acc[u];
    const float y = (x[0] + x[1]) + (x[2] + x[3]);
    return y != y && l == l;
}
// Bit r: one of the lanes r, r + 16, r + 32 and r + 48 has `bad` set.
__device__ __forceinline__ uint32_t rows_of_16(bool bad) {
    const uint64_t b = __builtin_amdgcn_ballot_w64(bad);
    const uint32_t x = (uint32_t)b | (uint32_t)(b >> 32);
    return (x | x >> 16) & 0xffffu;
}

// The lane, as a unit's code sees it: what is worked out from it stays inside the unit.  Taken
// out of the loop over units, all kernels' offsets would be held at once, and wide tiles have
// no registers for that.
__device__ __forceinline__ int unit_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// How rows of D elements lie in LDS and in lanes.
template <typename T, int D> struct Rows {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int CE = 16 / sizeof(T);          // elements per 16-byte chunk
    static constexpr int CPR = D / CE;                 // chunks per row
    static constexpr int RPI = 64 / CPR;               // rows per DMA instruction (1 KB)
    static constexpr int NI = 16 / RPI;                // DMA instructions per 16 rows
    static constexpr int NF = F16 ? D / 32 : D / 16;   // chunks of a K row a lane takes
    static constexpr int UT = D / 16;                  // 16-dim tiles of O^T
    static constexpr int VR = F16 ? UT : 4;            // V read offsets a lane keeps
    typedef T chunk_t __attribute__((ext_vector_type(CE)));
    // DMA: lane L of instruction u writes physical chunk L % CPR of row RPI u + L / CPR of a
    // 16-row group, which holds logical chunk (L % CPR) ^ swizzle.
    static __device__ __forceinline__ int drow(int lane) { return lane / CPR; }
    static __device__ __forceinline__ int dch(int lane) { return lane % CPR; }
    // LDS read offsets (elements) of the lane's K chunks inside 16 rows: fp16 lane (lr, lq)
    // takes row lr, dims 32 f + 8 lq .. + 7; fp32 dims D / 4 lq + 4 f .. + 3 (k-slot lq of MFMA
    // step s is dim D / 4 lq + s).
    static __device__ __forceinline__ void k_offsets(int (&rd)[NF], int lane) {
        const int lr = lane & 15, lq = lane >> 4;
#pragma unroll
        for (int f = 0; f < NF; f++) rd[f] = lr * D + CE * ((F16 ? 4 * f + lq : NF * lq + f) ^ kswz<T, D>(lr));
    }
    // ... of its V: fp16 (ds_read_tr4) key 4 lq + lr / 4, dims 16 u + 4 (lr % 4) .. + 3; fp32 row
    // 4 lq + kk, whose chunk the read adds.
    static __device__ __forceinline__ void v_offsets(int (&rd)[VR], int lane) {
        const int lr = lane & 15, lq = lane >> 4;
#pragma unroll
        for (int u = 0; u < VR; u++) {
            if constexpr (F16) {
                const int row = 4 * lq + (lr >> 2), col = 16 * u + 4 * (lr & 3);
                rd[u] = row * D + 8 * ((col >> 3) ^ vswz<T, D>(row)) + (col & 7);
            } else {
                rd[u] = (4 * lq + u) * D + (lr & 3);
            }
        }
    }
    // fp32: V of key 16 t + 4 lq + kk, dim 16 u + lr (base: the stage's V).
    static __device__ __forceinline__ float v_at(const float* base, const int (&rd)[VR], int lane, int t, int kk, int u) {
        const int lr = lane & 15, lq = lane >> 4;
        return base[rd[kk] + 16 * t * D + 4 * ((4 * u + (lr >> 2)) ^ vswz<T, D>(4 * lq + kk))];
    }
};

// m is what p = 2^(score - m) is taken against, low_max of a block's scores.  It moves only when a
// block's exceeds it by more than 2^kLazy; until then the sums are not rescaled.
// fp16: 2^7 below the maximum, and p at most 2^15, which fp16 holds as exactly as 1, so that weights of
// down to 2^-32 of the largest are in fp16's range, whose smallest number is 2^-24: taken against
// the maximum itself, the many positions of a long context that weigh less than 2^-25 each would
// all count as 0.
// fp32: the maximum, and p at most 2: sums do not overflow before V's own would, and score - m, whose
// rounding is p's, stays small (2^8 above the maximum a row of 257 positions was off by 3.5e-7, so 2.8e-7).
template <typename T> constexpr float kLazy = sizeof(T) == 2 ? 8.0f : 1.0f;
template <typename T> __device__ __forceinline__ float low_max(float x, float c) {
    return sizeof(T) == 2 ? __builtin_fmaf(x, c, -7.0f) : x * c;
}
template <typename T> __device__ __forceinline__ bool move_max(float mloc, float& m, float& alpha) {
    if (!__builtin_amdgcn_ballot_w64(mloc > m + kLazy<T>)) return false;
    const float m_new = mloc > m + kLazy<T> ? mloc : m;
    alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));   // 0 on the first move
    m = m_new;
    return true;
}

// A sum of many terms with what its roundings drop (x + y = s + e exactly): l of a long context whose
// positions weigh too little, each for itself, to be seen beside one that weighs more.
struct LongSum {
    float s = 0.0f, e = 0.0f;
    __device__ __forceinline__ void add(float x) {
        const float t = s + x, y = t - s;
        e += (s - (t - y)) + (x - y);
        s = t;
    }
    __device__ __forceinline__ void scale(float x) { s *= x; e *= x; }
    __device__ __forceinline__ float sum() const { return s + e; }
};

// Scores of a lane's row in a block: key 16 t + 4 lq + i of it counts where its bit of `mk` is
// set and it is one of the first `seen`.  Bit by bit in vector registers: comparisons would
// take a pair of scalar registers per score.
template <int NG>
__device__ __forceinline__ void hide(f4_t (&sc)[NG], uint64_t mk, int seen, int lane) {
    const uint64_t low = seen <= 0 ? 0 : seen >= 64 ? ~0ull : (1ull << seen) - 1;
    const uint64_t bits = (mk & low) >> (4 * (lane >> 4));
#pragma unroll
    for (int t = 0; t < NG; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t half = t < 2 ? (uint32_t)bits : (uint32_t)(bits >> 32);
            const uint32_t keep = (uint32_t)((int32_t)(half << (31 - 16 * (t & 1) - i)) >> 31);
            sc[t][i] = __uint_as_float((__float_as_uint(sc[t][i]) & keep) | (0xff800000u & ~keep));
        }
}

// Dims d0 .. d0 + 3 of row `row` of a wide tile: into the unit's record, or normalised into O.
struct RowOut {
    float* rec;       // the row's sum in the record, or null
    void*  o;         // its row of O
    float  inv;
};
template <typename T, int D, int TM>
__device__ __forceinline__ RowOut row_out(const cf_paged_attn_args_t& a, const PagedPlan& pl, const Unit& un, int kvh,
                                          const Work& w, int row, float m, float l, bool first) {
    if (un.n_ranges > 1) {
        float* const rec = record_of<TM, D>(a, pl, un, kvh);
        if (first) {
            rec[row] = m;
            rec[TM + row] = l;
        }
        return {rec + 2 * TM + row * D, nullptr, 1.0f};
    }
    const RowAt at = row_at(pl, pl.G, kvh, w.R0 + row);
    return {nullptr, (T*)a.o + ((int64_t)(un.s.row0 + at.tok) * a.H_q + at.h) * D, l == 0.0f ? 0.0f : 1.0f / l};
}
template <typename T>
__device__ __forceinline__ void put4(const RowOut& out, int d0, f4_t x) {
    if (out.rec) *(f4_t*)(out.rec + d0) = x;
    else store4((T*)out.o + d0, x * out.inv);
}

// Joins the ranges of cut tiles: O = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.  A
// workgroup per (tile, KV head) and ROWS rows: 256 / ROWS threads per row, D / 4 of them side
// by side over the dims, the rest sharing the ranges.
// Latency bounds it: 4 to 5 us, 2 of them any launch's.
template <typename T, int D, int TM, int ROWS>
__global__ __launch_bounds__(256)
void paged_merge(cf_paged_attn_args_t a, PagedPlan pl) {
    constexpr int DL = D / 4, SUBS = 256 / ROWS / DL;      // lanes over the dims, shares of the ranges
    static_assert(SUBS >= 1, "rows per workgroup");
    __shared__ float ml[2][ROWS][SUBS];
    __shared__ f4_t part[SUBS > 1 ? SUBS * ROWS * DL : 1];
    // The first tile's entry comes with the number of them (the list is longer than the grid's tiles).
    auto place = [&](int unit, int& group, int& kvh) {
        const int th = fastdiv(unit, pl.by_groups), tile_id = fastdiv(th, pl.by_kv);
        group = unit - th * pl.merge_groups;
        kvh = th - tile_id * a.H_kv;
        return tile_id;
    };
    int group, kvh;
    CutTile un = pl.cut_tiles[place(blockIdx.x, group, kvh)];
    const int cut_units = *pl.cut_count * a.H_kv * pl.merge_groups;
    asm volatile("" : "+s"(un.record), "+s"(un.n_ranges));
    const int G = pl.G;
    const int d4 = threadIdx.x % DL, sub = threadIdx.x / DL % SUBS, r = threadIdx.x / (DL * SUBS);
    for (int unit = blockIdx.x; unit < cut_units; unit += gridDim.x) {
        if (unit != (int)blockIdx.x) un = pl.cut_tiles[place(unit, group, kvh)];
        const int n_rows = min(un.s.n * G - un.tile * TM, TM);
        const float* const rec = pl.records + ((size_t)un.record * a.H_kv + kvh) * record_floats<TM, D>();
        const size_t step = (size_t)a.H_kv * record_floats<TM, D>();
        for (int row0 = group * ROWS; row0 < n_rows; row0 += pl.merge_groups * ROWS) {   // uniform
            const int row = row0 + r;
            float m = -INFINITY, l = 0.0f;
            f4_t acc = f4_t{0.f, 0.f, 0.f, 0.f};
            if (row < n_rows)
                for (int s0 = sub; s0 < un.n_ranges; s0 += 4 * SUBS) {
                    // Four ranges' loads at a time; one behind the last counts for nothing.
                    float ms[4], ls[4];
                    f4_t as[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int s = min(s0 + k * SUBS, un.n_ranges - 1);
                        ms[k] = rec[s * step + row];
                        ls[k] = rec[s * step + TM + row];
                        as[k] = *(const f4_t*)(rec + s * step + 2 * TM + row * D + 4 * d4);
                    }
                    float m_new = m;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (s0 + k * SUBS < un.n_ranges) m_new = fmaxf(m_new, ms[k]);
                    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                    const float wa = __builtin_amdgcn_exp2f(m - m_use);
                    m = m_new;
                    l *= wa;
                    acc *= wa;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (s0 + k * SUBS < un.n_ranges) {
                            const float wb = __builtin_amdgcn_exp2f(ms[k] - m_use);
                            l += ls[k] * wb;
                            acc += as[k] * wb;
                        }
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
                const RowAt at = row_at(pl, G, kvh, un.tile * TM + row);
                store4((T*)a.o + ((int64_t)(un.s.row0 + at.tok) * a.H_q + at.h) * D + 4 * d4, acc * inv);
            }
        }
    }
}

// Of the workspace: the number of cut tiles (256 bytes) and the list of them.
size_t header_bytes(int32_t max_records) { return 256 + ((size_t)max_records / 2 * sizeof(CutTile) + 255) / 256 * 256; }

// A unit looks for its sequence among all of them, so that the time of the tiles rises with the square
// of their number, that of the plain kernel with the positions (decode rows of 8 heads of 64 over 2,
// tiles and plain kernel: 1024 sequences of 16 positions 17 and 39 us, 16384 of 128 2.0 and 3.4 ms, 32768 of 16 7.5
// and 1.4 and of 128 7.8 and 6.6, 65536 of 128 31 and 13).  More than this many take the plain kernel.
constexpr int kMostSeqs = 32768;

}  // namespace

#endif  // CF_PAGED_TILES_H_
