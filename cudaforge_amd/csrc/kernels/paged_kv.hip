// paged_kv.hip — the pages of a step and the write of new K and V rows into them (gfx950).
//
// page_map: with c_b positions held and n_b tokens new, sequence b takes
// need_b = ceil((c_b + n_b) / P) - ceil(c_b / P) pages, the ones at places
// head + E_b .. of the ring with E_b the sum of need before b; token i of b is at position
// c_b + i and its slot is page * P + (c_b + i) % P.  Everything but the prefix sums is
// independent per token and per page.  A sequence that was not served and whose length counts the
// tokens all the same (in place) is known by its last entry, which is -1: it gets nothing, and
// when it ends, what it gives back are the entries that are pages.  Launch and latency bound it: 16 sequences 6.6 us, 256
// with 65000 tokens 9.5, 3000 with 63000 tokens 14.5.
//
// page_store: pages[slot[t]] = row t of K and V, with Q and K turned by their positions.  HBM
// bounds it: 8192 rows of 32 + 2 x 8 heads of 128 fp16, 201 MB, 41 to 43 us (4.8 TB/s; a large
// copy makes 5.2); 16 rows take 7 us, a launch.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "cdna4.h"

namespace {

using namespace cdna4;

// ------------------------------------------------------------------ map ---

constexpr int kMapThreads = 1024;
// The one-workgroup form: one sequence and four rows per thread (6.5 to 8 us over that range; by
// two launches 9.5 to 11.5).  It moves the pages of ended sequences too, at about 1 us per thousand
// more than two launches (64 requests of 512 pages ending at once: 31 and 11.5 us; 1024 of them 530
// and 83).  Pages come back as fast as tokens fill them, at most 4096 / page_size a step in the
// long run, so that costs less than the second launch for every step would.
constexpr int kMapOneSeqs = 1024;
constexpr int kMapOneTokens = 4096;

enum { kNotServed = -1, kEnded = -2, kEndedGaps = -3 };

// What the tokens and pages of one sequence need to know.
struct SeqPages {
    int c;         // positions held
    int n;         // new tokens (0 for an ended sequence)
    int first;     // place of its first new page behind the ring's head, kNotServed, kEnded or, where
                   // some of its entries are no pages, kEndedGaps
    int give;      // ended: place of its first page behind the free ones
};

struct MapDivs { FastDiv page, ring; };

// The counters as they are used: any content gives a place in the ring.
struct RingState { int head, avail, tail; };
__device__ __forceinline__ RingState ring_state(const int32_t* counters, int R, FastDiv by_ring) {
    RingState r;
    const int h = max(counters[0], 0);
    r.head = h - fastdiv(h, by_ring) * R;
    r.avail = min(max(counters[1], 0), R);
    r.tail = r.head + r.avail;                     // R <= 2^30
    if (r.tail >= R) r.tail -= R;
    return r;
}

__device__ __forceinline__ int ceil_pages(int x, int P, FastDiv by_page) {
    const int q = fastdiv(x, by_page);
    return q + (q * P < x ? 1 : 0);
}

// Entries of a row of the table that a sequence of len positions needs, the whole row where that is
// more than it has.
__device__ __forceinline__ int last_entry(const cf_page_map_args_t& a, FastDiv by_page, uint32_t len) {
    return len <= (uint32_t)(a.max_pages * a.page_size) ? ceil_pages((int)len, a.page_size, by_page) : a.max_pages;
}

// The page at place x behind the ring's head (x < avail), or -1 where the ring holds no page.
__device__ __forceinline__ int ring_page(const cf_page_map_args_t& a, int head, int x, FastDiv by_ring) {
    const int at = head + x;                       // < 2 R
    const int page = a.ring[at - fastdiv(at, by_ring) * a.ring_size];
    return (unsigned)page < (unsigned)a.num_pages ? page : -1;
}

// The slot of position pos of sequence b.
__device__ __forceinline__ int slot_of(const cf_page_map_args_t& a, const RingState& r, const MapDivs& dv, int b,
                                       const SeqPages& s, int pos) {
    if (s.first < 0) return -1;
    const int idx = fastdiv(pos, dv.page), before = ceil_pages(s.c, a.page_size, dv.page);
    const int page = idx < before ? a.table[(size_t)b * a.max_pages + idx] : ring_page(a, r.head, s.first + idx - before, dv.ring);
    return (unsigned)page < (unsigned)a.num_pages ? page * a.page_size + (pos - idx * a.page_size) : -1;
}

// A page behind the free ones, at place x of those that this call takes back.  Those that the ring
// has no place for are left out, as every place holds a free page then.
__device__ __forceinline__ void give_back(const cf_page_map_args_t& a, const RingState& r, int x, int page) {
    if (x >= a.ring_size - r.avail) return;
    const int at = r.tail + x;                     // < 2 R
    a.ring[at >= a.ring_size ? at - a.ring_size : at] = page;
}

// The pages among the first n entries of row b of the table, whose sequence has ended (kEndedGaps):
// by a wave, in their order.
__device__ __forceinline__ void give_back_gaps(const cf_page_map_args_t& a, const RingState& r, int b, const SeqPages& s,
                                               int n, int lane) {
    constexpr int kAtOnce = 4;
    const int32_t* const row = a.table + (size_t)b * a.max_pages;
    int place = s.give;
    for (uint32_t at = 0; at < (uint32_t)n; at += 64 * kAtOnce) {
        int page[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) page[k] = at + 64 * k + lane < (uint32_t)n ? row[at + 64 * k + lane] : -1;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const bool real = (unsigned)page[k] < (unsigned)a.num_pages;
            const uint64_t all = __builtin_amdgcn_ballot_w64(real);
            if (real) give_back(a, r, place + __builtin_popcountll(all & ((1ull << lane) - 1)), page[k]);
            place += __builtin_popcountll(all);
        }
    }
}

// Page j that changes hands with sequence b: into its table, or out of it into the ring.
__device__ __forceinline__ void move_page(const cf_page_map_args_t& a, const RingState& r, const MapDivs& dv, int b,
                                          const SeqPages& s, int j) {
    int32_t* const row = a.table + (size_t)b * a.max_pages;
    if (s.first == kEnded) {
        give_back(a, r, s.give + j, row[j]);
        return;
    }
    row[ceil_pages(s.c, a.page_size, dv.page) + j] = s.first >= 0 ? ring_page(a, r.head, s.first + j, dv.ring) : -1;
}

// How many of the first n entries of a row of the table are pages: by a wave, 512 entries at a time.
__device__ __forceinline__ int count_pages(const cf_page_map_args_t& a, const int32_t* row, int n, int lane) {
    constexpr int kAtOnce = 8;
    int count = 0;
    for (uint32_t at = 0; at < (uint32_t)n; at += 64 * kAtOnce) {
        int page[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) page[k] = at + 64 * k + lane < (uint32_t)n ? row[at + 64 * k + lane] : -1;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++)
            count += __builtin_popcountll(__builtin_amdgcn_ballot_w64((unsigned)page[k] < (unsigned)a.num_pages));
    }
    return count;
}

// For N rows at once, so that the LDS reads of one do not wait for another's: the last entry of
// start[0 .. n) that is not above x[j] (start[0] <= x[j]).
template <int N>
__device__ __forceinline__ void last_not_above(const int* start, int n, const int (&x)[N], int (&at)[N]) {
#pragma unroll
    for (int j = 0; j < N; j++) at[j] = 0;
    for (int step = kMapOneSeqs / 2; step > 0; step >>= 1) {
        if (step >= n) continue;
        int v[N];
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = start[min(at[j] + step, n - 1)];
#pragma unroll
        for (int j = 0; j < N; j++) at[j] += at[j] + step < n && v[j] <= x[j] ? step : 0;
    }
}

// What a sequence asks for and gives back.
struct Asked {
    int c, n;      // positions held; new tokens, negative for an ended sequence
    int need;      // new pages, kNotServed where its length passes the table, kStuck where it was not
                   // served before
    int back;      // ended: entries of its row that are pages
};
enum { kStuck = -2 };

// Those of sequences b0 .. b0 + PER - 1 of each thread of a workgroup of WAVES waves.  The rows of
// ended sequences are read by all its waves.
template <int PER, int WAVES> struct EndedList { int n; int2 row[PER * WAVES * 64]; };   // sequence and entries, then pages
template <int PER, int WAVES>
__device__ __forceinline__ void ask(const cf_page_map_args_t& a, FastDiv by_page, int b0, Asked (&s)[PER], EndedList<PER, WAVES>& ended) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int P = a.page_size, cap = a.max_pages * P;
    int raw[PER], last[PER], before[PER], place[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        raw[j] = b0 + j < a.B ? a.cache_lens[b0 + j] : 0;
        s[j].n = b0 + j < a.B ? a.new_lens[b0 + j] : 0;
        s[j].back = 0;
    }
    if (tid == 0) ended.n = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; j++) {
        s[j].c = min(max(raw[j], 0), cap);
        before[j] = ceil_pages(s[j].c, P, by_page);
        last[j] = 0;
        if (before[j] > 0) {
            if (s[j].n >= 0) last[j] = a.table[(size_t)(b0 + j) * a.max_pages + before[j] - 1];
            else ended.row[place[j] = atomicAdd(&ended.n, 1)] = {b0 + j, before[j]};
        }
    }
    __syncthreads();
    const int n = ended.n;
    if (n > 0) {
        for (int i = wave; i < n; i += WAVES) {
            const int2 e = ended.row[i];
            const int got = count_pages(a, a.table + (size_t)e.x * a.max_pages, e.y, lane);
            if (lane == 0) ended.row[i].y = got;
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < PER; j++) {
        if (s[j].n < 0) {
            s[j].need = 0;
            if (before[j] > 0) s[j].back = ended.row[place[j]].y;
            continue;
        }
        const uint32_t len = (uint32_t)s[j].c + (uint32_t)s[j].n;
        s[j].need = last[j] < 0 || raw[j] > cap ? kStuck : len > (uint32_t)cap ? kNotServed
                  : ceil_pages((int)len, P, by_page) - before[j];
    }
}

// Many sequences: their entries lie on as many lines of memory (3000 sequences: 14.5 us for the three
// launches; with page_map_scan reading the lines, in two launches, 16.7).
constexpr int kAskThreads = 64;
__global__ __launch_bounds__(kAskThreads)
void page_map_ask(cf_page_map_args_t a, FastDiv by_page) {
    __shared__ EndedList<1, kAskThreads / 64> ended;
    const int b = (int)blockIdx.x * kAskThreads + (int)threadIdx.x;
    Asked s[1];
    ask(a, by_page, b, s, ended);
    if (b < a.B) ((int4*)a.info)[b] = int4{s[0].c, s[0].n, s[0].need, s[0].back};
}

// One workgroup: the prefix sums, PER neighbouring sequences per thread.  ONE (one per
// thread, up to 1024 sequences and 4096 tokens): it then writes the tokens and pages too, each found by its
// number in the sums in LDS; else it leaves SeqPages per sequence in a.info for page_map_fill.
// ASKED: a.info holds what page_map_ask left.
template <bool ONE, int PER, bool ASKED>
__global__ __launch_bounds__(kMapThreads)
void page_map_scan(cf_page_map_args_t a, MapDivs dv) {
    constexpr int kWaves = kMapThreads / 64;
    __shared__ int part[4][kWaves];
    __shared__ int taken_s, refused_s, gaps_s;
    __shared__ SeqPages seq[ONE ? kMapOneSeqs : 1];
    __shared__ int row0[ONE ? kMapOneSeqs : 1], move0[ONE ? kMapOneSeqs : 1];
    __shared__ EndedList<ASKED ? 1 : PER, ASKED ? 1 : kWaves> ended_rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int P = a.page_size;
    const RingState r = ring_state(a.counters, a.ring_size, dv.ring);
    if (tid == 0) taken_s = refused_s = gaps_s = 0;
    int carry[4] = {0, 0, 0, 0};                   // rows, pages needed, taken back, moved
    for (int base = 0; base < a.B; base += PER * kMapThreads) {
        Asked ak[PER];
        int v[PER][4], sum[4] = {0, 0, 0, 0}, ex[4];
        bool gaps[PER];
        if constexpr (ASKED) {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int b = base + PER * tid + j;
                const int4 x = b < a.B ? ((const int4*)a.info)[b] : int4{0, 0, 0, 0};
                ak[j] = {x.x, x.y, x.z, x.w};
            }
        } else {
            ask(a, dv.page, base + PER * tid, ak, ended_rows);
        }
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int before = ceil_pages(ak[j].c, P, dv.page);
            const uint32_t len = (uint32_t)ak[j].c + (uint32_t)max(ak[j].n, 0);
            v[j][0] = max(ak[j].n, 0);
            v[j][1] = max(ak[j].need, 0);
            v[j][2] = ak[j].back;
            gaps[j] = ak[j].n < 0 && ak[j].back < before;
            if constexpr (ONE)
                v[j][3] = gaps[j] ? 0 : ak[j].n < 0 ? before : base + PER * tid + j < a.B ? last_entry(a, dv.page, len) - before : 0;
            else
                v[j][3] = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) sum[k] += v[j][k];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            ex[k] = wave_excl_sum(sum[k], lane);
            if (lane == 63) part[k][wave] = ex[k] + sum[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            int all = 0;
            for (int w = 0; w < kWaves; w++) {
                if (w == wave) ex[k] += carry[k] + all;
                all += part[k][w];
            }
            carry[k] += all;
        }
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int b = base + PER * tid + j;
            const bool ended = ak[j].n < 0;
            const bool served = !ended && (ak[j].need == 0 || (ak[j].need > 0 && ex[1] + ak[j].need <= r.avail));
            const SeqPages s = {ak[j].c, max(ak[j].n, 0), gaps[j] ? kEndedGaps : ended ? kEnded : served ? ex[1] : kNotServed, ex[2]};
            // Ends of what is taken rise with the sequences: the last one's counts.
            const uint64_t takes = __builtin_amdgcn_ballot_w64(served && v[j][1] > 0);
            const uint64_t refused = __builtin_amdgcn_ballot_w64(b < a.B && !served && !ended);
            if (takes && lane == 63 - __builtin_clzll(takes)) atomicMax(&taken_s, ex[1] + v[j][1]);
            if (refused && lane == 0) atomicAdd(&refused_s, __builtin_popcountll(refused));
            if (ONE && gaps[j]) gaps_s = 1;
            if (b < a.B) {
                a.seq_lens[b] = ended ? 0 : ak[j].need == kStuck ? a.cache_lens[b] : (int)min((uint32_t)s.c + (uint32_t)s.n, 0x7fffffffu);
                a.q_start[b] = ex[0];
                if constexpr (ONE) {
                    seq[b] = s;
                    row0[b] = ex[0];
                    move0[b] = ex[3];
                } else {
                    ((int4*)a.info)[b] = int4{s.c, s.n, s.first, s.give};
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) ex[k] += v[j][k];
        }
        __syncthreads();
    }
    if (tid == 0) {
        a.q_start[a.B] = carry[0];
        if constexpr (!ONE) {                      // counters_out may be counters
            a.info[4 * (size_t)a.B] = r.head;
            a.info[4 * (size_t)a.B + 1] = r.avail;
        }
        const int head = r.head + taken_s;         // < 2 R
        a.counters_out[0] = head - fastdiv(head, dv.ring) * a.ring_size;
        a.counters_out[1] = r.avail - taken_s + min(carry[2], a.ring_size - r.avail);
        a.counters_out[2] = refused_s;
    }
    if constexpr (ONE) {
        constexpr int N = kMapOneTokens / kMapThreads;
        int t[N], b[N], pos[N], slot[N];
#pragma unroll
        for (int j = 0; j < N; j++) t[j] = tid + j * kMapThreads;
        if (tid < a.T) {
            last_not_above(row0, a.B, t, b);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const SeqPages s = seq[b[j]];
                const uint32_t i = (uint32_t)(t[j] - row0[b[j]]);
                // Behind the last row; or new_lens whose sum passes 32 bits.
                const bool none = (uint32_t)t[j] >= (uint32_t)carry[0] || i >= (uint32_t)s.n || t[j] >= a.T;
                pos[j] = none ? -1 : s.c + (int)i;
                slot[j] = none ? -1 : slot_of(a, r, dv, b[j], s, pos[j]);
            }
#pragma unroll
            for (int j = 0; j < N; j++)
                if (t[j] < a.T) {
                    a.positions[t[j]] = pos[j];
                    a.slots[t[j]] = slot[j];
                }
        }
        for (uint32_t i = tid; i < (uint32_t)carry[3]; i += kMapThreads) {   // unsigned: up to 2^31 - 1 of them
            const int x[1] = {(int)i};
            int at[1];
            last_not_above(move0, a.B, x, at);
            move_page(a, r, dv, at[0], seq[at[0]], (int)i - move0[at[0]]);
        }
        for (int b = gaps_s ? wave : a.B; b < a.B; b += kWaves)
            if (seq[b].first == kEndedGaps) give_back_gaps(a, r, b, seq[b], ceil_pages(seq[b].c, P, dv.page), lane);
    }
}

// Workgroups (b, part): sequence b's tokens and pages, shared by its gridDim.y parts;
// b = B: the rows behind the last token.
constexpr int kFillThreads = 256;
__global__ __launch_bounds__(kFillThreads)
void page_map_fill(cf_page_map_args_t a, MapDivs dv, int b0) {
    const int b = b0 + (int)blockIdx.x;
    const uint32_t i0 = blockIdx.y * kFillThreads + threadIdx.x, step = gridDim.y * kFillThreads;
    const uint32_t row0 = (uint32_t)a.q_start[b];
    if (b == a.B) {
        for (uint32_t t = row0 + i0; t < (uint32_t)a.T; t += step) a.positions[t] = a.slots[t] = -1;
        return;
    }
    const RingState r = ring_state((const int32_t*)a.info + 4 * (size_t)a.B, a.ring_size, dv.ring);
    const int4 v = ((const int4*)a.info)[b];
    const SeqPages s = {v.x, v.y, v.z, v.w};
    for (uint32_t i = i0; i < (uint32_t)s.n && row0 + i < (uint32_t)a.T; i += step) {
        const uint32_t t = row0 + i;
        a.positions[t] = s.c + (int)i;
        a.slots[t] = slot_of(a, r, dv, b, s, s.c + (int)i);
    }
    const int before = ceil_pages(s.c, a.page_size, dv.page);
    if (s.first == kEndedGaps) {
        if (blockIdx.y == 0 && threadIdx.x < 64) give_back_gaps(a, r, b, s, before, threadIdx.x);
        return;
    }
    const int moves = s.first == kEnded ? before : last_entry(a, dv.page, (uint32_t)s.c + (uint32_t)s.n) - before;
    for (uint32_t j = i0; j < (uint32_t)moves; j += step) move_page(a, r, dv, b, s, (int)j);
}

// ------------------------------------------------------------------ store ---

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T e[N]; };

// One workgroup per row t: the cosines and sines of its position into LDS, then its K, V
// and Q rows in pieces of VEC elements: 16 bytes, or, where something is not 16-byte
// aligned, 2 (a pair to turn) or 1 (no rotation, any head size).
constexpr int kStoreThreads = 256;
template <typename T, int VEC>
__global__ __launch_bounds__(kStoreThreads)
void page_store(cf_page_store_args_t a, int64_t t0, FastDiv by_page, FastDiv by_pieces) {
    constexpr bool WIDE = VEC * sizeof(T) == 16;
    __shared__ float2 turn[CF_PAGE_ROPE_MAX_DIM / 2];
    const int64_t t = t0 + blockIdx.x;
    const int slot = a.slots[t];
    const int pos = a.rope ? a.positions[t] : 0;
    if (a.rope) {
        for (int i = threadIdx.x; i < a.d / 2; i += kStoreThreads) {
            // The angle in turns: whole ones dropped in 64 bits.
            double w = (double)pos * a.turns[i];
            w -= rint(w);
            float s, c;
            sincospif(2.0f * (float)w, &s, &c);
            turn[i] = float2{c, s};
        }
        __syncthreads();
    }
    const int pieces = a.d / VEC;                  // per head
    auto move = [&](const T* src, T* dst, bool turned, int piece) {
        Pack<T, VEC> x;
        if constexpr (WIDE) x = *(const Pack<T, VEC>*)src;
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) x.e[e] = src[e];
        if constexpr (VEC > 1)
            if (turned)
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 cs = turn[(piece * VEC + e) / 2];
                    const float u = (float)x.e[e], v = (float)x.e[e + 1];
                    x.e[e] = (T)(u * cs.x - v * cs.y);
                    x.e[e + 1] = (T)(u * cs.y + v * cs.x);
                }
        if constexpr (WIDE) *(Pack<T, VEC>*)dst = x;
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) dst[e] = x.e[e];
    };
    const int nkv = a.H_kv * pieces;
    if ((unsigned)slot < (unsigned)a.num_slots) {
        const int page = fastdiv(slot, by_page);
        const int64_t at = (int64_t)page * a.page_stride + (int64_t)(slot - page * a.page_size) * a.row_stride;
        const T* const k = (const T*)a.k + t * a.kv_stride;
        const T* const v = (const T*)a.v + t * a.kv_stride;
        for (int i = threadIdx.x; i < 2 * nkv; i += kStoreThreads) {
            const int which = i >= nkv, j = which ? i - nkv : i;
            const int h = fastdiv(j, by_pieces), piece = j - h * pieces;
            const int64_t to = at + (int64_t)h * a.head_stride + piece * VEC;
            move((which ? v : k) + (int64_t)j * VEC, (which ? (T*)a.v_pages : (T*)a.k_pages) + to, a.rope && !which, piece);
        }
    }
    if (a.q && pos >= 0) {
        const T* const q = (const T*)a.q + t * a.q_stride;
        T* const o = (T*)a.q_out + t * a.q_out_stride;
        for (int i = threadIdx.x; i < a.H_q * pieces; i += kStoreThreads) {
            const int h = fastdiv(i, by_pieces);
            move(q + (int64_t)i * VEC, o + (int64_t)i * VEC, true, i - h * pieces);
        }
    }
}

template <typename T>
int launch_store(const cf_page_store_args_t& a, hipStream_t st) {
    constexpr int kWide = 16 / sizeof(T);
    const uint64_t ptrs = (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)(uintptr_t)a.k_pages |
                          (uint64_t)(uintptr_t)a.v_pages | (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.q_out;
    const uint64_t steps = (uint64_t)a.kv_stride | (uint64_t)a.q_stride | (uint64_t)a.q_out_stride |
                           (uint64_t)a.page_stride | (uint64_t)a.row_stride | (uint64_t)a.head_stride | (uint64_t)a.d;
    const bool wide = ptrs % 16 == 0 && steps % kWide == 0;
    const FastDiv by_page = fastdiv_make(a.page_size);
    constexpr int64_t kMost = 1 << 23;             // rows of a launch: a grid has less than 2^32 threads
    for (int64_t t0 = 0; t0 < a.T; t0 += kMost) {
        const dim3 grid((unsigned)(a.T - t0 < kMost ? a.T - t0 : kMost)), block(kStoreThreads);
        if (wide) hipLaunchKernelGGL((page_store<T, kWide>), grid, block, 0, st, a, t0, by_page, fastdiv_make(a.d / kWide));
        else if (a.rope) hipLaunchKernelGGL((page_store<T, 2>), grid, block, 0, st, a, t0, by_page, fastdiv_make(a.d / 2));
        else hipLaunchKernelGGL((page_store<T, 1>), grid, block, 0, st, a, t0, by_page, fastdiv_make(a.d));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return 0;
}

}  // namespace

// Several launches need, per sequence, Asked or SeqPages, and once the ring's counters as they were.
extern "C" size_t cf_page_map_info_ints(int32_t B, int32_t T) {
    return B <= kMapOneSeqs && T <= kMapOneTokens ? 0 : 4 * (size_t)B + 2;
}

extern "C" int cf_launch_page_map(const cf_page_map_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    if (a->B <= 0 || a->T < 0 || a->page_size <= 0 || a->ring_size <= 0 || a->ring_size > (1 << 30))
        return (int)hipErrorInvalidValue;
    const MapDivs dv = {fastdiv_make(a->page_size), fastdiv_make(a->ring_size)};
    if (cf_page_map_info_ints(a->B, a->T) == 0) {
        hipLaunchKernelGGL((page_map_scan<true, 1, false>), dim3(1), dim3(kMapThreads), 0, st, *a, dv);
        return (int)hipGetLastError();
    }
    if (!a->info) return (int)hipErrorInvalidValue;
    // Four sequences a thread for more than a workgroup has threads: their loads wait together.
    hipError_t e;
    if (a->B <= kMapThreads) {
        hipLaunchKernelGGL((page_map_scan<false, 1, false>), dim3(1), dim3(kMapThreads), 0, st, *a, dv);
    } else {
        hipLaunchKernelGGL(page_map_ask, dim3((unsigned)((a->B - 1) / kAskThreads + 1)), dim3(kAskThreads), 0, st, *a, dv.page);
        if ((e = hipGetLastError()) != hipSuccess) return (int)e;
        hipLaunchKernelGGL((page_map_scan<false, 4, true>), dim3(1), dim3(kMapThreads), 0, st, *a, dv);
    }
    if ((e = hipGetLastError()) != hipSuccess) return (int)e;
    // Long chunks of few sequences are shared by several workgroups.
    const unsigned parts = (unsigned)(a->T / 2048 < 1 ? 1 : a->T / 2048 > 2048 / a->B ? (2048 / a->B < 1 ? 1 : 2048 / a->B) : a->T / 2048);
    constexpr int kMost = 1 << 23;                 // sequences of a launch: a grid has less than 2^32 threads
    for (int64_t b0 = 0; b0 <= a->B; b0 += kMost) {
        const unsigned n = (unsigned)(a->B + 1 - b0 < kMost ? a->B + 1 - b0 : kMost);
        hipLaunchKernelGGL(page_map_fill, dim3(n, parts), dim3(kFillThreads), 0, st, *a, dv, (int)b0);
        if ((e = hipGetLastError()) != hipSuccess) return (int)e;
    }
    return 0;
}

extern "C" int cf_launch_page_store(const cf_page_store_args_t* a, void* stream) {
    if (a->T <= 0 || a->d <= 0 || a->H_kv <= 0) return (int)hipErrorInvalidValue;
    return a->elem == CF_ELEM_F16 ? launch_store<_Float16>(*a, (hipStream_t)stream)
                                  : launch_store<float>(*a, (hipStream_t)stream);
}
