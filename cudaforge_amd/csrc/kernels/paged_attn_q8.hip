// paged_attn_q8.hip — attention of chunks of new tokens over a paged KV cache of 8-bit numbers
// (gfx950).  The sums, rows, positions and tiles are those of paged_attn.hip; K and V are codes times the
// power of two of their block.  Times below are of one call among others on one MI355X; "n rows over m"
// is n new tokens of a sequence of m positions in all, and heads are 32 of 128 over 8 KV heads and rows
// fp16 where none are named.

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
    const int lane = unit_lane();
    const int seen = min(min(s.len - s.n + tok + 1, s.len), key1);
    const int kvh = h / (a.at.H_q / a.at.H_kv);
    const int32_t* const table = a.at.table + (size_t)b * a.at.max_pages;
    const T* const q = (const T*)a.at.q + (int64_t)(s.row0 + tok) * a.at.q_stride + (int64_t)h * d;
    const uint8_t* const k = (const uint8_t*)a.at.k + (int64_t)kvh * a.at.head_stride;
    const uint8_t* const v = (const uint8_t*)a.at.v + (int64_t)kvh * a.at.head_stride;
    const float c = a.at.scale * kLog2e;
    float m = -INFINITY, acc[DIMS];
    LongSum l_run;
#pragma unroll
    for (int i = 0; i < DIMS; i++) acc[i] = 0.0f;
#pragma clang loop unroll(disable)
    for (uint32_t at0 = (uint32_t)key0; at0 < (uint32_t)max(seen, 0); at0 += 64) {    // unsigned: up to 2^31 positions
        const int k0 = (int)at0, key = k0 + lane;
        int64_t at = -1;
        int vpower = 0;
        float x = -INFINITY;
        if (key < seen) {
            const Cell cell = cell_of(a, dv, table, key);
            at = cell.at;
            if (at >= 0) {
                vpower = a.v_scales[cell.power + kvh];
                const float kpower = power_bits(a.k_scales[cell.power + kvh]);
                float dot = 0.0f;
#pragma clang loop unroll(disable)
                for (int e = 0; e < d; e++) dot = __builtin_fmaf((float)q[e], codes_f32<false>(k[at + e], kpower)[0], dot);
                x = dot * c;
            }
        }
        const float m_new = fmaxf(m, wave_max(x));
        // Positions that count, whatever they weigh: a NaN V touches the row from any of them.
        const uint64_t counts = __builtin_amdgcn_ballot_w64(key < seen && at >= 0);
        if (!counts) continue;
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2f(m - m_use), p = exp2f(x - m_use);
        m = m_new;
        l_run.scale(alpha);
        l_run.add(wave_sum(p));
        // Codes are few different numbers, so that roundings of a long sum would lean one way: 64
        // positions' by themselves first.
        float part[DIMS];
#pragma unroll
        for (int i = 0; i < DIMS; i++) part[i] = 0.0f;
#pragma clang loop unroll(disable)
        for (int j = 0; j < min(64, seen - k0); j++) {
            if (!(counts >> j & 1)) continue;  // not attended: its V may hold anything
            const int pbits = __builtin_amdgcn_readlane(__float_as_int(p), j);
            const float pj = __int_as_float(pbits);
            const int64_t row = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32) |
                                          (uint32_t)__builtin_amdgcn_readlane((int)at, j));
            const float power = power_bits(__builtin_amdgcn_readlane(vpower, j));
            if (pbits == 0) {                  // of weight 0: NaN only
#pragma unroll
                for (int i = 0; i < DIMS; i++)
                    if (lane + 64 * i < d) {
                        const float y = codes_f32<false>(v[row + lane + 64 * i], power)[0];
                        if (y != y) part[i] = y;
                    }
                continue;
            }
#pragma unroll
            for (int i = 0; i < DIMS; i++)
                if (lane + 64 * i < d)
                    part[i] = __builtin_fmaf(pj, codes_f32<false>(v[row + lane + 64 * i], power)[0], part[i]);
        }
#pragma unroll
        for (int i = 0; i < DIMS; i++) acc[i] = __builtin_fmaf(acc[i], alpha, part[i]);
    }
    const float l = l_run.sum();
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

// ---- On the matrix cores: d = 64 or 128, blocks of a multiple of 16 positions ----
//
// Codes go to LDS as they are and become 16-bit operands on their way to the matrix cores, one
// instruction for two, the power of their block with them: exact, so nothing is scaled afterwards.
// fp16 rows go with fp16 codes.  FP32 rows go with bf16 codes, and Q and the weights of V as sums of
// three bf16 numbers, whose 24 bits are FP32's own: three products for one, at 16 times the FP32
// MFMA's rate.

// T rows: what the matrix cores take, and in how many parts Q and the weights.
template <typename T> struct Parts;
template <> struct Parts<_Float16> {
    typedef _Float16 half_t;
    static constexpr int Q = 1, P = 2;
};
template <> struct Parts<float> {
    typedef __bf16 half_t;
    static constexpr int Q = 3, P = 3;
};
// x and y as sums of N numbers of B, part by part into elements e and e + 1 of `to`.  Two by two, as the
// converting instruction takes them (FP32 chunk below: 27.0 us, one at a time 28.3).
template <int N, typename B, typename V>
__device__ __forceinline__ void split_into(V (&to)[N], int e, float x, float y) {
    typedef B two_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; i++) {
        const two_t b = __builtin_convertvector(f2_t{x, y}, two_t);
        to[i][e] = b[0];
        to[i][e + 1] = b[1];
        x -= (float)b[0];
        y -= (float)b[1];
    }
}

// Rows of D codes in LDS and in lanes, in 16-byte chunks.
template <int D> struct Rows8 {
    static constexpr int CPR = D / 16;                 // chunks per row
    static constexpr int RPI = 64 / CPR;               // rows per DMA instruction (1 KB)
    static constexpr int NI = 16 / RPI;                // DMA instructions per 16 rows
    static constexpr int KF = D / 64;                  // chunks of a K row a lane takes
    static constexpr int UT = D / 16;                  // 16-dim tiles of O^T
    static __device__ __forceinline__ int drow(int lane) { return lane / CPR; }
    static __device__ __forceinline__ int dch(int lane) { return lane % CPR; }
    // Chunks are swizzled so that 8 lanes on 8 rows (K) and 16 lanes on 8 rows (V, rows 4 lq .. + 3
    // of an even group of 16 and of the odd one behind it) touch every bank once.
    static __device__ __forceinline__ int kswz(int row) { return D == 128 ? row & 7 : (row >> 1) & 3; }
    static __device__ __forceinline__ int vswz(int row, int odd) { return D == 128 ? (row & 3) | odd << 2 : ((row >> 1) & 1) | odd << 1; }
    // Lane (lr, lq) takes chunks 4 f + lq of K row lr: dims 64 f + 16 lq .. + 15, the k-slots of MFMA
    // steps 2 f and 2 f + 1.
    static __device__ __forceinline__ void k_offsets(int (&rd)[KF], int lane) {
        const int lr = lane & 15, lq = lane >> 4;
#pragma unroll
        for (int f = 0; f < KF; f++) rd[f] = lr * D + 16 * ((4 * f + lq) ^ kswz(lr));
    }
    // V (ds_read_tr8): positions 4 lq .. + 3 of two groups of 16, dims 16 u .. + 15.
    static __device__ __forceinline__ void v_offsets(int (&rd)[UT], int lane) {
        const int lr = lane & 15, lq = lane >> 4, odd = lr >> 3, row = 4 * lq + ((lr >> 1) & 3);
#pragma unroll
        for (int u = 0; u < UT; u++) rd[u] = (16 * odd + row) * D + 16 * (u ^ vswz(row, odd)) + 8 * (lr & 1);
    }
};

// The next 64 groups of 16 positions of a range, one per lane: where each starts (bytes), which
// of its positions count, and the powers of its K and V (those of a group of none are 2^0).
struct Groups8 {
    const int32_t* table;
    int lo, hi, info;        // lane: base + lane; info: positions, power of K << 16, of V << 24
    __device__ __forceinline__ void find(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, int kvh, int key, int key1) {
        const int page = table[fastdiv(min(key, a.at.max_pages * a.at.page_size - 1), pl.by_page)];
        const Group g = group_of(a.at, pl, page, key, key1);
        const int in = key - fastdiv(key, pl.by_page) * a.at.page_size;
        const int64_t p = ((int64_t)(g.mask ? page : 0) * (a.at.page_size / a.block) + fastdiv(in, dv.block)) * a.at.H_kv + kvh;
        const uint32_t kp = a.k_scales[p], vp = a.v_scales[p];
        lo = (int)g.at;
        hi = (int)(g.at >> 32);
        info = (int)(g.mask ? g.mask | kp << 16 | vp << 24 : 0x7f7f0000u);
    }
    __device__ __forceinline__ void load(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, int kvh, int base,
                                         int key0, int key1) {
        find(a, pl, dv, kvh, key0 + (base + unit_lane()) * 16, key1);
        asm volatile("" : "+v"(lo), "+v"(hi), "+v"(info));    // they have arrived
    }
    __device__ __forceinline__ int64_t at(int i) const {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i & 63) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane(lo, i & 63));
    }
    __device__ __forceinline__ uint32_t what(int i) const { return (uint32_t)__builtin_amdgcn_readlane(info, i & 63); }
};
__device__ __forceinline__ float k_power(uint32_t info) { return __uint_as_float((info << 7) & 0x7f800000u); }
__device__ __forceinline__ float v_power(uint32_t info) { return __uint_as_float((info >> 1) & 0x7f800000u); }

// 16 zeros, made where they are used: kept in registers for a whole kernel, wide tiles had no room.
__device__ __forceinline__ uint4 zeros() {
    uint32_t z = 0;
    asm volatile("" : "+v"(z));
    return uint4{z, z, z, z};
}

// Which of some V are NaN: bit 7 of the byte of each element of the lane's 16-byte chunk; and whether numbers
// among them are past the range of B, infinite on the matrix cores.
struct Nans {
    uint32_t w[4] = {0, 0, 0, 0};
    uint32_t past = 0;
    __device__ __forceinline__ bool any_but(const Nans& x) const {
        return ((w[0] & ~x.w[0]) | (w[1] & ~x.w[1]) | (w[2] & ~x.w[2]) | (w[3] & ~x.w[3])) != 0;
    }
};
// The least code (without its sign) that is past the range of B at a power: values reach 2^16 (fp16) or 2^128
// (bf16).  128: none.
template <typename B> __device__ __forceinline__ int least_past(int power) {
    const int e = (std::is_same<B, _Float16>::value ? 150 : 262) - power;      // exponent bits of that
    return e > 15 ? 128 : e > 0 ? e << 3 : max(4 >> min(-e, 2), 1);
}
template <typename B, int D>
__device__ __forceinline__ void find_nan(const cf_paged_q8_args_t& a, const Q8Divs& dv, int b, int kvh, int from, int to, Nans& found) {
    using R = Rows8<D>;
    const int lane = unit_lane(), sub = R::drow(lane);
    const int32_t* const table = a.at.table + (size_t)b * a.at.max_pages;
    const uint8_t* const v = (const uint8_t*)a.at.v + (int64_t)kvh * a.at.head_stride + 16 * R::dch(lane);
    Nans mine;
#pragma clang loop unroll(disable)
    for (int p0 = from; p0 < to; p0 += 64) {
        const int key = min(p0 + lane, to - 1);
        const Cell cell = cell_of(a, dv, table, key);
        const int power = cell.at >= 0 ? a.v_scales[cell.power + kvh] : 0;
#pragma clang loop unroll(disable)
        for (int r = sub; r < 64; r += R::RPI) {
            const int64_t row = (int64_t)((uint64_t)(uint32_t)__shfl((int)(cell.at >> 32), r) << 32 | (uint32_t)__shfl((int)cell.at, r));
            const int its_power = __shfl(power, r);
            const uint32_t whole = its_power == 255 ? 0x7f7f7f7fu : 0u, to_past = (uint32_t)(128 - least_past<B>(its_power)) * 0x01010101u;
            const uint4 x = row < 0 ? uint4{} : *(const uint4*)(v + row);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t nan = (((w[i] | whole) & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                mine.w[i] |= nan;
                mine.past |= ((w[i] & 0x7f7f7f7fu) + to_past) & 0x80808080u & ~nan;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int step = R::CPR; step < 64; step *= 2) mine.w[i] |= __shfl_xor(mine.w[i], step);
        found.w[i] |= mine.w[i];
    }
    found.past |= __builtin_amdgcn_ballot_w64(mine.past != 0) != 0;
}

// Rows row0 + bit of a unit (a bit of `rows` each), computed and stored by this wave, where a sum is NaN
// while l is a number (spoilt).  An element is NaN where a V that its row sees is; where V are that it does
// not see, or V past the range of the products' type are about (0 times those is NaN too), the plain
// loop computes the row again.
template <typename T, int D, int TM>
__device__ __forceinline__ void mend_rows8(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, const Unit& un,
                                           int kvh, const Work& w, int row0, uint32_t rows) {
    using R = Rows8<D>;
    using B = typename Parts<T>::half_t;
    const int lane = unit_lane();
    wait_vm<0>();                                             // what it stored is stored
    Nans seen;
    int upto = w.key0;
    for (; rows; rows &= rows - 1) {
        const int row = row0 + __builtin_ctz(rows);
        const RowAt at = row_at(pl, pl.G, kvh, w.R0 + row);
        const int sees = max(min(min(w.base + at.tok, un.s.len), w.key1), upto);     // rises with the rows
        find_nan<B, D>(a, dv, un.b, kvh, upto, sees, seen);
        upto = sees;
        Nans hidden;
        find_nan<B, D>(a, dv, un.b, kvh, sees, w.key1, hidden);
        float* const rec = un.n_ranges > 1 ? record_of<TM, D>(a.at, pl, un, kvh) : nullptr;
        T* const o = (T*)a.at.o + ((int64_t)(un.s.row0 + at.tok) * a.at.H_q + at.h) * D;
        if (seen.past | hidden.past || __builtin_amdgcn_ballot_w64(hidden.any_but(seen)) ||
            !__builtin_amdgcn_ballot_w64(seen.any_but(Nans{}))) {
            plain_row_q8<T, D / 64>(a, dv, un.s, un.b, at.tok, at.h, D, w.key0, w.key1, rec ? rec + row : nullptr, TM,
                                    rec + 2 * TM + row * D);
            continue;
        }
        if (lane >= R::CPR) continue;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (!((seen.w[e / 4] >> (8 * (e % 4) + 7)) & 1)) continue;
            if (rec) rec[2 * TM + row * D + 16 * lane + e] = NAN;
            else o[16 * lane + e] = (T)NAN;
        }
    }
}

// ---- Up to 16 rows, one wave with a ring of its own: no barrier. ----
template <int D, int STAGES = 2> struct Narrow8 {
    static constexpr int BK = 32, NS = STAGES;
    static constexpr int TILE = BK * D, STAGE = 2 * TILE;    // bytes
    static constexpr int RING = NS * STAGE;
};

// Positions [key0, key1) (key0 a multiple of 16) of (b, kvh) for the unit's rows: leaves m and
// the lane's share of l, and lane (lr, lq) with dims 16 u + 4 lq .. + 3 of row lr.
template <typename T, int D, int STAGES = 2>
__device__ __forceinline__ void narrow_range8(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, uint8_t* ring,
                                              const SeqRows& s, int b, int kvh, const Work& w, int key0, int key1,
                                              f4_t (&acc)[D / 16], float& m_run, float& l_run) {
    using R = Rows8<D>;
    using N = Narrow8<D, STAGES>;
    using B = typename Parts<T>::half_t;
    using C = Codes<B>;
    typedef typename C::eight_t eight_t;
    typedef T q8_t __attribute__((ext_vector_type(8)));
    constexpr int BK = N::BK, NG = BK / 16, NS = N::NS, TILE = N::TILE, STAGE = N::STAGE, NI = R::NI, NL = 2 * NG * NI, UT = R::UT;
    constexpr int QP = Parts<T>::Q, PP = Parts<T>::P, KS = D / 32;
    static_assert(NS * NL < 64, "vmcnt range");
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int drow = R::drow(lane), dch = R::dch(lane);
#pragma unroll
    for (int u = 0; u < UT; u++) acc[u] = f4_t{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = 0.0f;
    LongSum l;
    const int nblk = key1 > key0 ? (key1 - key0 + BK - 1) / BK : 0;
    if (nblk == 0) return;
    const float c = a.at.scale * kLog2e;
    const int seen = min(w.base + fastdiv(w.R0 + min(lr, w.n_rows - 1), pl.by_group), s.len);
    const int seen_all = min(w.base + fastdiv(w.R0, pl.by_group), s.len);

    // B operand Q^T: in step ks lane (lr, lq) holds dims 64 (ks / 2) + 16 lq + 8 (ks % 2) .. + 7 of row lr.  Its
    // loads wait together with those of the table.
    q8_t q[KS];
    {
        const RowAt at = row_at(pl, pl.G, kvh, w.R0 + min(lr, w.n_rows - 1));
        const T* const from = (const T*)a.at.q + (int64_t)(s.row0 + at.tok) * a.at.q_stride + at.h * D + 16 * lq;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] = *(const CF_GLOBAL q8_t*)(from + 64 * (ks / 2) + 8 * (ks % 2));
    }
    uint32_t koff[NI], voff[NI][2];
#pragma unroll
    for (int u = 0; u < NI; u++) {
        const int row = R::RPI * u + drow;
        koff[u] = (uint32_t)row * (uint32_t)a.at.row_stride + 16 * (dch ^ R::kswz(row));
        voff[u][0] = (uint32_t)row * (uint32_t)a.at.row_stride + 16 * (dch ^ R::vswz(row, 0));
        voff[u][1] = (uint32_t)row * (uint32_t)a.at.row_stride + 16 * (dch ^ R::vswz(row, 1));
    }
    int k_rd[R::KF], v_rd[UT];
    R::k_offsets(k_rd, lane);
    R::v_offsets(v_rd, lane);
    const uint32_t ring_base = __builtin_amdgcn_readfirstlane(lds_offset(ring));
    const uint8_t* const kp = (const uint8_t*)a.at.k + (int64_t)kvh * a.at.head_stride;
    const uint8_t* const vp = (const uint8_t*)a.at.v + (int64_t)kvh * a.at.head_stride;
    Groups8 groups = {a.at.table + (size_t)b * a.at.max_pages, 0, 0, 0};
    groups.load(a, pl, dv, kvh, 0, key0, key1);

    uint32_t info[NS][NG];
    auto issue = [&](int blk, auto stage_c) {
        constexpr int stage = decltype(stage_c)::value;
        if (blk > 0 && blk % (64 / NG) == 0) groups.load(a, pl, dv, kvh, blk * NG, key0, key1);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const int64_t at = groups.at(blk * NG + g);
            const uint32_t lds = ring_base + (uint32_t)(stage * STAGE + 16 * g * D);
#pragma unroll
            for (int u = 0; u < NI; u++) {
                lds_dma16_s(koff[u], kp + at, lds + u * 1024u);
                lds_dma16_s(voff[u][g & 1], vp + at, lds + (uint32_t)TILE + u * 1024u);
            }
            info[stage][g] = groups.what(blk * NG + g);
        }
    };

    eight_t qf[KS][QP];
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            if constexpr (QP == 1) {
                qf[ks][0][e] = q[ks][e];
                qf[ks][0][e + 1] = q[ks][e + 1];
            } else {
                split_into<QP, B>(qf[ks], e, q[ks][e], q[ks][e + 1]);
            }
        }
    wait_lds_reads();                                         // what the ring held before
    static_for<NS - 1>([&](auto i) {
        if (i < nblk) issue(i, i);
    });

    auto step = [&](int bi, auto stage_c) {
        constexpr int stage = decltype(stage_c)::value;
        if (bi + NS - 1 < nblk) {
            wait_lds_reads();                                 // the last reads of that stage
            issue(bi + NS - 1, std::integral_constant<int, (stage + NS - 1) % NS>{});
        }
        wait_ahead<NL, NS - 1>(min(NS - 1, nblk - 1 - bi));
        uint64_t mk = 0;
        uint32_t all = 0xffff;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            all &= info[stage][g];
            mk |= (uint64_t)(info[stage][g] & 0xffff) << (16 * g);
        }
        const bool full = (all & 0xffff) == 0xffff;
        uint8_t* const st = ring + stage * STAGE;
        if (!full) {
            // V where nothing counts: 0, as p = 0 times whatever it holds need not be.
#pragma unroll
            for (int u = 0; u < NG * NI; u++) {
                const int row = R::RPI * u + drow;
                if (!((mk >> row) & 1)) *(uint4*)(st + TILE + row * D + 16 * dch) = zeros();
            }
            wait_lds_reads();
        }
        const int k0 = key0 + bi * BK;
        // S^T: sc[t][i] = score(key k0 + 16 t + 4 lq + i, row lr).
        f4_t sc[NG];
#pragma unroll
        for (int t = 0; t < NG; t++) {
            sc[t] = f4_t{0.f, 0.f, 0.f, 0.f};
            const float power = k_power(info[stage][t]);
#pragma unroll
            for (int f = 0; f < R::KF; f++) {
                const uint4 x = *(const uint4*)(st + 16 * t * D + k_rd[f]);
                const eight_t k0f = C::of(x.x, power, x.y, power), k1f = C::of(x.z, power, x.w, power);
#pragma unroll
                for (int i = QP - 1; i >= 0; i--) {           // small parts first
                    sc[t] = C::mfma(k0f, qf[2 * f][i], sc[t]);
                    sc[t] = C::mfma(k1f, qf[2 * f + 1][i], sc[t]);
                }
            }
        }
        if (!full || k0 + BK > seen_all) hide(sc, mk, seen - k0, lane);
        float mloc = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
        for (int t = 1; t < NG; t++) mloc = fmaxf(mloc, fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])));
        mloc = low_max<T>(max_xor32(max_xor16(mloc)), c);     // -inf if the row sees nothing here
        float alpha;
        if (move_max<T>(mloc, m_run, alpha)) {
            l.scale(alpha);
#pragma unroll
            for (int u = 0; u < UT; u++) acc[u] *= alpha;
        }
        const float m_use = m_run == -INFINITY ? 0.0f : m_run;
        // O^T += V^T P^T, the lane's own scores being its B operand: in 32-key step j, k-slot e of lane
        // group lq is key 32 j + 16 (e / 4) + 4 lq + e % 4.  The weights in parts, so that their rounding
        // leaves the result: this wave waits on memory, not on products.
        float l_blk = 0.0f;
        eight_t pf[NG / 2][PP];
#pragma unroll
        for (int t = 0; t < NG; t++)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], c, -m_use));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i + 1], c, -m_use));
                l_blk += p0;
                l_blk += p1;
                split_into<PP, B>(pf[t / 2], 4 * (t & 1) + i, p0, p1);
            }
        l.add(l_blk);
#pragma unroll
        for (int j = 0; j < NG / 2; j++) {
            const float p0 = v_power(info[stage][2 * j]), p1 = v_power(info[stage][2 * j + 1]);
#pragma unroll
            for (int u = 0; u < UT; u++) {
                const lds_i2_t x = ds_read_tr8(st + TILE + 32 * j * D + v_rd[u]);
                const eight_t vf = C::of((uint32_t)x[0], p0, (uint32_t)x[1], p1);
#pragma unroll
                for (int i = PP - 1; i >= 0; i--) acc[u] = C::mfma(vf, pf[j][i], acc[u]);
            }
        }
    };
    for_each_stage<NS>(nblk, step);
    l_run = l.sum();
}

// A wave per unit, the units of neighbouring KV heads in one workgroup: they read the same
// cache rows at about the same time.  HBM bounds it: 64 rows over 4096 each, 537 MB, 101 us (5.3 TB/s);
// 16 rows over 1778 to 4096 positions, 114 MB, 29.2 us, 4 of them the merge's and 3 until the first
// codes are there (launch, lengths, table, powers).  Two stages of a ring: with 3 the same 16 rows take
// 30.0, with 4, which leave room for one workgroup a CU, 32.7.
template <int D> struct Heads8 {
    static constexpr int WAVES = 4, NS = 2;
    static constexpr int RING = Narrow8<D, NS>::RING;
    static constexpr int FIT = 160 * 1024 / (WAVES * RING), PER_CU = FIT < 4 ? FIT : 4;
};
template <typename T, int D>
__global__ __launch_bounds__(256, (Heads8<D>::PER_CU))
void paged_heads8(cf_paged_q8_args_t a, PagedPlan pl, Q8Divs dv) {
    using H = Heads8<D>;
    constexpr int BK = Narrow8<D>::BK, RING = H::RING;
    __shared__ __attribute__((aligned(16))) uint8_t ring_all[H::WAVES * RING];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const Geometry<16, BK, 1, true, true> geo(a.at, pl);
    if (geo.lists_cut_tiles()) return;
    for (int unit = (int)blockIdx.x * H::WAVES + wave;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.at.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        const Work w = unit_work<16, BK>(a.at, pl, un);
        const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
        f4_t acc[D / 16];
        float m, l;
        narrow_range8<T, D, H::NS>(a, pl, dv, ring_all + wave * RING, un.s, un.b, kvh, w, w.key0, w.key1, acc, m, l);
        l = add_xor32(add_xor16(l));
        const uint32_t again = rows_of_16(lr < w.n_rows && spoilt(acc, l));
        if (lr < w.n_rows) {
            const RowOut out = row_out<T, D, 16>(a.at, pl, un, kvh, w, lr, m, l, lq == 0);
#pragma unroll
            for (int u = 0; u < D / 16; u++) put4<T>(out, 16 * u + 4 * lq, acc[u]);
        }
        if (again) mend_rows8<T, D, 16>(a, pl, dv, un, kvh, w, 0, again);
    }
}

// Up to 16 rows by all waves of a workgroup: each takes a share of the unit's positions, and they
// join their m, l and sums in LDS (WAVES rings at `lds`, one each).  True where rows that this wave
// stored are spoilt.  Latency bounds it: an FP32 row of 12 heads of 64 over 257 6.6 us, 16 rows over 512 8.8.
template <typename T, int D, int TM, int WAVES>
__device__ __forceinline__ bool narrow_unit8(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, uint8_t* lds,
                                             const Unit& un, int kvh, const Work& w) {
    constexpr int RING = Narrow8<D>::RING, BK = Narrow8<D>::BK, LD = D + 4;
    static_assert(16 * (LD + 2) * 4 <= RING, "a wave's rows fit its ring");
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint8_t* const ring = lds + wave * RING;
    const int blocks = w.key1 > w.key0 ? (w.key1 - w.key0 + BK - 1) / BK : 0;
    const int per = (blocks + WAVES - 1) / WAVES * BK;
    const int k0 = min(w.key0 + wave * per, w.key1), k1 = min(k0 + per, w.key1);
    f4_t acc[D / 16];
    float m, l;
    narrow_range8<T, D>(a, pl, dv, ring, un.s, un.b, kvh, w, k0, k1, acc, m, l);
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
    for (int i = 64 * wave + lane; i < w.n_rows * (D / 4); i += 64 * WAVES) {
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
        put4<T>(row_out<T, D, TM>(a.at, pl, un, kvh, w, row, M, L, d4 == 0), 4 * d4, sum);
    }
    __syncthreads();                                          // the rings, before the next unit
    return __builtin_amdgcn_ballot_w64(again) != 0;
}

// The rows that the wave stored there.
template <typename T, int D, int TM, int WAVES>
__device__ __forceinline__ void mend_narrow8(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, const Unit& un,
                                             int kvh, const Work& w) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t rows = 0;
    for (int r = 0; r < w.n_rows; r++)
        if (r / (256 / D) % WAVES == wave) rows |= 1u << r;
    mend_rows8<T, D, TM>(a, pl, dv, un, kvh, w, 0, rows);
}

constexpr int kSplitWaves = 8;
template <typename T, int D>
__global__ __launch_bounds__(64 * kSplitWaves, 2)
void paged_split8(cf_paged_q8_args_t a, PagedPlan pl, Q8Divs dv) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kSplitWaves * Narrow8<D>::RING];
    const Geometry<16, 64, 1, false> geo(a.at, pl);
    for (int unit = (int)blockIdx.x;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.at.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        const Work w = unit_work<16, 64>(a.at, pl, un);
        if (narrow_unit8<T, D, 16, kSplitWaves>(a, pl, dv, lds, un, kvh, w)) mend_narrow8<T, D, 16, kSplitWaves>(a, pl, dv, un, kvh, w);
    }
}

// ---- Wide tiles: 8 waves of 16 NJ rows through one ring of 64-position blocks. ----
// A wave loads its eighth of a block's codes into registers a turn ahead, and puts them into the ring
// as 16-bit numbers: each code is converted once for the tile, and what the products read is as in
// attention over a 16-bit cache.  The two waves of a SIMD, w and w + 4, take turns: with phases cut by
// barriers, waves 0 .. 3 run products while waves 4 .. 7 run softmax, then the other way round.
// Products of turn i are S(i) = K_i Q^T and O += V_{i-1} P(i-1), so a stage of the ring is K_i with
// V_{i-1}.  Turn i of waves 0 .. 3 takes phases 2 i (products) and 2 i + 1, of the others 2 i + 1 and
// 2 i + 2.  Stage i, which turn i - 2 has left by the end of phase 2 i - 3, is written during the softmax
// phases before it, 2 i - 1 of waves 0 .. 3 and 2 i - 2 of the others: two stages do.
// The weights of V in two fp16 parts (FP32 rows: three of bf16), so that their rounding leaves the result.  In
// one part they cost half of the products with V, but the result is then off by 2.3e-4 of its size in the root
// mean square over 8192 positions and 2.8e-4 over 742 to 2717, so 2.07e-4 in two, which is its own rounding,
// and which rows that meets depends on how the whole batch is cut.
// NJ = 2: 2048 rows over 8192, 241 GFLOP in 330 us (730 TFLOP/s; 361 and 1090 with the second product; a large
// library product 1144; in one part 245 us): the products bound it.  FP32 (NJ = 1, three products for one): 840
// rows of 16 heads of 64 over 300 to 1129 positions 27.0 us, 3 rounds of launch and latency among them.
template <typename T, int D, int NJ> struct Wide8 {
    static constexpr int TM = 128 * NJ, BK = 64, NS = 2;
    static constexpr int TILE = BK * D, STAGE = 2 * TILE;    // 16-bit numbers
    static constexpr int QB = TM * D * (int)sizeof(T);       // bytes of Q, behind the stages
    static constexpr int LDS = NS * STAGE * 2 + QB > 8 * Narrow8<D>::RING ? NS * STAGE * 2 + QB : 8 * Narrow8<D>::RING;
};

// An address in scalar registers, which stays there: what a lane adds to it is 32 bits wide.
__device__ __forceinline__ const CF_GLOBAL uint8_t* uniform_at(const uint8_t* p) {
    const uint64_t x = (uint64_t)(uintptr_t)p;
    uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)x), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32));
    asm volatile("" : "+s"(lo), "+s"(hi));
    return (const CF_GLOBAL uint8_t*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// Returns the wave's rows that are spoilt, a bit each.
template <typename T, int D, int NJ>
__device__ __forceinline__ uint32_t wide8_unit(const cf_paged_q8_args_t& a, const PagedPlan& pl, const Q8Divs& dv, uint8_t* lds,
                                               const Unit& un, int kvh, const Work& w) {
    using R = Rows<_Float16, D>;
    using W = Wide8<T, D, NJ>;
    using B = typename Parts<T>::half_t;
    using C = Codes<B>;
    typedef typename C::eight_t eight_t;
    constexpr int BK = W::BK, TILE = W::TILE, STAGE = W::STAGE, UT = R::UT, NF = R::NF;
    constexpr int QP = Parts<T>::Q, PP = Parts<T>::P;
    constexpr int QC = D * (int)sizeof(T) / 16, QR = 64 / QC, QE = 16 / (int)sizeof(T);
    constexpr int CB = D / 8;                                // codes of a lane
    const int lane = unit_lane(), lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int G = pl.G;
    const float c = a.at.scale * kLog2e;
    const int wrow = 16 * NJ * wave;
    const bool active = wrow < w.n_rows;
    const int n = w.key1 > w.key0 ? (w.key1 - w.key0 + BK - 1) / BK : 0;
    f4_t acc[NJ][UT];
    LongSum l_run[NJ];
    float m_run[NJ];
    int seen[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        m_run[j] = -INFINITY;
#pragma unroll
        for (int u = 0; u < UT; u++) acc[j][u] = f4_t{0.f, 0.f, 0.f, 0.f};
        seen[j] = min(w.base + fastdiv(w.R0 + min(wrow + 16 * j + lr, w.n_rows - 1), pl.by_group), un.s.len);
    }
    const int seen_all = min(w.base + fastdiv(w.R0 + min(wrow, w.n_rows - 1), pl.by_group), un.s.len);

    if (n > 0) {
        // This wave's rows of a block: 8 half + 0 .. 7 of group `grp`, eight lanes a row.
        const int grp = wave >> 1, row = 8 * (wave & 1) + (lane >> 3), col = lane & 7;
        const uint32_t off = (uint32_t)row * (uint32_t)a.at.row_stride + CB * col;
        const int to_k = (16 * grp + row) * D + 8 * ((CB / 8 * col) ^ kswz<_Float16, D>(row));
        const int to_v = TILE + (16 * grp + row) * D + 8 * ((CB / 8 * col) ^ vswz<_Float16, D>(row));
        int k_rd[NF], v_rd[UT];
        R::k_offsets(k_rd, lane);
        R::v_offsets(v_rd, lane);
        _Float16* const ring = (_Float16*)lds;
        uint8_t* const qlds = lds + W::NS * STAGE * 2;
        const uint8_t* const kp = (const uint8_t*)a.at.k + (int64_t)kvh * a.at.head_stride;
        const uint8_t* const vp = (const uint8_t*)a.at.v + (int64_t)kvh * a.at.head_stride;

        // The next 64 blocks, one per lane: this wave's group of each, and which of them count as a whole.
        Groups8 groups = {a.at.table + (size_t)un.b * a.at.max_pages, 0, 0, 0};
        uint64_t whole = 0;
        auto key_of = [&](int i, int g) { return w.key0 + i * BK + 16 * g; };
        auto mask_of = [&](int i, int g) {                   // positions that count of group g of block i
            const int key = key_of(i, g);
            const int page = groups.table[fastdiv(min(key, a.at.max_pages * a.at.page_size - 1), pl.by_page)];
            return group_of(a.at, pl, page, key, w.key1).mask;
        };
        auto look = [&](int i) {
            groups.find(a, pl, dv, kvh, key_of(i + lane, grp), w.key1);
            uint32_t m = 0xffff;
#pragma unroll
            for (int g = 0; g < 4; g++) m &= mask_of(i + lane, g);
            asm volatile("" : "+v"(groups.lo), "+v"(groups.hi), "+v"(groups.info));
            whole = __builtin_amdgcn_ballot_w64(m == 0xffff);
        };
        // Stage i: codes and powers of block i's K and of block i - 1's V.  (Block n stands in where there is
        // none: page 0, and nothing of it counts.)
        typedef uint32_t words_t __attribute__((ext_vector_type(CB / 4)));
        words_t kcodes, vcodes;
        uint32_t kinfo = 0, vinfo = 0, wholes = 0;           // wholes: a bit for each of the last blocks
        int64_t v_at = 0;
        auto load = [&](int i) {
            if (i % 64 == 0) look(i);
            const int64_t at = groups.at(i);
            if (i == 0) v_at = at;
            kcodes = *(const CF_GLOBAL words_t*)(uniform_at(kp + at) + off);
            vcodes = *(const CF_GLOBAL words_t*)(uniform_at(vp + v_at) + off);
            vinfo = kinfo;
            kinfo = groups.what(i);
            v_at = at;
            wholes = wholes << 1 | (uint32_t)((whole >> (i & 63)) & 1);
        };
        auto put = [&](int at, words_t x, float power) {
            *(eight_t*)(ring + at) = C::of(x[0], power, x[1], power);
            if constexpr (CB == 16) *(eight_t*)(ring + (at ^ 8)) = C::of(x[2], power, x[3], power);
        };
        // V where nothing counts: 0, as p = 0 times whatever it holds need not be.
        auto write = [&](int i) {
            int odd = i & 1;
            asm volatile("" : "+s"(odd));
            const int stage = odd * STAGE;
            if ((vinfo & 0xffff) != 0xffff && !((vinfo >> row) & 1)) vcodes = words_t{};
            put(stage + to_k, kcodes, k_power(kinfo));
            put(stage + to_v, vcodes, v_power(vinfo));
        };

        {
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_offset(qlds)) + (uint32_t)(wrow * D * (int)sizeof(T));
#pragma unroll
            for (int u = 0; u < 16 * NJ / QR; u++) {
                const int r = QR * u + lane / QC;
                const RowAt at = row_at(pl, G, kvh, w.R0 + min(wrow + r, w.n_rows - 1));
                lds_dma16((const T*)a.at.q + (int64_t)(un.s.row0 + at.tok) * a.at.q_stride + at.h * D + QE * ((lane % QC) ^ (r & 7)),
                          __builtin_amdgcn_readfirstlane(to + u * 1024u));
            }
        }
        load(0);
        wait_vm<0>();
        // B operand Q^T: lane (lr, lq) takes dims 32 f + 8 lq .. + 7 of row lr.
        eight_t qf[NJ][NF][QP];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const T* const q = (const T*)qlds + (wrow + 16 * j + lr) * D;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                if constexpr (QP == 1) {
                    qf[j][f][0] = *(const eight_t*)(q + 8 * ((4 * f + lq) ^ (lr & 7)));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const T* const x = q + 4 * ((8 * f + 2 * lq + e / 4) ^ (lr & 7)) + e % 4;
                        split_into<QP, B>(qf[j][f], e, x[0], x[1]);
                    }
                }
            }
        }
        write(0);
        load(1);                                              // n >= 1: stages 0 and 1 exist
        wait_lds_reads();

        f4_t sc[NJ][4];
        eight_t pf[NJ][2][PP];

        // Fragment x of a turn: x < 2 UT is V^T (32-key step x / UT, dims 16 (x % UT)), the rest K
        // (key tile, then chunk).  They are read kAhead fragments before their products, in
        // exactly this order (2048 rows over 8192: 329 us, 8 ahead 333).
        constexpr int kAhead = 6, kV = 2 * UT, kAll = kV + 4 * NF;
        auto products = [&](int i, auto first_c, auto last_c) {   // fragments first .. last - 1
            constexpr int first = decltype(first_c)::value, last = decltype(last_c)::value;
            if (!active) return;
            int odd = i & 1;
            asm volatile("" : "+s"(odd));
            const _Float16* const st = ring + odd * STAGE;
            eight_t frag[kAhead];
            auto read = [&](auto x_c) {
                constexpr int x = decltype(x_c)::value;
                if constexpr (x < kV) {
                    const _Float16* const v = st + TILE + v_rd[x % UT] + 32 * (x / UT) * D;
                    frag[x % kAhead] = __builtin_bit_cast(eight_t, cat8(ds_read_tr4(v), ds_read_tr4(v + 16 * D)));
                } else if constexpr (x < kAll) {
                    frag[x % kAhead] = *(const eight_t*)(st + 16 * ((x - kV) % 4) * D + k_rd[(x - kV) / 4]);
                }
            };
            auto use = [&](auto x_c) {
                constexpr int x = decltype(x_c)::value;
                const eight_t f = frag[x % kAhead];
                // O^T += V^T P^T: in 32-key step s2, k-slot e of lane group lq is key
                // 32 s2 + 16 (e / 4) + 4 lq + e % 4, the lane's own scores.  p in its parts, small ones first.
                if constexpr (x < kV) {
#pragma unroll
                    for (int q = PP - 1; q >= 0; q--)
#pragma unroll
                        for (int j = 0; j < NJ; j++) acc[j][x % UT] = C::mfma(f, pf[j][x / UT][q], acc[j][x % UT]);
                } else {
                    // S^T: sc[j][t][e] = score(key 16 t + 4 lq + e of block i, row j).
                    constexpr int t = (x - kV) % 4, c0 = (x - kV) / 4;
#pragma unroll
                    for (int q = QP - 1; q >= 0; q--)
#pragma unroll
                        for (int j = 0; j < NJ; j++)
                            sc[j][t] = C::mfma(f, qf[j][c0][q], c0 == 0 && q == QP - 1 ? f4_t{0.f, 0.f, 0.f, 0.f} : sc[j][t]);
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
        const std::integral_constant<int, kV> to_v_end;
        const std::integral_constant<int, kAll> to_k_end;
        auto softmax = [&](int i, bool full) {
            if (!active) return;
            const int k0 = w.key0 + i * BK;
            const bool edge = !full || k0 + BK > seen_all;
            uint64_t mk = ~0ull;                              // positions that count
            if (!full) {
                mk = 0;
                for (int g = 0; g < 4; g++) mk |= (uint64_t)mask_of(i, g) << (16 * g);
            }
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
                    l_run[j].scale(alpha);
#pragma unroll
                    for (int u = 0; u < UT; u++) acc[j][u] *= alpha;
                }
                const float m_use = m_run[j] == -INFINITY ? 0.0f : m_run[j];
                float l_blk = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][t][e], c, -m_use));
                        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][t][e + 1], c, -m_use));
                        l_blk += p0 + p1;
                        split_into<PP, B>(pf[j][t >> 1], (t & 1) * 4 + e, p0, p1);
                    }
                l_run[j].add(l_blk);
            }
        };
        // Stage i into the ring, the codes of the next one on their way.
        auto refill = [&](int i) {
            if (i <= n) write(i);
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 <= n) load(i + 1);
            else wholes <<= 1;
            __builtin_amdgcn_sched_barrier(0);
        };
        // Everybody meets at every barrier, 2 n + 2 of them; each waits for its LDS accesses before.
        ring_barrier();
        auto half = [&](int i, int stage) {
            ring_barrier();
            refill(stage);
            softmax(i, (wholes >> (stage + 1 - i)) & 1);
            wait_lds_reads();
            ring_barrier();
        };
        if (wave < 4) {
            products(0, to_v_end, to_k_end);
            half(0, 1);
#pragma clang loop unroll(disable)
            for (int i = 1; i < n; i++) {
                products(i, from_v, to_k_end);
                half(i, i + 1);
            }
            products(n, from_v, to_v_end);
            ring_barrier();
        } else {
            refill(1);
            wait_lds_reads();
            ring_barrier();
            products(0, to_v_end, to_k_end);
            half(0, 2);
#pragma clang loop unroll(disable)
            for (int i = 1; i < n; i++) {
                products(i, from_v, to_k_end);
                half(i, i + 2);
            }
            products(n, from_v, to_v_end);
        }
    }
    uint32_t again_all = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int row = wrow + 16 * j + lr;
        const float l = add_xor32(add_xor16(l_run[j].sum()));
        const uint32_t again = rows_of_16(row < w.n_rows && spoilt(acc[j], l));
        if (row < w.n_rows) {
            const RowOut out = row_out<T, D, W::TM>(a.at, pl, un, kvh, w, row, m_run[j], l, lq == 0);
#pragma unroll
            for (int u = 0; u < UT; u++) put4<T>(out, 16 * u + 4 * lq, acc[j][u]);
        }
        again_all |= again << (16 * j);
    }
    ring_barrier();                                           // the ring's reads, before the next unit
    return again_all;
}

// Blocks of tiles of up to 16 rows that cost a wide tile's one (31 decode rows beside 4 chunks of 230 to 517
// rows: 106 us, with 2 111; 56 beside 8 of 300 rows 126 and 119).
constexpr int kNarrowCost8 = 4;
template <typename T, int D, int NJ>
__global__ __launch_bounds__(512, 2)
void paged_wide8(cf_paged_q8_args_t a, PagedPlan pl, Q8Divs dv) {
    using W = Wide8<T, D, NJ>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W::LDS];
    __shared__ int kept[4 * 64];
    const Geometry<W::TM, 64, kNarrowCost8, true, true> geo(a.at, pl, kept);
    if (geo.lists_cut_tiles()) return;
    for (int unit = (int)blockIdx.x;; unit += pl.step) {
        const int id = fastdiv(unit, pl.by_kv), kvh = unit - id * a.at.H_kv;
        Unit un;
        if (!geo.find(id, un)) break;
        Work w = unit_work<W::TM, 64>(a.at, pl, un);
        const bool narrow = w.n_rows <= 16;
        const uint32_t again = narrow ? narrow_unit8<T, D, W::TM, 8>(a, pl, dv, lds, un, kvh, w)
                                      : wide8_unit<T, D, NJ>(a, pl, dv, lds, un, kvh, w);
        if (!again) continue;
        if (!geo.find(id, un)) break;         // found anew: nothing is kept for this
        w = unit_work<W::TM, 64>(a.at, pl, un);
        if (narrow) mend_narrow8<T, D, W::TM, 8>(a, pl, dv, un, kvh, w);
        else mend_rows8<T, D, W::TM>(a, pl, dv, un, kvh, w, 16 * NJ * __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), again);
    }
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
            const int mid = lo + ((hi - lo) >> 1);
            if (a.at.q_start[mid] <= t) lo = mid; else hi = mid;
        }
        const SeqRows s = seq_rows(a.at, lo);
        if (t >= s.row0 && t < s.row0 + s.n) plain_row_q8<T, kAnyDims>(a, dv, s, lo, t - s.row0, h, a.at.d);
    }
}

// The plan of a call on the matrix cores: the kernel and how its work is cut.
enum Form8 { kHeads8, kSplit8, kWide1x8, kWide2x8 };   // kWide2x8: tiles of 256 rows, fp16
struct Plan8 {
    PagedPlan pl;
    Form8 form;
    int  wgs, merge_wgs;
    size_t bytes;         // workspace
};

// paged_split8 for sequences of up to 1024 positions, which it finishes in one range, as long as its units,
// a workgroup each, go in one round (us with paged_split8 and paged_heads8: 1 row over 512 7.3 and 10.5, 16
// over 512 8.8 and 12.9, 32 over 1024 16.7 and 20.2).  Longer ones: 1 over 2048 14.5 and 11.1, 16 over 2048 17.3
// and 20.1, 16 over 4096 40.9 and 32.2; where one of 16 is that long, only what it takes alone counts.
constexpr int64_t kSplitLen8 = 1024;
// Tiles of 256 rows read a block's K and V once for twice the rows, but are twice as long a piece of work.
// They pay where they fill three quarters of the chip by themselves (4 x 512 rows over 1024: 57 us, with 128
// rows 63; 2 x 2048 over 4096 272 and 329; 1024 over 1024, half the chip, 53 and 35.5), and where long
// ranges can be cut evenly (512 over 4608: 67 and 73; 4 x 230 over 2430 70.5 and 72.4; 700 over 1400, not cut,
// 66 and 43.5).
constexpr int64_t kLongLen8 = 2048;

bool fast_ok8(const cf_paged_q8_args_t& q) {
    const cf_paged_attn_args_t& a = q.at;
    const uint64_t ptrs = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)(uintptr_t)a.o;
    const uint64_t steps = (uint64_t)a.page_stride | (uint64_t)a.row_stride | (uint64_t)a.head_stride;
    const uint64_t es = a.elem == CF_ELEM_F16 ? 2 : 4;
    // Row numbers times the group and positions (with what is read ahead) stay in 31 bits, offsets
    // inside a group of rows in 32.
    return (a.d == 64 || a.d == 128) && q.block % 16 == 0 && ptrs % 16 == 0 && steps % 16 == 0 && a.q_stride * es % 16 == 0 &&
           a.scale > 0.0f && a.B <= kMostSeqs && (int64_t)a.T * (a.H_q / a.H_kv) <= (1 << 30) &&
           (int64_t)a.max_pages * a.page_size <= (1 << 30) && (uint64_t)a.row_stride * 16 < (1ull << 32);
}

// max_new and max_len only choose: the kernels' loops run until no unit is left, whatever the
// grid, and a sequence that is longer is computed all the same.
Plan8 make_plan8(const cf_paged_attn_args_t& a) {
    Plan8 p;
    const int64_t G = a.H_q / a.H_kv, cus = cu_count();
    const int64_t rows = (int64_t)a.max_new * G;              // of a sequence, at most
    const int64_t seqs = a.B < a.T ? a.B : a.T;
    auto tiles_of = [&](int64_t TM) {                         // tiles of the call, at most
        const int64_t t = ((int64_t)a.T * G + seqs * (TM - 1)) / TM;
        return rows <= TM && t > seqs ? seqs : t;
    };
    const bool f16 = a.elem == CF_ELEM_F16;
    if (rows <= 16) {
        const int64_t units = tiles_of(16) * a.H_kv;
        p.form = units <= cus && a.max_len <= kSplitLen8 ? kSplit8 : kHeads8;
    } else {
        const int64_t units = (int64_t)a.T * G / 256 * a.H_kv;
        const bool few_long = a.max_len > kLongLen8 && units >= cus / 8;
        p.form = f16 && (4 * units >= 3 * cus || few_long) ? kWide2x8 : kWide1x8;
    }
    const bool wide = p.form >= kWide1x8;
    const int64_t TM = !wide ? 16 : p.form == kWide2x8 ? 256 : 128;
    const int64_t BK = p.form == kHeads8 ? Narrow8<64>::BK : 64;
    const int64_t tiles = tiles_of(TM);
    // Units of a round: four waves of paged_heads8 a CU (d = 64: eight), though twice as many fit, as ranges
    // are longer then and records fewer (16 rows over 4096: 32.3 us, with twice as many 33.9; 1 over 16384 17.2
    // and 22.6).
    const int64_t per_cu = wide ? 1 : a.d == 128 ? 4 : 8;
    const int64_t fill = cus * per_cu > a.H_kv ? cus * per_cu / a.H_kv : 1;
    p.pl.fill = (int32_t)fill;
    // What is not worth cutting: a merge and the records cost some 5 us, and fp16 wide tiles take 2 to 2.7 us
    // a block (3 x 500 rows of 16 heads of 64 over 1200: 33.6 us, from 8 blocks on into ranges of 4 41.9; FP32
    // chunks of 129 to 411 rows over 300 to 1129 the other way round, 37 and 27).
    p.pl.min_blocks = (int32_t)(wide ? f16 ? 12 : 4 : 64 / BK);
    p.pl.one_blocks = (int32_t)((wide ? f16 ? 1536 : 512 : 128) / BK);
    p.pl.max_records = (int32_t)(4 * fill + 8);
    const bool cut = !a.uncut && p.form != kSplit8 && (a.max_len + BK - 1) / BK > (wide ? kFewOne / BK : p.pl.one_blocks);
    if (!cut) p.pl.one_blocks = INT32_MAX;                    // nor is what is longer than max_len
    p.bytes = cut ? header_bytes(p.pl.max_records) + (size_t)p.pl.max_records * a.H_kv * (TM * (a.d + 2)) * sizeof(float) : 0;
    int64_t units = (p.form == kHeads8 && cut && tiles <= fill ? 2 * fill : tiles + (cut ? 2 * fill : 0)) * a.H_kv;
    if (units > (1 << 22)) units = 1 << 22;
    p.wgs = (int)(p.form == kHeads8 ? (units + 3) / 4 : units);
    p.pl.step = p.form == kHeads8 ? 4 * p.wgs : p.wgs;
    p.pl.unit_wgs = p.wgs;
    if (cut) p.wgs++;                                         // lists the cut tiles
    const int64_t most_rows = rows < TM ? rows : TM;
    const int64_t merge_rows = p.form == kHeads8 ? 1 : 1024 / a.d;   // of a workgroup
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
int launch_tiles8(const cf_paged_q8_args_t& a, const Plan8& p, const Q8Divs& dv, hipStream_t st) {
    const dim3 grid((unsigned)p.wgs), mgrid((unsigned)p.merge_wgs);
    auto go = [&](auto tiles, int threads, auto merge) {
        hipLaunchKernelGGL(tiles, grid, dim3(threads), 0, st, a, p.pl, dv);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.merge_wgs == 0) return (int)e;
        hipLaunchKernelGGL(merge, mgrid, dim3(256), 0, st, a.at, p.pl);
        return (int)hipGetLastError();
    };
    if (p.form == kSplit8) {                                  // nothing is cut
        hipLaunchKernelGGL((paged_split8<T, D>), grid, dim3(64 * kSplitWaves), 0, st, a, p.pl, dv);
        return (int)hipGetLastError();
    }
    if (p.form == kHeads8) return go(paged_heads8<T, D>, 256, paged_merge<T, D, 16, 1>);
    if constexpr (sizeof(T) == 2)
        if (p.form == kWide2x8) return go(paged_wide8<T, D, 2>, 512, paged_merge<T, D, 256, 1024 / D>);
    return go(paged_wide8<T, D, 1>, 512, paged_merge<T, D, 128, 1024 / D>);
}

}  // namespace

extern "C" size_t cf_paged_attn_q8_bytes(const cf_paged_q8_args_t* a) { return fast_ok8(*a) ? make_plan8(a->at).bytes : 0; }

extern "C" int cf_launch_paged_attn_q8(const cf_paged_q8_args_t* a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    const cf_paged_attn_args_t& t = a->at;
    if (t.B <= 0 || t.T <= 0 || t.d <= 0 || t.d > 64 * kAnyDims || t.H_kv <= 0 || t.H_q % t.H_kv != 0 || a->block <= 0 ||
        t.page_size % a->block != 0)
        return (int)hipErrorInvalidValue;
    const Q8Divs dv = {fastdiv_make(t.page_size), fastdiv_make(a->block)};
    if (fast_ok8(*a)) {
        Plan8 p = make_plan8(t);
        if (p.bytes > 0 && !t.workspace) return (int)hipErrorInvalidValue;
        if (p.bytes > 0) {
            p.pl.cut_count = (int*)t.workspace;
            p.pl.cut_tiles = (CutTile*)((char*)t.workspace + 256);
            p.pl.records = (float*)((char*)t.workspace + header_bytes(p.pl.max_records));
        }
        if (t.elem == CF_ELEM_F16)
            return t.d == 64 ? launch_tiles8<_Float16, 64>(*a, p, dv, st) : launch_tiles8<_Float16, 128>(*a, p, dv, st);
        return t.d == 64 ? launch_tiles8<float, 64>(*a, p, dv, st) : launch_tiles8<float, 128>(*a, p, dv, st);
    }
    int64_t wgs = ((int64_t)t.T * t.H_q + 3) / 4;
    if (wgs > (1 << 22)) wgs = 1 << 22;        // a grid has less than 2^32 threads
    if (t.elem == CF_ELEM_F16) hipLaunchKernelGGL(paged_any_q8<_Float16>, dim3((unsigned)wgs), dim3(256), 0, st, *a, dv);
    else hipLaunchKernelGGL(paged_any_q8<float>, dim3((unsigned)wgs), dim3(256), 0, st, *a, dv);
    return (int)hipGetLastError();
}
