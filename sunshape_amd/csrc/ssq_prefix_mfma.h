// Matrix-core attention over VQ-coded pages for many query rows at once (ssq_decode_prefix): parameters, and
// the kernel template that ssq_prefix_mfma_*.hip instantiates.
//
// What it computes.  For a set of query rows of one KV head and a range of tokens, (o, m, l) = (sum_t e^{s_t - m} v_t,
// max_t s_t, sum_t e^{s_t - m}) in fp32, s_t = q . k_t with k_t the codewords that the token's codes name.
//
// Everything is held transposed: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16, a lane being one query row
// (its column) throughout, so the softmax's statistics and the rescale of O never cross lanes but for one exchange
// between a column's two halves, and S^T's accumulator is the P^T operand as it stands:
//   accumulator register i of half h holds matrix row 8 (i / 4) + 4 h + i % 4;  matrix row
//   m = 16 c + 8 a + 4 h + r is given the token 16 c + 8 h + 4 a + r of the 32-token tile, so register i holds
//   token 16 (i / 8) + 8 h + i % 8: the 8 consecutive tokens of one 16-byte piece of a dim-major value page,
//   which is the V^T operand, loaded straight into registers.
// K^T's operand is gathered codeword by codeword from the codebook in LDS: no key tile is ever written.  A
// codeword is stored as two 16-bit parts, c = hi + lo (the rounding of c, and of what that left: 2^-17 of c at most
// is dropped, 2^-23 with f16 parts), side by side, and the K slots of one MFMA take hi and lo of the same dims
// against the same query dims twice.  So one gather is one operand without a move, and the logits keep fp32's
// quality at twice the matrix-core work of 16-bit keys (their third part of all the work).
// Queries of 16 bits enter exactly (QT bf16 / f16); fp32 ones (rotated codecs) in two bf16 parts.
// Probabilities are rounded to the values' 16 bits for P.V, as in the other decode kernels; sums stay fp32.
//
// A wave holds 32 NR rows (NR 2: 64 rows per gathered operand, which the LDS needs to keep up) and takes every
// fourth tile of its item's range; the four waves' (o, m, l) join in LDS.  A workgroup (one per CU: the codebook
// fills the LDS, 128 KiB at head_dim 128) stages its KV head's codebook once and takes items in turn: a group
// of rows over a slice of the prefix, or a sequence's own rows over a piece of its own tokens.  The work of a
// tile's softmax (VALU) runs beside the next tile's scores (matrix cores).
#pragma once

#include "ssq_common.h"

struct SsqPrefixParams {
    ssq_decode_args a;  // own tokens' tables, lengths and mask; everything shared
    const int32_t* ptab;
    const int32_t* plen;
    int pcap;
    int G, rows;       // query rows of a KV head: (b, qi, g), g fastest
    int n_wg;          // workgroups per KV head
    int pre_nr, n_rg, n1;    // prefix items: n_rg groups of 32 pre_nr rows x n1 slices (n1 0: none)
    int own_nr, own_rg, n2;  // own items: sequences x own_rg groups of 32 own_nr rows x n2 pieces (n2 0: none)
    int own_tiles;     // tiles of a piece
    int psh;           // log2(page_size / 16)
    float* pre;        // o [n1][all rows][Dv], then m, l [n1][all rows]
    float* own;        // likewise for n2
};

// QT: how queries (and the codebook's parts) enter the matrix cores
enum { kQtBf16 = 0, kQtF16 = 1, kQtSplit = 2 };

#define SSQ_PREFIX_UNIT(name) int name(const SsqPrefixParams& p, hipStream_t st)
SSQ_PREFIX_UNIT(ssq_prefix_bf16);        // bf16 queries, bf16 values
SSQ_PREFIX_UNIT(ssq_prefix_f16);         // f16, f16
SSQ_PREFIX_UNIT(ssq_prefix_split_bf16);  // fp32 or other queries, bf16 values
SSQ_PREFIX_UNIT(ssq_prefix_split_f16);

namespace {

typedef float pv16f __attribute__((ext_vector_type(16)));
typedef __bf16 pv8bf __attribute__((ext_vector_type(8)));
typedef _Float16 pv8h __attribute__((ext_vector_type(8)));
typedef __bf16 pv2bf __attribute__((ext_vector_type(2)));
typedef _Float16 pv2h __attribute__((ext_vector_type(2)));
typedef float pv2f __attribute__((ext_vector_type(2)));
typedef unsigned int pv4u __attribute__((ext_vector_type(4)));

constexpr int kPfThreads = 256;
constexpr int kPfWaves = 4;
constexpr int kPfTile = 32;  // tokens
constexpr float kLog2e = 1.4426950408889634f;

// two fp32 to 16 bits (RNE), packed
template <bool F16>
__device__ __forceinline__ uint32_t pf_pack(float a, float b) {
    const pv2f f = {a, b};
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, pv2h));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, pv2bf));
}
template <bool F16>
__device__ __forceinline__ float pf_lo(uint32_t w) { return F16 ? ssq_f16_to_f32(w & 0xFFFFu) : __uint_as_float(w << 16); }
template <bool F16>
__device__ __forceinline__ float pf_hi(uint32_t w) { return F16 ? ssq_f16_to_f32(w >> 16) : __uint_as_float(w & 0xFFFF0000u); }

template <bool F16>
__device__ __forceinline__ pv16f pf_mfma(const uint4& a, const uint4& b, pv16f c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pv8h, a), __builtin_bit_cast(pv8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pv8bf, a), __builtin_bit_cast(pv8bf, b), c, 0, 0, 0);
}

// LDS: codebook parts [nb][256][2 bd] | scratch: staged query rows, then the waves' join | m, l [4][64]
template <int D>
struct PfLds {
    static constexpr int kBook = D * 256 * 4;
    static constexpr int kQRow = D + 8;                            // staged query row, 16-bit elements
    static constexpr int kJoinRow = 36;                            // floats: 32 dims, padded
    static constexpr int kQ = 64 * kQRow * 2;                      // 64 rows, or 32 rows in two parts
    static constexpr int kJoin = kPfWaves * 32 * kJoinRow * 4;
    static constexpr int kScratch = kQ > kJoin ? kQ : kJoin;
    static constexpr int kTotal = kBook + kScratch + 2 * kPfWaves * 64 * 4;
};

template <int D, int BD, int QT, int VT, int NR>
struct PfRun {
    static constexpr bool kF16 = QT == kQtF16;    // parts of the codebook and queries
    static constexpr bool kVF16 = VT == SSQ_F16;  // probabilities and values
    static constexpr int NB = D / BD, NW = NB / 4;
    static constexpr int NST = D / 8;                   // MFMAs of a 32 x 32 score tile
    static constexpr int NQ = D / 16;                    // query operands: 16 dims each
    static constexpr int DT = D / 32;
    static constexpr int QP = QT == kQtSplit ? 2 : 1;
    using L = PfLds<D>;

    struct Codes { uint32_t w[NW]; };
    struct Vals { uint4 v[2][DT]; };

    const SsqPrefixParams& p;
    const unsigned char* book;
    int lane, half, kv;
    uint4 q[QP][NR][NQ];
    // tokens
    const int32_t* table;
    int len, last_chunk, tile0, n_tiles, wave;  // this wave's tiles: tile0 + wave + 4 i, i < n_tiles
    int pg, pgn, batch;                         // table entries of 32 tiles, and of the 32 after them
    const uint8_t* cbase;
    const uint16_t* vbase;
    uint32_t voff, vstep;                       // lane and 32-dim offsets in a page, elements

    __device__ __forceinline__ int entries(int i0) const {  // lane: chunk (lane & 1) of tile i0 + lane / 2
        const int chunk = min(2 * (tile0 + wave + kPfWaves * (i0 + (lane >> 1))) + (lane & 1), last_chunk);
        return table[chunk >> p.psh];
    }
    __device__ __forceinline__ int page(int i, int c) const {  // uniform
        return __builtin_amdgcn_readlane((i >> 5) == batch ? pg : pgn, 2 * (i & 31) + c);
    }
    __device__ __forceinline__ int chunk_of(int i, int c) const {
        return min(2 * (tile0 + wave + kPfWaves * i) + c, last_chunk);
    }
    __device__ __forceinline__ void load_codes(int i, Codes& r) const {
        const int msk = (1 << p.psh) - 1;
        const int m = lane & 31, c = m >> 4;
        const int tok = 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);  // within its 16-token chunk
        const int pgc = c ? page(i, 1) : page(i, 0);
        const int at = (c ? (chunk_of(i, 1) & msk) : (chunk_of(i, 0) & msk)) * 16 + tok;
        const uint8_t* row = cbase + (int64_t)pgc * p.a.c_sb + (int64_t)at * p.a.c_st;
        if constexpr (NW >= 4) {
#pragma unroll
            for (int k = 0; k < NW / 4; ++k) {
                const uint4 x = reinterpret_cast<const uint4*>(row)[k];
                r.w[4 * k] = x.x; r.w[4 * k + 1] = x.y; r.w[4 * k + 2] = x.z; r.w[4 * k + 3] = x.w;
            }
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(row);
            r.w[0] = x.x; r.w[1] = x.y;
        }
    }
    __device__ __forceinline__ void load_vals(int i, Vals& r) const {
        const int msk = (1 << p.psh) - 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint16_t* src = vbase + (int64_t)page(i, c) * p.a.v_sb + (chunk_of(i, c) & msk) * 16;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) r.v[c][dt] = *reinterpret_cast<const uint4*>(src + voff + dt * vstep);
        }
    }
    // the K^T operand of step st: dims 16 (st / 2) + 8 half .., the hi parts (st even) or the lo parts
    __device__ __forceinline__ uint4 operand(const Codes& c, int st) const {
        const int s2 = st >> 1;
        const unsigned char* part = book + (st & 1) * (L::kBook / 2);
        if constexpr (BD == 8) {  // block 2 s2 + half
            const uint32_t code = (c.w[s2 >> 1] >> (16 * (s2 & 1) + 8 * half)) & 0xFFu;
            return *reinterpret_cast<const uint4*>(part + (2 * s2 + half) * 4096 + code * 16);
        } else if constexpr (BD == 4) {  // blocks 4 s2 + 2 half, + 1
            const uint32_t w = c.w[s2] >> (16 * half);
            const uint2 a = *reinterpret_cast<const uint2*>(part + (4 * s2 + 2 * half) * 2048 + (w & 0xFFu) * 8);
            const uint2 b = *reinterpret_cast<const uint2*>(part + (4 * s2 + 2 * half + 1) * 2048 + ((w >> 8) & 0xFFu) * 8);
            return make_uint4(a.x, a.y, b.x, b.y);
        } else {  // blocks 8 s2 + 4 half ..
            const uint32_t w = half ? c.w[2 * s2 + 1] : c.w[2 * s2];
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[k] = *reinterpret_cast<const uint32_t*>(part + (8 * s2 + 4 * half + k) * 1024 + ((w >> (8 * k)) & 0xFFu) * 4);
            return make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    __device__ __forceinline__ void scores(const Codes& c, pv16f (&s)[NR]) const {
        constexpr int kAhead = 4;
        uint4 k[kAhead];
#pragma unroll
        for (int st = 0; st < kAhead; ++st) k[st] = operand(c, st);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r] = pv16f{};
#pragma unroll
        for (int st = 0; st < NST; ++st) {
            const uint4 kk = k[st % kAhead];
            if (st + kAhead < NST) k[st % kAhead] = operand(c, st + kAhead);
            const int qi = st >> 1;
#pragma unroll
            for (int h = 0; h < QP; ++h)
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r] = pf_mfma<kF16>(kk, q[h][r][qi], s[r]);
        }
    }
};

// the lane 32 apart
__device__ __forceinline__ float pf_other(float v) { return __shfl_xor(v, 32); }

// One item: rows [R0, R0 + nr) of the KV head over tiles [t0, t1) of a sequence of `len` tokens; partials go to split
// `split` of ws.  The whole workgroup calls it.
template <int D, int BD, int QT, int VT, int NR>
__device__ __forceinline__ void pf_item(const SsqPrefixParams& p, unsigned char* lds, int kv, int R0, int nr,
                                        const int32_t* table, int len, int t0, int t1, const float* mask, float* ws,
                                        int n_split, int split) {
    using Run = PfRun<D, BD, QT, VT, NR>;
    using L = PfLds<D>;
    const ssq_decode_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n_rows = (int64_t)a.batch * a.num_q_heads * a.q_len;
    float* ws_o = ws + (int64_t)split * n_rows * D;
    float* ws_m = ws + (int64_t)n_split * n_rows * D + (int64_t)split * n_rows;
    float* ws_l = ws_m + (int64_t)n_split * n_rows;
    const int per_b = a.q_len * p.G;
    auto row_of = [&](int R, int& b, int& qi, int& h) {
        b = R / per_b;
        const int e = R - b * per_b;
        qi = e / p.G;
        h = kv * p.G + (e - qi * p.G);
    };
    auto rid_of = [&](int R) {
        int b, qi, h;
        row_of(R, b, qi, h);
        return ((int64_t)b * a.num_q_heads + h) * a.q_len + qi;
    };
    if (t0 >= t1) {  // nothing attended: the merge reads m alone
        for (int r = tid; r < nr; r += kPfThreads) ws_m[rid_of(R0 + r)] = -INFINITY;
        return;
    }
    unsigned char* scratch = lds + L::kBook;
    float* mL = reinterpret_cast<float*>(scratch + L::kScratch);  // [4][64]
    float* lL = mL + kPfWaves * 64;

    Run u{p, lds};
    u.lane = lane; u.half = half; u.kv = kv;
    u.table = table; u.len = len; u.last_chunk = (len - 1) >> 4;
    u.tile0 = t0; u.wave = wave;
    u.n_tiles = (t1 - t0 - wave + kPfWaves - 1) / kPfWaves;
    u.cbase = a.codes + (int64_t)kv * a.c_sh;
    u.vbase = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)kv * a.v_sh;
    u.voff = (uint32_t)col * (uint32_t)a.v_st + 8 * half;
    u.vstep = 32 * (uint32_t)a.v_st;
    u.batch = 0;
    u.pg = u.entries(0);
    u.pgn = u.entries(32);

    // ---- query rows: scaled in their dtype, permuted, as 16-bit parts [part][row][D] in LDS
    uint16_t* qL = reinterpret_cast<uint16_t*>(scratch);
    const int64_t* perm = a.perm + (int64_t)kv * a.perm_sh;
    constexpr int kRows = 32 * NR, kPer = kRows * D / kPfThreads, kBatch = kPer < 16 ? kPer : 16;
    const int j = tid % D;  // a thread's dim is the same for all its elements
    const int64_t pj = (int64_t)min((uint64_t)perm[j], (uint64_t)(D - 1));
#pragma unroll
    for (int e0 = 0; e0 < kPer; e0 += kBatch) {
        int64_t at[kBatch];
        float v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int r = (e0 + k) * (kPfThreads / D) + tid / D;
            int b, qi, h;
            row_of(R0 + min(r, nr - 1), b, qi, h);
            at[k] = (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + (int64_t)qi * a.q_sl + pj;
        }
        ssq_load_elems<kBatch>(a.q, a.q_dtype, at, v);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int r = (e0 + k) * (kPfThreads / D) + tid / D;
            float x = r < nr ? v[k] : 0.f;
            if (a.has_scale) x = ssq_round_to(x * a.scale, a.q_dtype);
            const uint32_t w = pf_pack<Run::kF16>(x, 0.f);
            qL[r * L::kQRow + j] = (uint16_t)w;
            if constexpr (Run::QP == 2) {
                const uint32_t w2 = pf_pack<false>(x - pf_lo<false>(w), 0.f);
                qL[(kRows + r) * L::kQRow + j] = (uint16_t)w2;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < Run::QP; ++h)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int st = 0; st < Run::NQ; ++st) {
                const uint16_t* row = qL + (h * kRows + 32 * r + col) * L::kQRow;
                u.q[h][r][st] = *reinterpret_cast<const uint4*>(row + 16 * st + 8 * half);
            }

    // this lane's mask rows
    const float* mrow[NR];
    if (mask) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            int b, qi, h;
            row_of(R0 + min(32 * r + col, nr - 1), b, qi, h);
            mrow[r] = mask + (int64_t)b * a.m_sb + (int64_t)h * a.m_sh + (int64_t)qi * a.m_sl;
        }
    }

    // ---- tiles
    float m_run[NR], l_run[NR];
    pv16f o[NR][Run::DT];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int dt = 0; dt < Run::DT; ++dt) o[r][dt] = pv16f{};
    }
    const int n = u.n_tiles;
    if (n > 0) {  // wave-uniform
        typename Run::Codes c0, c1;
        typename Run::Vals val;
        pv16f s[NR], s2[NR];
        u.load_codes(0, c0);
        u.load_vals(0, val);
        u.load_codes(min(1, n - 1), c1);
        u.scores(c0, s);
        for (int i = 0; i < n; ++i) {
            if ((i & 31) == 31) {  // the next tile starts the next 32 entries
                u.batch = (i >> 5) + 1;
                u.pg = u.pgn;
                u.pgn = u.entries(32 * (u.batch + 1));
            }
            u.load_codes(min(i + 2, n - 1), c0);
            const int tile = t0 + wave + kPfWaves * i;
            const int t_half = kPfTile * tile + 8 * half;  // register k: token t_half + 16 (k / 8) + k % 8
            const bool tail = kPfTile * (tile + 1) > len;  // uniform
            if (mask) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int t = min(t_half + 16 * (k >> 3) + (k & 7), len - 1);
                        s[r][k] += mrow[r][(int64_t)t * a.m_st];
                    }
            }
            if (tail) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (t_half + 16 * (k >> 3) + (k & 7) >= len) s[r][k] = -INFINITY;
#pragma unroll
                for (int c = 0; c < 2; ++c) {  // values behind the last token are unwritten
                    const int keep = len - (t_half + 16 * c);
#pragma unroll
                    for (int dt = 0; dt < Run::DT; ++dt) {
                        uint32_t w[4] = {val.v[c][dt].x, val.v[c][dt].y, val.v[c][dt].z, val.v[c][dt].w};
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k >= keep) w[k >> 1] &= (k & 1) ? 0x0000FFFFu : 0xFFFF0000u;
                        val.v[c][dt] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            // the running maximum moves only when a score passes it by kSoftmaxSlack
            float top[NR];
            bool over = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                top[r] = s[r][0];
#pragma unroll
                for (int k = 1; k < 16; ++k) top[r] = fmaxf(top[r], s[r][k]);
                over |= top[r] > m_run[r] + kSoftmaxSlack;
            }
            if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float mn = fmaxf(m_run[r], fmaxf(top[r], pf_other(top[r])));
                    const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[r] - mn) * kLog2e);
                    m_run[r] = mn;
                    l_run[r] *= f;
#pragma unroll
                    for (int dt = 0; dt < Run::DT; ++dt)
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[r][dt][k] *= f;
                }
            }
            // a masked score may be the type's lowest value, which times log2(e) is -inf: m is taken off first
            if (mask) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int k = 0; k < 16; ++k) s[r][k] -= m_run[r] == -INFINITY ? 0.f : m_run[r];
            }
            // the next tile's scores beside this tile's probabilities
            u.scores(c1, s2);
            uint4 pr[NR][2];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                // -inf while every score seen is (then the probabilities are exp(-inf) = 0)
                const float mb = mask || m_run[r] == -INFINITY ? 0.f : m_run[r] * kLog2e;
                float e[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    e[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][k], kLog2e, -mb));
                    l_run[r] += e[k];
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    pr[r][c] = make_uint4(pf_pack<Run::kVF16>(e[8 * c], e[8 * c + 1]), pf_pack<Run::kVF16>(e[8 * c + 2], e[8 * c + 3]),
                                          pf_pack<Run::kVF16>(e[8 * c + 4], e[8 * c + 5]), pf_pack<Run::kVF16>(e[8 * c + 6], e[8 * c + 7]));
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int dt = 0; dt < Run::DT; ++dt)
#pragma unroll
                    for (int r = 0; r < NR; ++r) o[r][dt] = pf_mfma<Run::kVF16>(val.v[c][dt], pr[r][c], o[r][dt]);
            u.load_vals(min(i + 1, n - 1), val);
#pragma unroll
            for (int r = 0; r < NR; ++r) s[r] = s2[r];
            const typename Run::Codes ct = c0;
            c1 = ct;
        }
    }
    // ---- the four waves' (m, l), then o, 32 rows x 32 dims at a time
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float l = l_run[r] + pf_other(l_run[r]);
        if (half == 0) {
            mL[wave * 64 + 32 * r + col] = m_run[r];
            lL[wave * 64 + 32 * r + col] = l;
        }
    }
    __syncthreads();  // also: every wave has read its query operands
    float* jL = reinterpret_cast<float*>(scratch);
    float f[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPfWaves; ++w) M = fmaxf(M, mL[w * 64 + 32 * r + col]);
        f[r] = m_run[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[r] - M) * kLog2e);
    }
    for (int r = tid; r < nr; r += kPfThreads) {
        float M = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kPfWaves; ++w) M = fmaxf(M, mL[w * 64 + r]);
#pragma unroll
        for (int w = 0; w < kPfWaves; ++w) {
            const float m = mL[w * 64 + r];
            if (m != -INFINITY) l += lL[w * 64 + r] * __builtin_amdgcn_exp2f((m - M) * kLog2e);
        }
        const int64_t rid = rid_of(R0 + r);
        ws_m[rid] = M;
        ws_l[rid] = l;
    }
    const int jr = tid >> 3, jd = (tid & 7) * 4;  // the row and dims this thread joins
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        if (32 * r >= nr) break;  // uniform
        const bool in = 32 * r + jr < nr;
        const int64_t rid = rid_of(R0 + min(32 * r + jr, nr - 1));
#pragma unroll
        for (int dt = 0; dt < Run::DT; ++dt) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // dims 8 k + 4 half ..
                float4 x = make_float4(o[r][dt][4 * k] * f[r], o[r][dt][4 * k + 1] * f[r], o[r][dt][4 * k + 2] * f[r], o[r][dt][4 * k + 3] * f[r]);
                if (f[r] == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
                *reinterpret_cast<float4*>(jL + (wave * 32 + col) * L::kJoinRow + 8 * k + 4 * half) = x;
            }
            __syncthreads();
            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kPfWaves; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(jL + (w * 32 + jr) * L::kJoinRow + jd);
                t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
            }
            if (in) *reinterpret_cast<float4*>(ws_o + rid * D + 32 * dt + jd) = t;
            __syncthreads();
        }
    }
}

template <int D, int BD, int QT, int VT>
__global__ __launch_bounds__(kPfThreads, 1) void k_prefix(const SsqPrefixParams p) {
    extern __shared__ __align__(16) unsigned char pf_lds[];
    const ssq_decode_args& a = p.a;
    const int tid = threadIdx.x;
    const int kv = blockIdx.x % a.num_kv_heads, w = blockIdx.x / a.num_kv_heads;
    // ---- the KV head's codebook as 16-bit parts
    {
        constexpr bool F16 = QT == kQtF16;
        const float* cent = a.cent + (int64_t)kv * a.cent_sh;
        const int nc = a.n_centroids, total = (D / BD) * nc;
        constexpr int kV = BD < 4 ? BD : 4;  // floats per load
        for (int e = tid; e < total * (BD / kV); e += kPfThreads) {
            const int cw = e / (BD / kV), part = e - cw * (BD / kV);
            const int blk = cw / nc, c = cw - blk * nc;
            float x[kV];
            const float* src = cent + (int64_t)cw * BD + part * kV;
            if constexpr (kV == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                x[0] = v.x; x[1] = v.y;
            }
            uint32_t hi[kV / 2], lo[kV / 2];
#pragma unroll
            for (int k = 0; k < kV / 2; ++k) {
                hi[k] = pf_pack<F16>(x[2 * k], x[2 * k + 1]);
                lo[k] = pf_pack<F16>(x[2 * k] - pf_lo<F16>(hi[k]), x[2 * k + 1] - pf_hi<F16>(hi[k]));
            }
            unsigned char* dst = pf_lds + (blk * 256 + c) * 2 * BD + part * 2 * kV;
            unsigned char* dlo = dst + PfLds<D>::kBook / 2;
            if constexpr (BD == 2) {
                *reinterpret_cast<uint32_t*>(dst) = hi[0];
                *reinterpret_cast<uint32_t*>(dlo) = lo[0];
            } else {
                *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(dlo) = make_uint2(lo[0], lo[1]);
            }
        }
    }
    __syncthreads();
    const int n_pre = p.n_rg * p.n1;
    const int n_items = n_pre + a.batch * p.own_rg * p.n2;
    for (int it = w; it < n_items; it += p.n_wg) {
        if (it < n_pre) {
            const int split = it / p.n_rg, rg = it - split * p.n_rg;  // the groups of one slice side by side
            const int len = max(0, min(p.plen[0], p.pcap));
            const int tiles = (len + kPfTile - 1) / kPfTile, per = (tiles + p.n1 - 1) / p.n1;
            const int R0 = rg * 32 * p.pre_nr, nr = min(32 * p.pre_nr, p.rows - R0);
            const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);
            if constexpr (QT != kQtSplit) {
                if (p.pre_nr == 2) {
                    pf_item<D, BD, QT, VT, 2>(p, pf_lds, kv, R0, nr, p.ptab, len, t0, t1, nullptr, p.pre, p.n1, split);
                    continue;
                }
            }
            pf_item<D, BD, QT, VT, 1>(p, pf_lds, kv, R0, nr, p.ptab, len, t0, t1, nullptr, p.pre, p.n1, split);
        } else {
            const int e = it - n_pre;
            const int split = e % p.n2, br = e / p.n2;
            const int b = br / p.own_rg, rg = br - b * p.own_rg;
            const int len = max(0, min(a.seq_lens[b], a.seq_len));
            const int tiles = (len + kPfTile - 1) / kPfTile;
            const int per_b = a.q_len * p.G;
            const int r0 = rg * 32 * p.own_nr, nr = min(32 * p.own_nr, per_b - r0);
            const int t0 = min(split * p.own_tiles, tiles), t1 = min(t0 + p.own_tiles, tiles);
            const int32_t* table = a.block_table + (int64_t)b * a.bt_sb;
            if constexpr (QT != kQtSplit) {
                if (p.own_nr == 2) {
                    pf_item<D, BD, QT, VT, 2>(p, pf_lds, kv, b * per_b + r0, nr, table, len, t0, t1, a.mask, p.own, p.n2, split);
                    continue;
                }
            }
            pf_item<D, BD, QT, VT, 1>(p, pf_lds, kv, b * per_b + r0, nr, table, len, t0, t1, a.mask, p.own, p.n2, split);
        }
    }
}

template <int D, int BD, int QT, int VT>
int launch_prefix(const SsqPrefixParams& p, hipStream_t st) {
    auto kern = k_prefix<D, BD, QT, VT>;
    int rc = ssq_allow_lds((const void*)kern, PfLds<D>::kTotal, "hipFuncSetAttribute(k_prefix)");
    if (rc) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.n_wg * p.a.num_kv_heads)), dim3(kPfThreads), PfLds<D>::kTotal, st, p);
    return ssq_check_hip(hipGetLastError(), "k_prefix launch");
}

template <int QT, int VT>
int launch_prefix_qv(const SsqPrefixParams& p, hipStream_t st) {
    if (p.a.head_dim == 64) {
        switch (p.a.block_dim) {
            case 2: return launch_prefix<64, 2, QT, VT>(p, st);
            case 4: return launch_prefix<64, 4, QT, VT>(p, st);
            default: return launch_prefix<64, 8, QT, VT>(p, st);
        }
    }
    switch (p.a.block_dim) {
        case 2: return launch_prefix<128, 2, QT, VT>(p, st);
        case 4: return launch_prefix<128, 4, QT, VT>(p, st);
        default: return launch_prefix<128, 8, QT, VT>(p, st);
    }
}

}  // namespace
