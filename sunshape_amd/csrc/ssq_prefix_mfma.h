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
// codeword is stored as two 16-bit parts, c = hi + lo (the rounding of c, and of what that left), and each 16 dims take
// one MFMA with the hi parts and one with the lo parts against the same query operand, half as much matrix-core work
// again.  Dropped is at most 2^-17 of a codeword with bf16 parts (one part would drop 2^-9); with f16 parts, which a
// power of two per KV head keeps off the subnormals, 2^-22 of it or 2^-38 of the head's largest one.
// Kept (passthrough) dims of a SunShape-Mixed codec, up to half of the head's, take a step per 16 more: their codewords are
// staged as zeros, and a token's kept values, two 8-byte pieces a lane and step, enter exactly, into sums of their own.
// Queries of 16 bits enter exactly (QT bf16 / f16); fp32 ones (rotated codecs) in two bf16 parts (2^-17 of a query dim
// is dropped; an infinite kept dim against a part of 0 gives NaN there).
// Probabilities are rounded to the values' 16 bits for P.V, as in the other decode kernels (two parts would take those
// products twice); sums stay fp32.
//
// A workgroup (one per CU: the codebook fills the LDS, 128 KiB at head_dim 128) stages its KV head's codebook once
// and takes items in turn.  A prefix item is a group of 32 NR rows (NR 2: 64 rows per gathered operand, which the
// LDS needs to keep up) over a slice of the prefix: each wave takes every fourth tile, and the four waves' (o, m, l)
// join in LDS.  An own item is one sequence's rows over a piece of its own tokens, by one wave: no barriers, four
// such latency chains side by side.  The work of a tile's softmax (VALU) runs beside the next tile's scores
// (matrix cores).
//
// Measured, one MI355X, whole calls with the merge: 128 sequences of 64 query heads (8 KV heads of 128 dims, byte codes of
// dim 4) on a prefix of 65,536 tokens with up to 1,024 own ones 415-424 us, 64 sequences of 32 on 32,768 73-76; attending
// every sequence's copy of the prefix by itself, 64 on 8,192: 122 against 55.  A tile of 32 tokens and 64 rows takes a wave
// 1.35 us, where the rate of a large library product (1.39 PFLOP/s) would take 1.16 for its 48 MFMAs, and the MFMAs
// alone, in this loop, 1.0: the matrix cores bound long prefixes, at 86 % of the rate that they reach.  Of a short one's
// 50 us, 3 to 4 are the codebook's staging, 3 the queries', 2.5 the first loads, 4 the join, 9 the own
// items, 8 the merge (a launch of its own).
//
// A row's maximum is its first tile's until the probabilities outgrow kPfOver; while a mask has hidden all its tokens
// there is none, and the first visible score sets it.  An infinite or NaN value counts wherever its tile is, also at
// probability 0 (0 times infinity is NaN), and a row of NaN scores is NaN, not one with nothing to attend.
#pragma once

#include "ssq_common.h"

#include <type_traits>

struct SsqPrefixParams {
    ssq_decode_args a;  // own tokens' tables, lengths and mask; everything shared
    const int32_t* ptab;
    const int32_t* plen;
    int pcap;
    int G, rows;       // query rows of a KV head: (b, qi, g), g fastest
    int n_wg;          // workgroups per KV head
    int pre_nr, n_rg, n1;    // prefix items: n_rg groups of 32 pre_nr rows x n1 slices (n1 0: none)
    int own_rg, n2;    // own items: sequences x own_rg groups of 32 rows x at most n2 pieces (n2 0: none)
    int own_min;       // the fewest tiles of a piece
    int psh;           // log2(page_size / 16)
    int q_vec;         // 16-bit query rows load in 16-byte pieces
    int kept;          // dims of the kept blocks, a multiple of 4, at most head_dim / 2
    float* pre;        // o [n1][all rows][Dv], then m, l [n1][all rows]
    float* own;        // likewise for n2
    int* own_per;      // tiles of a piece, chosen by the lengths (written for the merge)
};

// tiles of a prefix slice, and of a set of tokens
__host__ __device__ inline int ssq_prefix_tiles(int len) { return (len + 31) / 32; }
__host__ __device__ inline int ssq_prefix_slice(int len, int n1) { return (ssq_prefix_tiles(len) + n1 - 1) / n1; }

// QT: how queries (and the codebook's parts) enter the matrix cores
enum { kQtBf16 = 0, kQtF16 = 1, kQtSplit = 2 };

#define SSQ_PREFIX_UNIT(name) int name(const SsqPrefixParams& p, hipStream_t st)
SSQ_PREFIX_UNIT(ssq_prefix_bf16);        // bf16 queries, bf16 values
SSQ_PREFIX_UNIT(ssq_prefix_f16);         // f16, f16
SSQ_PREFIX_UNIT(ssq_prefix_split_bf16);  // fp32 or other queries, bf16 values
SSQ_PREFIX_UNIT(ssq_prefix_split_f16);
SSQ_PREFIX_UNIT(ssq_prefix_bf16_mixed);  // with kept blocks
SSQ_PREFIX_UNIT(ssq_prefix_f16_mixed);
SSQ_PREFIX_UNIT(ssq_prefix_split_bf16_mixed);
SSQ_PREFIX_UNIT(ssq_prefix_split_f16_mixed);

namespace {

typedef float pv16f __attribute__((ext_vector_type(16)));
typedef __bf16 pv8bf __attribute__((ext_vector_type(8)));
typedef _Float16 pv8h __attribute__((ext_vector_type(8)));
typedef __bf16 pv2bf __attribute__((ext_vector_type(2)));
typedef _Float16 pv2h __attribute__((ext_vector_type(2)));
typedef float pv2f __attribute__((ext_vector_type(2)));
typedef unsigned int pv4u __attribute__((ext_vector_type(4)));
typedef unsigned int pv2u __attribute__((ext_vector_type(2)));

constexpr int kPfThreads = 256;
constexpr int kPfWaves = 4;
constexpr int kPfTile = 32;  // tokens
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

// two fp32 values as packed parts
template <bool F16>
__device__ __forceinline__ void pf_split(float u, float v, uint32_t& hi, uint32_t& lo) {
    hi = pf_pack<F16>(u, v);
    lo = pf_pack<F16>(u - pf_lo<F16>(hi), v - pf_hi<F16>(hi));
}

template <bool F16>
__device__ __forceinline__ pv16f pf_mfma(const uint4& a, const uint4& b, pv16f c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pv8h, a), __builtin_bit_cast(pv8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pv8bf, a), __builtin_bit_cast(pv8bf, b), c, 0, 0, 0);
}

// LDS: codebook [nb]: the codewords' hi parts [256][bd], their lo parts | scratch: staged query rows, then the waves' join |
// m, l [4][64] | rows' offsets [2][64] | permutation [D] | kept dims' places in it [D / 2]
template <int D>
struct PfLds {
    static constexpr int kBook = D * 256 * 4;
    static constexpr int kQRow = D + 8;                            // staged query row, 16-bit elements
    static constexpr int kJoinRow = 36;                            // floats: 32 dims, padded
    static constexpr int kQ = 32 * (D + kQRow) * 2;                // 32 rows as they are, and permuted
    static constexpr int kJoin = kPfWaves * 32 * kJoinRow * 4;
    static constexpr int kScratch = kQ > kJoin ? kQ : kJoin;
    static constexpr int kPerm = kBook + kScratch + 2 * kPfWaves * 64 * 4 + 2 * 64 * 8;
    static constexpr int kKept = kPerm + 2 * D;
    static constexpr int kKeptMax = D / 2;                         // a multiple of 32
    static constexpr int kTotal = kKept + 2 * kKeptMax;
};

// HV: the codec keeps blocks
template <int D, int BD, int QT, int VT, int NR, bool HV>
struct PfRun {
    using L = PfLds<D>;
    static constexpr bool kF16 = QT == kQtF16;    // parts of the codebook and queries
    static constexpr bool kVF16 = VT == SSQ_F16;  // probabilities and values
    static constexpr int NB = D / BD, NW = NB / 4;
    static constexpr int NST = D / 8;                   // MFMAs of a 32 x 32 score tile
    static constexpr int NQ = D / 16;                    // query operands: 16 dims each
    static constexpr int DT = D / 32;
    static constexpr int QP = QT == kQtSplit ? 2 : 1;
    static constexpr int NK = HV ? L::kKeptMax / 16 : 0;  // steps of kept dims, at most
    static constexpr int KP = QT == kQtSplit && kVF16 ? 2 : 1;  // parts of a kept value: exact in its own type, or in two
    static constexpr bool kKept = HV;
    static constexpr bool kScaled = kF16 && !HV;  // scores come times the codebook's scale

    struct Codes { uint32_t w[NW]; };
    struct Vals { uint4 v[2][DT]; };
    template <int N>
    struct KeptOf {  // kept dims: queries, and the next tile's values
        uint4 q[QP][NR][N], v[N];
        int64_t o, on;  // as pc and pcn
        const uint16_t* base;
    };
    struct None {};

    const SsqPrefixParams& p;
    int lane, half;
    float inv;  // f16 parts: 1 / the codebook's scale
    uint32_t lds[2];
    uint4 q[QP][NR][NQ];
    // tokens
    const int32_t* table;
    int len, last_chunk, first, step, n_tiles;  // this wave's tiles: first + step i, i < n_tiles
    // of 32 tiles and the 32 after them (lane: piece lane & 1 of tile lane / 2), element offsets of the pieces' codes
    // and values
    int64_t pc, pv, pcn, pvn;
    int batch;
    const uint8_t* cbase;
    const uint16_t* vbase;
    uint32_t voff, vstep;                       // lane and 32-dim offsets in a page, elements
    std::conditional_t<HV, KeptOf<NK>, None> kept;

    __device__ __forceinline__ void entries(int i0, int64_t& oc, int64_t& ov, int64_t& ok) const {
        const int chunk = min(2 * (first + step * (i0 + (lane >> 1))) + (lane & 1), last_chunk);
        const int64_t page = table[chunk >> p.psh];
        const int at = 16 * (chunk & ((1 << p.psh) - 1));
        oc = page * p.a.c_sb + (int64_t)at * p.a.c_st;
        ov = page * p.a.v_sb + at;
        if constexpr (HV) ok = page * p.a.pt_sb + (int64_t)at * p.a.pt_st;
    }
    // this and the next 32 tiles' entries
    __device__ __forceinline__ void entries_now(int i0) {
        int64_t ok = 0;
        entries(i0, pc, pv, ok);
        pcn = pc;
        pvn = pv;
        if constexpr (HV) kept.o = kept.on = ok;
    }
    __device__ __forceinline__ void entries_next(int i0) {
        int64_t ok = 0;
        entries(i0, pcn, pvn, ok);
        if constexpr (HV) kept.on = ok;
    }
    __device__ __forceinline__ static int64_t of_lane(int64_t v, int l) {  // uniform
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), l);
        return (int64_t)(((uint64_t)hi << 32) | lo);
    }
    __device__ __forceinline__ void load_codes(int i, Codes& r) const {
        const int64_t o = (i >> 5) == batch ? pc : pcn;
        const int l = 2 * (i & 31);
        const int64_t o0 = of_lane(o, l), o1 = of_lane(o, l + 1);
        const uint8_t* row = cbase + (lane & 16 ? o1 : o0);  // cbase: this lane's token of a piece
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
    __device__ __forceinline__ void load_kept(int i) {
        if constexpr (HV) {
            const int64_t o = (i >> 5) == batch ? kept.o : kept.on;
            const int l = 2 * (i & 31);
            const int64_t o0 = of_lane(o, l), o1 = of_lane(o, l + 1);
            const uint16_t* row = kept.base + (lane & 16 ? o1 : o0);
#pragma unroll
            for (int k = 0; k < NK; ++k) {  // dims past the last: others, left out where they are used
                const int d = 16 * k + 8 * half;
                const uint2 x = *reinterpret_cast<const uint2*>(row + (d < p.kept ? d : 0));
                const uint2 y = *reinterpret_cast<const uint2*>(row + (d + 4 < p.kept ? d + 4 : 0));
                kept.v[k] = make_uint4(x.x, x.y, y.x, y.y);
            }
        }
    }
    __device__ __forceinline__ const uint16_t* val_row(int i, int c) const {
        return vbase + of_lane((i >> 5) == batch ? pv : pvn, 2 * (i & 31) + c);
    }
    __device__ __forceinline__ uint4 load_val(const uint16_t* row, int dt) const {
        return *reinterpret_cast<const uint4*>(row + voff + dt * vstep);
    }
    __device__ __forceinline__ void load_vals(int i, Vals& r) const {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) r.v[c][dt] = load_val(val_row(i, c), dt);
    }
    // the K^T operand of step st: dims 16 (st / 2) + 8 half .., the hi parts (st even) or the lo parts.  A gather's
    // address is code * 2 BD + a base, and the step's place in the instruction's 16-bit offset: lds[0] is the
    // codebook and this half's offset, lds[1] 64 KiB further.
    static constexpr int kPerHalf = 8 / BD, kBlk = 1024 * BD;  // blocks of a half's 8 dims; bytes of a block's tables
    template <class T>
    __device__ __forceinline__ T gather(uint32_t code, int at) const {  // at: a constant
        typedef const __attribute__((address_space(3))) T* Lds;
        return *(Lds)(code * (2 * BD) + lds[at >> 16] + (at & 0xFFFF));
    }
    __device__ __forceinline__ void set_book(const unsigned char* book) {
        lds[0] = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)book + half * (kPerHalf * kBlk);
        asm("" : "+v"(lds[0]));  // or the LDS's address is added again for every gather
        lds[1] = lds[0] + 65536;
        asm("" : "+v"(lds[1]));
    }
    __device__ __forceinline__ uint4 operand(const Codes& c, int st) const {
        const int s2 = st >> 1, at = s2 * 2 * kPerHalf * kBlk + (st & 1) * (kBlk / 2);
        if constexpr (BD == 8) {
            const pv4u x = gather<pv4u>(__builtin_amdgcn_ubfe(c.w[s2 >> 1], 16 * (s2 & 1) + 8 * half, 8), at);
            return make_uint4(x.x, x.y, x.z, x.w);
        } else if constexpr (BD == 4) {
            const uint32_t x = __builtin_amdgcn_ubfe(c.w[s2], 16 * half, 8), y = __builtin_amdgcn_ubfe(c.w[s2], 16 * half + 8, 8);
            const pv2u u = gather<pv2u>(x, at), v = gather<pv2u>(y, at + kBlk);
            return make_uint4(u.x, u.y, v.x, v.y);
        } else {
            const uint32_t w = half ? c.w[2 * s2 + 1] : c.w[2 * s2];
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = gather<uint32_t>((w >> (8 * k)) & 0xFFu, at + k * kBlk);
            return make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    // kAhead operands are gathered ahead of their MFMAs, across the end of a tile into the next one's codes: more do
    // not fit the registers beside 64 rows, and with 32 rows 8 of them cost more copies than they hide (64 sequences on
    // 32,768 tokens 81 us for 76)
    static constexpr int kAhead = 4;
    uint4 ring[kAhead];
    __device__ __forceinline__ void prime(const Codes& c) {
#pragma unroll
        for (int st = 0; st < kAhead; ++st) ring[st] = operand(c, st);
    }
    // beside(st): work for the vector units next to step st's MFMAs.  The barriers keep each step's gathers and
    // vector work between its MFMAs and the next ones: left alone, the compiler puts one kind after the other.
    // kept dims: the values asked for before, then those of tile i_kept are.
    template <class Beside>
    __device__ __forceinline__ void scores(const Codes& c, const Codes& next, int i_kept, pv16f (&s)[NR], Beside beside) {
#pragma unroll
        for (int st = 0; st < NST; ++st) {
            const uint4 kk = ring[st % kAhead];
#pragma unroll
            for (int h = 0; h < QP; ++h)
#pragma unroll
                for (int r = 0; r < NR; ++r) s[r] = pf_mfma<kF16>(kk, q[h][r][st >> 1], st || h ? s[r] : pv16f{});
            ring[st % kAhead] = st + kAhead < NST ? operand(c, st + kAhead) : operand(next, st + kAhead - NST);
            beside(st);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (HV) {  // in sums of their own, natural units
            pv16f t[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) t[r] = pv16f{};
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                if (16 * k >= p.kept) continue;  // uniform
                const int d = 16 * k + 8 * half;
                uint4 x = kept.v[k];
                if (d >= p.kept) x.x = x.y = 0u;
                if (d + 4 >= p.kept) x.z = x.w = 0u;
                uint4 part[KP];
                if constexpr (KP == 2) {
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) pf_split<kF16>(pf_lo<kVF16>(w[e]), pf_hi<kVF16>(w[e]), hi[e], lo[e]);
                    part[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    part[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                } else {
                    part[0] = x;
                }
#pragma unroll
                for (int h = 0; h < QP; ++h)
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int j = 0; j < KP; ++j) t[r] = pf_mfma<kF16>(part[j], kept.q[h][r][k], t[r]);
            }
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int k = 0; k < 16; ++k) s[r][k] = __builtin_fmaf(t[r][k], kLog2e, kF16 ? s[r][k] * inv : s[r][k]);
            load_kept(i_kept);
        }
    }
};

// the lane 32 apart
__device__ __forceinline__ float pf_other(float v) { return __shfl_xor(v, 32); }

// row R of a KV head's rows (b, qi, g): its sequence, query position and query head
__device__ __forceinline__ void pf_row(const SsqPrefixParams& p, int kv, int R, int& b, int& qi, int& h) {
    const int per_b = p.a.q_len * p.G;
    b = R / per_b;
    const int e = R - b * per_b;
    qi = e / p.G;
    h = kv * p.G + (e - qi * p.G);
}
__device__ __forceinline__ int64_t pf_rid(const SsqPrefixParams& p, int kv, int R) {
    int b, qi, h;
    pf_row(p, kv, R, b, qi, h);
    return ((int64_t)b * p.a.num_q_heads + h) * p.a.q_len + qi;
}
__device__ __forceinline__ int64_t pf_qrow(const SsqPrefixParams& p, int kv, int R) {
    int b, qi, h;
    pf_row(p, kv, R, b, qi, h);
    return (int64_t)b * p.a.q_sb + (int64_t)h * p.a.q_sh + (int64_t)qi * p.a.q_sl;
}

// element i of the queries (the split form takes any dtype), and an element scaled in its dtype
template <int QT>
__device__ __forceinline__ float pf_raw(const ssq_decode_args& a, int64_t i) {
    if constexpr (QT == kQtSplit) return ssq_load_elem(a.q, a.q_dtype, i);
    else return pf_lo<QT == kQtF16>(reinterpret_cast<const uint16_t*>(a.q)[i]);
}
// two elements scaled in their dtype, as packed 16-bit parts (a factor of 1 where there is no scale: exact)
template <int QT>
__device__ __forceinline__ void pf_parts(const ssq_decode_args& a, float scale, float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (QT == kQtSplit) {
        x = ssq_round_to(x * scale, a.q_dtype);
        y = ssq_round_to(y * scale, a.q_dtype);
        hi = pf_pack<false>(x, y);
        lo = pf_pack<false>(x - pf_lo<false>(hi), y - pf_hi<false>(hi));
    } else {
        hi = pf_pack<QT == kQtF16>(x * scale, y * scale);
        lo = 0;
    }
}

// eight consecutive dims
template <int QT>
__device__ __forceinline__ void pf_query8(const SsqPrefixParams& p, int64_t i, float (&x)[8]) {
    const ssq_decode_args& a = p.a;
    constexpr bool F16 = QT == kQtF16;
    if (QT != kQtSplit && p.q_vec) {  // uniform: rows of 16-byte pieces
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[2 * k] = pf_lo<F16>(w[k]);
            x[2 * k + 1] = pf_hi<F16>(w[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = pf_raw<QT>(a, i + k);
    }
}

// a wave's tokens: tiles first + step i (i < n) of a sequence of len > 0 tokens
template <class Run>
__device__ __forceinline__ void pf_tokens(Run& u, int kv, const int32_t* table, int len, int first, int step, int n) {
    const ssq_decode_args& a = u.p.a;
    u.table = table; u.len = len; u.last_chunk = (len - 1) >> 4;
    u.first = first; u.step = step; u.n_tiles = n;
    const int m = u.lane & 15;
    u.cbase = a.codes + (int64_t)kv * a.c_sh + (int64_t)(8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3)) * a.c_st;
    u.vbase = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)kv * a.v_sh;
    u.voff = (uint32_t)(u.lane & 31) * (uint32_t)a.v_st + 8 * u.half;
    u.vstep = 32 * (uint32_t)a.v_st;
    u.batch = 0;
    if constexpr (Run::kKept)
        u.kept.base = reinterpret_cast<const uint16_t*>(a.pt) + (int64_t)kv * a.pt_sh +
                      (int64_t)(8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3)) * a.pt_st;
    u.entries_now(0);
    if (n > 32) u.entries_next(32);
}

// Keeps a matrix-core operand in the accumulation registers, which the MFMAs read as well: the compiler otherwise
// parks what does not fit the 256 others there and copies it back for every use.
__device__ __forceinline__ void pf_pin(uint4& x) {
    pv4u v = {x.x, x.y, x.z, x.w};
    asm("" : "+a"(v));
    x = make_uint4(v.x, v.y, v.z, v.w);
}

// likewise an accumulator, where a branch that scales it would have all paths carry it in the others
__device__ __forceinline__ void pf_pin(pv16f& x) { asm("" : "+a"(x)); }

// max for numbers (an fmaxf would quieten its inputs first)
__device__ __forceinline__ float pf_max(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }
// Probabilities' sum of a lane's 16 tokens above which the running maximum moves (e^kSoftmaxSlack: each stays below it)
constexpr float kPfOver = 2980.958f;

// the first tiles' codes and values, asked for before the query rows are
template <class Run>
struct PfFirst {
    typename Run::Codes c1, c2, c3;
    typename Run::Vals val;
    __device__ __forceinline__ explicit PfFirst(Run& u) {
        if (u.n_tiles > 0) {  // wave-uniform
            u.load_codes(0, c1);
            u.load_codes(min(1, u.n_tiles - 1), c2);
            u.load_codes(min(2, u.n_tiles - 1), c3);
            u.load_vals(0, val);
            u.load_kept(0);
        }
    }
};

// The wave's tiles: a row's (m, l, o) over them, l over both halves.  mrow[r]: the additive mask's row of this lane's
// query row (MASK).
//
// One wave a SIMD issues one instruction every 4 cycles at best, so a tile costs its instructions: 48 MFMAs of 32 cycles
// for 64 rows of 128 dims leave room for about 340 others.  So the codebook is staged times log2(e): a probability is
// a subtraction and an exp2, and their sum, not a maximum per tile, tells when m has to move.  (With a mask the scores
// are taken back to natural units, where the type's lowest value stays what it is.)
template <bool MASK, int NR, class Run>
__device__ __forceinline__ void pf_tiles(Run& u, const PfFirst<Run>& first, const float* const (&mrow)[NR], float (&m_run)[NR],
                                         float (&l_run)[NR], pv16f (&o)[NR][Run::DT]) {
    const int n = u.n_tiles, len = u.len;
    if (n <= 0) return;  // wave-uniform
    typename Run::Codes c1 = first.c1, c2 = first.c2, c3 = first.c3;
    typename Run::Vals val = first.val;
    pv16f s[NR];  // scores and m: log2 units (scores times the codebook's scale), natural ones with a mask
    float m[NR], mb[NR];  // mb: m, or 0 while that is -inf (as the scores are: their probabilities are 0)
#pragma unroll
    for (int r = 0; r < NR; ++r) m[r] = -INFINITY;
    // tile i's mask, and its end where it holds the sequence's last token
    auto fix = [&](int i) {
        const int tile = u.first + u.step * i;
        const int t_half = kPfTile * tile + 8 * u.half;  // register k: token t_half + 16 (k / 8) + k % 8
        if constexpr (MASK) {
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int t = min(t_half + 16 * (k >> 3) + (k & 7), len - 1);
                    s[r][k] = __builtin_fmaf(s[r][k], Run::kScaled ? kLn2 * u.inv : kLn2, mrow[r][(int64_t)t * u.p.a.m_st]);
                }
        }
        if (kPfTile * (tile + 1) > len) {  // uniform
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
    };
    // a probability from its score
    auto prob = [&](float x, int r) {
        return __builtin_amdgcn_exp2f(MASK ? (x - mb[r]) * kLog2e : Run::kScaled ? __builtin_fmaf(x, u.inv, -mb[r]) : x - mb[r]);
    };
    auto top_of = [&](int r) {
        float top = s[r][0];
#pragma unroll
        for (int k = 1; k < 16; ++k) top = pf_max(top, s[r][k]);
        return pf_max(top, pf_other(top));
    };
    // raises m to the scores' maximum, by[r] >= 0 log2 units
    auto raise = [&](float (&by)[NR]) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float top = top_of(r);
            if (Run::kScaled && !MASK) top *= u.inv;
            const float mn = pf_max(m[r], top);
            by[r] = mn == -INFINITY ? 0.f : (mn - m[r]) * (MASK ? kLog2e : 1.f);
            m[r] = mn;
            mb[r] = mn == -INFINITY ? 0.f : mn;
        }
    };
    float by[NR];
    u.prime(c1);
    u.scores(c1, c2, min(1, n - 1), s, [](int) {});
    fix(0);
    raise(by);
    for (int i = 0; i < n; ++i) {
        if ((i & 31) == 31) {  // the next tile starts the next 32 entries (tiles up to i + 3 are asked for)
            u.batch = (i >> 5) + 1;
            u.pc = u.pcn;
            u.pv = u.pvn;
            if constexpr (Run::kKept) u.kept.o = u.kept.on;
            if (n > 32 * (u.batch + 1)) u.entries_next(32 * (u.batch + 1));
        }
        c1 = c2;
        c2 = c3;
        u.load_codes(min(i + 3, n - 1), c3);
        // the next tile's scores beside this tile's probabilities
        pv16f s2[NR];
        uint32_t pw[NR][8];  // P^T operands
        float e0[NR], lt[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) lt[r] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
        u.scores(c1, c2, min(i + 2, n - 1), s2, [&](int st) {
            constexpr int kPer = 16 / Run::NST;
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int x = 0; x < kPer; ++x) {
                    const int k = st * kPer + x;
                    const float e = prob(s[r][k], r);
                    lt[r] += e;
                    if (k & 1) pw[r][k >> 1] = pf_pack<Run::kVF16>(e0[r], e);
                    else e0[r] = e;
                }
        });
        bool over = false;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int dt = 0; dt < Run::DT; ++dt) pf_pin(o[r][dt]);
        // While a row has met hidden tokens only (m -inf), its probabilities, taken against 0, may underflow whatever
        // the scores are: these decide, not the sum.
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const bool none = m[r] == -INFINITY;
            over |= lt[r] > (none && !MASK ? -1.f : kPfOver);
            if (MASK && __builtin_amdgcn_ballot_w64(none) != 0) over |= none && top_of(r) > -INFINITY;
        }
        if (__builtin_amdgcn_ballot_w64(over) != 0) {  // m moves: once more from the scores
            raise(by);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float f = __builtin_amdgcn_exp2f(-by[r]);
                lt[r] = 0.f;
                l_run[r] *= f;
#pragma unroll
                for (int dt = 0; dt < Run::DT; ++dt) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[r][dt][k] *= f;
                    pf_pin(o[r][dt]);
                }
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const float x = prob(s[r][k], r), y = prob(s[r][k + 1], r);
                    pw[r][k >> 1] = pf_pack<Run::kVF16>(x, y);
                    lt[r] += x + y;
                }
            }
        }
        // P.V; a value operand's successor loads once it is used
        const uint16_t* vsrc[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) vsrc[c] = u.val_row(min(i + 1, n - 1), c);
#pragma unroll
        for (int r = 0; r < NR; ++r) l_run[r] += lt[r];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int dt = 0; dt < Run::DT; ++dt) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    o[r][dt] = pf_mfma<Run::kVF16>(val.v[c][dt], make_uint4(pw[r][4 * c], pw[r][4 * c + 1], pw[r][4 * c + 2], pw[r][4 * c + 3]), o[r][dt]);
                val.v[c][dt] = u.load_val(vsrc[c], dt);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r] = s2[r];
        if (i + 1 < n) fix(i + 1);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        l_run[r] += pf_other(l_run[r]);  // both halves' tokens
        m_run[r] = MASK || m[r] == -INFINITY ? m[r] : m[r] * kLn2;
        if (l_run[r] != l_run[r]) m_run[r] = 0.f;  // NaN scores: the maxima pass them over, the sum does not
    }
}

// A prefix item: rows [R0, R0 + nr) of the KV head over tiles [t0, t1) of the prefix (len tokens); partials go to
// slice `split`.  The whole workgroup calls it.  last: the workgroup's last item, after which the codebook's LDS is
// free for the join.
template <int D, int BD, int QT, int VT, int NR, bool HV>
__device__ __forceinline__ void pf_prefix_item(const SsqPrefixParams& p, unsigned char* lds, int kv, int R0, int nr,
                                               const uint16_t* permL, float inv, int len, int t0, int t1, int split, bool last) {
    using Run = PfRun<D, BD, QT, VT, NR, HV>;
    using L = PfLds<D>;
    const ssq_decode_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n_rows = (int64_t)a.batch * a.num_q_heads * a.q_len;
    float* ws_o = p.pre + (int64_t)split * n_rows * D;
    float* ws_m = p.pre + (int64_t)p.n1 * n_rows * D + (int64_t)split * n_rows;
    float* ws_l = ws_m + (int64_t)p.n1 * n_rows;
    unsigned char* scratch = lds + L::kBook;
    float* mL = reinterpret_cast<float*>(scratch + L::kScratch);  // [4][64]
    float* lL = mL + kPfWaves * 64;
    int64_t* rowL = reinterpret_cast<int64_t*>(lL + kPfWaves * 64);  // query rows' offsets, partial rows
    Run u{p};
    u.lane = lane; u.half = half; u.inv = inv;
    u.set_book(lds);
    pf_tokens(u, kv, p.ptab, len, t0 + wave, kPfWaves, (t1 - t0 - wave + kPfWaves - 1) / kPfWaves);
    const PfFirst<Run> first(u);

    // ---- query rows: pieces of 8 dims scaled in their dtype, as 16-bit parts; 32 rows of a part at a time go to
    // LDS as they are, are permuted there and become operands
    if (tid < 32 * NR) {
        const int R = R0 + min(tid, nr - 1);
        rowL[tid] = pf_qrow(p, kv, R);
        rowL[64 + tid] = pf_rid(p, kv, R);
    }
    __syncthreads();
    const float scale = a.has_scale ? a.scale : 1.f;
    constexpr int kPieces = 32 * D / 8 / kPfThreads;  // of 32 rows, per thread
    uint4 part[NR][Run::QP][kPieces];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int e = tid + k * kPfThreads, row = 32 * r + e / (D / 8), d = e % (D / 8) * 8;
            float x[8];
            pf_query8<QT>(p, rowL[row] + d, x);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pf_parts<QT>(a, scale, x[2 * i], x[2 * i + 1], hi[i], lo[i]);
                if (row >= nr) hi[i] = lo[i] = 0;
            }
            part[r][0][k] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (Run::QP == 2) part[r][1][k] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    uint16_t* rawL = reinterpret_cast<uint16_t*>(scratch);
    uint16_t* qL = rawL + 32 * D;
    const int j2 = tid % (D / 2);
    const uint32_t s0 = permL[2 * j2], s1 = permL[2 * j2 + 1];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int h = 0; h < Run::QP; ++h) {
            if (r || h) __syncthreads();  // the operands before are read
#pragma unroll
            for (int k = 0; k < kPieces; ++k) reinterpret_cast<uint4*>(rawL)[tid + k * kPfThreads] = part[r][h][k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 32 * (D / 2) / kPfThreads; ++k) {
                const int row = tid / (D / 2) + k * (2 * kPfThreads / D);
                reinterpret_cast<uint32_t*>(qL + row * L::kQRow)[j2] = rawL[row * D + s0] | ((uint32_t)rawL[row * D + s1] << 16);
            }
            __syncthreads();
#pragma unroll
            for (int st = 0; st < Run::NQ; ++st) {
                u.q[h][r][st] = *reinterpret_cast<const uint4*>(qL + col * L::kQRow + 16 * st + 8 * half);
                if constexpr (NR == 2) pf_pin(u.q[h][r][st]);
            }
            if constexpr (HV) {
                const uint16_t* keptL = reinterpret_cast<const uint16_t*>(lds + L::kKept);
#pragma unroll
                for (int k = 0; k < Run::NK; ++k) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = keptL[16 * k + 8 * half + 2 * e], y = keptL[16 * k + 8 * half + 2 * e + 1];
                        w[e] = (x < D ? qL[col * L::kQRow + x] : 0u) | (y < D ? (uint32_t)qL[col * L::kQRow + y] << 16 : 0u);
                    }
                    u.kept.q[h][r][k] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }

    const float* mrow[NR] = {};
    float m_run[NR], l_run[NR];
    pv16f o[NR][Run::DT];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int dt = 0; dt < Run::DT; ++dt) {
            o[r][dt] = pv16f{};
            pf_pin(o[r][dt]);
        }
    }
    pf_tiles<false, NR>(u, first, mrow, m_run, l_run, o);

    // ---- the four waves' (m, l), then o, 32 rows x 32 dims at a time (at weight 0 too: an infinite or NaN value
    // counts as in one pass; a wave without tiles has zeros)
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        if (half == 0) {
            mL[wave * 64 + 32 * r + col] = m_run[r];
            lL[wave * 64 + 32 * r + col] = l_run[r];
        }
    }
    __syncthreads();  // also: every wave is past its gathers
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
        const int64_t rid = rowL[64 + r];
        ws_m[rid] = M;
        ws_l[rid] = l;
    }
    const int jr = tid >> 3, jd = (tid & 7) * 4;  // the row and dims this thread joins
    constexpr int kTileF = kPfWaves * 32 * L::kJoinRow;  // floats of a (32 rows, 32 dims) tile of every wave
    float* jL = reinterpret_cast<float*>(last ? lds : scratch);
    auto join = [&](const float* src, int r, int dt) {
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kPfWaves; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(src + (w * 32 + jr) * L::kJoinRow + jd);
            t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
        }
        if (32 * r + jr < nr) *reinterpret_cast<float4*>(ws_o + rowL[64 + 32 * r + jr] * D + 32 * dt + jd) = t;
    };
    static_assert(NR * Run::DT * kTileF * 4 <= L::kBook + L::kScratch, "the last item's join fits the codebook's LDS");
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int dt = 0; dt < Run::DT; ++dt) {
            float* dst = jL + (last ? (r * Run::DT + dt) * kTileF : 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // dims 8 k + 4 half ..
                const float4 x = make_float4(o[r][dt][4 * k] * f[r], o[r][dt][4 * k + 1] * f[r], o[r][dt][4 * k + 2] * f[r], o[r][dt][4 * k + 3] * f[r]);
                *reinterpret_cast<float4*>(dst + (wave * 32 + col) * L::kJoinRow + 8 * k + 4 * half) = x;
            }
            if (!last) {  // uniform
                __syncthreads();
                join(jL, r, dt);
                __syncthreads();
            }
        }
    if (last) {
        __syncthreads();
#pragma unroll 2
        for (int t = 0; t < NR * Run::DT; ++t) join(jL + t * kTileF, t / Run::DT, t % Run::DT);
    }
}

// An own item: rows [R0, R0 + nr) (nr <= 32) of one sequence over tiles [t0, t1) of its own tokens, by one wave.
template <int D, int BD, int QT, int VT, bool MASK, bool HV>
__device__ __forceinline__ void pf_own_item(const SsqPrefixParams& p, const unsigned char* book, const uint16_t* permL, float inv,
                                            int kv, int R0, int nr, const int32_t* table, int len, int t0, int t1, int split) {
    using Run = PfRun<D, BD, QT, VT, 1, HV>;
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    Run u{p};
    u.lane = lane; u.half = half; u.inv = inv;
    u.set_book(book);
    pf_tokens(u, kv, table, len, t0, 1, t1 - t0);
    // query operands straight from memory: a lane's row, its half of every 16 permuted dims, all loads in flight
    const int R = R0 + min(col, nr - 1);
    const int64_t qrow = pf_qrow(p, kv, R);
    float x[Run::NQ + Run::NK][8];
#pragma unroll
    for (int st = 0; st < Run::NQ; ++st) {
        const uint4 pw = *reinterpret_cast<const uint4*>(permL + 16 * st + 8 * half);
        const uint32_t w[4] = {pw.x, pw.y, pw.z, pw.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) x[st][k] = pf_raw<QT>(a, qrow + ((w[k >> 1] >> (16 * (k & 1))) & 0xFFFFu));
    }
    if constexpr (HV) {
        const uint16_t* keptL = reinterpret_cast<const uint16_t*>(book + PfLds<D>::kKept);
#pragma unroll
        for (int st = 0; st < Run::NK; ++st)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t at = keptL[16 * st + 8 * half + k];
                x[Run::NQ + st][k] = at < D ? pf_raw<QT>(a, qrow + permL[at]) : 0.f;
            }
    }
    const PfFirst<Run> first(u);
    const float scale = a.has_scale ? a.scale : 1.f;
#pragma unroll
    for (int st = 0; st < Run::NQ + Run::NK; ++st) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            pf_parts<QT>(a, scale, x[st][2 * k], x[st][2 * k + 1], hi[k], lo[k]);
            if (col >= nr) hi[k] = lo[k] = 0;
        }
        const uint4 part[2] = {make_uint4(hi[0], hi[1], hi[2], hi[3]), make_uint4(lo[0], lo[1], lo[2], lo[3])};
#pragma unroll
        for (int h = 0; h < Run::QP; ++h) {
            if constexpr (HV) {
                if (st >= Run::NQ) {
                    u.kept.q[h][0][st - Run::NQ] = part[h];
                    continue;
                }
            }
            u.q[h][0][st] = part[h];
        }
    }
    const float* mrow[1] = {nullptr};
    if constexpr (MASK) {
        int b, qi, h;
        pf_row(p, kv, R, b, qi, h);
        mrow[0] = a.mask + (int64_t)b * a.m_sb + (int64_t)h * a.m_sh + (int64_t)qi * a.m_sl;
    }
    float m_run[1] = {-INFINITY}, l_run[1] = {0.f};
    pv16f o[1][Run::DT];
#pragma unroll
    for (int dt = 0; dt < Run::DT; ++dt) o[0][dt] = pv16f{};
    pf_tiles<MASK, 1>(u, first, mrow, m_run, l_run, o);
    if (col < nr) {
        const int64_t n_rows = (int64_t)a.batch * a.num_q_heads * a.q_len, rid = pf_rid(p, kv, R);
        float* ws_m = p.own + (int64_t)p.n2 * n_rows * D + (int64_t)split * n_rows;
        float* dst = p.own + ((int64_t)split * n_rows + rid) * D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < Run::DT; ++dt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float4*>(dst + 32 * dt + 8 * k) =
                    make_float4(o[0][dt][4 * k], o[0][dt][4 * k + 1], o[0][dt][4 * k + 2], o[0][dt][4 * k + 3]);
        if (half == 0) {
            ws_m[rid] = m_run[0];
            ws_m[(int64_t)p.n2 * n_rows + rid] = l_run[0];
        }
    }
}

// inclusive wave sum: row shifts by 1, 2, 4 and 8, then lane 15 and lane 31 of the rows below
__device__ __forceinline__ int pf_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// The sequences' own tokens, cut by their lengths (which only the device knows): pieces of `per` tiles, the size that
// gives every wave of the KV head about one, numbered sequence by sequence; wave v takes pieces v, v + n_waves, ...
// Every number follows from seq_lens, so all waves agree and a call repeats itself bit for bit.
template <int D, int BD, int QT, int VT, bool HV>
__device__ __forceinline__ void pf_own(const SsqPrefixParams& p, const unsigned char* book, const uint16_t* permL, float inv, int kv, int v) {
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & 63;
    const int n_waves = p.n_wg * kPfWaves, ns = a.batch * p.own_rg, per_b = a.q_len * p.G;
    auto tiles_of = [&](int s) {  // of sequence and row group s
        return s < ns ? ssq_prefix_tiles(max(0, min(a.seq_lens[s / p.own_rg], a.seq_len))) : 0;
    };
    const int t_first = tiles_of(lane);
    auto count = [&](int per) {  // pieces of all sequences
        int c = __builtin_amdgcn_readlane(pf_scan((t_first + per - 1) / per), 63);
        for (int s0 = 64; s0 < ns; s0 += 64) c += __builtin_amdgcn_readlane(pf_scan((tiles_of(s0 + lane) + per - 1) / per), 63);
        return c;
    };
    // pieces of the fewest tiles, or larger ones where that is more than a piece a wave
    int per = p.own_min, n = count(per);
    if (n > n_waves) {
        const int total = count(1);
        per = max(per, (total + n_waves - 1) / n_waves);
        n = count(per);
        for (int k = 0; k < 6 && n > n_waves && ns <= n_waves; ++k) {
            per += (per + 3) / 4;
            n = count(per);
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.own_per[0] = per;
    int s0 = 0, base = 0, t = t_first, c = (t_first + per - 1) / per, inc = pf_scan(c);
    for (int it = v; it < n; it += n_waves) {
        while (it >= base + __builtin_amdgcn_readlane(inc, 63)) {  // it < n: ends before s0 passes ns
            base += __builtin_amdgcn_readlane(inc, 63);
            s0 += 64;
            t = tiles_of(s0 + lane);
            c = (t + per - 1) / per;
            inc = pf_scan(c);
        }
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + inc > it));
        const int split = it - base - __builtin_amdgcn_readlane(inc - c, l);
        const int s = s0 + l, b = s / p.own_rg, r0 = (s - b * p.own_rg) * 32;
        const int t0 = split * per, t1 = min(t0 + per, __builtin_amdgcn_readlane(t, l));
        const int len = max(0, min(a.seq_lens[b], a.seq_len));
        const int32_t* table = a.block_table + (int64_t)b * a.bt_sb;
        if (a.mask) pf_own_item<D, BD, QT, VT, true, HV>(p, book, permL, inv, kv, b * per_b + r0, min(32, per_b - r0), table, len, t0, t1, split);
        else pf_own_item<D, BD, QT, VT, false, HV>(p, book, permL, inv, kv, b * per_b + r0, min(32, per_b - r0), table, len, t0, t1, split);
    }
}

template <int D, int BD, int QT, int VT, bool HV>
__global__ __launch_bounds__(kPfThreads, 1) void k_prefix(const SsqPrefixParams p) {
    extern __shared__ __align__(16) unsigned char pf_lds[];
    using L = PfLds<D>;
    const ssq_decode_args& a = p.a;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = blockIdx.x % a.num_kv_heads, w = blockIdx.x / a.num_kv_heads;
    uint16_t* permL = reinterpret_cast<uint16_t*>(pf_lds + L::kPerm);
    // a permuted dim's source, for this thread's staging and for the waves' own rows
    const int64_t pj = (int64_t)min((uint64_t)a.perm[(int64_t)kv * a.perm_sh + tid % D], (uint64_t)(D - 1));
    const int plen = p.n1 ? max(0, min(p.plen[0], p.pcap)) : 0;
    float inv = 1.f;
    // ---- the KV head's codebook times log2(e) (and, in f16 parts, a power of two) as 16-bit parts: a thread takes the
    // same codeword (or half of one, at 8 dims) of every block, all of them in flight; workgroups start at different
    // blocks, since those of one KV head share an L2
    {
        constexpr bool F16 = QT == kQtF16;
        constexpr int NB = D / BD, kV = BD < 4 ? BD : 4, kParts = BD / kV;  // floats of a piece, pieces of a codeword
        const float* cent = a.cent + (int64_t)kv * a.cent_sh;
        const int nc = a.n_centroids;
        auto block = [&](int i) { return (i + w) & (NB - 1); };
        auto zero = [&](int i) { return HV && ssq_is_heavy(a.heavy_mask[0], a.heavy_mask[1], block(i)); };
        float x[NB][kParts][kV];  // at most 128 floats a lane
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const float* src = cent + block(i) * nc * BD;  // uniform
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                const int e = min(tid + j * kPfThreads, nc * kParts - 1);
                if constexpr (kV == 4) {
                    const float4 v = reinterpret_cast<const float4*>(src)[e];
                    x[i][j][0] = v.x; x[i][j][1] = v.y; x[i][j][2] = v.z; x[i][j][3] = v.w;
                } else {
                    const float2 v = reinterpret_cast<const float2*>(src)[e];
                    x[i][j][0] = v.x; x[i][j][1] = v.y;
                }
            }
        }
        float unit = kLog2e;
        if constexpr (F16) {
            // The power of two takes the head's largest codeword to [2^13, 2^14): what the low parts drop, half a step of
            // f16's subnormals (2^-25) where they are small, is then at most 2^-38 of it, whatever the keys' size.
            // Scores are scaled back where the maximum is subtracted.  A codeword without a finite value does not count.
            auto largest = [&](bool all) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    float t = 0.f;
#pragma unroll
                    for (int j = 0; j < kParts; ++j)
#pragma unroll
                        for (int k = 0; k < kV; ++k) {
                            const float y = __builtin_fabsf(x[i][j][k]);
                            t = pf_max(t, all || y < INFINITY ? y : 0.f);
                        }
                    top = pf_max(top, zero(i) ? 0.f : t);
                }
                return ssq_wave_max(top);
            };
            float top = largest(true);
            if (!(top < INFINITY)) top = largest(false);  // uniform
            float* topL = reinterpret_cast<float*>(pf_lds + L::kBook);
            if ((tid & 63) == 0) topL[wave] = top;
            __syncthreads();
            top = fmaxf(fmaxf(topL[0], topL[1]), fmaxf(topL[2], topL[3]));
            const int up = top > 0.f ? max(-100, min(100, 14 - __builtin_amdgcn_frexp_expf(top))) : 0;
            unit = kLog2e * __uint_as_float((uint32_t)(127 + up) << 23);
            inv = __uint_as_float((uint32_t)(127 - up) << 23);
            inv = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(inv)));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            unsigned char* blk = pf_lds + block(i) * 1024 * BD;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                uint32_t hi[kV / 2], lo[kV / 2];
#pragma unroll
                for (int k = 0; k < kV / 2; ++k) {
                    pf_split<F16>(x[i][j][2 * k] * unit, x[i][j][2 * k + 1] * unit, hi[k], lo[k]);
                    if (zero(i)) hi[k] = lo[k] = 0;
                }
                // past the last codeword: it again
                unsigned char* dst = blk + min(tid + j * kPfThreads, nc * kParts - 1) * 2 * kV;
                if constexpr (BD == 2) {
                    *reinterpret_cast<uint32_t*>(dst) = hi[0];
                    *reinterpret_cast<uint32_t*>(dst + 512 * BD) = lo[0];
                } else {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(dst + 512 * BD) = make_uint2(lo[0], lo[1]);
                }
            }
        }
        if (tid < D) permL[tid] = (uint16_t)pj;
        if constexpr (HV) {  // where kept dim tid is
            if (tid < L::kKeptMax) {
                int at = 0xFFFF, left = tid / BD;
                for (int blk = 0; blk < NB; ++blk)
                    if (ssq_is_heavy(a.heavy_mask[0], a.heavy_mask[1], blk) && left-- == 0) at = blk * BD + tid % BD;
                reinterpret_cast<uint16_t*>(pf_lds + L::kKept)[tid] = (uint16_t)at;
            }
        }
    }
    __syncthreads();
    // (from the last workgroup down: a small prefix has the first ones)
    if (p.n2) pf_own<D, BD, QT, VT, HV>(p, pf_lds, permL, inv, kv, (p.n_wg - 1 - w) * kPfWaves + wave);
    // ---- the prefix: slices past its length are not read by the merge either
    const int tiles = ssq_prefix_tiles(plen), per = p.n1 ? ssq_prefix_slice(plen, p.n1) : 0;
    const int n_pre = per ? p.n_rg * ((tiles + per - 1) / per) : 0;
    for (int it = w; it < n_pre; it += p.n_wg) {
        const int split = it / p.n_rg, rg = it - split * p.n_rg;  // the groups of one slice side by side
        const int R0 = rg * 32 * p.pre_nr, nr = min(32 * p.pre_nr, p.rows - R0);
        const int t0 = split * per, t1 = min(t0 + per, tiles);
        if constexpr (QT != kQtSplit && !HV) {
            if (p.pre_nr == 2) {
                pf_prefix_item<D, BD, QT, VT, 2, HV>(p, pf_lds, kv, R0, nr, permL, inv, plen, t0, t1, split, it + p.n_wg >= n_pre);
                continue;
            }
        }
        pf_prefix_item<D, BD, QT, VT, 1, HV>(p, pf_lds, kv, R0, nr, permL, inv, plen, t0, t1, split, it + p.n_wg >= n_pre);
    }
}

template <int D, int BD, int QT, int VT, bool HV>
int launch_prefix(const SsqPrefixParams& p, hipStream_t st) {
    auto kern = k_prefix<D, BD, QT, VT, HV>;
    int rc = ssq_allow_lds((const void*)kern, PfLds<D>::kTotal, "hipFuncSetAttribute(k_prefix)");
    if (rc) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.n_wg * p.a.num_kv_heads)), dim3(kPfThreads), PfLds<D>::kTotal, st, p);
    return ssq_check_hip(hipGetLastError(), "k_prefix launch");
}

template <int QT, int VT, bool HV>
int launch_prefix_qv(const SsqPrefixParams& p, hipStream_t st) {
    if (p.a.head_dim == 64) {
        switch (p.a.block_dim) {
            case 2: return launch_prefix<64, 2, QT, VT, HV>(p, st);
            case 4: return launch_prefix<64, 4, QT, VT, HV>(p, st);
            default: return launch_prefix<64, 8, QT, VT, HV>(p, st);
        }
    }
    switch (p.a.block_dim) {
        case 2: return launch_prefix<128, 2, QT, VT, HV>(p, st);
        case 4: return launch_prefix<128, 4, QT, VT, HV>(p, st);
        default: return launch_prefix<128, 8, QT, VT, HV>(p, st);
    }
}

}  // namespace
