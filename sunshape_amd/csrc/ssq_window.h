// Causal attention over VQ-coded pages with 16- or 8-bit values, a sliding window and sinks (ssq_decode_window):
// parameters, and the kernel template that ssq_window_*.hip instantiates.
//
// What it computes.  Row i of the Lq newest tokens of a sequence of n tokens stands at p = n - Lq + i and sees the
// tokens j <= p with j > p - window or j < sinks:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = e^{q . k_j},  lse = log sum_j w_j,
// k_j the codewords that token j's codes name, v_j the stored value, times its page's scale for 8-bit values.
//
// Everything is held transposed: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32, a lane's column being one
// query row throughout, so the softmax's statistics and the rescale of O stay in the lane but for one exchange between
// the four lane groups.  A tile has 4 x CH tokens, CH = 16 (8-bit values) or 8: lane group h = lane / 16 is given the
// CH tokens that follow CH h, which is one 16-byte piece of a dim-major value page per dim: the V^T operand.
// Matrix row m = 4 g + i of score product s is token CH g + 4 s + i, so the four accumulator registers of group h
// hold tokens CH h + 4 s .. + 3: P^T's operand as it stands, with no lane crossed.
// K^T's operand is gathered codeword by codeword from the codebook in LDS.  A codeword is stored as two f16 parts of
// c 2^k (hi = its rounding, lo = the rounding of what that left; k per KV head, so that the largest codeword is
// below 2^15), next to each other: a gather feeds hi and lo as the two halves of the K dimension against the
// query's dims given twice.  Dropped is 2^-22 of a codeword, or 2^-40 of the head's largest.  Queries enter as f16 at
// a power of two of the row's own: exact for 16-bit ones (elements below 2^-29 of the row's largest apart), fp32 ones
// in two parts.
// Probabilities are 2^(x - m), m kept 14 below the row's running maximum, so that f16 holds them with 11 bits down to 2^-28 of
// the largest (8-bit and f16 values; with bf16 values they are rounded to bf16, as in the other decode kernels, and kept small
// enough that their sums of such values are finite: kWinTop).  What is joined is averages with their sums, not sums.  A page's scale
// joins them before the rounding, relative to the largest scale that the row has met, which its O is kept in units of: f16 then has
// 11 bits down to 2^-20 of the row's largest probability at the least (and nothing below 2^-31), as a tile with a page whose scale is less than
// 2^-8 of that takes its products in 32 bits (kWinFar).
//
// Bound by memory for long contexts: 64 sequences of 32,768 tokens (32 / 8 heads of 128, 8-bit values, 2.69 GB) take 424 us,
// 6.3 TB/s, where a probe that only reads reaches 6.85; by about 10 us before the first tile (loads, lengths, codebook, queries) and 5
// of the join for short ones: one sequence of 517 tokens 11.7 us.  What k_window_wide takes from many rows is in ssq_window_wide.h.
#pragma once

#include "ssq_common.h"

#include <type_traits>

struct SsqWindowParams {
    ssq_decode_args a;
    int window, sinks;       // window: INT_MAX where everything is seen
    int out_dtype;
    int n_pages;
    const float* v_scale;
    int64_t vs_sb, vs_sh;
    int G, rows, rgroups;    // query rows of a (sequence, KV head): (qi, g), g fastest; groups of item_rows
    int items;               // batch * rgroups
    int n_wg;                // workgroups per KV head
    int form;                // kWinTeam: a workgroup's waves share whole items; kWinShares: each wave has an equal share of all
                             // tiles (WinCut); kWinWide: each workgroup has, over items of 256 rows
    int item_rows, workers;  // rows of an item; those that share the tiles of a KV head
    int fixed, least;        // an item's cost beside its tiles, and the smallest share, both in tiles
    int psh;                 // log2(page_size / 16)
    int q_vec, out_vec;      // query rows load in 16-byte pieces; four values of the output store as one
    float* part;             // [Hkv][workers][2] slots of item_rows x (Dv + 2): o, then m (log2 units), l
    int* meta;               // [items][2]: first worker * 2 + its slot, and pieces
};

#define SSQ_WINDOW_UNIT(name) int name(const SsqWindowParams& p, hipStream_t st)
SSQ_WINDOW_UNIT(ssq_window_64_e4m3);
SSQ_WINDOW_UNIT(ssq_window_64_bf16);
SSQ_WINDOW_UNIT(ssq_window_64_f16);
SSQ_WINDOW_UNIT(ssq_window_128_e4m3);
SSQ_WINDOW_UNIT(ssq_window_128_bf16);
SSQ_WINDOW_UNIT(ssq_window_128_f16);

// waves of a workgroup: two a SIMD, so that one's matrix products run beside the other's vector work.  (32 rows a wave, half as
// many gathers for a row, leave registers for one: 20 rows a sequence 43 us for 36, a chunk of 512 tokens 162 for 119.)
constexpr int kWinWaves = 8, kWinThreads = kWinWaves * 64, kWinRows = 16, kWinWideRows = 256;
enum { kWinTeam, kWinShares, kWinWide };

// what the tiles of an item follow from, beside its length
struct WinShape { int window, sinks, q_len, G, rows; };
__host__ __device__ __forceinline__ WinShape win_shape(const SsqWindowParams& p) {
    return {p.window, p.sinks, p.a.q_len, p.G, p.rows};
}
// tiles of an item that some row of it sees
struct WinTiles {
    int p_lo, p_hi;      // the first and last row's positions
    int n, n_sink, from; // tile i: i < n_sink ? i : from + i - n_sink
};
template <int TT, int ROWS>
__host__ __device__ __forceinline__ WinTiles win_tiles(const WinShape& p, int len, int row0) {
    WinTiles t;
    const int last = (row0 + ROWS < p.rows ? row0 + ROWS : p.rows) - 1;
    t.p_lo = len - p.q_len + row0 / p.G;
    t.p_hi = len - p.q_len + last / p.G;
    t.n = t.n_sink = t.from = 0;
    if (t.p_hi < 0) return t;
    const int lo = t.p_lo >= p.window ? t.p_lo - p.window + 1 : 0;
    const int ns = ((p.sinks < t.p_hi + 1 ? p.sinks : t.p_hi + 1) + TT - 1) / TT;
    if (lo / TT > ns) {
        t.n_sink = ns;
        t.from = lo / TT;
    }
    t.n = t.n_sink + t.p_hi / TT - t.from + 1;
    return t;
}

namespace {

typedef float w4f __attribute__((ext_vector_type(4)));
typedef _Float16 w8h __attribute__((ext_vector_type(8)));
typedef _Float16 w2h __attribute__((ext_vector_type(2)));
typedef __bf16 w8b __attribute__((ext_vector_type(8)));
typedef __bf16 w2b __attribute__((ext_vector_type(2)));
typedef float w2f __attribute__((ext_vector_type(2)));
typedef unsigned int w4u __attribute__((ext_vector_type(4)));
typedef unsigned int w2u __attribute__((ext_vector_type(2)));

constexpr float kWinLog2e = 1.4426950408889634f, kWinLn2 = 0.6931471805599453f;
constexpr float kWinNone = -3.0e38f;  // m of a row that has met nothing
// log2 of the largest probability when m moves, and of what moves it.  f16 holds the most below 2^15.5.  bf16 holds as many bits of any
// size, but its values reach 2^128: what a row's probabilities sum to stays below 1 there, so that O, which is divided by the sum
// at the end, never passes its values (a lane's sum is at most kWinMass when a tile begins, a row's four lanes' 2^-2, and a tile adds 64 * 2^-6.5 at most;
// past kWinMass m moves 4 up).
template <int VT>
constexpr float kWinTop = VT == SSQ_BF16 ? -8.f : 14.f;
template <int VT>
constexpr float kWinOver = VT == SSQ_BF16 ? -6.5f : 15.5f;
constexpr float kWinMass = 0.0625f;
constexpr float kWinScale = 7.888609052210118e-31f;  // 2^-100, the smallest unit of O
constexpr float kWinFar = 0.00390625f;  // 2^-8: of the unit, what a page's scale has to be for its probabilities to go to f16 with it

__device__ __forceinline__ w4f win_mfma(const uint4& a, const uint4& b, w4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w8h, a), __builtin_bit_cast(w8h, b), c, 0, 0, 0);
}
template <int VT>
__device__ __forceinline__ w4f win_mfma_v(const uint4& a, const uint4& b, w4f c) {
    if constexpr (VT == SSQ_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w8b, a), __builtin_bit_cast(w8b, b), c, 0, 0, 0);
    else
        return win_mfma(a, b, c);
}
__device__ __forceinline__ uint32_t win_pack_h(float a, float b) {  // RNE
    const w2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, w2h));
}
template <int VT>
__device__ __forceinline__ uint32_t win_pack_p(float a, float b) {
    const w2f f = {a, b};
    if constexpr (VT == SSQ_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, w2b));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, w2h));
}
__device__ __forceinline__ float win_h(uint32_t w, int i) { return ssq_f16_to_f32(i ? w >> 16 : w & 0xFFFFu); }
// x rounded to f16, and the rounding of what that left (CHECKED: 0 beside an infinity)
template <bool CHECKED>
__device__ __forceinline__ void win_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = win_pack_h(x, y);
    const float u = x - win_h(hi, 0), v = y - win_h(hi, 1);
    lo = CHECKED ? win_pack_h(__builtin_isfinite(u) ? u : 0.f, __builtin_isfinite(v) ? v : 0.f) : win_pack_h(u, v);
}
// four e4m3 values as two packed pairs of f16 (exact)
__device__ __forceinline__ w2u win_e4m3(uint32_t w) {
    w2u r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    return r;
}
// exponent e with x < 2^e, of a positive finite x (0: 0)
__device__ __forceinline__ int win_exp(float x) { return x > 0.f ? __builtin_amdgcn_frexp_expf(x) : 0; }

// four values to the output's dtype, as one piece
__device__ __forceinline__ void win_store4(void* out, int dtype, int64_t i, w4f z) {
    if (dtype == SSQ_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + i) = make_float4(z[0], z[1], z[2], z[3]);
    } else {
        const uint2 w = dtype == SSQ_BF16 ? make_uint2(win_pack_p<SSQ_BF16>(z[0], z[1]), win_pack_p<SSQ_BF16>(z[2], z[3]))
                                          : make_uint2(win_pack_h(z[0], z[1]), win_pack_h(z[2], z[3]));
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + i) = w;
    }
}

// a wave's LDS writes before this point are seen by its reads after it (one wave's LDS operations execute in order)
__device__ __forceinline__ void win_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 32-bit products, a lane's value of its dim and its row's probability each, of a token a lane group: what a page far below the
// unit takes, whose f16 would have bits to lose (16 of these for one of 16 bits, and rare: with such a page in every tile 64 sequences
// of 32,768 take 886 us for 424)
__device__ __forceinline__ w4f win_mfma_32(float a, float b, w4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// four e4m3 values
__device__ __forceinline__ w4f win_e4m3_32(uint32_t w) {
    return w4f{__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1), __builtin_amdgcn_cvt_f32_fp8((int)w, 2),
               __builtin_amdgcn_cvt_f32_fp8((int)w, 3)};
}
// a part w of an average, or infinite as it is (its weight is above 0, whatever 32 bits make of it)
__device__ __forceinline__ float win_part(float z, float w) { return fabsf(z) == INFINITY ? z : z * w; }
__device__ __forceinline__ w4f win_part(w4f z, float w) { return w4f{win_part(z[0], w), win_part(z[1], w), win_part(z[2], w), win_part(z[3], w)}; }
// whether a lane's largest score, or its sum, takes m up
template <int VT>
__device__ __forceinline__ bool win_over(float top, float m, float l) {
    if constexpr (VT == SSQ_BF16) return (top > m + kWinOver<VT>) | (l > kWinMass);
    else return top > m + kWinOver<VT>;
}
// a group's value over the four lane groups of a column
__device__ __forceinline__ float win_max4(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float win_sum4(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// A kernel's arguments, to be loaded where they are used: taken from the parameter, all 60 words of them would stay in scalar
// registers across the loops, and those that do not fit in lanes of vector registers, which the tiles need.
typedef const __attribute__((address_space(4))) SsqWindowParams* WinArgs;
__device__ __forceinline__ WinArgs win_args() {
    WinArgs k = (WinArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return k;
}

// Equal shares of the items' tiles: the items of a KV head lie end to end on a cost axis, fixed + tiles each, and worker w (a
// wave, those of a workgroup n_wg apart; or a workgroup) takes [w share, (w + 1) share).  An item inside one share is written out by its
// wave; one that spans several leaves a partial in each: slot 0 of a worker for the item its share starts in, slot 1 for one that
// starts in it.  Everything follows from the lengths, which the host does not see.  Waves that wait for nobody keep the memory
// busy through one another's beginnings and ends.
template <int TT, int ROWS>
struct WinCut {
    int share, total;
    int c0, v0;  // this lane's cost and inclusive sum over the first 64 items
    __device__ __forceinline__ static int length(WinArgs p, int i) { return p->a.seq_lens[min(i, p->items - 1) / p->rgroups]; }
    __device__ __forceinline__ static int cost(WinArgs p, int i, int len) {
        if (i >= p->items) return 0;
        const WinShape s{p->window, p->sinks, p->a.q_len, p->G, p->rows};
        return p->fixed + win_tiles<TT, ROWS>(s, max(0, min(len, p->a.seq_len)), i % p->rgroups * ROWS).n;
    }
    __device__ __forceinline__ static int scan(int v) {  // inclusive, over the wave
        v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
        return v;
    }
    // (the whole wave calls these two; len: length(lane), asked for before)
    __device__ __forceinline__ void init(WinArgs p, int lane, int len) {
        c0 = cost(p, lane, len);
        v0 = scan(c0);
        total = __builtin_amdgcn_readlane(v0, 63);
        for (int i = SSQ_WAVE; i < p->items; i += SSQ_WAVE)
            total += __builtin_amdgcn_readlane(scan(cost(p, i + lane, length(p, i + lane))), 63);
        share = max((total + p->workers - 1) / p->workers, p->least);
    }
    // the item that holds cost position x < total, and its start.  Once a worker: the items behind it follow one by one (131,072 short
    // sequences 2.2 ms, 61 with a search for each).
    __device__ __forceinline__ void find(WinArgs p, int lane, int x, int& item, int& s) const {  // (uniform results)
        int base = 0, mine = c0, v = v0;
        for (int f = 0;;) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(base + v > x);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                item = f + l;
                s = base + __builtin_amdgcn_readlane(v, l) - __builtin_amdgcn_readlane(mine, l);
                return;
            }
            base += __builtin_amdgcn_readlane(v, 63);
            f += SSQ_WAVE;
            if (f >= p->items) break;  // not reached for x < total
            mine = cost(p, f + lane, length(p, f + lane));
            v = scan(mine);
        }
        item = p->items;
        s = x;
    }
};

// LDS: codebook | the waves' query rows, and their join | m, l [waves][16] | reduction [waves] | permutation [D]
// A KV head's codebook: 64 (32) floats a thread, all asked for at once, staged in LDS as two f16 parts times 2^k.
template <int D, int BD>
struct WinBook {
    static constexpr int kPer = D / BD * 256 / kWinThreads;
    float c[kPer][BD];
    __device__ __forceinline__ void load(WinArgs p, int kv, int tid) {
        const float* cent = p->a.cent + (int64_t)kv * p->a.cent_sh;
        auto entry = [&](int k, const float* src) {
            if constexpr (BD >= 4) {
#pragma unroll
                for (int d = 0; d < BD; d += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(src + d);
                    c[k][d] = x.x; c[k][d + 1] = x.y; c[k][d + 2] = x.z; c[k][d + 3] = x.w;
                }
            } else {
                const float2 x = *reinterpret_cast<const float2*>(src);
                c[k][0] = x.x; c[k][1] = x.y;
            }
        };
        const int n = p->a.n_centroids;  // entry e = tid + k * kWinThreads: block e / 256, codeword e % 256
        const float* src = cent + ((tid >> 8) * n + min(tid & 255, n - 1)) * BD;
#pragma unroll
        for (int k = 0; k < kPer; ++k) entry(k, src + k * (kWinThreads / 256 * BD) * n);
    }
    // The whole workgroup; returns k.  Entry e is at 4 BD e: BD 2 hi, lo; 4 hi, hi, lo, lo; 8 four words hi, four lo.
    __device__ __forceinline__ int stage(unsigned char* smem, float* red, int tid, int lane, int wave) const {
        // the largest finite codeword; infinite ones (rare) cost a second look and checks on the way
        auto largest = [&](auto checked) {
            float most = 0.f;
#pragma unroll
            for (int k = 0; k < kPer; ++k)
#pragma unroll
                for (int d = 0; d < BD; ++d) {
                    const float z = fabsf(c[k][d]);
                    most = fmaxf(most, !checked || z < INFINITY ? z : 0.f);
                }
            most = ssq_wave_max(most);
            __syncthreads();
            if (lane == 0) red[wave] = most;
            __syncthreads();
            most = 0.f;
#pragma unroll
            for (int w = 0; w < kWinWaves; ++w) most = fmaxf(most, red[w]);
            return most;
        };
        float most = largest(std::false_type{});
        const bool infinite = most == INFINITY;  // uniform
        if (infinite) most = largest(std::true_type{});
        const int book_exp = min(15 - win_exp(most), 126), n_centroids = win_args()->a.n_centroids;
        auto put = [&](auto checked) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int e = tid + k * kWinThreads;
                const float scale = (e & 255) < n_centroids ? ldexpf(1.f, book_exp) : 0.f;
                uint32_t hi[BD / 2], lo[BD / 2];
#pragma unroll
                for (int d = 0; d < BD; d += 2) win_split<checked>(c[k][d] * scale, c[k][d + 1] * scale, hi[d / 2], lo[d / 2]);
                unsigned char* at = smem + e * (4 * BD);
                if constexpr (BD == 8) {
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(at + 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                } else if constexpr (BD == 4) {
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
                } else {
                    *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], lo[0]);
                }
            }
        };
        if (infinite) put(std::true_type{});
        else put(std::false_type{});
        __syncthreads();
        return book_exp;
    }
};

template <int D>
struct WinLds {
    static constexpr int kBook = D * 256 * 4;
    static constexpr int kJoinRows = 4;
    static constexpr int kJoinRow = D + 4;  // floats
    static constexpr int kQRow = 2 * D + 16;  // bytes of a 16-bit query row; 8 of them a wave at a time, or 4 of 32 bits
    static constexpr int kQ = kWinWaves * 8 * kQRow, kJoin = kWinWaves * kJoinRows * kJoinRow * 4;
    static constexpr int kMl = kBook + (kQ > kJoin ? kQ : kJoin);
    static constexpr int kRed = kMl + 2 * kWinWaves * kWinRows * 4;
    static constexpr int kPerm = kRed + kWinWaves * 4;
    static constexpr int kTotal = kPerm + 2 * D;
};

// D: head_dim and value_dim, BD: block_dim, VT: value dtype, QP: query parts
template <int D, int BD, int VT, int QP>
struct WinRun {
    static constexpr bool kV8 = VT == SSQ_E4M3;
    static constexpr int CH = kV8 ? 16 : 8;        // tokens of a lane group
    static constexpr int TT = 4 * CH;              // tokens of a tile
    static constexpr int NS = CH / 4;              // score products (16 tokens each)
    static constexpr int NB = D / BD;
    static constexpr int NCL = NB / 4;             // codes of a token that a lane gathers
    static constexpr int NW = (NCL + 3) / 4;       // in words
    static constexpr int DT = D / 16;
    static constexpr int NK = D / 16;              // score MFMAs of 16 tokens (a lane's four dims, hi and lo, each)
    static constexpr int NQ = BD == 8 ? NK / 2 : NK;  // query operands
    static constexpr int NE = D / 4;               // query dims of a lane
    using L = WinLds<D>;

    static constexpr int NST = NS * NK;            // score steps of a tile
    static constexpr int kAhead = 4;               // operands gathered ahead

    struct Codes { uint32_t w[NS][NW]; };
    struct Vals {
        w4u v[DT];
        float scale;
    };

    int lane, col, grp;
    int window, sinks, n_pages, psh;
    uint32_t c_sb, c_st, v_sb, vs_sb;  // strides (v_sb in bytes)
    const float* v_scale;           // of this KV head
    uint32_t book;                  // LDS address of the codebook, and this group's blocks in it
    uint4 q[QP][NQ];
    float fac;                      // scores to log2 units
    // the item
    int pos;                        // this column's position
    WinTiles t{};
    const int32_t* table;
    int last_tok;
    // addresses
    const uint8_t* cbase;           // this lane's token of a chunk, its codes
    const uint8_t* vbase;
    uint32_t vstep;                 // 16 dims, bytes

    __device__ __forceinline__ int tile_of(int i) const { return i < t.n_sink ? i : t.from + i - t.n_sink; }
    // the page table's entry of chunk g of tile i: its page (always one of the cache's) and place in it
    __device__ __forceinline__ void entry(int i, int g, int& page, int& at) const {
        const int tok = min(TT * tile_of(i) + CH * g, last_tok & ~(CH - 1));
        page = min((uint32_t)table[(tok >> 4) >> psh], (uint32_t)(n_pages - 1));
        at = tok & ((16 << psh) - 1);
    }
    struct Place { int page, at; };
    __device__ __forceinline__ Place place(int i, int g) const {
        Place e;
        entry(i, g, e.page, e.at);
        return e;
    }
    __device__ __forceinline__ int code_chunk() const { return (lane >> 2) & 3; }
    __device__ __forceinline__ void load_codes(const Place& e, Codes& r) const {
        const uint8_t* row = cbase + (uint64_t)(uint32_t)e.page * c_sb + (uint32_t)e.at * c_st;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const uint8_t* src = row + 4 * s * c_st;
            if constexpr (NCL == 16) {
                const w4u x = __builtin_nontemporal_load(reinterpret_cast<const w4u*>(src));
                r.w[s][0] = x.x; r.w[s][1] = x.y; r.w[s][2] = x.z; r.w[s][3] = x.w;
            } else if constexpr (NCL == 8) {
                const w2u x = __builtin_nontemporal_load(reinterpret_cast<const w2u*>(src));
                r.w[s][0] = x.x; r.w[s][1] = x.y;
            } else if constexpr (NCL == 4) {
                r.w[s][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src));
            } else {
                r.w[s][0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(src));
            }
        }
    }
    __device__ __forceinline__ const uint8_t* val_row(const Place& e) const {
        return vbase + (uint64_t)(uint32_t)e.page * v_sb + (uint32_t)e.at * (kV8 ? 1u : 2u);
    }
    __device__ __forceinline__ w4u load_val(const uint8_t* row, int dt) const {
        return __builtin_nontemporal_load(reinterpret_cast<const w4u*>(row + dt * vstep));
    }
    __device__ __forceinline__ void load_vals(const Place& e, Vals& r) const {
        r.scale = load_scale(e);
        const uint8_t* row = val_row(e);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) r.v[dt] = load_val(row, dt);
    }
    __device__ __forceinline__ float load_scale(const Place& e) const {
        if constexpr (kV8) return v_scale[(uint64_t)(uint32_t)e.page * vs_sb];
        else return 1.f;
    }

    template <class T>
    __device__ __forceinline__ T gather(uint32_t code, int at) const {  // at: a constant below 65,536
        typedef const __attribute__((address_space(3))) T* Lds;
        return *(Lds)(uintptr_t)(code * (4 * BD) + book + at);
    }
    // the operand of score step st: product st / NK, this lane's dims 4 (st % NK) .. + 3, hi and lo (with codewords of 8
    // dims: hi or lo of 8 dims)
    __device__ __forceinline__ uint4 operand(const Codes& c, int st) const {
        const int s = st / NK, k = st % NK;
        auto code = [&](int j) { return __builtin_amdgcn_ubfe(c.w[s][j >> 2], 8 * (j & 3), 8); };
        if constexpr (BD == 8) {
            const w4u x = gather<w4u>(code(k >> 1), (k >> 1) * 8192 + 16 * (k & 1));
            return make_uint4(x.x, x.y, x.z, x.w);
        } else if constexpr (BD == 4) {
            const w4u x = gather<w4u>(code(k), k * 4096);
            return make_uint4(x.x, x.y, x.z, x.w);
        } else {
            const w2u x = gather<w2u>(code(2 * k), k * 4096), y = gather<w2u>(code(2 * k + 1), k * 4096 + 2048);
            return make_uint4(x.x, x.y, y.x, y.y);
        }
    }
    // A tile's scores.  Gathers run kAhead steps before their products; the barriers keep the compiler from gathering a whole
    // tile ahead, which does not fit the registers.
    __device__ __forceinline__ void scores(const Codes& c, w4f (&s)[NS]) const {
        uint4 ring[kAhead];
#pragma unroll
        for (int st = 0; st < kAhead; ++st) ring[st] = operand(c, st);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < NST; ++st) {
            const uint4 x = ring[st % kAhead];
            w4f& acc = s[st / NK];
#pragma unroll
            for (int h = 0; h < QP; ++h) acc = win_mfma(x, q[h][BD == 8 ? st % NK / 2 : st % NK], st % NK || h ? acc : w4f{});
            if (st + kAhead < NST) ring[st % kAhead] = operand(c, st + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // bits [0, n) of a chunk's tokens
    __device__ __forceinline__ static uint32_t below(int n) { return (1u << min(max(n, 0), CH)) - 1u; }
    // the chunk's tokens that some row at a position from `first` to `last` sees; with the two swapped, that all do
    __device__ __forceinline__ uint32_t sees(int first, int last, int tok) const {
        return below(last + 1 - tok) & (~below(max(max(first, 0) - window, -1) + 1 - tok) | below(sinks - tok));
    }
    // the value operand of 8 tokens from 8 jj of this lane's chunk, those in `gone` (a bit a token of the chunk) as 0
    __device__ __forceinline__ uint4 vals(const w4u& v, int jj) const {
        if constexpr (kV8) {
            const w2u a = win_e4m3(v[2 * jj]), b = win_e4m3(v[2 * jj + 1]);
            return make_uint4(a.x, a.y, b.x, b.y);
        } else {
            return make_uint4(v.x, v.y, v.z, v.w);
        }
    }
    // all bits of the values of the chunk's tokens whose bit is set
    __device__ __forceinline__ static w4u spread(uint32_t bits) {
        w4u r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = spread_word(bits, k);
        return r;
    }
    __device__ __forceinline__ static uint32_t spread_word(uint32_t bits, int k) {  // its word k
        if constexpr (kV8) {
            const uint32_t b = (bits >> (4 * k)) & 0xFu;
            return ((b * 0x00204081u) & 0x01010101u) * 0xFFu;  // a bit to a byte each
        } else {
            const uint32_t b = bits >> (2 * k);
            return (b & 1u ? 0xFFFFu : 0u) | (b & 2u ? 0xFFFF0000u : 0u);
        }
    }
    // the top bit of each value that is infinite or NaN
    __device__ __forceinline__ static uint32_t wild(uint32_t w) {
        if constexpr (kV8) return (w & 0x7F7F7F7Fu) + 0x01010101u;
        else return (w & 0x7FFF7FFFu) + (VT == SSQ_BF16 ? 0x00800080u : 0x04000400u);
    }
    // Infinite and NaN values (16 bits) that this column's row sees in tiles i0, i0 + step, .. below i1, put into its O: a dim is
    // infinite, or NaN, whatever the probabilities.  Whether a row sees one of a kind is a product of ones.
    __device__ __forceinline__ void put_wild(int i0, int i1, int step, w4f (&o)[DT]) const {
        constexpr uint32_t one = VT == SSQ_BF16 ? 0x3F80u : 0x3C00u, infinity = VT == SSQ_BF16 ? 0x7F80u : 0x7C00u;
        uint32_t nan = 0, inf = 0, neg = 0;  // a bit a (dt, e)
        for (int i = i0; i < i1; i += step) {
            const uint8_t* row = val_row(place(i, grp));
            const w4u on = spread(sees(pos, pos, TT * tile_of(i) + CH * grp)) & (one * 0x10001u);
            const uint4 seen = make_uint4(on.x, on.y, on.z, on.w);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const w4u v = load_val(row, dt);
                uint32_t kind[3][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t a = v[k] & 0xFFFFu, b = v[k] >> 16;
                    kind[0][k] = ((a & 0x7FFFu) > infinity ? one : 0u) | ((b & 0x7FFFu) > infinity ? one << 16 : 0u);
                    kind[1][k] = (a == infinity ? one : 0u) | (b == infinity ? one << 16 : 0u);
                    kind[2][k] = (a == (infinity | 0x8000u) ? one : 0u) | (b == (infinity | 0x8000u) ? one << 16 : 0u);
                }
                auto any = [&](const uint32_t (&x)[4]) {
                    const w4f z = win_mfma_v<VT>(make_uint4(x[0], x[1], x[2], x[3]), seen, w4f{});
                    uint32_t r = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) r |= (__float_as_uint(fminf(z[e], 1.f)) >> 29 & 1u) << e;  // a count: 0, or 1 and more
                    return r;
                };
                nan |= any(kind[0]) << (4 * dt);
                inf |= any(kind[1]) << (4 * dt);
                neg |= any(kind[2]) << (4 * dt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        nan |= inf & neg;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t x = __float_as_uint(o[dt][e]);
                auto put = [&](uint32_t bits, uint32_t y) {
                    const uint32_t on = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 4 * dt + e, 1);
                    x = (x & ~on) | (y & on);
                };
                put(inf, 0x7F800000u);
                put(neg, 0xFF800000u);
                put(nan, 0x7FC00000u);
                o[dt][e] = __uint_as_float(x);
            }
    }
};

template <int D, int BD, int VT, int QP, bool TEAM>
__global__ __launch_bounds__(kWinThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_window(const SsqWindowParams) {
    using W = WinRun<D, BD, VT, QP>;
    using L = typename W::L;
    constexpr int TT = W::TT, CH = W::CH, NS = W::NS, DT = W::DT, NE = W::NE;
    constexpr int kStep = TEAM ? kWinWaves : 1;  // from a wave's tile to its next
    extern __shared__ __align__(16) unsigned char smem[];
    WinArgs p = win_args();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = blockIdx.x % p->a.num_kv_heads, wg = blockIdx.x / p->a.num_kv_heads;
    float* red = reinterpret_cast<float*>(smem + L::kRed);
    uint16_t* perm = reinterpret_cast<uint16_t*>(smem + L::kPerm);
    float* mls = reinterpret_cast<float*>(smem + L::kMl);

    // ---- the codebook, behind the permutation
    // (No branches around these loads or the first tiles': they return in order, and a wait behind a branch is for all of them.)
    const int64_t at_perm = p->a.perm[(int64_t)kv * p->a.perm_sh + min(tid, D - 1)];
    const int first_len = TEAM ? 0 : WinCut<TT, kWinRows>::length(p, lane);
    WinBook<D, BD> book;
    book.load(p, kv, tid);
    if (tid < D) perm[tid] = (uint16_t)((uint64_t)at_perm < (uint64_t)D ? at_perm : D - 1);

    W u;
    u.lane = lane; u.col = lane & 15; u.grp = lane >> 4;
    u.window = p->window; u.sinks = p->sinks; u.n_pages = p->n_pages; u.psh = p->psh;
    u.c_sb = (uint32_t)p->a.c_sb; u.c_st = (uint32_t)p->a.c_st; u.v_sb = (uint32_t)p->a.v_sb * (W::kV8 ? 1 : 2); u.vs_sb = (uint32_t)p->vs_sb;
    u.v_scale = p->v_scale + (int64_t)kv * p->vs_sh;
    const int q_len = p->a.q_len;
    u.book = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)smem + u.grp * (W::NCL * 1024 * BD);
    asm("" : "+v"(u.book));  // opaque, or every block's address takes a register instead of the gather's offset field
    u.cbase = p->a.codes + (int64_t)kv * p->a.c_sh + (int64_t)(u.col & 3) * u.c_st + u.grp * W::NCL;
    u.vbase = reinterpret_cast<const uint8_t*>(p->a.v) + ((int64_t)kv * p->a.v_sh + (int64_t)u.col * p->a.v_st) * (W::kV8 ? 1 : 2);
    u.vstep = 16 * (uint32_t)p->a.v_st * (W::kV8 ? 1 : 2);

    // ---- what is to be done: an item's tiles [i0, i1), and where they go (slot -1: the output)
    WinCut<TT, kWinRows> cut;
    const int worker = TEAM ? wg : wave * p->n_wg + wg;
    int x = 0, x_begin = 0, x_end = 0, ahead = worker;  // the next item, and its cost position
    if constexpr (!TEAM) {
        cut.init(p, lane, first_len);
        x = x_begin = (int)min((int64_t)worker * cut.share, (int64_t)cut.total);
        x_end = (int)min((int64_t)(worker + 1) * cut.share, (int64_t)cut.total);
        if (x_begin < x_end) cut.find(p, lane, x_begin, ahead, x);
    }
    int b = 0, row0 = 0, nr = 0, len = 0, i0 = 0, i1 = 0, slot = -1;
    auto next = [&]() {
        p = win_args();
        for (;;) {
            const int item = __builtin_amdgcn_readfirstlane(ahead), start = x;
            if ((!TEAM && x >= x_end) || item >= p->items) return false;
            ahead = item + (TEAM ? p->n_wg : 1);
            b = item / p->rgroups;
            row0 = (item - b * p->rgroups) * kWinRows;
            len = max(0, min(p->a.seq_lens[b], p->a.seq_len));
            nr = min(kWinRows, p->rows - row0);
            u.t = win_tiles<TT, kWinRows>(WinShape{u.window, u.sinks, q_len, p->G, p->rows}, len, row0);
            slot = -1;
            i0 = TEAM ? wave : 0;
            i1 = u.t.n;
            if constexpr (!TEAM) {
                const int cost = p->fixed + u.t.n;
                x = start + cost;
                i0 = max(0, x_begin - start - p->fixed);
                i1 = max(0, min(u.t.n, x_end - start - p->fixed));
                if (u.t.n == 0 ? start < x_begin : i1 <= i0) continue;  // its part here is of the fixed cost
                const bool mine = i0 == 0 && i1 == u.t.n;
                if (!mine) slot = start < x_begin ? 0 : 1;
                if (i0 == 0 && kv == 0 && lane == 0) {  // pieces, for the merge
                    p->meta[2 * item] = 2 * worker + (slot > 0 ? 1 : 0);
                    p->meta[2 * item + 1] = mine ? 1 : (start + cost - 1) / cut.share - worker + 1;
                }
            }
            return true;
        }
    };
    // ---- its first loads: the tiles', then the query rows'
    // the places of the next tile's values and of the codes after the next tile's; the codes of this and the next tile
    typename W::Place pv{}, pc{};
    typename W::Codes c0, c1;
    typename W::Vals val;
    // Query rows come in 16-byte pieces, 1 KiB a wave at once, kPieces times: 16 rows of 16 bits, or 8 of 32 (those behind are
    // loaded when their turn comes).
    constexpr int kPieces = D / 32;
    uint4 qraw[kPieces];
    int last_i = 0;
    // piece k of a batch from row r0 on: its row and byte in it
    auto q_at = [&](int k, int r0, int& r, int& byte) {
        constexpr int row_bytes = QP == 2 ? 4 * D : 2 * D;
        const int o = (k * SSQ_WAVE + lane) * 16;
        r = r0 + o / row_bytes;
        byte = o % row_bytes;
    };
    auto q_load = [&](int k, int r0) {
        int r, byte;
        q_at(k, r0, r, byte);
        const int row = row0 + max(0, min(r, nr - 1)), qi = row / p->G, h = kv * p->G + row - qi * p->G;
        constexpr int size = QP == 2 ? 4 : 2;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(p->a.q) + ((int64_t)b * p->a.q_sb + (int64_t)h * p->a.q_sh + (int64_t)qi * p->a.q_sl) * size + byte;
        if (p->q_vec) return *reinterpret_cast<const uint4*>(src);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = size == 4 ? reinterpret_cast<const uint32_t*>(src)[e]
                             : (uint32_t)reinterpret_cast<const uint16_t*>(src)[2 * e] | (uint32_t)reinterpret_cast<const uint16_t*>(src)[2 * e + 1] << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto load = [&]() {
        u.table = p->a.block_table + (int64_t)b * p->a.bt_sb;
        u.last_tok = max(u.t.p_hi, 0);
        u.pos = len - q_len + min(row0 + u.col, p->rows - 1) / p->G;
        // (a wave without tiles loads the last one's)
        const int i = max(0, min(i0, i1 - 1));
        last_i = i0 < i1 ? i1 - 1 - (i1 - 1 - i0) % kStep : i;
        const int in = min(i + kStep, last_i);
        pc = u.place(i, u.code_chunk());
        pv = u.place(i, u.grp);
        const typename W::Place pcn = u.place(in, u.code_chunk()), pvn = u.place(in, u.grp);
        const typename W::Place pc2 = u.place(min(i + 2 * kStep, last_i), u.code_chunk());
#pragma unroll
        for (int k = 0; k < kPieces; ++k) qraw[k] = q_load(k, 0);
        u.load_codes(pc, c0);
        u.load_codes(pcn, c1);
        u.load_vals(pv, val);
        pc = pc2;
        pv = pvn;
    };
    int book_exp;  // the codebook is staged times 2^book_exp
    // ---- the query rows as operands: f16, at a power of two of each row's
    auto query_of = [&](auto type) {
        constexpr int dtype = decltype(type)::value, wide = dtype == SSQ_F32 ? 1 : 0;
        const bool in = u.col < nr;
        const float scale = p->a.has_scale ? p->a.scale : 1.f;  // (a factor of 1 is exact)
        // through the wave's LDS rows, 8 (4) at a time, permuted on the way back
        unsigned char* rows = smem + L::kBook + wave * 8 * L::kQRow;
        const int row_bytes = L::kQRow << wide, per = 8 >> wide;
        uint32_t idx[NE / 2];
#pragma unroll
        for (int k = 0; k < NE / 8; ++k) {
            const uint4 w = reinterpret_cast<const uint4*>(perm + u.grp * NE)[k];
            idx[4 * k] = w.x; idx[4 * k + 1] = w.y; idx[4 * k + 2] = w.z; idx[4 * k + 3] = w.w;
        }
        float y[NE];
#pragma unroll
        for (int k = 0; k < NE; ++k) y[k] = 0.f;
        for (int r0 = 0; r0 < nr; r0 += per) {
            if (wide && r0 == 8)  // the second batch of 32-bit rows
#pragma unroll
                for (int k = 0; k < kPieces; ++k) qraw[k] = q_load(k, 8);
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                int r, byte;
                q_at(k, wide ? r0 & 8 : 0, r, byte);
                if (r >= r0 && r < r0 + per) *reinterpret_cast<uint4*>(rows + (r - r0) * row_bytes + byte) = qraw[k];
            }
            win_lds_sync();
            if (u.col >= r0 && u.col < r0 + per) {
                const unsigned char* mine = rows + (u.col - r0) * row_bytes;
#pragma unroll
                for (int k = 0; k < NE; ++k) {
                    const uint32_t j = k & 1 ? idx[k / 2] >> 16 : idx[k / 2] & 0xFFFFu;
                    y[k] = ssq_bits_to_f32(wide ? reinterpret_cast<const uint32_t*>(mine)[j] : reinterpret_cast<const uint16_t*>(mine)[j], dtype);
                }
            }
            win_lds_sync();
        }
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < NE; ++k) {
            y[k] = in ? ssq_round_to(y[k] * scale, dtype) : 0.f;
            const float z = fabsf(y[k]);
            most = fmaxf(most, z < INFINITY ? z : 0.f);
        }
        const int up = min(15 - win_exp(win_max4(most)), 126);
        const float s = ldexpf(1.f, up);
        u.fac = ldexpf(kWinLog2e, max(-book_exp - up, -126));  // above 0
        uint32_t hi[NE / 2], lo[NE / 2];
#pragma unroll
        for (int k = 0; k < NE; k += 2) win_split<true>(y[k] * s, y[k + 1] * s, hi[k / 2], lo[k / 2]);
#pragma unroll
        for (int h = 0; h < QP; ++h) {
            const uint32_t* w = h ? lo : hi;
#pragma unroll
            for (int k = 0; k < W::NQ; ++k) {
                if constexpr (BD == 8) u.q[h][k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                else if constexpr (BD == 4) u.q[h][k] = make_uint4(w[2 * k], w[2 * k + 1], w[2 * k], w[2 * k + 1]);
                else u.q[h][k] = make_uint4(w[2 * k], w[2 * k], w[2 * k + 1], w[2 * k + 1]);
            }
        }
    };
    auto query = [&]() {
        if constexpr (QP == 2) query_of(std::integral_constant<int, SSQ_F32>{});
        else if (p->a.q_dtype == SSQ_BF16) query_of(std::integral_constant<int, SSQ_BF16>{});
        else query_of(std::integral_constant<int, SSQ_F16>{});
    };

    __syncthreads();  // the permutation
    bool more = next();
    load();
    book_exp = book.stage(smem, red, tid, lane, wave);
    while (more) {
        query();

        // ---- this wave's tiles.  Loads return in order: a place is asked for a tile before it is used, and before that
        // tile's values.
        float m = kWinNone, l = 0.f, unit = W::kV8 ? kWinScale : 1.f, inv_unit = 1.f / unit;
        w4f o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = w4f{};
        for (int i = i0; i < i1; i += kStep) {
            w4f s[NS];
            u.scores(c0, s);
            c0 = c1;
            u.load_codes(pc, c1);
            pc = u.place(min(i + 3 * kStep, last_i), u.code_chunk());
            const int t0 = TT * u.tile_of(i), tok = t0 + CH * u.grp;
            // tokens of the tile that some row does not see (uniform)
            const bool edge = (t0 + TT - 1 > u.t.p_lo) | ((t0 <= u.t.p_hi - u.window) & (t0 + TT > u.sinks));
            bool apart = false;  // an infinite or NaN value that some rows see and others do not
            if (edge) {
                const uint32_t any = u.sees(u.t.p_lo, u.t.p_hi, tok), all = u.sees(u.t.p_hi, u.t.p_lo, tok);
                const uint32_t mine = u.sees(u.pos, u.pos, tok);
#pragma unroll
                for (int e = 0; e < CH; ++e) s[e >> 2][e & 3] = mine >> e & 1u ? s[e >> 2][e & 3] : -INFINITY;
                if (mine == 0) val.scale = 0.f;  // not this row's page, or none of this tile's
                const w4u off = W::spread(~any);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) val.v[dt] &= ~off;
                if (q_len > 1) {
                    const w4u part = W::spread(~all) & (W::kV8 ? 0x80808080u : 0x80008000u);
                    uint32_t found = 0;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) found |= W::wild(val.v[dt][k]) & part[k];
                    apart = __builtin_amdgcn_ballot_w64(found != 0) != 0;
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int e = 1; e < CH; ++e) top = fmaxf(top, s[e >> 2][e & 3]);
            top *= u.fac;
            if (__builtin_amdgcn_ballot_w64(win_over<VT>(top, m, l)) != 0) {
                float mn = fmaxf(m, win_max4(top) - kWinTop<VT>);
                if (VT == SSQ_BF16 && win_max4(l) > kWinMass) mn = fmaxf(mn, m + 4.f);
                const float f = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
            }
            float by = 1.f;    // this group's page scale, in units of O
            bool far = false;  // a page's is too far below them
            if constexpr (W::kV8) {
                // (positive floats compare as their bits; rows have units of their own where they do not see the same pages)
                const uint32_t bits = __float_as_uint(val.scale);
                if (__builtin_amdgcn_ballot_w64(bits > __float_as_uint(unit)) != 0) {
                    const float big = fmaxf(unit, win_max4(val.scale));
                    const float f = unit / big;
                    unit = big;
                    inv_unit = 1.f / unit;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
                }
                by = val.scale * inv_unit;
                far = __builtin_amdgcn_ballot_w64((by < kWinFar) & (val.scale > 0.f)) != 0;
            }
#pragma unroll
            for (int e = 0; e < CH; e += 2) {
                const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], u.fac, -m));
                const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][(e & 3) + 1], u.fac, -m));
                l += x0 + x1;
                s[e >> 2][e & 3] = W::kV8 ? x0 * by : x0;
                s[e >> 2][(e & 3) + 1] = W::kV8 ? x1 * by : x1;
            }
            if constexpr (W::kV8) {
                if (far) {  // in 32 bits; rows of one position at a time if `apart`, as below, else all
                    for (int at = apart ? u.t.p_lo : u.t.p_hi; at <= u.t.p_hi; ++at) {
                        const uint32_t on = apart ? u.sees(at, at, tok) : ~0u;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            w4f z = o[dt];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const w4f y = win_e4m3_32(val.v[dt][k] & W::spread_word(on, k));
#pragma unroll
                                for (int e = 0; e < 4; ++e) z = win_mfma_32(y[e], s[k][e], z);
                                __builtin_amdgcn_sched_barrier(0);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[dt][e] = !apart || u.pos == at ? z[e] : o[dt][e];
                        }
                    }
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) val.v[dt] = w4u{};
                    apart = false;
                }
            }
            uint32_t pw[CH / 2];
#pragma unroll
            for (int e = 0; e < CH; e += 2) pw[e / 2] = win_pack_p<VT>(s[e >> 2][e & 3], s[e >> 2][(e & 3) + 1]);
            if (apart) {
                // The rows of one position at a time, the values that they do not see as 0; the products below then add nothing.
                for (int at = u.t.p_lo; at <= u.t.p_hi; ++at) {
                    const w4u on = W::spread(u.sees(at, at, tok));
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        w4f z = o[dt];
#pragma unroll
                        for (int jj = 0; jj < CH / 8; ++jj)
                            z = win_mfma_v<VT>(u.vals(val.v[dt] & on, jj), make_uint4(pw[4 * jj], pw[4 * jj + 1], pw[4 * jj + 2], pw[4 * jj + 3]), z);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[dt][e] = u.pos == at ? z[e] : o[dt][e];
                    }
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) val.v[dt] = w4u{};
            }
            const uint8_t* next_row = u.val_row(pv);
            val.scale = u.load_scale(pv);
            pv = u.place(min(i + 2 * kStep, last_i), u.grp);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {  // a value operand's successor loads once it is used
#pragma unroll
                for (int jj = 0; jj < CH / 8; ++jj)
                    o[dt] = win_mfma_v<VT>(u.vals(val.v[dt], jj), make_uint4(pw[4 * jj], pw[4 * jj + 1], pw[4 * jj + 2], pw[4 * jj + 3]), o[dt]);
                val.v[dt] = u.load_val(next_row, dt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        l = win_sum4(l);
        if constexpr (!W::kV8) {
            // A probability that 16 bits hold as 0, or a rescale by one that 32 do, makes NaN of an infinity: what is not finite is looked at
            // again (scores of NaN leave l NaN).
            float odd = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(o[dt][e], 0.f, odd);
            if (__builtin_amdgcn_ballot_w64(odd != 0.f) != 0) u.put_wild(i0, i1, kStep, o);
        }
        // What the row's values average to here: everything that is joined or stored is a finite average of finite values, whatever
        // their size (O in its units times the unit need not be).
        const float inv = 1.f / l;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = l == 0.f ? w4f{} : W::kV8 ? o[dt] * inv * unit : o[dt] * inv;

        p = win_args();
        if constexpr (TEAM) {
            // ---- the waves' join, 4 rows at a time
            if (lane < kWinRows) {
                mls[wave * kWinRows + lane] = m;
                mls[(kWinWaves + wave) * kWinRows + lane] = l;
            }
            __syncthreads();
            float* join = reinterpret_cast<float*>(smem + L::kBook);
            constexpr int kRow = L::kJoinRow;
#pragma unroll 1
            for (int r0 = 0; r0 < nr; r0 += L::kJoinRows) {
                if ((u.col & ~3) == r0) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const w4f z = o[dt];
                        *reinterpret_cast<float4*>(join + (wave * 4 + (u.col & 3)) * kRow + 16 * dt + 4 * u.grp) = make_float4(z[0], z[1], z[2], z[3]);
                    }
                }
                __syncthreads();
                const int r = r0 + tid / D, dv = tid % D;
                if (tid < 4 * D && r < nr) {
                    float mr = kWinNone, lt = 0.f, ot = 0.f, lw[kWinWaves];
#pragma unroll
                    for (int w = 0; w < kWinWaves; ++w) mr = fmaxf(mr, mls[w * kWinRows + r]);
#pragma unroll
                    for (int w = 0; w < kWinWaves; ++w) {
                        lw[w] = mls[(kWinWaves + w) * kWinRows + r] * __builtin_amdgcn_exp2f(mls[w * kWinRows + r] - mr);
                        lt += lw[w];
                    }
                    const float part = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
                    for (int w = 0; w < kWinWaves; ++w) ot += win_part(join[(w * 4 + r - r0) * kRow + dv], lw[w] * part);
                    const int row = row0 + r, qi = row / p->G, h = kv * p->G + row - qi * p->G;
                    ssq_store_elem(p->a.out, p->out_dtype, (int64_t)b * p->a.o_sb + (int64_t)h * p->a.o_sh + (int64_t)qi * p->a.o_sl + dv,
                                   ot);
                    if (p->a.lse && dv == 0)
                        p->a.lse[((int64_t)b * p->a.num_q_heads + h) * p->a.q_len + qi] = lt == 0.f ? -INFINITY : (mr + log2f(lt)) * kWinLn2;
                }
                __syncthreads();
            }
        } else if (u.col < nr) {
            if (slot < 0) {
                const int row = row0 + u.col, qi = row / p->G, h = kv * p->G + row - qi * p->G;
                const int64_t at = (int64_t)b * p->a.o_sb + (int64_t)h * p->a.o_sh + (int64_t)qi * p->a.o_sl + 4 * u.grp;
                const int dtype = p->out_dtype;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const w4f z = o[dt];
                    if (p->out_vec) win_store4(p->a.out, dtype, at + 16 * dt, z);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e) ssq_store_elem(p->a.out, dtype, at + 16 * dt + e, z[e]);
                }
                if (p->a.lse && u.grp == 0)
                    p->a.lse[((int64_t)b * p->a.num_q_heads + h) * p->a.q_len + qi] = l == 0.f ? -INFINITY : (m + log2f(l)) * kWinLn2;
            } else {
                float* dst = p->part + ((int64_t)(kv * p->workers + worker) * 2 + slot) * (kWinRows * (D + 2));
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const w4f z = o[dt];
                    *reinterpret_cast<float4*>(dst + u.col * D + 16 * dt + 4 * u.grp) = make_float4(z[0], z[1], z[2], z[3]);
                }
                if (u.grp == 0) {
                    dst[kWinRows * D + u.col] = m;
                    dst[kWinRows * D + kWinRows + u.col] = l;
                }
            }
        }
        more = next();
        if (more) load();
    }
}

// n of N pieces (m, l, average) joined to (M, L, average o): averages weighted by their share of the sum, which no size of values
// takes past them.
template <int N, int E, class T>
__device__ __forceinline__ void win_join(float& M, float& L, T (&o)[E], const float (&m)[N], const float (&l)[N], const T (&op)[N][E], int n) {
    float mt = M, w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) mt = j < n ? fmaxf(mt, m[j]) : mt;
    const float w0 = L * __builtin_amdgcn_exp2f(M - mt);
    float sum = w0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = j < n ? l[j] * __builtin_amdgcn_exp2f(m[j] - mt) : 0.f;
        sum += w[j];
    }
    M = mt;
    L = sum;
    const float part = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = win_part(o[e], w0 * part);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (j >= n) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += win_part(op[j][e], w[j] * part);
    }
}

}  // namespace

#include "ssq_window_wide.h"

namespace {

// Joins the pieces of the items that waves shared: a query row by one wave of four, or by all W waves of a workgroup where pieces
// may be many; lanes over the value dims, 8 pieces in flight a wave.
template <int D, int W>
__global__ __launch_bounds__((W > 1 ? W : 4) * SSQ_WAVE) void k_window_merge(const SsqWindowParams p) {
    constexpr bool WIDE = W > 1;
    constexpr int E = D / SSQ_WAVE, kAhead = 8;
    __shared__ float mo[W][D], ml[W][2];
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t id = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;  // (sequence, KV head, row)
    const int64_t bk = id / p.rows;
    const int row = (int)(id - bk * p.rows), b = (int)(bk / a.num_kv_heads), kv = (int)(bk - (int64_t)b * a.num_kv_heads);
    if (b >= a.batch) return;
    const int item = b * p.rgroups + row / kWinRows, r = row % kWinRows;
    constexpr int n = kWinRows, slot = n * (D + 2);
    const int first = p.meta[2 * item], pieces = p.meta[2 * item + 1];
    if (pieces <= 1) return;
    const float* base = p.part + (int64_t)kv * p.workers * 2 * slot;
    auto at = [&](int i) { return base + (int64_t)(i ? 2 * ((first >> 1) + i) : first) * slot; };
    float M = kWinNone, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int i0 = WIDE ? wave * kAhead : 0; i0 < pieces; i0 += W * kAhead) {
        float m[kAhead], lp[kAhead], op[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            m[j] = kWinNone;
            if (i0 + j >= pieces) continue;
            const float* src = at(i0 + j);
            m[j] = src[n * D + r];
            lp[j] = src[n * D + n + r];
#pragma unroll
            for (int e = 0; e < E; ++e) op[j][e] = src[r * D + lane * E + e];
        }
        win_join<kAhead, E>(M, l, o, m, lp, op, pieces - i0);
    }
    if constexpr (WIDE) {
        if (lane == 0) {
            ml[wave][0] = M;
            ml[wave][1] = l;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) mo[wave][lane * E + e] = o[e];
        __syncthreads();
        if (wave) return;
        float m[W], lp[W], op[W][E];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            m[w] = ml[w][0];
            lp[w] = ml[w][1];
#pragma unroll
            for (int e = 0; e < E; ++e) op[w][e] = mo[w][lane * E + e];
        }
        M = kWinNone;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        win_join<W, E>(M, l, o, m, lp, op, (pieces + kAhead - 1) / kAhead);  // (the waves behind had none)
    }
    const int qi = row / p.G, h = kv * p.G + row - qi * p.G;
#pragma unroll
    for (int e = 0; e < E; ++e)
        ssq_store_elem(a.out, p.out_dtype, (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)qi * a.o_sl + lane * E + e,
                       o[e]);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.num_q_heads + h) * a.q_len + qi] = l == 0.f ? -INFINITY : (M + log2f(l)) * kWinLn2;
}

// An item of few may have as many pieces as there are workers; of many, each has few.  (One of 131,071 tokens: 16 waves a row 5.9
// us; when pieces were read eight at a time, some twice, 9.4, and 4 waves 20; 64 of 66 tiles: one 4, four 5.)
template <int D>
int win_merge(const SsqWindowParams& p, hipStream_t st) {
    if (p.form == kWinWide) {
        hipLaunchKernelGGL(k_window_wide_merge<D>, dim3((unsigned)(p.items * p.a.num_kv_heads * kWinWaves)), dim3(D / 32 * SSQ_WAVE), 0, st, p);
        return ssq_check_hip(hipGetLastError(), "k_window_wide_merge launch");
    }
    const int64_t rows = (int64_t)p.a.batch * p.a.num_kv_heads * p.rows;
    const int pieces = p.workers / p.items;
    if (pieces >= 32) hipLaunchKernelGGL((k_window_merge<D, 16>), dim3((unsigned)rows), dim3(1024), 0, st, p);
    else if (pieces > 8) hipLaunchKernelGGL((k_window_merge<D, 4>), dim3((unsigned)rows), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_window_merge<D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
    return ssq_check_hip(hipGetLastError(), "k_window_merge launch");
}
template <int D, int BD, int VT, int QP>
int win_launch(const SsqWindowParams& p, hipStream_t st) {
    static_assert(WinLds<D>::kTotal <= 160 * 1024 && WideLds<D>::kTotal <= 160 * 1024, "a workgroup's LDS");
    auto kern = p.form == kWinTeam ? k_window<D, BD, VT, QP, true> : p.form == kWinShares ? k_window<D, BD, VT, QP, false> : k_window_wide<D, BD, VT, QP>;
    const int lds = p.form == kWinWide ? WideLds<D>::kTotal : WinLds<D>::kTotal;
    int rc = ssq_allow_lds((const void*)kern, lds, "hipFuncSetAttribute(k_window)");
    if (rc) return rc;
    hipLaunchKernelGGL(kern, dim3(p.n_wg * p.a.num_kv_heads), dim3(kWinThreads), lds, st, p);
    rc = ssq_check_hip(hipGetLastError(), "k_window launch");
    return rc || p.form == kWinTeam ? rc : win_merge<D>(p, st);
}
template <int D, int BD, int VT>
int win_form(const SsqWindowParams& p, hipStream_t st) {
    return p.a.q_dtype == SSQ_F32 ? win_launch<D, BD, VT, 2>(p, st) : win_launch<D, BD, VT, 1>(p, st);
}
template <int D, int VT>
int win_blocks(const SsqWindowParams& p, hipStream_t st) {
    switch (p.a.block_dim) {
        case 2: return win_form<D, 2, VT>(p, st);
        case 4: return win_form<D, 4, VT>(p, st);
        default: return win_form<D, 8, VT>(p, st);
    }
}

}  // namespace
