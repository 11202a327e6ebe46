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
// the largest (8-bit and f16 values; with bf16 values they are rounded to bf16, as in the other decode kernels).  A page's scale
// joins them before the rounding, relative to the largest scale met, which O is kept in units of.
#pragma once

#include "ssq_common.h"

struct SsqWindowParams {
    ssq_decode_args a;
    int window, sinks;       // window: INT_MAX where everything is seen
    int out_dtype;
    int n_pages;
    const float* v_scale;
    int64_t vs_sb, vs_sh;
    int G, rows, rgroups;    // query rows of a (sequence, KV head): (qi, g), g fastest; groups of 16 NR rows
    int items;               // batch * rgroups
    int n_wg;                // workgroups per KV head
    int whole;               // a workgroup takes whole items; else equal shares of all their tiles (WinCut)
    int fixed, least;        // an item's cost beside its tiles, and the smallest share, both in tiles
    int psh;                 // log2(page_size / 16)
    float* part;             // [Hkv][n_wg][2] slots of 16 NR rows x (Dv + 2): o, then m (log2 units), l
    int* meta;               // [items][2]: first workgroup * 2 + its slot, and pieces
};

#define SSQ_WINDOW_UNIT(name) int name(const SsqWindowParams& p, int nr, hipStream_t st)
SSQ_WINDOW_UNIT(ssq_window_64_e4m3);
SSQ_WINDOW_UNIT(ssq_window_64_bf16);
SSQ_WINDOW_UNIT(ssq_window_64_f16);
SSQ_WINDOW_UNIT(ssq_window_128_e4m3);
SSQ_WINDOW_UNIT(ssq_window_128_bf16);
SSQ_WINDOW_UNIT(ssq_window_128_f16);

// waves of a workgroup: two a SIMD, so that one's matrix products run beside the other's vector work; with 32 query rows
// the registers hold one
__host__ __device__ constexpr int win_waves(int nr) { return nr == 1 ? 8 : 4; }

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
template <int TT>
__host__ __device__ __forceinline__ WinTiles win_tiles(const WinShape& p, int len, int row0, int rows_per) {
    WinTiles t;
    const int last = (row0 + rows_per < p.rows ? row0 + rows_per : p.rows) - 1;
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
constexpr float kWinTop = 14.f, kWinOver = 15.5f;  // log2 of the largest probability when m moves, and of what moves it
constexpr float kWinScale = 7.888609052210118e-31f;  // 2^-100, the smallest unit of O

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
// x rounded to f16, and the rounding of what that left (0 beside an infinity or NaN)
__device__ __forceinline__ void win_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = win_pack_h(x, y);
    const float u = x - win_h(hi, 0), v = y - win_h(hi, 1);
    lo = win_pack_h(__builtin_isfinite(u) ? u : 0.f, __builtin_isfinite(v) ? v : 0.f);
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

// Equal shares of the items' tiles: the items of a KV head lie end to end on a cost axis, fixed + tiles each, and
// workgroup w takes [w share, (w + 1) share).  An item inside one share is written out by its workgroup; one that spans
// several leaves a partial in each: slot 0 of a workgroup for the item its share starts in, slot 1 for one that starts in
// it.  Everything follows from the lengths, which the host does not see.
template <int TT, int RP>
struct WinCut {
    int share, total;
    __device__ __forceinline__ static int cost(WinArgs p, int i) {
        if (i >= p->items) return 0;
        const int b = i / p->rgroups, g = i - b * p->rgroups;
        const WinShape s{p->window, p->sinks, p->a.q_len, p->G, p->rows};
        return p->fixed + win_tiles<TT>(s, max(0, min(p->a.seq_lens[b], p->a.seq_len)), g * RP, RP).n;
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
    // (the whole wave calls these two)
    __device__ __forceinline__ void init(WinArgs p, int lane) {
        total = 0;
        for (int i = 0; i < p->items; i += SSQ_WAVE) total += __builtin_amdgcn_readlane(scan(cost(p, i + lane)), 63);
        share = (max((total + p->n_wg - 1) / p->n_wg, p->least) + 7) & ~7;
    }
    // the item that holds cost position x < total, its start and cost
    __device__ __forceinline__ void find(WinArgs p, int lane, int x, int& item, int& s, int& c) const {
        int base = 0;
        for (int f = 0; f < p->items; f += SSQ_WAVE) {
            const int mine = cost(p, f + lane), v = scan(mine);
            const uint64_t hit = __builtin_amdgcn_ballot_w64(base + v > x);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                item = f + l;
                c = __builtin_amdgcn_readlane(mine, l);
                s = base + __builtin_amdgcn_readlane(v, l) - c;
                return;
            }
            base += __builtin_amdgcn_readlane(v, 63);
        }
        item = p->items;
        s = x;
        c = 0;
    }
};

// LDS: codebook | scratch: query parts, then the waves' join | m, l [waves][RP] | rows' factors [RP] | reduction [waves] | permutation [D]
template <int D, int NR, int QP>
struct WinLds {
    static constexpr int RP = 16 * NR, kWaves = win_waves(NR);
    static constexpr int kBook = D * 256 * 4;
    static constexpr int kJoinRows = 4;
    static constexpr int kJoinRow = D + 4;  // floats
    static constexpr int kQRow = D + 8;      // f16 elements
    static constexpr int kQ = RP * kQRow * 2 * QP;
    static constexpr int kJoin = kWaves * kJoinRows * kJoinRow * 4;
    static constexpr int kScratch = kQ > kJoin ? kQ : kJoin;
    static constexpr int kMl = kBook + kScratch;
    static constexpr int kFac = kMl + 2 * kWaves * RP * 4;
    static constexpr int kRed = kFac + RP * 4;
    static constexpr int kPerm = kRed + kWaves * 4;
    static constexpr int kTotal = kPerm + 2 * D;
};

// D: head_dim and value_dim, BD: block_dim, VT: value dtype, NR: columns of 16 query rows, QP: query parts
template <int D, int BD, int VT, int NR, int QP>
struct WinRun {
    static constexpr bool kV8 = VT == SSQ_E4M3;
    static constexpr int CH = kV8 ? 16 : 8;        // tokens of a lane group
    static constexpr int TT = 4 * CH;              // tokens of a tile
    static constexpr int NS = CH / 4;              // score products (16 tokens each)
    static constexpr int NB = D / BD;
    static constexpr int NCL = NB / 4;             // codes of a token that a lane gathers
    static constexpr int NW = (NCL + 3) / 4;       // in words
    static constexpr int DT = D / 16;
    static constexpr int RP = 16 * NR;
    static constexpr int NK = D / 16;              // score MFMAs of 16 tokens (a lane's four dims, hi and lo, each)
    static constexpr int NQ = BD == 8 ? NK / 2 : NK;  // query operands
    using L = WinLds<D, NR, QP>;

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
    uint4 q[QP][NR][NQ];
    float fac[NR];                  // scores to log2 units
    // the item
    int pos[NR];                    // this column's positions
    WinTiles t;
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
    __device__ __forceinline__ void scores(const Codes& c, w4f (&s)[NS][NR]) const {
        uint4 ring[kAhead];
#pragma unroll
        for (int st = 0; st < kAhead; ++st) ring[st] = operand(c, st);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < NST; ++st) {
            const uint4 x = ring[st % kAhead];
#pragma unroll
            for (int h = 0; h < QP; ++h)
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    w4f& acc = s[st / NK][n];
                    acc = win_mfma(x, q[h][n][BD == 8 ? st % NK / 2 : st % NK], st % NK || h ? acc : w4f{});
                }
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
        for (int k = 0; k < 4; ++k) {
            if constexpr (kV8) {
                const uint32_t b = (bits >> (4 * k)) & 0xFu;
                r[k] = ((b * 0x00204081u) & 0x01010101u) * 0xFFu;  // a bit to a byte each
            } else {
                const uint32_t b = bits >> (2 * k);
                r[k] = (b & 1u ? 0xFFFFu : 0u) | (b & 2u ? 0xFFFF0000u : 0u);
            }
        }
        return r;
    }
    // the top bit of each value that is infinite or NaN
    __device__ __forceinline__ static uint32_t wild(uint32_t w) {
        if constexpr (kV8) return (w & 0x7F7F7F7Fu) + 0x01010101u;
        else return (w & 0x7FFF7FFFu) + (VT == SSQ_BF16 ? 0x00800080u : 0x04000400u);
    }
};

template <int D, int BD, int VT, int NR, int QP>
__global__ __launch_bounds__(win_waves(NR) * SSQ_WAVE) __attribute__((amdgpu_waves_per_eu(NR == 1 ? 2 : 1, NR == 1 ? 2 : 1))) void k_window(const SsqWindowParams) {
    using W = WinRun<D, BD, VT, NR, QP>;
    using L = typename W::L;
    constexpr int RP = W::RP, TT = W::TT, CH = W::CH, NS = W::NS, DT = W::DT;
    constexpr int kWinWaves = win_waves(NR), kWinThreads = kWinWaves * SSQ_WAVE;
    extern __shared__ __align__(16) unsigned char smem[];
    WinArgs p = win_args();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = blockIdx.x % p->a.num_kv_heads, wg = blockIdx.x / p->a.num_kv_heads;
    float* red = reinterpret_cast<float*>(smem + L::kRed);
    uint16_t* perm = reinterpret_cast<uint16_t*>(smem + L::kPerm);
    float* mls = reinterpret_cast<float*>(smem + L::kMl);
    float* facs = reinterpret_cast<float*>(smem + L::kFac);

    // ---- the codebook, 64 (32) floats a thread, all asked for at once
    constexpr int kPer = W::NB * 256 / kWinThreads;
    int book_exp;  // the codebook is staged times 2^book_exp
    {
        const float* cent = p->a.cent + (int64_t)kv * p->a.cent_sh;
        const int n_centroids = p->a.n_centroids;
        float c[kPer][BD];
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int e = tid + k * kWinThreads, blk = e >> 8, w = e & 255;
            const float* src = cent + (int64_t)(blk * n_centroids + min(w, n_centroids - 1)) * BD;
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
        }
        if (tid < D) {
            const uint64_t j = (uint64_t)p->a.perm[(int64_t)kv * p->a.perm_sh + tid];
            perm[tid] = (uint16_t)(j < (uint64_t)D ? j : D - 1);
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k)
#pragma unroll
            for (int d = 0; d < BD; ++d) {
                const float x = fabsf(c[k][d]);
                most = fmaxf(most, x < INFINITY ? x : 0.f);
            }
        most = ssq_wave_max(most);
        if (lane == 0) red[wave] = most;
        __syncthreads();
        most = 0.f;
#pragma unroll
        for (int w = 0; w < kWinWaves; ++w) most = fmaxf(most, red[w]);
        book_exp = min(15 - win_exp(most), 126);
        const float scale = ldexpf(1.f, book_exp);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int e = tid + k * kWinThreads;
            uint32_t hi[BD / 2], lo[BD / 2];
#pragma unroll
            for (int d = 0; d < BD; d += 2) {
                const bool in = (e & 255) < n_centroids;
                win_split(in ? c[k][d] * scale : 0.f, in ? c[k][d + 1] * scale : 0.f, hi[d / 2], lo[d / 2]);
            }
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
    }

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

    WinCut<TT, RP> cut;
    int x = wg, x_end = 0;
    const int whole = p->whole;
    if (!whole) {
        cut.init(p, lane);
        x = min((int64_t)wg * cut.share, (int64_t)cut.total);
        x_end = min((int64_t)(wg + 1) * cut.share, (int64_t)cut.total);
    }
    const int x_begin = x;
    for (;;) {
        // ---- the next item and this workgroup's tiles of it
        p = win_args();
        int item, i0 = 0, i1, slot = -1, start = 0, c = 0;
        if (whole) {
            if (x >= p->items) break;
            item = x;
            x += p->n_wg;
        } else {
            if (x >= x_end) break;
            cut.find(p, lane, x, item, start, c);
            if (item >= p->items) break;
            x = start + c;
        }
        item = __builtin_amdgcn_readfirstlane(item);
        const int b = item / p->rgroups, row0 = (item - b * p->rgroups) * RP;
        const int len = max(0, min(p->a.seq_lens[b], p->a.seq_len)), rows = p->rows, G = p->G;
        u.t = win_tiles<TT>(WinShape{u.window, u.sinks, q_len, G, rows}, len, row0, RP);
        i1 = u.t.n;
        if (!whole) {
            i0 = max(0, x_begin - start - p->fixed);
            i1 = max(0, min(u.t.n, x_end - start - p->fixed));
            if (u.t.n == 0 ? start < x_begin : i1 <= i0) continue;  // its part here is of the fixed cost
            const bool mine = i0 == 0 && i1 == u.t.n;
            if (!mine) slot = start < x_begin ? 0 : 1;
            if (i0 == 0 && kv == 0 && tid == 0) {  // pieces, for the merge
                const int w_last = (start + c - 1) / cut.share;
                p->meta[2 * item] = 2 * wg + (slot > 0 ? 1 : 0);
                p->meta[2 * item + 1] = mine ? 1 : w_last - wg + 1;
            }
        }
        const int nr = min(RP, rows - row0);

        // ---- its query rows: scaled in their dtype, permuted, in f16 at a power of two of each row's
        __syncthreads();  // (the codebook is staged, the last join is read)
        {
            constexpr int kLpr = D / 4;  // lanes of a row, 4 dims each
            uint16_t* qs = reinterpret_cast<uint16_t*>(smem + L::kBook);
#pragma unroll
            for (int r0 = 0; r0 < RP; r0 += kWinThreads / kLpr) {
                const int r = r0 + tid / kLpr, j = 4 * (tid % kLpr);
                if (RP < kWinThreads / kLpr && r >= RP) break;  // whole waves
                const int row = row0 + r, qi = row / G, h = kv * G + row - qi * G;
                float y[4] = {0.f, 0.f, 0.f, 0.f}, most = 0.f;
                if (r < nr) {
                    const int64_t at = (int64_t)b * p->a.q_sb + (int64_t)h * p->a.q_sh + (int64_t)qi * p->a.q_sl;
                    int64_t idx[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) idx[k] = at + perm[j + k];
                    ssq_load_elems(p->a.q, p->a.q_dtype, idx, y);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (p->a.has_scale) y[k] = ssq_round_to(y[k] * p->a.scale, p->a.q_dtype);
                    const float z = fabsf(y[k]);
                    most = fmaxf(most, z < INFINITY ? z : 0.f);
                }
#pragma unroll
                for (int o = 1; o < kLpr; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
                const int up = min(15 - win_exp(most), 126);
                const float s = ldexpf(1.f, up);
                uint32_t hi[2], lo[2];
                win_split(y[0] * s, y[1] * s, hi[0], lo[0]);
                win_split(y[2] * s, y[3] * s, hi[1], lo[1]);
                *reinterpret_cast<uint2*>(qs + r * L::kQRow + j) = make_uint2(hi[0], hi[1]);
                if constexpr (QP == 2) *reinterpret_cast<uint2*>(qs + (RP + r) * L::kQRow + j) = make_uint2(lo[0], lo[1]);
                if (tid % kLpr == 0) facs[r] = ldexpf(kWinLog2e, max(-book_exp - up, -126));  // above 0
            }
        }
        // this wave's first places
        const int n_mine = i1 > i0 + wave ? (i1 - i0 - wave + kWinWaves - 1) / kWinWaves : 0;
        const int last_i = i0 + wave + kWinWaves * (n_mine - 1);
        u.table = p->a.block_table + (int64_t)b * p->a.bt_sb;
        u.last_tok = u.t.p_hi;
        // the places of the next tile's values and of the codes after the next tile's; the codes of this and the next tile
        typename W::Place pv{}, pc{};
        typename W::Codes c0, c1;
        typename W::Vals val;
        if (n_mine > 0) {
            const int i = i0 + wave, in = min(i + kWinWaves, last_i);
            pc = u.place(i, u.code_chunk());
            pv = u.place(i, u.grp);
            const typename W::Place pcn = u.place(in, u.code_chunk()), pvn = u.place(in, u.grp);
            const typename W::Place pc2 = u.place(min(i + 2 * kWinWaves, last_i), u.code_chunk());
            u.load_codes(pc, c0);
            u.load_codes(pcn, c1);
            u.load_vals(pv, val);
            pc = pc2;
            pv = pvn;
        }
        __syncthreads();
        {
            const uint16_t* qs = reinterpret_cast<const uint16_t*>(smem + L::kBook);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                u.fac[n] = facs[16 * n + u.col];
                u.pos[n] = len - q_len + min(row0 + 16 * n + u.col, rows - 1) / G;
#pragma unroll
                for (int h = 0; h < QP; ++h) {
                    const uint16_t* src = qs + (h * RP + 16 * n + u.col) * L::kQRow + u.grp * (D / 4);
#pragma unroll
                    for (int k = 0; k < W::NQ; ++k) {
                        if constexpr (BD == 8) {
                            u.q[h][n][k] = *reinterpret_cast<const uint4*>(src + 8 * k);
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(src + 4 * k);
                            if constexpr (BD == 4) u.q[h][n][k] = make_uint4(w.x, w.y, w.x, w.y);
                            else u.q[h][n][k] = make_uint4(w.x, w.x, w.y, w.y);
                        }
                    }
                }
            }
        }

        // ---- this wave's tiles
        float m[NR], l[NR], unit = W::kV8 ? kWinScale : 1.f, inv_unit = 1.f / unit;
        w4f o[NR][DT];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            m[n] = kWinNone;
            l[n] = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[n][dt] = w4f{};
        }
        // Loads return in order: a place is asked for a tile before it is used, and before that tile's values.
        for (int i = i0 + wave; i < i1; i += kWinWaves) {
            w4f s[NS][NR];
            u.scores(c0, s);
            c0 = c1;
            u.load_codes(pc, c1);
            pc = u.place(min(i + 3 * kWinWaves, last_i), u.code_chunk());
            const int t0 = TT * u.tile_of(i), tok = t0 + CH * u.grp;
            // tokens of the tile that some row does not see (uniform)
            const bool edge = (t0 + TT - 1 > u.t.p_lo) | ((t0 <= u.t.p_hi - u.window) & (t0 + TT > u.sinks));
            bool apart = false;  // an infinite or NaN value that some rows see and others do not
            if (edge) {
                const uint32_t any = u.sees(u.t.p_lo, u.t.p_hi, tok), all = u.sees(u.t.p_hi, u.t.p_lo, tok);
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const uint32_t mine = u.sees(u.pos[n], u.pos[n], tok);
#pragma unroll
                    for (int e = 0; e < CH; ++e) s[e >> 2][n][e & 3] = mine >> e & 1u ? s[e >> 2][n][e & 3] : -INFINITY;
                }
                if (any == 0) val.scale = 0.f;  // no page of this tile's
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
            float top[NR];
            bool over = false;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                top[n] = s[0][n][0];
#pragma unroll
                for (int e = 1; e < CH; ++e) top[n] = fmaxf(top[n], s[e >> 2][n][e & 3]);
                top[n] *= u.fac[n];
                over |= top[n] > m[n] + kWinOver;
            }
            if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float mn = fmaxf(m[n], win_max4(top[n]) - kWinTop);
                    const float f = __builtin_amdgcn_exp2f(m[n] - mn);
                    m[n] = mn;
                    l[n] *= f;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][dt][e] *= f;
                }
            }
            float by = 1.f;  // this group's page scale, in units of O
            if constexpr (W::kV8) {
                const uint32_t bits = __float_as_uint(val.scale);
                uint32_t big = max(max((uint32_t)__builtin_amdgcn_readlane((int)bits, 0), (uint32_t)__builtin_amdgcn_readlane((int)bits, 16)),
                                   max((uint32_t)__builtin_amdgcn_readlane((int)bits, 32), (uint32_t)__builtin_amdgcn_readlane((int)bits, 48)));
                if (big > __float_as_uint(unit)) {  // uniform: positive floats compare as their bits
                    const float f = unit / __uint_as_float(big);
                    unit = __uint_as_float(big);
                    inv_unit = 1.f / unit;
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][dt][e] *= f;
                }
                by = val.scale * inv_unit;
            }
            uint32_t pw[NR][CH / 2];
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < CH; e += 2) {
                    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][n][e & 3], u.fac[n], -m[n]));
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][n][(e & 3) + 1], u.fac[n], -m[n]));
                    l[n] += x0 + x1;
                    pw[n][e / 2] = W::kV8 ? win_pack_p<VT>(x0 * by, x1 * by) : win_pack_p<VT>(x0, x1);
                }
            if (apart) {
                // The rows of one position at a time, the values that they do not see as 0; the products below then add nothing.
                for (int at = u.t.p_lo; at <= u.t.p_hi; ++at) {
                    const w4u on = W::spread(u.sees(at, at, tok));
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            w4f y = o[n][dt];
#pragma unroll
                            for (int jj = 0; jj < CH / 8; ++jj)
                                y = win_mfma_v<VT>(u.vals(val.v[dt] & on, jj), make_uint4(pw[n][4 * jj], pw[n][4 * jj + 1], pw[n][4 * jj + 2], pw[n][4 * jj + 3]), y);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][dt][e] = u.pos[n] == at ? y[e] : o[n][dt][e];
                        }
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) val.v[dt] = w4u{};
            }
            const uint8_t* next_row = u.val_row(pv);
            val.scale = u.load_scale(pv);
            pv = u.place(min(i + 2 * kWinWaves, last_i), u.grp);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {  // a value operand's successor loads once it is used
#pragma unroll
                for (int jj = 0; jj < CH / 8; ++jj) {
                    const uint4 v = u.vals(val.v[dt], jj);
#pragma unroll
                    for (int n = 0; n < NR; ++n)
                        o[n][dt] = win_mfma_v<VT>(v, make_uint4(pw[n][4 * jj], pw[n][4 * jj + 1], pw[n][4 * jj + 2], pw[n][4 * jj + 3]), o[n][dt]);
                }
                val.v[dt] = u.load_val(next_row, dt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        // ---- the waves' join, 4 rows at a time
        p = win_args();
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            l[n] = win_sum4(l[n]);
            if (lane < 16) {
                mls[wave * RP + 16 * n + lane] = m[n];
                mls[(kWinWaves + wave) * RP + 16 * n + lane] = l[n];
            }
        }
        __syncthreads();
        float f[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            float mt = kWinNone;
#pragma unroll
            for (int w = 0; w < kWinWaves; ++w) mt = fmaxf(mt, mls[w * RP + 16 * n + u.col]);
            f[n] = __builtin_amdgcn_exp2f(m[n] - mt) * unit;
        }
        float* join = reinterpret_cast<float*>(smem + L::kBook);
        constexpr int kRow = L::kJoinRow;
#pragma unroll 1
        for (int r0 = 0; r0 < nr; r0 += L::kJoinRows) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
                if (r0 / 16 == n && (u.col & ~3) == (r0 & 15)) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        *reinterpret_cast<float4*>(join + (wave * 4 + (u.col & 3)) * kRow + 16 * dt + 4 * u.grp) =
                            make_float4(o[n][dt][0] * f[n], o[n][dt][1] * f[n], o[n][dt][2] * f[n], o[n][dt][3] * f[n]);
                }
            __syncthreads();
            for (int e = tid; e < 4 * D; e += kWinThreads) {
                const int r = r0 + e / D, dv = e % D;
                if (r >= nr) continue;
                float mt = kWinNone;
#pragma unroll
                for (int w = 0; w < kWinWaves; ++w) mt = fmaxf(mt, mls[w * RP + r]);
                float lt = 0.f, ot = 0.f;
#pragma unroll
                for (int w = 0; w < kWinWaves; ++w) {
                    lt += mls[(kWinWaves + w) * RP + r] * __builtin_amdgcn_exp2f(mls[w * RP + r] - mt);
                    ot += join[(w * 4 + r - r0) * kRow + dv];
                }
                if (slot < 0) {
                    const int row = row0 + r, qi = row / p->G, h = kv * p->G + row - qi * p->G;
                    ssq_store_elem(p->a.out, p->out_dtype, (int64_t)b * p->a.o_sb + (int64_t)h * p->a.o_sh + (int64_t)qi * p->a.o_sl + dv,
                                   lt == 0.f ? 0.f : ot / lt);
                    if (p->a.lse && dv == 0)
                        p->a.lse[((int64_t)b * p->a.num_q_heads + h) * p->a.q_len + qi] = lt == 0.f ? -INFINITY : (mt + log2f(lt)) * kWinLn2;
                } else {
                    float* dst = p->part + ((int64_t)(kv * p->n_wg + wg) * 2 + slot) * (RP * (D + 2));
                    dst[r * D + dv] = ot;
                    if (dv == 0) {
                        dst[RP * D + r] = mt;
                        dst[RP * D + RP + r] = lt;
                    }
                }
            }
            __syncthreads();
        }
    }
}

// Joins the pieces of the items that workgroups shared.  One wave a query row, lanes over the value dims.
template <int RP, int D>
__global__ __launch_bounds__(256) void k_window_merge(const SsqWindowParams p) {
    constexpr int E = D / SSQ_WAVE;
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & 63;
    const int id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (sequence, KV head, row)
    const int bk = id / p.rows, row = id - bk * p.rows, b = bk / a.num_kv_heads, kv = bk - b * a.num_kv_heads;
    if (b >= a.batch) return;
    const int item = b * p.rgroups + row / RP, r = row % RP;
    const int first = p.meta[2 * item], pieces = p.meta[2 * item + 1];
    if (pieces <= 1) return;
    const float* base = p.part + (int64_t)kv * p.n_wg * 2 * (RP * (D + 2));
    auto at = [&](int i) { return base + (int64_t)(i ? 2 * ((first >> 1) + i) : first) * (RP * (D + 2)); };
    float M = kWinNone;
    for (int i = lane; i < pieces; i += SSQ_WAVE) M = fmaxf(M, at(i)[RP * D + r]);
    M = ssq_wave_max(M);
    float l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    constexpr int kAhead = 8;
    for (int i0 = 0; i0 < pieces; i0 += kAhead) {
        float w[kAhead], lp[kAhead], op[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const float* src = at(min(i0 + j, pieces - 1));
            w[j] = src[RP * D + r];
            lp[j] = src[RP * D + RP + r];
#pragma unroll
            for (int e = 0; e < E; ++e) op[j][e] = src[r * D + lane * E + e];
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i0 + j >= pieces) continue;
            const float f = __builtin_amdgcn_exp2f(w[j] - M);
            l += lp[j] * f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += op[j][e] * f;
        }
    }
    const int qi = row / p.G, h = kv * p.G + row - qi * p.G;
#pragma unroll
    for (int e = 0; e < E; ++e)
        ssq_store_elem(a.out, p.out_dtype, (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)qi * a.o_sl + lane * E + e,
                       l == 0.f ? 0.f : o[e] / l);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.num_q_heads + h) * a.q_len + qi] = l == 0.f ? -INFINITY : (M + log2f(l)) * kWinLn2;
}

template <int D, int BD, int VT, int NR, int QP>
int win_launch(const SsqWindowParams& p, hipStream_t st) {
    using L = WinLds<D, NR, QP>;
    static_assert(L::kTotal <= 160 * 1024, "a workgroup's LDS");
    auto kern = k_window<D, BD, VT, NR, QP>;
    constexpr int kWinThreads = win_waves(NR) * SSQ_WAVE;
    int rc = ssq_allow_lds((const void*)kern, L::kTotal, "hipFuncSetAttribute(k_window)");
    if (rc) return rc;
    hipLaunchKernelGGL(kern, dim3(p.n_wg * p.a.num_kv_heads), dim3(kWinThreads), L::kTotal, st, p);
    rc = ssq_check_hip(hipGetLastError(), "k_window launch");
    if (rc || p.whole) return rc;
    const int64_t rows = (int64_t)p.a.batch * p.a.num_kv_heads * p.rows;
    hipLaunchKernelGGL((k_window_merge<16 * NR, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
    return ssq_check_hip(hipGetLastError(), "k_window_merge launch");
}
template <int D, int BD, int VT>
int win_rows(const SsqWindowParams& p, int nr, hipStream_t st) {
    const bool split = p.a.q_dtype == SSQ_F32;
    if (nr == 1) return split ? win_launch<D, BD, VT, 1, 2>(p, st) : win_launch<D, BD, VT, 1, 1>(p, st);
    return split ? win_launch<D, BD, VT, 2, 2>(p, st) : win_launch<D, BD, VT, 2, 1>(p, st);
}
template <int D, int VT>
int win_blocks(const SsqWindowParams& p, int nr, hipStream_t st) {
    switch (p.a.block_dim) {
        case 2: return win_rows<D, 2, VT>(p, nr, st);
        case 4: return win_rows<D, 4, VT>(p, nr, st);
        default: return win_rows<D, 8, VT>(p, nr, st);
    }
}

}  // namespace
