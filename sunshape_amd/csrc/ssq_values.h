// Values to 8-bit pages (ssq_append_values, and ssq_append8's values): e4m3 with one fp32 scale per (page, KV head).
//
// scale = the smallest power of two s >= 2^-100 with |v| <= 448 s for every finite value of the page's tokens, and no less
// than the page's scale unless its first token (offset 0) is among the new ones.  Stored is v / s rounded to e4m3 (RNE; the
// division is exact).  Where the scale grows, the page's earlier tokens are taken to the new one: their bytes times old /
// new, rounded again, which changes what falls below e4m3's normal range (2^-6 of the scale) and nothing else.  NaN and
// infinities are stored as NaN and do not count for the scale.  The earlier tokens of a page are those before its
// first new one; bytes behind the new ones stay.
//
// A run is the tokens of a row (b, .) that go to one page; it starts at its first one, whose wave takes the run whole, so
// a page's scale needs no atomic and nothing depends on an order.  A wave looks at kRunChunk positions of a row for starts,
// for one head of up to 128 dims or two of up to 64 at a time: a lane holds two dims of up to 16 tokens, which become two
// 16-byte rows of the dim-major page in registers (ValWave::small; ValWave::run serves any run).  Bound by bytes for prompts;
// for a step by its chain of loads (slots, then values, scale and page together).  32,768 tokens of 8 heads of 128 dims, bf16
// (101 MB): 38 us, 2.7 TB/s (65 with runs through LDS, 61 with runs in registers and value types at run time), a wave's one load, wait and
// store; 37 times 5 rows of 2 heads of 64, a third of them padding: 8.3 us.
#pragma once

#include "ssq_common.h"

#include <type_traits>

struct SsqValues {
    const void* v;
    int v_dtype;
    int64_t v_sb, v_sh, v_ss;
    int batch, heads, seq_len, value_dim;
    uint8_t* pages;
    int64_t vp_sb, vp_sh, vp_sd;
    float* scale;
    int64_t vs_sb, vs_sh;
    const int64_t* slots;
    int64_t sm_sb, n_slots;
    int page_size, page_log;  // page_log -1: no power of two
    int vec;                  // pairs of dims load as one word
    int chunks, hgroups;      // waves: batch x chunks of a row x groups of heads
    int two;                  // a wave takes two heads (at most 64 dims)
};

constexpr int kRunChunk = 16;

namespace {

constexpr float kValLeast = 7.888609052210118e-31f;  // 2^-100

// the smallest power of two s >= 2^-100 with x <= 448 s (448 = 0.875 * 2^9)
__device__ __forceinline__ float val_scale(float x) {
    if (!(x > 448.f * kValLeast)) return kValLeast;
    const int e = __builtin_amdgcn_frexp_expf(x);
    return ldexpf(1.f, e - 9 + (__builtin_amdgcn_frexp_mantf(x) > 0.875f ? 1 : 0));
}
// x / s (s a power of two: times its inverse, exact) as what e4m3 rounds; infinities go to NaN
__device__ __forceinline__ float val_in(float x, float inv) {
    return fabsf(x) < INFINITY ? x * inv : __builtin_nanf("");
}
// four fp32 values, |x| <= 448 or NaN, to e4m3 (RNE)
__device__ __forceinline__ uint32_t val_pack(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ void val_unpack(uint32_t w, float (&x)[4]) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
}
// bytes [0, n) of a 16-byte row times f
__device__ __forceinline__ uint4 val_rescale(uint4 row, int n, float f) {
    uint32_t w[4] = {row.x, row.y, row.z, row.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float x[4];
        val_unpack(w[k], x);
        const uint32_t y = val_pack(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
        const int left = n - 4 * k;  // uniform
        const uint32_t take = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        w[k] = (y & take) | (w[k] & ~take);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A wave's runs: those that start at positions [16 chunk, 16 chunk + 16) of row b, for its heads.
struct ValWave {
    const SsqValues& p;
    int lane, b, head, dim, L;  // this lane's head and first dim (two of every 2 L), lanes of a head
    bool on;                    // its head exists

    struct At { int page, off; };
    __device__ __forceinline__ At at(int s) const {  // page -1: padding, or past the row
        At r{-1, 0};
        if (s < 0 || s >= p.seq_len) return r;
        const int64_t slot = p.slots[(int64_t)b * p.sm_sb + s];
        if (slot < 0 || slot >= p.n_slots) return r;
        r.page = (int)(p.page_log >= 0 ? slot >> p.page_log : slot / p.page_size);
        r.off = (int)(slot - (int64_t)r.page * p.page_size);
        return r;
    }
    __device__ __forceinline__ void load2(int s, int d, float (&x)[2]) const {
        const int64_t i = (int64_t)b * p.v_sb + (int64_t)head * p.v_sh + (int64_t)s * p.v_ss + d;
        x[0] = x[1] = 0.f;
        if (!on || d >= p.value_dim) return;
        if (p.vec) {  // uniform
            if (p.v_dtype == SSQ_F32) {
                const float2 w = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p.v) + i);
                x[0] = w.x; x[1] = w.y;
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(p.v) + i);
                x[0] = ssq_bits_to_f32(w & 0xFFFFu, p.v_dtype);
                x[1] = ssq_bits_to_f32(w >> 16, p.v_dtype);
            }
        } else {
            x[0] = ssq_load_elem(p.v, p.v_dtype, i);
            if (d + 1 < p.value_dim) x[1] = ssq_load_elem(p.v, p.v_dtype, i + 1);
        }
    }
    __device__ __forceinline__ static float most(float m, const float (&x)[2]) {
        const float u = fabsf(x[0]), w = fabsf(x[1]);
        return fmaxf(m, fmaxf(u < INFINITY ? u : 0.f, w < INFINITY ? w : 0.f));
    }
    __device__ __forceinline__ uint8_t* row(int page, int d) const {
        return p.pages + (int64_t)page * p.vp_sb + (int64_t)head * p.vp_sh + (int64_t)d * p.vp_sd;
    }

    // One run: it starts at position s0; the 64 positions from there are this wave's lanes (r: theirs).
    __device__ __forceinline__ void run(int s0, At r) const {
        const int page = __builtin_amdgcn_readfirstlane(r.page);
        const float held = on ? p.scale[(int64_t)page * p.vs_sb + (int64_t)head * p.vs_sh] : kValLeast;
        const int D = p.value_dim, step = 2 * L;
        // ---- the run's tokens: the largest value, the first offset
        float top = 0.f;
        int n = 0, first = p.page_size, lead = 0;
        bool in_order = true, in_row = true;  // offsets ascend by one; positions do
        uint64_t bits = 0;                    // the run's positions from s0 (the first 64)
        for (int base = 0;; base += SSQ_WAVE) {
            if (base) r = at(s0 + base + lane);
            const uint64_t live = __builtin_amdgcn_ballot_w64(r.page >= 0), same = __builtin_amdgcn_ballot_w64(r.page == page);
            const uint64_t other = live & ~same;
            const uint64_t mine = other ? same & ((1ull << __builtin_ctzll(other)) - 1ull) : same;
            if (base == 0) {
                bits = mine;
                lead = __builtin_amdgcn_readfirstlane(r.off);
            }
            // rows 8 at a time
            uint64_t left = mine;
            while (left) {
                float y[8][2];
                int k = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j][0] = y[j][1] = 0.f;
                    if (left) {  // uniform
                        const int l = __builtin_ctzll(left);
                        left &= left - 1;
                        const int off = __builtin_amdgcn_readlane(r.off, l);
                        first = min(first, off);
                        in_order &= off == lead + n + j;
                        in_row &= base + l == n + j;
                        load2(s0 + base + l, dim, y[j]);
                        k = j + 1;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = most(top, y[j]);
                n += k;
            }
            for (int d = dim + step; d < (D + step - 1) / step * step; d += step)  // dims past the first 2 L
                for (uint64_t w = mine; w; w &= w - 1) {
                    float y[2];
                    load2(s0 + base + __builtin_ctzll(w), d, y);
                    top = most(top, y);
                }
            if (other || s0 + base + SSQ_WAVE >= p.seq_len) break;
        }
        for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float need = val_scale(top);
        const float now = first > 0 ? fmaxf(held, need) : need, inv = 1.f / now, again = held * inv;
        const bool grown = first > 0 && now != held;
        if (on && dim == 0) p.scale[(int64_t)page * p.vs_sb + (int64_t)head * p.vs_sh] = now;
        // ---- the held bytes, then the new ones, whole 16-byte rows where offsets and positions ascend together
        for (int d0 = dim; d0 < (D + step - 1) / step * step; d0 += step) {
            for (int e = 0; e < 2; ++e) {
                const int d = d0 + e;
                if (grown && on && d < D)
                    for (int c = 0; c < first; c += 16) {
                        uint4* dst = reinterpret_cast<uint4*>(row(page, d) + c);
                        *dst = val_rescale(*dst, min(16, first - c), again);
                    }
            }
            int k = 0;  // tokens written
            if (in_order && in_row) {
                while (k < n) {
                    const int off = first + k;
                    if (off % 16 == 0 && n - k >= 16) {
                        float y[16][2];
#pragma unroll
                        for (int j = 0; j < 16; ++j) load2(s0 + k + j, d0, y[j]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (!on || d0 + e >= D) continue;
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[i] = val_pack(val_in(y[4 * i][e], inv), val_in(y[4 * i + 1][e], inv), val_in(y[4 * i + 2][e], inv),
                                                val_in(y[4 * i + 3][e], inv));
                            *reinterpret_cast<uint4*>(row(page, d0 + e) + off) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        k += 16;
                    } else {
                        put(s0 + k, page, off, d0, inv);
                        ++k;
                    }
                }
                continue;
            }
            for (int base = 0; k < n; base += SSQ_WAVE) {
                const At q = at(s0 + base + lane);
                uint64_t mine = __builtin_amdgcn_ballot_w64(q.page == page);
                if (base == 0) mine = bits;
                while (mine && k < n) {
                    const int l = __builtin_ctzll(mine);
                    mine &= mine - 1;
                    put(s0 + base + l, page, __builtin_amdgcn_readlane(q.off, l), d0, inv);
                    ++k;
                }
                if (s0 + base + SSQ_WAVE >= p.seq_len) break;
            }
        }
    }
    // one token's two values, a byte each
    __device__ __forceinline__ void put(int s, int page, int off, int d, float inv) const {
        float y[2];
        load2(s, d, y);
        const uint32_t w = val_pack(val_in(y[0], inv), val_in(y[1], inv), 0.f, 0.f);
        if (on && d < p.value_dim) row(page, d)[off] = (uint8_t)w;
        if (on && d + 1 < p.value_dim) row(page, d + 1)[off] = (uint8_t)(w >> 8);
    }
    // A run of n <= 16 tokens at ascending offsets from `first` in a page of 16, at the positions s0 + (the bits of `mine`): one
    // 16-byte row a dim, the held bytes and the new ones.  Everything is asked for at once.
    template <int DT>
    __device__ __forceinline__ void small(int s0, uint64_t mine, int n, int page, int first) const {
        using Raw = std::conditional_t<DT == SSQ_F32, uint2, uint32_t>;  // a token's two values
        constexpr int kSize = DT == SSQ_F32 ? 4 : 2;
        Raw raw[16];
        const bool one = on && dim < p.value_dim;  // (pairs load whole: value_dim is even)
        const uint8_t* src = reinterpret_cast<const uint8_t*>(p.v) + ((int64_t)b * p.v_sb + (int64_t)head * p.v_sh + (one ? dim : 0)) * kSize;
#pragma unroll
        for (int j = 0; j < 16; ++j) {  // (those behind the last repeat it)
            raw[j] = *reinterpret_cast<const Raw*>(src + (int64_t)(s0 + __builtin_ctzll(mine)) * p.v_ss * kSize);
            const uint64_t rest = mine & (mine - 1);
            mine = rest ? rest : mine;
        }
        float* at_scale = p.scale + (int64_t)page * p.vs_sb + (int64_t)head * p.vs_sh;
        const float held = *at_scale;
        uint8_t* dst = row(page, one ? dim : 0);
        uint4 old[2];
        old[0] = old[1] = make_uint4(0, 0, 0, 0);
        if (n < 16) {  // uniform
            old[0] = *reinterpret_cast<const uint4*>(dst);
            old[1] = *reinterpret_cast<const uint4*>(dst + (one ? p.vp_sd : 0));
        }
        auto value = [&](int j, int e) {
            if constexpr (DT == SSQ_F32) return __uint_as_float(e ? raw[j].y : raw[j].x);
            else return ssq_bits_to_f32(e ? raw[j] >> 16 : raw[j] & 0xFFFFu, DT);
        };
        // (NaN leaves a maximum as it is; infinite ones are rare, and take a second look)
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(fabsf(value(j, 0)), fabsf(value(j, 1))));
        const bool wild = __builtin_amdgcn_ballot_w64(top == INFINITY) != 0;
        if (wild) {
            top = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float x[2] = {value(j, 0), value(j, 1)};
                top = most(top, x);
            }
        }
        if (!one) top = 0.f;
        for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float need = val_scale(top);
        const float now = first > 0 ? fmaxf(held, need) : need, inv = 1.f / now, again = held * inv;
        const bool grown = first > 0 && now != held;
        if (on && dim == 0) *at_scale = now;
        if (!one) return;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            uint32_t w[4];
            if (wild) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = val_pack(val_in(value(4 * k, e), inv), val_in(value(4 * k + 1, e), inv), val_in(value(4 * k + 2, e), inv),
                                    val_in(value(4 * k + 3, e), inv));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = val_pack(value(4 * k, e) * inv, value(4 * k + 1, e) * inv, value(4 * k + 2, e) * inv, value(4 * k + 3, e) * inv);
            }
            if (n < 16) {  // uniform
                if (grown) old[e] = val_rescale(old[e], first, again);
                const uint32_t ow[4] = {old[e].x, old[e].y, old[e].z, old[e].w};
                // w moved up by `first` bytes (uniform)
                const int ws = first >> 2, bs = 8 * (first & 3);
                uint32_t nw[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t hi = 0, lo = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j == k - ws) hi = w[j];
                        if (j == k - ws - 1) lo = w[j];
                    }
                    nw[k] = bs ? (hi << bs) | (lo >> (32 - bs)) : hi;
                    uint32_t take = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (4 * k + j >= first && 4 * k + j < first + n) take |= 0xFFu << (8 * j);
                    nw[k] = (ow[k] & ~take) | (nw[k] & take);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = nw[k];
            }
            *reinterpret_cast<uint4*>(dst + e * p.vp_sd) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ void chunk(int c) const {
        const int s0 = kRunChunk * c;
        // the chunk's positions and those after them, and the 64 before
        const At r = at(s0 + lane), back = at(s0 - 64 + lane);
        const uint64_t live = __builtin_amdgcn_ballot_w64(r.page >= 0), before = __builtin_amdgcn_ballot_w64(back.page >= 0);
        uint64_t own = live & ((1ull << kRunChunk) - 1ull);
        if (!own) return;
        int prev = -1;
        if (before) {
            prev = __builtin_amdgcn_readlane(back.page, 63 - __builtin_clzll(before));
        } else {
            for (int s = s0 - 64; s > 0; s -= SSQ_WAVE) {
                const At q = at(s - 1 - lane);
                const uint64_t any = __builtin_amdgcn_ballot_w64(q.page >= 0);
                if (any) {
                    prev = __builtin_amdgcn_readlane(q.page, __builtin_ctzll(any));
                    break;
                }
            }
        }
        while (own) {
            const int l = __builtin_ctzll(own), page = __builtin_amdgcn_readlane(r.page, l);
            own &= own - 1;
            if (page == prev) continue;
            prev = page;
            // the run's positions among the 64: up to the next one of another page
            const uint64_t from = ~0ull << l, same = __builtin_amdgcn_ballot_w64(r.page == page) & from, other = live & ~same & from;
            const uint64_t mine = other ? same & ((1ull << __builtin_ctzll(other)) - 1ull) : same;
            const int n = __builtin_popcountll(mine), first = __builtin_amdgcn_readlane(r.off, l);
            const bool is = mine >> lane & 1ull;
            const int rank = __builtin_popcountll(mine & ((1ull << lane) - 1ull));
            const bool whole = (other || s0 + SSQ_WAVE >= p.seq_len) && __builtin_amdgcn_ballot_w64(is && r.off != first + rank) == 0;
            if (!whole || p.page_size != 16 || p.value_dim > 2 * L || !p.vec) run(s0 + l, at(s0 + l + lane));
            else if (p.v_dtype == SSQ_BF16) small<SSQ_BF16>(s0, mine, n, page, first);
            else if (p.v_dtype == SSQ_F16) small<SSQ_F16>(s0, mine, n, page, first);
            else small<SSQ_F32>(s0, mine, n, page, first);
        }
    }
};

// waves of a call: id -> row, chunk of it, group of heads
__device__ __forceinline__ void val_wave(const SsqValues& p, int64_t id, int lane) {
    const int hg = (int)(id % p.hgroups);
    const int64_t bc = id / p.hgroups;
    const int c = (int)(bc % p.chunks);
    const int64_t b = bc / p.chunks;
    if (b >= p.batch) return;
    const int L = p.two ? 32 : 64, head = p.two ? 2 * hg + lane / 32 : hg;
    const ValWave w{p, lane, (int)b, min(head, p.heads - 1), 2 * (lane & (L - 1)), L, head < p.heads};
    w.chunk(c);
}

}  // namespace
