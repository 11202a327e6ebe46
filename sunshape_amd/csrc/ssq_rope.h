// Per-head RMS norm and position rotation of rows [B, H, S, D] (ssq_qk_norm_rope, ssq_append).
//
//   u = (x * r) * w, r = 1 / sqrt(mean(x^2) + eps);  (u1, u2) -> (u1 c - u2 s, u2 c + u1 s).
//
// The sum of squares and r are held in 64 bits: the squares of 16-bit values are exact there and the
// order of the sum does not show after r is rounded to 32 bits, so a row's result does not depend on how
// its dims are spread over lanes, and the codes an append picks do not depend on the kernel that serves
// it.  Products and sums after that are fp32, each rounded (-ffp-contract=off), in the order above.
#pragma once

#include "ssq_common.h"

namespace {

typedef __bf16 rope_bf2 __attribute__((ext_vector_type(2)));
typedef float rope_f2 __attribute__((ext_vector_type(2)));

// two fp32 values rounded to a 16-bit dtype (RNE; NaN stays NaN), packed
template <int DT>
__device__ __forceinline__ uint32_t rope_pack2(float a, float b) {
    if constexpr (DT == SSQ_BF16) {
        const rope_f2 f = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, rope_bf2));
    } else {
        return ssq_f32_to_f16(a) | (ssq_f32_to_f16(b) << 16);
    }
}
__device__ __forceinline__ float rope_round(float x, int dt) {  // to dtype dt, as fp32
    if (dt == SSQ_BF16) return ssq_bf16_to_f32(rope_pack2<SSQ_BF16>(x, 0.f) & 0xFFFFu);
    if (dt == SSQ_F16) return ssq_f16_to_f32(ssq_f32_to_f16(x));
    return x;
}
__device__ __forceinline__ void rope_store(void* p, int dt, int64_t i, float x) {
    if (dt == SSQ_F32) reinterpret_cast<float*>(p)[i] = x;
    else if (dt == SSQ_BF16) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)rope_pack2<SSQ_BF16>(x, 0.f);
    else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)ssq_f32_to_f16(x);
}

// elements of one 16-byte piece
template <int DT>
struct RopeVec {
    static constexpr int N = DT == SSQ_F32 ? 4 : 8;
};

template <int DT>
__device__ __forceinline__ void rope_unpack(const uint4& v, float (&x)[RopeVec<DT>::N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == SSQ_F32) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == SSQ_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            x[2 * i] = ssq_f16_to_f32(w[i] & 0xFFFFu);
            x[2 * i + 1] = ssq_f16_to_f32(w[i] >> 16);
        }
    }
}
template <int DT>
__device__ __forceinline__ uint4 rope_packv(const float (&x)[RopeVec<DT>::N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == SSQ_F32) w[i] = __float_as_uint(x[i]);
        else w[i] = rope_pack2<DT>(x[2 * i], x[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 1 / sqrt(sum / D + eps), inv_d = 1 / D.  The hardware's estimate r has about 24 bits; with e = 1 - m r^2 the step
// r (1 + e / 2 + 3 e^2 / 8) leaves 64 bits' rounding alone, at a fifth of the operations of a division,
// a square root and a reciprocal.  An infinite mean gives 0; a mean of 0 with eps = 0, NaN (0 * inf).
__device__ __forceinline__ float rope_rstd(double sum, double inv_d, double eps) {
    const double m = __builtin_fma(sum, inv_d, eps);
    const double r = __builtin_amdgcn_rsq(m);
    const double e = __builtin_fma(-(m * r), r, 1.0);
    const double y = __builtin_fma(r * e, __builtin_fma(e, 0.375, 0.5), r);
    return (float)(m == __builtin_inf() ? 0.0 : y);
}

// the row of the tables for token (b, s), or -1 for a position outside them
__device__ __forceinline__ int64_t rope_pos(const ssq_rope& t, int b, int s) {
    const int64_t pos = t.positions[(int64_t)b * t.p_sb + (int64_t)s * t.p_ss];
    return pos >= 0 && pos < t.max_pos ? pos : -1;
}

// One normed and rotated dim of a row by itself: raw(i) is element i, wt(i) its weight.
template <class Raw, class Wt>
__device__ __forceinline__ float rope_dim(const ssq_rope& t, int64_t pos, int dim, bool norm, float r, Raw raw, Wt wt) {
    auto u = [&](int i) { return norm ? (raw(i) * r) * wt(i) : raw(i); };
    const float x = u(dim);
    if (!t.cos || dim >= t.rot_dim) return x;
    const int half = t.rot_dim >> 1;
    const bool first = t.interleaved ? !(dim & 1) : dim < half;
    const int other = t.interleaved ? dim ^ 1 : first ? dim + half : dim - half;
    const int i = t.interleaved ? dim >> 1 : first ? dim : dim - half;
    const float y = u(other);
    const int64_t at = (pos < 0 ? 0 : pos) * t.ld + i;
    const float c = pos < 0 ? __builtin_nanf("") : t.cos[at], s = pos < 0 ? __builtin_nanf("") : t.sin[at];
    const float a = x * c, b = y * s;
    return first ? a - b : a + b;
}

}  // namespace

// Rows of one or two tensors of a dtype (queries and keys), as a kernel takes them.
struct SsqRopeRows {
    const void* x[2];
    void* y[2];
    int64_t x_sb[2], x_sh[2], x_ss[2], y_sb[2], y_sh[2], y_ss[2];
    const void* w[2];
    int32_t heads[2], batch, seq_len, head_dim, dtype;
    ssq_rope t;
};

namespace {

constexpr int kRopeThreads = 256;

struct RopeParams {
    SsqRopeRows r;
    int lpr, lpr_log;  // lanes per row, a power of two
    int groups;        // head groups per token
    int64_t items;     // tokens * groups
    double inv_d;      // 1 / head_dim
};

// LDS floats of the weights: two rows of the widest head dim
template <int DT, bool NORM>
constexpr int rope_lds() { return NORM ? 4 * RopeVec<DT>::N * SSQ_WAVE : 4; }

// Bytes bound it: every element is read and written once, 7 operations each.  A lane takes a unit of two
// 16-byte pieces that hold both dims of its pairs ([i, i + V) and [i + rot / 2, ..) of the halves, 2 V
// consecutive dims when interleaved), so a pair never crosses lanes and only the norm's sum does (within
// the D / 2V lanes of a row).  A lane keeps its unit for HEADS heads of one token, whose loads are in
// flight together, with the token's table entries in registers and the weights in LDS.  blk: the workgroup.
template <int DT, bool NORM, int HEADS>
__device__ __forceinline__ void rope_units(const RopeParams& p, int64_t blk, float* wl) {
    constexpr int V = RopeVec<DT>::N, kRow = 2 * V * SSQ_WAVE;
    const SsqRopeRows& R = p.r;
    const ssq_rope& t = R.t;
    const int u = threadIdx.x & (p.lpr - 1);
    const int64_t item = (blk * kRopeThreads + threadIdx.x) >> p.lpr_log;
    const bool live = item < p.items;
    const int64_t it = live ? item : p.items - 1;
    const int64_t tok = it / p.groups;
    const int h0 = (int)(it - tok * p.groups) * HEADS;
    const int b = (int)(tok / R.seq_len), s = (int)(tok - (int64_t)b * R.seq_len);
    const int H = R.heads[0] + R.heads[1], D = R.head_dim;
    const int rot = t.cos ? t.rot_dim : 0;
    // the unit's two pieces
    const bool turned = u < rot / (2 * V);
    int o0, o1;
    if (turned && !t.interleaved) {
        o0 = u * V;
        o1 = (rot >> 1) + u * V;
    } else {  // adjacent pieces: interleaved pairs, or dims past rot (whose units count on from rot's)
        o0 = 2 * u * V;
        o1 = o0 + V;
    }
    uint4 x0[HEADS], x1[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        const int h = min(h0 + k, H - 1);
        const int j = h >= R.heads[0];
        const int64_t row = (int64_t)b * R.x_sb[j] + (int64_t)(j ? h - R.heads[0] : h) * R.x_sh[j] + (int64_t)s * R.x_ss[j];
        const char* src = reinterpret_cast<const char*>(R.x[j]) + row * (16 / V);
        x0[k] = *reinterpret_cast<const uint4*>(src + o0 * (16 / V));
        x1[k] = *reinterpret_cast<const uint4*>(src + o1 * (16 / V));
    }
    if constexpr (NORM) {
        for (int i = threadIdx.x; i < 2 * D; i += kRopeThreads) {
            const int j = i >= D;
            wl[j * kRow + i - j * D] = R.w[j] ? ssq_load_elem(R.w[j], t.w_dtype, i - j * D) : 0.f;
        }
        __syncthreads();
    }
    float c[V], sn[V];
    if (turned) {
        const int64_t pos = rope_pos(t, b, s);
        const float* cr = t.cos + (pos < 0 ? 0 : pos) * t.ld + u * V;
        const float* sr = t.sin + (pos < 0 ? 0 : pos) * t.ld + u * V;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 a = *reinterpret_cast<const float4*>(cr + i), d = *reinterpret_cast<const float4*>(sr + i);
            c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
            sn[i] = d.x; sn[i + 1] = d.y; sn[i + 2] = d.z; sn[i + 3] = d.w;
        }
        if (pos < 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = sn[i] = __builtin_nanf("");
        }
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        const int h = min(h0 + k, H - 1);
        const int j = h >= R.heads[0];
        float a[V], d[V];
        rope_unpack<DT>(x0[k], a);
        rope_unpack<DT>(x1[k], d);
        if constexpr (NORM) {
            if (R.w[j]) {  // the same for a whole row, not for a wave: the shuffles stay within a row's lanes
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum = __builtin_fma((double)a[i], (double)a[i], sum);
                    sum = __builtin_fma((double)d[i], (double)d[i], sum);
                }
                for (int o = p.lpr >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
                const float r = rope_rstd(sum, p.inv_d, t.eps);
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const float4 w0 = *reinterpret_cast<const float4*>(&wl[j * kRow + o0 + i]);
                    const float4 w1 = *reinterpret_cast<const float4*>(&wl[j * kRow + o1 + i]);
                    a[i] = (a[i] * r) * w0.x; a[i + 1] = (a[i + 1] * r) * w0.y;
                    a[i + 2] = (a[i + 2] * r) * w0.z; a[i + 3] = (a[i + 3] * r) * w0.w;
                    d[i] = (d[i] * r) * w1.x; d[i + 1] = (d[i + 1] * r) * w1.y;
                    d[i + 2] = (d[i + 2] * r) * w1.z; d[i + 3] = (d[i + 3] * r) * w1.w;
                }
            }
        }
        if (turned) {
            if (t.interleaved) {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    float m = a[i] * c[i >> 1], n = a[i + 1] * sn[i >> 1], q = a[i + 1] * c[i >> 1], e = a[i] * sn[i >> 1];
                    a[i] = m - n;
                    a[i + 1] = q + e;
                    constexpr int W = V / 2;
                    m = d[i] * c[W + (i >> 1)]; n = d[i + 1] * sn[W + (i >> 1)];
                    q = d[i + 1] * c[W + (i >> 1)]; e = d[i] * sn[W + (i >> 1)];
                    d[i] = m - n;
                    d[i + 1] = q + e;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float m = a[i] * c[i], n = d[i] * sn[i], q = d[i] * c[i], e = a[i] * sn[i];
                    a[i] = m - n;
                    d[i] = q + e;
                }
            }
        }
        if (live && h0 + k < H) {
            const int64_t row = (int64_t)b * R.y_sb[j] + (int64_t)(j ? h - R.heads[0] : h) * R.y_sh[j] + (int64_t)s * R.y_ss[j];
            char* dst = reinterpret_cast<char*>(R.y[j]) + row * (16 / V);
            *reinterpret_cast<uint4*>(dst + o0 * (16 / V)) = rope_packv<DT>(a);
            *reinterpret_cast<uint4*>(dst + o1 * (16 / V)) = rope_packv<DT>(d);
        }
    }
}

}  // namespace

// argument checks of the rotation (host); the caller has checked head_dim
int ssq_rope_check(const ssq_rope& t, int head_dim, bool norm);
// normed and rotated rows, x -> y
int ssq_rope_run(const SsqRopeRows& r, hipStream_t st);
// whether the unit kernel serves the rows: whole 16-byte pieces, a power of two of them per row
bool ssq_rope_units_ok(const SsqRopeRows& r, int& lpr);
