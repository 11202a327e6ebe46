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

// 1 / sqrt(mean + eps) of a sum of squares over D dims
__device__ __forceinline__ float rope_rstd(double sum, int D, double eps) {
    return (float)(1.0 / __builtin_sqrt(sum / (double)D + eps));
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

// argument checks of the rotation (host); the caller has checked head_dim
int ssq_rope_check(const ssq_rope& t, int head_dim, bool norm);
// normed and rotated rows, x -> y
int ssq_rope_run(const SsqRopeRows& r, hipStream_t st);
