// Norm and rotation of queries and keys, one pass (ssq_qk_norm_rope; mathematics in ssq_rope.h).
//
// Bytes bound it: every element is read and written once, 7 operations each.  A lane takes a unit of two
// 16-byte pieces that hold both dims of its pairs ([i, i + V) and [i + rot / 2, ..) of the halves, 2 V
// consecutive dims when interleaved), so a pair never crosses lanes and only the norm's sum does (within
// the D / 2V lanes of a row).  A lane keeps its unit for kHeads heads of one token, whose loads are in
// flight together, with the token's table entries in registers and the weights in LDS.
#include "ssq_rope.h"

namespace {

constexpr int kRopeThreads = 256;

struct RopeParams {
    SsqRopeRows r;
    int lpr, lpr_log;  // lanes per row, a power of two
    int groups;        // head groups per token
    int64_t items;     // tokens * groups
};

template <int DT, bool NORM, int HEADS>
__global__ __launch_bounds__(kRopeThreads) void k_rope_units(const RopeParams p) {
    constexpr int V = RopeVec<DT>::N;
    __shared__ __align__(16) float wl[NORM ? 2 : 1][NORM ? 2 * V * SSQ_WAVE : 4];
    const SsqRopeRows& R = p.r;
    const ssq_rope& t = R.t;
    const int u = threadIdx.x & (p.lpr - 1);
    const int64_t item = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) >> p.lpr_log;
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
            wl[j][i - j * D] = R.w[j] ? ssq_load_elem(R.w[j], t.w_dtype, i - j * D) : 0.f;
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
                const float r = rope_rstd(sum, D, t.eps);
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const float4 w0 = *reinterpret_cast<const float4*>(&wl[j][o0 + i]);
                    const float4 w1 = *reinterpret_cast<const float4*>(&wl[j][o1 + i]);
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

// Any head dim, alignment and rotated width: a wave per row, a lane per pair (and per dim past rot_dim).
__global__ __launch_bounds__(kRopeThreads) void k_rope_any(const RopeParams p) {
    const SsqRopeRows& R = p.r;
    const ssq_rope& t = R.t;
    const int lane = threadIdx.x & (SSQ_WAVE - 1);
    const int H = R.heads[0] + R.heads[1], D = R.head_dim;
    const int64_t row = (int64_t)blockIdx.x * (kRopeThreads / SSQ_WAVE) + threadIdx.x / SSQ_WAVE;
    if (row >= (int64_t)R.batch * R.seq_len * H) return;  // whole waves
    const int64_t tok = row / H;
    const int h = (int)(row - tok * H), j = h >= R.heads[0], hh = j ? h - R.heads[0] : h;
    const int b = (int)(tok / R.seq_len), s = (int)(tok - (int64_t)b * R.seq_len);
    const int64_t xr = (int64_t)b * R.x_sb[j] + (int64_t)hh * R.x_sh[j] + (int64_t)s * R.x_ss[j];
    const int64_t yr = (int64_t)b * R.y_sb[j] + (int64_t)hh * R.y_sh[j] + (int64_t)s * R.y_ss[j];
    const bool norm = R.w[j] != nullptr;
    float r = 1.f;
    if (norm) {
        double sum = 0.0;
        for (int i = lane; i < D; i += SSQ_WAVE) {
            const double x = (double)ssq_load_elem(R.x[j], R.dtype, xr + i);
            sum = __builtin_fma(x, x, sum);
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        r = rope_rstd(sum, D, t.eps);
    }
    const int rot = t.cos ? t.rot_dim : 0;
    const int64_t pos = rot ? rope_pos(t, b, s) : 0;
    auto raw = [&](int i) { return ssq_load_elem(R.x[j], R.dtype, xr + i); };
    auto wt = [&](int i) { return ssq_load_elem(R.w[j], t.w_dtype, i); };
    // both dims of a pair are read before either is written: rows may be rotated in place
    for (int i = lane; i < (rot >> 1); i += SSQ_WAVE) {
        const int d0 = t.interleaved ? 2 * i : i, d1 = t.interleaved ? 2 * i + 1 : i + (rot >> 1);
        const float y0 = rope_dim(t, pos, d0, norm, r, raw, wt), y1 = rope_dim(t, pos, d1, norm, r, raw, wt);
        rope_store(R.y[j], R.dtype, yr + d0, y0);
        rope_store(R.y[j], R.dtype, yr + d1, y1);
    }
    for (int i = rot + lane; i < D; i += SSQ_WAVE) {
        const float y = rope_dim(t, pos, i, norm, r, raw, wt);
        rope_store(R.y[j], R.dtype, yr + i, y);
    }
}

template <int DT, int HEADS>
int launch_units(const RopeParams& p, unsigned blocks, hipStream_t st) {
    if (p.r.w[0] || p.r.w[1])
        hipLaunchKernelGGL((k_rope_units<DT, true, HEADS>), dim3(blocks), dim3(kRopeThreads), 0, st, p);
    else
        hipLaunchKernelGGL((k_rope_units<DT, false, HEADS>), dim3(blocks), dim3(kRopeThreads), 0, st, p);
    return ssq_check_hip(hipGetLastError(), "k_rope_units launch");
}

// whether the unit kernel serves the rows: whole 16-byte pieces, a power of two of them per row
bool units_ok(const SsqRopeRows& r, int& lpr) {
    const int size = r.dtype == SSQ_F32 ? 4 : 2, V = 16 / size;
    const int rot = r.t.cos ? r.t.rot_dim : 0;
    if (r.head_dim % (2 * V) || rot % (2 * V)) return false;
    lpr = r.head_dim / (2 * V);
    if (lpr > SSQ_WAVE || (lpr & (lpr - 1))) return false;
    if (rot && ((uintptr_t)r.t.cos % 16 || (uintptr_t)r.t.sin % 16 || r.t.ld % 4)) return false;
    for (int j = 0; j < 2; ++j) {
        if (!r.heads[j]) continue;
        const int64_t st[6] = {r.x_sb[j], r.x_sh[j], r.x_ss[j], r.y_sb[j], r.y_sh[j], r.y_ss[j]};
        for (int64_t v : st)
            if (v % V) return false;
        if ((uintptr_t)r.x[j] % 16 || (uintptr_t)r.y[j] % 16) return false;
    }
    return true;
}

}  // namespace

int ssq_rope_check(const ssq_rope& t, int head_dim, bool norm) {
    if (t.cos) {
        SSQ_REQUIRE(t.sin && t.positions, "the rotation needs cos, sin and positions");
        SSQ_REQUIRE(t.rot_dim >= 2 && t.rot_dim % 2 == 0 && t.rot_dim <= head_dim,
                    "rot_dim must be even and in [2, head_dim], got %d", t.rot_dim);
        SSQ_REQUIRE(t.max_pos >= 1 && t.ld >= t.rot_dim / 2, "bad rotation table (max_pos %d, row stride %lld)", t.max_pos,
                    (long long)t.ld);
        SSQ_REQUIRE(t.interleaved == 0 || t.interleaved == 1, "interleaved must be 0 or 1");
    }
    if (norm) {
        SSQ_REQUIRE(t.w_dtype >= SSQ_F32 && t.w_dtype <= SSQ_F16, "bad norm weight dtype");
        SSQ_REQUIRE(t.eps >= 0.0, "eps must be >= 0");
    }
    return SSQ_OK;
}

int ssq_rope_run(const SsqRopeRows& r, hipStream_t st) {
    RopeParams p{};
    p.r = r;
    const int64_t tokens = (int64_t)r.batch * r.seq_len;
    const int H = r.heads[0] + r.heads[1];
    if (tokens == 0 || H == 0) return SSQ_OK;
    int lpr = 0;
    if (!units_ok(r, lpr)) {
        const int64_t blocks = (tokens * H + 3) / 4;
        SSQ_UNSUPPORTED(blocks <= 0x7fffffff, "too many rows");
        hipLaunchKernelGGL(k_rope_any, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, p);
        return ssq_check_hip(hipGetLastError(), "k_rope_any launch");
    }
    p.lpr = lpr;
    while ((1 << p.lpr_log) < lpr) ++p.lpr_log;
    // one head per lane while the rows leave lanes idle (latency is what counts there), else four
    const bool many = tokens * H * lpr >= (int64_t)ssq_device_cus() * 2048;
    p.groups = many ? (H + 3) / 4 : H;
    p.items = tokens * p.groups;
    const int64_t blocks = (p.items * lpr + kRopeThreads - 1) / kRopeThreads;
    SSQ_UNSUPPORTED(blocks <= 0x7fffffff, "too many rows");
    const unsigned n = (unsigned)blocks;
    if (r.dtype == SSQ_BF16) return many ? launch_units<SSQ_BF16, 4>(p, n, st) : launch_units<SSQ_BF16, 1>(p, n, st);
    if (r.dtype == SSQ_F16) return many ? launch_units<SSQ_F16, 4>(p, n, st) : launch_units<SSQ_F16, 1>(p, n, st);
    return many ? launch_units<SSQ_F32, 4>(p, n, st) : launch_units<SSQ_F32, 1>(p, n, st);
}

extern "C" int ssq_qk_norm_rope(const ssq_rope_args* a, void* stream) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_rope_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_rope_args size %u != library's %zu", a->struct_size, sizeof(ssq_rope_args));
    SSQ_REQUIRE(a->dtype >= SSQ_F32 && a->dtype <= SSQ_F16, "bad dtype");
    SSQ_REQUIRE(a->batch >= 0 && a->seq_len >= 0 && a->head_dim >= 1 && a->head_dim <= 1024, "bad batch/seq_len/head_dim");
    SSQ_REQUIRE(a->num_q_heads >= 1 && a->num_k_heads >= 0 && a->num_q_heads + (int64_t)a->num_k_heads <= 1 << 20,
                "bad head counts");
    SSQ_REQUIRE(a->q && a->q_out, "q and q_out must be non-NULL");
    SSQ_REQUIRE(a->num_k_heads == 0 || (a->k && a->k_out), "k and k_out must be non-NULL");
    int rc = ssq_rope_check(a->rope, a->head_dim, a->q_weight || (a->num_k_heads && a->k_weight));
    if (rc) return rc;
    SsqRopeRows r{};
    r.x[0] = a->q; r.y[0] = a->q_out; r.w[0] = a->q_weight; r.heads[0] = a->num_q_heads;
    r.x_sb[0] = a->q_sb; r.x_sh[0] = a->q_sh; r.x_ss[0] = a->q_ss;
    r.y_sb[0] = a->qo_sb; r.y_sh[0] = a->qo_sh; r.y_ss[0] = a->qo_ss;
    r.heads[1] = a->num_k_heads;
    if (a->num_k_heads) {
        r.x[1] = a->k; r.y[1] = a->k_out; r.w[1] = a->k_weight;
        r.x_sb[1] = a->k_sb; r.x_sh[1] = a->k_sh; r.x_ss[1] = a->k_ss;
        r.y_sb[1] = a->ko_sb; r.y_sh[1] = a->ko_sh; r.y_ss[1] = a->ko_ss;
    }
    r.batch = a->batch; r.seq_len = a->seq_len; r.head_dim = a->head_dim; r.dtype = a->dtype;
    r.t = a->rope;
    return ssq_rope_run(r, (hipStream_t)stream);
}
