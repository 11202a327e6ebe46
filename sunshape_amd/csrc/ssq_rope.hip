// Norm and rotation of queries and keys, one pass (ssq_qk_norm_rope; mathematics and the unit kernel's body in
// ssq_rope.h).
//
// Measured, one MI355X: 32,768 tokens of 32 + 8 heads of 128 dims, bf16 with norm: 131-134 us for 688 MB, 5.1-5.2 TB/s,
// a copy's rate; a step of 64 tokens 4.2 us, 7.5 with the call (latency of one chain: position, table, row).
#include "ssq_rope.h"

namespace {

template <int DT, bool NORM, int HEADS>
__global__ __launch_bounds__(kRopeThreads) void k_rope_units(const RopeParams p) {
    __shared__ __align__(16) float wl[rope_lds<DT, NORM>()];
    rope_units<DT, NORM, HEADS>(p, blockIdx.x, wl);
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
        r = rope_rstd(sum, p.inv_d, t.eps);
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

}  // namespace

bool ssq_rope_units_ok(const SsqRopeRows& r, int& lpr) {
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
    p.inv_d = 1.0 / (double)r.head_dim;
    const int64_t tokens = (int64_t)r.batch * r.seq_len;
    const int H = r.heads[0] + r.heads[1];
    if (tokens == 0 || H == 0) return SSQ_OK;
    int lpr = 0;
    if (!ssq_rope_units_ok(r, lpr)) {
        const int64_t blocks = (tokens * H + 3) / 4;
        SSQ_UNSUPPORTED(blocks <= 0x7fffffff, "too many rows");
        hipLaunchKernelGGL(k_rope_any, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, p);
        return ssq_check_hip(hipGetLastError(), "k_rope_any launch");
    }
    p.lpr = lpr;
    while ((1 << p.lpr_log) < lpr) ++p.lpr_log;
    // One head per lane while the rows leave lanes idle (latency is what counts there), else four, which read a token's
    // table entries once: 40 heads of 128 dims in bf16, us with one and with four: 64 tokens 3.6 and 6.0, 2,048 11.3
    // and 11.9, 4,096 19.9 and 20.1, 8,192 35.2 and 33.6; fp32, 512 6.3 and 7.5, 2,048 18.3 and 16.4
    const bool many = tokens * H * lpr >= (int64_t)ssq_device_cus() * 4096;
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
    SSQ_REQUIRE((int64_t)a->batch * a->seq_len <= 0x7fffffff, "too many tokens");
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
