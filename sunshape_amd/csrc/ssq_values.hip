// ssq_append_values: values to 8-bit pages (ssq_values.h).
#include "ssq_values.h"

int ssq_values_check(const ssq_values_args* a);
SsqValues ssq_values_params(const ssq_values_args& a);

namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads, 6) void k_append_values(const SsqValues p) {
    val_wave(p, (int64_t)blockIdx.x * (kThreads / SSQ_WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x / SSQ_WAVE),
             threadIdx.x & (SSQ_WAVE - 1));
}

}  // namespace

int ssq_values_check(const ssq_values_args* a) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_values_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_values_args size %u != library's %zu", a->struct_size, sizeof(ssq_values_args));
    SSQ_REQUIRE(a->v && a->v_pages && a->v_scale && a->slot_mapping, "v, v_pages, v_scale and slot_mapping must be non-NULL");
    SSQ_REQUIRE(a->v_dtype >= SSQ_F32 && a->v_dtype <= SSQ_F16, "bad v_dtype");
    SSQ_REQUIRE(a->batch >= 0 && a->seq_len >= 0 && a->num_kv_heads >= 1 && a->num_kv_heads <= 65535, "bad batch/heads/seq_len");
    SSQ_REQUIRE(a->value_dim >= 1 && a->value_dim <= 8192, "value_dim must be in [1, 8192]");
    SSQ_REQUIRE(a->page_size >= 16 && a->page_size % 16 == 0, "8-bit pages need a page_size that is a multiple of 16");
    SSQ_REQUIRE(a->num_pages >= 0 && a->num_pages <= 0x7fffffff, "bad num_pages");
    SSQ_REQUIRE((uintptr_t)a->v_pages % 16 == 0 && a->vp_sb % 16 == 0 && a->vp_sh % 16 == 0 && a->vp_sd % 16 == 0,
                "8-bit value rows must be 16-byte aligned");
    SSQ_REQUIRE((int64_t)a->batch * a->seq_len <= 0x7fffffff - 64, "too many rows");
    return SSQ_OK;
}

SsqValues ssq_values_params(const ssq_values_args& a) {
    SsqValues p{};
    p.v = a.v; p.v_dtype = a.v_dtype; p.v_sb = a.v_sb; p.v_sh = a.v_sh; p.v_ss = a.v_ss;
    p.batch = a.batch; p.heads = a.num_kv_heads; p.seq_len = a.seq_len; p.value_dim = a.value_dim;
    p.pages = reinterpret_cast<uint8_t*>(a.v_pages); p.vp_sb = a.vp_sb; p.vp_sh = a.vp_sh; p.vp_sd = a.vp_sd;
    p.scale = a.v_scale; p.vs_sb = a.vs_sb; p.vs_sh = a.vs_sh;
    p.slots = a.slot_mapping; p.sm_sb = a.sm_sb;
    p.n_slots = a.num_pages * a.page_size;
    p.page_size = a.page_size;
    p.page_log = -1;
    for (int l = 4; l < 31; ++l)
        if (a.page_size == 1 << l) p.page_log = l;
    const int pair = a.v_dtype == SSQ_F32 ? 8 : 4;
    p.vec = a.value_dim % 2 == 0 && (uintptr_t)a.v % pair == 0 && a.v_sb % 2 == 0 && a.v_sh % 2 == 0 && a.v_ss % 2 == 0;
    p.chunks = (a.seq_len + kRunChunk - 1) / kRunChunk;
    p.two = a.value_dim <= 64 && a.num_kv_heads > 1;
    p.hgroups = p.two ? (a.num_kv_heads + 1) / 2 : a.num_kv_heads;
    return p;
}

extern "C" int ssq_append_values(const ssq_values_args* a, void* stream) {
    int rc = ssq_values_check(a);
    if (rc) return rc;
    if (a->batch == 0 || a->seq_len == 0 || a->num_pages == 0) return SSQ_OK;
    const SsqValues p = ssq_values_params(*a);
    const int64_t waves = (int64_t)p.batch * p.chunks * p.hgroups, per = kThreads / SSQ_WAVE;
    SSQ_UNSUPPORTED((waves + per - 1) / per <= 0x7fffffff, "too many rows");
    hipLaunchKernelGGL(k_append_values, dim3((unsigned)((waves + per - 1) / per)), dim3(kThreads), 0, (hipStream_t)stream, p);
    return ssq_check_hip(hipGetLastError(), "k_append_values launch");
}
