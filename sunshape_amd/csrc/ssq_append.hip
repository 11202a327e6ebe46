// Append of raw keys and values to a paged cache (ssq_append): the keys' norm and rotation (ssq_rope.h), the
// nearest-codeword search (arithmetic in ssq_encode_math.h: the codes are those of ssq_encode over the
// rotated keys) and the values' transpose into dim-major pages.
//
// Few rows (a decode step): one launch, k_append_few.  A workgroup serves one block of some keys of a KV head:
// it rotates just that block's dims (and, with a norm, reads the whole row for its sum, from L2 after the first
// block), keeps the block's codebook in LDS and splits a key's scan over `slices` lanes.  Workgroups past
// the blocks copy the values.  One chain of loads bounds it, so everything whose address is known is asked for at once.
//
// Many rows: k_append_prep writes the pages' values and the rotated keys side by side, and ssq_encode, which is
// where the time goes, takes those.
#include "ssq_encode_math.h"
#include "ssq_rope.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kValTok = 64;    // tokens of a value tile, at most
constexpr int kValDims = 128;  // dims of a value tile
constexpr int kStageFloats = 10 * 1024;  // codebook floats (with norms) per LDS stage

struct AppendParams {
    ssq_encode_args e;
    ssq_rope t;
    const void* kw;
    int64_t n_slots;  // num_pages * page_size
    const void* v;
    void* vp;
    int64_t v_sb, v_sh, v_ss, vp_sb, vp_sh, vp_sd;
    int v_dtype, vp_dtype, value_dim;
    int slices;    // lanes per (key, block)
    int chunk;     // codewords per LDS stage
    int row_vec;   // key rows load as 16-byte pieces
    int dchunks;   // value dims in chunks of kValDims
    int vtok;      // tokens of a value tile: 64, or 16 where there are few
    int v_vec;     // value rows load as 16-byte pieces
    int vp_vec;    // pages take 16-byte stores of 8 (16-bit) or 4 (32-bit) tokens
    int64_t* slots_out;  // sanitized slots (many rows) or NULL
};

__device__ __forceinline__ int64_t slot_of(const AppendParams& p, int i) {  // -1: nothing is written
    const int b = i / p.e.seq_len, s = i - b * p.e.seq_len;
    const int64_t slot = p.e.slot_mapping[(int64_t)b * p.e.sm_sb + s];
    return slot >= 0 && slot < p.n_slots ? slot : -1;
}

// LDS of a value tile: raw elements of the page dtype, one padding dword per row
__host__ __device__ constexpr int val_row(int size) { return kValDims * size + 4; }

// where a token's values go in its head's pages, and its slot within the page (-1: nowhere)
struct ValSlots {
    int64_t base[kValTok];
    int off[kValTok];
};

// Tokens [vtok tile, +vtok) (flat over the batch), dims [128 dc, +128) of one KV head: rows in, pages out.  A
// page holds a dim's tokens side by side, so a run of tokens in consecutive slots of a page that starts on
// an 8-slot boundary leaves as whole 16-byte pieces; any other token by itself.
__device__ __forceinline__ void value_tile(const AppendParams& p, unsigned char* lds, ValSlots& vs, int tile, int kv, int dc) {
    const ssq_encode_args& a = p.e;
    const int tid = threadIdx.x;
    const int n = a.batch * a.seq_len;
    const int i0 = tile * p.vtok, nt = min(p.vtok, n - i0);
    const int d0 = dc * kValDims, nd = min(kValDims, p.value_dim - d0);
    const int size = p.vp_dtype == SSQ_F32 ? 4 : 2;
    const int row = val_row(size);
    const int page = a.page_size;
    if (tid < kValTok) {
        const int64_t slot = tid < nt ? slot_of(p, i0 + tid) : -1;
        const int64_t pg = slot / page;
        vs.off[tid] = slot < 0 ? -1 : (int)(slot - pg * page);
        vs.base[tid] = slot < 0 ? 0 : pg * p.vp_sb + (int64_t)kv * p.vp_sh + (int64_t)d0 * p.vp_sd + (slot - pg * page);
        if (p.slots_out && kv == 0 && dc == 0 && tid < nt) p.slots_out[i0 + tid] = slot;
    }
    if (!p.v) return;  // the whole workgroup
    auto vrow = [&](int t) {
        const int i = i0 + t, b = i / a.seq_len, s = i - b * a.seq_len;
        return (int64_t)b * p.v_sb + (int64_t)kv * p.v_sh + (int64_t)s * p.v_ss + d0;
    };
    if (p.v_vec) {  // same 16-bit dtype: pieces of 8
        const int pieces = nd >> 3;
        for (int e = tid; e < nt * pieces; e += kThreads) {
            const int t = e / pieces, q = e - t * pieces;
            const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.v) + vrow(t) + 8 * q);
            uint32_t* dst = reinterpret_cast<uint32_t*>(lds + t * row + 16 * q);  // rows are 4-byte aligned
            dst[0] = w.x; dst[1] = w.y; dst[2] = w.z; dst[3] = w.w;
        }
    } else {
        for (int e = tid; e < nt * nd; e += kThreads) {
            const int t = e / nd, d = e - t * nd;
            unsigned char* dst = lds + t * row + d * size;
            if (p.v_dtype == p.vp_dtype) {
                if (size == 4) *reinterpret_cast<uint32_t*>(dst) = reinterpret_cast<const uint32_t*>(p.v)[vrow(t) + d];
                else *reinterpret_cast<uint16_t*>(dst) = reinterpret_cast<const uint16_t*>(p.v)[vrow(t) + d];
            } else {
                rope_store(dst, p.vp_dtype, 0, ssq_load_elem(p.v, p.v_dtype, vrow(t) + d));
            }
        }
    }
    __syncthreads();
    // groups of 8 tokens, cut so that the first token's run meets 8-slot boundaries
    const int lead = vs.off[0] < 0 ? 0 : vs.off[0] & 7;
    const int groups = (nt + lead + 7) >> 3;
    // lanes: the group's parity fastest (both halves of a 16-token page), then dims
    for (int e = tid; e < groups * nd; e += kThreads) {
        const int pair = e / (2 * nd), rest = e - pair * 2 * nd;
        const bool odd = 2 * pair + 1 >= groups;  // the group without a partner
        const int g = odd ? 2 * pair : 2 * pair + (rest & 1), d = odd ? rest : rest >> 1;
        const int ta = max(8 * g - lead, 0), tb = min(8 * g - lead + 8, nt);
        const int64_t dd = (int64_t)d * p.vp_sd;
        bool whole = p.vp_vec && tb - ta == 8 && vs.off[ta] >= 0 && (vs.off[ta] & 7) == 0;
        if (whole) {  // one page: its size is a multiple of 8
            const int64_t b0 = vs.base[ta];
#pragma unroll
            for (int k = 1; k < 8; ++k) whole = whole && vs.off[ta + k] == vs.off[ta] + k && vs.base[ta + k] == b0 + k;
        }
        if (whole) {
            const int64_t at = vs.base[ta] + dd;
            if (size == 2) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = *reinterpret_cast<const uint16_t*>(lds + (ta + 2 * k) * row + 2 * d) |
                           ((uint32_t)*reinterpret_cast<const uint16_t*>(lds + (ta + 2 * k + 1) * row + 2 * d) << 16);
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.vp) + at) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = *reinterpret_cast<const uint32_t*>(lds + (ta + k) * row + 4 * d);
                uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p.vp) + at);
                dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
                dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            continue;
        }
        for (int t = ta; t < tb; ++t) {
            if (vs.off[t] < 0) continue;
            const int64_t at = vs.base[t] + dd;
            if (size == 2) reinterpret_cast<uint16_t*>(p.vp)[at] = *reinterpret_cast<const uint16_t*>(lds + t * row + 2 * d);
            else reinterpret_cast<uint32_t*>(p.vp)[at] = *reinterpret_cast<const uint32_t*>(lds + t * row + 4 * d);
        }
    }
}

// Many rows: workgroups [0, rope_blocks) rotate the keys, the others write the values (and, for kv 0 and the first
// dims, the sanitized slots).  They share nothing; one launch lets the values' transposes run beside the rotation.
template <int DT, bool NORM>
__global__ __launch_bounds__(kThreads) void k_append_prep(const AppendParams p, const RopeParams rp, int rope_blocks, int tiles) {
    constexpr int kLds = kValTok * val_row(4) > rope_lds<DT, NORM>() * 4 ? kValTok * val_row(4) : rope_lds<DT, NORM>() * 4;
    __shared__ __align__(16) unsigned char lds[kLds];
    __shared__ ValSlots vs;
    static_assert(kThreads == kRopeThreads, "one block size");
    if ((int)blockIdx.x < rope_blocks) {
        rope_units<DT, NORM, 4>(rp, blockIdx.x, reinterpret_cast<float*>(lds));
        return;
    }
    const int e = blockIdx.x - rope_blocks, dk = e / tiles;  // tiles of a KV head side by side
    value_tile(p, lds, vs, e - dk * tiles, dk % p.e.num_kv_heads, dk / p.e.num_kv_heads);
}

// BD: the block dim at compile time (1, 2, 4 or 8), or 0 for any other up to 16.  x: keys (or value tiles),
// y: KV heads, z: blocks, then value dims.
template <int BD>
__global__ __launch_bounds__(kThreads) void k_append_few(const AppendParams p) {
    constexpr int kX = BD ? BD : 16;
    extern __shared__ __align__(16) unsigned char few_lds[];
    unsigned char* lds = few_lds;
    const ssq_encode_args& a = p.e;
    const int kv = blockIdx.y, blk = blockIdx.z;
    const int n = a.batch * a.seq_len;
    if (blk >= a.n_blocks) {
        __shared__ ValSlots vs;
        if ((int)blockIdx.x * p.vtok < n) value_tile(p, lds, vs, blockIdx.x, kv, blk - a.n_blocks);
        return;
    }
    const int S = p.slices, sl = threadIdx.x & (S - 1);
    const int k0 = blockIdx.x * (kThreads / S);
    if (k0 >= n) return;  // the whole workgroup
    const int i = k0 + (int)(threadIdx.x / S);
    const bool live = i < n;
    const int bd = BD ? BD : a.block_dim, nc = a.n_centroids, D = a.head_dim;
    const int cw = ssq_code_width(nc);
    const bool heavy = ssq_is_heavy(a.heavy_mask[0], a.heavy_mask[1], blk);
    const float* met = a.metric ? a.metric + (int64_t)kv * a.metric_sh + (int64_t)blk * bd * D + blk * bd : nullptr;
    const int64_t* perm = a.perm + (int64_t)kv * a.perm_sh + (int64_t)blk * bd;
    const int ii = live ? i : n - 1;
    const int b = ii / a.seq_len, s = ii - b * a.seq_len;
    const int64_t slot = slot_of(p, ii);
    const int64_t krow = (int64_t)b * a.k_sb + (int64_t)kv * a.k_sh + (int64_t)s * a.k_ss;
    // the block's dims, their partners, weights and table entries (dims are the same for the whole workgroup)
    const bool norm = p.kw != nullptr, turn = p.t.cos != nullptr;
    const int half = p.t.rot_dim >> 1;
    bool rot[kX], first[kX];
    int64_t at[2 * kX], wat[2 * kX];
    int ti[kX];
#pragma unroll
    for (int d = 0; d < kX; ++d) {
        const int dim = d < bd ? (int)min((uint64_t)perm[d], (uint64_t)(D - 1)) : 0;
        rot[d] = turn && dim < p.t.rot_dim;
        first[d] = p.t.interleaved ? !(dim & 1) : dim < half;
        const int other = !rot[d] ? dim : p.t.interleaved ? dim ^ 1 : first[d] ? dim + half : dim - half;
        ti[d] = !rot[d] ? 0 : p.t.interleaved ? dim >> 1 : first[d] ? dim : dim - half;
        at[d] = krow + dim;
        at[kX + d] = krow + other;
        wat[d] = dim;
        wat[kX + d] = other;
    }
    float xr[2 * kX], wv[2 * kX], cv[kX], sv[kX];
    ssq_load_elems<2 * kX>(a.keys, a.k_dtype, at, xr);
    const int64_t pos = turn ? rope_pos(p.t, b, s) : 0;
    if (turn) {  // uniform
        const int64_t trow = (pos < 0 ? 0 : pos) * p.t.ld;
#pragma unroll
        for (int d = 0; d < kX; ++d) {
            cv[d] = p.t.cos[trow + ti[d]];
            sv[d] = p.t.sin[trow + ti[d]];
        }
    }
    float r = 1.f;
    if (norm) {  // the key's S lanes share the row's sum
        ssq_load_elems<2 * kX>(p.kw, p.t.w_dtype, wat, wv);
        double sum = 0.0;
        if (p.row_vec) {
            const int per = a.k_dtype == SSQ_F32 ? 4 : 8;
            const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(a.keys) + krow * (16 / per));
            for (int q = sl; q < D / per; q += S) {
                const uint4 w = src[q];
                if (a.k_dtype == SSQ_F32) {
                    float x[4];
                    rope_unpack<SSQ_F32>(w, x);
#pragma unroll
                    for (int k = 0; k < 4; ++k) sum = __builtin_fma((double)x[k], (double)x[k], sum);
                } else {
                    float x[8];
                    if (a.k_dtype == SSQ_BF16) rope_unpack<SSQ_BF16>(w, x);
                    else rope_unpack<SSQ_F16>(w, x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum = __builtin_fma((double)x[k], (double)x[k], sum);
                }
            }
        } else {
            for (int q = sl; q < D; q += S) {
                const double x = (double)ssq_load_elem(a.keys, a.k_dtype, krow + q);
                sum = __builtin_fma(x, x, sum);
            }
        }
        for (int o = S >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        r = rope_rstd(sum, D, p.t.eps);
    }
    float x[kX];
#pragma unroll
    for (int d = 0; d < kX; ++d) {  // as rope_dim
        float u = norm ? (xr[d] * r) * wv[d] : xr[d];
        if (rot[d]) {
            const float v = norm ? (xr[kX + d] * r) * wv[kX + d] : xr[kX + d];
            const float c = pos < 0 ? __builtin_nanf("") : cv[d], sn = pos < 0 ? __builtin_nanf("") : sv[d];
            const float y = u * c, z = v * sn;
            u = first[d] ? y - z : y + z;
        }
        x[d] = norm || turn ? rope_round(u, a.k_dtype) : u;
    }
    int64_t crow = 0, prow = 0;
    if (slot >= 0) {
        const int64_t page = slot / a.page_size, off = slot - page * a.page_size;
        crow = page * a.c_sb + (int64_t)kv * a.c_sh + off * a.c_st;
        prow = page * a.pt_sb + (int64_t)kv * a.pt_sh + off * a.pt_st;
    }
    const bool put = live && slot >= 0 && sl == 0;
    if (heavy) {  // the whole workgroup: code 0, values kept
        if (put) {
            store_code(a.codes, cw, crow + blk, 0u);
            const int ps = a.pt_dense ? blk : heavy_ordinal(a.heavy_mask[0], a.heavy_mask[1], blk);
#pragma unroll
            for (int d = 0; d < kX; ++d)
                if (d < bd) rope_store(a.pt, a.pt_dtype, prow + (int64_t)ps * bd + d, x[d]);
        }
        return;
    }
    auto map = [&](float (&c)[kX]) {  // into the metric space
        float y[kX];
#pragma unroll
        for (int k = 0; k < kX; ++k)
            if (k < bd) y[k] = metric_row(met + (int64_t)k * D, c, bd);
#pragma unroll
        for (int k = 0; k < kX; ++k)
            if (k < bd) c[k] = y[k];
    };
    if (met) map(x);
    const float xn = sq_norm(x, bd);
    const bool direct = a.direct_dist != 0;
    float* cb = reinterpret_cast<float*>(lds);  // [chunk][bd]
    float* cn = cb + (size_t)p.chunk * bd;      // [chunk]
    const float* cent = a.cent + (int64_t)kv * a.cent_sh + (int64_t)blk * nc * bd;
    float e_min = INFINITY;
    uint32_t j_best = 0;
    for (int j0 = 0; j0 < nc; j0 += p.chunk) {
        const int m = min(p.chunk, nc - j0);
        __syncthreads();  // the previous stage's reads are done
        for (int e = threadIdx.x; e < m; e += kThreads) {
            float c[kX];
#pragma unroll
            for (int d = 0; d < kX; ++d)
                if (d < bd) c[d] = cent[(int64_t)(j0 + e) * bd + d];
            if (met) map(c);
#pragma unroll
            for (int d = 0; d < kX; ++d)
                if (d < bd) cb[(size_t)e * bd + d] = c[d];
            cn[e] = sq_norm(c, bd);
        }
        __syncthreads();
        if (direct) {
            for (int j = sl; j < m; j += S) take_min(direct_dist2(x, cb + (size_t)j * bd, bd), (uint32_t)(j0 + j), e_min, j_best);
        } else {
            int j = sl;
            for (; j + 3 * S < m; j += 4 * S) {  // four codewords' LDS reads in flight
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = mm_dist2(x, xn, cb + (size_t)(j + u * S) * bd, cn[j + u * S], bd);
#pragma unroll
                for (int u = 0; u < 4; ++u) take_min(v[u], (uint32_t)(j0 + j + u * S), e_min, j_best);
            }
            for (; j < m; j += S) take_min(mm_dist2(x, xn, cb + (size_t)j * bd, cn[j], bd), (uint32_t)(j0 + j), e_min, j_best);
        }
    }
    // the key's lanes: the smaller distance, then the smaller index
    float f_best = __builtin_sqrtf(e_min);
    for (int o = S >> 1; o > 0; o >>= 1) {
        const float of = __shfl_xor(f_best, o);
        const uint32_t oj = (uint32_t)__shfl_xor((int)j_best, o);
        if (of < f_best || (of == f_best && oj < j_best)) {
            f_best = of;
            j_best = oj;
        }
    }
    if (put) store_code(a.codes, cw, crow + blk, j_best);
}

int check(const ssq_append_args* a) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_append_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_append_args size %u != library's %zu", a->struct_size, sizeof(ssq_append_args));
    const ssq_encode_args& e = a->enc;
    if (e.struct_size != sizeof(ssq_encode_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_encode_args size %u != library's %zu", e.struct_size, sizeof(ssq_encode_args));
    SSQ_REQUIRE(e.keys && e.perm && e.cent && e.codes, "keys, perm, cent and codes must be non-NULL");
    SSQ_REQUIRE(e.slot_mapping && e.page_size >= 1, "append needs a slot_mapping and page_size >= 1");
    SSQ_REQUIRE(a->num_pages >= 0 && a->num_pages <= INT64_MAX / e.page_size, "bad num_pages");
    SSQ_REQUIRE(e.batch >= 0 && e.num_kv_heads >= 1 && e.num_kv_heads <= 65535 && e.seq_len >= 0, "bad batch/heads/seq_len");
    SSQ_REQUIRE((int64_t)e.batch * e.seq_len <= 0x7fffffff - kThreads, "too many rows");
    SSQ_REQUIRE(e.k_dtype >= SSQ_F32 && e.k_dtype <= SSQ_F16, "bad k_dtype");
    SSQ_REQUIRE(e.head_dim >= 1 && e.head_dim <= 1024, "head_dim must be in [1, 1024]");
    SSQ_REQUIRE(e.block_dim >= 1 && e.block_dim <= 16 && e.head_dim % e.block_dim == 0,
                "head_dim must be divisible by block_dim (block_dim <= 16)");
    SSQ_REQUIRE(e.n_blocks == e.head_dim / e.block_dim && e.n_blocks <= 128, "bad n_blocks");
    SSQ_REQUIRE(e.n_centroids >= 1 && e.n_centroids <= kMaxCentroids, "n_centroids must be in [1, %d]", kMaxCentroids);
    if (e.n_centroids > 256) {
        const int cw = ssq_code_width(e.n_centroids);
        SSQ_REQUIRE((uintptr_t)e.codes % cw == 0, "%d-bit codes must be %d-byte aligned", 8 * cw, cw);
    }
    const bool any_heavy = e.heavy_mask[0] || e.heavy_mask[1];
    SSQ_REQUIRE(!any_heavy || e.pt, "heavy blocks need a passthrough output");
    if (any_heavy) SSQ_REQUIRE(e.pt_dtype >= SSQ_F32 && e.pt_dtype <= SSQ_F16, "bad pt_dtype");
    SSQ_REQUIRE(e.direct_dist == 0 || e.direct_dist == 1, "direct_dist must be 0 or 1");
    // 2 and 3 serve some codebooks only; a refusal by ssq_encode would come after the values are written
    SSQ_UNSUPPORTED(e.kernel == 0 || e.kernel == 1, "append takes kernel 0, or 1 for the exact scan, not %d", e.kernel);
    int rc = ssq_rope_check(a->rope, e.head_dim, a->k_weight != nullptr);
    if (rc) return rc;
    if (a->v) {
        SSQ_REQUIRE(a->v_pages, "values need v_pages");
        SSQ_REQUIRE(a->v_dtype >= SSQ_F32 && a->v_dtype <= SSQ_F16 && a->vp_dtype >= SSQ_F32 && a->vp_dtype <= SSQ_F16,
                    "bad value dtype");
        SSQ_REQUIRE(a->value_dim >= 1 && a->value_dim <= 8192, "value_dim must be in [1, 8192]");
    }
    return SSQ_OK;
}

// One launch up to about 2^26 (key, block, codeword) triples.
constexpr int64_t kFewWork = (int64_t)1 << 26;
bool few(const ssq_append_args& a) {
    const ssq_encode_args& e = a.enc;
    if (e.kernel != 0) return false;
    const int64_t rows = (int64_t)e.batch * e.seq_len * e.num_kv_heads * e.n_blocks;
    return rows <= kFewWork && rows * e.n_centroids <= kFewWork;
}

bool turns(const ssq_append_args& a) { return a.k_weight || a.rope.cos; }

int64_t rows_bytes(const ssq_append_args& a) {
    const ssq_encode_args& e = a.enc;
    const int64_t n = (int64_t)e.batch * e.seq_len * e.num_kv_heads * e.head_dim * (e.k_dtype == SSQ_F32 ? 4 : 2);
    return turns(a) ? (n + 255) & ~(int64_t)255 : 0;
}

AppendParams params(const ssq_append_args& a) {
    AppendParams p{};
    p.e = a.enc;
    p.t = a.rope;
    if (!p.t.cos) p.t.rot_dim = 0;
    p.kw = a.k_weight;
    p.n_slots = a.num_pages * a.enc.page_size;
    p.v = a.v;
    p.vp = a.v_pages;
    p.v_sb = a.v_sb; p.v_sh = a.v_sh; p.v_ss = a.v_ss;
    p.vp_sb = a.vp_sb; p.vp_sh = a.vp_sh; p.vp_sd = a.vp_sd;
    p.v_dtype = a.v_dtype; p.vp_dtype = a.vp_dtype; p.value_dim = a.v ? a.value_dim : 0;
    p.dchunks = (p.value_dim + kValDims - 1) / kValDims;
    const ssq_encode_args& e = a.enc;
    const int per = e.k_dtype == SSQ_F32 ? 4 : 8;
    p.row_vec = (uintptr_t)e.keys % 16 == 0 && e.head_dim % per == 0 && e.k_sb % per == 0 && e.k_sh % per == 0 && e.k_ss % per == 0;
    p.vtok = (int64_t)a.enc.batch * a.enc.seq_len > 1024 ? kValTok : 16;
    p.v_vec = a.v && a.v_dtype == a.vp_dtype && a.v_dtype != SSQ_F32 && (uintptr_t)a.v % 16 == 0 && a.value_dim % 8 == 0 &&
              a.v_sb % 8 == 0 && a.v_sh % 8 == 0 && a.v_ss % 8 == 0;
    const int vper = a.vp_dtype == SSQ_F32 ? 4 : 8;
    p.vp_vec = a.v && (uintptr_t)a.v_pages % 16 == 0 && e.page_size % 8 == 0 && a.vp_sb % vper == 0 && a.vp_sh % vper == 0 &&
               a.vp_sd % vper == 0;
    return p;
}

// the values and the sanitized slots, and the keys' rotation beside them where its unit kernel serves them
int run_prep(const AppendParams& p, const SsqRopeRows& r, bool turn, unsigned vtiles, hipStream_t st) {
    RopeParams rp{};
    rp.r = r;
    int lpr = 0;
    int64_t rope_blocks = 0;
    const bool units = turn && ssq_rope_units_ok(r, lpr);
    if (units) {
        rp.lpr = lpr;
        while ((1 << rp.lpr_log) < lpr) ++rp.lpr_log;
        rp.groups = (r.heads[0] + 3) / 4;
        rp.items = (int64_t)r.batch * r.seq_len * rp.groups;
        rope_blocks = (rp.items * lpr + kThreads - 1) / kThreads;
    } else if (turn) {
        int rc = ssq_rope_run(r, st);
        if (rc) return rc;
    }
    const int64_t blocks = rope_blocks + (int64_t)vtiles * p.e.num_kv_heads * (p.dchunks ? p.dchunks : 1);
    SSQ_UNSUPPORTED(blocks <= 0x7fffffff, "too many rows");
    const dim3 grid((unsigned)blocks), block(kThreads);
    const int rb = (int)rope_blocks, vt = (int)vtiles;
    const bool norm = units && r.w[0];
    if (!units || r.dtype == SSQ_BF16) {
        if (norm) hipLaunchKernelGGL((k_append_prep<SSQ_BF16, true>), grid, block, 0, st, p, rp, rb, vt);
        else hipLaunchKernelGGL((k_append_prep<SSQ_BF16, false>), grid, block, 0, st, p, rp, rb, vt);
    } else if (r.dtype == SSQ_F16) {
        if (norm) hipLaunchKernelGGL((k_append_prep<SSQ_F16, true>), grid, block, 0, st, p, rp, rb, vt);
        else hipLaunchKernelGGL((k_append_prep<SSQ_F16, false>), grid, block, 0, st, p, rp, rb, vt);
    } else {
        if (norm) hipLaunchKernelGGL((k_append_prep<SSQ_F32, true>), grid, block, 0, st, p, rp, rb, vt);
        else hipLaunchKernelGGL((k_append_prep<SSQ_F32, false>), grid, block, 0, st, p, rp, rb, vt);
    }
    return ssq_check_hip(hipGetLastError(), "k_append_prep launch");
}

}  // namespace

extern "C" size_t ssq_append_workspace_size(const ssq_append_args* a) {
    if (check(a) != SSQ_OK || few(*a)) return 0;
    return (size_t)(rows_bytes(*a) + (int64_t)a->enc.batch * a->enc.seq_len * 8);
}

extern "C" int ssq_append(const ssq_append_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc) return rc;
    const ssq_encode_args& e = a->enc;
    const int64_t n = (int64_t)e.batch * e.seq_len;
    if (n == 0) return SSQ_OK;
    hipStream_t st = (hipStream_t)stream;
    AppendParams p = params(*a);
    const unsigned vtiles = (unsigned)((n + p.vtok - 1) / p.vtok);
    if (few(*a)) {
        // lanes per key: enough to fill the device, at least 16 codewords each
        const int64_t units = n * e.num_kv_heads * e.n_blocks;
        p.slices = 8;
        while (p.slices < 64 && units * p.slices < (int64_t)ssq_device_cus() * 1024 && p.slices * 16 <= e.n_centroids) p.slices *= 2;
        const int stage = kStageFloats / (e.block_dim + 1);
        p.chunk = e.n_centroids < stage ? e.n_centroids : stage;
        const int per = kThreads / p.slices;
        const unsigned ktiles = (unsigned)((n + per - 1) / per);
        dim3 grid(ktiles > vtiles ? ktiles : vtiles, e.num_kv_heads, e.n_blocks + p.dchunks);
        size_t lds = (size_t)p.chunk * (e.block_dim + 1) * 4;
        const size_t vlds = a->v ? (size_t)p.vtok * val_row(a->vp_dtype == SSQ_F32 ? 4 : 2) : 0;
        if (vlds > lds) lds = vlds;
        switch (e.block_dim) {
            case 1: hipLaunchKernelGGL(k_append_few<1>, grid, dim3(kThreads), lds, st, p); break;
            case 2: hipLaunchKernelGGL(k_append_few<2>, grid, dim3(kThreads), lds, st, p); break;
            case 4: hipLaunchKernelGGL(k_append_few<4>, grid, dim3(kThreads), lds, st, p); break;
            case 8: hipLaunchKernelGGL(k_append_few<8>, grid, dim3(kThreads), lds, st, p); break;
            default: hipLaunchKernelGGL(k_append_few<0>, grid, dim3(kThreads), lds, st, p); break;
        }
        return ssq_check_hip(hipGetLastError(), "k_append_few launch");
    }
    const int64_t rows = rows_bytes(*a);
    SSQ_REQUIRE(workspace && workspace_bytes >= (size_t)(rows + n * 8), "workspace too small: %zu < %lld bytes", workspace_bytes,
                (long long)(rows + n * 8));
    SSQ_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
    p.slots_out = reinterpret_cast<int64_t*>(reinterpret_cast<char*>(workspace) + rows);
    ssq_encode_args enc = e;
    enc.slot_mapping = p.slots_out;
    enc.sm_sb = e.seq_len;
    SsqRopeRows r{};
    if (turns(*a)) {
        r.x[0] = e.keys; r.y[0] = workspace; r.w[0] = a->k_weight; r.heads[0] = e.num_kv_heads;
        r.x_sb[0] = e.k_sb; r.x_sh[0] = e.k_sh; r.x_ss[0] = e.k_ss;
        // token-major, as projections come
        r.y_ss[0] = (int64_t)e.num_kv_heads * e.head_dim;
        r.y_sh[0] = e.head_dim;
        r.y_sb[0] = r.y_ss[0] * e.seq_len;
        r.batch = e.batch; r.seq_len = e.seq_len; r.head_dim = e.head_dim; r.dtype = e.k_dtype;
        r.t = a->rope;
        enc.keys = workspace;
        enc.k_sb = r.y_sb[0]; enc.k_sh = r.y_sh[0]; enc.k_ss = r.y_ss[0];
    }
    rc = run_prep(p, r, turns(*a), vtiles, st);
    if (rc) return rc;
    return ssq_encode(&enc, stream);
}
