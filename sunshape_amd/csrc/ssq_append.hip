// Append of raw keys and values to a paged cache (ssq_append): the keys' norm and rotation (ssq_rope.h), the
// nearest-codeword search (arithmetic in ssq_encode_math.h: the codes are those of ssq_encode over the
// rotated keys) and the values' transpose into dim-major pages.
//
// Few rows (a decode step): one launch, k_append_few.  A workgroup serves one block of some keys of a KV head:
// it rotates just that block's dims, keeps the block's codebook in LDS and splits a key's scan over 4 to 64
// lanes.  The first workgroups write the values.  Loads that wait for one another bound it, so the keys' whole
// rows (which the norm needs anyhow), the codebook, the permutation, slots and positions are all asked for at once,
// and only the table's and weights' entries after them.  64 sequences' step (8 heads of 128 dims, 256 codewords of dim
// 4, norm and rotation, values): 9.3 us in a trace (8.2 a call among others, whose launches overlap), of which 1.0 the
// values, 1.1 the norm, 0.9 the rotation, 2 the scan's vector instructions and about 4 the launch and the first loads.  With
// 8-bit values (k_append_few8, the first workgroups as in ssq_values.h) 7.0 a call; 11.6 as two launches.
//
// Many rows: k_append_prep writes the pages' values and the rotated keys side by side, and ssq_encode, which is
// where the time goes, takes those.  8,192 tokens of the same layer: 19.8 us for 67 MB (3.4 TB/s) and 61.5 us.
#include "ssq_encode_math.h"
#include "ssq_rope.h"
#include "ssq_values.h"

#include <math.h>

int ssq_values_check(const ssq_values_args* a);
SsqValues ssq_values_params(const ssq_values_args& a);

namespace {

constexpr int kThreads = 256;
constexpr int kValTok = 16;    // tokens of a value tile
constexpr int kOneTok = 4;     // tokens of a workgroup where they go one by one
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
    int chunk;     // codewords per LDS stage
    int row_vec;   // key rows load as 16-byte pieces
    int dchunks;   // value dims in chunks of kValDims
    int vone;      // value tokens one by one
    int vseq;      // value tiles per sequence
    int vtiles;    // value tiles
    int ktiles;    // workgroups per block and KV head (few rows)
    int krow;      // LDS bytes of a key row (few rows)
    int page_log;  // log2 of the page size, or -1
    double inv_d;  // 1 / head_dim
    int v_vec;     // value rows load as 16-byte pieces
    int vp_vec;    // pages take 16-byte stores of 8 (16-bit) or 4 (32-bit) tokens
    int64_t* slots_out;  // sanitized slots (many rows) or NULL
};

__device__ __forceinline__ int64_t slot_of(const AppendParams& p, int b, int s) {  // -1: nothing is written
    const int64_t slot = p.e.slot_mapping[(int64_t)b * p.e.sm_sb + s];
    return slot >= 0 && slot < p.n_slots ? slot : -1;
}

// slot = page * page_size + off
__device__ __forceinline__ void split_slot(const AppendParams& p, int64_t slot, int64_t& page, int& off) {
    const int size = p.e.page_size;
    if (p.page_log >= 0) {
        page = slot >> p.page_log;
        off = (int)slot & (size - 1);
    } else if ((uint64_t)slot >> 32 == 0) {
        const uint32_t q = (uint32_t)slot / (uint32_t)size;
        page = q;
        off = (int)((uint32_t)slot - q * (uint32_t)size);
    } else {
        page = slot / size;
        off = (int)(slot - page * size);
    }
}

// token i of the batch, [B, S] flat
__device__ __forceinline__ void split_token(const AppendParams& p, int i, int& b, int& s) {
    b = p.e.seq_len == 1 ? i : i / p.e.seq_len;
    s = i - b * p.e.seq_len;
}

// LDS row of a value tile: raw elements of the page dtype and 16 bytes, which puts the two groups of 8 tokens on
// other banks
__host__ __device__ constexpr int val_row(int size) { return kValDims * size + 16; }
constexpr int kValLds = kValTok * val_row(4);

// where a token's values go in its head's pages, and its slot within the page (-1: nowhere)
struct ValSlots {
    int64_t base[kValTok];
    int off[kValTok];
};

// Up to 16 tokens of a sequence, dims [128 dc, +128) of one KV head: rows in, pages out.  A page holds a dim's tokens
// side by side, so 8 tokens in consecutive slots of a page from an 8-slot boundary leave as one 16-byte piece, any
// other token by itself.  Tiles begin where the sequence's first slot, counted on, is a multiple of 16:
// a prompt into whole pages then has pieces only, and two lanes fill a 16-token page's 32 bytes of a dim.
// One load and one store a lane, and many small workgroups to cover the slots' latency: 1,024 tokens' keys and values
// (8 heads of 128 dims) took 7.5 us by tiles of 64 tokens and take 6.4.
__device__ __forceinline__ void value_tile(const AppendParams& p, unsigned char* lds, ValSlots& vs, int tile, int kv, int dc) {
    const ssq_encode_args& a = p.e;
    const int tid = threadIdx.x;
    const int b = tile / p.vseq, end = (tile - b * p.vseq + 1) * kValTok;
    const int64_t first = slot_of(p, b, 0);
    const int s1 = end - (first < 0 ? 0 : (int)first & (kValTok - 1)), s0 = max(s1 - kValTok, 0);
    const int nt = min(s1, a.seq_len) - s0;
    if (nt <= 0) return;  // the whole workgroup
    const int d0 = dc * kValDims, nd = min(kValDims, p.value_dim - d0);
    const int size = p.vp_dtype == SSQ_F32 ? 4 : 2;
    const int row = val_row(size);
    if (tid < nt) {
        const int64_t slot = slot_of(p, b, s0 + tid);
        int64_t pg;
        int off;
        split_slot(p, slot < 0 ? 0 : slot, pg, off);
        vs.off[tid] = slot < 0 ? -1 : off;
        vs.base[tid] = slot < 0 ? 0 : pg * p.vp_sb + (int64_t)kv * p.vp_sh + (int64_t)d0 * p.vp_sd + off;
        if (p.slots_out && kv == 0 && dc == 0) p.slots_out[(int64_t)b * a.seq_len + s0 + tid] = slot;
    }
    if (!p.v) return;  // the whole workgroup
    const int64_t vrow = (int64_t)b * p.v_sb + (int64_t)kv * p.v_sh + (int64_t)s0 * p.v_ss + d0;
    if (p.v_vec) {  // same 16-bit dtype: pieces of 8
        const int pieces = nd >> 3;
        for (int e = tid; e < nt * pieces; e += kThreads) {
            const int t = e / pieces, q = e - t * pieces;
            *reinterpret_cast<uint4*>(lds + t * row + 16 * q) =
                *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.v) + vrow + (int64_t)t * p.v_ss + 8 * q);
        }
    } else {
        for (int e = tid; e < nt * nd; e += kThreads) {
            const int t = e / nd, d = e - t * nd;
            const int64_t at = vrow + (int64_t)t * p.v_ss + d;
            unsigned char* dst = lds + t * row + d * size;
            if (p.v_dtype != p.vp_dtype) rope_store(dst, p.vp_dtype, 0, ssq_load_elem(p.v, p.v_dtype, at));
            else if (size == 4) *reinterpret_cast<uint32_t*>(dst) = reinterpret_cast<const uint32_t*>(p.v)[at];
            else *reinterpret_cast<uint16_t*>(dst) = reinterpret_cast<const uint16_t*>(p.v)[at];
        }
    }
    __syncthreads();
    // both groups of 8 tokens of a dim side by side; a sequence's first tile lacks its first cut tokens
    const int cut = s0 - (s1 - kValTok);
    for (int e = tid; e < 2 * nd; e += kThreads) {
        const int g = e & 1, d = e >> 1;
        const int ta = max(8 * g - cut, 0), tb = min(8 * g - cut + 8, nt);
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

// Tokens [4 tile, +4) one by one: where a sequence brings few tokens, few share a page's 16-byte piece.
__device__ __forceinline__ void value_rows(const AppendParams& p, int tile, int kv, int dc) {
    const ssq_encode_args& a = p.e;
    const int d0 = dc * kValDims, nd = min(kValDims, p.value_dim - d0), d = threadIdx.x & (kValDims - 1);
    const int n = a.batch * a.seq_len;
    constexpr int kStep = kThreads / kValDims, kSteps = kOneTok / kStep;
    static_assert(kThreads % kValDims == 0 && kOneTok % kStep == 0, "rows per step");
    uint32_t w[kSteps];
    int64_t slot[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int i = tile * kOneTok + k * kStep + (int)(threadIdx.x / kValDims);
        slot[k] = -1;
        if (i < n) {
            int b, s;
            split_token(p, i, b, s);
            slot[k] = slot_of(p, b, s);
            if (p.slots_out && kv == 0 && dc == 0 && d == 0) p.slots_out[i] = slot[k];
            if (d >= nd || !p.v) slot[k] = -1;
            else w[k] = ssq_load_bits(p.v, p.v_dtype, (int64_t)b * p.v_sb + (int64_t)kv * p.v_sh + (int64_t)s * p.v_ss + d0 + d);
        }
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        if (slot[k] < 0) continue;
        int64_t pg;
        int off;
        split_slot(p, slot[k], pg, off);
        const int64_t at = pg * p.vp_sb + (int64_t)kv * p.vp_sh + (int64_t)(d0 + d) * p.vp_sd + off;
        if (p.v_dtype != p.vp_dtype) rope_store(p.vp, p.vp_dtype, at, ssq_bits_to_f32(w[k], p.v_dtype));
        else if (p.v_dtype == SSQ_F32) reinterpret_cast<uint32_t*>(p.vp)[at] = w[k];
        else reinterpret_cast<uint16_t*>(p.vp)[at] = (uint16_t)w[k];
    }
}

constexpr int kPrepHeads = 2;  // with 4, 101 registers a lane leave room for half the value workgroups: 22.6 us for 20.0

// Many rows: workgroups [0, rope_blocks) rotate the keys, the others write the values (and, for kv 0 and the first
// dims, the sanitized slots).  They share nothing; one launch lets the values' transposes run beside the rotation.
template <int DT, bool NORM>
__global__ __launch_bounds__(kThreads) void k_append_prep(const AppendParams p, const RopeParams rp, int rope_blocks, int tiles) {
    constexpr int kLds = kValLds > rope_lds<DT, NORM>() * 4 ? kValLds : rope_lds<DT, NORM>() * 4;
    __shared__ __align__(16) unsigned char lds[kLds];
    __shared__ ValSlots vs;
    static_assert(kThreads == kRopeThreads, "one block size");
    if ((int)blockIdx.x < rope_blocks) {
        rope_units<DT, NORM, kPrepHeads>(rp, blockIdx.x, reinterpret_cast<float*>(lds));
        return;
    }
    const int e = blockIdx.x - rope_blocks, dk = e / tiles;  // tiles of a KV head side by side
    const int dc = dk / p.e.num_kv_heads, kv = dk - dc * p.e.num_kv_heads;
    if (p.vone) value_rows(p, e - dk * tiles, kv, dc);
    else value_tile(p, lds, vs, e - dk * tiles, kv, dc);
}

constexpr int kScan = 16;  // codewords of a lane whose distances are held at once

// Clamped pre-sqrt values v[u] >= 0 of codewords j0 + u stride against the least distance so far: the first codeword
// with the smallest correctly rounded sqrt wins.  The square roots of all are not taken: the smallest v has the
// smallest one, and equal ones come from values less than 2^-21 apart relatively (below 2^-126, a few units of the
// smallest subnormal), so only where a second value lies that close are they compared.  Four operations a
// codeword, where keeping the first minimum as it goes takes its exact branch at almost every step of
// so short a scan, in one lane or another.
__device__ __forceinline__ void first_least(const float (&v)[kScan], uint32_t j0, uint32_t stride, float& f_best, uint32_t& j_best) {
    float least = v[0];
#pragma unroll
    for (int u = 1; u < kScan; ++u) least = __builtin_fminf(least, v[u]);
    const float f = __builtin_sqrtf(least);
    if (!(f < f_best)) return;
    const float near = least * 0x1.00001p+0f + 0x1.0p-146f;
    int at = 0, n = 0;
#pragma unroll
    for (int u = kScan - 1; u >= 0; --u) {
        const bool c = v[u] <= near;
        at = c ? u : at;
        n += c ? 1 : 0;
    }
    if (n > 1) {
#pragma unroll
        for (int u = kScan - 1; u >= 0; --u)
            if (v[u] <= near && __builtin_sqrtf(v[u]) == f) at = u;
    }
    f_best = f;
    j_best = j0 + (uint32_t)at * stride;
}

// A key's row into LDS by its S lanes, and, if asked, its lane's share of the sum of squares.
template <int DT, int S>
__device__ __forceinline__ double stage_row(const AppendParams& p, int64_t at, unsigned char* dst, int sl) {
    constexpr int V = RopeVec<DT>::N, kAhead = 4;
    const int D = p.e.head_dim;
    const bool norm = p.kw != nullptr;
    double sum = 0.0;
    if (p.row_vec) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p.e.keys) + at * (16 / V));
        const int units = D / V;
        for (int q0 = sl; q0 < units; q0 += kAhead * S) {
            uint4 w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (q0 + k * S < units) w[k] = src[q0 + k * S];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (q0 + k * S >= units) continue;
                *reinterpret_cast<uint4*>(dst + 16 * (q0 + k * S)) = w[k];
                if (!norm) continue;
                float x[V];
                rope_unpack<DT>(w[k], x);
#pragma unroll
                for (int i = 0; i < V; ++i) sum = __builtin_fma((double)x[i], (double)x[i], sum);
            }
        }
    } else {
        for (int q = sl; q < D; q += S) {
            const uint32_t w = ssq_load_bits(p.e.keys, DT, at + q);
            if constexpr (DT == SSQ_F32) reinterpret_cast<uint32_t*>(dst)[q] = w;
            else reinterpret_cast<uint16_t*>(dst)[q] = (uint16_t)w;
            const double x = (double)ssq_bits_to_f32(w, DT);
            sum = __builtin_fma(x, x, sum);
        }
    }
    return sum;
}

// The dims of one block of a key, normed, rotated and rounded as rope_dim does it, from its row in LDS.
template <int DT, int N>
__device__ __forceinline__ void block_dims(const unsigned char* row, const int (&dim)[N], const int (&other)[N],
                                           const bool (&rot)[N], const bool (&first)[N], bool norm, bool turn, float r,
                                           const float (&w0)[N], const float (&w1)[N], const float (&cv)[N], const float (&sv)[N],
                                           float (&x)[N]) {
    auto elem = [&](int i) {
        if constexpr (DT == SSQ_F32) return reinterpret_cast<const float*>(row)[i];
        else return ssq_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[i], DT);
    };
#pragma unroll
    for (int d = 0; d < N; ++d) x[d] = elem(dim[d]);
    if (norm) {
#pragma unroll
        for (int d = 0; d < N; ++d) x[d] = (x[d] * r) * w0[d];
    }
    if (turn) {
#pragma unroll
        for (int d = 0; d < N; ++d) {
            float v = elem(other[d]);
            if (norm) v = (v * r) * w1[d];
            const float y = x[d] * cv[d], z = v * sv[d], t = first[d] ? y - z : y + z;
            x[d] = rot[d] ? t : x[d];
        }
    }
    if (norm || turn) {
#pragma unroll
        for (int d = 0; d < N; ++d) x[d] = rope_round(x[d], DT);
    }
}

// BD: the block dim at compile time (1, 2, 4 or 8), or 0 for any other up to 16; S: lanes of a key.  x: value
// tiles, then blocks and their tiles of keys; y: KV heads.  V8: the values go to 8-bit pages (p8), p8_blocks workgroups a head.
template <int BD, int S, bool V8>
__device__ __forceinline__ void append_few(const AppendParams& p, const SsqValues* p8, int p8_blocks) {
    constexpr int kX = BD ? BD : 16, kPer = kThreads / S;
    extern __shared__ __align__(16) unsigned char few_lds[];
    const ssq_encode_args& a = p.e;
    const int kv = blockIdx.y, n = a.batch * a.seq_len;
    int kt = blockIdx.x;
    if constexpr (V8) {
        if (kt < p8_blocks) {
            const int64_t w = (int64_t)kt * (kThreads / SSQ_WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x / SSQ_WAVE);
            if (kv < p8->hgroups) val_wave(*p8, w * p8->hgroups + kv, threadIdx.x & (SSQ_WAVE - 1));
            return;
        }
        kt -= p8_blocks;
    } else if (kt < p.vtiles * p.dchunks) {
        __shared__ ValSlots vs;
        const int dc = kt / p.vtiles, tile = kt - dc * p.vtiles;
        if (p.vone) value_rows(p, tile, kv, dc);
        else value_tile(p, few_lds, vs, tile, kv, dc);
        return;
    }
    if constexpr (!V8) kt -= p.vtiles * p.dchunks;
    const int blk = kt / p.ktiles;
    kt -= blk * p.ktiles;
    const int sl = threadIdx.x & (S - 1), local = (int)threadIdx.x / S, i = kt * kPer + local;
    const bool live = i < n;
    const int bd = BD ? BD : a.block_dim, nc = a.n_centroids, D = a.head_dim;
    const int cw = ssq_code_width(nc);
    const bool heavy = ssq_is_heavy(a.heavy_mask[0], a.heavy_mask[1], blk);
    const float* met = a.metric ? a.metric + (int64_t)kv * a.metric_sh + (int64_t)blk * bd * D + blk * bd : nullptr;
    int b, s;
    split_token(p, live ? i : n - 1, b, s);
    const bool norm = p.kw != nullptr, turn = p.t.cos != nullptr;
    // LDS: the codebook's stage [chunk][bd] and norms [chunk], then the key rows
    float* cb = reinterpret_cast<float*>(few_lds);
    float* cn = cb + (size_t)p.chunk * bd;
    unsigned char* row = few_lds + (((size_t)p.chunk * (bd + 1) * 4 + 15) & ~(size_t)15) + (size_t)local * p.krow;

    // everything whose address is known
    const int64_t slot = slot_of(p, b, s);
    const int64_t pos = turn ? rope_pos(p.t, b, s) : 0;
    const float* cent = a.cent + (int64_t)kv * a.cent_sh + (int64_t)blk * nc * bd;
    float c0[kX];
    const bool mine0 = (int)threadIdx.x < min(p.chunk, nc);
    if (mine0) {
#pragma unroll
        for (int d = 0; d < kX; ++d)
            if (d < bd) c0[d] = cent[threadIdx.x * bd + d];
    }
    const int64_t* perm = a.perm + (int64_t)kv * a.perm_sh + (int64_t)blk * bd;
    int dim[kX];
#pragma unroll
    for (int d = 0; d < kX; ++d) dim[d] = d < bd ? (int)min((uint64_t)perm[d], (uint64_t)(D - 1)) : 0;
    const int64_t at = (int64_t)b * a.k_sb + (int64_t)kv * a.k_sh + (int64_t)s * a.k_ss;
    double sum = a.k_dtype == SSQ_BF16  ? stage_row<SSQ_BF16, S>(p, at, row, sl)
                 : a.k_dtype == SSQ_F16 ? stage_row<SSQ_F16, S>(p, at, row, sl)
                                        : stage_row<SSQ_F32, S>(p, at, row, sl);
    // the block's dims, their partners and table entries
    const int half = p.t.rot_dim >> 1;
    int other[kX];
    bool rot[kX], first[kX];
    float cv[kX], sv[kX], w0[kX], w1[kX];
#pragma unroll
    for (int d = 0; d < kX; ++d) {
        const int m = dim[d];
        rot[d] = turn && m < p.t.rot_dim;
        first[d] = p.t.interleaved ? !(m & 1) : m < half;
        other[d] = !rot[d] ? m : p.t.interleaved ? m ^ 1 : first[d] ? m + half : m - half;
    }
    if (turn) {
        const float* cr = p.t.cos + (pos < 0 ? 0 : pos) * p.t.ld;
        const float* sr = p.t.sin + (pos < 0 ? 0 : pos) * p.t.ld;
#pragma unroll
        for (int d = 0; d < kX; ++d) {
            const int ti = !rot[d] ? 0 : p.t.interleaved ? dim[d] >> 1 : min(dim[d], other[d]);
            cv[d] = cr[ti];
            sv[d] = sr[ti];
        }
    }
    if (norm) {
#pragma unroll
        for (int d = 0; d < kX; ++d) {
            w0[d] = ssq_load_elem(p.kw, p.t.w_dtype, dim[d]);
            w1[d] = ssq_load_elem(p.kw, p.t.w_dtype, other[d]);
        }
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
    auto stage = [&](float (&c)[kX], int e) {
        if (met) map(c);
#pragma unroll
        for (int d = 0; d < kX; ++d)
            if (d < bd) cb[e * bd + d] = c[d];
        cn[e] = sq_norm(c, bd);
    };
    if (mine0) stage(c0, threadIdx.x);
    __syncthreads();

    float r = 1.f;
    if (norm) {  // the key's lanes' shares
#pragma unroll
        for (int o = S >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        r = rope_rstd(sum, p.inv_d, p.t.eps);
    }
    if (turn && pos < 0) {  // a position outside the tables
#pragma unroll
        for (int d = 0; d < kX; ++d) cv[d] = sv[d] = __builtin_nanf("");
    }
    float x[kX];
    if (a.k_dtype == SSQ_BF16) block_dims<SSQ_BF16>(row, dim, other, rot, first, norm, turn, r, w0, w1, cv, sv, x);
    else if (a.k_dtype == SSQ_F16) block_dims<SSQ_F16>(row, dim, other, rot, first, norm, turn, r, w0, w1, cv, sv, x);
    else block_dims<SSQ_F32>(row, dim, other, rot, first, norm, turn, r, w0, w1, cv, sv, x);
    int64_t crow = 0, prow = 0;
    if (slot >= 0) {
        int64_t page;
        int off;
        split_slot(p, slot, page, off);
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
    if (met) map(x);
    const float xn = sq_norm(x, bd);
    const bool direct = a.direct_dist != 0;
    float f_best = INFINITY;
    uint32_t j_best = 0;
    for (int j0 = 0; j0 < nc; j0 += p.chunk) {
        const int m = min(p.chunk, nc - j0);
        // codewords past the first kThreads, and past the first stage
        if (j0) __syncthreads();  // the previous stage's reads are done
        for (int e = threadIdx.x + (j0 ? 0 : kThreads); e < m; e += kThreads) {
            float c[kX];
#pragma unroll
            for (int d = 0; d < kX; ++d)
                if (d < bd) c[d] = cent[(int64_t)(j0 + e) * bd + d];
            stage(c, e);
        }
        if (j0 || m > kThreads) __syncthreads();
        for (int g = 0; g < m; g += kScan * S) {  // the next kScan codewords of each lane
            float v[kScan];
            if (!direct && g + kScan * S <= m) {
                const float* c = cb + (g + sl) * bd;
                const float* q = cn + g + sl;
#pragma unroll
                for (int u = 0; u < kScan; ++u) v[u] = __builtin_fmaxf(mm_dist2(x, xn, c + u * S * bd, q[u * S], bd), 0.f);
            } else if (!direct) {
#pragma unroll
                for (int u = 0; u < kScan; ++u) {
                    const int j = g + sl + u * S, jj = min(j, m - 1);
                    const float y = mm_dist2(x, xn, cb + jj * bd, cn[jj], bd);
                    v[u] = j < m ? __builtin_fmaxf(y, 0.f) : INFINITY;  // NaN: 0, as clamp_min's
                }
            } else {  // at most 25 codewords and keys: small code counts
#pragma unroll 1
                for (int u = 0; u < kScan; ++u) {
                    const int j = g + sl + u * S;
                    const float y = direct_dist2(x, cb + min(j, m - 1) * bd, bd);
#pragma unroll
                    for (int k = 0; k < kScan; ++k) v[k] = k != u ? v[k] : j < m ? __builtin_fmaxf(y, 0.f) : INFINITY;
                }
            }
            first_least(v, (uint32_t)(j0 + g + sl), (uint32_t)S, f_best, j_best);
        }
    }
    // the key's lanes: the smaller distance, then the smaller index
#pragma unroll
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
template <int BD, int S>
__global__ __launch_bounds__(kThreads) void k_append_few(const AppendParams p) { append_few<BD, S, false>(p, nullptr, 0); }
// (a kernel of its own: the values' registers would cost the 16-bit one waves)
template <int BD, int S>
__global__ __launch_bounds__(kThreads) void k_append_few8(const AppendParams p, const SsqValues p8, int p8_blocks) {
    append_few<BD, S, true>(p, &p8, p8_blocks);
}

bool uses_grid(const ssq_encode_args& e) {  // as ssq_encode chooses
    return e.kernel == 0 && e.grid && !e.direct_dist && ssq_encode_grid_supported(&e);
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
    if (uses_grid(e)) {  // likewise
        const uint64_t need = ssq_encode_grid_bytes(&e);
        SSQ_REQUIRE((uintptr_t)e.grid % 16 == 0, "the grid must be 16-byte aligned");
        SSQ_REQUIRE(e.grid_bytes >= need, "grid too small for this codebook (%llu < %llu bytes)",
                    (unsigned long long)e.grid_bytes, (unsigned long long)need);
    }
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

// One launch or two and the encode's?  The few kernel stages a codebook per 4 to 64 keys, the encode's screen spreads it
// over 512; measured, calls in a row, 8 heads of 128 dims, us in one launch and through the encode:
//   256 codewords of dim 4: 64 tokens 8.5 and 18.8, 256 14.2 and 20.2, 512 22.8 and 18.5;  of dim 2: 128 tokens 12.1 and
//   21.2, 256 20.0 and 17.5;  of dim 8: 512 tokens 20.3 and 24.7, 1,024 33.5 and 22.1;  4,096 of dim 4: 4 tokens 11.4
//   and 23.2, 16 28.2 and 31.4, 64 42 and 22
// -- about 2^24 (key, block, codeword) triples.  Codebooks of at most 256 codewords that ssq_encode serves by its exact
// scan, whose workgroups take more keys than most calls have, stay: 16 of dim 4, 4,096 tokens 90 and 253, 8,192 167 and
// 427; 128 of dim 8, 8,192 tokens 165 and 2,157; up to as many workgroups as one launch holds with ease.
bool few(const ssq_append_args& a) {
    const ssq_encode_args& e = a.enc;
    if (e.kernel != 0) return false;
    const bool scan = !uses_grid(e) && (e.n_centroids < 256 || (e.n_centroids == 256 && (e.direct_dist || e.block_dim > 10)));
    const int64_t rows = (int64_t)e.batch * e.seq_len * e.num_kv_heads * e.n_blocks;
    return scan ? rows <= 1 << 26 : rows <= 1 << 24 && rows * e.n_centroids <= 1 << 24;
}

bool turns(const ssq_append_args& a) { return a.k_weight || a.rope.cos; }

int64_t rows_bytes(const ssq_append_args& a) {
    const ssq_encode_args& e = a.enc;
    const int64_t n = (int64_t)e.batch * e.seq_len * e.num_kv_heads * e.head_dim * (e.k_dtype == SSQ_F32 ? 4 : 2);
    return turns(a) ? (n + 255) & ~(int64_t)255 : 0;
}

AppendParams params(const ssq_append_args& a) {
    AppendParams p{};
    const ssq_encode_args& e = a.enc;
    p.e = e;
    p.t = a.rope;
    if (!p.t.cos) p.t.rot_dim = 0;
    p.kw = a.k_weight;
    p.n_slots = a.num_pages * a.enc.page_size;
    p.page_log = -1;
    for (int l = 0; l < 31; ++l)
        if (e.page_size == 1 << l) p.page_log = l;
    p.inv_d = 1.0 / (double)e.head_dim;
    p.v = a.v;
    p.vp = a.v_pages;
    p.v_sb = a.v_sb; p.v_sh = a.v_sh; p.v_ss = a.v_ss;
    p.vp_sb = a.vp_sb; p.vp_sh = a.vp_sh; p.vp_sd = a.vp_sd;
    p.v_dtype = a.v_dtype; p.vp_dtype = a.vp_dtype; p.value_dim = a.v ? a.value_dim : 0;
    p.dchunks = (p.value_dim + kValDims - 1) / kValDims;
    const int per = e.k_dtype == SSQ_F32 ? 4 : 8;
    p.row_vec = (uintptr_t)e.keys % 16 == 0 && e.head_dim % per == 0 && e.k_sb % per == 0 && e.k_sh % per == 0 && e.k_ss % per == 0;
    p.vone = e.seq_len < 8;
    p.vseq = (e.seq_len + 2 * (kValTok - 1)) / kValTok;  // a first tile of one token, at worst
    p.vtiles = p.vone ? (int)(((int64_t)e.batch * e.seq_len + kOneTok - 1) / kOneTok) : e.batch * p.vseq;
    p.v_vec = a.v && a.v_dtype == a.vp_dtype && a.v_dtype != SSQ_F32 && (uintptr_t)a.v % 16 == 0 && a.value_dim % 8 == 0 &&
              a.v_sb % 8 == 0 && a.v_sh % 8 == 0 && a.v_ss % 8 == 0;
    const int vper = a.vp_dtype == SSQ_F32 ? 4 : 8;
    p.vp_vec = a.v && (uintptr_t)a.v_pages % 16 == 0 && e.page_size % 8 == 0 && a.vp_sb % vper == 0 && a.vp_sh % vper == 0 &&
               a.vp_sd % vper == 0;
    return p;
}

// the values and the sanitized slots, and the keys' rotation beside them where its unit kernel serves them
int run_prep(const AppendParams& p, const SsqRopeRows& r, bool turn, hipStream_t st) {
    RopeParams rp{};
    rp.r = r;
    rp.inv_d = p.inv_d;
    int lpr = 0;
    int64_t rope_blocks = 0;
    const bool units = turn && ssq_rope_units_ok(r, lpr);
    if (units) {
        rp.lpr = lpr;
        while ((1 << rp.lpr_log) < lpr) ++rp.lpr_log;
        rp.groups = (r.heads[0] + kPrepHeads - 1) / kPrepHeads;
        rp.items = (int64_t)r.batch * r.seq_len * rp.groups;
        rope_blocks = (rp.items * lpr + kThreads - 1) / kThreads;
    } else if (turn) {
        int rc = ssq_rope_run(r, st);
        if (rc) return rc;
    }
    const int64_t blocks = rope_blocks + (int64_t)p.vtiles * p.e.num_kv_heads * (p.dchunks ? p.dchunks : 1);
    SSQ_UNSUPPORTED(blocks <= 0x7fffffff, "too many rows");
    const dim3 grid((unsigned)blocks), block(kThreads);
    const int rb = (int)rope_blocks, vt = p.vtiles;
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

template <int BD, int S>
void launch_few(const AppendParams& p, const SsqValues* p8, int p8_blocks, dim3 grid, size_t lds, hipStream_t st) {
    if (p8) hipLaunchKernelGGL((k_append_few8<BD, S>), grid, dim3(kThreads), lds, st, p, *p8, p8_blocks);
    else hipLaunchKernelGGL((k_append_few<BD, S>), grid, dim3(kThreads), lds, st, p);
}
template <int S>
int launch_few(const AppendParams& p, const SsqValues* p8, int p8_blocks, dim3 grid, size_t lds, hipStream_t st) {
    switch (p.e.block_dim) {
        case 1: launch_few<1, S>(p, p8, p8_blocks, grid, lds, st); break;
        case 2: launch_few<2, S>(p, p8, p8_blocks, grid, lds, st); break;
        case 4: launch_few<4, S>(p, p8, p8_blocks, grid, lds, st); break;
        case 8: launch_few<8, S>(p, p8, p8_blocks, grid, lds, st); break;
        default: launch_few<0, S>(p, p8, p8_blocks, grid, lds, st); break;
    }
    return ssq_check_hip(hipGetLastError(), "k_append_few launch");
}

}  // namespace

extern "C" size_t ssq_append_workspace_size(const ssq_append_args* a) {
    if (check(a) != SSQ_OK || few(*a)) return 0;
    return (size_t)(rows_bytes(*a) + (int64_t)a->enc.batch * a->enc.seq_len * 8);
}

// v8: the values' 8-bit append, beside the keys' (a->v NULL) in the one launch of few rows, else in one of its own
static int append_run(const ssq_append_args* a, const ssq_values_args* v8, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc) return rc;
    const ssq_encode_args& e = a->enc;
    const int64_t n = (int64_t)e.batch * e.seq_len;
    if (n == 0) return SSQ_OK;
    hipStream_t st = (hipStream_t)stream;
    AppendParams p = params(*a);
    if (few(*a)) {
        // Lanes of a key, by (key, block) pairs: more where pairs are few (the chain of loads and a lane's scan bound the
        // call), fewer where they are many (what every lane does besides its scan does), us with 16, 8 and 4, 256
        // codewords of dim 4: 8,192 pairs 7.4, 7.5, 9.1; 16,384 9.4, 8.6, 9.4; 65,536 23, 17.2, 14.3; 4 for at most 64
        // codewords, a scan of 16 each: 512 pairs 8.4, 8.2, 5.2.  A whole wave where the scan is long and the keys
        // too few for the device (4,096 codewords, 4 tokens: 11.9 with 64, 32 with 8; 64 tokens 79 and 44).  A
        // workgroup's key rows fit 20 KiB of LDS.
        const int64_t units = n * e.num_kv_heads * e.n_blocks;
        const int row = e.head_dim * (e.k_dtype == SSQ_F32 ? 4 : 2);
        p.krow = ((row + 15) & ~15) + 16;  // rows on other LDS banks
        int S = e.n_centroids <= 64 || units >= 32768 ? 4 : units <= 8192 ? 16 : 8;
        if (units * 8 < (int64_t)ssq_device_cus() * 256 && e.n_centroids >= 1024) S = SSQ_WAVE;
        while (S < SSQ_WAVE && kThreads / S * p.krow > 20 * 1024) S = S == 16 ? SSQ_WAVE : 2 * S;
        const int stage = kStageFloats / (e.block_dim + 1);
        p.chunk = e.n_centroids < stage ? e.n_centroids : stage;
        const int per = kThreads / S;
        p.ktiles = (int)((n + per - 1) / per);
        SsqValues p8{};
        int64_t p8_blocks = 0;
        if (v8 && a->num_pages > 0) {
            p8 = ssq_values_params(*v8);
            p8_blocks = ((int64_t)p8.batch * p8.chunks + kThreads / SSQ_WAVE - 1) / (kThreads / SSQ_WAVE);
        }
        const SsqValues* vp = v8 ? &p8 : nullptr;
        const int64_t xs = p8_blocks + (int64_t)p.vtiles * p.dchunks + (int64_t)p.ktiles * e.n_blocks;
        SSQ_UNSUPPORTED(xs <= 0x7fffffff, "too many rows");
        dim3 grid((unsigned)xs, e.num_kv_heads);
        size_t lds = (((size_t)p.chunk * (e.block_dim + 1) * 4 + 15) & ~(size_t)15) + (size_t)per * p.krow;
        const size_t vlds = a->v && !p.vone ? (size_t)kValTok * val_row(a->vp_dtype == SSQ_F32 ? 4 : 2) : 0;
        if (vlds > lds) lds = vlds;
        switch (S) {
            case 4: return launch_few<4>(p, vp, (int)p8_blocks, grid, lds, st);
            case 8: return launch_few<8>(p, vp, (int)p8_blocks, grid, lds, st);
            case 16: return launch_few<16>(p, vp, (int)p8_blocks, grid, lds, st);
            default: return launch_few<SSQ_WAVE>(p, vp, (int)p8_blocks, grid, lds, st);
        }
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
    rc = run_prep(p, r, turns(*a), st);
    if (rc == SSQ_OK && v8) rc = ssq_append_values(v8, stream);
    if (rc) return rc;
    return ssq_encode(&enc, stream);
}

extern "C" int ssq_append(const ssq_append_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return append_run(a, nullptr, workspace, workspace_bytes, stream);
}

// The values of an 8-bit append are those of ssq_append_values, the rest those of ssq_append without values.

namespace {

int check8(const ssq_append8_args* a, ssq_append_args& keys, ssq_values_args& v) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_append8_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_append8_args size %u != library's %zu", a->struct_size, sizeof(ssq_append8_args));
    keys = a->app;
    keys.v = nullptr;
    int rc = check(&keys);
    if (rc) return rc;
    SSQ_REQUIRE(a->app.vp_dtype == SSQ_E4M3, "append8 writes 8-bit values");
    const ssq_encode_args& e = keys.enc;
    v = ssq_values_args{};
    v.struct_size = sizeof(v);
    v.v = a->app.v; v.v_dtype = a->app.v_dtype; v.v_sb = a->app.v_sb; v.v_sh = a->app.v_sh; v.v_ss = a->app.v_ss;
    v.batch = e.batch; v.num_kv_heads = e.num_kv_heads; v.seq_len = e.seq_len; v.value_dim = a->app.value_dim;
    v.v_pages = a->app.v_pages; v.vp_sb = a->app.vp_sb; v.vp_sh = a->app.vp_sh; v.vp_sd = a->app.vp_sd;
    v.v_scale = a->v_scale; v.vs_sb = a->vs_sb; v.vs_sh = a->vs_sh;
    v.slot_mapping = e.slot_mapping; v.sm_sb = e.sm_sb;
    v.page_size = e.page_size; v.num_pages = a->app.num_pages;
    return ssq_values_check(&v);
}

}  // namespace

extern "C" size_t ssq_append8_workspace_size(const ssq_append8_args* a) {
    ssq_append_args keys;
    ssq_values_args v;
    return check8(a, keys, v) == SSQ_OK ? ssq_append_workspace_size(&keys) : 0;
}

extern "C" int ssq_append8(const ssq_append8_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    ssq_append_args keys;
    ssq_values_args v;
    int rc = check8(a, keys, v);
    return rc == SSQ_OK ? append_run(&keys, &v, workspace, workspace_bytes, stream) : rc;
}
