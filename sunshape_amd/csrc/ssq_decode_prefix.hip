// Decode for a batch that shares a prefix (ssq_decode_prefix): every query row attends the prefix's tokens and
// its own sequence's, one softmax over both.
//
//   m = max(m_p, m_o),  l = l_p e^{m_p - m} + l_o e^{m_o - m},  out = (o_p e^{m_p - m} + o_o e^{m_o - m}) / l
//
// with (o, m, l) = (sum_t e^{s_t - m} v_t, max_t s_t, sum_t e^{s_t - m}) of a set of tokens.  The prefix is one
// sequence whose query rows are all sequences' rows of a KV head, so its codes and values are read once for them.
// Both parts leave fp32 (o, m, l) in the workspace, per context split, and a merge joins them.
//
// Byte-code codecs of head_dim 64 and 128 take the matrix-core kernel (ssq_prefix_mfma.h), one launch for the prefix
// and the own tokens; every other problem the decode kernels (ssq_decode_partials).
#include "ssq_prefix_mfma.h"

#include <math.h>

int ssq_decode_validate(const ssq_decode_args* a);
int ssq_decode_partial_splits(const ssq_decode_args* a, int& split_len);
int ssq_decode_partials(const ssq_decode_args* a, void* ws, size_t bytes, hipStream_t st);

namespace {

constexpr int kMergeRows = 4;
constexpr int kMergeBatch = 8;  // partials in flight per lane
constexpr int kMergeDims = 4;   // value dims per lane per pass

struct MergeParams {
    ssq_decode_args a;
    // The prefix's partials: for each query position and each chunk of `chunk` sequences a block of
    // n1 (the last chunk n1_last) splits x (num_q_heads * sequences) rows: o, then m, then l.
    const float* pre;
    int chunk, n1, n1_last;
    // the own tokens' partials, n2 splits x (batch * num_q_heads * q_len) rows (0: none)
    const float* own;
    int n2;
    int len1, len1_last, len2;  // tokens of a split
    const int32_t* plen;
};

// Whether a query row holds a NaN (a wave's question).
__device__ __forceinline__ bool nan_query(const ssq_decode_args& a, int b, int h, int qi, int lane) {
    const int64_t at = (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + (int64_t)qi * a.q_sl;
    bool is = false;
    for (int d = lane; d < a.head_dim; d += SSQ_WAVE) {
        const float x = ssq_load_elem(a.q, a.q_dtype, at + d);
        is |= x != x;
    }
    return __builtin_amdgcn_ballot_w64(is) != 0;
}

// One wave per query row.  A lane takes a split's (m, l), 64 at a time; the splits that hold tokens are then
// joined with lane j on value dims j, j + 64, ...: bytes bound it, and splits without tokens cost no o.  Those
// with tokens count also at weight 0: 0 times an infinite or NaN value is NaN, as in one pass over all tokens.
__global__ __launch_bounds__(kMergeRows * SSQ_WAVE) void k_merge_prefix(const MergeParams p) {
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & (SSQ_WAVE - 1);
    const int64_t n_rows = (int64_t)a.batch * a.num_q_heads * a.q_len;
    const int64_t rid = (int64_t)blockIdx.x * kMergeRows + __builtin_amdgcn_readfirstlane(threadIdx.x / SSQ_WAVE);
    if (rid >= n_rows) return;  // whole waves
    const int qi = (int)(rid % a.q_len);
    const int h = (int)(rid / a.q_len % a.num_q_heads);
    const int b = (int)(rid / a.q_len / a.num_q_heads);
    const int Dv = a.value_dim;
    // this row's prefix block
    int n1 = p.n1, len1 = p.len1;
    int64_t at0 = 0, rows1 = n_rows, row1 = rid;
    if (p.n1) {
        const int c = b / p.chunk, cn = min(p.chunk, a.batch - c * p.chunk);
        if ((int64_t)(c + 1) * p.chunk >= a.batch) {
            n1 = p.n1_last;
            len1 = p.len1_last;
        }
        const int rest = a.batch % p.chunk ? a.batch % p.chunk : p.chunk;
        const int64_t per_q = (int64_t)a.num_q_heads * ((int64_t)(a.batch - rest) * p.n1 + (int64_t)rest * p.n1_last);
        at0 = (per_q * qi + (int64_t)a.num_q_heads * c * p.chunk * p.n1) * (Dv + 2);
        rows1 = (int64_t)a.num_q_heads * cn;
        row1 = (int64_t)h * cn + (b - c * p.chunk);
    }
    const int n1_all = n1;
    const int n2 = p.n2;
    const float* pre_o = p.pre + at0;
    const float* pre_m = pre_o + rows1 * n1_all * Dv;
    const float* pre_l = pre_m + rows1 * n1_all;
    const float* own_m = p.own + n_rows * p.n2 * Dv;
    const float* own_l = own_m + n_rows * p.n2;
    const int n = n1 + n2;
    const int t1 = n1 ? p.plen[0] : 0, t2 = n2 ? a.seq_lens[b] : 0;
    float M = -INFINITY, L = 0.f;
    for (int d0 = 0; d0 < Dv; d0 += kMergeDims * SSQ_WAVE) {
        float Mr = -INFINITY, Lr = 0.f, o[kMergeDims];
#pragma unroll
        for (int k = 0; k < kMergeDims; ++k) o[k] = 0.f;
        for (int s0 = 0; s0 < n; s0 += SSQ_WAVE) {
            const int s = s0 + lane;
            const bool pre = s < n1;
            const int64_t at = pre ? (int64_t)s * rows1 + row1 : (int64_t)(s - n1) * n_rows + rid;
            const float m = s < n ? (pre ? pre_m : own_m)[at] : -INFINITY;
            const float l = m != -INFINITY ? (pre ? pre_l : own_l)[at] : 0.f;
            const float Mc = fmaxf(Mr, ssq_wave_max(m));
            const float f = Mr == -INFINITY ? 0.f : __expf(Mr - Mc);  // earlier passes, rescaled
            const float w = m == -INFINITY ? 0.f : __expf(m - Mc);
            Lr = Lr * f + ssq_wave_sum(l * w);
#pragma unroll
            for (int k = 0; k < kMergeDims; ++k) o[k] *= f;
            const bool holds = pre ? (int64_t)s * len1 < t1 : s < n && (int64_t)(s - n1) * p.len2 < t2;
            uint64_t live = __builtin_amdgcn_ballot_w64(holds);
            while (live) {  // wave-uniform
                float ov[kMergeBatch][kMergeDims], wv[kMergeBatch];
#pragma unroll
                for (int i = 0; i < kMergeBatch; ++i) {
                    const int src = live ? __builtin_ctzll(live) : 0;
                    wv[i] = live ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), src)) : 0.f;
                    const int sp = s0 + src;
                    const float* ob = live ? (sp < n1 ? pre_o + ((int64_t)sp * rows1 + row1) * Dv
                                                      : p.own + ((int64_t)(sp - n1) * n_rows + rid) * Dv)
                                           : nullptr;
#pragma unroll
                    for (int k = 0; k < kMergeDims; ++k)
                        ov[i][k] = ob && d0 + k * SSQ_WAVE < Dv ? ob[min(d0 + k * SSQ_WAVE + lane, Dv - 1)] : 0.f;
                    live &= live - 1;
                }
#pragma unroll
                for (int i = 0; i < kMergeBatch; ++i)
#pragma unroll
                    for (int k = 0; k < kMergeDims; ++k) o[k] += ov[i][k] * wv[i];
            }
            Mr = Mc;
        }
        // the decode kernels leave a row of NaN scores as one without tokens
        if (Mr == -INFINITY && nan_query(a, b, h, qi, lane)) Mr = Lr = __builtin_nanf("");
#pragma unroll
        for (int k = 0; k < kMergeDims; ++k) {
            const int dv = d0 + k * SSQ_WAVE + lane;
            if (dv < Dv)  // a row with nothing to attend gives 0
                ssq_store_elem(a.out, a.v_dtype, (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)qi * a.o_sl + dv,
                               Mr == -INFINITY ? 0.f : o[k] / Lr);
        }
        M = Mr;
        L = Lr;
    }
    if (a.lse && lane == 0) a.lse[rid] = M == -INFINITY ? -INFINITY : M + logf(L);
}

// The same for the matrix-core kernel's partials, n1 prefix slices and n2 own pieces x (batch * num_q_heads * q_len)
// rows, of which those with tokens are written.  Loads that wait for one another bound it (partials come from
// other XCDs), so the lengths, every (m, l) and the first few o of both kinds are asked for at once, and what
// the lengths rule out is dropped after.  Lane j has dims D / 64 j ...
struct MergeFlat {
    ssq_decode_args a;
    const float* pre;
    const float* own;
    int n1, n2, pcap;
    int pair;  // pairs of output dims store as one word
    const int32_t* plen;
    const int* own_per;
};

template <int D>
__global__ __launch_bounds__(kMergeRows * SSQ_WAVE) void k_merge_flat(const MergeFlat p) {
    constexpr int E = D / SSQ_WAVE, kMl = 3;      // n1 <= 128, n2 <= 32
    constexpr int kAhead = 8, kAheadOwn = 2;      // most sequences have one or two pieces; unwritten ones cost their bytes
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & (SSQ_WAVE - 1);
    const int64_t n_rows = (int64_t)a.batch * a.num_q_heads * a.q_len;
    const int64_t at_row = (int64_t)blockIdx.x * kMergeRows + __builtin_amdgcn_readfirstlane(threadIdx.x / SSQ_WAVE);
    if (at_row >= n_rows) return;  // whole waves
    const int rid = (int)at_row;
    const int bh = rid / a.q_len, qi = rid - bh * a.q_len, b = bh / a.num_q_heads, h = bh - b * a.num_q_heads;
    auto o_of = [&](const float* part, int i, float (&o)[E]) {
        const float* src = part + ((int64_t)i * n_rows + rid) * D + lane * E;
        if constexpr (E == 2) {
            const float2 x = *reinterpret_cast<const float2*>(src);
            o[0] = x.x; o[1] = x.y;
        } else {
            o[0] = src[0];
        }
    };
    float m[kMl], l[kMl], o1[kAhead][E], o2[kAheadOwn][E];
#pragma unroll
    for (int i = 0; i < kMl; ++i) {
        const int s = i * SSQ_WAVE + lane, n = s < p.n1 ? p.n1 : p.n2;
        const float* part = s < p.n1 ? p.pre : p.own;
        m[i] = -INFINITY;
        l[i] = 0.f;
        if (s < p.n1 + p.n2) {
            const float* src = part + (int64_t)n * n_rows * D + (int64_t)(s < p.n1 ? s : s - p.n1) * n_rows + rid;
            m[i] = src[0];
            l[i] = src[(int64_t)n * n_rows];
        }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < p.n1) o_of(p.pre, i, o1[i]);  // uniform
#pragma unroll
    for (int i = 0; i < kAheadOwn; ++i)
        if (i < p.n2) o_of(p.own, i, o2[i]);
    int n1 = 0, n2 = 0;  // those with tokens, as the kernel cut them
    if (p.n1) {
        const int len = max(0, min(p.plen[0], p.pcap)), per = ssq_prefix_slice(len, p.n1);
        n1 = per ? (ssq_prefix_tiles(len) + per - 1) / per : 0;
    }
    if (p.n2) {
        const int per = p.own_per[0];
        n2 = (ssq_prefix_tiles(max(0, min(a.seq_lens[b], a.seq_len))) + per - 1) / per;
    }
    float M = -INFINITY, L = 0.f, w[kMl];
#pragma unroll
    for (int i = 0; i < kMl; ++i) {
        const int s = i * SSQ_WAVE + lane;
        if (s < p.n1 ? s >= n1 : s - p.n1 >= n2) m[i] = -INFINITY;
        M = fmaxf(M, m[i]);
    }
    M = ssq_wave_max(M);
#pragma unroll
    for (int i = 0; i < kMl; ++i) {
        w[i] = m[i] == -INFINITY ? 0.f : __expf(m[i] - M);
        L += m[i] == -INFINITY ? 0.f : l[i] * w[i];
    }
    L = ssq_wave_sum(L);
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    auto weight = [&](int s) {
        const float x = s < SSQ_WAVE ? w[0] : s < 2 * SSQ_WAVE ? w[1] : w[2];  // uniform
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), s & (SSQ_WAVE - 1)));
    };
    // at weight 0 too: an infinite or NaN value counts as in one pass over all tokens
    auto add = [&](const float* part, int first, int n, const auto& ahead) {
        constexpr int kHave = sizeof(ahead) / sizeof(ahead[0]);
#pragma unroll
        for (int i = 0; i < kHave; ++i) {
            if (i >= n) continue;  // uniform
            const float f = weight(first + i);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += ahead[i][e] * f;
        }
        for (int i0 = kHave; i0 < n; i0 += kAhead) {
            float x[kAhead][E];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (i0 + i < n) o_of(part, i0 + i, x[i]);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (i0 + i >= n) continue;
                const float f = weight(first + i0 + i);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += x[i][e] * f;
            }
        }
    };
    add(p.pre, 0, n1, o1);
    add(p.own, p.n1, n2, o2);
    const int64_t at = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)qi * a.o_sl + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = M == -INFINITY ? 0.f : o[e] / L;  // a row with nothing to attend gives 0
    if (E == 2 && p.pair) {
        const uint32_t x = a.v_dtype == SSQ_BF16 ? pf_pack<false>(o[0], o[E - 1]) : pf_pack<true>(o[0], o[E - 1]);
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + at) = x;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) ssq_store_elem(a.out, a.v_dtype, at + e, o[e]);
    }
    if (a.lse && lane == 0) a.lse[rid] = M == -INFINITY ? -INFINITY : M + logf(L);
}

struct PrefixPlan {
    int chunk, n1, n1_last, n2;
    int len1, len1_last, len2;  // tokens of a split
    size_t pre_bytes, own_bytes;
    bool fast;  // the matrix-core kernel
    SsqPrefixParams fp;
};

int kept_dims(const ssq_decode_args& d) {
    return (__builtin_popcountll(d.heavy_mask[0]) + __builtin_popcountll(d.heavy_mask[1])) * d.block_dim;
}

// Problems of the matrix-core kernel: pages of whole 16-token pieces, byte codes, codewords of 2, 4 or 8 dims, at most
// half of the dims kept.
bool fast_shape(const ssq_decode_args& d) {
    if (d.kernel != 0 || (d.head_dim != 64 && d.head_dim != 128) || d.value_dim != d.head_dim) return false;
    if (d.block_dim != 2 && d.block_dim != 4 && d.block_dim != 8) return false;
    if (d.n_centroids > 256 || (d.code_bits != 0 && d.code_bits != 8) || d.page_size % 16) return false;
    if (const int kept = kept_dims(d)) {  // compact rows of whole 8-byte pieces in the values' dtype
        if (kept > d.head_dim / 2 || kept % 4 || d.pt_dense || d.pt_dtype != d.v_dtype) return false;
        if ((uintptr_t)d.pt % 8 || d.pt_sb % 4 || d.pt_sh % 4 || d.pt_st % 4) return false;
    }
    if (d.v_dtype != SSQ_BF16 && d.v_dtype != SSQ_F16) return false;
    if ((uintptr_t)d.cent % 16 || d.cent_sh % 4) return false;
    const int64_t cal = d.n_blocks >= 16 ? 16 : d.n_blocks, unit = d.code_bits ? 4 : 1;  // code rows load in pieces
    if ((uintptr_t)d.codes % cal || (d.c_sb * unit) % cal || (d.c_sh * unit) % cal || (d.c_st * unit) % cal) return false;
    if ((uintptr_t)d.v % 16 || d.v_sb % 8 || d.v_sh % 8 || d.v_st % 8) return false;
    return d.v_st >= 0 && d.v_st <= 1 << 22;  // 32-bit offsets inside a page
}

// How the prefix and the own tokens are cut into items (ssq_prefix_mfma.h).
void fast_plan(const ssq_prefix_args& a, PrefixPlan& pl) {
    const ssq_decode_args& d = a.dec;
    SsqPrefixParams& f = pl.fp;
    f = SsqPrefixParams{};
    f.a = d;
    if (d.code_bits == 8) {  // 8-bit words are the byte rows
        f.a.c_sb *= 4; f.a.c_sh *= 4; f.a.c_st *= 4;
    }
    f.ptab = a.prefix_table;
    f.plen = a.prefix_len;
    f.pcap = a.prefix_cap;
    f.G = d.num_q_heads / d.num_kv_heads;
    const int per_b = f.G * d.q_len;
    f.rows = per_b * d.batch;
    const int cus = ssq_device_cus();
    f.n_wg = cus / d.num_kv_heads > 0 ? cus / d.num_kv_heads : 1;
    while ((16 << f.psh) < d.page_size) ++f.psh;
    f.q_vec = d.q_dtype != SSQ_F32 && (uintptr_t)d.q % 16 == 0 && d.q_sb % 8 == 0 && d.q_sh % 8 == 0 && d.q_sl % 8 == 0;
    const bool split = !(d.q_dtype == SSQ_BF16 && d.v_dtype == SSQ_BF16) && !(d.q_dtype == SSQ_F16 && d.v_dtype == SSQ_F16);
    f.kept = kept_dims(d);
    f.own_rg = (per_b + 31) / 32;
    f.pre_nr = 1;
    if (a.prefix_cap > 0) {
        // Rows of an item and slices of the prefix: the fewest hundredths of a microsecond by what items measured: 10 us
        // and 1.35 per tile of a wave with 64 rows, 3 and 0.98 with 32 (twice the gathers, but fewer queries to move
        // through LDS); and 6 where the prefix's items leave a KV head too few workgroups for its own items, which then
        // wait for one another.  8 heads of 128 dims, 4 query heads each, 64 own tokens, us with 32 and with 64 rows:
        // 16 sequences on 4,096 tokens 19.7 and 21.6, on 65,536 53.4 and 49.2; 48 sequences 25.9 and 25.8, 122 and 95.6.
        // The costs are those of 128 dims; at 64 the choice is the same but for close calls: 14.6 and 15.8, 41.6 and
        // 37.4; 20.2 and 19.9, 94.2 and 74.9; of 2 heads with 7 each, 128 sequences on 8,192 28.8, the choice, and 26.2.
        // Workgroups left for the own items or not: 8 sequences on 4,096 tokens 18.6 and 26.0, 48 on 1,000 19.8
        // and 26.1.  Split queries and kept dims leave no registers for 64 rows.
        const int most = split || f.kept || f.rows <= 32 ? 1 : 2, tiles = (a.prefix_cap + 31) / 32;
        // pieces of two tiles, of sequences taken to fill half of their tables
        const int64_t own_items = d.seq_len > 0 ? (int64_t)d.batch * f.own_rg * ((d.seq_len + 127) / 128) : 0;
        const int64_t room = f.n_wg - (own_items + 3) / 4;
        int64_t best = INT64_MAX;
        for (int nr = 1; nr <= most; ++nr) {
            const int n_rg = (f.rows + 32 * nr - 1) / (32 * nr);
            const int n1_most = 4 * f.n_wg / n_rg;  // about four rounds
            for (int n1 = 1; n1 <= 128 && (n1 == 1 || (n1 * 4 <= tiles && n1 <= n1_most)); ++n1) {
                const int items = n_rg * n1, rounds = (items + f.n_wg - 1) / f.n_wg;
                const int wave = ((tiles + n1 - 1) / n1 + 3) / 4;
                const int64_t cost = (int64_t)rounds * (nr == 1 ? 300 + 98 * (int64_t)wave : 1000 + 135 * (int64_t)wave) +
                                     (own_items && items > room ? 600 : 0);
                if (cost < best) {
                    best = cost;
                    f.pre_nr = nr;
                    f.n_rg = n_rg;
                    f.n1 = n1;
                }
            }
        }
    }
    if (d.seq_len > 0) {
        // The fewest tiles of a wave's piece: 2 (a piece's own cost is about 5), as many as keep the partials to
        // 32 per row, and to 16 per wave where every sequence is as long as the tables.
        const int64_t tiles = ssq_prefix_tiles(d.seq_len), waves = 4 * (int64_t)f.n_wg;
        int64_t least = 2;
        if ((tiles + 31) / 32 > least) least = (tiles + 31) / 32;
        const int64_t all = d.batch * (int64_t)f.own_rg * tiles;
        if ((all + 16 * waves - 1) / (16 * waves) > least) least = (all + 16 * waves - 1) / (16 * waves);
        f.own_min = (int)(least < tiles ? least : tiles);
        f.n2 = (int)((tiles + f.own_min - 1) / f.own_min);
    }
    const int64_t rows = (int64_t)d.batch * d.num_q_heads * d.q_len;
    pl.n1 = pl.n1_last = f.n1;
    pl.n2 = f.n2;
    pl.pre_bytes = ((size_t)(rows * f.n1 * (d.value_dim + 2) * 4) + 255) & ~(size_t)255;  // 16-byte stores in both parts
    pl.own_bytes = f.n2 ? (size_t)(rows * f.n2 * (d.value_dim + 2) * 4) + 256 : 0;  // and the pieces' size
}

// where the kernel leaves the pieces' size for the merge: behind the own tokens' partials
int* own_per_of(const PrefixPlan& pl, void* workspace) {
    return reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + pl.pre_bytes + pl.own_bytes - 256);
}

int fast_launch(const PrefixPlan& pl, void* workspace, hipStream_t st) {
    SsqPrefixParams f = pl.fp;
    f.pre = reinterpret_cast<float*>(workspace);
    f.own = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + pl.pre_bytes);
    const ssq_decode_args& d = f.a;
    if (f.n2) f.own_per = own_per_of(pl, workspace);
    const bool bf = d.v_dtype == SSQ_BF16;
    if (d.q_dtype != d.v_dtype) {
        if (f.kept) return bf ? ssq_prefix_split_bf16_mixed(f, st) : ssq_prefix_split_f16_mixed(f, st);
        return bf ? ssq_prefix_split_bf16(f, st) : ssq_prefix_split_f16(f, st);
    }
    if (f.kept) return bf ? ssq_prefix_bf16_mixed(f, st) : ssq_prefix_f16_mixed(f, st);
    return bf ? ssq_prefix_bf16(f, st) : ssq_prefix_f16(f, st);
}

// sequences [b0, b0 + n) at query position qi as one sequence of n query rows per head, attending the prefix
ssq_decode_args prefix_part(const ssq_prefix_args& a, int b0, int n, int qi) {
    ssq_decode_args d = a.dec;
    const int size = d.q_dtype == SSQ_F32 ? 4 : 2;
    d.q = reinterpret_cast<const void*>((uintptr_t)d.q + (uintptr_t)(((int64_t)b0 * d.q_sb + (int64_t)qi * d.q_sl) * size));
    d.q_sl = d.q_sb;
    d.q_sb = 0;
    d.batch = 1;
    d.q_len = n;
    d.mask = nullptr;
    d.lse = nullptr;
    d.block_table = a.prefix_table;
    d.bt_sb = 0;
    d.seq_lens = a.prefix_len;
    d.seq_len = a.prefix_cap;
    d.num_splits = 0;
    return d;
}

int check(const ssq_prefix_args* a) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_prefix_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_prefix_args size %u != library's %zu", a->struct_size, sizeof(ssq_prefix_args));
    ssq_decode_args d = a->dec;
    if (d.struct_size != sizeof(ssq_decode_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_decode_args size %u != library's %zu", d.struct_size, sizeof(ssq_decode_args));
    SSQ_REQUIRE(d.layout == SSQ_PAGED, "a shared prefix needs the paged layout");
    SSQ_REQUIRE(d.scores == nullptr, "decode with a shared prefix writes no raw scores");
    SSQ_REQUIRE(d.kernel == 0 || d.kernel == 1, "kernel must be 0 or 1");
    SSQ_REQUIRE(d.num_splits == 0, "num_splits must be 0");
    SSQ_REQUIRE(a->prefix_cap >= 0 && a->prefix_cap <= 1 << 30, "prefix_cap must be in [0, 2^30]");
    SSQ_REQUIRE(d.seq_len <= 1 << 30, "seq_len must be at most 2^30");
    SSQ_REQUIRE(a->prefix_cap == 0 || (a->prefix_table && a->prefix_len), "a prefix needs prefix_table and prefix_len");
    SSQ_REQUIRE((int64_t)d.batch * (d.num_q_heads > 0 ? d.num_q_heads : 1) <= (1 << 24) && d.q_len <= 1 << 16 &&
                    (int64_t)d.batch * d.num_q_heads * d.q_len <= 0x7fffffff,
                "too many query rows");
    SSQ_REQUIRE((int64_t)d.batch * (d.num_kv_heads > 0 ? d.num_kv_heads : 1) <= 65535, "batch * num_kv_heads > 65535");
    if (d.seq_len == 0 || !d.block_table) {  // no own tokens: the rest is checked as the prefix's problem
        SSQ_REQUIRE(d.seq_len == 0, "paged layout needs block_table and seq_lens");
        static const int32_t none = 0;
        d.block_table = &none;
        d.seq_lens = &none;
    }
    return ssq_decode_validate(&d);
}

int make_plan(const ssq_prefix_args& a, PrefixPlan& pl) {
    const ssq_decode_args& d = a.dec;
    pl = PrefixPlan{};
    pl.chunk = d.batch;
    pl.fast = fast_shape(d);
    if (pl.fast) {
        fast_plan(a, pl);
        return SSQ_OK;
    }
    if (a.prefix_cap > 0) {
        // up to 64 query rows of a KV head take the matrix-core decode kernels (16 rows per pass over the
        // pages); any number the generic one (8 rows per pass)
        const int G = d.num_q_heads / d.num_kv_heads;
        if (d.kernel == 0 && (int64_t)G * d.batch > 64) pl.chunk = 64 / G > 0 ? 64 / G : 1;
        if (pl.chunk > d.batch) pl.chunk = d.batch;
        const int rest = d.batch % pl.chunk ? d.batch % pl.chunk : pl.chunk;
        const ssq_decode_args whole = prefix_part(a, 0, pl.chunk, 0), last = prefix_part(a, d.batch - rest, rest, 0);
        pl.n1 = ssq_decode_partial_splits(&whole, pl.len1);
        pl.n1_last = ssq_decode_partial_splits(&last, pl.len1_last);
        if (pl.n1 == 0 || pl.n1_last == 0) return SSQ_ERR_UNSUPPORTED;
        const int64_t rows = (int64_t)d.num_q_heads * ((int64_t)(d.batch - rest) * pl.n1 + (int64_t)rest * pl.n1_last);
        pl.pre_bytes = (size_t)(rows * d.q_len * (d.value_dim + 2) * 4);
    }
    if (d.seq_len > 0) {
        pl.n2 = ssq_decode_partial_splits(&d, pl.len2);
        if (pl.n2 == 0) return SSQ_ERR_UNSUPPORTED;
        pl.own_bytes = (size_t)d.batch * d.num_q_heads * d.q_len * pl.n2 * (d.value_dim + 2) * 4;
    }
    return SSQ_OK;
}

}  // namespace

// A call's plan, for tests that mean to reach a form of the matrix-core kernel (zeros where it does not serve the
// call): rows of a prefix item / 32, row groups, slices, workgroups per KV head, own pieces at most, their fewest tiles.
int ssq_decode_prefix_plan(const ssq_prefix_args* a, int32_t* out) {
    PrefixPlan pl;
    int rc = check(a);
    if (rc == SSQ_OK) rc = make_plan(*a, pl);
    if (rc) return rc;
    const SsqPrefixParams f = pl.fast ? pl.fp : SsqPrefixParams{};
    const int32_t v[6] = {f.n1 ? f.pre_nr : 0, f.n_rg, f.n1, f.n_wg, f.n2, f.own_min};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
    return SSQ_OK;
}

extern "C" size_t ssq_decode_prefix_workspace_size(const ssq_prefix_args* a) {
    PrefixPlan pl;
    if (check(a) != SSQ_OK || make_plan(*a, pl) != SSQ_OK) return 0;
    return pl.pre_bytes + pl.own_bytes;
}

extern "C" int ssq_decode_prefix(const ssq_prefix_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc) return rc;
    const ssq_decode_args& d = a->dec;
    PrefixPlan pl;
    rc = make_plan(*a, pl);
    if (rc) return rc;
    SSQ_REQUIRE(workspace_bytes >= pl.pre_bytes + pl.own_bytes, "workspace too small: %zu < %zu bytes", workspace_bytes,
                pl.pre_bytes + pl.own_bytes);
    SSQ_REQUIRE(workspace || pl.pre_bytes + pl.own_bytes == 0, "workspace is NULL");
    hipStream_t st = (hipStream_t)stream;
    const float* pre = reinterpret_cast<const float*>(workspace);
    const float* own = reinterpret_cast<const float*>(reinterpret_cast<char*>(workspace) + pl.pre_bytes);
    const int64_t rows = (int64_t)d.batch * d.num_q_heads * d.q_len;
    const dim3 grid((unsigned)((rows + kMergeRows - 1) / kMergeRows)), block(kMergeRows * SSQ_WAVE);
    if (pl.fast) {
        if (pl.n1 || pl.n2) rc = fast_launch(pl, workspace, st);
        if (rc) return rc;
        MergeFlat m{};
        m.a = d;
        m.pre = pre; m.own = own;
        m.n1 = pl.n1; m.n2 = pl.n2;
        m.plen = a->prefix_len;
        m.pcap = a->prefix_cap;
        m.pair = (uintptr_t)d.out % 4 == 0 && d.o_sb % 2 == 0 && d.o_sh % 2 == 0 && d.o_sl % 2 == 0;
        if (pl.n2) m.own_per = own_per_of(pl, workspace);
        if (d.head_dim == 64) hipLaunchKernelGGL(k_merge_flat<64>, grid, block, 0, st, m);
        else hipLaunchKernelGGL(k_merge_flat<128>, grid, block, 0, st, m);
        return ssq_check_hip(hipGetLastError(), "k_merge_flat launch");
    }
    MergeParams m{};
    m.a = d;
    m.pre = pre;
    m.chunk = pl.chunk;
    m.n1 = pl.n1;
    m.n1_last = pl.n1_last;
    m.own = own;
    m.n2 = pl.n2;
    m.len1 = pl.len1;
    m.len1_last = pl.len1_last;
    m.len2 = pl.len2;
    m.plen = a->prefix_len;
    if (pl.n1) {
        char* at = reinterpret_cast<char*>(workspace);
        for (int qi = 0; qi < d.q_len; ++qi)
            for (int b0 = 0; b0 < d.batch; b0 += pl.chunk) {
                const int n = d.batch - b0 < pl.chunk ? d.batch - b0 : pl.chunk;
                ssq_decode_args part = prefix_part(*a, b0, n, qi);
                part.num_splits = b0 + pl.chunk >= d.batch ? pl.n1_last : pl.n1;
                const size_t bytes = (size_t)d.num_q_heads * n * part.num_splits * (d.value_dim + 2) * 4;
                rc = ssq_decode_partials(&part, at, bytes, st);
                if (rc) return rc;
                at += bytes;
            }
    }
    if (pl.n2) {
        ssq_decode_args own = d;
        own.num_splits = pl.n2;
        own.lse = nullptr;
        rc = ssq_decode_partials(&own, const_cast<float*>(m.own), pl.own_bytes, st);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(k_merge_prefix, grid, block, 0, st, m);
    return ssq_check_hip(hipGetLastError(), "k_merge_prefix launch");
}
