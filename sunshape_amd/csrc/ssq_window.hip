// Causal attention over pages with a sliding window, sinks and 8-bit values (ssq_decode_window): the checks and the plan
// of a call.  The kernel is in ssq_window.h, its instantiations in ssq_window_*.hip.
#include "ssq_window.h"

#include <limits.h>

int ssq_decode_validate(const ssq_decode_args* a);

namespace {

struct Plan {
    SsqWindowParams p;
    size_t part_bytes, bytes;
};

int check(const ssq_window_args* a) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_window_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_window_args size %u != library's %zu", a->struct_size, sizeof(ssq_window_args));
    ssq_decode_args d = a->dec;
    const bool v8 = d.v_dtype == SSQ_E4M3;
    SSQ_REQUIRE(d.layout == SSQ_PAGED, "decode_window takes pages");
    SSQ_REQUIRE(d.v, "decode_window needs values");
    SSQ_REQUIRE(!d.scores && !d.mask, "decode_window takes no mask and gives no scores");
    SSQ_REQUIRE(d.seq_len >= d.page_size, "decode_window needs a block table of at least one page");
    SSQ_REQUIRE(a->window >= 0 && a->sinks >= 0, "window and sinks must not be negative");
    SSQ_REQUIRE(a->out_dtype >= SSQ_F32 && a->out_dtype <= SSQ_F16, "bad out_dtype");
    SSQ_REQUIRE(a->num_pages >= 1 && a->num_pages <= INT_MAX, "bad num_pages");
    SSQ_REQUIRE(!v8 || a->v_scale, "8-bit values need v_scale");
    SSQ_REQUIRE(v8 || !a->v_scale, "v_scale goes with 8-bit values");
    SSQ_REQUIRE(d.batch >= 0 && d.num_q_heads >= 0 && d.q_len >= 0 && d.num_kv_heads >= 1, "bad batch/heads/q_len");
    SSQ_REQUIRE((int64_t)d.batch * (d.num_q_heads > 0 ? d.num_q_heads : 1) <= (1 << 24) && d.q_len <= 1 << 20 &&
                    (int64_t)d.batch * d.num_q_heads * d.q_len <= 1 << 30,
                "too many query rows");
    if (v8) d.v_dtype = SSQ_F16;  // the decode's checks know 16 bits, and calls with something to do
    if (d.batch == 0) d.batch = 1;
    if (d.num_q_heads == 0) d.num_q_heads = d.num_kv_heads;
    if (d.q_len == 0) d.q_len = 1;
    int rc = ssq_decode_validate(&d);
    if (rc) return rc;
    SSQ_UNSUPPORTED(!d.heavy_mask[0] && !d.heavy_mask[1], "decode_window serves codecs without passthrough blocks");
    SSQ_UNSUPPORTED((d.head_dim == 64 || d.head_dim == 128) && d.value_dim == d.head_dim,
                    "decode_window serves head_dim 64 or 128 with value_dim the same, not %d and %d", d.head_dim, d.value_dim);
    SSQ_UNSUPPORTED(d.block_dim == 2 || d.block_dim == 4 || d.block_dim == 8, "decode_window serves block_dim 2, 4 or 8, not %d",
                    d.block_dim);
    SSQ_UNSUPPORTED(d.n_centroids <= 256 && d.code_bits == 0, "decode_window serves byte codes (at most 256 codewords)");
    SSQ_UNSUPPORTED(v8 || d.v_dtype == SSQ_BF16 || d.v_dtype == SSQ_F16, "decode_window serves values of 8 or 16 bits");
    SSQ_UNSUPPORTED(d.page_size >= 16, "decode_window serves page sizes from 16, not %d", d.page_size);  // and they divide 256
    SSQ_UNSUPPORTED(d.seq_len <= 1 << 30, "the block table is too long");
    SSQ_REQUIRE((uintptr_t)d.cent % 16 == 0 && d.cent_sh % 4 == 0, "centroids must be 16-byte aligned");
    const int64_t piece = d.n_blocks / 4;  // bytes of a token's codes that a lane loads at once
    SSQ_REQUIRE((uintptr_t)d.codes % piece == 0 && d.c_sb % piece == 0 && d.c_sh % piece == 0 && d.c_st % piece == 0,
                "code rows must be aligned to %lld bytes", (long long)piece);
    const int64_t per = v8 ? 16 : 8;
    SSQ_REQUIRE((uintptr_t)d.v % 16 == 0 && d.v_sb % per == 0 && d.v_sh % per == 0 && d.v_st % per == 0,
                "value rows must be 16-byte aligned");
    SSQ_REQUIRE(d.v_st >= 0 && d.v_st <= 1 << 22, "the values' dim stride must be at most 2^22");
    SSQ_REQUIRE(d.c_sb >= 0 && d.c_sb < 1ll << 31 && d.c_st >= 0 && d.c_st <= 1 << 22 && d.v_sb >= 0 && d.v_sb < 1ll << 30 &&
                    a->vs_sb >= 0 && a->vs_sb < 1ll << 30,
                "page strides must be below 2^30 elements");
    SSQ_UNSUPPORTED(d.num_kv_heads <= 1 << 16, "too many KV heads");
    return SSQ_OK;
}

// The most tiles of tt tokens of an item of `rows` rows (any length that the tables hold; a window's tiles depend on where it ends).
int64_t most_tiles(const SsqWindowParams& p, int tt, int rows) {
    const int64_t all = ((int64_t)p.a.seq_len + tt - 1) / tt;
    if (p.window == INT_MAX) return all;
    const int64_t seen = ((int64_t)p.window + rows + tt - 1) / tt + 1 + ((int64_t)p.sinks + tt - 1) / tt;
    return seen < all ? seen : all;
}

// A workgroup's waves on one item at a time, joined in LDS and written out, or every wave an equal share of all tiles and a
// second launch that joins them?  Together an item takes as many rounds as it has tiles / 8, and items wait for the longest
// one's; shares cost the join, about 9 us.  By what calls took, tenths of a microsecond: a round of 8 tiles 26 where all CUs
// have one to load, 19 where less than three quarters have, 23 where groups of rows share the tokens; 50 an item, 80 a call; a tile
// of a share 32 (24), 170 a call.  Measured us together and in shares, 32 / 8 heads of 128: 1 sequence of 1,100 tokens 15.6 and
// 18.1, of 4,100 26.8 and 18.3; 16 of 2,100 20.7 and 25.5; 48 of 4,100 59.7 and 57.8, of 600 23.9 and 24.7; 128 of 600 43.7 and
// 37.9; 16 times 5 rows under a window of 1,001 22.2 and 33.9; 64 under one of 4,096 70.4 and 73.5; 14 / 2 heads of 64: 128 of
// 4,100 26.9 and 36.0.  Past 80 tiles lengths may differ by more than a round is worth (48 ragged ones of up to 8,192 92.0 and 82.3).
bool team(const SsqWindowParams& p, int64_t most) {
    if (most > 80) return false;
    const int64_t turns = (p.items + p.n_wg - 1) / p.n_wg;
    const bool shared = p.rgroups > 1;
    const int64_t round = shared ? 23 : 4 * (int64_t)p.items >= 3 * (int64_t)p.n_wg ? 26 : 19;
    const int64_t together = turns * ((most > 8 ? most : 8) * round / 8 + 50) + 80;
    const int64_t shares = 170 + (shared ? 24 : 32) * (int64_t)p.items * (most + p.fixed) / (p.n_wg * kWinWaves);
    return together <= shares;
}

// Items of 256 rows, whose workgroups decode a tile once for all of them?  They take longer to start and to join, and leave
// waves idle where rows end.  By what calls took, tenths of a microsecond: head_dim 128 a tile of 64 tokens 24 a wave of 16 rows
// and 240 a call, a tile of 32 tokens 15 a workgroup of 256 and 370 a call; head_dim 64 16 and 180, a tile of 64 18 and 270.  Measured
// us by 16 rows and by 256, 32 / 8 heads of 128: 1 sequence of 16,384 and 33 new tokens 50 and 57, 64 69 and 60, 512 338 and 235;
// 64 of 2,048 29 and 42; 32 times 64 of 8,192 697 and 480; 512 under a window of 1,024 49 and 48, of 4,096 97 and 89, 8 times 229
// and 149; 16 prompts of 512 468 and 130; 14 / 2 heads of 64: 300 of 4,096 33.1 and 32.7, of 16,384 76 and 62.
bool wide(const SsqWindowParams& p) {
    if (p.rows <= kWinWideRows / 2) return false;
    const bool small = p.a.head_dim == 64;
    auto tiles = [&](int rows, int tt) {  // of all items of a KV head
        int64_t seen = p.a.seq_len;
        if (p.window != INT_MAX) {
            const int64_t most = (int64_t)p.window + p.sinks + rows / p.G + tt;
            if (most < seen) seen = most;
        }
        return (int64_t)p.a.batch * ((p.rows + rows - 1) / rows) * ((seen + tt - 1) / tt);
    };
    const int64_t few = (small ? 180 : 240) + (small ? 16 : 24) * tiles(kWinRows, 64) / (p.n_wg * kWinWaves);
    const int64_t many = (small ? 270 : 370) + (small ? 18 : 15) * tiles(kWinWideRows, small ? 64 : 32) / p.n_wg;
    return many <= few;
}

int make_plan(const ssq_window_args& a, Plan& pl) {
    const ssq_decode_args& d = a.dec;
    SsqWindowParams& p = pl.p;
    p = SsqWindowParams{};
    p.a = d;
    p.window = a.window > 0 ? a.window : INT_MAX;
    p.sinks = a.sinks;
    p.out_dtype = a.out_dtype;
    p.n_pages = (int)a.num_pages;
    p.v_scale = a.v_scale;
    p.vs_sb = a.vs_sb;
    p.vs_sh = a.vs_sh;
    p.G = d.num_q_heads / d.num_kv_heads;
    p.rows = p.G * d.q_len;
    const int cus = ssq_device_cus();
    p.n_wg = cus / d.num_kv_heads > 0 ? cus / d.num_kv_heads : 1;
    p.least = 2;
    const bool many = wide(p);
    // (An item of 256 rows costs 5 to 8 tiles of its own.  With 5 and 8, in turn: 16 prompts of 512 tokens 130 and 146 us, one of 8,192
    // 900 and 860, 4 of 2,048 287 and 275, 512 tokens of 16,384 235 both.)
    p.fixed = many ? 5 : 2;
    p.item_rows = many ? kWinWideRows : kWinRows;
    p.rgroups = (p.rows + p.item_rows - 1) / p.item_rows;
    p.items = d.batch * p.rgroups;
    const int tt = many ? 4096 / d.head_dim : d.v_dtype == SSQ_E4M3 ? 64 : 32;
    const int64_t most = most_tiles(p, tt, p.item_rows);
    p.form = many ? kWinWide : team(p, most) ? kWinTeam : kWinShares;
    // the cost axis that shares are cut from has 32 bits
    SSQ_UNSUPPORTED(p.form == kWinTeam || p.items * (most + p.fixed) < 1ll << 31, "too many query rows for so long a context");
    if (p.form == kWinTeam && p.n_wg > p.items) p.n_wg = p.items;
    p.workers = p.form == kWinShares ? p.n_wg * kWinWaves : p.n_wg;
    while ((16 << p.psh) < d.page_size) ++p.psh;
    const int per = d.q_dtype == SSQ_F32 ? 4 : 8;
    p.q_vec = (uintptr_t)d.q % 16 == 0 && d.q_sb % per == 0 && d.q_sh % per == 0 && d.q_sl % per == 0;
    const int size = p.out_dtype == SSQ_F32 ? 16 : 8;
    p.out_vec = (uintptr_t)d.out % size == 0 && d.o_sb % 4 == 0 && d.o_sh % 4 == 0 && d.o_sl % 4 == 0;
    pl.part_bytes = p.form == kWinTeam ? 0 : (size_t)d.num_kv_heads * p.workers * 2 * p.item_rows * (d.value_dim + 2) * 4;
    pl.bytes = p.form == kWinTeam ? 0 : pl.part_bytes + (size_t)p.items * 8;
    return SSQ_OK;
}

}  // namespace

extern "C" size_t ssq_decode_window_workspace_size(const ssq_window_args* a) {
    if (check(a) != SSQ_OK || a->dec.batch == 0 || a->dec.num_q_heads == 0 || a->dec.q_len == 0) return 0;
    Plan pl;
    return make_plan(*a, pl) == SSQ_OK ? pl.bytes : 0;
}

extern "C" int ssq_decode_window(const ssq_window_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(a);
    if (rc) return rc;
    const ssq_decode_args& d = a->dec;
    if (d.batch == 0 || d.num_q_heads == 0 || d.q_len == 0) return SSQ_OK;
    Plan pl;
    rc = make_plan(*a, pl);
    if (rc) return rc;
    SSQ_REQUIRE(workspace_bytes >= pl.bytes && (workspace || pl.bytes == 0), "workspace too small: %zu < %zu bytes", workspace_bytes,
                pl.bytes);
    SSQ_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
    pl.p.part = reinterpret_cast<float*>(workspace);
    pl.p.meta = reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + pl.part_bytes);
    hipStream_t st = (hipStream_t)stream;
    const bool small = d.head_dim == 64;
    switch (d.v_dtype) {
        case SSQ_E4M3: return small ? ssq_window_64_e4m3(pl.p, st) : ssq_window_128_e4m3(pl.p, st);
        case SSQ_BF16: return small ? ssq_window_64_bf16(pl.p, st) : ssq_window_128_bf16(pl.p, st);
        default: return small ? ssq_window_64_f16(pl.p, st) : ssq_window_128_f16(pl.p, st);
    }
}
