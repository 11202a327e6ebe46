// ssq_decode_window for many query rows of a sequence and KV head (a prompt's chunk): k_window_wide.  Included by ssq_window.h.
//
// The formulas and the numbers' forms are k_window's: S^T = K Q^T and O^T = V^T P^T, K in two f16 parts, probabilities in 16 bits
// with the page's scale in them.  What differs is who decodes.  Sixteen rows at a time, a token's codewords are gathered
// from the codebook once per 16 rows: a chunk of 512 tokens (4 heads a KV head) spent 44 us of 87 in the LDS, two thirds of
// it bank conflicts, and 46 in VALU instructions, with 21 us of matrix products.  Here eight waves of 32 rows share a tile of
// 4096 / D tokens: each thread gathers 8 dims of a token and takes 8 tokens of a value dim, converted, to LDS rows that
// v_mfma_f32_32x32x16 operands are read from without conflicts.  The codebook leaves room for one tile: its successor is
// gathered into registers while the tile is used, and written between two barriers.
//
// What bounds it: an operand of 1 KiB from LDS feeds one product of 32 cycles, so four SIMDs' products take what the LDS
// can give; a step of 32 tokens (head_dim 128) takes 1.5 us, its products 0.7, its LDS reads 0.8, the probabilities 0.4.  Beside that about
// 37 us of start, partials and join.  Measured us by 16 rows and here: 512 new tokens of 16,384 seeing 4,096 97 and 88, seeing
// all 338 and 234; 16 prompts of 512 468 and 134 (what is chosen: wide() in ssq_window.hip).  Eight operands ahead in place of four: no
// gain.  Partials in the registers' order (a store is 1 KiB, the join reads what it wrote) 95 -> 89; by rows: 16 bytes each.
//
// Matrix row m = 8 a + 4 g + i (a lane's register 4 a + i in group g = lane / 32) of a score block of 32 is token
// 16 (a / 2) + 8 g + 4 (a % 2) + i: registers 8 t .. 8 t + 7 are then the P^T operand of the block's 16 tokens from 16 t.
#pragma once

namespace {

typedef float w16f __attribute__((ext_vector_type(16)));

template <int VT>
__device__ __forceinline__ w16f wide_mfma(const uint4& a, const uint4& b, w16f c) {
    if constexpr (VT == SSQ_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(w8b, a), __builtin_bit_cast(w8b, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(w8h, a), __builtin_bit_cast(w8h, b), c, 0, 0, 0);
}
__device__ __forceinline__ w16f wide_mfma_32(float a, float b, w16f c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
// a barrier for LDS alone: global loads stay in flight
__device__ __forceinline__ void wide_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int D>
struct WideLds {
    static constexpr int TT = 4096 / D;              // tokens of a tile: 8 dims of a token a thread
    static constexpr int kBook = D * 256 * 4;
    static constexpr int kKRow = 2 * D + 16;         // bytes of a token's hi (lo) parts
    static constexpr int kLo = TT * kKRow;           // from hi to lo
    static constexpr int kVRow = 2 * TT + 16;        // bytes of a value dim
    static constexpr int kK = kBook, kV = kK + 2 * kLo, kScale = kV + D * kVRow, kFlag = kScale + 32, kRed = kFlag + 4 * kWinWaves,
                         kPerm = kRed + 4 * kWinWaves, kWild = kPerm + 2 * D, kTotal = kWild + 3 * kWinThreads;
    static constexpr int kQRow = 2 * D + 16;         // a query row on its way, 8 (4) a wave, in the tile's place
    static_assert(kWinWaves * 8 * kQRow <= 2 * kLo, "the queries' rows");
};

template <int D, int BD, int VT, int QP>
__global__ __launch_bounds__(kWinThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_window_wide(const SsqWindowParams) {
    using L = WideLds<D>;
    constexpr bool kV8 = VT == SSQ_E4M3;
    constexpr int TT = L::TT, ROWS = kWinWideRows, WR = ROWS / kWinWaves;
    constexpr int NK = D / 16, DT = D / 32, NB = TT / 32, NT = TT / 16, NE = D / 2, NC = 8 / BD;
    extern __shared__ __align__(16) unsigned char smem[];
    WinArgs p = win_args();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, grp = lane >> 5;
    const int kv = blockIdx.x % p->a.num_kv_heads, wg = blockIdx.x / p->a.num_kv_heads;
    float* red = reinterpret_cast<float*>(smem + L::kRed);
    uint16_t* perm = reinterpret_cast<uint16_t*>(smem + L::kPerm);
    float* scales = reinterpret_cast<float*>(smem + L::kScale);
    uint32_t* flags = reinterpret_cast<uint32_t*>(smem + L::kFlag);  // a wave's: some value of its piece is infinite or NaN
    unsigned char* wilds = smem + L::kWild;                          // then: a thread's 8 tokens that are NaN, inf, -inf

    const int64_t at_perm = p->a.perm[(int64_t)kv * p->a.perm_sh + min(tid, D - 1)];
    const int first_len = WinCut<TT, ROWS>::length(p, lane);
    int book_exp;
    WinCut<TT, ROWS> cut;
    WinBook<D, BD> book;
    book.load(p, kv, tid);
    if (tid < D) perm[tid] = (uint16_t)((uint64_t)at_perm < (uint64_t)D ? at_perm : D - 1);
    cut.init(p, lane, first_len);
    const int x_begin = (int)min((int64_t)wg * cut.share, (int64_t)cut.total), x_end = (int)min((int64_t)(wg + 1) * cut.share, (int64_t)cut.total);
    int x = x_begin, ahead = 0;  // the next item, and its cost position
    if (x_begin < x_end) cut.find(p, lane, x_begin, ahead, x);

    // ---- this thread's piece of a tile: 8 dims of a token, and 8 tokens of a value dim
    const int window = p->window, sinks = p->sinks, q_len = p->a.q_len, n_pages = p->n_pages, psh = p->psh;
    const int ktok = tid / (D / 8), kdim = tid % (D / 8), vdim = tid / (TT / 8), vtok = tid % (TT / 8);
    const uint32_t c_sb = (uint32_t)p->a.c_sb, c_st = (uint32_t)p->a.c_st, v_sb = (uint32_t)p->a.v_sb * (kV8 ? 1 : 2), vs_sb = (uint32_t)p->vs_sb;
    const uint8_t* cbase = p->a.codes + (int64_t)kv * p->a.c_sh + (ktok & 15) * (int64_t)c_st + kdim * NC;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(p->a.v) + ((int64_t)kv * p->a.v_sh + (int64_t)vdim * p->a.v_st + 8 * (vtok & 1)) * (kV8 ? 1 : 2);
    const float* v_scale = p->v_scale + (int64_t)kv * p->vs_sh;
    unsigned char* const kput = smem + L::kK + ktok * L::kKRow + 16 * kdim;
    unsigned char* const vput = smem + L::kV + vdim * L::kVRow + 16 * vtok;
    const unsigned char* const kget = smem + L::kK + (16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3)) * L::kKRow + 16 * grp;
    const unsigned char* const vget = smem + L::kV + col * L::kVRow + 16 * grp;

    int b = 0, row0 = 0, nr = 0, len = 0, i0 = 0, i1 = 0, slot = -1, last_tok = 0;
    WinTiles t{};
    const int32_t* table = nullptr;
    auto next = [&]() {
        p = win_args();
        for (;;) {
            const int item = __builtin_amdgcn_readfirstlane(ahead), start = x;
            if (x >= x_end || item >= p->items) return false;
            ahead = item + 1;
            b = item / p->rgroups;
            row0 = (item - b * p->rgroups) * ROWS;
            len = max(0, min(p->a.seq_lens[b], p->a.seq_len));
            nr = min(ROWS, p->rows - row0);
            t = win_tiles<TT, ROWS>(WinShape{window, sinks, q_len, p->G, p->rows}, len, row0);
            const int cost = p->fixed + t.n;
            x = start + cost;
            i0 = max(0, x_begin - start - p->fixed);
            i1 = max(0, min(t.n, x_end - start - p->fixed));
            if (t.n == 0 ? start < x_begin : i1 <= i0) continue;  // its part here is of the fixed cost
            const bool mine = i0 == 0 && i1 == t.n;
            slot = mine ? -1 : start < x_begin ? 0 : 1;
            if (i0 == 0 && kv == 0 && tid == 0) {  // pieces, for the merge
                p->meta[2 * item] = 2 * wg + (slot > 0 ? 1 : 0);
                p->meta[2 * item + 1] = mine ? 1 : (start + cost - 1) / cut.share - wg + 1;
            }
            table = p->a.block_table + (int64_t)b * p->a.bt_sb;
            last_tok = max(t.p_hi, 0);
            return true;
        }
    };
    auto tile_of = [&](int i) { return i < t.n_sink ? i : t.from + i - t.n_sink; };
    // the page (always one of the cache's) and place in it of the 16 tokens around `off` in tile i
    struct Place { int page, at; };
    auto place = [&](int i, int off) {
        const int tok = min(TT * tile_of(min(i, max(i1 - 1, 0))) + (off & ~15), last_tok & ~15);
        return Place{(int)min((uint32_t)table[(tok >> 4) >> psh], (uint32_t)(n_pages - 1)), tok & ((16 << psh) - 1)};
    };
    // ---- a tile's pieces on their way
    uint32_t codes = 0, codes_next = 0;  // of the tile that is gathered next, and of the one after it
    w4u raw{};
    float scale = 1.f;
    Place pk{}, pv{}, ps{};
    auto scale_at = [&](int i) {
        if constexpr (kV8) ps = place(i, 16 * min(tid, NT - 1));
    };
    auto load_scale = [&]() {
        if constexpr (kV8) scale = v_scale[(uint64_t)(uint32_t)ps.page * vs_sb];
    };
    auto load_codes = [&]() {
        const uint8_t* src = cbase + (uint64_t)(uint32_t)pk.page * c_sb + (uint32_t)pk.at * c_st;
        if constexpr (NC == 4) return *reinterpret_cast<const uint32_t*>(src);
        else if constexpr (NC == 2) return (uint32_t)*reinterpret_cast<const uint16_t*>(src);
        else return (uint32_t)*src;
    };
    auto load_vals = [&]() {
        const uint8_t* row = vbase + (uint64_t)(uint32_t)pv.page * v_sb + (uint32_t)pv.at * (kV8 ? 1u : 2u);
        if constexpr (kV8) {
            const w2u x = *reinterpret_cast<const w2u*>(row);
            raw.x = x.x; raw.y = x.y;
        } else {
            raw = *reinterpret_cast<const w4u*>(row);
        }
    };
    uint4 khi, klo;
    auto gather = [&]() {
        const unsigned char* at = smem + kdim * NC * (1024 * BD);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const unsigned char* e = at + j * (1024 * BD) + ((codes >> (8 * j)) & 0xFFu) * (4 * BD);
            if constexpr (BD == 8) {
                const uint4 h = reinterpret_cast<const uint4*>(e)[0], l = reinterpret_cast<const uint4*>(e)[1];
                hi[0] = h.x; hi[1] = h.y; hi[2] = h.z; hi[3] = h.w;
                lo[0] = l.x; lo[1] = l.y; lo[2] = l.z; lo[3] = l.w;
            } else if constexpr (BD == 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(e);
                hi[2 * j] = w.x; hi[2 * j + 1] = w.y; lo[2 * j] = w.z; lo[2 * j + 1] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(e);
                hi[j] = w.x; lo[j] = w.y;
            }
        }
        khi = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        klo = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    };
    auto put_keys = [&](int i) {
        if (kV8 && tid < NT) scales[(i & 1) * NT + tid] = scale;
        *reinterpret_cast<uint4*>(kput) = khi;
        *reinterpret_cast<uint4*>(kput + L::kLo) = klo;
    };
    auto put_vals = [&]() {
        // Infinities and NaN are kept out of the tile, for the rows that do not see them, and noted.
        uint32_t wild = 0;
        if constexpr (kV8) {
            wild = (((raw.x & 0x7F7F7F7Fu) + 0x01010101u) | ((raw.y & 0x7F7F7F7Fu) + 0x01010101u)) & 0x80808080u;
        } else {
            constexpr uint32_t up = VT == SSQ_BF16 ? 0x00800080u : 0x04000400u;
#pragma unroll
            for (int k = 0; k < 4; ++k) wild |= (raw[k] & 0x7FFF7FFFu) + up;
            wild &= 0x80008000u;
        }
        const bool any = __builtin_amdgcn_ballot_w64(wild != 0) != 0;
        if (any) {
            uint32_t nan = 0, inf = 0, neg = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                constexpr int bits = kV8 ? 8 : 16, each = 32 / bits;
                const uint32_t z = (raw[j / each] >> (bits * (j % each))) & ((1u << bits) - 1u), mag = z & ((1u << (bits - 1)) - 1u);
                constexpr uint32_t infinity = kV8 ? 0x7Fu : VT == SSQ_BF16 ? 0x7F80u : 0x7C00u;
                if (mag < infinity) continue;
                if (kV8 || mag > infinity) nan |= 1u << j;
                else if (z == mag) inf |= 1u << j;
                else neg |= 1u << j;
                raw[j / each] &= ~(((1u << bits) - 1u) << (bits * (j % each)));
            }
            wilds[tid] = (unsigned char)nan;
            wilds[kWinThreads + tid] = (unsigned char)inf;
            wilds[2 * kWinThreads + tid] = (unsigned char)neg;
        }
        if (lane == 0) flags[wave] = any ? 1u : 0u;
        if constexpr (kV8) {
            const w2u x = win_e4m3(raw.x), y = win_e4m3(raw.y);
            *reinterpret_cast<uint4*>(vput) = make_uint4(x.x, x.y, y.x, y.y);
        } else {
            *reinterpret_cast<uint4*>(vput) = make_uint4(raw.x, raw.y, raw.z, raw.w);
        }
    };
    // ---- the wave's query rows: 1 KiB a piece
    constexpr int kSize = QP == 2 ? 4 : 2, kRowBytes = D * kSize, kPieces = WR * kRowBytes / (SSQ_WAVE * 16);
    uint4 qraw[kPieces];
    auto load_rows = [&]() {
        const int wr0 = row0 + WR * wave, n = max(1, min(WR, p->rows - wr0));
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int o = (k * SSQ_WAVE + lane) * 16, row = min(wr0 + min(o / kRowBytes, n - 1), p->rows - 1), qi = row / p->G, h = kv * p->G + row - qi * p->G;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(p->a.q) + ((int64_t)b * p->a.q_sb + (int64_t)h * p->a.q_sh + (int64_t)qi * p->a.q_sl) * kSize + o % kRowBytes;
            if (p->q_vec) {
                qraw[k] = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    z[e] = kSize == 4 ? reinterpret_cast<const uint32_t*>(src)[e]
                                      : (uint32_t)reinterpret_cast<const uint16_t*>(src)[2 * e] | (uint32_t)reinterpret_cast<const uint16_t*>(src)[2 * e + 1] << 16;
                qraw[k] = make_uint4(z[0], z[1], z[2], z[3]);
            }
        }
    };
    // ---- as operands: f16, at a power of two of each row's; fac takes scores to log2 units
    uint4 q[QP][NK];
    float fac = 1.f;
    auto query_of = [&](auto type) {
        constexpr int dtype = decltype(type)::value, wide = dtype == SSQ_F32 ? 1 : 0;
        const int n = max(0, min(WR, p->rows - row0 - WR * wave));
        const float qs = p->a.has_scale ? p->a.scale : 1.f;  // (a factor of 1 is exact)
        // through the wave's LDS rows, `per` at a time: permuted there by all lanes, kEach dims each, and read back as operands
        unsigned char* rows = smem + L::kK + wave * 8 * L::kQRow;
        constexpr int row_bytes = L::kQRow << wide, per = 8 >> wide, kEach = D * per / SSQ_WAVE, kLoads = per * kRowBytes / (SSQ_WAVE * 16);
        const int pr = lane & (per - 1), pd = lane / per * kEach;
        uint32_t idx[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) idx[k] = perm[pd + k];
        float y[NE];
#pragma unroll
        for (int k = 0; k < NE; ++k) y[k] = 0.f;
#pragma unroll
        for (int r0 = 0; r0 < WR; r0 += per) {
#pragma unroll
            for (int k = 0; k < kLoads; ++k) {
                const int o = (k * SSQ_WAVE + lane) * 16;
                *reinterpret_cast<uint4*>(rows + o / kRowBytes * row_bytes + o % kRowBytes) = qraw[r0 / per * kLoads + k];
            }
            win_lds_sync();
            uint32_t w[kEach];
#pragma unroll
            for (int k = 0; k < kEach; ++k)
                w[k] = wide ? reinterpret_cast<const uint32_t*>(rows + pr * row_bytes)[idx[k]] : reinterpret_cast<const uint16_t*>(rows + pr * row_bytes)[idx[k]];
            win_lds_sync();
#pragma unroll
            for (int k = 0; k < kEach; k += 16 / kSize) {
                uint4 z;
                if constexpr (wide) z = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
                else z = make_uint4(w[k] | w[k + 1] << 16, w[k + 2] | w[k + 3] << 16, w[k + 4] | w[k + 5] << 16, w[k + 6] | w[k + 7] << 16);
                *reinterpret_cast<uint4*>(rows + pr * row_bytes + (pd + k) * kSize) = z;
            }
            win_lds_sync();
            if (col >= r0 && col < r0 + per) {
                const unsigned char* mine = rows + (col - r0) * row_bytes + 8 * grp * kSize;
#pragma unroll
                for (int c = 0; c < NK; ++c)
#pragma unroll
                    for (int e = 0; e < kSize / 2; ++e) {
                        const uint4 z = *reinterpret_cast<const uint4*>(mine + 16 * c * kSize + 16 * e);
                        const uint32_t u[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
                        for (int k = 0; k < 16 / kSize; ++k)
                            y[8 * c + 4 * e + k] = ssq_bits_to_f32(wide ? u[k & 3] : k & 1 ? u[k / 2] >> 16 : u[k / 2] & 0xFFFFu, dtype);
                    }
            }
            win_lds_sync();
        }
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < NE; ++k) {
            y[k] = col < n ? ssq_round_to(y[k] * qs, dtype) : 0.f;
            const float z = fabsf(y[k]);
            most = fmaxf(most, z < INFINITY ? z : 0.f);
        }
        const int up = min(15 - win_exp(fmaxf(most, __shfl_xor(most, 32))), 126);
        const float s = ldexpf(1.f, up);
        fac = ldexpf(kWinLog2e, max(-book_exp - up, -126));  // above 0
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) win_split<true>(y[8 * c + 2 * k] * s, y[8 * c + 2 * k + 1] * s, hi[k], lo[k]);
            q[0][c] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (QP == 2) q[QP - 1][c] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    };
    // bits [0, n) of 8 tokens; the tokens from tok that some row at a position from `first` to `last` sees
    auto below = [](int n) { return (1u << min(max(n, 0), 8)) - 1u; };
    auto sees = [&](int first, int last, int tok) {
        return below(last + 1 - tok) & (~below(max(max(first, 0) - window, -1) + 1 - tok) | below(sinks - tok));
    };

    auto first = [&]() {  // an item's first loads
        pk = place(i0, ktok);
        pv = place(i0, 8 * vtok);
        scale_at(i0);
        const Place pk1 = place(i0 + 1, ktok), pk2 = place(i0 + 2, ktok);
        codes = load_codes();
        load_scale();
        if constexpr (QP == 1) load_rows();  // (32 bits beside the codebook's registers do not fit)
        pk = pk1;
        codes_next = load_codes();
        load_vals();
        pk = pk2;
        pv = place(i0 + 1, 8 * vtok);
        scale_at(i0 + 1);
    };
    // tile i's keys and scales, and the values of the one before it, take their places
    auto step = [&](int i) {
        wide_sync();
        put_keys(i);
        put_vals();
        codes = codes_next;
        codes_next = load_codes();
        load_scale();
        load_vals();
        pk = place(i + 3, ktok);
        scale_at(i + 2);
        pv = place(i + 1, 8 * vtok);
        wide_sync();
    };
    bool more = next();
    if (more) first();
    book_exp = book.stage(smem, red, tid, lane, wave);
    // A wave's work goes M(0) X(0) M(1) X(1) .. M(n): M(i) the matrix products of tile i's scores and of tile i - 1's values, X(i)
    // tile i's probabilities.  Waves 0 to 3 take a step before each M, waves 4 to 7, which share their SIMDs, behind it: the
    // tile's place holds keys i and values i - 1 for both, and one's matrix products run beside the other's vector work.
    const bool late = wave >= kWinWaves / 2;
    while (more) {
        if constexpr (QP == 2) load_rows();
        if constexpr (QP == 2) query_of(std::integral_constant<int, SSQ_F32>{});
        else if (p->a.q_dtype == SSQ_BF16) query_of(std::integral_constant<int, SSQ_BF16>{});
        else query_of(std::integral_constant<int, SSQ_F16>{});
        gather();
        wide_sync();  // the queries have left the tile's place
        put_keys(i0);
        codes = codes_next;
        codes_next = load_codes();
        load_scale();
        pk = place(i0 + 3, ktok);
        scale_at(i0 + 2);

        // this wave's rows, a lane's and the first and last one's positions
        const int wr0 = row0 + WR * wave, row = wr0 + col, base = len - q_len;
        const int pos = base + min(row, p->rows - 1) / p->G;
        const int p_lo = base + min(wr0, p->rows - 1) / p->G, p_hi = base + (min(wr0 + WR, p->rows) - 1) / p->G;
        const bool busy = wr0 < p->rows && p_hi >= 0;
        float m = kWinNone, l = 0.f, unit = kV8 ? kWinScale : 1.f, inv_unit = 1.f / unit;
        w16f o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = w16f{};
        w16f s[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) s[k] = w16f{};
        wide_sync();
        // nothing of tile i for this wave
        auto hidden = [&](int i) {
            const int t0 = TT * tile_of(i);
            return !busy | (i < i0) | (i >= i1) | (t0 > p_hi) | ((t0 + TT <= max(p_lo, 0) - window + 1) & (t0 >= sinks));
        };
        uint4 pw[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) pw[c] = uint4{};
        bool far = false;  // 8-bit values: tile i - 1 has a page far below the unit; its probabilities are in s, in 32 bits, and 0 in pw
        for (int i = i0; i <= i1; ++i) {
            if (!late && i > i0) step(i);
            if constexpr (kV8) {
                if (far) {
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            const uint4 v = *reinterpret_cast<const uint4*>(vget + 32 * dt * L::kVRow + 32 * c);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int j = 0; j < 8; ++j) o[dt] = wide_mfma_32(win_h(w[j / 2], j & 1), s[c / 2][8 * (c % 2) + j], o[dt]);
                        }
                }
                far = false;
            }
            gather();  // the next tile's (past the last: some tile's)
            const bool none = hidden(i);
            if (!none) {
                // operand st: hi, lo in turn of 16 dims of a block, read kAhead before its products
                constexpr int NST = 2 * NK * NB, kAhead = 4;
                auto operand = [&](int st) {
                    return *reinterpret_cast<const uint4*>(kget + 32 * (st / (2 * NK)) * L::kKRow + 32 * (st % (2 * NK) / 2) + st % 2 * L::kLo);
                };
                uint4 ring[kAhead];
#pragma unroll
                for (int st = 0; st < kAhead; ++st) ring[st] = operand(st);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int st = 0; st < NST; ++st) {
                    const uint4 k = ring[st % kAhead];
                    w16f& z = s[st / (2 * NK)];
#pragma unroll
                    for (int h = 0; h < QP; ++h) z = wide_mfma<SSQ_F16>(k, q[h][st % (2 * NK) / 2], st % (2 * NK) || h ? z : w16f{});
                    if (st + kAhead < NST) ring[st % kAhead] = operand(st + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (!hidden(i - 1)) {
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        o[dt] = wide_mfma<VT>(*reinterpret_cast<const uint4*>(vget + 32 * dt * L::kVRow + 32 * c), pw[c], o[dt]);
                uint32_t found = 0;
#pragma unroll
                for (int w = 0; w < kWinWaves; ++w) found |= flags[w];
                if (__builtin_amdgcn_readfirstlane(found) != 0) {  // a row has a dim's infinities and NaN of the tokens that it sees
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int dim = 32 * dt + 8 * (e / 4) + 4 * grp + e % 4;
                            if (!flags[dim / (D / kWinWaves)]) continue;
                            uint32_t nan = 0, inf = 0, neg = 0;
                            for (int j = 0; j < TT / 8; ++j) {
                                const uint32_t mine = sees(pos, pos, TT * tile_of(i - 1) + 8 * j);
                                const unsigned char* w = wilds + dim * (TT / 8) + j;
                                nan |= mine & w[0];
                                inf |= mine & w[kWinThreads];
                                neg |= mine & w[2 * kWinThreads];
                            }
                            if (inf) o[dt][e] += INFINITY;
                            if (neg) o[dt][e] -= INFINITY;
                            if (nan) o[dt][e] = NAN;
                        }
                }
            }
            if (late && i < i1) step(i + 1);
            if (!none) {
                const int t0 = TT * tile_of(i);
                // tokens of the tile that some row does not see (uniform)
                const bool edge = (t0 + TT - 1 > p_lo) | ((t0 <= p_hi - window) & (t0 + TT > sinks));
                float sc[NT];
#pragma unroll
                for (int c = 0; c < NT; ++c) sc[c] = kV8 ? scales[(i & 1) * NT + c] : 1.f;
                if (edge) {
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        const uint32_t mine = sees(pos, pos, t0 + 16 * c + 8 * grp);
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[c / 2][8 * (c % 2) + j] = mine >> j & 1u ? s[c / 2][8 * (c % 2) + j] : -INFINITY;
                        const int at = t0 + 16 * c;  // of a page that this row sees
                        if (!((at <= pos) & ((at + 15 > max(pos, 0) - window) | (at < sinks)))) sc[c] = 0.f;
                    }
                }
                float top = s[0][0];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[n][e]);
                top *= fac;
                if (__builtin_amdgcn_ballot_w64(win_over<VT>(top, m, l)) != 0) {
                    float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)) - kWinTop<VT>);
                    if (VT == SSQ_BF16 && fmaxf(l, __shfl_xor(l, 32)) > kWinMass) mn = fmaxf(mn, m + 4.f);
                    const float f = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= f;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        if constexpr (kV8) o[dt] *= f;
                        else
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[dt][e] = win_part(o[dt][e], f);  // (f may be 0)
                    }
                }
                if constexpr (kV8) {  // a row's units: the largest scale of a page that it sees
                    float big = sc[0];
#pragma unroll
                    for (int c = 1; c < NT; ++c) big = fmaxf(big, sc[c]);
                    if (__builtin_amdgcn_ballot_w64(big > unit) != 0) {
                        big = fmaxf(unit, big);
                        const float f = unit / big;
                        unit = big;
                        inv_unit = 1.f / unit;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
                    }
                }
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    uint32_t w[4];
                    const float by = kV8 ? sc[c] * inv_unit : 1.f;
                    if constexpr (kV8) far |= __builtin_amdgcn_ballot_w64((by < kWinFar) & (sc[c] > 0.f)) != 0;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 2][8 * (c % 2) + j], fac, -m));
                        float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 2][8 * (c % 2) + j + 1], fac, -m));
                        l += x0 + x1;
                        if constexpr (kV8) {
                            s[c / 2][8 * (c % 2) + j] = x0 *= by;
                            s[c / 2][8 * (c % 2) + j + 1] = x1 *= by;
                        }
                        w[j / 2] = win_pack_p<VT>(x0, x1);
                    }
                    pw[c] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (far) {
#pragma unroll
                    for (int c = 0; c < NT; ++c) pw[c] = uint4{};
                }
            }
        }
        l += __shfl_xor(l, 32);
        // what the row's values average to here, as in k_window
        const float inv = 1.f / l;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = l == 0.f ? w16f{} : kV8 ? o[dt] * inv * unit : o[dt] * inv;

        p = win_args();
        if (WR * wave + col < nr) {
            if (slot < 0) {
                const int qi = row / p->G, h = kv * p->G + row - qi * p->G;
                const int64_t at = (int64_t)b * p->a.o_sb + (int64_t)h * p->a.o_sh + (int64_t)qi * p->a.o_sl + 4 * grp;
                const int dtype = p->out_dtype;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        w4f z;
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] = o[dt][4 * a + e];
                        if (p->out_vec) win_store4(p->a.out, dtype, at + 32 * dt + 8 * a, z);
                        else
#pragma unroll
                            for (int e = 0; e < 4; ++e) ssq_store_elem(p->a.out, dtype, at + 32 * dt + 8 * a + e, z[e]);
                    }
                if (p->a.lse && grp == 0)
                    p->a.lse[((int64_t)b * p->a.num_q_heads + h) * p->a.q_len + qi] = l == 0.f ? -INFINITY : (m + log2f(l)) * kWinLn2;
            } else {
                float* dst = p->part + ((int64_t)(kv * p->workers + wg) * 2 + slot) * (ROWS * (D + 2));
                const int r = WR * wave + col;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int a = 0; a < 4; ++a)  // as the registers lie: a store is 1 KiB
                        *reinterpret_cast<float4*>(dst + ((wave * DT + dt) * 4 + a) * 256 + lane * 4) =
                            make_float4(o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]);
                if (grp == 0) {
                    dst[ROWS * D + r] = m;
                    dst[ROWS * D + ROWS + r] = l;
                }
            }
        }
        more = next();
        if (more) first();
    }
}

// Joins the pieces of the items that workgroups shared: 32 rows a workgroup, 32 value dims a wave, in the registers' order.
template <int D>
__global__ __launch_bounds__(D / 32 * SSQ_WAVE) void k_window_wide_merge(const SsqWindowParams p) {
    constexpr int ROWS = kWinWideRows, WR = ROWS / kWinWaves, DT = D / 32, kAhead = 4;
    const ssq_decode_args& a = p.a;
    const int lane = threadIdx.x & 63, dt = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, grp = lane >> 5;
    const int w = blockIdx.x % kWinWaves, unit = blockIdx.x / kWinWaves, kv = unit % a.num_kv_heads, item = unit / a.num_kv_heads;
    const int b = item / p.rgroups, r = WR * w + col, row = (item - b * p.rgroups) * ROWS + r;
    const int first = p.meta[2 * item], pieces = p.meta[2 * item + 1];
    if (pieces <= 1 || row - col >= p.rows) return;
    const int64_t slot = (int64_t)ROWS * (D + 2);
    const float* base = p.part + (int64_t)kv * p.workers * 2 * slot;
    float M = kWinNone, l = 0.f;
    w4f o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = w4f{};
    for (int i0 = 0; i0 < pieces; i0 += kAhead) {
        float m[kAhead], lp[kAhead];
        w4f op[kAhead][4];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            m[j] = kWinNone;
            if (i0 + j >= pieces) continue;
            const float* src = base + (int64_t)(i0 + j ? 2 * ((first >> 1) + i0 + j) : first) * slot;
            m[j] = src[ROWS * D + r];
            lp[j] = src[ROWS * D + ROWS + r];
#pragma unroll
            for (int k = 0; k < 4; ++k) op[j][k] = *reinterpret_cast<const w4f*>(src + ((w * DT + dt) * 4 + k) * 256 + lane * 4);
        }
        win_join<kAhead, 4>(M, l, o, m, lp, op, pieces - i0);
    }
    if (row >= p.rows) return;
    const int qi = row / p.G, h = kv * p.G + row - qi * p.G;
    const int64_t at = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)qi * a.o_sl + 32 * dt + 4 * grp;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const w4f z = o[k];
        if (p.out_vec) win_store4(a.out, p.out_dtype, at + 8 * k, z);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) ssq_store_elem(a.out, p.out_dtype, at + 8 * k + e, z[e]);
    }
    if (a.lse && dt == 0 && grp == 0) a.lse[((int64_t)b * a.num_q_heads + h) * a.q_len + qi] = l == 0.f ? -INFINITY : (M + log2f(l)) * kWinLn2;
}

}  // namespace
