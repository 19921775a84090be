// dsa_chunk_fp4.h - the kernels for few rows on DSA_KV_MXFP4 rows: dense attention of a
// chunk's tokens (include/dsa_chunk.h) and attention over lists of positions
// (dsa_mla_decode, dsa_mla_prefill).  Part of dsa_chunk.hip.

// ---------------------------------------------------------------------------
// 16 QB rows (heads of tokens) a workgroup, tiles of 64 positions.
//   K      wave w: positions 16 w .. +15 of the tile in its registers, straight from the cache, two
//          tiles ahead: a row's codes are 256 bytes, so a lane's 7 loads hold a quarter of a row
//   QK^T   wave w: those 16 positions x all rows, 16x16x32.  The codes are converted between the matrix
//          instructions, once, and written to LDS from there: the tile is V, and K is never read from LDS
//   P      exp2 against a fixed reference, bf16, exchanged through LDS
//   PV     wave w: O^T[dims 128 w .. +127 x all rows]
// QB = 1: 16 rows, two workgroups a CU, one V buffer, two barriers a tile; PV in 16x16x32.
// QB = 2: 32 rows, one workgroup a CU (Q alone takes 144 registers), two V buffers, one barrier a tile.
// What bounds them: not memory (rows are 400 bytes: 512 tokens x 2048 of 32 heads from HBM 128 us, 3.3 TB/s; a
// third of 1536 tokens over 3000 rows, from the caches, 105) nor the matrix units (1531 tokens x 2048 of 16 heads:
// 169 us, 0.65 PFLOP/s; matrix units busy 24 % of the cycles, vector instructions 35, LDS 40), but the chain of a
// wave's tile - codes, conversion, scores, exp2, LDS, barrier, product - with one or two waves on a SIMD to run
// beside it.  Without one part of it (wrong results) that case, at 185 us, took: without PV 151, without V's writes
// 141, without both 120, without the conversion 163, without the scores' products 164.  A pair of tiles takes 1.6
// to 1.9 us, a QB = 2 tile 1.3 to 1.5. Kept on the way (303 us at first, 128-row blocks with most rows empty 702):
// loads without a branch around them, so that a wait counts only older ones, two tiles ahead; fsw(), after whose
// first form bank conflicts were 26.7 M cycles and are 1.7 M; Q loaded once for a workgroup (185 -> 172, with the
// lane numbers formed anew in qk(): 222 registers of 256 over lists, 218 dense), beside the first rows' look-up and without
// divisions (172 -> 169; 64 entries each for 1536 tokens 31 -> 28).  Not kept: rows loaded along their bytes and
// turned through LDS (98 M L1 accesses become 39 M, but LDS has the wait then: 185 -> 200); QB = 2 with half the
// next tile's conversions behind PV's products and half behind the scores' (lists 318 -> 313, dense 50.3 -> 50.9:
// the chain is as long).
// ---------------------------------------------------------------------------
constexpr int FTILE = 64;                    // positions of a tile
// V in LDS: rows of 1 KB, piece c of row r at c ^ fsw(r).  A write takes eight rows' pieces of one number at a time,
// which meet no bank of 32 twice (the low three bits tell the rows apart); half a transposed read two pieces of each of
// eight rows, or four of each of four, no bank of 64 (the upper three, or two).
__device__ __forceinline__ int fsw(int r) { return 9 * (r & 1) + 4 * ((r >> 1) & 1) + 2 * ((r >> 2) & 1); }
template <int QB>
struct FewLay {
    static constexpr int ROWS = 16 * QB;
    static constexpr int VT = FTILE * NSTRIDE, PT = FTILE * ROWS * 2;
    static constexpr int NB = QB == 1 ? 1 : 2;                            // V and P buffers
    static constexpr int PLACES = QB == 1 ? 2 * CUS : CUS;
};

template <int QB, bool LIST>
__global__ void __launch_bounds__(NTHR) __attribute__((amdgpu_waves_per_eu(QB == 1 ? 2 : 1, QB == 1 ? 2 : 1)))
dsa_mla_fp4_few_kernel(const ChunkParams p) {
    using L = FewLay<QB>;
    constexpr int VT = L::VT, PT = L::PT, NB = L::NB, ROWS = L::ROWS;
    // NB tiles of V, then NB of P
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[NB * (VT + PT)];
    __shared__ __attribute__((aligned(16))) int32_t s_rows[SPAN];
    __shared__ uint32_t s_skip[SPAN / TILE];                               // bit j: position j of 32 has no row
    __shared__ float s_top[NWAVE][ROWS];
    __shared__ int32_t s_misc[4];            // [0] a row that may be read, [1] again, [2] O may have passed fp32, [3] it has
    const lds_ptr T0 = (lds_ptr)s_tile, PX = T0 + NB * VT;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work work;
    if constexpr (LIST) work = list_work(p, ROWS);
    else work = find_work(p, ROWS, L::PLACES);
    const Block& blk = work.blk;
    const int split = work.split, per = work.per;
    if (blk.rows == 0) return;
    int lim_lo, lim_hi;
    if constexpr (LIST) lim_lo = lim_hi = p.topk;
    else lim_lo = limit_in(p, blk, blk.first + blk.r0 / p.H), lim_hi = limit_in(p, blk, blk.first + (blk.r0 + blk.rows - 1) / p.H);
    const bool too_long = !LIST && blk.len > p.max_len;
    const int k0 = (int)min((int64_t)split * per, (int64_t)lim_hi);
    const int k1 = too_long ? k0 : (int)min(LIST ? (int64_t)lim_hi : min((int64_t)lim_hi, p.pages.limit), (int64_t)k0 + per);
    if (!LIST && p.ns > 1 && k1 <= k0) return;      // (the join knows; that of lists reads every split)

    // scores: this lane's row of each block of 16, its positions 16 wave + 4 q .. +3 of a tile, and the dims
    // 128 q .. +127 and 512 + 32 j + 8 q .. +7 (j < 2) of a product's operands
    const int q = lane >> 4;
    // Row k of the block: its token after the block's first one's, and its head.  (Of a list all rows are one token's;
    // elsewhere a division where a token has fewer heads than the block rows.)
    struct HeadOf {
        int tok, head;
    };
    const int tok0 = LIST ? 0 : blk.r0 / p.H, head0 = blk.r0 - tok0 * p.H;
    auto head_of = [&](int k) -> HeadOf {
        if constexpr (LIST) return {0, blk.r0 + k};
        int t = 0, h = head0 + k;
        if (p.H >= ROWS) t = h >= p.H ? 1 : 0;
        else t = h / p.H;
        return {tok0 + t, h - t * p.H};
    };
    int limit[QB];
#pragma unroll
    for (int h = 0; h < QB; ++h)
        limit[h] = LIST ? 0 : limit_in(p, blk, blk.first + head_of(min(16 * h + (lane & 15), blk.rows - 1)).tok);
    const int64_t q0 = LIST ? token_at(blk.first, p.s_q, p.q_sb, p.q_st) : (int64_t)blk.first * p.q_st;
    // Q once for the workgroup, 16 bytes a lane of neighbouring ones; each lane's part comes back through LDS (in
    // qf's order a load of 64 lanes touches 64 cache lines, and every wave would read all rows).
    constexpr int QU = 72, QSTRIDE = 16 * QU + 16, QN = (ROWS * QU + 255) / 256;
    static_assert(ROWS * QSTRIDE <= NB * VT, "Q fits the tile buffers");
    u32x4 qraw[QN];
    auto load_q = [&] {
        const int tid = 64 * wave + fresh_lane();
#pragma unroll
        for (int n = 0; n < QN; ++n) {
            const int u = min(tid + 256 * n, ROWS * QU - 1);
            const HeadOf r = head_of(min(u / QU, blk.rows - 1));
            const __bf16* qp = p.q + q0 + (int64_t)r.tok * p.q_st + (int64_t)r.head * p.q_sh;
            qraw[n] = *reinterpret_cast<const u32x4*>(qp + 8 * (u % QU));
        }
    };

    // ---- positions [c0, c0 + SPAN) below k1 -> cache rows (positions without one: some row that is there) ----
    int ntiles = 0, n_valid = 0;
    auto resolve = [&](int c0, auto beside) {
        if constexpr (LIST) {
            n_valid = resolve_list(p, blk, c0, k1, s_rows, s_misc, beside);
            ntiles = (n_valid + FTILE - 1) / FTILE;
        } else {
            const int tid = 64 * wave + fresh_lane();
            const int at = c0 + 8 * tid;
            int32_t id[8], blk_i[8], some = -1;
            uint32_t skip = 0;
            // (positions past the end look up the last one's row: no branch splits the eight reads)
            if (p.pages.table) {
                const int32_t* const table = p.pages.table + blk.b * p.pages.table_stride;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = min(at + e, k1 - 1);
                    blk_i[e] = p.pages.shift >= 0 ? k >> p.pages.shift : k / p.pages.block_size;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) id[e] = table[blk_i[e]];
                beside();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t r = (int64_t)id[e] * p.pages.block_size + (min(at + e, k1 - 1) - blk_i[e] * p.pages.block_size);
                    id[e] = r >= 0 && r < p.rows ? (int32_t)r : -1;
                }
            } else {
                beside();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t r = blk.b * p.pages.batch_stride + min(at + e, k1 - 1);
                    id[e] = r < p.rows ? (int32_t)r : -1;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                skip |= at + e >= k1 || id[e] < 0 ? 1u << e : 0u;
                some = max(some, id[e]);
            }
            __syncthreads();                       // the previous span is done with its rows and tiles
            if (tid == 0) s_misc[0] = -1;
            __syncthreads();
            if (some >= 0) s_misc[0] = some;       // any of them will do
            __syncthreads();
            const int32_t safe = __builtin_amdgcn_readfirstlane(s_misc[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) id[e] = id[e] < 0 ? max(safe, 0) : id[e];
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<int4*>(&s_rows[8 * tid + e]) = int4{id[e], id[e + 1], id[e + 2], id[e + 3]};
            reinterpret_cast<unsigned char*>(s_skip)[tid] = (unsigned char)skip;
            ntiles = safe < 0 ? 0 : (min(k1 - c0, SPAN) + FTILE - 1) / FTILE;
            __syncthreads();
        }
    };

    const int nspans = k1 > k0 ? (int)(((int64_t)k1 - k0 + SPAN - 1) / SPAN) : 0;
    auto start_of = [&](int c) { return (int)(k0 + (int64_t)c * SPAN); };
    // (Q beside the first span's rows)
    bool ready = nspans > 0;
    if (ready) resolve(start_of(0), load_q);
    else load_q();
    u32x4 qf[QB][KS / 2];
    {
        const int ln = fresh_lane();
#pragma unroll
        for (int n = 0; n < QN; ++n) {
            const int u = 64 * wave + ln + 256 * n;
            if (u < ROWS * QU) lds_st<u32x4>(T0 + (u / QU) * QSTRIDE + 16 * (u % QU), qraw[n]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < QB; ++h)
#pragma unroll
            for (int ks = 0; ks < KS / 2; ++ks)
                qf[h][ks] = lds_ld<u32x4>(T0 + (16 * h + (ln & 15)) * QSTRIDE +
                                          (ks < 16 ? 256 * (ln >> 4) + 16 * ks : 64 * ks + 16 * (ln >> 4)));
        __syncthreads();
    }

    // This lane's quarter of row lane % 16 of its wave's 16
    struct Raw {
        u32x4 v[6];            // codes of dims 128 q + 32 j .. +31 (j < 4), RoPE values 32 (j - 4) + 8 q .. +7
        unsigned s;            // the codes' four scales
    };
    auto fetch = [&](Raw& x, int i) {
        const int ln = opaque(lane), lq = ln >> 4;
        const uint32_t id = (uint32_t)s_rows[i * FTILE + 16 * wave + (ln & 15)];
        const unsigned char* const at = p.kv + (uint64_t)id * (uint32_t)p.row_bytes;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = *reinterpret_cast<const u32x4*>(at + 64 * lq + 16 * j);
        x.s = *reinterpret_cast<const unsigned*>(at + FP4_SCALE_OFF + 4 * lq);
#pragma unroll
        for (int j = 4; j < 6; ++j) x.v[j] = *reinterpret_cast<const u32x4*>(at + FP4_ROPE_OFF + 64 * (j - 4) + 16 * lq);
    };
    auto scale_of = [&](const Raw& x, int j) -> unsigned { return (x.s >> (8 * j)) & 0xFFu; };
    // (as in the other kernels: NoPE values that are not finite must not reach rows that do not attend them.  Only
    // scale bytes from 253 on give any.)  Bit r: those of this wave's position r, which are cleared.
    auto scan = [&](Raw& x) -> uint32_t {
        bool high = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) high |= scale_of(x, j) >= 253u;
        if (__builtin_amdgcn_ballot_w64(high) == 0) return 0;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 v = fp4_to_bf16(x.v[j][i], scale_of(x, j));
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (v[w] & 0x7F800000u) == 0x7F800000u || (v[w] & 0x7F80u) == 0x7F80u;
            }
        const uint64_t who = __builtin_amdgcn_ballot_w64(odd);
        const uint32_t two = (uint32_t)who | (uint32_t)(who >> 32), rows = (two | two >> 16) & 0xFFFFu;
        if ((rows >> (lane & 15)) & 1) {
            x.s = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[j] = u32x4{0, 0, 0, 0};
        }
        return rows;
    };

    const float c_s = p.scale_log2;
    float m_ref[QB] = {}, l_lane[QB] = {};
    bool any[QB] = {};

    // S^T[4 positions of this lane x its rows]; the converted codes go to V's tile at vt
    auto qk = [&](const Raw& x, lds_ptr vt, f32x4 (&s)[QB]) {
        const int ln = opaque(lane), lr = 16 * wave + (ln & 15);
        const lds_ptr vr = vt + lr * NSTRIDE + 256 * (ln >> 4);
        const int sw = 16 * fsw(lr);
        f32x4 a[2] = {};                       // two chains: the blocks of rows, or the even and odd k-steps
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            const unsigned e = scale_of(x, j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 k = fp4_to_bf16(x.v[j][i], e);
#pragma unroll
                for (int h = 0; h < QB; ++h) {
                    f32x4& c = a[QB == 2 ? h : i & 1];
                    c = mfma16(k, qf[h][4 * j + i], c);
                }
                lds_st<u32x4>(vr + (sw ^ (16 * (4 * j + i))), k);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < QB; ++h) {
                f32x4& c = a[QB == 2 ? h : i];
                c = mfma16(x.v[4 + i], qf[h][16 + i], c);
            }
        if constexpr (QB == 2) s[0] = a[0], s[1] = a[1];
        else s[0] = a[0] + a[1];
    };
    // does every row of the block attend all of this wave's positions of tile i?
    auto skips = [&](int i) -> uint32_t {
        return LIST ? 0u : (__builtin_amdgcn_readfirstlane(s_skip[2 * i + (wave >> 1)]) >> (16 * (wave & 1))) & 0xFFFFu;
    };
    // scores of tile i (its codes to vt), masked
    auto scores = [&](Raw& x, int i, int c0, lds_ptr vt, f32x4 (&s)[QB]) {
        const uint32_t skip = skips(i);
        const int at = i * FTILE + 16 * wave;
        const bool m = at + 16 > (LIST ? n_valid : lim_lo - c0) || skip != 0;
        uint32_t nan = 0;
        if (!LIST && m) nan = scan(x);
        qk(x, vt, s);
        if (m) {
            const int q4 = opaque(lane) >> 4 << 2;
#pragma unroll
            for (int h = 0; h < QB; ++h) {
                const int left = (LIST ? n_valid : limit[h] - c0) - at;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = q4 + r;
                    const bool on = j < left && !((skip >> j) & 1);
                    any[h] = any[h] || on;
                    const float v = (nan >> j) & 1 ? __builtin_nanf("") : s[h][r];
                    s[h][r] = on ? v : -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < QB; ++h) any[h] = true;
        }
    };
    // over the lanes that share a row, then over the waves
    auto lanes = [&](float v, auto f) {
        v = f(v, __shfl_xor(v, 16, 64));
        return f(v, __shfl_xor(v, 32, 64));
    };
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto put = [&](int h, float v) {
        if (opaque(lane) < 16) s_top[wave][16 * h + opaque(lane)] = v;
    };
    auto got = [&](int w, int h) { return s_top[w][16 * h + (opaque(lane) & 15)]; };
    // the largest of a row's scores in the tile
    auto top_of = [&](const f32x4 (&s)[QB], float (&top)[QB]) {
#pragma unroll
        for (int h = 0; h < QB; ++h) put(h, lanes(fmaxf(fmaxf(s[h][0], s[h][1]), fmaxf(s[h][2], s[h][3])), larger));
        __syncthreads();
#pragma unroll
        for (int h = 0; h < QB; ++h) top[h] = fmaxf(fmaxf(got(0, h), got(1, h)), fmaxf(got(2, h), got(3, h)));
        __syncthreads();
    };
    // P of wave w's positions: of QB = 2 the half k = w of a 32x32x16 step pair, lane (hi, row) 8 positions:
    // 4 hi .. +3, then 8 + 4 hi .. +3; of QB = 1 half w & 1 of 16x16x32 step w / 2, lane (q, row) 8 positions: 4 q .. +3
    // of either wave
    auto p_out = [&](const f32x4 (&s)[QB], lds_ptr px) {
        const int ln = opaque(lane), lq = ln >> 4;
#pragma unroll
        for (int h = 0; h < QB; ++h) {
            f32x4 e;
#pragma unroll
            for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][r], c_s, -m_ref[h]));
            l_lane[h] += (e[0] + e[1]) + (e[2] + e[3]);
            const lds_ptr to = QB == 1 ? px + 1024 * (wave >> 1) + 8 * (wave & 1) + 16 * ln
                                       : px + ((2 * wave + (lq & 1)) * ROWS + 16 * h + (ln & 15)) * 16 + 8 * (lq >> 1);
            lds_st<u32x2>(to, __builtin_bit_cast(u32x2, __builtin_convertvector(e, bf16x4)));
        }
    };
    // V^T by transposed reads: a group of 16 lanes reads four rows' 16 dims, and a lane then has one dim of four
    // positions
    f32x16 o[QB == 2 ? 4 : 1];                 // QB = 2: dims 128 wave + 32 m .. +31
    f32x4 o16[QB == 1 ? 8 : 1];                // QB = 1: dims 128 wave + 16 m .. +15
    // (QB = 1: the LDS addresses are kept in registers through the loop, as far as there are any left)
    auto pv = [&](lds_cptr vt, lds_cptr px) {
        const int ln = QB == 1 && LIST ? lane : opaque(lane);
        const int g16 = ln >> 4, i16 = ln & 15, rr = i16 >> 2, pp = i16 & 3;
        constexpr int N = 16, AHEAD = 3;
        u32x4 v[AHEAD], pb[QB == 2 ? 4 : 2];
        if constexpr (QB == 2) {
            const int lhi = ln >> 5, vx = 2 * (g16 & 1) + (pp >> 1);
            const lds_cptr v0 = vt + (4 * lhi + rr) * NSTRIDE + 256 * wave + 8 * (pp & 1);
            auto v_frag = [&](int i) -> u32x4 {
                const lds_cptr at = v0 + 16 * (i >> 2) * NSTRIDE;
                const int c = (4 * (i & 3) + vx) ^ fsw(4 * lhi + rr);         // (row 8 further on: the same)
                const s16x4 va = lds_read_tr16(at + 16 * c), vb = lds_read_tr16(at + 8 * NSTRIDE + 16 * c);
                return __builtin_bit_cast(u32x4, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
            };
#pragma unroll
            for (int u = 0; u < 4; ++u) pb[u] = lds_ld<u32x4>(px + ((2 * u + lhi) * ROWS + (ln & 31)) * 16);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) v[i] = v_frag(i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                o[i & 3] = mfma_bf16(v[i % AHEAD], pb[i >> 2], o[i & 3]);
                if (i + AHEAD < N) v[i % AHEAD] = v_frag(i + AHEAD);
            }
        } else {
            const lds_cptr v0 = vt + (4 * g16 + rr) * NSTRIDE + 256 * wave + 8 * (pp & 1);
            auto v_frag = [&](int i) -> u32x4 {
                const lds_cptr at = v0 + 32 * (i >> 3) * NSTRIDE + 16 * ((2 * (i & 7) + (pp >> 1)) ^ fsw(4 * g16 + rr));
                const s16x4 va = lds_read_tr16(at), vb = lds_read_tr16(at + 16 * NSTRIDE);      // (the same swizzle)
                return __builtin_bit_cast(u32x4, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
            };
#pragma unroll
            for (int u = 0; u < 2; ++u) pb[u] = lds_ld<u32x4>(px + 1024 * u + 16 * ln);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) v[i] = v_frag(i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                o16[i & 7] = mfma16(v[i % AHEAD], pb[i >> 3], o16[i & 7]);
                if (i + AHEAD < N) v[i % AHEAD] = v_frag(i + AHEAD);
            }
        }
    };

    bool first = true, again = false;
    // scores and probabilities of tile i, then its registers take tile i + 2
    auto take = [&](Raw& x, int i, int c0) {
        // (one V buffer: every wave is done with the tile before)
        if constexpr (NB == 1) tile_barrier();
        f32x4 s[QB];
        scores(x, i, c0, T0 + (NB == 1 ? 0 : (i & 1) * VT), s);
        // (past the last tile: that one again.  Behind a branch, the wait for the tile before would have to
        // take in these loads too.)
        fetch(x, min(i + 2, ntiles - 1));
        if (first) {
            float top[QB];
            top_of(s, top);
#pragma unroll
            for (int h = 0; h < QB; ++h) {
                m_ref[h] = top[h] == -INFINITY ? 0.0f : top[h] * c_s;
                m_ref[h] -= (float)lift_of<false>(k1 - k0, false);
            }
            first = false;
        }
        p_out(s, PX + (NB == 1 ? 0 : (i & 1) * PT));
        // (every wave's V and P of tile i are there; two buffers: and every wave is done with tile i - 1)
        tile_barrier();
    };
    while (true) {
        if constexpr (QB == 2) {
#pragma unroll
            for (int m = 0; m < 4; ++m) o[m] = f32x16{};
        } else {
#pragma unroll
            for (int m = 0; m < 8; ++m) o16[m] = f32x4{};
        }
#pragma unroll
        for (int h = 0; h < QB; ++h) l_lane[h] = 0.0f;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            if (!ready) resolve(c0, [] {});
            ready = false;
            if (ntiles == 0) continue;
            Raw x0, x1;
            fetch(x0, 0);
            fetch(x1, min(1, ntiles - 1));
            take(x0, 0, c0);
            // (a loop without a branch inside: where paths meet, the waits take the fewest loads in flight)
            int i = 0;
            for (; i + 2 < ntiles; i += 2) {
                pv(T0, PX);
                take(x1, i + 1, c0);
                pv(T0 + (NB - 1) * VT, PX + (NB - 1) * PT);
                take(x0, i + 2, c0);
            }
            pv(T0, PX);
            if (i + 1 < ntiles) {
                take(x1, i + 1, c0);
                pv(T0 + (NB - 1) * VT, PX + (NB - 1) * PT);
            }
        }
        // row sums over the lanes and waves that share a row (-1: no position, below every sum; a NaN stays one)
        const int lift = lift_of<false>(k1 - k0, false);
        __syncthreads();
        if (threadIdx.x == 0) s_misc[1] = 0, s_misc[2] = 0, s_misc[3] = 0;
#pragma unroll
        for (int h = 0; h < QB; ++h) {
            const float l = lanes(l_lane[h], [](float a, float b) { return a + b; });
            const uint64_t anys = __builtin_amdgcn_ballot_w64(any[h]);
            put(h, (anys >> (opaque(lane) & 15)) & 0x0001000100010001ull ? l : -1.0f);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < QB; ++h) {
            float l = 0.0f;
            bool on = false;
#pragma unroll
            for (int w = 0; w < NWAVE; ++w) {
                const float v = got(w, h);
                on = on || v != -1.0f;
                l += v == -1.0f ? 0.0f : v;
            }
            any[h] = on;
            l_lane[h] = l;
            const bool held = l > __builtin_ldexpf(1.0f, lift - 40) && l < __builtin_ldexpf(1.0f, lift + 40);
            if (!again && on && !held) s_misc[1] = 1;
            if (on && l >= 0.5f) s_misc[2] = 1;
        }
        __syncthreads();
        bool served = again || __builtin_amdgcn_readfirstlane(s_misc[1]) == 0;
        if (!again && __builtin_expect(served && __builtin_amdgcn_readfirstlane(s_misc[2]) != 0, false)) {
            float z = 0.0f;                    // (as in the tiled kernel)
            if constexpr (QB == 2) {
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int r = 0; r < 16; ++r) z = __builtin_fmaf(o[m][r], 0.0f, z);
            } else {
#pragma unroll
                for (int m = 0; m < 8; ++m)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = __builtin_fmaf(o16[m][r], 0.0f, z);
            }
            if (z != 0.0f) s_misc[3] = 1;
            __syncthreads();
            served = __builtin_amdgcn_readfirstlane(s_misc[3]) == 0;
        }
        if (served) break;
        again = true;
        float top[QB];
#pragma unroll
        for (int h = 0; h < QB; ++h) top[h] = -INFINITY;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            resolve(c0, [] {});
            for (int i = 0; i < ntiles; ++i) {
                Raw x;
                fetch(x, i);
                f32x4 s[QB];
                scores(x, i, c0, T0, s);
                float t[QB];
                top_of(s, t);
#pragma unroll
                for (int h = 0; h < QB; ++h) top[h] = fmaxf(top[h], t[h]);
            }
        }
#pragma unroll
        for (int h = 0; h < QB; ++h) {
            m_ref[h] = top[h] == -INFINITY ? 0.0f : top[h] * c_s;
            m_ref[h] -= (float)lift_of<false>(k1 - k0, true);
        }
    }

    // ---- O / l, LSE: rows' values from the scoring lanes to the lanes that hold O ----
    // (lane numbers anew: none of what follows is kept through the tile loop)
    const int lift = lift_of<false>(k1 - k0, again);
    const int ln = fresh_lane();
    __syncthreads();
    if (wave == 0 && ln < 16) {
#pragma unroll
        for (int h = 0; h < QB; ++h) {
            const int r = 16 * h + ln;
            const float lse = too_long ? __builtin_nanf("")
                                       : (m_ref[h] + (float)lift + __builtin_amdgcn_logf(__builtin_ldexpf(l_lane[h], -lift))) * LN2;
            s_top[0][r] = too_long ? __builtin_nanf("") : (any[h] ? 1.0f / l_lane[h] : 0.0f);
            const int64_t at = (int64_t)blk.first * p.H + blk.r0 + r;
            if (r >= blk.rows) {
            } else if (p.ns > 1) {
                p.part_lse[(int64_t)split * p.T * p.H + at] = any[h] || too_long ? lse : -FLT_MAX;
            } else if (p.lse) {
                p.lse[at] = any[h] || too_long ? lse : INFINITY;
            }
        }
    }
    __syncthreads();
    // O's values by quads of dims: quad k of this lane is dims 128 wave + dim_of(k) .. +3 of row orow
    constexpr int QUADS = QB == 2 ? 16 : 8;
    const int orow = QB == 2 ? ln & 31 : ln & 15;
    auto dim_of = [&](int k) { return QB == 2 ? 8 * k + 4 * (ln >> 5) : 16 * k + 4 * (ln >> 4); };
    const float inv = s_top[0][orow];
    auto quad = [&](int k) -> f32x4 {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (QB == 2 ? o[QB == 2 ? k >> 2 : 0][4 * (k & 3) + i] : o16[QB == 1 ? k : 0][i]) * inv;
        return v;
    };
    if (p.ns == 1) {
        constexpr int OUT_STRIDE = D_VO * 2 + 16;
        static_assert(ROWS * OUT_STRIDE <= NB * VT, "the stage fits the tile buffers");
#pragma unroll
        for (int k = 0; k < QUADS; ++k)
            lds_st<u32x2>(T0 + orow * OUT_STRIDE + 2 * (128 * wave + dim_of(k)),
                          __builtin_bit_cast(u32x2, __builtin_convertvector(quad(k), bf16x4)));
        __syncthreads();
        const bool wide = ((p.o_sb | p.o_st | p.o_sh) & 7) == 0 && ((uintptr_t)p.out & 15) == 0;
        const int64_t o0 = LIST ? token_at(blk.first, p.s_q, p.o_sb, p.o_st) : (int64_t)blk.first * p.o_st;
        for (int k = 0; k < ROWS / NWAVE; ++k) {
            const int r = ROWS / NWAVE * wave + k;
            if (r >= blk.rows) break;
            const HeadOf at = head_of(r);
            const u32x4 v = lds_ld<u32x4>(T0 + r * OUT_STRIDE + 16 * ln);
            __bf16* const dst = p.out + o0 + (int64_t)at.tok * p.o_st + (int64_t)at.head * p.o_sh + 8 * ln;
            if (wide) {
                *reinterpret_cast<u32x4*>(dst) = v;
            } else {
                reinterpret_cast<u32x2*>(dst)[0] = u32x2{v[0], v[1]};
                reinterpret_cast<u32x2*>(dst)[1] = u32x2{v[2], v[3]};
            }
        }
    } else {
        constexpr int PST = D_VO + 16;                     // a wave's 128 dims of a row, and a pad
        static_assert(NWAVE * ROWS * PST <= NB * VT, "four waves' stages fit the tile buffers");
        const lds_ptr stg = T0 + wave * ROWS * PST;
#pragma unroll
        for (int k = 0; k < QUADS; ++k) lds_st<f32x4>(stg + orow * PST + 4 * dim_of(k), quad(k));
        float* const dst0 = p.part_o + ((int64_t)split * p.T * p.H + (int64_t)blk.first * p.H + blk.r0) * D_VO;
#pragma unroll
        for (int k = 0; k < ROWS / 2; ++k) {
            const int r = 2 * k + (ln >> 5);
            const f32x4 v = lds_ld<f32x4>(stg + r * PST + 16 * (ln & 31));
            if (r < blk.rows) *reinterpret_cast<f32x4*>(dst0 + (int64_t)r * D_VO + 128 * wave + 4 * (ln & 31)) = v;
        }
    }
}
