// dsa_chunk_fp4.h - the narrow kernel of DSA_KV_MXFP4 rows: dense attention of a
// chunk's tokens (include/dsa_chunk.h) and attention over lists of positions
// (dsa_mla_decode, dsa_mla_prefill).  Part of dsa_chunk.hip.

// ---------------------------------------------------------------------------
// 32 rows (heads of tokens) a workgroup, two workgroups a CU, tiles of 32 positions.
//   K      wave w: 16 positions (half w % 2) in its registers straight from the cache, two tiles
//          ahead: a row's codes are 256 bytes, so a lane's 7 loads hold its quarter of a row
//   QK^T   wave w: those 16 positions x 16 rows (half w / 2), 16x16x32, the codes converted between
//          the matrix instructions and written to LDS from there, half of the dims by each of the two
//          waves that hold them: the tile is V of the next step, and K is never read from LDS
//   P, PV  as in dsa_mla_chunk_narrow_kernel; V and P in two buffers, so that a tile takes one barrier
// ---------------------------------------------------------------------------

template <bool LIST>
__global__ void __launch_bounds__(NTHR) __attribute__((amdgpu_waves_per_eu(2, 2)))
dsa_mla_fp4_narrow_kernel(const ChunkParams p) {
    constexpr int VT = TILE * NSTRIDE, PT = 2 * 2 * NARROW * 16;
    // two tiles of V, then two of P: [tile % 2][u][hi][row] x 8 positions
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[2 * VT + 2 * PT];
    __shared__ __attribute__((aligned(16))) int32_t s_rows[SPAN];
    __shared__ uint32_t s_skip[SPAN / TILE];                               // bit j: position j of the tile has no row
    __shared__ float s_top[2][NARROW];
    __shared__ int32_t s_misc[4];            // [0] a row that may be read, [1] again, [2] O may have passed fp32, [3] it has
    const lds_ptr T0 = (lds_ptr)s_tile, PX = T0 + 2 * VT;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work work = LIST ? list_work(p, NARROW) : find_work(p, NARROW, 2 * CUS);
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

    // scores: this lane's row of the 16 of its wave, its positions 16 half + 4 q .. +3 of a tile, and the dims
    // 128 j + 32 q .. +31 (j < 4) and 512 + 32 j + 8 q .. +7 (j < 2) of a product's operands
    const int half = wave & 1, rh = wave >> 1, q = lane >> 4;
    const int my = 16 * rh + (lane & 15);
    const int row = blk.r0 + min(my, blk.rows - 1);
    const int tok = blk.first + row / p.H;
    const int limit = LIST ? 0 : limit_in(p, blk, tok);
    u32x4 qf[KS / 2];
    {
        const __bf16* qp = p.q + (LIST ? token_at(tok, p.s_q, p.q_sb, p.q_st) : (int64_t)tok * p.q_st) + (int64_t)(row % p.H) * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS / 2; ++ks) {
            const int d = ks < 16 ? 128 * (ks >> 2) + 32 * q + 8 * (ks & 3) : 32 * ks + 8 * q;
            qf[ks] = *reinterpret_cast<const u32x4*>(qp + d);
        }
    }

    // ---- positions [c0, c0 + SPAN) below k1 -> cache rows (positions without one: some row that is there) ----
    int ntiles = 0, n_valid = 0;
    auto resolve = [&](int c0) {
        if constexpr (LIST) {
            n_valid = resolve_list(p, blk, c0, k1, s_rows, s_misc);
            ntiles = (n_valid + TILE - 1) / TILE;
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
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t r = (int64_t)id[e] * p.pages.block_size + (min(at + e, k1 - 1) - blk_i[e] * p.pages.block_size);
                    id[e] = r >= 0 && r < p.rows ? (int32_t)r : -1;
                }
            } else {
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
            ntiles = safe < 0 ? 0 : (min(k1 - c0, SPAN) + TILE - 1) / TILE;
            __syncthreads();
        }
    };

    // This lane's part of a tile: row c16 of its wave's 16
    struct Raw {
        u32x4 c[4];            // codes of dims 128 j + 32 q .. +31: block 4 j + q of its row
        u32x4 s;               // the row's scales; byte q of dword j is that block's
        u32x4 r[2];            // RoPE
    };
    auto fetch = [&](Raw& x, int i) {
        const int ln = opaque(lane);
        const uint32_t id = (uint32_t)s_rows[i * TILE + 16 * half + (ln & 15)];
        const unsigned char* const at = p.kv + (uint64_t)id * (uint32_t)p.row_bytes;
        const unsigned char* const mine = at + 16 * (ln >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.c[j] = *reinterpret_cast<const u32x4*>(mine + 64 * j);
        x.s = *reinterpret_cast<const u32x4*>(at + FP4_SCALE_OFF);
#pragma unroll
        for (int j = 0; j < 2; ++j) x.r[j] = *reinterpret_cast<const u32x4*>(mine + FP4_ROPE_OFF + 64 * j);
    };
    auto scale_of = [&](const Raw& x, int j) -> unsigned { return (x.s[j] >> (8 * (opaque(lane) >> 4))) & 0xFFu; };
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
            for (int s = 0; s < 4; ++s) {
                const u32x4 v = fp4_to_bf16(x.c[j][s], scale_of(x, j));
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (v[w] & 0x7F800000u) == 0x7F800000u || (v[w] & 0x7F80u) == 0x7F80u;
            }
        const uint64_t who = __builtin_amdgcn_ballot_w64(odd);
        const uint32_t two = (uint32_t)who | (uint32_t)(who >> 32), rows = (two | two >> 16) & 0xFFFFu;
        if ((rows >> (lane & 15)) & 1) {
            x.s = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) x.c[j] = u32x4{0, 0, 0, 0};
        }
        return rows;
    };

    const float c_s = p.scale_log2;
    f32x16 o[4];
    float m_ref = 0.0f, l_lane = 0.0f;
    bool any = false;

    // S^T[4 positions of this lane x its row]; the converted codes go to V's tile at vt
    auto qk = [&](const Raw& x, lds_ptr vt) -> f32x4 {
        const int ln = opaque(lane), lr = 16 * half + (ln & 15);
        const lds_ptr vr = vt + lr * NSTRIDE;
        const int piece = 16 * ((4 * (ln >> 4)) ^ nsw(lr));
        f32x4 a = {}, b = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            const unsigned e = scale_of(x, j);
            u32x4 k[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                k[s] = fp4_to_bf16(x.c[j][s], e);
                if (s & 1) b = mfma16(k[s], qf[4 * j + s], b);
                else a = mfma16(k[s], qf[4 * j + s], a);
            }
            if (rh == (j >> 1)) {
#pragma unroll
                for (int s = 0; s < 4; ++s) lds_st<u32x4>(vr + 256 * j + (piece ^ (16 * s)), k[s]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        a = mfma16(x.r[0], qf[16], a);
        b = mfma16(x.r[1], qf[17], b);
        return a + b;
    };
    auto masked = [&](int i, int c0) -> bool {
        if constexpr (LIST) return (i + 1) * TILE > n_valid;
        else return c0 + (i + 1) * TILE > lim_lo || __builtin_amdgcn_readfirstlane(s_skip[i]) != 0;
    };
    auto mask = [&](f32x4& s, uint32_t nan, int i, int c0) {
        const uint32_t skip = LIST ? 0u : s_skip[i];
        const int left = LIST ? n_valid - i * TILE : limit - (c0 + i * TILE), q4 = opaque(lane) >> 4 << 2;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = q4 + r, j = 16 * half + at;
            const bool on = j < left && !((skip >> j) & 1);
            any = any || on;
            const float v = (nan >> at) & 1 ? __builtin_nanf("") : s[r];
            s[r] = on ? v : -INFINITY;
        }
    };
    // scores of tile i (its codes to vt), masked
    auto scores = [&](Raw& x, int i, int c0, lds_ptr vt) -> f32x4 {
        const bool m = masked(i, c0);
        uint32_t nan = 0;
        if (!LIST && m) nan = scan(x);
        f32x4 s = qk(x, vt);
        if (m) mask(s, nan, i, c0);
        else any = true;
        return s;
    };
    // the largest of a row's scores in both halves of the tile
    auto top_of = [&](const f32x4& s) -> float {
        float m = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (q == 0) s_top[half][my] = m;
        __syncthreads();
        m = fmaxf(s_top[0][my], s_top[1][my]);
        __syncthreads();
        return m;
    };
    auto p_out = [&](const f32x4& s, lds_ptr px) {
        f32x4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c_s, -m_ref));
        l_lane += (e[0] + e[1]) + (e[2] + e[3]);
        // (the order of a lane's eight positions in the product: 4 hi .. +3, then 8 + 4 hi .. +3)
        lds_st<u32x2>(px + ((2 * half + (q & 1)) * NARROW + my) * 16 + 8 * (q >> 1),
                      __builtin_bit_cast(u32x2, __builtin_convertvector(e, bf16x4)));
    };
    auto pv = [&](lds_cptr vt, lds_cptr px) {
        const int ln = opaque(lane), lhi = ln >> 5;
        const int g16 = ln >> 4, i16 = ln & 15, rr = i16 >> 2, pp = i16 & 3;
        const int vx = 2 * (g16 & 1) + (pp >> 1);
        const lds_cptr v0 = vt + (4 * lhi + rr) * NSTRIDE + 256 * wave + 8 * (pp & 1);
        auto v_frag = [&](int i) -> u32x4 {
            const lds_cptr at = v0 + 16 * (i >> 2) * NSTRIDE;
            const int c = (4 * (i & 3) + vx) ^ (4 * rr + lhi);                // row 8 further on: nsw + 2
            const s16x4 va = lds_read_tr16(at + 16 * c), vb = lds_read_tr16(at + 8 * NSTRIDE + 16 * (c ^ 2));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        u32x4 pb[2], v[3];
        pb[0] = lds_ld<u32x4>(px + (lhi * NARROW + (ln & 31)) * 16);
#pragma unroll
        for (int i = 0; i < 3; ++i) v[i] = v_frag(i);
        pb[1] = lds_ld<u32x4>(px + ((2 + lhi) * NARROW + (ln & 31)) * 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[i & 3] = mfma_bf16(v[i % 3], pb[i >> 2], o[i & 3]);
            if (i + 3 < 8) v[i % 3] = v_frag(i + 3);
        }
    };

    const int nspans = k1 > k0 ? (int)(((int64_t)k1 - k0 + SPAN - 1) / SPAN) : 0;
    auto start_of = [&](int c) { return (int)(k0 + (int64_t)c * SPAN); };
    bool first = true, again = false;
    // scores and probabilities of tile i, then its registers take tile i + 2
    auto take = [&](Raw& x, int i, int c0) {
        const f32x4 s = scores(x, i, c0, T0 + (i & 1) * VT);
        if (i + 2 < ntiles) fetch(x, i + 2);
        if (first) {
            const float top = top_of(s) * c_s;
            m_ref = top == -INFINITY ? 0.0f : top;
            m_ref -= (float)lift_of<false>(k1 - k0, false);
            first = false;
        }
        p_out(s, PX + (i & 1) * PT);
        // (every wave's V and P of tile i are there, and every wave is done with tile i - 1)
        tile_barrier();
    };
    while (true) {
#pragma unroll
        for (int m = 0; m < 4; ++m) o[m] = f32x16{};
        l_lane = 0.0f;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            resolve(c0);
            if (ntiles == 0) continue;
            Raw x0, x1{};
            fetch(x0, 0);
            if (ntiles > 1) fetch(x1, 1);
            take(x0, 0, c0);
            for (int i = 0; i < ntiles; i += 2) {
                pv(T0, PX);
                if (i + 1 < ntiles) {
                    take(x1, i + 1, c0);
                    pv(T0 + VT, PX + PT);
                }
                if (i + 2 < ntiles) take(x0, i + 2, c0);
            }
        }
        // row sums over the lanes and halves that share a row
        float l = l_lane;
        l += __shfl_xor(l, 16, 64), l += __shfl_xor(l, 32, 64);
        const uint64_t anys = __builtin_amdgcn_ballot_w64(any);
        any = ((anys >> (lane & 15)) & 0x0001000100010001ull) != 0;
        __syncthreads();
        if (threadIdx.x == 0) s_misc[1] = 0, s_misc[2] = 0, s_misc[3] = 0;
        if (q == 0) s_top[half][my] = any ? l : -1.0f;
        __syncthreads();
        // (a half with no position: -1, below every sum; a NaN stays one)
        const float l0 = s_top[0][my], l1 = s_top[1][my];
        any = !(l0 == -1.0f && l1 == -1.0f);
        l = (l0 == -1.0f ? 0.0f : l0) + (l1 == -1.0f ? 0.0f : l1);
        const int lift = lift_of<false>(k1 - k0, false);
        const bool held = l > __builtin_ldexpf(1.0f, lift - 40) && l < __builtin_ldexpf(1.0f, lift + 40);
        if (!again && any && !held) s_misc[1] = 1;
        if (any && l >= 0.5f) s_misc[2] = 1;
        l_lane = l;
        __syncthreads();
        bool served = again || __builtin_amdgcn_readfirstlane(s_misc[1]) == 0;
        if (!again && __builtin_expect(served && __builtin_amdgcn_readfirstlane(s_misc[2]) != 0, false)) {
            float z = 0.0f;                    // (as in the tiled kernel)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r) z = __builtin_fmaf(o[m][r], 0.0f, z);
            if (z != 0.0f) s_misc[3] = 1;
            __syncthreads();
            served = __builtin_amdgcn_readfirstlane(s_misc[3]) == 0;
        }
        if (served) break;
        again = true;
        float top = -INFINITY;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            resolve(c0);
            for (int i = 0; i < ntiles; ++i) {
                Raw x;
                fetch(x, i);
                top = fmaxf(top, top_of(scores(x, i, c0, T0)));
            }
        }
        m_ref = top == -INFINITY ? 0.0f : top * c_s;
        m_ref -= (float)lift_of<false>(k1 - k0, true);
    }

    // ---- O / l, LSE: rows' values from the scoring lanes to the lanes that hold O ----
    const int lift = lift_of<false>(k1 - k0, again);
    const float lse = too_long ? __builtin_nanf("")
                               : (m_ref + (float)lift + __builtin_amdgcn_logf(__builtin_ldexpf(l_lane, -lift))) * LN2;
    __syncthreads();
    // (lane numbers anew: none of what follows is kept through the tile loop)
    const int ln = fresh_lane(), mine = 16 * rh + (ln & 15);
    if (ln < 16 && half == 0) {
        s_top[0][mine] = too_long ? __builtin_nanf("") : (any ? 1.0f / l_lane : 0.0f);
        const int64_t at = (int64_t)blk.first * p.H + blk.r0 + mine;
        if (mine >= blk.rows) {
        } else if (p.ns > 1) {
            p.part_lse[(int64_t)split * p.T * p.H + at] = any || too_long ? lse : -FLT_MAX;
        } else if (p.lse) {
            p.lse[at] = any || too_long ? lse : INFINITY;
        }
    }
    __syncthreads();
    const int hi = ln >> 5, r32 = ln & 31;
    const float inv = s_top[0][r32];
    if (p.ns == 1) {
        constexpr int OUT_STRIDE = D_VO * 2 + 16;
        static_assert(32 * OUT_STRIDE <= 2 * VT, "the stage fits the tile buffers");
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = {o[m][4 * g] * inv, o[m][4 * g + 1] * inv, o[m][4 * g + 2] * inv, o[m][4 * g + 3] * inv};
                lds_st<u32x2>(T0 + r32 * OUT_STRIDE + 2 * (128 * wave + 32 * m + 8 * g + 4 * hi),
                              __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4)));
            }
        __syncthreads();
        const bool o16 = ((p.o_sb | p.o_st | p.o_sh) & 7) == 0 && ((uintptr_t)p.out & 15) == 0;
        for (int k = 0; k < 8; ++k) {
            const int r = 8 * wave + k;
            if (r >= blk.rows) break;
            const int t = blk.first + (blk.r0 + r) / p.H, h = (blk.r0 + r) % p.H;
            const u32x4 v = lds_ld<u32x4>(T0 + r * OUT_STRIDE + 16 * ln);
            __bf16* const dst = p.out + (LIST ? token_at(t, p.s_q, p.o_sb, p.o_st) : (int64_t)t * p.o_st) + (int64_t)h * p.o_sh + 8 * ln;
            if (o16) {
                *reinterpret_cast<u32x4*>(dst) = v;
            } else {
                reinterpret_cast<u32x2*>(dst)[0] = u32x2{v[0], v[1]};
                reinterpret_cast<u32x2*>(dst)[1] = u32x2{v[2], v[3]};
            }
        }
    } else {
        constexpr int PST = D_VO + 16;
        static_assert(4 * 32 * PST <= 2 * VT + 2 * PT, "four waves' stages fit the tile buffers");
        const lds_ptr stg = T0 + wave * 32 * PST;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = {o[m][4 * g] * inv, o[m][4 * g + 1] * inv, o[m][4 * g + 2] * inv, o[m][4 * g + 3] * inv};
                lds_st<f32x4>(stg + r32 * PST + 4 * (32 * m + 8 * g + 4 * hi), v);
            }
        float* const dst0 = p.part_o + ((int64_t)split * p.T * p.H + (int64_t)blk.first * p.H + blk.r0) * D_VO;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int r = 2 * k + (ln >> 5);
            const f32x4 v = lds_ld<f32x4>(stg + r * PST + 16 * (ln & 31));
            if (r < blk.rows) *reinterpret_cast<f32x4*>(dst0 + (int64_t)r * D_VO + 128 * wave + 4 * (ln & 31)) = v;
        }
    }
}
