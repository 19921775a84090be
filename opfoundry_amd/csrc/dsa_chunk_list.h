// dsa_chunk_list.h - calls over lists of positions (dsa_mla_decode, dsa_mla_prefill on
// DSA_KV_MXFP4 rows): their workgroups, and their entries' cache rows.  Part of dsa_chunk.hip.

// The work of a call over lists: a workgroup takes m heads of one token.  The groups of a token read the
// same rows and lie 8 workgroups apart, on one XCD; the last tokens % 8 are taken group by group.
__device__ __forceinline__ Work list_work(const ChunkParams& p, int32_t m) {
    const int32_t groups = (p.H + m - 1) / m;
    int32_t t = blockIdx.x, g = 0;
    if (groups > 1) {
        const int32_t whole = p.T / 8 * 8 * groups;
        if (t < whole) {
            const int32_t blk = t / (8 * groups), rem = t - blk * 8 * groups;
            g = rem >> 3;
            t = 8 * blk + (rem & 7);
        } else {
            const int32_t i = t - whole;
            g = i % groups;
            t = p.T / 8 * 8 + i / groups;
        }
    }
    // (a prompt's last tokens have the longest lists: first)
    if (p.causal == 2) t = p.T - 1 - t;
    Work w{};
    w.blk.b = t / p.s_q;
    w.blk.first = t;
    w.blk.r0 = g * m;
    w.blk.rows = min(m, p.H - w.blk.r0);
    w.split = blockIdx.y;
    w.per = p.per_split;
    return w;
}
// Addresses of token t's first head, in elements.
__device__ __forceinline__ int64_t token_at(int32_t t, int32_t s_q, int64_t sb, int64_t st) {
    const int32_t b = t / s_q;
    return b * sb + (t - b * s_q) * st;
}

// Entries [c0, c0 + SPAN) below k1 of a token's list -> the cache rows of the valid ones, without gaps, and how
// many; the last 64 are filled up with the first row.  `counts`: four words of LDS; `beside`: done while
// the entries are on their way.  (Ends with a barrier; begins
// with one that ends the use of the span before.)
template <class Beside>
__device__ __forceinline__ int32_t resolve_list(const ChunkParams& p, const Block& blk, int c0, int k1, int32_t* s_rows,
                                                int32_t* counts, Beside beside) {
    const int lane = fresh_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = 64 * wave + lane;
    const int32_t tt = blk.first - blk.b * p.s_q;
    const int32_t* const idx = p.indices + blk.b * p.idx_sb + tt * p.idx_st;
    int32_t j[8], ent[8], row[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int k = c0 + 8 * tid + e;
        j[e] = k < k1 ? idx[k] : -1;
    }
    beside();
    const int64_t len = p.lens ? (int64_t)p.lens[blk.b] : p.list_len;
    int64_t jmax = len;
    if (p.causal == 1) jmax = min(len, len - p.s_q + tt + 1);
    else if (p.causal == 2) jmax = min(len, blk.b + p.causal_offset + 1);
    const bool paged = p.pages.table != nullptr;
    const int32_t* const table = p.pages.table + blk.b * p.pages.table_stride;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        ent[e] = dsa_rows::topk_block(j[e], jmax, p.pages.block_size, p.pages.shift);
        if (paged && ent[e] >= 0) ent[e] = table[ent[e]];
    }
    int32_t n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // (a negative entry's rows lie below 0)
        row[e] = ent[e] < 0 ? -1
                            : (int32_t)dsa_rows::topk_finish(j[e], 0, ent[e], paged, p.pages.block_size, p.pages.shift,
                                                             blk.b * p.pages.batch_stride, p.rows);
        n += row[e] >= 0 ? 1 : 0;
    }
    const int32_t upto = (int32_t)wave_incl_scan((uint32_t)n);
    __syncthreads();
    if (lane == 63) counts[wave] = upto;
    __syncthreads();
    int32_t at = upto - n, total = 0;
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) {
        const int32_t c = counts[w];
        at += w < wave ? c : 0;
        total += c;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (row[e] >= 0) s_rows[at++] = row[e];
    total = __builtin_amdgcn_readfirstlane(total);
    __syncthreads();
    const int32_t end = (total + 63) / 64 * 64;
    if (tid < 64 && total + tid < end) s_rows[total + tid] = s_rows[0];
    __syncthreads();
    return total;
}
