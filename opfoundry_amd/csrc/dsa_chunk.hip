// dsa_chunk.hip - gfx950 kernels of dsa_mla_chunk (include/dsa_chunk.h): dense
// attention of a chunk's tokens over the paged latent cache.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>
#include <algorithm>

#include "../../include/dsa_chunk.h"
#include "dsa_seq.h"

namespace {

#include "dsa_lds.h"

constexpr int D_QK = DSA_MLA_D_QK, D_VO = DSA_MLA_D_VO;
constexpr int NWAVE = 4, NTHR = 64 * NWAVE;
constexpr int TILE = 32;
constexpr int CUS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr unsigned FP8_SCALE_LIMIT_BITS = 0x43000000u;   // 128.0f

struct ChunkParams {
    const __bf16* q;
    int64_t q_st, q_sh;
    const int32_t* indptr;
    const int32_t* lens;
    const unsigned char* kv;
    int64_t rows, row_bytes;
    dsa_seq::Pages pages;
    __bf16* out;
    int64_t o_st, o_sh;
    float* lse;
    float* part_o;       // fp32 partials [split][t][h][512] and their LSE [split][t][h] (log2 units kept as ln)
    float* part_lse;
    int32_t T, B, H, causal, max_len, ns, per_split;
    float scale_log2;
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
    return x;
}

// positions that token t of sequence b attends: [0, limit)
__device__ __forceinline__ int64_t limit_of(const ChunkParams& p, int32_t b, int32_t t) {
    const int64_t len = p.lens[b];
    const int64_t own = dsa_seq::position_of(p.indptr, p.lens, b, t) + 1;
    const int64_t lim = p.causal && own < len ? own : len;
    return lim < 0 ? 0 : lim;
}

// One workgroup per (token, head, split): each wave takes every fourth position,
// a lane 8 NoPE values and one RoPE value; the four waves' sums are joined in LDS.
template <int FMT>
__global__ void __launch_bounds__(NTHR) dsa_mla_chunk_row_kernel(const ChunkParams p) {
    __shared__ float s_o[NWAVE][D_VO];
    __shared__ float s_m[NWAVE], s_l[NWAVE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(blockIdx.x / (unsigned)p.H), h = (int)(blockIdx.x % (unsigned)p.H), split = blockIdx.y;
    const int32_t b = seq_of(p.indptr, p.B, t);
    if (b == NO_SEQ) return;
    const int64_t limit = limit_of(p, b, t);
    const bool too_long = p.lens[b] > p.max_len;
    const int64_t k0 = (int64_t)split * p.per_split, k1 = min(limit, k0 + p.per_split);
    float q[9], o[8] = {};
    const __bf16* qp = p.q + (int64_t)t * p.q_st + (int64_t)h * p.q_sh;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (float)qp[8 * lane + i];
    q[8] = (float)qp[512 + lane];
    float m = -INFINITY, l = 0.0f;
    bool bad = false;
    for (int64_t j = k0 + wave; j < k1; j += NWAVE) {
        const int64_t row = dsa_seq::row_of(p.pages, b, j, p.rows);
        if (row < 0) continue;
        const unsigned char* r = p.kv + row * p.row_bytes;
        float k[9];
        if constexpr (FMT == DSA_KV_BF16) {
            const __bf16* rb = (const __bf16*)r;
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = (float)rb[8 * lane + i];
            k[8] = (float)rb[512 + lane];
        } else {
            const u32x2 c = *reinterpret_cast<const u32x2*>(r + 8 * lane);
            const float sc = *reinterpret_cast<const float*>(r + 512 + 4 * (lane >> 4));
            bad |= __builtin_amdgcn_ballot_w64(__float_as_uint(sc) >= FP8_SCALE_LIMIT_BITS) != 0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
                k[4 * w] = lo[0] * sc, k[4 * w + 1] = lo[1] * sc, k[4 * w + 2] = hi[0] * sc, k[4 * w + 3] = hi[1] * sc;
            }
            k[8] = (float)reinterpret_cast<const __bf16*>(r + 528)[lane];
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 9; ++i) s = __builtin_fmaf(q[i], k[i], s);
        s = wave_sum(s) * p.scale_log2;
        const float mn = fmaxf(m, s);
        const float a = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(s - mn);
        l = l * a + e;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __builtin_fmaf(e, k[i], o[i] * a);
        m = mn;
    }
    const bool any = l != 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s_o[wave][8 * lane + i] = o[i];
    if (lane == 0) s_m[wave] = any ? m : -INFINITY, s_l[wave] = bad || too_long ? __builtin_nanf("") : l;
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) mm = fmaxf(mm, s_m[w]);
    float f[NWAVE];
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w] - mm);
        ll += s_l[w] * (s_l[w] == s_l[w] ? f[w] : 1.0f);
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    const float lse = (mm + __builtin_amdgcn_logf(ll)) * LN2;
    const int d = 2 * threadIdx.x;
    float v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < NWAVE; ++w) x += f[w] == 0.0f ? 0.0f : s_o[w][d + i] * f[w];
        v[i] = x * inv;
    }
    if (p.ns > 1) {
        const int64_t at = ((int64_t)split * p.T + t) * p.H + h;
        p.part_o[at * D_VO + d] = v[0], p.part_o[at * D_VO + d + 1] = v[1];
        if (threadIdx.x == 0) p.part_lse[at] = ll == 0.0f ? -FLT_MAX : lse;
    } else {
        __bf16* op = p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh;
        op[d] = (__bf16)v[0], op[d + 1] = (__bf16)v[1];
        if (threadIdx.x == 0 && p.lse) p.lse[(int64_t)t * p.H + h] = ll == 0.0f ? INFINITY : lse;
    }
}

// Joins the partials of a row's splits, one wave a row: a lane holds 8 of its 512
// values.  Splits past the row's positions wrote nothing and are not read.
__global__ void __launch_bounds__(NTHR) dsa_mla_chunk_combine_kernel(const ChunkParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * NWAVE + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)p.T * p.H) return;
    const int t = (int)(row / p.H), h = (int)(row - (int64_t)t * p.H);
    const int32_t b = seq_of(p.indptr, p.B, t);
    if (b == NO_SEQ) return;
    const int64_t limit = limit_of(p, b, t);
    const int ns = (int)min((int64_t)p.ns, (limit + p.per_split - 1) / p.per_split);
    const int64_t step = (int64_t)p.T * p.H;
    const float mine = lane < ns ? p.part_lse[lane * step + row] : -FLT_MAX;     // at most 64 splits
    float top = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const bool any = __builtin_amdgcn_ballot_w64(mine != -FLT_MAX) != 0;
    const float w = mine == -FLT_MAX ? 0.0f : __builtin_amdgcn_exp2f((mine - top) * LOG2E);
    const float total = wave_sum(w);
    float o[8] = {};
    for (int s = 0; s < ns; ++s) {
        const float f = __shfl(w, s, 64);
        if (f == 0.0f) continue;
        const float* src = p.part_o + (s * step + row) * D_VO + 8 * lane;
        const f32x4 x = *reinterpret_cast<const f32x4*>(src), y = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(f, x[i], o[i]), o[4 + i] = __builtin_fmaf(f, y[i], o[4 + i]);
    }
    const float nan = p.lens[b] > p.max_len ? __builtin_nanf("") : 0.0f;
    const float inv = any ? 1.0f / total + nan : nan;
    const f32x8 r = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv};
    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_convertvector(r, bf16x8));
    u32x2* const dst = reinterpret_cast<u32x2*>(p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + 8 * lane);
    dst[0] = u32x2{v[0], v[1]};
    dst[1] = u32x2{v[2], v[3]};
    if (lane == 0 && p.lse) p.lse[row] = nan != 0.0f ? nan : (any ? top + __builtin_amdgcn_logf(total) * LN2 : INFINITY);
}

// ------------------------------------------------------------------- host

int splits_of(const dsa_mla_chunk_args* a, int32_t* per) {
    int ns = a->num_splits;
    if (ns == 0) {
        // about two workgroups per CU, at least 256 positions each
        const int64_t blocks = std::max<int64_t>(1, (int64_t)a->T * a->H / 32);
        const int64_t want = std::max<int64_t>(1, 2 * CUS / blocks);
        ns = (int)std::min<int64_t>({want, std::max(1, a->max_kv_len / 256), DSA_MLA_MAX_SPLITS});
    }
    const int64_t each = (a->max_kv_len + (int64_t)ns - 1) / ns;
    *per = (int32_t)std::min<int64_t>(INT32_MAX - TILE + 1, std::max<int64_t>(TILE, (each + TILE - 1) / TILE * TILE));
    return ns;
}

size_t workspace_of(int ns, int64_t T, int64_t H) {
    return ns > 1 ? (size_t)ns * T * H * (D_VO + 1) * sizeof(float) : 0;
}

int validate(const dsa_mla_chunk_args* a) {
    if (!a) return DSA_ERR_NULL_POINTER;
    if (a->kv_format != DSA_KV_BF16 && a->kv_format != DSA_KV_FP8_656) return DSA_ERR_BAD_FORMAT;
    if (a->T < 0 || a->B < 0 || a->H < 1 || a->max_kv_len < 0 || a->kv_total_rows < 0 || a->kv_total_rows > INT32_MAX)
        return DSA_ERR_BAD_SHAPE;
    if (a->max_kv_len > DSA_MLA_MAX_LIST) return DSA_ERR_BAD_SHAPE;
    if (a->num_splits < 0 || a->num_splits > DSA_MLA_MAX_SPLITS) return DSA_ERR_BAD_SPLITS;
    // (rows of queries, with a block of each sequence's own, stay below 2^31)
    if ((int64_t)a->T * a->H + (int64_t)128 * a->B > INT32_MAX) return DSA_ERR_BAD_SHAPE;
    const int64_t least = a->kv_format == DSA_KV_BF16 ? D_QK : DSA_MLA_FP8_ROW_BYTES;
    const int64_t unit = a->kv_format == DSA_KV_BF16 ? 2 : 1;
    if (a->kv_stride_row != 0 &&
        (a->kv_stride_row < least || (a->kv_stride_row * unit) % 16 || a->kv_stride_row * unit > UINT32_MAX))
        return DSA_ERR_BAD_STRIDE;
    if (a->block_table) {
        if (a->block_size < 1 || a->table_blocks < 0 || (int64_t)a->block_size * a->table_blocks > INT32_MAX)
            return DSA_ERR_BAD_SHAPE;
        if (a->block_table_stride < 0) return DSA_ERR_BAD_STRIDE;
    } else if (a->kv_batch_stride < 0) {
        return DSA_ERR_BAD_STRIDE;
    }
    if (a->T == 0 || a->B == 0) return DSA_OK;
    if (!a->q || !a->out || !a->q_indptr || !a->seq_lens || (a->kv_total_rows > 0 && !a->kv_cache))
        return DSA_ERR_NULL_POINTER;
    if (a->q_stride_t < 0 || a->q_stride_h < 0 || (a->q_stride_t % 8) || (a->q_stride_h % 8) || a->o_stride_t < 0 ||
        a->o_stride_h < 0 || (a->o_stride_t % 4) || (a->o_stride_h % 4))
        return DSA_ERR_BAD_STRIDE;
    if (((uintptr_t)a->q & 15) || ((uintptr_t)a->kv_cache & 15) || ((uintptr_t)a->out & 7)) return DSA_ERR_BAD_STRIDE;
    return DSA_OK;
}

}  // namespace

extern "C" {

int dsa_mla_chunk_num_splits(const dsa_mla_chunk_args* a, int32_t* num_splits) {
    if (!num_splits) return DSA_ERR_NULL_POINTER;
    const int rc = validate(a);
    if (rc) return rc;
    int32_t per;
    *num_splits = splits_of(a, &per);
    return DSA_OK;
}

int dsa_mla_chunk_workspace_size(const dsa_mla_chunk_args* a, size_t* bytes) {
    if (!bytes) return DSA_ERR_NULL_POINTER;
    const int rc = validate(a);
    if (rc) return rc;
    int32_t per;
    *bytes = a->B == 0 ? 0 : workspace_of(splits_of(a, &per), a->T, a->H);
    return DSA_OK;
}

int dsa_mla_chunk(const dsa_mla_chunk_args* a, void* ws, size_t ws_bytes, void* stream) {
    const int rc = validate(a);
    if (rc) return rc;
    if (a->T == 0 || a->B == 0) return DSA_OK;
    ChunkParams p{};
    p.ns = splits_of(a, &p.per_split);
    const size_t need = workspace_of(p.ns, a->T, a->H);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) return DSA_ERR_WORKSPACE;
    p.q = (const __bf16*)a->q;
    p.q_st = a->q_stride_t, p.q_sh = a->q_stride_h;
    p.indptr = a->q_indptr, p.lens = a->seq_lens;
    p.kv = (const unsigned char*)a->kv_cache;
    p.rows = a->kv_total_rows;
    p.row_bytes = a->kv_format == DSA_KV_BF16 ? 2 * (a->kv_stride_row ? a->kv_stride_row : D_QK)
                                              : (a->kv_stride_row ? a->kv_stride_row : DSA_MLA_FP8_ROW_BYTES);
    p.pages = dsa_seq::make_pages(a->block_table, a->block_table_stride, a->table_blocks, a->block_size,
                                  a->kv_batch_stride);
    p.out = (__bf16*)a->out;
    p.o_st = a->o_stride_t, p.o_sh = a->o_stride_h;
    p.lse = a->lse;
    p.part_o = (float*)ws;
    p.part_lse = p.part_o + (size_t)p.ns * a->T * a->H * D_VO;
    p.T = a->T, p.B = a->B, p.H = a->H, p.causal = a->causal, p.max_len = a->max_kv_len;
    p.scale_log2 = a->sm_scale * LOG2E;
    const dim3 grid((unsigned)((int64_t)a->T * a->H), (unsigned)p.ns);
    if (a->kv_format == DSA_KV_BF16)
        hipLaunchKernelGGL(dsa_mla_chunk_row_kernel<DSA_KV_BF16>, grid, dim3(NTHR), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(dsa_mla_chunk_row_kernel<DSA_KV_FP8_656>, grid, dim3(NTHR), 0, (hipStream_t)stream, p);
    if (hipGetLastError() != hipSuccess) return DSA_ERR_HIP;
    if (p.ns > 1) {
        const int64_t rows = (int64_t)a->T * a->H;
        hipLaunchKernelGGL(dsa_mla_chunk_combine_kernel, dim3((unsigned)((rows + NWAVE - 1) / NWAVE)), dim3(NTHR), 0,
                           (hipStream_t)stream, p);
        if (hipGetLastError() != hipSuccess) return DSA_ERR_HIP;
    }
    return DSA_OK;
}

}  // extern "C"
