// dsa_chunk.hip - gfx950 kernels of dsa_mla_chunk (include/dsa_chunk.h): dense
// attention of a chunk's tokens over the paged latent cache.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>
#include <cmath>
#include <algorithm>
#include <type_traits>

#include "../../include/dsa_chunk.h"
#include "dsa_overlap.h"
#include "dsa_seq.h"

namespace {

#include "dsa_lds.h"

constexpr int D_QK = DSA_MLA_D_QK, D_VO = DSA_MLA_D_VO;
constexpr int NWAVE = 4, NTHR = 64 * NWAVE;
constexpr int TILE = 32;
constexpr int CUS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr float FP16_MAX = 65504.0f;
constexpr unsigned FP8_SCALE_LIMIT_BITS = 0x43000000u;   // 128.0f

constexpr int NARROW = 32;                   // rows of a workgroup of the kernel for few rows
// What a workgroup of a kernel takes, us: `start`, and `tile` for each 32 positions (`pair` where two
// share a CU).
struct Kernel {
    float start, tile, pair;
};
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
    int32_t common;      // of H and the rows of a block (block_start)
    int32_t* dealt;      // where the positions of a split that the device chose are kept for the join (null:
                         // splits of per_split positions)
    float scale_log2;
    Kernel kernel;
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

// ---------------------------------------------------------------------------
// The tiled kernel: one workgroup per 128 rows and split.  A row is one head of
// one token; a block holds 128 consecutive rows of one sequence (token-major), so
// any head count fills it, and all its rows attend the same cache rows but for the
// causal end.  The cache rows come in tiles of 32, three tile buffers deep:
//   QK^T   wave w: S^T[32 positions x its 32 rows], 36 k-steps of 32x32x16, Q in registers
//   P      exp2 against a fixed reference (the first tile's maximum of the row, which stands
//          for 2^lift), 16 bits, exchanged through LDS
//   PV     wave w: O^T[dims 128 w .. +127 x 128 rows] in 256 accumulation registers
// Iteration i computes QK^T of tile i + 1, then PV of tile i with the exponentials of
// tile i + 1 between its matrix instructions: one barrier a tile.  Q and O are 400 of a
// CU's 512 KB of registers, which is why a workgroup is 128 rows and fills a CU.
// Measured (1024 tokens of 128 heads, 8192 bf16 rows before them): 1.98 ms, 1.25 PFLOP/s, 92 % of what
// a product of two 16384 x 16384 matrices reaches here (2.06 ms in sessions where the card holds a lower
// clock); matrix units busy 54 % of the cycles at 1.8 to 2.2 GHz.  656-byte rows (two prompts of 1915 and
// 1782 tokens): 1.27 ms, 750 TFLOP/s, 2.4 us a tile: every wave converts the whole tile's codes for its
// scores (8 vector instructions to a matrix instruction, matrix units busy 30 %).  A shared tile of
// converted codes has no room beside V's two and the three raw ones.  A workgroup's Q and O pass through
// memory once, 8 us each; the next workgroup's Q read ahead from within the loop, whose loads are waited
// for in order, cost more there than it saved (1296 -> 1367 us).
// ---------------------------------------------------------------------------
constexpr int BLOCK = 128;                   // rows of a workgroup
constexpr int SPAN = 2048;                   // positions resolved to cache rows at a time
// A tile in LDS: NoPE row r at r * NOPE_STRIDE, its 16-byte piece c at c ^ nope_sw(r); RoPE
// row r at ROPE_OFF + 128 r, piece c at c ^ rope_sw(r).  The pad moves every row by four
// banks groups and the XOR parts rows four apart, so that the K reads (one piece of 16
// rows) and the transposed V reads (four pieces of four rows) meet no bank twice.
constexpr int NOPE_STRIDE = 1088;
constexpr int ROPE_OFF = TILE * NOPE_STRIDE;
constexpr int TILE_BYTES = ROPE_OFF + TILE * 128;
constexpr int P_BYTES = 2 * NWAVE * 64 * 16;
constexpr int KS_NOPE = 32, KS = 36;         // 16-deep k-steps of NoPE, and with RoPE
constexpr int LPW = TILE / NWAVE + 1;        // loads of a wave and tile
// 656-byte rows: the rows as they lie in the cache, back to back (41 pieces of 16 bytes each), three
// tiles of them; V in two tiles of fp16 NoPE values in the layout above.
constexpr int FP8_ROW = DSA_MLA_FP8_ROW_BYTES;
constexpr int RAW_PIECES = TILE * FP8_ROW / 16;          // 1312
constexpr int RAW_LOADS = (RAW_PIECES + 63) / 64;        // 21 loads of 1 KB
constexpr int RAW_BYTES = RAW_LOADS * 1024;
constexpr int RAW_LPW = (RAW_LOADS + NWAVE - 1) / NWAVE; // of wave 0 (6); the others 5
static_assert(RAW_LOADS == NWAVE * (RAW_LPW - 1) + 1 && RAW_PIECES % 64 == 32, "the last load is wave 0's, half of it spare");
constexpr int V_BYTES = TILE * NOPE_STRIDE;
__device__ __forceinline__ int nope_sw(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int rope_sw(int r) { return (r >> 1) & 7; }

__device__ __forceinline__ f32x16 mfma_bf16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// O += A B on an accumulation register tile; the wait states before it (a vector write of
// an operand: two) and around accesses of O from outside (o_fence) are written out, since
// the compiler does not see a matrix instruction here.
template <bool F16>
__device__ __forceinline__ void mfma_o(f32x16& acc, u32x4 a, u32x4 b) {
    if constexpr (F16)
        asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
    else
        asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
// This lane's v or that of the lane 32 further (a ballot, which every lane takes part in, whatever its own v)
__device__ __forceinline__ bool either(bool v) {
    const uint64_t all = __builtin_amdgcn_ballot_w64(v);
    return (((uint32_t)all | (uint32_t)(all >> 32)) >> (threadIdx.x & 31)) & 1;
}
// 8 e4m3 codes -> 8 bf16 (exact)
__device__ __forceinline__ u32x4 codes_bf16(unsigned c0, unsigned c1) {
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c0, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c0, 1.0f, true)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c1, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c1, 1.0f, true))};
}
__device__ __forceinline__ void o_fence(f32x16 (&o)[16]) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7"
                 : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]),
                   "+a"(o[8]), "+a"(o[9]), "+a"(o[10]), "+a"(o[11]), "+a"(o[12]), "+a"(o[13]), "+a"(o[14]), "+a"(o[15]));
}

// A workgroup's rows: those of sequence b from row r0 (of its n * H) on.
struct Block {
    int32_t b, r0, rows;       // rows = 0: nothing to do
    int32_t first;             // token of row 0 of the sequence
    int32_t len, end;          // positions; token t is position len - end + t
};
__device__ __forceinline__ Block find_block(const ChunkParams& p, int64_t x, int32_t m) {
    auto start = [&](int32_t i) { return dsa_seq::block_start(min(max(p.indptr[i], 0), p.T), i, p.H, m, p.common); };
    Block k{};
    k.b = count_upto(p.B, x, start);
    if (k.b >= p.B) return k;
    const int64_t local = x - start(k.b);
    k.first = min(max(p.indptr[k.b], 0), p.T);
    k.end = p.indptr[k.b + 1];
    k.len = p.lens[k.b];
    const int64_t left = (int64_t)(min(max(k.end, 0), p.T) - k.first) * p.H - local * m;
    if (local < 0 || left <= 0) return k;
    k.r0 = (int32_t)(local * m);
    k.rows = (int32_t)min(left, (int64_t)m);
    return k;
}
// positions that token t (of the block's sequence) attends: [0, limit)
__device__ __forceinline__ int32_t limit_in(const ChunkParams& p, const Block& k, int32_t t) {
    const int64_t own = (int64_t)k.len - k.end + t + 1;
    return (int32_t)max((int64_t)0, p.causal ? min(own, (int64_t)k.len) : (int64_t)k.len);
}

// The power of two that P of a row's reference score stands for, of a split of n positions.
// 656-byte rows: P in fp16 loses up to 2^-25 where it is below 2^-14, which n positions could add up to n 2^-25
// of a row's sum.  Past 2^14 positions the first tile's maximum is 2^lift instead of 1, so that the loss stays below
// 2^-11 of it; P may then grow by 16 - lift powers of two before the row starts again.
// bf16 rows, whose values and P have the range of fp32: O passes it where a sum of P above 1 meets values near the
// largest.  With the maximum at 2^-15 most rows' sums stay below 1/2, and O below the largest value; for the others O
// is looked at, and a row starts again with its exact maximum so low that n of them add up to 1/2 at most.
template <bool FP8>
__device__ __forceinline__ int lift_of(int32_t n, bool again) {
    const int bits = n <= 1 ? 0 : 32 - __builtin_clz((unsigned)n - 1);         // ceil(log2 n)
    if (FP8) return max(0, min(14, bits - 14));
    return again ? -1 - bits : -15;
}

constexpr float PART_BYTES_US = 5.3e6f;            // at which splits' partials are written and read again
constexpr float JOIN_SPLIT_US = 0.1f;              // and what the join's wait for one more split costs

// Reductions and a running sum over a wave's lanes by moves within and between its rows of 16.
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t moved(int32_t v, int32_t none) {
    return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
template <class T, class F>
__device__ __forceinline__ T scan(T v, T none, F op) {
    auto step = [&](auto ctrl, auto rows) {
        v = op(v, __builtin_bit_cast(T, moved<decltype(ctrl)::value, decltype(rows)::value>(
                      __builtin_bit_cast(int32_t, v), __builtin_bit_cast(int32_t, none))));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});        // from 1, 2, 4, 8 lanes below
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});        // row 0's last lane to row 1, 2's to 3
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});        // lane 31 to rows 2 and 3
    return v;
}
template <class T, class F>
__device__ __forceinline__ T over_lanes(T v, T none, F op) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, scan(v, none, op)), 63));
}

// Parts of at most b that `a` has (an integer division takes ten times the code, which a workgroup's first
// waves fetch).
__device__ __forceinline__ int32_t parts(int32_t a, int32_t b) {
    return dsa_seq::parts_by(a, b, __builtin_amdgcn_rcpf((float)b));
}

// The block, the split and the positions of a split of a workgroup.  The host knows a bound of the
// lengths alone.  Where it leaves the splits to the device (`dealt`, at most 64 sequences: a lane holds
// one), each lane prices one split size about the even share of a workgroup's place on the chip
// (`places`: one a CU, or two) and the cheapest is taken: the longest split where all workgroups have a
// place, else their sum with half of a split at the end; and what the partials and their join cost.
// The workgroups are then numbered without gaps, and a sequence's splits are even: workgroups with nothing
// to do between the others make the dispatcher, which hands them to XCDs and shader engines in turn,
// leave CUs idle while others hold three.  16 sequences of 7130 to 19272 bf16 rows, 16 heads: 66 us, of
// 506 workgroups (77 in 16 splits by the bound of the lengths, 366 of them with work); 66 too where that
// bound is four times as much (173).  7 sequences of 1994 to 4772 rows and 28 to 258 tokens of 40 heads:
// 374 us (402 in 2).  Finding it out takes 1.5 us: one token of 128 heads over 1483 656-byte rows 19.1
// and, in 20 splits by the caller's count, 17.3.  Of 50 ragged calls it was 4 % above the best of 13
// counts on average (23 % below to 17 % above).
struct Work {
    Block blk;
    int32_t split, per;
};
__device__ __forceinline__ Work find_work(const ChunkParams& p, int32_t m, int32_t places) {
    // Blocks of one sequence follow one another and read the same rows: four at a time on one XCD
    // (workgroups go to the eight in turn).
    uint32_t x = blockIdx.x;
    if (x < (gridDim.x & ~31u) && (p.dealt || m == NARROW)) x = (x & ~31u) | (x & 7) << 2 | ((x >> 3) & 3);
    // (the last block first: later tokens attend more, and the long ones must not come last)
    if (!p.dealt) return {find_block(p, (int64_t)gridDim.x - 1 - x, m), (int32_t)blockIdx.y, p.per_split};
    const int lane = threadIdx.x & 63, i = min(lane, p.B - 1);
    const int32_t first = min(max(p.indptr[i], 0), p.T), end = p.indptr[i + 1], len = p.lens[i];
    const int64_t rows = lane < p.B ? (int64_t)max(0, min(max(end, 0), p.T) - first) * p.H : 0;
    const int32_t blocks = (int32_t)((rows + m - 1) / m);
    const int32_t tiles = rows > 0 ? (int32_t)((min((int64_t)min(max(len, 0), p.max_len), p.pages.limit) + TILE - 1) / TILE) : 0;
    const float all = over_lanes((float)blocks * (float)tiles, 0.0f, [](float u, float v) { return u + v; });
    const int32_t most = over_lanes(max(tiles, 1), 1, [](int32_t u, int32_t v) { return max(u, v); });
    const int32_t least = parts(most, p.ns);          // no more than ns splits of any
    const float want = all / (float)places * __builtin_amdgcn_exp2f((float)(lane - 15) * 0.1f);
    const int32_t size = lane == 63 ? most : max(least, min(most, (int32_t)fminf(want, 1.0e9f) + 1));
    const float inv = 0.99999f * __builtin_amdgcn_rcpf((float)size);
    float groups = 0.0f;
    const float blocks_f = (float)blocks, tiles_f = (float)tiles;
    for (int j0 = 0; j0 < p.B; j0 += 4)               // (lanes past the last hold no blocks)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            auto at = [&](float v) {
                return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, v), j0 + j));
            };
            groups = __builtin_fmaf(at(blocks_f), __builtin_ceilf(at(tiles_f) * inv), groups);
        }
    const Kernel k = p.kernel;
    const float room = (float)places, tile = groups > (float)CUS && k.pair > 0.0f ? k.pair : k.tile;
    float us = groups <= room ? k.start + tile * (float)size
                              : (tile * all + k.start * groups) / room + 0.5f * tile * (float)size;
    us += groups * (float)m * (2.0f * 4.0f * (D_VO + 1) / PART_BYTES_US) + JOIN_SPLIT_US * (float)most * inv;
    if (lane != 63 && groups > (float)gridDim.x) us = FLT_MAX;
    const float best = over_lanes(us, FLT_MAX, [](float u, float v) { return fminf(u, v); });
    const uint64_t at = __builtin_amdgcn_ballot_w64(us == best);
    int32_t per = __builtin_amdgcn_readlane(size, at ? __builtin_ctzll(at) : 63);
    // the workgroups up to and with a sequence's; whole sequences where the estimate was too low
    uint32_t upto;
    int32_t splits;
    while (true) {
        splits = parts(tiles, per);
        upto = scan((uint32_t)min((int64_t)blocks * splits, ((int64_t)1 << 26) - 1), 0u,
                    [](uint32_t u, uint32_t v) { return u + v; });
        if (per == most || __builtin_amdgcn_ballot_w64(upto > gridDim.x) == 0) break;
        per = most;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.dealt = per;
    Work w{};
    const int b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= x));
    if (b >= p.B) return w;
    const int32_t nb = __builtin_amdgcn_readlane(blocks, b), ns = __builtin_amdgcn_readlane(splits, b);
    const int32_t local = (int32_t)(x - ((uint32_t)__builtin_amdgcn_readlane(upto, b) - (uint32_t)nb * ns));
    w.split = __builtin_amdgcn_readfirstlane(parts(local + 1, nb) - 1);
    w.per = TILE * parts(__builtin_amdgcn_readlane(tiles, b), ns);
    w.blk.b = b;
    w.blk.first = __builtin_amdgcn_readlane(first, b), w.blk.end = __builtin_amdgcn_readlane(end, b);
    w.blk.len = __builtin_amdgcn_readlane(len, b);
    w.blk.r0 = __builtin_amdgcn_readfirstlane((nb - 1 - (local - w.split * nb)) * m);
    w.blk.rows = (int32_t)min((int64_t)(min(max(w.blk.end, 0), p.T) - w.blk.first) * p.H - w.blk.r0, (int64_t)m);
    return w;
}

// the kernel's argument block, in the constant address space
typedef const __attribute__((address_space(4))) ChunkParams* Args;

template <int FMT>
__global__ void __launch_bounds__(NTHR) __attribute__((amdgpu_waves_per_eu(1, 1)))
dsa_mla_chunk_tile_kernel(const ChunkParams p) {
    constexpr bool FP8 = FMT == DSA_KV_FP8_656;
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[FP8 ? 2 * V_BYTES + 3 * RAW_BYTES : 3 * TILE_BYTES];
    __shared__ __attribute__((aligned(16))) float s_scale[FP8 ? 2 * 4 * TILE : 4];    // [tile % 2][group][position]
    __shared__ __attribute__((aligned(16))) unsigned char s_p[2 * P_BYTES];
    __shared__ __attribute__((aligned(16))) int32_t s_rows[SPAN];     // cache rows of a span's positions
    __shared__ uint32_t s_skip[SPAN / TILE];                          // bit j: position j of the tile has no row
    __shared__ uint32_t s_nan[SPAN / TILE];                           // bit j: its row holds a NaN or infinity
    __shared__ int32_t s_misc[4];                                     // [0] a row that may be read, [1] restart, [2] O may
                                                                      // have passed fp32, [3] and has
    __shared__ float s_inv[BLOCK];
    const lds_ptr T0 = (lds_ptr)s_tile, PX = (lds_ptr)s_p;
    const LDS_AS int32_t* const rows_l = (const LDS_AS int32_t*)s_rows;
    // The arguments as the code outside the tile loop reads them: anew where it needs them, so
    // that none is kept in a register across the loop.
    auto args = []() -> Args {
        Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hi = lane >> 5, r32 = lane & 31;
    const Work work = find_work(p, BLOCK, CUS);
    const Block& blk = work.blk;
    const int split = work.split, per = work.per;
    if (blk.rows == 0) return;
    const int t_lo = blk.first + blk.r0 / p.H, t_hi = blk.first + (blk.r0 + blk.rows - 1) / p.H;
    const int lim_lo = limit_in(p, blk, t_lo), lim_hi = limit_in(p, blk, t_hi);
    const bool too_long = blk.len > p.max_len;
    const int k0 = (int)min((int64_t)split * per, (int64_t)lim_hi);
    // (positions without a page end the sequence as far as its rows go)
    const int k1 = too_long ? k0 : (int)min(min((int64_t)lim_hi, p.pages.limit), (int64_t)k0 + per);
    // a split with no positions writes nothing: the combine does not read it
    if (p.ns > 1 && k1 <= k0) return;

    // this lane's row (rows past the block's end are computed on its last one and not stored)
    const int row = blk.r0 + min(32 * wave + r32, blk.rows - 1);
    const int tok = blk.first + row / p.H, head = row % p.H;
    const int limit = limit_in(p, blk, tok);
    // Q: lane (hi, r32) holds 8 dims of row r32 in qf[ks], the k-step's half `hi`: dims 16 ks + 8 hi .. +7; of
    // 656-byte rows, whose codes come 16 to a read, dims 32 j + 16 hi .. +15 in qf[2 j] and qf[2 j + 1] (the order
    // of the dims within a pair of k-steps is free as long as K has the same)
    // They come by way of the tile buffers, 12 k-steps at a time and two such parts in flight: a load of a wave
    // takes 1 KB of one row after the other, where fragments read from memory touch 64 places (with the epilogue's
    // rows stored together 2002 -> 1999 us for 1024 tokens over 8192 bf16 rows, 1302 -> 1292 for the two prompts).
    // In LDS row r of a part is at 384 r, its 16-byte piece c at c ^ (r >> 1) % 8.
    u32x4 qf[KS];
    {
        constexpr int PART = 12, LINE = 32 * PART, BYTES = 32 * LINE;
        static_assert(NWAVE * 2 * BYTES <= sizeof(s_tile) && KS == 3 * PART);
        const uint64_t mine = (uint64_t)(p.q + (int64_t)tok * p.q_st + (int64_t)head * p.q_sh);
        const lds_ptr qb = T0 + wave * 2 * BYTES;
        uint64_t src[PART];
#pragma unroll
        for (int k = 0; k < PART; ++k) {
            const int at = 64 * (k % 3) + lane, r8 = at / 24, r = 8 * (k / 3) + r8;        // piece 64 k + lane
            src[k] = __shfl(mine, r, 64) + 16 * ((at - 24 * r8) ^ ((r >> 1) & 7));
        }
        auto request = [&](int part) {
#pragma unroll
            for (int k = 0; k < PART; ++k)
                lds_dma16((const void*)(src[k] + part * LINE), qb + (part & 1) * BYTES + 1024 * k);
        };
        auto take = [&](int part) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = 0; j < PART; ++j) {
                const int ks = PART * part + j;
                const int c = FP8 && ks < KS_NOPE ? 4 * (j >> 1) + 2 * hi + (j & 1) : 2 * j + hi;
                qf[ks] = lds_ld<u32x4>(qb + (part & 1) * BYTES + r32 * LINE + 16 * (c ^ ((r32 >> 1) & 7)));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        };
        request(0);
        request(1);
        wait_vm<PART>();
        take(0);
        request(2);
        wait_vm<PART>();
        take(1);
        wait_vm<0>();
        take(2);
    }

    // ---- positions [c0, c0 + SPAN) below k1 -> cache rows ----
    // A position without a row, and those from k1 on, are read as some row that exists (every
    // read is of the cache's own rows that the sequence attends) and masked.
    int ntiles = 0;
    auto resolve = [&](int c0) {
        const Args a = args();
        const int64_t rows = a->rows;
        const int32_t bs = a->pages.block_size, shift = a->pages.shift;
        const int32_t* const table = a->pages.table;
        const int tid = 64 * wave + fresh_lane();
        const int at = c0 + 8 * tid;
        int32_t id[8];
        // (positions past the end look up the last one's row: no branch splits the eight reads)
        if (!table) {
            const int64_t base = blk.b * a->pages.batch_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t r = base + min(at + e, k1 - 1);
                id[e] = r < rows ? (int32_t)r : -1;
            }
        } else {
            const int32_t* const mine = table + blk.b * a->pages.table_stride;
            int32_t blk_i[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int q = min(at + e, k1 - 1);
                blk_i[e] = shift >= 0 ? q >> shift : q / bs;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) id[e] = mine[blk_i[e]];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t r = (int64_t)id[e] * bs + (min(at + e, k1 - 1) - blk_i[e] * bs);
                id[e] = r >= 0 && r < rows ? (int32_t)r : -1;
            }
        }
        uint32_t skip = 0;
        int32_t some = -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            skip |= at + e >= k1 || id[e] < 0 ? 1u << e : 0u;
            some = max(some, id[e]);
        }
        __syncthreads();                       // the previous span is done with its rows and tiles
        if (tid == 0) s_misc[0] = -1;
        if (tid < SPAN / TILE) s_nan[tid] = 0;
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
    };

    // ---- tile i of the span -> buffer `slot`.  bf16: wave w rows 8 w .. 8 w + 7 and their RoPE;
    // 656-byte rows: the tile's pieces, load k = w, w + 4, .. of wave w ----
    auto slot_of = [&](int s) -> lds_ptr { return T0 + s * (FP8 ? V_BYTES : TILE_BYTES); };
    auto raw_of = [&](int s) -> lds_ptr { return T0 + 2 * V_BYTES + s * RAW_BYTES; };
    struct Rows {
        int32_t r[8];
        int32_t rope;
    };
    // 656-byte rows whose tile is one run of the cache (dense rows, pages of whole tiles): a load's source
    // is the run's start plus its number and the lane
    const bool runs = FP8 && p.row_bytes == FP8_ROW && (!p.pages.table || p.pages.block_size % TILE == 0);
    auto load_rows = [&](int i) -> Rows {
        Rows g{};
        if constexpr (!FP8) {
            const LDS_AS int32_t* at = rows_l + i * TILE + 8 * wave;
            const u32x4 a = lds_ld<u32x4>((lds_cptr)at), b = lds_ld<u32x4>((lds_cptr)(at + 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g.r[e] = __builtin_amdgcn_readfirstlane((int)a[e]);
                g.r[4 + e] = __builtin_amdgcn_readfirstlane((int)b[e]);
            }
            g.rope = at[opaque(lane) >> 3];
        } else {
            g.r[0] = runs && __builtin_amdgcn_readfirstlane(s_skip[i]) == 0 ? __builtin_amdgcn_readfirstlane(rows_l[i * TILE]) : -1;
            g.r[1] = i;
        }
        return g;
    };
    auto issue = [&](const Rows& g, int slot) {
        const int ln = opaque(lane);
        if constexpr (!FP8) {
            const lds_ptr tb = slot_of(slot);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 8 * wave + e;
                const unsigned char* base = p.kv + (uint64_t)(uint32_t)g.r[e] * (uint32_t)p.row_bytes;
                lds_dma16_s(base, 16u * (unsigned)(ln ^ nope_sw(r)), tb + r * NOPE_STRIDE);
            }
            const int r = 8 * wave + (ln >> 3);
            lds_dma16(p.kv + (uint64_t)(uint32_t)g.rope * (uint32_t)p.row_bytes + 1024 + 16 * ((ln & 7) ^ rope_sw(r)),
                      tb + ROPE_OFF + 8 * wave * 128);
        } else {
            // load k takes pieces 64 k .. +63; the last one's spare lanes repeat one of its pieces into the
            // slot's padding
            const lds_ptr rb = raw_of(slot) + 1024 * wave;
            if (g.r[0] >= 0) {
                const unsigned char* base = p.kv + (uint64_t)(uint32_t)g.r[0] * FP8_ROW + 1024 * wave;
#pragma unroll
                for (int e = 0; e < RAW_LPW - 1; ++e) lds_dma16_s(base + 1024 * NWAVE * e, 16u * ln, rb + 1024 * NWAVE * e);
                if (wave == 0)
                    lds_dma16_s(base + 1024 * (RAW_LOADS - 1), 16u * (ln & 31), rb + 1024 * (RAW_LOADS - 1));
            } else {
                // piece / 41 is its row in the tile
                const int i = g.r[1];
#pragma unroll 1
                for (int k = wave; k < RAW_LOADS; k += NWAVE) {
                    const unsigned piece = min(64u * k + ln, (unsigned)RAW_PIECES - 1), rt = piece / 41u;
                    const uint32_t row = (uint32_t)rows_l[i * TILE + (int)rt];
                    lds_dma16(p.kv + ((uint64_t)row * (uint32_t)p.row_bytes + 16u * (piece - 41u * rt)),
                              raw_of(slot) + 1024 * k);
                }
            }
        }
    };

    // In a tile that some row of the block does not attend whole, a row of the cache may hold anything,
    // and 0 x NaN is NaN: one with a NaN or infinity among its NoPE values is cleared, and the scores of
    // those that do attend it become NaN.  (bf16: a wave looks at the rows that it loaded.)
    auto scan = [&](int i, int slot) {
        const int ln = opaque(lane);
        uint32_t bad = 0;
        if constexpr (!FP8) {
            const lds_ptr tb = slot_of(slot) + 8 * wave * NOPE_STRIDE + 16 * ln;
#pragma unroll 2
            for (int e = 0; e < 8; ++e) {
                const u32x4 v = lds_ld<u32x4>(tb + e * NOPE_STRIDE);
                bool odd = false;
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (v[w] & 0x7F800000u) == 0x7F800000u || (v[w] & 0x7F80u) == 0x7F80u;
                if (__builtin_amdgcn_ballot_w64(odd)) {
                    lds_st<u32x4>(tb + e * NOPE_STRIDE, u32x4{0, 0, 0, 0});
                    bad |= 1u << e;
                }
            }
        } else {
            // two rows of 32 pieces a read: e4m3 has no infinity, and its NaN has all bits but the sign set
            const lds_ptr tb = raw_of(slot) + (8 * wave + (ln >> 5)) * FP8_ROW + 16 * (ln & 31);
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
                const u32x4 v = lds_ld<u32x4>(tb + 2 * e * FP8_ROW);
                unsigned odd = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= ((v[w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                const uint64_t who = __builtin_amdgcn_ballot_w64(odd != 0);
                const bool lo = (uint32_t)who != 0, up = (who >> 32) != 0;
                if (ln < 32 ? lo : up) lds_st<u32x4>(tb + 2 * e * FP8_ROW, u32x4{0, 0, 0, 0});
                bad |= (lo ? 1u : 0u) << (2 * e) | (up ? 2u : 0u) << (2 * e);
            }
        }
        if (bad && ln == 0) reinterpret_cast<unsigned char*>(s_nan)[4 * i + wave] = (unsigned char)bad;
    };

    // ---- 656-byte rows: V of the raw tile -> fp16.  Piece g = 4 u + m of wave w is rows 16 u .. +15, dims
    // 128 w + 32 m .. +31, the V block that its own PV group (u, m) reads: a buffer is refilled by its readers.
    // v_cvt_scalef32 applies the power of two of the row's scale exactly, the product its mantissa (both in
    // fp16).  The scales go to s_scale for the scores; one outside [0, 128) is NaN there, and its row 0 in V.
    struct Scale {
        float sc;          // 0 where the scale is out of range
        f16x2 m;           // its mantissa, twice
    };
    auto deq_scale = [&](lds_cptr rb, int par, int u) -> Scale {
        const int ln = opaque(lane);
        const int r = 16 * u + (ln >> 2);
        const float s = lds_ld<float>(rb + r * FP8_ROW + 512 + 4 * wave);
        const bool bad = __float_as_uint(s) >= FP8_SCALE_LIMIT_BITS;
        if ((ln & 3) == 0) *(LDS_AS float*)&s_scale[(4 * par + wave) * TILE + r] = bad ? __builtin_nanf("") : s;
        Scale d;
        d.sc = bad ? 0.0f : s;
        const _Float16 m16 = (_Float16)__uint_as_float((__float_as_uint(d.sc) & 0x007FFFFFu) | 0x3F800000u);
        d.m = f16x2{m16, m16};
        return d;
    };
    auto deq_load = [&](lds_cptr rb, int g) -> u32x2 {
        const int ln = opaque(lane);
        return lds_ld<u32x2>(rb + (16 * (g >> 2) + (ln >> 2)) * FP8_ROW + 128 * wave + 32 * (g & 3) + 8 * (ln & 3));
    };
    auto deq_store = [&](lds_ptr vb, int g, u32x2 c, const Scale& d) {
        const int ln = opaque(lane);
        const int r = 16 * (g >> 2) + (ln >> 2), ch = 16 * wave + 4 * (g & 3) + (ln & 3);
        const u32x4 v = {__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[0], d.sc, false) * d.m),
                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[0], d.sc, true) * d.m),
                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[1], d.sc, false) * d.m),
                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[1], d.sc, true) * d.m)};
        lds_st<u32x4>(vb + r * NOPE_STRIDE + 16 * (ch ^ nope_sw(r)), v);
    };
    auto dequant = [&](lds_cptr rb, lds_ptr vb, int par) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const Scale d = deq_scale(rb, par, u);
#pragma unroll
            for (int m = 0; m < 4; ++m) deq_store(vb, 4 * u + m, deq_load(rb, 4 * u + m), d);
        }
    };

    const float c_s = p.scale_log2;
    auto landed = [&](auto keep) {
        wait_vm<decltype(keep)::value>();
        asm volatile("" ::: "memory");
    };
    f32x16 o[16];
    float m_ref = 0.0f, l_lane = 0.0f;
    float p_top = 0.0f;          // 656-byte rows: the largest P (fp16 holds up to 2^16)
    bool first_tile = true, any = false;

    // PV's first operands of a tile (bf16 rows): read in the last steps of the scores before it (1024 tokens of
    // 128 heads over 8192 rows 2000 -> 1978 us; 656-byte rows, whose scores leave no idle reads: 1294 -> 1307)
    struct First {
        u32x4 p[NWAVE], v;
    };
    // V^T block m of the wave's dims, positions 16 u .. +15 (transposed reads of rows 4 hi .. +3 and 8 further)
    auto v_block = [&](lds_cptr vt, int ln, int u, int m) -> u32x4 {
        const int lhi = ln >> 5, g16 = ln >> 4, i16 = ln & 15, rr = i16 >> 2, pp = i16 & 3;
        const int vx = 2 * (g16 & 1) + (pp >> 1);
        const lds_cptr v_a = vt + (4 * lhi + rr) * NOPE_STRIDE + 16 * (vx ^ lhi) + 8 * (pp & 1) + 256 * wave;
        const lds_cptr v_b = vt + (4 * lhi + rr + 8) * NOPE_STRIDE + 16 * (vx ^ (lhi + 2)) + 8 * (pp & 1) + 256 * wave;
        const s16x4 va = lds_read_tr16(v_a + 16 * u * NOPE_STRIDE + 64 * m);
        const s16x4 vb = lds_read_tr16(v_b + 16 * u * NOPE_STRIDE + 64 * m);
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto p_block = [&](lds_cptr px, int ln, int u, int h) -> u32x4 { return lds_ld<u32x4>(px + ((u * NWAVE + h) * 64 + ln) * 16); };
    auto read_first = [&](First& f, int i, lds_cptr vt, lds_cptr px) {
        if (i < NWAVE) f.p[i] = p_block(px, lane, 0, i);
        else f.v = v_block(vt, lane, 0, 0);
    };
    auto none = [](int) {};
    // (last(i), i = 0 .. 4, is called in the last five steps)
    auto qk = [&](lds_cptr kt, auto&& last) -> f32x16 {
        const int ln = lane, lhi = ln >> 5, lr = ln & 31;
        const lds_cptr k_even = kt + lr * NOPE_STRIDE + 16 * (lhi ^ nope_sw(lr));
        const lds_cptr k_odd = kt + lr * NOPE_STRIDE + 16 * ((2 + lhi) ^ nope_sw(lr));
        const lds_cptr k_rope = kt + ROPE_OFF + 128 * lr;
        const int rsw = rope_sw(lr);
        constexpr int AHEAD = 6;
        auto k_at = [&](int ks) -> lds_cptr {
            return ks < KS_NOPE ? ((ks & 1) ? k_odd : k_even) + 64 * (ks >> 1) : k_rope + 16 * ((2 * (ks - KS_NOPE) + lhi) ^ rsw);
        };
        u32x4 kb[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kb[i] = lds_ld<u32x4>(k_at(i));
        f32x16 acc = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            __builtin_amdgcn_sched_barrier(0);
            acc = mfma_bf16(kb[ks % AHEAD], qf[ks], acc);
            if (ks + AHEAD < KS) kb[ks % AHEAD] = lds_ld<u32x4>(k_at(ks + AHEAD));
            if (ks >= KS - 5) last(ks - (KS - 5));
        }
        __builtin_amdgcn_sched_barrier(0);
        return acc;
    };
    // ---- 656-byte rows: S^T from the raw codes, which bf16 holds exactly.  The scale of 128 dims is a
    // position's own, so each group is a chain of its own: S = sum_g scale_g (K_g q_g) + K_rope q_rope.
    // (The fp8 matrix instructions, with Q in two exact e4m3 parts, sum their products with 13 bits against the
    // largest, scores off by 2^-15, and were no faster: two prompts of 1700 to 2048 tokens 1.40 ms, this 1.38.) ----
    auto qk8 = [&](lds_cptr raw, int par) -> f32x16 {
        const int ln = opaque(lane), lhi = ln >> 5, lr = ln & 31;
        const lds_cptr kn = raw + lr * FP8_ROW + 16 * lhi;
        const lds_cptr kr = kn + 528;
        const lds_cptr sc = (lds_cptr)(LDS_AS float*)&s_scale[4 * par * TILE] + 16 * lhi;
        constexpr int AHEAD = 3;               // reads of 16 codes, each two k-steps
        u32x4 kb[AHEAD];
        auto k_frag = [&](int j) { return lds_ld<u32x4>(j < KS_NOPE / 2 ? kn + 32 * j : kr + 32 * (j - KS_NOPE / 2)); };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kb[i] = k_frag(i);
        f32x16 s = {};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x16 a = {};
            f32x4 f[4];
#pragma unroll
            for (int j = 4 * g; j < 4 * g + 4; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                const u32x4 c = kb[j % AHEAD];
                a = mfma_bf16(codes_bf16(c[0], c[1]), qf[2 * j], a);
                a = mfma_bf16(codes_bf16(c[2], c[3]), qf[2 * j + 1], a);
                kb[j % AHEAD] = k_frag(j + AHEAD);
                if (j == 4 * g + 1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[i] = lds_ld<f32x4>(sc + 4 * TILE * g + 32 * i);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(a[r], f[r >> 2][r & 3], s[r]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            s = mfma_bf16(kb[(KS_NOPE / 2 + j) % AHEAD], qf[KS_NOPE + j], s);
            if (j + AHEAD < 4) kb[(KS_NOPE / 2 + j) % AHEAD] = k_frag(KS_NOPE / 2 + j + AHEAD);
        }
        __builtin_amdgcn_sched_barrier(0);
        return s;
    };
    auto masked = [&](int i, int c0) { return c0 + (i + 1) * TILE > lim_lo || __builtin_amdgcn_readfirstlane(s_skip[i]) != 0; };
    // lane (hi, r32), register r: position 8 (r / 4) + 4 hi + r % 4 of the tile, row r32 of the wave
    auto mask = [&](f32x16& s, int i, int c0) {
        const uint32_t skip = s_skip[i];
        const int pos0 = c0 + i * TILE;
        if (masked(i, c0)) {
            asm volatile("");
            const uint32_t nan = s_nan[i];
            const int left = limit - pos0, h4 = 4 * opaque(hi);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int j = 8 * (r >> 2) + h4 + (r & 3);
                const bool on = j < left && !((skip >> j) & 1);
                any = any || on;
                const float v = (nan >> j) & 1 ? __builtin_nanf("") : s[r];
                s[r] = on ? v : -INFINITY;
            }
        } else {
            any = true;
        }
    };
    auto top_of = [&](const f32x16& s) -> float {
        float m = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
        return fmaxf(m, __shfl_xor(m, 32, 64));
    };
    auto p_half = [&](const float* e, int u, lds_ptr px) {
        const int ln = opaque(lane);
        float lt = 0.0f;
#pragma unroll
        for (int r = 8 * u; r < 8 * u + 8; ++r) lt += e[r];
        l_lane += lt;
        if constexpr (FP8) {
            u32x4 h;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const f16x2 v = {(_Float16)e[8 * u + 2 * w], (_Float16)e[8 * u + 2 * w + 1]};
                h[w] = __builtin_bit_cast(unsigned, v);
                p_top = fmaxf(p_top, fmaxf(e[8 * u + 2 * w], e[8 * u + 2 * w + 1]));
            }
            lds_st<u32x4>(px + ((u * NWAVE + wave) * 64 + ln) * 16, h);
            return;
        }
        const f32x8 a = {e[8 * u], e[8 * u + 1], e[8 * u + 2], e[8 * u + 3], e[8 * u + 4], e[8 * u + 5], e[8 * u + 6], e[8 * u + 7]};
        lds_st<u32x4>(px + ((u * NWAVE + wave) * 64 + ln) * 16, __builtin_bit_cast(u32x4, __builtin_convertvector(a, bf16x8)));
    };
    auto p_first = [&](f32x16& s, lds_ptr px) {
        if (first_tile) {
            // no position of the first tile attended: any reference, checked at the end
            const float top = top_of(s) * c_s;
            m_ref = top == -INFINITY ? 0.0f : top;
            m_ref -= (float)lift_of<FP8>(k1 - k0, false);
            first_tile = false;
        }
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c_s, -m_ref));
        p_half(e, 0, px);
        p_half(e, 1, px);
    };
    // (656-byte rows, with_exp: the next tile but one, raw at draw, goes to V's own buffer, piece by piece)
    auto pv = [&](lds_ptr vt, lds_cptr px, First& f, const f32x16& sn, float* en, auto with_exp, lds_cptr draw, int dpar) {
        const int ln = FP8 ? opaque(lane) : lane;
        u32x4 v_cur = {};
        if constexpr (!FP8) v_cur = f.v;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if constexpr (FP8) {
#pragma unroll
                for (int h = 0; h < NWAVE; ++h) f.p[h] = p_block(px, ln, u, h);
                v_cur = v_block(vt, ln, u, 0);
            }
            Scale ds;
            if constexpr (FP8 && decltype(with_exp)::value) ds = deq_scale(draw, dpar, u);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                __builtin_amdgcn_sched_barrier(0);
                u32x4 v_nxt = v_cur;
                if (m + 1 < 4) v_nxt = v_block(vt, ln, u, m + 1);
                else if (!FP8 && u == 0) v_nxt = v_block(vt, ln, 1, 0);
                u32x2 codes;
                if constexpr (FP8 && decltype(with_exp)::value) codes = deq_load(draw, 4 * u + m);
#pragma unroll
                for (int h = 0; h < NWAVE; ++h) {
                    mfma_o<FP8>(o[4 * m + h], v_cur, f.p[h]);
                    if (!FP8 && u == 0 && m == 3) f.p[h] = p_block(px, ln, 1, h);
                }
                if constexpr (decltype(with_exp)::value) {
                    const int r0 = 8 * u + 2 * m;
                    en[r0] = __builtin_amdgcn_exp2f(__builtin_fmaf(sn[r0], c_s, -m_ref));
                    en[r0 + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sn[r0 + 1], c_s, -m_ref));
                }
                if constexpr (FP8 && decltype(with_exp)::value) deq_store(vt, 4 * u + m, codes, ds);
                v_cur = v_nxt;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    const int nspans = k1 > k0 ? (k1 - k0 + SPAN - 1) / SPAN : 0;
    // Pass 0; where its reference did not serve one of the rows: the largest score of every row, and the pass
    // again with that as the reference.  A row of 656-byte rows needs it whose later scores pass its first tile's by
    // 11 (16 powers of two), one of bf16 rows by 28 less the logarithm of how many do; its whole block then takes
    // 2.7 times as long (1024 tokens of 128 heads over 8192 rows, all blocks: bf16 1.96 -> 5.33 ms, 656-byte rows
    // 2.75 -> 7.84; the 32-row kernel on 32 tokens of 16 heads 41 -> 83 us and 41 -> 76).
    bool again = false;
    while (true) {
        // (0 x 0 + 0: cleared where they are, without the registers that zeros to copy would take)
        const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < 16; ++m)
            asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(o[m]) : "v"(zero));
        o_fence(o);
        l_lane = 0.0f;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = k0 + c * SPAN;
            resolve(c0);
            if (ntiles == 0) continue;
            if constexpr (!FP8) {
            issue(load_rows(0), 0);
            if (ntiles > 1) issue(load_rows(1), 1);
            Rows next = load_rows(min(2, ntiles - 1));
            if (ntiles > 1) landed(std::integral_constant<int, LPW>{}); else landed(std::integral_constant<int, 0>{});
            if (masked(0, c0)) scan(0, 0);
            tile_barrier();
            f32x16 s0 = qk(slot_of(0), none);
            mask(s0, 0, c0);
            p_first(s0, PX);
            int cur = 0;
            for (int i = 0; i + 1 < ntiles; ++i) {
                const int nxt = cur == 2 ? 0 : cur + 1;
                // tile i + 1, the only one in flight, has landed; the barrier shows every wave's P of
                // tile i, and every wave is done with tile i - 1, whose buffer takes tile i + 2
                landed(std::integral_constant<int, 0>{});
                if (masked(i + 1, c0)) scan(i + 1, nxt);
                tile_barrier();
                __builtin_amdgcn_sched_barrier(0);
                if (i + 2 < ntiles) issue(next, nxt == 2 ? 0 : nxt + 1);
                __builtin_amdgcn_sched_barrier(0);
                First f;
                f32x16 sn = qk(slot_of(nxt), [&](int k) { read_first(f, k, slot_of(cur), PX + (i & 1) * P_BYTES); });
                if (i + 3 < ntiles) next = load_rows(i + 3);
                mask(sn, i + 1, c0);
                float en[16];
                pv(slot_of(cur), PX + (i & 1) * P_BYTES, f, sn, en, std::true_type{}, T0, 0);
                const lds_ptr px = PX + ((i + 1) & 1) * P_BYTES;
                p_half(en, 0, px);
                p_half(en, 1, px);
                cur = nxt;
            }
            tile_barrier();
            float en[16];
            First f;
#pragma unroll
            for (int k = 0; k < 5; ++k) read_first(f, k, slot_of(cur), PX + ((ntiles - 1) & 1) * P_BYTES);
            pv(slot_of(cur), PX + ((ntiles - 1) & 1) * P_BYTES, f, f32x16{}, en, std::false_type{}, T0, 0);
            } else {
                // Iteration j: scores of tile j from raw slot j % 3; PV of tile j - 1 from V buffer (j - 1) % 2,
                // with the exponentials of tile j and the conversion of tile j + 1 into that buffer.
                auto ready = [&](int i) {          // tile i lies whole in its slot
                    landed(std::integral_constant<int, 0>{});
                    tile_barrier();
                    if (i < ntiles && masked(i, c0)) {
                        scan(i, i % 3);
                        tile_barrier();
                    }
                };
                issue(load_rows(0), 0);
                ready(0);
                if (ntiles > 1) issue(load_rows(1), 1);
                dequant(raw_of(0), slot_of(0), 0);
                Rows next = load_rows(min(2, ntiles - 1));
                ready(1);
                if (ntiles > 2) issue(next, 2);
                f32x16 s0 = qk8(raw_of(0), 0);
                next = load_rows(min(3, ntiles - 1));
                mask(s0, 0, c0);
                p_first(s0, PX);
                if (ntiles > 1) dequant(raw_of(1), slot_of(1), 1);
                for (int j = 1; j < ntiles; ++j) {
                    // (the barrier also shows tile j's V and scales and tile j - 1's P, and every wave is
                    // done with tile j - 1's raw slot, which takes tile j + 2)
                    ready(j + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    if (j + 2 < ntiles) issue(next, (j + 2) % 3);
                    __builtin_amdgcn_sched_barrier(0);
                    f32x16 sn = qk8(raw_of(j % 3), j & 1);
                    if (j + 3 < ntiles) next = load_rows(j + 3);
                    mask(sn, j, c0);
                    float en[16];
                    First f;
                    pv(slot_of((j - 1) & 1), PX + ((j - 1) & 1) * P_BYTES, f, sn, en, std::true_type{}, raw_of((j + 1) % 3),
                       (j + 1) & 1);
                    const lds_ptr px = PX + (j & 1) * P_BYTES;
                    p_half(en, 0, px);
                    p_half(en, 1, px);
                }
                tile_barrier();
                float en[16];
                First f;
                pv(slot_of((ntiles - 1) & 1), PX + ((ntiles - 1) & 1) * P_BYTES, f, f32x16{}, en, std::false_type{}, T0, 0);
            }
        }
        o_fence(o);
        if (again) break;
        // The reference served if the sum (bf16 P, which has the range of fp32) or the largest P (fp16) lies where
        // its type holds it, and if O, which is at most the sum times the largest value, did not pass fp32.  The sum
        // is at least the first tile's maximum, 2^lift; it grows past 2^40 times that only where later scores do.
        const float l = l_lane + __shfl_xor(l_lane, 32, 64);
        const bool have = either(any);
        const float top_p = FP8 ? fmaxf(p_top, __shfl_xor(p_top, 32, 64)) : 0.0f;
        __syncthreads();
        if (wave == 0) s_misc[1] = 0, s_misc[2] = 0, s_misc[3] = 0;
        __syncthreads();
        const int lift = lift_of<FP8>(k1 - k0, false);
        const bool held = FP8 ? top_p >= __builtin_ldexpf(0.5f, lift) && top_p <= FP16_MAX
                              : l > __builtin_ldexpf(1.0f, lift - 40) && l < __builtin_ldexpf(1.0f, lift + 40);
        if (have && !held) s_misc[1] = 1;
        if (!FP8 && have && l >= 0.5f) s_misc[2] = 1;
        __syncthreads();
        bool served = __builtin_amdgcn_readfirstlane(s_misc[1]) == 0;
        if (!FP8 && __builtin_expect(served && __builtin_amdgcn_readfirstlane(s_misc[2]) != 0, false)) {
            // (0 times what is not finite is NaN; tile after tile, without copies of all of O)
            float t = 0.0f;
#pragma unroll
            for (int m = 0; m < 16; ++m) {
                asm volatile("" : "+a"(o[m]), "+v"(t));
#pragma unroll
                for (int r = 0; r < 16; ++r) t = __builtin_fmaf(o[m][r], 0.0f, t);
            }
            asm volatile("" : "+v"(t));
            if (t != 0.0f) s_misc[3] = 1;
            __syncthreads();
            served = __builtin_amdgcn_readfirstlane(s_misc[3]) == 0;
        }
        if (served) break;
        again = true;
        float top = -INFINITY;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = k0 + c * SPAN;
            resolve(c0);
            for (int i = 0; i < ntiles; ++i) {
                issue(load_rows(i), 0);
                landed(std::integral_constant<int, 0>{});
                f32x16 s;
                if constexpr (FP8) {
                    tile_barrier();
                    if (masked(i, c0)) scan(i, 0);
                    dequant(raw_of(0), slot_of(0), 0);
                    tile_barrier();
                    s = qk8(raw_of(0), 0);
                } else {
                    if (masked(i, c0)) scan(i, 0);
                    tile_barrier();
                    s = qk(slot_of(0), none);
                }
                mask(s, i, c0);
                top = fmaxf(top, top_of(s));
                tile_barrier();
            }
        }
        m_ref = top == -INFINITY ? 0.0f : top * c_s;
        m_ref -= (float)lift_of<FP8>(k1 - k0, true);
    }

    // ---- O / l, LSE ----
    // (lane and wave numbers anew: none of what follows is kept through the tile loop)
    const int ln = fresh_lane(), hi_ = ln >> 5, r_ = ln & 31;
    int wv = wave;
    asm volatile("" : "+s"(wv));
    const Args a_ = args();
    const int ns = a_->ns, H = a_->H;
    const int64_t TH = (int64_t)a_->T * H;
    const float l = l_lane + __shfl_xor(l_lane, 32, 64);
    const bool have = either(any);
    const bool mine = 32 * wv + r_ < blk.rows;
    const int lift = lift_of<FP8>(k1 - k0, again);
    const float lse = too_long ? __builtin_nanf("")
                               : (m_ref + (float)lift + __builtin_amdgcn_logf(__builtin_ldexpf(l, -lift))) * LN2;
    if (hi_ == 0) {
        s_inv[32 * wv + r_] = too_long ? __builtin_nanf("") : (have ? 1.0f / l : 0.0f);
        const int64_t at = (int64_t)blk.first * H + blk.r0 + 32 * wv + r_;      // rows are token-major
        if (mine && ns > 1) a_->part_lse[split * TH + at] = have ? lse : -FLT_MAX;
        else if (mine && a_->lse) a_->lse[at] = have || too_long ? lse : INFINITY;
    }
    __syncthreads();
    float inv[NWAVE];
#pragma unroll
    for (int h = 0; h < NWAVE; ++h) inv[h] = s_inv[32 * h + r_];
    const int d0 = 128 * wv + 4 * hi_;
    if (ns == 1) {
        const int64_t o_st = a_->o_st, o_sh = a_->o_sh;
        __bf16* const out = a_->out;
        // 32 rows at a time through LDS, so that a wave's store is one whole 1 KB row
        constexpr int OUT_STRIDE = D_VO * 2 + 16;
        static_assert(32 * OUT_STRIDE <= TILE_BYTES, "the stage fits a tile buffer");
        const int st_w = opaque(r_ * OUT_STRIDE + 2 * d0);
        const bool o16 = ((o_st | o_sh) & 7) == 0 && ((uintptr_t)out & 15) == 0;
#pragma unroll
        for (int h = 0; h < NWAVE; ++h) {
            const lds_ptr stg = slot_of(h & 1);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16& a = o[4 * m + h];
                    const f32x4 v = {a[4 * g] * inv[h], a[4 * g + 1] * inv[h], a[4 * g + 2] * inv[h], a[4 * g + 3] * inv[h]};
                    lds_st<u32x2>(stg + st_w + 2 * (32 * m + 8 * g), __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4)));
                }
            }
            __syncthreads();
            // the wave's eight rows, read together
            u32x4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = lds_ld<u32x4>(stg + (8 * wv + k) * OUT_STRIDE + 16 * ln);
            const int r0 = 32 * h + 8 * wv;
            int t = (blk.r0 + r0) / H, hh = (blk.r0 + r0) - t * H;
            t += blk.first;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (r0 + k >= blk.rows) break;
                __bf16* const dst = out + t * o_st + hh * o_sh + 8 * ln;
                if (o16) {
                    *reinterpret_cast<u32x4*>(dst) = v[k];
                } else {
                    reinterpret_cast<u32x2*>(dst)[0] = u32x2{v[k][0], v[k][1]};
                    reinterpret_cast<u32x2*>(dst)[1] = u32x2{v[k][2], v[k][3]};
                }
                if (++hh == H) hh = 0, ++t;
            }
        }
    } else {
        // fp32 partials: the wave's 128 dims of two rows a store
        constexpr int PST = D_VO + 16;
        static_assert(4 * 32 * PST <= 3 * TILE_BYTES, "four waves' stages fit the tile buffers");
        const lds_ptr stg = T0 + wv * 32 * PST;
        const int st_w = opaque(r_ * PST + 16 * hi_);
        float* const dst0 = a_->part_o + (split * TH + (int64_t)blk.first * H + blk.r0) * D_VO;
#pragma unroll
        for (int h = 0; h < NWAVE; ++h) {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16& a = o[4 * m + h];
                    const f32x4 v = {a[4 * g] * inv[h], a[4 * g + 1] * inv[h], a[4 * g + 2] * inv[h], a[4 * g + 3] * inv[h]};
                    lds_st<f32x4>(stg + st_w + 4 * (32 * m + 8 * g), v);
                }
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int r = 2 * k + (ln >> 5);
                const f32x4 v = lds_ld<f32x4>(stg + r * PST + 16 * (ln & 31));
                if (32 * h + r < blk.rows)
                    *reinterpret_cast<f32x4*>(dst0 + (int64_t)(32 * h + r) * D_VO + 128 * wv + 4 * (ln & 31)) = v;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The narrow kernel: 32 rows a workgroup, two workgroups a CU, for single tokens and
// few heads, where the cache rows' way through memory counts and not the products.
//   QK^T   wave w: 16 positions (half w % 2 of the tile) x 16 rows (half w / 2), 16x16x32
//   P      as in the tiled kernel, one buffer: P of a tile is read before the next's is written
//   PV     wave w: O^T[dims 128 w .. +127 x 32 rows] in 64 registers
// Two barriers a tile; one workgroup's waits are the other's time.
// Measured (16 sequences of 7130 to 19272 bf16 rows, 1 to 4 tokens of 16 heads): 59 us, 290 MB read at
// 4.9 TB/s, 96 % of a large copy's rate.  One token of 128 heads over 1483 656-byte rows: 14.4 us in
// 64 workgroups of 3 tiles, a chain of memory round trips (1.5 us to the split, then pages, rows, partials).
// ---------------------------------------------------------------------------
// A tile in LDS: NoPE rows of 1 KB, piece c of row r at c ^ nsw(r): the K reads (one piece of 16 rows) find 16
// values of nsw, the transposed V reads (four pieces of four rows) pieces that part at bit 2.  Conflicts take
// 270 of a tile's 790 LDS cycles (1040-byte rows and c ^ 4 (r % 4): 400 of 880, and 233 us where this is 202:
// 256 single tokens of 16 heads over 4096 656-byte rows).
constexpr int NSTRIDE = 1024;
__device__ __forceinline__ int nsw(int r) { return 4 * (r & 3) + ((r >> 2) & 3); }
constexpr int NROPE_OFF = TILE * NSTRIDE;
constexpr int NTILE = NROPE_OFF + TILE * 128;
constexpr int NLIST = 512;                   // entries of the row list
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return mfma_bf16(a, b, c);
}

// RUNS: a tile lies in one page (or in a flat cache), so that its rows follow its first one's
template <int FMT, bool RUNS>
__global__ void __launch_bounds__(NTHR) __attribute__((amdgpu_waves_per_eu(2, 2)))
dsa_mla_chunk_narrow_kernel(const ChunkParams p) {
    constexpr bool FP8 = FMT == DSA_KV_FP8_656;
    constexpr int VT = TILE * NSTRIDE;                               // 656-byte rows: one V tile, two raw slots
    constexpr int BYTES = FP8 ? VT + 2 * RAW_BYTES : 2 * NTILE;
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[BYTES];
    __shared__ __attribute__((aligned(16))) unsigned char s_p[2 * 2 * 32 * 16];     // [u][hi][row] x 8 positions
    __shared__ int32_t s_rows[NLIST];        // RUNS: the first row of every tile; else every position's
    __shared__ float s_top[2][NARROW];
    __shared__ uint32_t s_nan;               // bit j: position j's row holds a NaN or infinity
    __shared__ int32_t s_misc[4];            // [0] a row that may be read, [1] again, [2] a scale out of range
                                             // (bf16: O may have passed fp32), [3] it has
    const lds_ptr T0 = (lds_ptr)s_tile, PX = (lds_ptr)s_p;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work work = find_work(p, NARROW, 2 * CUS);
    const Block& blk = work.blk;
    const int split = work.split, per = work.per;
    if (blk.rows == 0) return;
    const int lim_lo = limit_in(p, blk, blk.first + blk.r0 / p.H);
    const int lim_hi = limit_in(p, blk, blk.first + (blk.r0 + blk.rows - 1) / p.H);
    const bool too_long = blk.len > p.max_len;
    const int k0 = (int)min((int64_t)split * per, (int64_t)lim_hi);
    const int k1 = too_long ? k0 : (int)min(min((int64_t)lim_hi, p.pages.limit), (int64_t)k0 + per);
    if (p.ns > 1 && k1 <= k0) return;

    // scores: this lane's row of the 16 of its wave, and its positions 16 half + 4 q .. +3 of a tile
    const int half = wave & 1, q = lane >> 4;
    const int my = 16 * (wave >> 1) + (lane & 15);
    const int row = blk.r0 + min(my, blk.rows - 1);
    const int tok = blk.first + row / p.H;
    const int limit = limit_in(p, blk, tok);
    u32x4 qf[KS / 2];
    {
        const __bf16* qp = p.q + (int64_t)tok * p.q_st + (int64_t)(row % p.H) * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS / 2; ++ks) {
            // (656-byte rows: 16 codes a read, the two k-steps of 64 dims share them)
            const int d = FP8 && ks < 16 ? 64 * (ks >> 1) + 16 * q + 8 * (ks & 1) : 32 * ks + 8 * q;
            qf[ks] = *reinterpret_cast<const u32x4*>(qp + d);
        }
    }

    // ---- positions [c0, c0 + span) below k1 -> the row list; -1: no row ----
    constexpr int STEP = RUNS ? TILE : 1;
    constexpr int span = NLIST * STEP;
    int ntiles = 0;
    int32_t safe = -1;                       // a row that is there
    auto resolve = [&](int c0) {
        __syncthreads();
        const int count = (min(k1 - c0, span) + STEP - 1) / STEP;
        int32_t some = -1;
        for (int e = threadIdx.x; e < NLIST; e += NTHR) {
            int64_t r = -1;
            if (e < count) r = dsa_seq::row_of(p.pages, blk.b, c0 + e * STEP, p.rows);
            s_rows[e] = (int32_t)r;
            some = max(some, (int32_t)r);
        }
        if (threadIdx.x == 0) s_misc[0] = -1;
        __syncthreads();
        if (some >= 0) s_misc[0] = some;
        __syncthreads();
        safe = __builtin_amdgcn_readfirstlane(s_misc[0]);
        ntiles = safe < 0 ? 0 : (min(k1 - c0, span) + TILE - 1) / TILE;
    };
    // RUNS: a tile's first row, read ahead of its use
    auto base_of = [&](int i) -> int32_t { return RUNS && i < NLIST ? s_rows[i] : 0; };
    // a tile's positions that have a row (bit j clear: none, or past k1)
    auto has_of = [&](int32_t base, int i, int c0) -> uint32_t {
        const int left = k1 - (c0 + i * TILE);
        if constexpr (RUNS) {
            const int64_t n = base < 0 ? 0 : min((int64_t)left, p.rows - base);
            return n >= TILE ? ~0u : (1u << n) - 1u;
        } else {
            const int j = lane & 31;
            return (uint32_t)__builtin_amdgcn_ballot_w64(j < left && s_rows[i * TILE + j] >= 0);
        }
    };
    // cache row of position j of tile i (some row that is there, for one without)
    auto row_at = [&](int32_t base, uint32_t has, int i, int j) -> uint32_t {
        const bool ok = (has >> j) & 1;
        return (uint32_t)(ok ? (RUNS ? base + j : s_rows[i * TILE + j]) : safe);
    };

    auto slot_of = [&](int s) -> lds_ptr { return FP8 ? T0 + VT + s * RAW_BYTES : T0 + s * NTILE; };
    auto issue = [&](int32_t base, uint32_t has, int i, int slot) {
        const int ln = opaque(lane);
        const lds_ptr tb = slot_of(slot);
        if constexpr (!FP8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 8 * wave + e;
                const uint32_t at = __builtin_amdgcn_readfirstlane(row_at(base, has, i, r));
                lds_dma16_s(p.kv + (uint64_t)at * (uint32_t)p.row_bytes, 16u * (unsigned)(ln ^ nsw(r)), tb + r * NSTRIDE);
            }
            const int r = 8 * wave + (ln >> 3);
            lds_dma16(p.kv + (uint64_t)row_at(base, has, i, r) * (uint32_t)p.row_bytes + 1024 + 16 * ((ln & 7) ^ rope_sw(r)),
                      tb + NROPE_OFF + 8 * wave * 128);
        } else if (RUNS && has == ~0u && p.row_bytes == FP8_ROW) {
            const unsigned char* from = p.kv + (uint64_t)(uint32_t)base * FP8_ROW + 1024 * wave;
#pragma unroll
            for (int e = 0; e < RAW_LPW - 1; ++e) lds_dma16_s(from + 1024 * NWAVE * e, 16u * ln, tb + 1024 * wave + 1024 * NWAVE * e);
            if (wave == 0) lds_dma16_s(from + 1024 * (RAW_LOADS - 1), 16u * (ln & 31), tb + 1024 * (RAW_LOADS - 1));
        } else {
#pragma unroll 1
            for (int k = wave; k < RAW_LOADS; k += NWAVE) {
                const unsigned piece = min(64u * k + ln, (unsigned)RAW_PIECES - 1), rt = piece / 41u;
                lds_dma16(p.kv + ((uint64_t)row_at(base, has, i, (int)rt) * (uint32_t)p.row_bytes + 16u * (piece - 41u * rt)), tb + 1024 * k);
            }
        }
    };
    // this wave's loads have landed, but for those of the newest tile where `one_more` is in flight
    // (656-byte rows: RAW_LPW of wave 0, one fewer of the others)
    auto landed = [&](bool one_more) {
        if (FP8 && one_more) {
            if (wave == 0) wait_vm<RAW_LPW>();
            else wait_vm<RAW_LPW - 1>();
        } else {
            wait_vm<0>();
        }
        asm volatile("" ::: "memory");
    };
    // (as in the tiled kernel: rows that some row of the block does not attend must not reach it; of 656-byte
    // rows one with a scale out of range too)
    auto scan = [&](int slot) {
        const int ln = opaque(lane);
        uint32_t bad = 0;
        if constexpr (!FP8) {
            const lds_ptr tb = slot_of(slot) + 8 * wave * NSTRIDE + 16 * ln;
#pragma unroll 2
            for (int e = 0; e < 8; ++e) {
                const u32x4 v = lds_ld<u32x4>(tb + e * NSTRIDE);
                bool odd = false;
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (v[w] & 0x7F800000u) == 0x7F800000u || (v[w] & 0x7F80u) == 0x7F80u;
                if (__builtin_amdgcn_ballot_w64(odd)) {
                    lds_st<u32x4>(tb + e * NSTRIDE, u32x4{0, 0, 0, 0});
                    bad |= 1u << e;
                }
            }
        } else {
            const lds_ptr tb = slot_of(slot) + (8 * wave + (ln >> 5)) * FP8_ROW + 16 * (ln & 31);
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
                const u32x4 v = lds_ld<u32x4>(tb + 2 * e * FP8_ROW);
                unsigned odd = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= ((v[w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                // (its scales, each by one lane)
                const lds_ptr sp = slot_of(slot) + (8 * wave + 2 * e + (ln >> 5)) * FP8_ROW + 512 + 4 * (ln & 3);
                if (lds_ld<unsigned>(sp) >= FP8_SCALE_LIMIT_BITS) odd = 1;
                const uint64_t who = __builtin_amdgcn_ballot_w64(odd != 0);
                const bool lo = (uint32_t)who != 0, up = (who >> 32) != 0;
                if (ln < 32 ? lo : up) {
                    lds_st<u32x4>(tb + 2 * e * FP8_ROW, u32x4{0, 0, 0, 0});
                    lds_st<unsigned>(sp, 0u);
                }
                bad |= (lo ? 1u : 0u) << (2 * e) | (up ? 2u : 0u) << (2 * e);
            }
        }
        if (ln == 0) reinterpret_cast<unsigned char*>(&s_nan)[wave] = (unsigned char)bad;
    };

    const float c_s = p.scale_log2;
    f32x16 o[4];
    float m_ref = 0.0f, l_lane = 0.0f, p_top = 0.0f;
    bool any = false;
    // 656-byte rows: a scale outside [0, 128) in a tile that every row of the block attends whole (in others
    // scan() has seen to it): all of them are NaN
    bool range_bad = false;

    // S^T[4 positions of this lane x its row]
    auto qk = [&](lds_cptr kt) -> f32x4 {
        const int ln = opaque(lane), lq = ln >> 4, lr = 16 * half + (ln & 15);
        if constexpr (!FP8) {
            const lds_cptr kn = kt + lr * NSTRIDE, kr = kt + NROPE_OFF + 128 * lr;
            const int sw = nsw(lr);
            auto k_at = [&](int ks) -> lds_cptr {
                return ks < 16 ? kn + 256 * (ks >> 2) + 16 * ((4 * (ks & 3) + lq) ^ sw) : kr + 16 * ((4 * (ks - 16) + lq) ^ rope_sw(lr));
            };
            constexpr int AHEAD = 6;
            u32x4 kb[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) kb[i] = lds_ld<u32x4>(k_at(i));
            f32x4 a = {}, b = {};
#pragma unroll
            for (int ks = 0; ks < KS / 2; ++ks) {
                __builtin_amdgcn_sched_barrier(0);
                if (ks & 1) b = mfma16(kb[ks % AHEAD], qf[ks], b);
                else a = mfma16(kb[ks % AHEAD], qf[ks], a);
                if (ks + AHEAD < KS / 2) kb[ks % AHEAD] = lds_ld<u32x4>(k_at(ks + AHEAD));
            }
            return a + b;
        } else {
            // With the scores, between their matrix instructions, V of the tile goes to T0 as fp16: each wave
            // converts the dims that it reads, piece (u, m) = rows 16 u .. +15, dims 128 wave + 32 m .. +31 (as
            // the tiled kernel does)
            const int vr = ln >> 2;
            u32x2 codes[8];
            float vs[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const lds_cptr r = kt + (16 * u + vr) * FP8_ROW;
                vs[u] = lds_ld<float>(r + 512 + 4 * wave);
#pragma unroll
                for (int m = 0; m < 4; ++m) codes[4 * u + m] = lds_ld<u32x2>(r + 128 * wave + 32 * m + 8 * (ln & 3));
            }
            const lds_cptr kn = kt + lr * FP8_ROW + 16 * lq;
            auto k_at = [&](int j) -> lds_cptr { return j < 8 ? kn + 64 * j : kn + 528 + 64 * (j - 8); };
            constexpr int AHEAD = 4;
            u32x4 kb[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) kb[j] = lds_ld<u32x4>(k_at(j));
            // a position's four scales
            f32x4 sc[4];
            f32x4 s = {}, g[4];
            f16x2 mm;
            float vsc;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                if ((j & 1) == 0) g[j >> 1] = f32x4{};
                const u32x4 k = kb[j % AHEAD];
                g[j >> 1] = mfma16(codes_bf16(k[0], k[1]), qf[2 * j], g[j >> 1]);
                g[j >> 1] = mfma16(codes_bf16(k[2], k[3]), qf[2 * j + 1], g[j >> 1]);
                if (j + AHEAD < 10) kb[j % AHEAD] = lds_ld<u32x4>(k_at(j + AHEAD));
                if (j == 5) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[r] = lds_ld<f32x4>(kt + (16 * half + 4 * lq + r) * FP8_ROW + 512);
                }
                if ((j & 3) == 0) {
                    vsc = vs[j >> 2];
                    range_bad |= __float_as_uint(vsc) >= FP8_SCALE_LIMIT_BITS;
                    const _Float16 m16 = (_Float16)__uint_as_float((__float_as_uint(vsc) & 0x007FFFFFu) | 0x3F800000u);
                    mm = f16x2{m16, m16};
                }
                const u32x2 c = codes[j];
                const u32x4 v = {__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[0], vsc, false) * mm),
                                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[0], vsc, true) * mm),
                                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[1], vsc, false) * mm),
                                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[1], vsc, true) * mm)};
                const int r = 16 * (j >> 2) + vr;
                lds_st<u32x4>(T0 + r * NSTRIDE + 256 * wave + 16 * ((4 * (j & 3) + (ln & 3)) ^ nsw(vr)), v);
            }
            s = mfma16(kb[8 % AHEAD], qf[16], s);
            s = mfma16(kb[9 % AHEAD], qf[17], s);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(g[i][r], sc[r][i], s[r]);
            return s;
        }
    };
    auto masked = [&](uint32_t has, int i, int c0) { return c0 + (i + 1) * TILE > lim_lo || has != ~0u; };
    auto mask = [&](f32x4& s, uint32_t has, int i, int c0) {
        if (masked(has, i, c0)) {
            const uint32_t nan = s_nan;
            const int left = limit - (c0 + i * TILE);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * half + 4 * q + r;
                const bool on = j < left && ((has >> j) & 1);
                any = any || on;
                const float v = (nan >> j) & 1 ? __builtin_nanf("") : s[r];
                s[r] = on ? v : -INFINITY;
            }
        } else {
            any = true;
        }
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
    auto p_out = [&](const f32x4& s) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c_s, -m_ref));
        l_lane += (e[0] + e[1]) + (e[2] + e[3]);
        u32x2 w;
        if constexpr (FP8) {
            p_top = fmaxf(p_top, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
            const f16x2 a = {(_Float16)e[0], (_Float16)e[1]}, b = {(_Float16)e[2], (_Float16)e[3]};
            w = u32x2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
        } else {
            const f32x4 v = {e[0], e[1], e[2], e[3]};
            w = __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
        }
        // (the order of a lane's eight positions in the product: 4 hi .. +3, then 8 + 4 hi .. +3)
        lds_st<u32x2>(PX + ((2 * half + (q & 1)) * 32 + my) * 16 + 8 * (q >> 1), w);
    };
    auto pv = [&](lds_cptr vt) {
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
        pb[0] = lds_ld<u32x4>(PX + (lhi * 32 + (ln & 31)) * 16);
#pragma unroll
        for (int i = 0; i < 3; ++i) v[i] = v_frag(i);
        pb[1] = lds_ld<u32x4>(PX + ((2 + lhi) * 32 + (ln & 31)) * 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            o[i & 3] = mfma32<FP8>(v[i % 3], pb[i >> 2], o[i & 3]);
            if (i + 3 < 8) v[i % 3] = v_frag(i + 3);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    const int nspans = k1 > k0 ? (int)(((int64_t)k1 - k0 + span - 1) / span) : 0;
    auto start_of = [&](int c) { return (int)(k0 + (int64_t)c * span); };
    bool first = true, all_nan = false;
    bool again = false;
    while (true) {
#pragma unroll
        for (int m = 0; m < 4; ++m) o[m] = f32x16{};
        l_lane = 0.0f;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            resolve(c0);
            if (ntiles == 0) continue;
            auto at = [&](int i) { return __builtin_amdgcn_readfirstlane(base_of(i)); };
            int32_t b0 = at(0), b1 = at(1);
            uint32_t has = has_of(b0, 0, c0), has1 = ntiles > 1 ? has_of(b1, 1, c0) : 0;
            issue(b0, has, 0, 0);
            if (FP8 && ntiles > 1) issue(b1, has1, 1, 1);
            // Q is waited for here, with the first tiles' loads in flight: left to its first use, the compiler's
            // wait would stand in the loop and drain every tile's loads
#pragma unroll
            for (int ks = 0; ks < KS / 2; ++ks) asm volatile("" : "+v"(qf[ks]));
            for (int i = 0; i < ntiles; ++i) {
                const int slot = i & 1;
                // tile i, the older of those in flight, has landed
                landed(i + 1 < ntiles);
                const bool m = masked(has, i, c0);
                if (!FP8 && m) scan(slot);
                tile_barrier();
                if (FP8 && m) {
                    scan(slot);
                    tile_barrier();
                }
                // bf16: every wave is done with tile i - 1, whose buffer takes tile i + 1
                if (!FP8 && i + 1 < ntiles) issue(b1, has1, i + 1, slot ^ 1);
                const int32_t ahead = base_of(i + 2);
                f32x4 s = qk(slot_of(slot));
                mask(s, has, i, c0);
                if (first) {
                    const float top = top_of(s) * c_s;
                    m_ref = top == -INFINITY ? 0.0f : top;
                    m_ref -= (float)lift_of<FP8>(k1 - k0, false);
                    first = false;
                }
                p_out(s);
                const int32_t b2 = __builtin_amdgcn_readfirstlane(ahead);
                const uint32_t has2 = i + 2 < ntiles ? has_of(b2, i + 2, c0) : 0;
                tile_barrier();
                // 656-byte rows: every wave is done with the raw slot, which takes tile i + 2
                if (FP8 && i + 2 < ntiles) issue(b2, has2, i + 2, slot);
                pv(FP8 ? (lds_cptr)T0 : (lds_cptr)slot_of(slot));
                has = has1, b1 = b2, has1 = has2;
            }
        }
        // row sums over the lanes and halves that share a row (s_top: free)
        float l = l_lane, t = FP8 ? p_top : 0.0f;
        l += __shfl_xor(l, 16, 64), l += __shfl_xor(l, 32, 64);
        t = fmaxf(t, __shfl_xor(t, 16, 64)), t = fmaxf(t, __shfl_xor(t, 32, 64));
        const uint64_t anys = __builtin_amdgcn_ballot_w64(any);
        any = ((anys >> (lane & 15)) & 0x0001000100010001ull) != 0;
        __syncthreads();
        if (threadIdx.x == 0) s_misc[1] = 0, s_misc[2] = 0, s_misc[3] = 0;
        if (q == 0) s_top[half][my] = any ? l : 0.0f;
        __syncthreads();
        l = s_top[0][my] + s_top[1][my];
        __syncthreads();
        if (q == 0) s_top[half][my] = any ? (FP8 ? t : 1.0f) : -1.0f;
        __syncthreads();
        t = fmaxf(s_top[0][my], s_top[1][my]);
        any = t >= 0.0f;
        const int lift = lift_of<FP8>(k1 - k0, false);
        const bool held = FP8 ? t >= __builtin_ldexpf(0.5f, lift) && t <= FP16_MAX
                              : l > __builtin_ldexpf(1.0f, lift - 40) && l < __builtin_ldexpf(1.0f, lift + 40);
        if (!again && any && !held) s_misc[1] = 1;
        if (FP8 ? range_bad : any && l >= 0.5f) s_misc[2] = 1;
        l_lane = l;
        __syncthreads();
        all_nan = too_long || (FP8 && s_misc[2] != 0);
        bool served = again || __builtin_amdgcn_readfirstlane(s_misc[1]) == 0;
        if (!FP8 && !again && __builtin_expect(served && __builtin_amdgcn_readfirstlane(s_misc[2]) != 0, false)) {
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
        p_top = 0.0f;
        float top = -INFINITY;
        for (int c = 0; c < nspans; ++c) {
            const int c0 = start_of(c);
            resolve(c0);
            for (int i = 0; i < ntiles; ++i) {
                const int32_t base = __builtin_amdgcn_readfirstlane(base_of(i));
                const uint32_t has = has_of(base, i, c0);
                issue(base, has, i, 0);
                landed(false);
                tile_barrier();
                if (masked(has, i, c0)) {
                    scan(0);
                    tile_barrier();
                }
                f32x4 s = qk(slot_of(0));
                mask(s, has, i, c0);
                top = fmaxf(top, top_of(s));       // (its barriers also end the slot's use)
            }
        }
        m_ref = top == -INFINITY ? 0.0f : top * c_s;
        m_ref -= (float)lift_of<FP8>(k1 - k0, true);
    }

    // ---- O / l, LSE: rows' values from the scoring lanes to the lanes that hold O ----
    const int lift = lift_of<FP8>(k1 - k0, again);
    const float lse = all_nan ? __builtin_nanf("")
                              : (m_ref + (float)lift + __builtin_amdgcn_logf(__builtin_ldexpf(l_lane, -lift))) * LN2;
    __syncthreads();
    if (q == 0 && half == 0) {
        s_top[0][my] = all_nan ? __builtin_nanf("") : (any ? 1.0f / l_lane : 0.0f);
        const int64_t at = (int64_t)blk.first * p.H + blk.r0 + my;
        if (my >= blk.rows) {
        } else if (p.ns > 1) {
            p.part_lse[(int64_t)split * p.T * p.H + at] = any || all_nan ? lse : -FLT_MAX;
        } else if (p.lse) {
            p.lse[at] = any || all_nan ? lse : INFINITY;
        }
    }
    __syncthreads();
    const int hi = lane >> 5, r32 = lane & 31;
    const float inv = s_top[0][r32];
    if (p.ns == 1) {
        constexpr int OUT_STRIDE = D_VO * 2 + 16;
        static_assert(32 * OUT_STRIDE <= BYTES, "the stage fits the tile buffers");
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = {o[m][4 * g] * inv, o[m][4 * g + 1] * inv, o[m][4 * g + 2] * inv, o[m][4 * g + 3] * inv};
                lds_st<u32x2>(T0 + r32 * OUT_STRIDE + 2 * (128 * wave + 32 * m + 8 * g + 4 * hi),
                              __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4)));
            }
        __syncthreads();
        const bool o16 = ((p.o_st | p.o_sh) & 7) == 0 && ((uintptr_t)p.out & 15) == 0;
        for (int k = 0; k < 8; ++k) {
            const int r = 8 * wave + k;
            if (r >= blk.rows) break;
            const int t = blk.first + (blk.r0 + r) / p.H, h = (blk.r0 + r) % p.H;
            const u32x4 v = lds_ld<u32x4>(T0 + r * OUT_STRIDE + 16 * lane);
            __bf16* const dst = p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + 8 * lane;
            if (o16) {
                *reinterpret_cast<u32x4*>(dst) = v;
            } else {
                reinterpret_cast<u32x2*>(dst)[0] = u32x2{v[0], v[1]};
                reinterpret_cast<u32x2*>(dst)[1] = u32x2{v[2], v[3]};
            }
        }
    } else {
        constexpr int PST = D_VO + 16;
        static_assert(4 * 32 * PST <= BYTES, "four waves' stages fit the tile buffers");
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
            const int r = 2 * k + (lane >> 5);
            const f32x4 v = lds_ld<f32x4>(stg + r * PST + 16 * (lane & 31));
            if (r < blk.rows) *reinterpret_cast<f32x4*>(dst0 + (int64_t)r * D_VO + 128 * wave + 4 * (lane & 31)) = v;
        }
    }
}

// Joins the partials of a row's splits, SHARES waves a row: a lane holds 8 of its 512 values,
// wave i takes splits i, i + SHARES, ...  Splits past the row's positions wrote nothing and add nothing.
// Bound by a chain of memory round trips where there are few rows (128 rows of 16 splits 4.1 us, 6.8 with one
// wave a row and the loads in turn), by the partials' bytes where there are many (40040 rows of 1 to 3 splits 39 us).
template <int SHARES>
__global__ void __launch_bounds__(NTHR) dsa_mla_chunk_combine_kernel(const ChunkParams p) {
    __shared__ __attribute__((aligned(16))) float s_o[SHARES > 1 ? SHARES * D_VO : 4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int share = SHARES > 1 ? wave : 0;
    const int64_t row = (int64_t)blockIdx.x * (NWAVE / SHARES) + wave / SHARES;
    const int64_t step = (int64_t)p.T * p.H;
    if (row >= step) return;
    const int t = (int)(row / p.H), h = (int)(row - (int64_t)t * p.H);
    // Requested at once, before it is known which of them are needed: the sequences' bounds, every
    // split's sum and (where a row has four waves) a wave's first eight partials.
    const int32_t i0 = min(lane, p.B - 1);
    const int32_t start_l = p.indptr[i0], end_l = p.indptr[i0 + 1], len_l = p.lens[i0];
    const int32_t dealt = p.dealt ? *p.dealt : 0;
    const float lse_l = p.part_lse[min(lane, p.ns - 1) * step + row];
    const float* const src = p.part_o + row * D_VO + 8 * lane;
    f32x4 x[8], y[8];
    auto fetch = [&](int s0, int last) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const float* const at = src + min(s0 + s * SHARES, last) * step * D_VO;
            x[s] = *reinterpret_cast<const f32x4*>(at), y[s] = *reinterpret_cast<const f32x4*>(at + 4);
        }
    };
    if constexpr (SHARES > 1) fetch(share, p.ns - 1);
    int64_t limit;
    int32_t len;
    if (p.B <= 64) {
        const int32_t b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < p.B && end_l <= t));
        if (b >= p.B || t < __builtin_amdgcn_readlane(start_l, b)) return;
        len = __builtin_amdgcn_readlane(len_l, b);
        const int64_t own = (int64_t)len - __builtin_amdgcn_readlane(end_l, b) + t + 1;
        limit = max((int64_t)0, p.causal ? min(own, (int64_t)len) : (int64_t)len);
    } else {
        const int32_t b = seq_of(p.indptr, p.B, t);
        if (b == NO_SEQ) return;
        len = p.lens[b];
        limit = limit_of(p, b, t);
    }
    int32_t per = p.per_split;
    if (p.dealt) {
        // (as find_work has it; 1 where there is no position, and no split is read)
        const int32_t tiles = (int32_t)((min((int64_t)min(max(len, 1), p.max_len), p.pages.limit) + TILE - 1) / TILE);
        per = TILE * max(1, parts(tiles, max(1, parts(tiles, dealt))));
    }
    const int ns = (int)min((int64_t)p.ns, (min(limit, p.pages.limit) + per - 1) / per);
    const float mine = lane < ns ? lse_l : -FLT_MAX;
    float top = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const bool any = __builtin_amdgcn_ballot_w64(mine != -FLT_MAX) != 0;
    // (a weight of 1 is 2^-7 here, so that 64 partials near the largest value stay in fp32 together)
    const float w = mine == -FLT_MAX ? 0.0f : 0x1p-7f * __builtin_amdgcn_exp2f((mine - top) * LOG2E);
    const float total = wave_sum(w);
    float o[8] = {};
    // eight splits' loads in flight at a time; the last one's again past it.  One of no weight is not added
    // (its partial may hold anything).
    for (int s0 = share; s0 < ns; s0 += 8 * SHARES) {
        if (SHARES == 1 || s0 != share) fetch(s0, ns - 1);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const float f = __shfl(w, s0 + s * SHARES, 64);          // 0 past the last
            if (f != 0.0f) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = __builtin_fmaf(f, x[s][i], o[i]);
                    o[4 + i] = __builtin_fmaf(f, y[s][i], o[4 + i]);
                }
            }
        }
    }
    const float nan = len > p.max_len ? __builtin_nanf("") : 0.0f;
    const float inv = any ? 1.0f / total + nan : nan;
    __bf16* const dst = p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh;
    if constexpr (SHARES == 1) {
        const f32x8 r = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv};
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_convertvector(r, bf16x8));
        u32x2* const d = reinterpret_cast<u32x2*>(dst + 8 * lane);
        d[0] = u32x2{v[0], v[1]};
        d[1] = u32x2{v[2], v[3]};
    } else {
        f32x4* const mine_o = reinterpret_cast<f32x4*>(s_o + share * D_VO + 8 * lane);
        mine_o[0] = f32x4{o[0], o[1], o[2], o[3]};
        mine_o[1] = f32x4{o[4], o[5], o[6], o[7]};
        __syncthreads();
        static_assert(D_VO == 2 * NTHR);
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int i = 0; i < SHARES; ++i) a += s_o[i * D_VO + 2 * threadIdx.x], c += s_o[i * D_VO + 2 * threadIdx.x + 1];
        const f32x2 r = {a * inv, c * inv};
        *reinterpret_cast<uint32_t*>(dst + 2 * threadIdx.x) = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
    }
    if (lane == 0 && share == 0 && p.lse)
        p.lse[row] = nan != 0.0f ? nan : (any ? top + __builtin_amdgcn_logf(0x1p7f * total) * LN2 : INFINITY);
}

// ------------------------------------------------------------------- host

// The kernel and split count of a call: those of least expected time, from the call's sizes
// alone.  A workgroup takes `start` us and `tile` us for each 32 positions (`pair` where two
// share a CU); past one workgroup a CU (two of the narrow kernel) they run in rounds; the
// cache's rows come at most at `BYTES_US` (splits of a sequence and blocks of rows find each
// other's in the caches); a split writes and reads its fp32 partials.  Fitted to 3600 calls of
// both kernels (1 to 200 sequences of 1 to 400 tokens, 1 to 128 heads, 64 to 60000 positions,
// 1 to 64 splits): the choice is 1.9 % above the fastest candidate on average, 27 % at most
// (15 tokens of 32 heads over 21979 bf16 rows, 75 us in 32 splits and 59 in 48).  Measured on
// the two sides of it, us: one token of 128 heads over 1501 rows, 128-row blocks 25.2, 32-row 17.7;
// 256 of 16 heads over 4096 302 and 217; 200 of 128 heads over 1000 78 and 120; 512 tokens of
// 16 heads over the same 4096 rows 90 (4 splits) and 120.
constexpr Kernel KERNELS[2][2] = {       // [656-byte rows][narrow]
    {{6.3f, 1.83f, 0.0f}, {6.4f, 1.15f, 1.81f}},
    {{10.6f, 2.47f, 0.0f}, {8.3f, 1.48f, 2.07f}},
};
constexpr float BYTES_US = 8.5e6f, FIRST_US = 10.7f, JOIN_US = 3.7f;
constexpr int COUNTS[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 28, 32, 40, 48, 56, 64};

constexpr int64_t MAX_GROUPS = ((int64_t)1 << 32) / NTHR - 1, MAX_SPLIT_ROWS = MAX_GROUPS * NWAVE;

// Four waves join a row where there are few rows of many splits, one wave elsewhere.  A call with one
// and with four, us: 16 rows of 48 splits 22.7 and 17.4; 128 of 32 27.0 and 23.6, of 8 20.4 and 19.6, of 2
// 19.9 and 19.9; 512 of 16 30.3 and 28.5, of 4 21.4 and 22.0; 1024 of 32 38.0 and 37.2, of 8 26.4 and 27.2;
// 2048 of 8 35.0 and 36.7; 4096 of 4 34.2 and 39.0.
constexpr int64_t FEW_ROWS = 1024;
constexpr int FOUR_FROM = 5;

struct Plan {
    bool narrow;
    int ns;              // at most
    int32_t per;         // positions of a split
    bool deal;           // the device chooses the split's positions
};

float expected_us(const dsa_mla_chunk_args* a, bool narrow, int64_t blocks, int ns) {
    const bool fp8 = a->kv_format == DSA_KV_FP8_656;
    const Kernel& k = KERNELS[fp8][narrow];
    const int64_t tiles = (a->max_kv_len + (int64_t)TILE - 1) / TILE, each = (tiles + ns - 1) / ns;
    const float groups = (float)blocks * ns;
    auto in_rounds = [](float us, float rounds) {
        return us * (rounds <= 1.0f ? 1.0f : rounds <= 3.0f ? std::ceil(rounds) : rounds + 0.5f);
    };
    float us = narrow && groups > CUS ? in_rounds(k.start + each * k.pair, groups / (2 * CUS))
                                      : in_rounds(k.start + each * k.tile, groups / CUS);
    const float row = fp8 ? DSA_MLA_FP8_ROW_BYTES : DSA_MLA_BF16_ROW_BYTES;
    us = std::max(us, FIRST_US + (float)a->B * a->max_kv_len * row / BYTES_US);
    if (ns > 1) us += JOIN_US + (float)ns * a->T * a->H * (2 * 4 * (D_VO + 1)) / PART_BYTES_US;
    return us;
}

Plan plan_of(const dsa_mla_chunk_args* a) {
    Plan best{};
    float least = INFINITY;
    for (int n = 0; n < 2; ++n) {
        const int32_t m = n ? NARROW : BLOCK;
        const int64_t blocks = dsa_seq::block_start(a->T, a->B, a->H, m, dsa_seq::common(a->H, m));
        for (const int c : COUNTS) {
            const int ns = a->num_splits ? a->num_splits : c;
            // (a split of fewer positions than a tile is none; 64 splits of a grid's y extent)
            if (ns > 1 && !a->num_splits && (int64_t)a->max_kv_len < (int64_t)ns * TILE) break;
            if (ns > 1 && (int64_t)a->T * a->H > MAX_SPLIT_ROWS) break;
            const float us = expected_us(a, n != 0, blocks, ns);
            if (us < least) least = us, best.narrow = n != 0, best.ns = ns;
            if (a->num_splits) break;
        }
    }
    // up to twice as many splits, of the size that the lengths ask for
    best.deal = !a->num_splits && best.ns > 1 && a->B <= 64;
    if (best.deal) best.ns = std::min(2 * best.ns, (int)DSA_MLA_MAX_SPLITS);
    const int64_t each = (a->max_kv_len + (int64_t)best.ns - 1) / best.ns;
    best.per = (int32_t)std::min<int64_t>(INT32_MAX - TILE + 1, std::max<int64_t>(TILE, (each + TILE - 1) / TILE * TILE));
    return best;
}

size_t workspace_of(int ns, int64_t T, int64_t H) {
    // (and 16 bytes for the dealt split)
    return ns > 1 ? (size_t)ns * T * H * (D_VO + 1) * sizeof(float) + 16 : 0;
}

int validate(const dsa_mla_chunk_args* a) {
    if (!a) return DSA_ERR_NULL_POINTER;
    if (a->kv_format != DSA_KV_BF16 && a->kv_format != DSA_KV_FP8_656) return DSA_ERR_BAD_FORMAT;
    if (a->T < 0 || a->B < 0 || a->H < 1 || a->max_kv_len < 0 || a->kv_total_rows < 0 || a->kv_total_rows > INT32_MAX)
        return DSA_ERR_BAD_SHAPE;
    if (a->max_kv_len > DSA_MLA_MAX_LIST) return DSA_ERR_BAD_SHAPE;
    if (a->num_splits < 0 || a->num_splits > DSA_MLA_MAX_SPLITS) return DSA_ERR_BAD_SPLITS;
    // (a grid holds below 2^32 threads: workgroups of 32 rows, and the join's of 4)
    const int64_t rows = (int64_t)a->T * a->H;
    if (rows + (int64_t)NARROW * a->B > MAX_GROUPS * NARROW) return DSA_ERR_BAD_SHAPE;
    if (a->num_splits > 1 && rows > MAX_SPLIT_ROWS) return DSA_ERR_BAD_SHAPE;
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
    if (!(a->sm_scale > 0.0f && a->sm_scale <= FLT_MAX)) return DSA_ERR_UNSUPPORTED;
    if (a->T == 0 || a->B == 0) return DSA_OK;
    if (!a->q || !a->out || !a->q_indptr || !a->seq_lens || (a->kv_total_rows > 0 && !a->kv_cache))
        return DSA_ERR_NULL_POINTER;
    if (dsa_overlap::within({a->T, a->H, a->o_stride_t, a->o_stride_h, D_VO})) return DSA_ERR_BAD_STRIDE;
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
    *num_splits = plan_of(a).ns;
    return DSA_OK;
}

int dsa_mla_chunk_workspace_size(const dsa_mla_chunk_args* a, size_t* bytes) {
    if (!bytes) return DSA_ERR_NULL_POINTER;
    const int rc = validate(a);
    if (rc) return rc;
    *bytes = a->T == 0 || a->B == 0 ? 0 : workspace_of(plan_of(a).ns, a->T, a->H);
    return DSA_OK;
}

int dsa_mla_chunk(const dsa_mla_chunk_args* a, void* ws, size_t ws_bytes, void* stream) {
    const int rc = validate(a);
    if (rc) return rc;
    if (a->T == 0 || a->B == 0) return DSA_OK;
    ChunkParams p{};
    const Plan plan = plan_of(a);
    p.ns = plan.ns;
    p.per_split = plan.per;
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
    p.dealt = plan.deal ? (int32_t*)(p.part_lse + (size_t)p.ns * a->T * a->H) : nullptr;
    p.kernel = KERNELS[a->kv_format == DSA_KV_FP8_656][plan.narrow];
    p.T = a->T, p.B = a->B, p.H = a->H, p.causal = a->causal, p.max_len = a->max_kv_len;
    p.scale_log2 = a->sm_scale * LOG2E;
    const bool narrow = plan.narrow;
    const bool runs = !a->block_table || a->block_size % TILE == 0;
    const int32_t m = narrow ? NARROW : BLOCK;
    p.common = dsa_seq::common(a->H, m);
    const int64_t most = dsa_seq::block_start(a->T, a->B, a->H, m, p.common);
    const int64_t places = plan.narrow ? 2 * CUS : CUS;
    const dim3 blocks((unsigned)(plan.deal ? std::min(most * p.ns, most <= places / 4 ? places : 3 * places + most) : most),
                      plan.deal ? 1u : (unsigned)p.ns);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, blocks, dim3(NTHR), 0, (hipStream_t)stream, p); };
    const bool fp8 = a->kv_format == DSA_KV_FP8_656;
    if (!narrow) launch(fp8 ? dsa_mla_chunk_tile_kernel<DSA_KV_FP8_656> : dsa_mla_chunk_tile_kernel<DSA_KV_BF16>);
    else if (fp8) launch(runs ? dsa_mla_chunk_narrow_kernel<DSA_KV_FP8_656, true> : dsa_mla_chunk_narrow_kernel<DSA_KV_FP8_656, false>);
    else launch(runs ? dsa_mla_chunk_narrow_kernel<DSA_KV_BF16, true> : dsa_mla_chunk_narrow_kernel<DSA_KV_BF16, false>);
    if (hipGetLastError() != hipSuccess) return DSA_ERR_HIP;
    if (p.ns > 1) {
        const int64_t rows = (int64_t)a->T * a->H;
        if (rows <= FEW_ROWS && p.ns >= FOUR_FROM)
            hipLaunchKernelGGL(dsa_mla_chunk_combine_kernel<4>, dim3((unsigned)rows), dim3(NTHR), 0, (hipStream_t)stream, p);
        else
            hipLaunchKernelGGL(dsa_mla_chunk_combine_kernel<1>, dim3((unsigned)((rows + NWAVE - 1) / NWAVE)), dim3(NTHR),
                               0, (hipStream_t)stream, p);
        if (hipGetLastError() != hipSuccess) return DSA_ERR_HIP;
    }
    return DSA_OK;
}

}  // extern "C"
