// dsa_prep.hip - gfx950 kernels in front of the attention: norms of queries and
// keys with the position rotation (dsa_qk_norm_rope), and the write of latent
// rows and index keys into the paged caches (dsa_kv_append), of
// include/dsa_chunk.h.
//
// Both are one pass over memory: a row lives in the registers of one wave, 8
// values (16 bytes) a lane, between its load and its store.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "../../include/dsa_chunk.h"
#include "dsa_overlap.h"
#include "dsa_seq.h"

namespace {

#include "dsa_lds.h"

constexpr int WAVES = 4;                 // waves of a workgroup
constexpr int ROT = DSA_MLA_D_ROPE;      // rotated values of a row

// ---- sums over 16 and over 64 lanes, result in every one of them ----
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
template <class F>
__device__ __forceinline__ float all16(float x, F f) {
    x = f(x, dpp<0xB1>(x));      // lanes 1, 0, 3, 2
    x = f(x, dpp<0x4E>(x));      // lanes 2, 3, 0, 1
    x = f(x, dpp<0x141>(x));     // the 8 lanes mirrored
    x = f(x, dpp<0x140>(x));     // the 16 lanes mirrored
    return x;
}
template <class F>
__device__ __forceinline__ float all4(float x, F f) {
    x = f(x, dpp<0xB1>(x));
    x = f(x, dpp<0x4E>(x));
    return x;
}
__device__ __forceinline__ float sum16(float x) {
    return all16(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float sum64(float x) {
    x = sum16(x);
    x += __shfl_xor(x, 16, 64);
    x += __shfl_xor(x, 32, 64);
    return x;
}
__device__ __forceinline__ float max_abs(float a, float b) { return fmaxf(a, b); }

// ---- 8 values of a lane ----
struct V8 {
    float v[8];
};
__device__ __forceinline__ V8 unpack8(u32x4 x) {
    V8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.v[2 * i] = __uint_as_float(x[i] << 16);
        r.v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
    }
    return r;
}
__device__ __forceinline__ u32x4 pack8(const V8& r) {
    const f32x8 a = {r.v[0], r.v[1], r.v[2], r.v[3], r.v[4], r.v[5], r.v[6], r.v[7]};
    return __builtin_bit_cast(u32x4, __builtin_convertvector(a, bf16x8));
}
__device__ __forceinline__ V8 load8f(const float* p) {
    V8 r;
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = a[i], r.v[4 + i] = b[i];
    return r;
}

// A lane's factors of the rotation: its 8 values are numbers 8 c .. 8 c + 7 of
// the 64 rotated ones (c = 0 .. 7).  own[e] multiplies value e, other[e] its
// partner in the pair (with the sign of its place in it).
struct Turn {
    V8 own, other;
};
template <int ROPE>
__device__ __forceinline__ Turn load_turn(const float* cos_sin, int64_t n_pos, int64_t pos, int c, bool inverse) {
    Turn t;
    if constexpr (ROPE == DSA_ROPE_NONE) return t;
    const bool known = pos >= 0 && pos < n_pos;
    const float* row = cos_sin + (known ? pos : 0) * ROT;
    const float flip = inverse ? -1.0f : 1.0f;
    if constexpr (ROPE == DSA_ROPE_INTERLEAVED) {
        f32x4 co = {}, si = {};
        if (n_pos > 0) {
            co = *reinterpret_cast<const f32x4*>(row + 4 * c);
            si = *reinterpret_cast<const f32x4*>(row + 32 + 4 * c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.own.v[2 * i] = t.own.v[2 * i + 1] = co[i];
            t.other.v[2 * i] = -flip * si[i];
            t.other.v[2 * i + 1] = flip * si[i];
        }
    } else {
        V8 si = {};
        t.own = V8{};
        if (n_pos > 0) {
            t.own = load8f(row + 8 * (c & 3));
            si = load8f(row + 32 + 8 * (c & 3));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) t.other.v[i] = c < 4 ? -flip * si.v[i] : flip * si.v[i];
    }
    if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t.own.v[i] = __builtin_nanf("");
    }
    return t;
}
// The lane's values turned; the partner of a halves pair sits 4 lanes away, so
// every lane of the wave takes part and `on` says whether this one's are rotated.
template <int ROPE>
__device__ __forceinline__ void turn8(V8& x, const Turn& t, bool on) {
    if constexpr (ROPE == DSA_ROPE_NONE) return;
    V8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float partner = ROPE == DSA_ROPE_INTERLEAVED ? x.v[i ^ 1] : __shfl_xor(x.v[i], 4, 64);
        y.v[i] = __builtin_fmaf(x.v[i], t.own.v[i], partner * t.other.v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = on ? y.v[i] : x.v[i];
}

// The norm of a row spread over LANES lanes, `in` saying whether this lane's
// values are under it: mean and variance from fp32 sums (the variance from the
// differences to the mean, so that a large mean loses nothing).
template <int LANES>
__device__ __forceinline__ void norm8(V8& x, int kind, bool in, float inv_n, float eps, bool has_w, const V8& w, bool has_b,
                                      const V8& b) {
    if (kind == DSA_NORM_NONE) return;
    auto total = [](float s) { return LANES == 64 ? sum64(s) : sum16(s); };
    float mean = 0.0f;
    if (kind == DSA_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x.v[i];
        mean = total(in ? s : 0.0f) * inv_n;
    }
    V8 d;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        d.v[i] = x.v[i] - mean;
        s = __builtin_fmaf(d.v[i], d.v[i], s);
    }
    const float r = 1.0f / sqrtf(total(in ? s : 0.0f) * inv_n + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float y = d.v[i] * r;
        if (has_w) y *= w.v[i];
        if (has_b) y += b.v[i];
        x.v[i] = in ? y : x.v[i];
    }
}

// Sequences and positions of the N tokens from t on (include/dsa_chunk.h); NO_SEQ for one of none.  Up to
// 64 sequences are read at once, a lane each, so that a token waits for one load and not for three in turn.
template <int N>
struct Located {
    int32_t b[N];
    int64_t pos[N];
};
template <int N>
__device__ __forceinline__ Located<N> locate(const int32_t* indptr, const int32_t* lens, int32_t B, int32_t t) {
    Located<N> r;
    if (B <= 64) {
        const int lane = threadIdx.x & 63, i = min(lane, B - 1);
        const int32_t start = indptr[i], end = indptr[i + 1], len = lens[i];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int32_t b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < B && end <= t + k));
            const int32_t at = min(b, B - 1);
            r.b[k] = b < B && t + k >= __builtin_amdgcn_readlane(start, at) ? b : NO_SEQ;
            r.pos[k] = (int64_t)__builtin_amdgcn_readlane(len, at) - __builtin_amdgcn_readlane(end, at) + t + k;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            r.b[k] = seq_of(indptr, B, t + k);
            r.pos[k] = r.b[k] == NO_SEQ ? -1 : dsa_seq::position_of(indptr, lens, r.b[k], t + k);
        }
    }
    return r;
}

// ---------------------------------------------------------------------------
// Norms and rotation of queries and keys.  A wave takes GROUP heads of one
// token of one stream: their loads are all in flight before the first is used,
// and the rotation's factors and the weights are read once for them.  D = 512
// and 576: a row of 64 lanes (and, for 576, the last 64 values of 8 rows in one
// further load); D = 128: four rows of 16 lanes.
// Bound by memory: 4096 tokens of 129 rows of 512, 1.08 GB in 195 us, 5.6 TB/s (a 1 GiB copy: 5.1); 1531 tokens
// of 65 rows of 128, 51 MB in 12 us, 4.2 TB/s; 3000 of 129 rows of 576, 892 MB in 158 us, 5.6 TB/s.  Two tokens of
// 129 rows of 576 take 6.2 us: 3.1 for one row without a norm, a launch and its chain of two loads, 1.6 more for 8 rows
// each in 16 waves a token, 1.6 more for the key's norm, which runs over all 8 places of its wave where one is taken
// (one row with a norm 5.2, eight 5.6).
// ---------------------------------------------------------------------------
template <int D>
constexpr int GROUP = D == 128 ? 16 : 8;

template <int D, int ROPE>
__global__ void __launch_bounds__(64 * WAVES) dsa_qk_norm_rope_kernel(const dsa_qk_norm_rope_args p, int q_groups,
                                                                      int groups) {
    constexpr int G = GROUP<D>;
    constexpr int PER = D == 128 ? 4 : 1;            // rows of a load
    constexpr int LOADS = G / PER;
    const int lane = threadIdx.x & 63;
    const int job = (int)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = job / groups, g = job - t * groups;
    if (t >= p.T) return;
    const bool is_q = g < q_groups;
    const dsa_norm_rope_rows& s = is_q ? p.q : p.k;
    const int h0 = (is_q ? g : g - q_groups) * G;
    const int heads = min(G, s.H - h0);
    // this lane's 16-byte piece of its row, and the row's number in a load
    const int piece = D == 128 ? lane & 15 : lane, sub = D == 128 ? lane >> 4 : 0;
    const __bf16* x = (const __bf16*)s.x + (int64_t)t * s.stride_t + (int64_t)h0 * s.stride_h;
    // every load of the rows goes out before the token's position is known
    u32x4 v[LOADS], tail = {};
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int h = PER * j + sub;
        if (h < heads) v[j] = *reinterpret_cast<const u32x4*>(x + (int64_t)h * s.stride_h + 8 * piece);
    }
    if constexpr (D == 576) {
        const int h = lane >> 3;
        if (h < heads) tail = *reinterpret_cast<const u32x4*>(x + (int64_t)h * s.stride_h + 512 + 8 * (lane & 7));
    }
    int64_t pos;
    if (p.positions) {
        pos = p.positions[t];
    } else if (ROPE != DSA_ROPE_NONE || p.q_indptr) {
        const Located<1> at = locate<1>(p.q_indptr, p.seq_lens, p.B, t);
        if (at.b[0] == NO_SEQ) return;
        pos = at.pos[0];
    } else {
        pos = 0;
    }
    const int turned = piece - p.rot_off / 8;          // piece of the rotated 64
    const bool rot = turned >= 0 && turned < 8, in = 8 * piece < p.norm_dim;
    const int rot_tail = D == 576 ? (lane & 7) : 0;    // the tail's lanes hold pieces 64 + (lane & 7)
    const bool tail_rot = p.rot_off == 512;
    Turn turn = load_turn<ROPE>(p.cos_sin, p.n_pos, pos, (D == 576 && tail_rot) ? rot_tail : turned & 7,
                                p.inverse != 0);
    V8 w{}, b{};
    if (in && s.weight) w = load8f(s.weight + 8 * piece);
    if (in && s.bias) b = load8f(s.bias + 8 * piece);
    __bf16* o = (__bf16*)s.out + (int64_t)t * s.out_stride_t + (int64_t)h0 * s.out_stride_h;
    const float inv_n = 1.0f / (float)p.norm_dim;

#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int h = PER * j + sub;
        V8 y = unpack8(v[j]);
        norm8<D == 128 ? 16 : 64>(y, s.norm, in, inv_n, p.eps, s.weight != nullptr, w, s.bias != nullptr, b);
        turn8<ROPE>(y, turn, rot);
        if (h < heads) *reinterpret_cast<u32x4*>(o + (int64_t)h * s.out_stride_h + 8 * piece) = pack8(y);
    }
    if constexpr (D == 576) {
        const int h = lane >> 3;
        V8 y = unpack8(tail);
        turn8<ROPE>(y, turn, tail_rot);
        if (h < heads) *reinterpret_cast<u32x4*>(o + (int64_t)h * s.out_stride_h + 512 + 8 * (lane & 7)) = pack8(y);
    }
}

// ---------------------------------------------------------------------------
// Append: waves 0 .. T-1 write one latent row each, the waves after them the
// index keys of four tokens each (16 lanes a key).  Each waits for its sequence's
// bounds, then for its page and its position's angles; its values, requested
// first, are there by then.  That chain is what a call takes: one token 2.9 us, 128
// 3.7, 4099 tokens of V4 fp8 rows 5.5 (7.7 MB), 9238 of 656-byte rows and index
// keys 11.8 (24 MB; 11548 waves, of which 7168 fit the chip at a time).
// ---------------------------------------------------------------------------
struct AppendParams {
    dsa_kv_append_args a;
    dsa_seq::Pages pages;
};

// e4m3fn codes of 8 values: round to nearest even, saturating at 448, NaN to NaN
__device__ __forceinline__ u32x2 e4m3x8(const V8& x) {
    u32x2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float c[4];
        unsigned nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = x.v[4 * h + i];
            c[i] = fminf(fmaxf(f, -448.0f), 448.0f);
            // (an infinity is no value of the type either)
            const unsigned bits = __float_as_uint(f);
            if ((bits & 0x7FFFFFFFu) >= 0x7F800000u) nan |= (0x7Fu | ((bits >> 24) & 0x80u)) << (8 * i), c[i] = 0.0f;
        }
        unsigned w = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        w = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], (int)w, true);
        out[h] = w | nan;
    }
    return out;
}
__device__ __forceinline__ float amax8(const V8& x) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x.v[i]));
    return a;
}
// e of the least power of two 2^e >= amax / 448 = amax / (1.75 * 2^8)
__device__ __forceinline__ int scale_exponent(float amax) {
    const unsigned bits = __float_as_uint(amax);
    if (bits == 0) return 0;
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(-126, min(127, e));
}

template <int ROPE>
__device__ __forceinline__ void append_latent(const AppendParams& p, int t) {
    const dsa_kv_append_args& a = p.a;
    const int lane = threadIdx.x & 63;
    const int fmt = a.kv_format;
    const bool wide = fmt == DSA_KV_BF16 || fmt == DSA_KV_FP8_656 || fmt == DSA_KV_MXFP8;   // 576 values
    const __bf16* x = (const __bf16*)a.kv + (int64_t)t * a.kv_stride_t;
    const u32x4 raw = *reinterpret_cast<const u32x4*>(x + 8 * lane);
    u32x4 raw_tail = {};
    if (wide && lane < 8) raw_tail = *reinterpret_cast<const u32x4*>(x + 512 + 8 * lane);
    V8 w{};
    if (a.weight) w = load8f(a.weight + 8 * lane);

    const Located<1> at = locate<1>(a.q_indptr, a.seq_lens, a.B, t);
    if (at.b[0] == NO_SEQ) return;
    const int64_t pos = at.pos[0];
    const Turn turn = load_turn<ROPE>(a.cos_sin, a.n_pos, pos, lane & 7, false);      // in flight beside the page's
    const int64_t row = dsa_seq::row_of(p.pages, at.b[0], pos, a.cache_rows);
    if (row < 0) return;
    V8 v = unpack8(raw), tail = unpack8(raw_tail);
    norm8<64>(v, a.norm, true, 1.0f / 512.0f, a.eps, a.weight != nullptr, w, false, w);
    if (wide) turn8<ROPE>(tail, turn, true);
    else turn8<ROPE>(v, turn, lane >= 56);

    unsigned char* const dst = (unsigned char*)a.cache + row * a.stride_row * (fmt == DSA_KV_BF16 || fmt == DSA_KV_BF16_D512 ? 2 : 1);
    unsigned char* const rope = (unsigned char*)a.cache_rope + row * a.rope_stride_row * 2;
    if (fmt == DSA_KV_BF16 || fmt == DSA_KV_BF16_D512) {
        *reinterpret_cast<u32x4*>(dst + 16 * lane) = pack8(v);
        if (wide && lane < 8) *reinterpret_cast<u32x4*>(dst + 1024 + 16 * lane) = pack8(tail);
    } else if (fmt == DSA_KV_FP8_656) {
        const float amax = all16(amax8(v), max_abs);
        const float scale = amax / 448.0f;
        V8 c;
#pragma unroll
        for (int i = 0; i < 8; ++i) c.v[i] = v.v[i] / scale;
        if (!(scale > 0.0f)) {                 // zeros, and the NaNs, which the largest value does not see
#pragma unroll
            for (int i = 0; i < 8; ++i) c.v[i] = v.v[i] != v.v[i] ? v.v[i] : 0.0f;
        }
        *reinterpret_cast<u32x2*>(dst + 8 * lane) = e4m3x8(c);
        if ((lane & 15) == 0) *reinterpret_cast<float*>(dst + 512 + 4 * (lane >> 4)) = scale;
        if (lane < 8) *reinterpret_cast<u32x4*>(dst + 528 + 16 * lane) = pack8(tail);
    } else {
        const int e = scale_exponent(all4(amax8(v), max_abs));
        V8 c;
#pragma unroll
        for (int i = 0; i < 8; ++i) c.v[i] = ldexpf(v.v[i], -e);
        const u32x2 codes = e4m3x8(c);
        if (wide) {
            *reinterpret_cast<u32x2*>(dst + 8 * lane) = codes;
            if ((lane & 3) == 0) ((unsigned char*)a.cache_scale)[row * a.scale_stride_row + (lane >> 2)] = (unsigned char)(e + 127);
            if (lane < 8) *reinterpret_cast<u32x4*>(rope + 16 * lane) = pack8(tail);
        } else if (lane < 56) {
            *reinterpret_cast<u32x2*>(dst + 8 * lane) = codes;
            if ((lane & 3) == 0) dst[DSA_MLA_V4_NOPE + (lane >> 2)] = (unsigned char)(e + 127);
        } else {
            *reinterpret_cast<u32x4*>(rope + 16 * (lane - 56)) = pack8(v);
        }
    }
}

template <int ROPE>
__device__ __forceinline__ void append_index(const AppendParams& p, int t0) {
    const dsa_kv_append_args& a = p.a;
    const int lane = threadIdx.x & 63, piece = lane & 15;
    const int t = t0 + (lane >> 4);
    const bool there = t < a.T;
    const u32x4 raw = *reinterpret_cast<const u32x4*>((const __bf16*)a.index_k + (int64_t)min(t, a.T - 1) * a.index_stride_t + 8 * piece);
    V8 w{}, bias{};
    if (a.index_weight) w = load8f(a.index_weight + 8 * piece);
    if (a.index_bias) bias = load8f(a.index_bias + 8 * piece);
    const Located<4> at = locate<4>(a.q_indptr, a.seq_lens, a.B, t0);
    const int k = lane >> 4;
    const int32_t b = there ? (k & 2 ? (k & 1 ? at.b[3] : at.b[2]) : (k & 1 ? at.b[1] : at.b[0])) : NO_SEQ;
    const int64_t pos = k & 2 ? (k & 1 ? at.pos[3] : at.pos[2]) : (k & 1 ? at.pos[1] : at.pos[0]);
    const int64_t row = b == NO_SEQ ? -1 : dsa_seq::row_of(p.pages, b, pos, a.index_rows);
    const Turn turn = load_turn<ROPE>(a.cos_sin, a.n_pos, pos, piece & 7, false);
    V8 v = unpack8(raw);
    norm8<16>(v, a.index_norm, true, 1.0f / 128.0f, a.index_eps, a.index_weight != nullptr, w,
              a.index_bias != nullptr, bias);
    turn8<ROPE>(v, turn, piece < 8);
    if (there && row >= 0)
        *reinterpret_cast<u32x4*>((__bf16*)a.index_cache + row * a.index_stride_row + 8 * piece) = pack8(v);
}

__global__ void __launch_bounds__(64 * WAVES) dsa_kv_append_kernel(const AppendParams p, int latent_jobs) {
    const int job = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (job < latent_jobs) {
        if (p.a.rope == DSA_ROPE_INTERLEAVED) append_latent<DSA_ROPE_INTERLEAVED>(p, job);
        else if (p.a.rope == DSA_ROPE_HALVES) append_latent<DSA_ROPE_HALVES>(p, job);
        else append_latent<DSA_ROPE_NONE>(p, job);
    } else if (p.a.index_k && 4 * (job - latent_jobs) < p.a.T) {
        const int t0 = 4 * (job - latent_jobs);
        if (p.a.index_rope == DSA_ROPE_INTERLEAVED) append_index<DSA_ROPE_INTERLEAVED>(p, t0);
        else if (p.a.index_rope == DSA_ROPE_HALVES) append_index<DSA_ROPE_HALVES>(p, t0);
        else append_index<DSA_ROPE_NONE>(p, t0);
    }
}

// ------------------------------------------------------------------- host
constexpr int64_t MAX_JOBS = (((int64_t)1 << 32) / (64 * WAVES) - 1) * WAVES;      // a grid holds below 2^32 threads

bool kind_ok(int v) { return v >= 0 && v <= 2; }
bool ptr16(const void* q) { return ((uintptr_t)q & 15) == 0; }

int check_rows(const dsa_norm_rope_rows& s, int T, int D, int rope) {
    if (s.H < 0) return DSA_ERR_BAD_SHAPE;
    if (s.H == 0) return DSA_OK;
    if (!kind_ok(s.norm)) return DSA_ERR_UNSUPPORTED;
    if (s.norm == DSA_NORM_NONE && (s.weight || s.bias)) return DSA_ERR_UNSUPPORTED;
    if (T == 0) return DSA_OK;
    if (!s.x || !s.out) return DSA_ERR_NULL_POINTER;
    if ((s.stride_t % 8) || (s.stride_h % 8) || (s.out_stride_t % 8) || (s.out_stride_h % 8)) return DSA_ERR_BAD_STRIDE;
    if (s.stride_t < 0 || s.stride_h < 0) return DSA_ERR_BAD_STRIDE;
    if ((s.H > 1 && s.out_stride_h < D) || (T > 1 && s.out_stride_t < D)) return DSA_ERR_BAD_STRIDE;
    if (s.x == s.out && ((s.H > 1 && s.stride_h != s.out_stride_h) || (T > 1 && s.stride_t != s.out_stride_t)))
        return DSA_ERR_BAD_STRIDE;
    if (!ptr16(s.x) || !ptr16(s.out) || !ptr16(s.weight) || !ptr16(s.bias)) return DSA_ERR_BAD_STRIDE;
    return DSA_OK;
}

// Rows of an output share memory with one another, with the other output's, or with an input's other than
// their own in place.
bool outputs_overlap(const dsa_qk_norm_rope_args& a) {
    using dsa_overlap::Rows;
    using dsa_overlap::wide;
    struct Part {
        Rows rows;
        int64_t at;            // address, in elements (all are 16-byte aligned)
        wide end;
    };
    auto part = [&](const dsa_norm_rope_rows& s, const void* p, int64_t st, int64_t sh) {
        const Rows r{a.T, s.H, st, sh, a.D};
        const int64_t at = (int64_t)((uintptr_t)p >> 1);
        return Part{r, at, at + dsa_overlap::extent(r)};
    };
    auto overlap = [](const Part& x, const Part& o) {
        return x.at < o.end && o.at < x.end && dsa_overlap::between(x.rows, o.rows, o.at - x.at);
    };
    Part x[2], o[2];
    int n = 0;
    for (const dsa_norm_rope_rows* s : {&a.q, &a.k}) {
        if (s->H == 0) continue;
        x[n] = part(*s, s->x, s->stride_t, s->stride_h);
        o[n] = part(*s, s->out, s->out_stride_t, s->out_stride_h);
        if (dsa_overlap::within(o[n].rows) || (s->x != s->out && overlap(x[n], o[n]))) return true;
        ++n;
    }
    return n == 2 && (overlap(x[0], o[1]) || overlap(x[1], o[0]) || overlap(o[0], o[1]));
}

template <int D>
int launch_norm_rope(const dsa_qk_norm_rope_args* a, hipStream_t stream) {
    const int qg = (a->q.H + GROUP<D> - 1) / GROUP<D>, kg = (a->k.H + GROUP<D> - 1) / GROUP<D>;
    const int64_t jobs = (int64_t)a->T * (qg + kg);
    if (jobs == 0) return DSA_OK;
    if (jobs > MAX_JOBS) return DSA_ERR_BAD_SHAPE;
    if (outputs_overlap(*a)) return DSA_ERR_BAD_STRIDE;
    const dim3 grid((unsigned)((jobs + WAVES - 1) / WAVES)), block(64 * WAVES);
    if (a->rope == DSA_ROPE_INTERLEAVED)
        hipLaunchKernelGGL((dsa_qk_norm_rope_kernel<D, DSA_ROPE_INTERLEAVED>), grid, block, 0, stream, *a, qg, qg + kg);
    else if (a->rope == DSA_ROPE_HALVES)
        hipLaunchKernelGGL((dsa_qk_norm_rope_kernel<D, DSA_ROPE_HALVES>), grid, block, 0, stream, *a, qg, qg + kg);
    else
        hipLaunchKernelGGL((dsa_qk_norm_rope_kernel<D, DSA_ROPE_NONE>), grid, block, 0, stream, *a, qg, qg + kg);
    return hipGetLastError() == hipSuccess ? DSA_OK : DSA_ERR_HIP;
}

}  // namespace

extern "C" {

int dsa_qk_norm_rope(const dsa_qk_norm_rope_args* a, void* stream) {
    if (!a) return DSA_ERR_NULL_POINTER;
    if (a->T < 0 || a->B < 0 || a->n_pos < 0) return DSA_ERR_BAD_SHAPE;
    if (a->D != 128 && a->D != 512 && a->D != 576) return DSA_ERR_UNSUPPORTED;
    if (!kind_ok(a->rope)) return DSA_ERR_UNSUPPORTED;
    if (a->norm_dim < 8 || a->norm_dim > (a->D < 512 ? a->D : 512) || a->norm_dim % 8) return DSA_ERR_BAD_SHAPE;
    if (a->rot_off < 0 || a->rot_off > a->D - ROT || a->rot_off % ROT) return DSA_ERR_BAD_SHAPE;
    if (!(a->eps >= 0.0f)) return DSA_ERR_BAD_SHAPE;
    int rc = check_rows(a->q, a->T, a->D, a->rope);
    if (!rc) rc = check_rows(a->k, a->T, a->D, a->rope);
    if (rc) return rc;
    if (a->T == 0 || (a->q.H == 0 && a->k.H == 0)) return DSA_OK;
    if (a->rope != DSA_ROPE_NONE) {
        if (a->n_pos > 0 && !a->cos_sin) return DSA_ERR_NULL_POINTER;
        if (!ptr16(a->cos_sin)) return DSA_ERR_BAD_STRIDE;
    }
    if (!a->positions && (a->q_indptr || a->rope != DSA_ROPE_NONE)) {
        if (a->B == 0) return DSA_OK;        // rows of no sequence
        if (!a->q_indptr || !a->seq_lens) return DSA_ERR_NULL_POINTER;
    }
    switch (a->D) {
        case 128: return launch_norm_rope<128>(a, (hipStream_t)stream);
        case 512: return launch_norm_rope<512>(a, (hipStream_t)stream);
        default: return launch_norm_rope<576>(a, (hipStream_t)stream);
    }
}

int dsa_kv_append(const dsa_kv_append_args* args, void* stream) {
    if (!args) return DSA_ERR_NULL_POINTER;
    AppendParams p;
    p.a = *args;
    dsa_kv_append_args& a = p.a;
    if (a.T < 0 || a.B < 0 || a.n_pos < 0 || a.cache_rows < 0 || a.index_rows < 0) return DSA_ERR_BAD_SHAPE;
    if (!kind_ok(a.rope) || !kind_ok(a.index_rope) || !kind_ok(a.index_norm)) return DSA_ERR_UNSUPPORTED;
    if (a.norm != DSA_NORM_NONE && a.norm != DSA_NORM_RMS) return DSA_ERR_UNSUPPORTED;
    if (a.norm == DSA_NORM_NONE && a.weight) return DSA_ERR_UNSUPPORTED;
    if (a.index_norm == DSA_NORM_NONE && (a.index_weight || a.index_bias)) return DSA_ERR_UNSUPPORTED;
    if (a.kv_format < DSA_KV_BF16 || a.kv_format > DSA_KV_MXFP8_V4) return DSA_ERR_BAD_FORMAT;
    if (!(a.eps >= 0.0f) || !(a.index_eps >= 0.0f)) return DSA_ERR_BAD_SHAPE;
    if (a.block_table) {
        if (a.block_size < 1 || a.table_blocks < 0 || (int64_t)a.block_size * a.table_blocks > INT32_MAX)
            return DSA_ERR_BAD_SHAPE;
        if (a.block_table_stride < 0) return DSA_ERR_BAD_STRIDE;
    } else {
        if (a.kv_batch_stride < 0 || (a.kv_batch_stride == 0 && a.B > 1)) return DSA_ERR_BAD_STRIDE;
    }
    if (a.T == 0 || a.B == 0 || (!a.kv && !a.index_k)) return DSA_OK;
    if (!a.q_indptr || !a.seq_lens) return DSA_ERR_NULL_POINTER;
    const bool rotates = (a.kv && a.rope != DSA_ROPE_NONE) || (a.index_k && a.index_rope != DSA_ROPE_NONE);
    if (rotates && a.n_pos > 0 && !a.cos_sin) return DSA_ERR_NULL_POINTER;
    if (!ptr16(a.cos_sin)) return DSA_ERR_BAD_STRIDE;
    if (a.kv) {
        const bool bf16 = a.kv_format == DSA_KV_BF16 || a.kv_format == DSA_KV_BF16_D512;
        const bool streams = a.kv_format == DSA_KV_MXFP8 || a.kv_format == DSA_KV_MXFP8_V4;
        const bool scales = a.kv_format == DSA_KV_MXFP8;
        const int64_t least = a.kv_format == DSA_KV_BF16 ? 576 : a.kv_format == DSA_KV_FP8_656 ? 656 : 512;
        if (a.stride_row == 0) a.stride_row = least;
        if (a.scale_stride_row == 0) a.scale_stride_row = 16;
        if (a.rope_stride_row == 0) a.rope_stride_row = ROT;
        if (a.cache_rows > 0 && (!a.cache || (streams && !a.cache_rope) || (scales && !a.cache_scale)))
            return DSA_ERR_NULL_POINTER;
        if (a.stride_row < least || a.stride_row % (bf16 ? 8 : 16)) return DSA_ERR_BAD_STRIDE;
        if (streams && (a.rope_stride_row < ROT || a.rope_stride_row % 8)) return DSA_ERR_BAD_STRIDE;
        if (scales && (a.scale_stride_row < 16 || a.scale_stride_row % 16)) return DSA_ERR_BAD_STRIDE;
        if (a.kv_stride_t < 0 || a.kv_stride_t % 8) return DSA_ERR_BAD_STRIDE;
        if (!ptr16(a.kv) || !ptr16(a.weight) || !ptr16(a.cache) || (streams && !ptr16(a.cache_rope)) ||
            (scales && !ptr16(a.cache_scale)))
            return DSA_ERR_BAD_STRIDE;
    }
    if (a.index_k) {
        if (a.index_stride_row == 0) a.index_stride_row = 128;
        if (a.index_rows > 0 && !a.index_cache) return DSA_ERR_NULL_POINTER;
        if (a.index_stride_row < 128 || a.index_stride_row % 8 || a.index_stride_t < 0 || a.index_stride_t % 8)
            return DSA_ERR_BAD_STRIDE;
        if (!ptr16(a.index_k) || !ptr16(a.index_weight) || !ptr16(a.index_bias) || !ptr16(a.index_cache))
            return DSA_ERR_BAD_STRIDE;
    }
    p.pages = dsa_seq::make_pages(a.block_table, a.block_table_stride, a.table_blocks, a.block_size, a.kv_batch_stride);
    const int latent = a.kv ? a.T : 0;
    const int64_t jobs = (int64_t)latent + (a.index_k ? ((int64_t)a.T + 3) / 4 : 0);
    if (jobs > MAX_JOBS) return DSA_ERR_BAD_SHAPE;
    hipLaunchKernelGGL(dsa_kv_append_kernel, dim3((unsigned)((jobs + WAVES - 1) / WAVES)), dim3(64 * WAVES), 0,
                       (hipStream_t)stream, p, latent);
    return hipGetLastError() == hipSuccess ? DSA_OK : DSA_ERR_HIP;
}

}  // extern "C"
