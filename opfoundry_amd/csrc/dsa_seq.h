// dsa_seq.h - which sequence and position a chunk's token has, and which cache
// row a position has: the rules of include/dsa_chunk.h, for the kernels (device)
// and their CPU test (host).
//
// hipcc compiles these for host and device; a host-only test defines
// __host__ and __device__ as empty before including this file.
#ifndef DSA_SEQ_H_
#define DSA_SEQ_H_

#include <stdint.h>

namespace dsa_seq {

// The pages of a call.  One cache row per (sequence, position).
struct Pages {
    const int32_t* table;      // NULL: flat
    int64_t table_stride;
    int64_t batch_stride;      // flat: rows of a sequence (0: every sequence starts at row 0)
    int64_t limit;             // positions at or past it have no row
    int32_t block_size, shift; // shift = log2(block_size) for a power of two, else -1
};

__host__ __device__ inline Pages make_pages(const int32_t* table, int64_t table_stride, int32_t table_blocks,
                                            int32_t block_size, int64_t batch_stride) {
    Pages g;
    g.table = table;
    g.table_stride = table_stride;
    g.batch_stride = batch_stride;
    g.block_size = block_size;
    g.shift = -1;
    for (int s = 0; s < 31; ++s)
        if (block_size == (1 << s)) g.shift = s;
    g.limit = table ? (int64_t)table_blocks * block_size : (batch_stride > 0 ? batch_stride : INT64_MAX);
    return g;
}

// Cache row of position p of sequence b, or -1 where it has none inside [0, rows).
__host__ __device__ inline int64_t row_of(const Pages& g, int32_t b, int64_t p, int64_t rows) {
    if (p < 0 || p >= g.limit) return -1;
    int64_t row;
    if (g.table) {
        const int32_t q = (int32_t)p;         // below table_blocks * block_size, which the host keeps in 31 bits
        const int32_t blk = g.shift >= 0 ? q >> g.shift : q / g.block_size;
        row = (int64_t)g.table[(int64_t)b * g.table_stride + blk] * g.block_size + (q - blk * g.block_size);
    } else {
        row = (int64_t)b * g.batch_stride + p;
    }
    return row >= 0 && row < rows ? row : -1;
}

// Position of token t (in sequence b) of the chunk.
__host__ __device__ inline int64_t position_of(const int32_t* indptr, const int32_t* lens, int32_t b, int32_t t) {
    return (int64_t)lens[b] - indptr[b + 1] + t;
}

// Blocks of `m` rows that a grid gives sequence b, whose tokens have H rows each: sequence b
// starts at block_start(b), its own blocks come first among those up to block_start(b + 1), and
// the grid has block_start(B) of them, which needs no count of the sequences before it.  With
// g = gcd(H, m) a sequence's rows are a multiple of g, so that it leaves at most m - g of its
// last block unused, and that much is added for each: with A = indptr_b H + b (m - g),
// floor((A + n H + m - g) / m) - floor(A / m) >= ceil(n H / m).  (A whole block for each would
// leave every second block of single tokens with H = m empty, and with them every second XCD.)
__host__ __device__ inline int32_t common(int32_t H, int32_t m) {
    while (m) {
        const int32_t r = H % m;
        H = m;
        m = r;
    }
    return H;
}
__host__ __device__ inline int64_t block_start(int64_t indptr_b, int32_t b, int32_t H, int32_t m, int32_t g) {
    return (indptr_b * H + (int64_t)b * (m - g)) / m;
}

// ceil(a / b) of 0 <= a < 2^31 and 1 <= b <= 2^26 by a reciprocal of b that is off by at most 2^-23 of
// itself: exact where it is below 2^20, else at least that and at most 2^-19 more.  (Rounding a, b, the
// reciprocal and the product moves the quotient by less than 2^-21 of itself: below 2^20 its floor is then
// off by one at most, and two steps reach the ceiling; above, the share added first outweighs it.)
__host__ __device__ inline int32_t parts_by(int32_t a, int32_t b, float reciprocal) {
    uint32_t q = (uint32_t)((float)a * reciprocal);
    q += q >> 20;
    q += q * (uint32_t)b < (uint32_t)a ? 1 : 0;
    q += q * (uint32_t)b < (uint32_t)a ? 1 : 0;
    return (int32_t)q;
}

}  // namespace dsa_seq

#endif  // DSA_SEQ_H_
