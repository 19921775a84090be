// Host build of opfoundry_amd/csrc/dsa_seq.h (the chunk operators' rules of sequences, pages and
// blocks) for tests/test_chunk_cpu.py: the two HIP qualifiers are defined empty, so g++ compiles
// exactly the functions the device code runs.
#define __host__
#define __device__
#include "../../opfoundry_amd/csrc/dsa_seq.h"

extern "C" {

int64_t seq_row(const int32_t* table, int64_t table_stride, int32_t blocks, int32_t block_size, int64_t batch_stride,
                int32_t b, int64_t p, int64_t rows) {
    return dsa_seq::row_of(dsa_seq::make_pages(table, table_stride, blocks, block_size, batch_stride), b, p, rows);
}
int64_t seq_position(const int32_t* indptr, const int32_t* lens, int32_t b, int32_t t) {
    return dsa_seq::position_of(indptr, lens, b, t);
}
int32_t seq_common(int32_t H, int32_t m) { return dsa_seq::common(H, m); }
int64_t seq_block_start(int64_t indptr, int32_t b, int32_t H, int32_t m) {
    return dsa_seq::block_start(indptr, b, H, m, dsa_seq::common(H, m));
}
int32_t seq_parts(int32_t a, int32_t b, float reciprocal) { return dsa_seq::parts_by(a, b, reciprocal); }

}  // extern "C"
