// dsa_list.h - attention of query tokens over lists of positions on DSA_KV_MXFP4
// rows: the kernels are dsa_chunk.hip's, the entry points dsa_mla.hip's.
#ifndef DSA_LIST_H_
#define DSA_LIST_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsa_list {

// The fields have the meaning (and the validated ranges) of dsa_mla_decode_args and
// dsa_mla_prefill_args; strides in elements, row_bytes in bytes.
struct Call {
    const void* q;
    int64_t q_sb, q_st, q_sh;
    const void* kv;
    int64_t rows, row_bytes;
    const int32_t* block_table;
    int64_t table_stride;
    int32_t block_size;
    int64_t batch_stride;
    const int32_t* seq_lens;       // NULL: every sequence is `len` long
    int64_t len;
    const int32_t* indices;
    int64_t idx_sb, idx_st;
    void* out;
    int64_t o_sb, o_st, o_sh;
    float* lse;
    float* part_o;                 // ns > 1: fp32 partials [split][B * s_q][H][512] and their LSE (-FLT_MAX: empty)
    float* part_lse;
    int32_t B, s_q, H, topk;
    int32_t causal;                // 1: j <= L - s_q + t, 2: j <= b + causal_offset
    int64_t causal_offset;
    float scale_log2;
    int32_t ns, per_split;         // split s takes entries [s * per_split, (s + 1) * per_split)
};

// `heads` of a workgroup: 128 or 32 (one a CU), or 16 (two a CU).  0 or DSA_ERR_HIP.
__attribute__((visibility("hidden"))) int launch(const Call& c, int heads, hipStream_t stream);

}  // namespace dsa_list

#endif  // DSA_LIST_H_
