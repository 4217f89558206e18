// Launch interface of the token-step operators (include/hipvoc_ops.h states what they compute).  Host code (ops.inc.cpp) has checked the
// arguments; everything only the device can see (page numbers, lengths, offsets) is checked by the kernels, which never follow a bad one.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hipvoc_ops.h"
#include "ops_index.hpp"

namespace hipvoc {

// bits of the deferred error word of a handle
enum OpsErr { OPS_ERR_POSITION = 1, OPS_ERR_PAGE = 2, OPS_ERR_LENGTH = 4 };

hipError_t launch_take_error(int *err, int word, hipStream_t s);      // err[word] = err[0], err[0] = 0

struct KvMoveArgs {
    hipvoc_kv_cache c;
    hipvoc_kv_rows r;
    int page_shift;
    void *k, *v;                  // the call's rows: source of a write, destination of a read
    int64_t k_stride, v_stride;
    int dtype, n_rows;
    int *err;
};
hipError_t launch_kv_write(const KvMoveArgs &a, hipStream_t s);
hipError_t launch_kv_read(const KvMoveArgs &a, hipStream_t s);

struct AttnArgs {
    hipvoc_kv_cache c;
    int page_shift;
    const void *q;
    void *out;
    float *lse;
    int64_t q_stride, out_stride;
    int dtype, n_heads, group;           // group: query heads per key head
    const int32_t *table;
    int64_t table_stride;
    int table_width;
    const int32_t *lens;
    int n_seqs, max_len, window;
    float scale_log2;                    // scale * log2(e): softmax in powers of two
    // the plan (ops_index.hpp)
    int heads, workers, least;           // pairs per sequence; 0 workers: a workgroup per pair, nothing to join
    float *part;                         // slots [workers + n_seqs * heads][query heads of a pair][head_dim], then (m, l) of each
    int64_t *before;                     // [n_seqs + 1] tiles (of one pair) before each sequence
    int *err;
};
hipError_t launch_attention_decode(const AttnArgs &a, hipStream_t s);

struct NormArgs {
    const void *x, *residual, *weight;
    void *sum, *y;
    float *scales;
    int64_t x_stride, residual_stride, sum_stride, y_stride;
    int dtype, out_dtype, group;         // group 0: the row
    float eps;
    int rows, cols;
};
hipError_t launch_add_rmsnorm(const NormArgs &a, hipStream_t s);

struct Q4Args {
    const uint8_t *codes;
    const void *scales, *mins;
    int n_out, n_in, group;
    const void *x;
    int64_t x_stride;
    int x_dtype;
    const float *x_scale;
    int x_groups;
    void *y;
    int64_t y_stride;
    int y_dtype, n_rows;
};
hipError_t launch_q4_matvec(const Q4Args &a, hipStream_t s);

}  // namespace hipvoc
