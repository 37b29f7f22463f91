// What the calls that write the paged 8-bit cache share (kvcache.hip, rope.hip).
#pragma once

#include "quant8.h"

namespace nnc {

struct KvArgs {
    Ragged g;
    int8_t *k, *v;
    float *k_scale, *v_scale;
    void *k_rows, *v_rows;
    int64_t k_ld, v_ld;
    int k_col, v_col, kv_heads, dim;
};

// false with an error recorded
bool kv_args(const char* name, Tensor* k, Tensor* v, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale,
             Tensor* v_scale, Tensor* table, Tensor* starts, Tensor* lengths, int k_col, int v_col, KvArgs* a);
// nnc_hip_kv_write's kernels for arguments that are in order, rows not 0
void launch_write(const char* name, bool f16, const KvArgs& a);

}  // namespace nnc
