// window.cuh - causal attention with a sliding window and first tokens that stay visible.
#pragma once

#include "common.cuh"

namespace lg {

struct WindowArgs {
    const void *q, *k, *v;
    void* out;
    long long q_stride, k_stride, v_stride, q_batch, k_batch, v_batch;
    const int *pos0, *lens;
    int batch, n, m, q_heads, kv_heads, window, sinks;
    float scale_log2;  // of the scores, times log2(e)
};

}  // namespace lg
