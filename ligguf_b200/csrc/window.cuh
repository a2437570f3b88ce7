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

// One warp a query head of a row: 32 keys at a time, a key a lane for the scores, D/32 elements a lane
// for the sum over values.
template <typename T, typename Out, int D>
__global__ void __launch_bounds__(256) window_rows_kernel(const WindowArgs a) {
    constexpr int E = D / 32;
    __shared__ float qs[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long w = blockIdx.x * 8ll + warp;
    if (w >= static_cast<long long>(a.batch) * a.n * a.q_heads) return;
    const int h = static_cast<int>(w % a.q_heads);
    const long long row = w / a.q_heads;
    const int b = static_cast<int>(row / a.n), i = static_cast<int>(row % a.n), g = h / (a.q_heads / a.kv_heads);
    const int len = max(0, min(a.lens ? a.lens[b] : a.m, a.m));
    const long long p = static_cast<long long>(a.pos0 ? a.pos0[b] : len - a.n) + i;
    const T* q = static_cast<const T*>(a.q) + b * a.q_batch + i * a.q_stride + h * D;
    const T* k = static_cast<const T*>(a.k) + b * a.k_batch + g * D;
    const T* v = static_cast<const T*>(a.v) + b * a.v_batch + g * D;
#pragma unroll
    for (int e = 0; e < E; ++e) qs[warp][lane * E + e] = KvTraits<T>::to_float(q[lane * E + e]) * a.scale_log2;
    __syncwarp();
    const int last = static_cast<int>(max(0ll, min(p + 1, static_cast<long long>(len))));  // keys below pass the causal mask
    const int first = a.window ? static_cast<int>(max(0ll, min(p - a.window + 1, static_cast<long long>(last)))) : 0;
    float m = -INFINITY, s = 0.f, o[E] = {};
    for (int part = 0; part < 2; ++part) {
        const int j0 = part ? first : 0, j1 = part ? last : min(a.window ? min(a.sinks, first) : 0, last);
        for (int jb = j0; jb < j1; jb += 32) {
            const int j = jb + lane;
            float x = -INFINITY;
            if (j < j1) {
                x = 0.f;
                const T* kr = k + j * a.k_stride;
                for (int e = 0; e < D; ++e) x = fmaf(KvTraits<T>::to_float(kr[e]), qs[warp][e], x);
            }
            const float mn = fmaxf(m, warp_max(x));
            const float c = m == -INFINITY ? 0.f : exp2f(m - mn), pr = x == -INFINITY ? 0.f : exp2f(x - mn);
            m = mn;
            s = s * c + warp_sum(pr);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= c;
            for (int t = 0; t < 32 && jb + t < j1; ++t) {
                const float pt = __shfl_sync(0xffffffffu, pr, t);
                const T* vr = v + (jb + t) * a.v_stride + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(pt, KvTraits<T>::to_float(vr[e]), o[e]);
            }
        }
    }
    Out* out = static_cast<Out*>(a.out) + w * D + lane * E;
    const float inv = s > 0.f ? 1.0f / s : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = KvTraits<Out>::from_float(o[e] * inv);
}

}  // namespace lg
