// kv4_decode.cuh - one token of each sequence over the 4-bit cache.
#pragma once

#include "kv4.cuh"
#include "rope_rows.cuh"

namespace lg {

struct Kv4DecodeArgs {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    void* out;
    void *k_rows, *v_rows;
    const float *q_gamma, *k_gamma;
    const double* turns;
    const int* pos_rows;
    int pos, n_rows, q_heads, kv_heads, pairs, norm, n_context, layout, rows_type;
    float eps, magnitude, scale;
    int window, sinks;
    uint8_t* tiles;  // first tile of (layer, sequence 0, head 0)
    long long tiles_per_head;
    int* err;
};

// Error word of the status call, beside the waits' codes: a decode position beyond the context.
enum : int { KERR_POSITION = 16 };

// One head's 8 elements a lane (D/8 lanes, the same in every group of lanes): norm and rotation.
template <int D>
__device__ __forceinline__ void rope_head8(float (&x)[8], int l, const float* gamma, int norm, float eps,
                                           const float2* cs, int pairs, int layout, float* xs) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        ss = head_sum<D / 8>(ss);
        const float rs = 1.0f / sqrtf(ss / static_cast<float>(D) + eps);
        float g[8];
        load8(gamma + l * 8, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (x[i] * rs) * g[i];
    }
    const int group = (threadIdx.x & 31) / (D / 8);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) xs[group * D + l * 8 + i] = x[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = 8 * l + i;
        if (e < 2 * pairs) {
            const bool low = layout == 0 ? !(e & 1) : e < pairs;
            const int other = layout == 0 ? e ^ 1 : low ? e + pairs : e - pairs;
            const float2 w = cs[layout == 0 ? e >> 1 : low ? e : e - pairs];
            x[i] = x[i] * w.x + (low ? -xs[group * D + other] : xs[group * D + other]) * w.y;
        }
    }
    __syncwarp();
}

template <typename T>
__device__ __forceinline__ void store_rows8(void* rows, int type, long long at, const float (&y)[8]) {
    if (type == 0)
        store8(static_cast<float*>(rows) + at, y);
    else if (type == 1)
        store8(static_cast<__half*>(rows) + at, y);
    else
        store8(static_cast<__nv_bfloat16*>(rows) + at, y);
}

// Block (KV head, row): 8 warps walk the visible positions in turn, one position at a time, each with its
// own running maximum and sums; then they are joined.
template <typename In, int D, int NREP>
__global__ void __launch_bounds__(256) kv4_decode_kernel(const Kv4DecodeArgs a) {
    constexpr int L = D / 8;
    __shared__ float2 cs[D / 2];
    __shared__ float qs[NREP][D], kn[D], vn[D], xs[8][256];
    __shared__ float wm[8][NREP], wl[8][NREP], wo[8][NREP][D];
    const int g = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pos = a.pos_rows ? a.pos_rows[r] : a.pos;
    const bool over = pos >= a.n_context;
    const int l = lane % L;
    uint8_t* head_tiles = a.tiles + (static_cast<long long>(r) * a.kv_heads + g) * a.tiles_per_head * Kv4<D>::kTileBytes;
    In* out = static_cast<In*>(a.out) + (static_cast<long long>(r) * a.q_heads + g * NREP) * D;
    if (pos < 0 || over) {
        if (over && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = KERR_POSITION;
        const float z[8] = {};
        for (int u = threadIdx.x; u < NREP * L; u += 256) store8(out + u * 8, z);
        if (threadIdx.x < L) {
            const long long at = (static_cast<long long>(r) * a.kv_heads + g) * D + threadIdx.x * 8;
            if (a.k_rows) store_rows8<In>(a.k_rows, a.rows_type, at, z);
            if (a.v_rows) store_rows8<In>(a.v_rows, a.rows_type, at, z);
        }
        return;
    }
    for (int i = threadIdx.x; i < a.pairs; i += 256) cs[i] = rope_turn(a.turns, i, pos, a.magnitude);
    __syncthreads();
    for (int job = warp; job < NREP + 2; job += 8) {
        const bool isq = job < NREP;
        const In* src = isq         ? static_cast<const In*>(a.q) + r * a.q_stride + (g * NREP + job) * D
                        : job == NREP ? static_cast<const In*>(a.k) + r * a.k_stride + g * D
                                      : static_cast<const In*>(a.v) + r * a.v_stride + g * D;
        float x[8];
        load8(src + l * 8, x);
        if (job <= NREP) rope_head8<D>(x, l, isq ? a.q_gamma : a.k_gamma, a.norm, a.eps, cs, a.pairs, a.layout, xs[warp]);
        float* dst = isq ? qs[job] : job == NREP ? kn : vn;
        if (lane < L)
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[l * 8 + i] = x[i] * (isq ? a.scale : 1.f);
        if (!isq) {
            uint32_t codes;
            const __half d = kv4_quantize8(x, codes);
            if (lane < L) {
                uint8_t* tile = head_tiles + static_cast<long long>(pos / kKv4Tile) * Kv4<D>::kTileBytes;
                if (job == NREP)
                    kv4_store8<D, false>(tile, pos % kKv4Tile, l, codes, d);
                else
                    kv4_store8<D, true>(tile, pos % kKv4Tile, l, codes, d);
                void* rows = job == NREP ? a.k_rows : a.v_rows;
                if (rows) {
                    float y[8];
                    kv4_values8(codes, d, y);
                    store_rows8<In>(rows, a.rows_type, (static_cast<long long>(r) * a.kv_heads + g) * D + l * 8, y);
                }
            }
        }
    }
    __syncthreads();
    constexpr int E = D / 32;
    float m[NREP], ls[NREP], o[NREP][E];
#pragma unroll
    for (int h = 0; h < NREP; ++h) {
        m[h] = -INFINITY, ls[h] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[h][e] = 0.f;
    }
    const int first = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const int sinks = a.window ? min(a.sinks, first) : 0;
    const int count = sinks + (pos - first) + 1;  // the last is the token itself
    for (int i = warp; i < count; i += 8) {
        const int j = i < sinks ? i : first + (i - sinks);
        float kx[E], vx[E];
        if (i == count - 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) kx[e] = kn[lane * E + e], vx[e] = vn[lane * E + e];
        } else {
            const uint8_t* tile = head_tiles + static_cast<long long>(j / kKv4Tile) * Kv4<D>::kTileBytes;
            const int p = j % kKv4Tile;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int el = lane * E + e, sc = 2 * (p * Kv4<D>::kGroups + el / 32);
                const int kc = tile[kv4_key_byte(p, el >> 1)] >> (4 * (el & 1)) & 15;
                const int vc = tile[Kv4<D>::kCodes + kv4_value_byte(p, el >> 1)] >> (4 * (el & 1)) & 15;
                kx[e] = (kc - 8) * __half2float(*reinterpret_cast<const __half*>(tile + Kv4<D>::kKeyScales + sc));
                vx[e] = (vc - 8) * __half2float(*reinterpret_cast<const __half*>(tile + Kv4<D>::kValueScales + sc));
            }
        }
#pragma unroll
        for (int h = 0; h < NREP; ++h) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(kx[e], qs[h][lane * E + e], s);
            s = warp_sum(s);
            const float mn = fmaxf(m[h], s), c = m[h] == -INFINITY ? 0.f : expf(m[h] - mn), w = expf(s - mn);
            m[h] = mn;
            ls[h] = ls[h] * c + w;
#pragma unroll
            for (int e = 0; e < E; ++e) o[h][e] = fmaf(w, vx[e], o[h][e] * c);
        }
    }
#pragma unroll
    for (int h = 0; h < NREP; ++h) {
        wm[warp][h] = m[h], wl[warp][h] = ls[h];
#pragma unroll
        for (int e = 0; e < E; ++e) wo[warp][h][lane * E + e] = o[h][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NREP * D; i += 256) {
        const int h = i / D;
        float M = -INFINITY, s = 0.f, t = 0.f;
        for (int w = 0; w < 8; ++w) M = fmaxf(M, wm[w][h]);
        for (int w = 0; w < 8; ++w) {
            const float c = wm[w][h] == -INFINITY ? 0.f : expf(wm[w][h] - M);
            s = fmaf(wl[w][h], c, s);
            t = fmaf(wo[w][h][i % D], c, t);
        }
        out[i] = KvTraits<In>::from_float(t / s);
    }
}

}  // namespace lg
