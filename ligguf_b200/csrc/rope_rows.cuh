// rope_rows.cuh - one pass over the rows of a layer's projections: per-head RMS norm, rotation by
// position and, for the 4-bit cache, quantization.
//
//   y = x / sqrt(mean(x^2) + eps) * gamma
//   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),  t = position * f_i
//
// The angle is formed in fp64 as a number of turns, position * f_i / 2pi, of which the whole turns drop
// exactly; what is left goes to fp32 sine and cosine.  (Formed in fp32, the angle of position 100000
// is off by up to 0.004 radians.)
//
// A thread holds 8 consecutive elements of a head (a "unit"), D/8 lanes a head, so the sum of squares
// and a quantized block's extremes are shuffles within 16 (8) and 4 lanes.
#pragma once

#include "common.cuh"
#include "kv4.cuh"

namespace lg {

struct RopeRowsArgs {
    const void *q, *k, *v;  // q or v may be null (no queries / no cache)
    long long q_stride, k_stride, v_stride;
    void *q_out, *k_out;  // rotated rows; null where not wanted
    long long q_out_stride, k_out_stride;
    const float *q_gamma, *k_gamma;
    const double* turns;  // [pairs] turns per position
    const int* pos;       // positions, or null: pos0 + token
    int n, pos0, q_heads, kv_heads, pairs, norm;
    float eps, magnitude;
    // 4-bit cache (tiles null: none)
    uint8_t* tiles;  // first tile of (layer, sequence, head 0)
    long long tiles_per_head;
    void *k_rows, *v_rows;  // the rows as the cache holds them, or null
    int units_per_block;
};

// cos and sin of position * f, times the magnitude; turns = f / 2pi.
__device__ __forceinline__ float2 rope_turn(double turns, int pos, float magnitude) {
    const double t = static_cast<double>(pos) * turns;
    float s, c;
    sincospif(static_cast<float>(2.0 * (t - rint(t))), &s, &c);
    return make_float2(magnitude * c, magnitude * s);
}

// Sum over the 2^k lanes of a head.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Layouts of the rotation: adjacent pairs lie within a thread; halves whose distance is a whole number
// of units are exchanged by a shuffle, others through shared memory.
enum : int { kRopeAdjacent = 0, kRopeHalves = 1, kRopeHalvesOdd = 2 };

// Where the table in shared memory holds pair i: threads of neighbouring units read neighbouring entries.
template <int kLayout>
__device__ __forceinline__ int rope_slot(int i) {
    return kLayout == kRopeAdjacent ? (i & 3) * 16 + (i >> 2) : (i & 7) * 8 + (i >> 3);
}

// 8 elements of a row as they were loaded.
template <typename T>
struct Units {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) v[i] = *(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) KvTraits<T>::unpack(v[i], x + i * KvTraits<T>::kElemsPer16B);
    }
};

// One unit of a token: norm, rotation, and its stores.  Warp-collective.
template <typename In, typename Out, int D, int kLayout>
__device__ __forceinline__ void rope_rows_unit(const RopeRowsArgs& a, long long tok, int pos, int u, bool live, int q_units,
                                               int k_units, float (&x)[8], const float2* cs, float* xch) {
    constexpr int L = D / 8;
    const int kind = u < q_units ? 0 : u < q_units + k_units ? 1 : 2;  // q, k, v
    const int hu = u - (kind == 0 ? 0 : kind == 1 ? q_units : q_units + k_units);
    const int head = hu / L, l = hu % L;
    if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        ss = head_sum<L>(ss);
        if (kind < 2) {
            const float rs = 1.0f / sqrtf(ss / static_cast<float>(D) + a.eps);
            float g[8];
            load8((kind ? a.k_gamma : a.q_gamma) + l * 8, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (x[i] * rs) * g[i];
        }
    }
    if constexpr (kLayout == kRopeAdjacent) {
        if (kind < 2)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * l + i < a.pairs) {
                    const float2 w = cs[rope_slot<kLayout>(4 * l + i)];
                    const float x0 = x[2 * i], x1 = x[2 * i + 1];
                    x[2 * i] = x0 * w.x - x1 * w.y;
                    x[2 * i + 1] = x0 * w.y + x1 * w.x;
                }
    } else if constexpr (kLayout == kRopeHalves) {
        const int hl = a.pairs / 8;  // units of a half
        const bool low = l < hl;
        const int from = low ? l + hl : l - hl;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(0xffffffffu, x[i], from & (L - 1), L);
            if (kind < 2 && l < 2 * hl) {
                const float2 w = cs[rope_slot<kLayout>(8 * (low ? l : l - hl) + i)];
                x[i] = x[i] * w.x + (low ? -other : other) * w.y;
            }
        }
    } else {
        float* xs = xch + (threadIdx.x & ~31) * 8;  // this warp's heads
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) xs[(threadIdx.x & 31) * 8 + i] = x[i];
        __syncwarp();
        const float* hx = xs + (threadIdx.x & 31 & ~(L - 1)) * 8;
        if (kind < 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = 8 * l + i;
                if (e < 2 * a.pairs) {
                    const bool low = e < a.pairs;
                    const float2 w = cs[rope_slot<kLayout>(low ? e : e - a.pairs)];
                    const float other = hx[low ? e + a.pairs : e - a.pairs];
                    x[i] = x[i] * w.x + (low ? -other : other) * w.y;
                }
            }
    }
    if (kind == 0) {
        if (live && a.q_out) store8(static_cast<Out*>(a.q_out) + tok * a.q_out_stride + hu * 8, x);
    } else if (kind == 1) {
        if (live && a.k_out) store8(static_cast<Out*>(a.k_out) + tok * a.k_out_stride + hu * 8, x);
    }
    if (a.tiles && __any_sync(0xffffffffu, kind > 0)) {
        uint32_t codes;
        const __half d = kv4_quantize8(x, codes);
        if (live && kind > 0) {
            uint8_t* tile = a.tiles + (head * a.tiles_per_head + pos / kKv4Tile) * Kv4<D>::kTileBytes;
            if (kind == 1)
                kv4_store8<D, false>(tile, pos % kKv4Tile, l, codes, d);
            else
                kv4_store8<D, true>(tile, pos % kKv4Tile, l, codes, d);
            Out* rows = static_cast<Out*>(kind == 1 ? a.k_rows : a.v_rows);
            if (rows) {
                float y[8];
                kv4_values8(codes, d, y);
                store8(rows + (tok * a.kv_heads * L + hu) * 8, y);
            }
        }
    }
}

// Block (token, part of its units): a token's rotation is computed once for all its heads, with the first
// kRopeAhead units of every thread already in flight.
constexpr int kRopeAhead = 4;
template <typename In, typename Out, int D, int kLayout>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeRowsArgs a) {
    constexpr int L = D / 8;  // units (lanes) of a head
    __shared__ float2 cs[64];
    __shared__ float xch[kLayout == kRopeHalvesOdd ? 256 * 8 : 1];
    const long long tok = blockIdx.x;
    const int q_units = a.q ? a.q_heads * L : 0, k_units = a.kv_heads * L;
    const int total = q_units + k_units + (a.v ? k_units : 0);
    const int u1 = min(total, static_cast<int>(blockIdx.y + 1) * a.units_per_block);
    const int pos = a.pos ? a.pos[tok] : a.pos0 + static_cast<int>(tok);
    const int lane = threadIdx.x & 31;
    bool first = true;
    // Whole warps stay together: the shuffles below need every lane (units past the end work on zeros).
    for (int u0 = blockIdx.y * a.units_per_block + (threadIdx.x & ~31); first || u0 < u1; u0 += kRopeAhead * blockDim.x) {
        Units<In> x[kRopeAhead];
#pragma unroll
        for (int n = 0; n < kRopeAhead; ++n) {
            const int u = u0 + n * blockDim.x + lane;
            if (u < u1) {
                const In* src = u < q_units ? static_cast<const In*>(a.q) + tok * a.q_stride + u * 8
                                : u < q_units + k_units
                                    ? static_cast<const In*>(a.k) + tok * a.k_stride + (u - q_units) * 8
                                    : static_cast<const In*>(a.v) + tok * a.v_stride + (u - q_units - k_units) * 8;
                x[n].load(src);
            } else {
                x[n].zero();
            }
        }
        if (first) {
            for (int i = threadIdx.x; i < a.pairs; i += blockDim.x)
                cs[rope_slot<kLayout>(i)] = rope_turn(a.turns[i], pos, a.magnitude);
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int n = 0; n < kRopeAhead; ++n) {
            const int u = u0 + n * blockDim.x + lane;
            if (u - lane >= u1) break;
            float y[8];
            x[n].get(y);
            rope_rows_unit<In, Out, D, kLayout>(a, tok, pos, u, u < u1, q_units, k_units, y, cs, xch);
        }
    }
}

}  // namespace lg
