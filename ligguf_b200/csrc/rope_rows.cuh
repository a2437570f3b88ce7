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
    int parts;       // blocks of a token
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

// What a head's elements are multiplied by, from the sum of their squares.  (One rounding: 1 / sqrtf has two, a 2-norm
// error of 8.5e-8 in place of 7.5e-8, and takes the prompts' kernel from 33 to 41.7 us for 7777 tokens.)
template <int D>
__device__ __forceinline__ float rms_factor(float ss, float eps) {
    return rsqrtf(fmaf(ss, 1.0f / D, eps));
}
// The rotation of a pair (a, b) by w = (cos, sin), with its roundings spelt out: both kernels that write the cache take
// these and rms_factor, so that a key is the same there whether it came with a prompt or alone.  (rope_pairs_kernel,
// which writes none, leaves the roundings to the compiler: 32.8 us for its prompt, 38.7 with these.)
__device__ __forceinline__ float rope_first(float a, float b, float2 w) { return fmaf(a, w.x, -__fmul_rn(b, w.y)); }
__device__ __forceinline__ float rope_second(float a, float b, float2 w) { return fmaf(b, w.x, __fmul_rn(a, w.y)); }

// Layouts of the rotation: adjacent pairs lie within a thread; halves whose distance is a whole number
// of units are exchanged by a shuffle, others through shared memory.
enum : int { kRopeAdjacent = 0, kRopeHalves = 1, kRopeHalvesOdd = 2 };

// The place of pair i's cosine and sine in a token's table: threads of neighbouring units read neighbouring entries
// (an entry of two pairs, read as 16 bytes).
__device__ __forceinline__ int rope_slot(int i) { return ((i & 7) >> 1) * 16 + (i >> 3) * 2 + (i & 1); }

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
            const float rs = rms_factor<D>(ss, a.eps);
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
                    const float2 w = cs[rope_slot(4 * l + i)];
                    const float x0 = x[2 * i], x1 = x[2 * i + 1];
                    x[2 * i] = rope_first(x0, x1, w);
                    x[2 * i + 1] = rope_second(x0, x1, w);
                }
    } else if constexpr (kLayout == kRopeHalves) {
        const int hl = a.pairs / 8;  // units of a half
        const bool low = l < hl;
        const int from = low ? l + hl : l - hl;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(0xffffffffu, x[i], from & (L - 1), L);
            if (kind < 2 && l < 2 * hl) {
                const float2 w = cs[rope_slot(8 * (low ? l : l - hl) + i)];
                x[i] = low ? rope_first(x[i], other, w) : rope_second(other, x[i], w);
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
                    const float2 w = cs[rope_slot(low ? e : e - a.pairs)];
                    const float other = hx[low ? e + a.pairs : e - a.pairs];
                    x[i] = low ? rope_first(x[i], other, w) : rope_second(other, x[i], w);
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

// Two units of a head that one thread takes together: the halves of eight rotated pairs (or, past the rotated
// part and for adjacent pairs, neighbours), so a rotation needs no exchange and reads its table once.
template <int D, int kLayout>
__device__ __forceinline__ int2 rope_two_units(int dl, int pairs) {
    if (kLayout == kRopeHalves) {
        const int hl = pairs / 8;
        if (dl < hl) return make_int2(dl, dl + hl);
    }
    return make_int2(2 * dl, 2 * dl + 1);  // (past the rotated part: 2 hl + 2 (dl - hl))
}

// Heads that are normed and rotated: block (token, part), a pair of units of kTake heads a thread.  Bound by the bytes
// of the rows, each read and written once, if only enough of them are on their way.  What a thread does hangs on its
// loads, the token's rotations (fp64, then sine and cosine: hidden by the loads) and a barrier, so it takes about as many
// heads as 64 registers hold: one of 32 bits, two of 16, with 24 to 72 bytes of spills.  7777 tokens of 40 heads in fp16:
// 33 us (4.9 TB/s; 28 without the norm); one head a thread 43, four heads, whose registers halve the threads, 36; blocks that stay and are fed by
// bulk copies into shared memory 35 to 37: shared memory's rate bounds them.
template <typename In, typename Out, int D, int kLayout, int kTake>
__global__ void __launch_bounds__(256, 4) rope_pairs_kernel(const RopeRowsArgs a) {
    constexpr int L = D / 8, DL = L / 2;
    __shared__ __align__(16) float2 cs[64];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (a kernel that needs these results waits for them)
    const long long tok = blockIdx.x / a.parts;
    const int pos = a.pos ? a.pos[tok] : a.pos0 + static_cast<int>(tok);
    const int item = blockIdx.x % a.parts * blockDim.x + threadIdx.x;
    auto table = [&]() {
        if (threadIdx.x < 64)
            cs[rope_slot(threadIdx.x)] = static_cast<int>(threadIdx.x) < a.pairs ? rope_turn(a.turns[threadIdx.x], pos, a.magnitude) : make_float2(1.f, 0.f);
        __syncthreads();
    };  // (whole warps: pair_items is a multiple of 32)
    const int qh = a.q ? a.q_heads : 0, heads = qh + a.kv_heads;
    // Heads h0, h0 + step, .. below end: queries' or keys', never both, so that a thread has one set of norm weights.
    const int dl = item % DL, of = item / DL, q_step = (qh + kTake - 1) / kTake, k_step = (heads - qh + kTake - 1) / kTake;
    const bool keys = of >= q_step, live = of < q_step + k_step;
    const int h0 = keys ? qh + of - q_step : of, step = keys ? k_step : q_step, end = live ? (keys ? heads : qh) : 0;
    const int2 two = rope_two_units<D, kLayout>(dl, a.pairs);
    const In* src = keys ? static_cast<const In*>(a.k) + tok * a.k_stride - qh * D : static_cast<const In*>(a.q) + tok * a.q_stride;
    Units<In> x[kTake][2];
#pragma unroll
    for (int n = 0; n < kTake; ++n) {
        const int h = h0 + n * step;
        if (h < end) {
            x[n][0].load(src + h * D + two.x * 8);
            x[n][1].load(src + h * D + two.y * 8);
        } else {
            x[n][0].zero();
            x[n][1].zero();
        }
    }
    float g[16];
    auto weights = [&]() {
        const float4* gamma = reinterpret_cast<const float4*>(keys ? a.k_gamma : a.q_gamma);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 u = gamma[two.x * 2 + i], v = gamma[two.y * 2 + i];
            g[4 * i] = u.x, g[4 * i + 1] = u.y, g[4 * i + 2] = u.z, g[4 * i + 3] = u.w;
            g[8 + 4 * i] = v.x, g[9 + 4 * i] = v.y, g[10 + 4 * i] = v.z, g[11 + 4 * i] = v.w;
        }
    };
    if (kTake > 1 && a.norm && live) weights();
    table();
    if (kTake == 1 && a.norm && live) weights();  // (later: fewer registers)
    float rs[kTake];
    if (a.norm) {  // the heads' sums side by side: their exchanges wait for one another's results otherwise
#pragma unroll
        for (int n = 0; n < kTake; ++n) {
            float p[8], r[8], s0 = 0.f, s1 = 0.f;
            x[n][0].get(p);
            x[n][1].get(r);
#pragma unroll
            for (int i = 0; i < 8; ++i) s0 = fmaf(p[i], p[i], s0), s1 = fmaf(r[i], r[i], s1);
            rs[n] = s0 + s1;
        }
#pragma unroll
        for (int o = 1; o < DL; o <<= 1)
#pragma unroll
            for (int n = 0; n < kTake; ++n) rs[n] += __shfl_xor_sync(0xffffffffu, rs[n], o);
#pragma unroll
        for (int n = 0; n < kTake; ++n) rs[n] = rms_factor<D>(rs[n], a.eps);
    }
    float4 w[4];  // two rotations each
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = kLayout == kRopeAdjacent || dl < a.pairs / 8 ? *reinterpret_cast<const float4*>(cs + rope_slot(8 * dl + 2 * i))
                                                            : make_float4(1.f, 0.f, 1.f, 0.f);
    Out* dst = keys ? static_cast<Out*>(a.k_out) + tok * a.k_out_stride - qh * D : static_cast<Out*>(a.q_out) + tok * a.q_out_stride;
#pragma unroll
    for (int n = 0; n < kTake; ++n) {
        const int h = h0 + n * step;
        float p[8], r[8];
        x[n][0].get(p);
        x[n][1].get(r);
        if (a.norm)
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = (p[i] * rs[n]) * g[i], r[i] = (r[i] * rs[n]) * g[8 + i];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float4 v = w[i / 2];
            float& a0 = kLayout == kRopeHalves ? p[i] : i < 4 ? p[2 * i] : r[2 * i - 8];
            float& b0 = kLayout == kRopeHalves ? r[i] : i < 4 ? p[2 * i + 1] : r[2 * i - 7];
            float& a1 = kLayout == kRopeHalves ? p[i + 1] : i < 4 ? p[2 * i + 2] : r[2 * i - 6];
            float& b1 = kLayout == kRopeHalves ? r[i + 1] : i < 4 ? p[2 * i + 3] : r[2 * i - 5];
            const float x0 = a0, y0 = b0, x1 = a1, y1 = b1;
            a0 = x0 * v.x - y0 * v.y;
            b0 = x0 * v.y + y0 * v.x;
            a1 = x1 * v.z - y1 * v.w;
            b1 = x1 * v.w + y1 * v.z;
        }
        if (h < end) {
            store8(dst + h * D + two.x * 8, p);
            store8(dst + h * D + two.y * 8, r);
        }
    }
}

// Heads that are quantized too, and with them the others of the call; and halves that are not whole units apart: a
// unit a thread, in 32 registers.  Block (token, part of its units).  A prompt of 2048 tokens of 48 heads in fp32 (32 rotated, 16
// quantized): 19.6 us, 4.0 TB/s; keys and values by tiles of the cache, their codes put together in shared memory, and
// the queries by rope_pairs_kernel beside them took 23 to 25.
template <typename In, typename Out, int D, int kLayout>
__global__ void __launch_bounds__(256) rope_units_kernel(const RopeRowsArgs a) {
    constexpr int L = D / 8;  // units (lanes) of a head
    __shared__ __align__(16) float2 cs[64];
    __shared__ float xch[kLayout == kRopeHalvesOdd ? 256 * 8 : 1];
    const long long tok = blockIdx.x / a.parts;
    const int part = blockIdx.x % a.parts;
    const int pos = a.pos ? a.pos[tok] : a.pos0 + static_cast<int>(tok);
    for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) cs[rope_slot(i)] = rope_turn(a.turns[i], pos, a.magnitude);
    __syncthreads();
    const int q_units = a.q ? a.q_heads * L : 0, k_units = a.kv_heads * L;
    const int u1 = min(q_units + k_units + (a.v ? k_units : 0), (part + 1) * a.units_per_block);
    // Whole warps stay together: the shuffles need every lane (units past the end work on zeros).
    for (int u0 = part * a.units_per_block + static_cast<int>(threadIdx.x & ~31); u0 < u1; u0 += blockDim.x) {
        const int u = u0 + (threadIdx.x & 31);
        float x[8] = {};
        if (u < u1) {
            const In* src = u < q_units ? static_cast<const In*>(a.q) + tok * a.q_stride + u * 8
                            : u < q_units + k_units ? static_cast<const In*>(a.k) + tok * a.k_stride + (u - q_units) * 8
                                                    : static_cast<const In*>(a.v) + tok * a.v_stride + (u - q_units - k_units) * 8;
            load8(src, x);
        }
        rope_rows_unit<In, Out, D, kLayout>(a, tok, pos, u, u < u1, q_units, k_units, x, cs, xch);
    }
}

}  // namespace lg
