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
    int kv_heads_per_block; // of a block that takes tiles of keys and values
    int parts;              // blocks of a token, and the units of each
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

// A prompt's keys and values: block (tile of 16 positions, a few KV heads).  A thread holds 8 elements of one
// position, the same of every head, so it forms its rotations once; a head's codes are put together in shared
// memory and leave as whole 16-byte words (byte by byte they cost more than the rest of the kernel).  Positions
// of the tile outside the prompt keep their bytes: such tiles are written byte by byte.
constexpr int kKv4AppendBlocks = 3;  // resident on an SM
constexpr int kRopePairRow = 64 + 8;  // table entries of a position: two positions of a warp in other banks
template <typename In, typename Out, int D, int kLayout>
__global__ void __launch_bounds__(256, kKv4AppendBlocks) kv4_append_kernel(const RopeRowsArgs a) {
    constexpr int L = D / 8, kHeads = 256 / (16 * L), TB = Kv4<D>::kTileBytes;  // heads at a time
    __shared__ float2 cs[16 * kRopePairRow];
    __shared__ uint4 staging[kHeads * TB / 16];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the queries' kernel needs nothing of this one's
    const int block = blockIdx.x;
    const int groups = (a.kv_heads + a.kv_heads_per_block - 1) / a.kv_heads_per_block;
    const int t0 = a.pos0 / kKv4Tile * kKv4Tile + block / groups * kKv4Tile;
    const int h0 = block % groups * a.kv_heads_per_block, h1 = min(a.kv_heads, h0 + a.kv_heads_per_block);
    const int l = threadIdx.x % L, p = threadIdx.x / L % 16, sub = threadIdx.x / (16 * L);
    const int pos = t0 + p;
    const bool live = pos >= a.pos0 && pos < a.pos0 + a.n;
    const bool whole = t0 >= a.pos0 && t0 + kKv4Tile <= a.pos0 + a.n;
    const long long tok = pos - a.pos0;
    Units<In> k, v;
    auto load = [&](int h) {
        if (live && h < h1) {
            k.load(static_cast<const In*>(a.k) + tok * a.k_stride + h * D + l * 8);
            v.load(static_cast<const In*>(a.v) + tok * a.v_stride + h * D + l * 8);
        } else {
            k.zero();
            v.zero();
        }
    };
    load(h0 + sub);
    for (int i = threadIdx.x; i < 16 * a.pairs; i += 256)
        cs[i / a.pairs * kRopePairRow + rope_slot<kLayout>(i % a.pairs)] = rope_turn(a.turns[i % a.pairs], t0 + i / a.pairs, a.magnitude);
    __syncthreads();
    // This thread's rotations: of its four pairs, or of the eight pairs it has a half of.
    constexpr int kTurns = kLayout == kRopeAdjacent ? 4 : 8;
    float2 w[kTurns];
    const int hl = a.pairs / 8;
    const bool low = l < hl;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const int pair = kLayout == kRopeAdjacent ? 4 * l + i : 8 * (low ? l : l - hl) + i;
        w[i] = (kLayout == kRopeAdjacent ? pair < a.pairs : l < 2 * hl) ? cs[p * kRopePairRow + rope_slot<kLayout>(pair)] : make_float2(1.f, 0.f);
    }
    float g[8];
    if (a.norm) load8(a.k_gamma + l * 8, g);
    uint8_t* stage = reinterpret_cast<uint8_t*>(staging) + sub * TB;
    for (int h = h0 + sub; h - sub < h1; h += kHeads) {
        float x[8], y[8];
        k.get(x);
        v.get(y);
        load(h + kHeads);
        if (a.norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
            const float rs = rsqrtf(head_sum<L>(ss) * (1.0f / D) + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (x[i] * rs) * g[i];
        }
        if constexpr (kLayout == kRopeAdjacent) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = x[2 * i], x1 = x[2 * i + 1];
                x[2 * i] = x0 * w[i].x - x1 * w[i].y;
                x[2 * i + 1] = x0 * w[i].y + x1 * w[i].x;
            }
        } else {
            const int from = (low ? l + hl : l < 2 * hl ? l - hl : l) & (L - 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float other = __shfl_sync(0xffffffffu, x[i], from, L);
                x[i] = x[i] * w[i].x + (low ? -other : other) * w[i].y;
            }
        }
        uint32_t kc, vc;
        const __half kd = kv4_quantize8(x, kc), vd = kv4_quantize8(y, vc);
        uint8_t* tile = a.tiles + (h * a.tiles_per_head + t0 / kKv4Tile) * TB;
        const bool on = live && h < h1;
        if (on) {
            uint8_t* dst = whole ? stage : tile;
            kv4_store8<D, false>(dst, p, l, kc, kd);
            kv4_store8<D, true>(dst, p, l, vc, vd);
        }
        if (whole) {
            __syncthreads();
            if (h < h1)
                for (int i = threadIdx.x % (16 * L); i < TB / 16; i += 16 * L)
                    reinterpret_cast<uint4*>(tile)[i] = reinterpret_cast<const uint4*>(stage)[i];
        }
        if (on && a.k_rows) {
            float z[8];
            kv4_values8(kc, kd, z);
            store8(static_cast<Out*>(a.k_rows) + (tok * a.kv_heads + h) * D + l * 8, z);
        }
        if (on && a.v_rows) {
            float z[8];
            kv4_values8(vc, vd, z);
            store8(static_cast<Out*>(a.v_rows) + (tok * a.kv_heads + h) * D + l * 8, z);
        }
        if (whole) __syncthreads();
    }
}

// One head's two units in p and r: norm, rotation.  Lanes of D/16 hold a head.
template <int D, int kLayout>
__device__ __forceinline__ void rope_two(const RopeRowsArgs& a, const float* gamma, int dl, int2 two, const float2* cs,
                                         float (&p)[8], float (&r)[8]) {
    if (a.norm) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s0 = fmaf(p[i], p[i], s0), s1 = fmaf(r[i], r[i], s1);
        const float rs = rsqrtf(head_sum<D / 16>(s0 + s1) * (1.0f / D) + a.eps);
        float g[8];
        load8(gamma + two.x * 8, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (p[i] * rs) * g[i];
        load8(gamma + two.y * 8, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = (r[i] * rs) * g[i];
    }
    if constexpr (kLayout == kRopeHalves) {
        if (dl < a.pairs / 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 w = cs[rope_slot<kLayout>(8 * dl + i)];
                const float x0 = p[i], x1 = r[i];
                p[i] = x0 * w.x - x1 * w.y;
                r[i] = x0 * w.y + x1 * w.x;
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float* z = i < 4 ? p + 2 * i : r + 2 * (i - 4);
            if (8 * dl + i < a.pairs) {
                const float2 w = cs[rope_slot<kLayout>(8 * dl + i)];
                const float x0 = z[0], x1 = z[1];
                z[0] = x0 * w.x - x1 * w.y;
                z[1] = x0 * w.y + x1 * w.x;
            }
        }
    }
}

// Heads that are only normed and rotated, a block a token, by pairs of units; a thread takes the same pair of
// every head it takes.
template <typename In, typename Out, int D, int kLayout>
__global__ void __launch_bounds__(256) rope_pairs_kernel(const RopeRowsArgs a) {
    constexpr int DL = D / 16, kTake = sizeof(In) == 4 ? 1 : 2;  // heads of a thread at a time
    __shared__ float2 cs[64];
    const int qh = a.q ? a.q_heads : 0, heads = qh + (a.tiles ? 0 : a.kv_heads);
    const int dl = threadIdx.x % DL, step = blockDim.x / DL, h0 = threadIdx.x / DL;
    const int2 two = rope_two_units<D, kLayout>(dl, a.pairs);
    const long long tok = blockIdx.x;
    Units<In> x[2 * kTake];
    auto load = [&](int h) {
#pragma unroll
        for (int n = 0; n < kTake; ++n, h += step) {
            if (h < heads) {
                const In* src = h < qh ? static_cast<const In*>(a.q) + tok * a.q_stride + h * D
                                       : static_cast<const In*>(a.k) + tok * a.k_stride + (h - qh) * D;
                x[2 * n].load(src + two.x * 8);
                x[2 * n + 1].load(src + two.y * 8);
            } else {
                x[2 * n].zero();
                x[2 * n + 1].zero();
            }
        }
    };
    load(h0);
    const int pos = a.pos ? a.pos[tok] : a.pos0 + static_cast<int>(tok);
    for (int i = threadIdx.x; i < a.pairs; i += blockDim.x)
        cs[rope_slot<kLayout>(i)] = rope_turn(a.turns[i], pos, a.magnitude);
    __syncthreads();
    for (int h = h0; h - h0 < heads; h += kTake * step) {
        if (h != h0) load(h);
#pragma unroll
        for (int n = 0; n < kTake; ++n) {
            const int hn = h + n * step;
            float p[8], r[8];
            x[2 * n].get(p);
            x[2 * n + 1].get(r);
            rope_two<D, kLayout>(a, hn < qh ? a.q_gamma : a.k_gamma, dl, two, cs, p, r);
            if (hn < heads) {
                Out* dst = hn < qh ? static_cast<Out*>(a.q_out) + tok * a.q_out_stride + hn * D
                                   : static_cast<Out*>(a.k_out) + tok * a.k_out_stride + (hn - qh) * D;
                store8(dst + two.x * 8, p);
                store8(dst + two.y * 8, r);
            }
        }
    }
    // Launched beside kv4_append_kernel, whose completion this grid's stands for.
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Block (token, part of its units), a unit a thread: few tokens, and halves that are not whole units apart.  A
// token's rotation is computed once for the block's heads, with its first loads already in flight.
constexpr int kRopeAhead = 4;  // units a thread has in flight
template <typename In, typename Out, int D, int kLayout>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeRowsArgs a) {
    constexpr int L = D / 8;  // units (lanes) of a head
    __shared__ float2 cs[64];
    __shared__ float xch[kLayout == kRopeHalvesOdd ? 256 * 8 : 1];
    const int part = blockIdx.x % a.parts;
    const long long tok = blockIdx.x / a.parts;
    const int q_units = a.q ? a.q_heads * L : 0, k_units = a.kv_heads * L;
    const int pos = a.pos ? a.pos[tok] : a.pos0 + static_cast<int>(tok);
    const int u1 = min(q_units + k_units + (a.v ? k_units : 0), (part + 1) * a.units_per_block);
    const int lane = threadIdx.x & 31;
    bool first = true;
    // Whole warps stay together: the shuffles below need every lane (units past the end work on zeros).
    for (int u0 = part * a.units_per_block + static_cast<int>(threadIdx.x & ~31); first || u0 < u1; u0 += kRopeAhead * blockDim.x) {
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
        }
        first = false;
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
