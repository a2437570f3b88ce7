// kv4.cuh - the 4-bit key/value cache: its layout in HBM and the quantizer.
//
// Values.  32 consecutive elements of a head share a scale d (fp16) and have codes 0..15; an element is
// (code - 8) * d (GGUF's Q4_0).
//
// Layout.  A tile is 16 consecutive positions of one KV head of one sequence and layer, 18*D bytes:
//   [0, 8D)     key codes      [8D, 16D)  value codes
//   [16D, 17D)  key scales     [17D, 18D) value scales, each [16 positions][D/32] fp16
// Tiles of one head are consecutive, so the attention kernel streams one contiguous run.  The codes lie
// as the A operand of mma.m16n8k16 wants them, so that a lane unpacks a fragment from one 32-bit word
// with four ANDs and one shift and no exchange between lanes:
//   keys:   A rows are the 16 positions, A columns 16 elements j*16.. of the head.  Word j of lane
//           4g + t holds rows g, g+8 and columns 2t, 2t+1, 2t+8, 2t+9; column 2t + b + 8c is element
//           16j + 4t + 2b + c.
//   values: A rows are 16 elements i*16.. of the head (row g is element 16i + 2g, row g+8 element
//           16i + 2g + 1), A columns the 16 positions; word i of lane 4g + t as above.
// The nibbles of a word, low to high: (keys: row g: columns 2t, 2t+8; row g+8: columns 2t, 2t+8;
// values: column 2t: rows g, g+8; column 2t+8: rows g, g+8) in the low 16 bits, the same of column + 1
// in the high 16.  So w & 0x000F000F and w & 0x00F000F0 are two registers of the fragment, and the
// same of w >> 8 the other two.  Every position owns whole bytes (one byte is two neighbouring elements
// of one position), so appending a position never reads or disturbs another's.
// Words: [D/64 chunks of four words][32 lanes][4 words]: a lane loads 16 bytes, a warp 512 in a row.
#pragma once

#include "common.cuh"

namespace lg {

constexpr int kKv4Tile = 16;  // positions of a tile
template <int D>
struct Kv4 {
    static constexpr int kGroups = D / 32;
    static constexpr int kCodes = 8 * D;          // bytes of a tile's key (or value) codes
    static constexpr int kKeyScales = 16 * D;     // offsets of the scales
    static constexpr int kValueScales = 17 * D;
    static constexpr int kTileBytes = 18 * D;
};

// Byte offset, within a tile's key codes, of the byte that holds elements 2e, 2e+1 of position p.
__host__ __device__ __forceinline__ int kv4_key_byte(int p, int e) {
    const int j = e >> 3, t = (e >> 1) & 3, b = e & 1;
    return (j >> 2) * 512 + ((p & 7) * 4 + t) * 16 + (j & 3) * 4 + 2 * b + (p >> 3);
}
// Same for the value codes.
__host__ __device__ __forceinline__ int kv4_value_byte(int p, int e) {
    const int i = e >> 3, g = e & 7;
    return (i >> 2) * 512 + (g * 4 + ((p & 7) >> 1)) * 16 + (i & 3) * 4 + 2 * (p & 1) + (p >> 3);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Quantizes 8 of a block's 32 elements; lanes 4i..4i+3 of a warp hold a block (every lane of the warp
// calls it).  Returns the scale; code pair i (elements 2i, 2i+1 of the 8) is byte i of `codes`.
__device__ __forceinline__ __half kv4_quantize8(const float (&x)[8], uint32_t& codes) {
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        hi = max_nan(hi, x[i]);
        lo = min_nan(lo, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const float m = hi >= -lo ? hi : lo;  // a NaN anywhere made both NaN
    const bool finite = fabsf(m) <= 3.402823466e+38f;
    const __half d = finite ? __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.f), 65504.f))
                            : __ushort_as_half(static_cast<unsigned short>(0x7FFFu));
    const float df = __half2float(d);
    const float inv = (finite && df != 0.f) ? 1.0f / df : 0.f;
    codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // The scale is rounded first, so the codes answer to the value that is stored.
        const float c = fminf(fmaxf(rintf(x[i] * inv) + 8.f, 0.f), 15.f);  // a NaN gives 0
        codes |= static_cast<uint32_t>(c) << (4 * i);
    }
    return d;
}
// What the cache holds for those 8 elements.
__device__ __forceinline__ void kv4_values8(uint32_t codes, __half d, float (&x)[8]) {
    const float df = __half2float(d);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int>((codes >> (4 * i)) & 15u) - 8) * df;
}
// Stores 8 elements (number l of the head's D/8) of position p of a tile.
template <int D, bool kValues>
__device__ __forceinline__ void kv4_store8(uint8_t* tile, int p, int l, uint32_t codes, __half d) {
    uint8_t* c = tile + (kValues ? Kv4<D>::kCodes : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        c[kValues ? kv4_value_byte(p, 4 * l + i) : kv4_key_byte(p, 4 * l + i)] = static_cast<uint8_t>(codes >> (8 * i));
    if ((l & 3) == 0)
        *reinterpret_cast<__half*>(tile + (kValues ? Kv4<D>::kValueScales : Kv4<D>::kKeyScales) +
                                   2 * (p * Kv4<D>::kGroups + (l >> 2))) = d;
}
// Loads them back: codes and scale.
template <int D, bool kValues>
__device__ __forceinline__ uint32_t kv4_load8(const uint8_t* tile, int p, int l, __half& d) {
    const uint8_t* c = tile + (kValues ? Kv4<D>::kCodes : 0);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        codes |= static_cast<uint32_t>(
                     c[kValues ? kv4_value_byte(p, 4 * l + i) : kv4_key_byte(p, 4 * l + i)])
                 << (8 * i);
    d = *reinterpret_cast<const __half*>(tile + (kValues ? Kv4<D>::kValueScales : Kv4<D>::kKeyScales) +
                                         2 * (p * Kv4<D>::kGroups + (l >> 2)));
    return codes;
}

// 8 consecutive elements of a row, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        KvTraits<T>::unpack(*reinterpret_cast<const uint4*>(p), x);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *(reinterpret_cast<float4*>(p) + 1) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        union {
            T h[8];
            uint4 v;
        } u;
#pragma unroll
        for (int i = 0; i < 8; ++i) u.h[i] = KvTraits<T>::from_float(x[i]);
        *reinterpret_cast<uint4*>(p) = u.v;
    }
}

// ---------------------------------------------------------------------------- conversions
struct Kv4IoArgs {
    uint8_t* tiles;  // first tile of (layer, first sequence, head 0)
    long long tiles_per_head;
    int kv_heads, n_seqs, pos0, n;
    void *k, *v;  // rows or blocks (either may be null)
};

// Cache rows as numbers: one thread per 8 elements of K or V (blockIdx.y).
template <typename Out, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4IoArgs a) {
    constexpr int L = D / 8;
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    const int per_row = a.kv_heads * L;
    if (i >= static_cast<long long>(a.n) * per_row) return;
    const int r = static_cast<int>(i / per_row), u = static_cast<int>(i % per_row), head = u / L, l = u % L;
    const int p = a.pos0 + r;
    const uint8_t* tile = a.tiles + (head * a.tiles_per_head + p / kKv4Tile) * Kv4<D>::kTileBytes;
    Out* dst = static_cast<Out*>(blockIdx.y ? a.v : a.k);
    if (!dst) return;
    __half d;
    const uint32_t codes = blockIdx.y ? kv4_load8<D, true>(tile, p % kKv4Tile, l, d)
                                      : kv4_load8<D, false>(tile, p % kKv4Tile, l, d);
    float x[8];
    kv4_values8(codes, d, x);
    store8(dst + i * 8, x);
}

// Q4_0 blocks in (kLoad) or out: one thread per block of K or V (blockIdx.y) of every sequence.
template <int D, bool kLoad>
__global__ void __launch_bounds__(256) kv4_blocks_kernel(const Kv4IoArgs a) {
    constexpr int G = D / 32;
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    const int per_row = a.kv_heads * G;
    if (i >= static_cast<long long>(a.n_seqs) * a.n * per_row) return;
    const long long row = i / per_row;
    const int u = static_cast<int>(i % per_row), head = u / G, grp = u % G;
    const long long seq = row / a.n;
    const int p = a.pos0 + static_cast<int>(row % a.n);
    uint8_t* tile = a.tiles + ((seq * a.kv_heads + head) * a.tiles_per_head + p / kKv4Tile) * Kv4<D>::kTileBytes;
    unsigned short* blk = static_cast<unsigned short*>(blockIdx.y ? a.v : a.k) + i * 9;
    if (kLoad) {
        uint32_t w[8];  // 16-bit words of the block: the scale, then bytes of codes
#pragma unroll
        for (int s = 0; s < 8; ++s) w[s] = blk[1 + s];
        const __half d = __ushort_as_half(blk[0]);
        // Element e < 16 is the low nibble of byte e, element e + 16 its high nibble.
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint32_t codes = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int byte = (8 * s + e) & 15;
                const uint32_t v = (w[byte >> 1] >> (8 * (byte & 1) + (s >= 2 ? 4 : 0))) & 15u;
                codes |= v << (4 * e);
            }
            if (blockIdx.y)
                kv4_store8<D, true>(tile, p % kKv4Tile, 4 * grp + s, codes, d);
            else
                kv4_store8<D, false>(tile, p % kKv4Tile, 4 * grp + s, codes, d);
        }
    } else {
        uint32_t c[4];
        __half d;
#pragma unroll
        for (int s = 0; s < 4; ++s)
            c[s] = blockIdx.y ? kv4_load8<D, true>(tile, p % kKv4Tile, 4 * grp + s, d)
                              : kv4_load8<D, false>(tile, p % kKv4Tile, 4 * grp + s, d);
        blk[0] = __half_as_ushort(d);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            uint32_t w = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int e = 2 * s + b;  // byte number
                const uint32_t v = ((c[e >> 3] >> (4 * (e & 7))) & 15u) | (((c[2 + (e >> 3)] >> (4 * (e & 7))) & 15u) << 4);
                w |= v << (8 * b);
            }
            blk[1 + s] = static_cast<unsigned short>(w);
        }
    }
}

}  // namespace lg
