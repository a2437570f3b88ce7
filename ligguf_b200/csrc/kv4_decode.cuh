// kv4_decode.cuh - one token of each sequence: norm, rotation, append, attention over the 4-bit cache.
//
//   out_h = sum_j w_j v_j / sum_j w_j,  w_j = 2^(x_j),  x_j = log2(e) * scale * (q_h . k_j)
//
// over the visible cached positions j and the token's own unquantized k, v.
//
// Bound by the cache's bytes (18 D a tile of 16 positions and KV head) as long as the arithmetic on them
// stays short, so both products run on the tensor cores (mma.m16n8k16, fp16 operands, fp32 sums) straight
// from the packed codes:
//   - Keys: a code n (0..15) masked into the low mantissa bits of a half is the subnormal n * 2^-24, and
//     shifted by a nibble n * 2^-20: exact operands that cost one AND for two codes.  The powers of two are
//     taken out of the fp32 results, and the -8 of (n - 8) d is added to a group's sum.  The tensor cores
//     align products by their operands' exponent fields and cut off what lies 24 bits below the largest, and
//     a subnormal's field is that of 2^-14: so the queries' hi parts are whole numbers, which makes every
//     product and sum of hi parts exact, cut or not.
//   - Values: the weights cannot be whole numbers, and with subnormal codes that cut costs 7 bits (results
//     were off by 9e-6).  So 0x6400 is OR-ed in by the same instruction (1024 + n, or 1024 + 16 n), and one
//     packed subtraction (or multiply-add) makes it n - 8: normal halves, exact as well.
//   - S^T = K Q^T: 16 positions x 8 columns.  The key scales multiply the fp32 sums of their 32 elements.
//   - Queries and weights are split into two halves each, hi + lo, which together hold 22 bits, so the
//     results are those of fp32 arithmetic.  Up to four query heads a KV head share one product: columns
//     0-3 are the hi parts of the heads, 4-7 the lo parts, which cost nothing then.  The two parts of a
//     score lie two lanes apart, so a warp takes tiles in pairs: one exchange leaves the lanes of the hi
//     columns with the first tile's scores and those of the lo columns with the second's, and no lane
//     does another's softmax again.  With eight heads the lo parts are a second product into the same
//     sums, and every lane has heads of its own.
//   - O^T += V^T W: the value scales are multiplied into the weights, one B operand for each 32 elements.
//     The weights go from the sums' layout to the operand's by transposing 8x8 fragments (movmatrix).
//   - Weights carry value scales of any size, so the running maximum is that of x_j + (exponent of the
//     largest scale of row j): |weight * scale| stays in [0, 2^15] of fp16's range whatever the scales.
//     It is only moved when a row exceeds it by 2^8, a vote of the warp per tile.
//
// The work is one list: (row, KV head) items, each some units for its start and end, its visible tiles, and
// one unit for the token itself, cut into equal contiguous shares of as many blocks as fit at once, whatever
// the lengths of the sequences; the cut is computed by every block from the positions, which may be in
// device memory.  In a share, the 8 warps take pairs of tiles in turn, each with its own ring of bulk copies
// and its own running sums, which the block joins per item.  Items that several blocks share are joined by
// the last of them to finish, in the order of the blocks, so results repeat bit for bit.
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
    float eps, magnitude, scale_log2;
    int window, sinks;
    uint8_t* tiles;  // first tile of (layer, sequence 0, head 0)
    long long tiles_per_head;
    float* parts;    // [blocks][2] partial results
    int* tickets;    // [n_rows * kv_heads], zero between calls
    float per_block; // 1 / blocks of the launch
    int* err;        // [kKv4ErrWords], in host memory
};

// The status call's words: a wait's code, and whether a row's position was beyond the context.  Each has its own,
// or the later of the two would hide that a block gave up and left tickets behind.
enum : int { kKv4ErrWait = 0, kKv4ErrPosition = 1, kKv4ErrWords = 2 };

// Eight warps a block; two blocks an SM, or one of twice the registers for eight heads a KV head (232 of them; 64 and 8
// heads of 128: one token over 32768 positions 22.8 us, 16 sequences of 8192 64.8 us, where 32 and 8 heads take 22.8
// and 51.4).  At 128 registers, head_dim 128 spills 112 to 124 bytes.  (One block of sixteen
// warps is slower: nothing covers its starts and joins. 24 sequences: 58.8 us against 47.)
__host__ __device__ constexpr int kv4_warps(int) { return 8; }
__host__ __device__ constexpr int kv4_blocks_per_sm(int nrep) { return nrep > 4 ? 1 : 2; }
// Units that an item counts beside its tiles and its token: what a block spends on entering and joining an
// item, in tiles (24, 40, 56, 72: 16 streams of 4100 positions 33.0, 32.2, 31.6, 31.4 us, 24 sequences up to 8191
// 44.6, 44.3, 44.0, 44.4 us).
constexpr int kKv4ItemUnits = 56;
// Units a block has at least: with fewer, a short context's join takes longer than its tiles (512 positions of four
// KV heads: 8.8 us with 16, 9.3 with 24, 13 with 96, where one block takes a head).
constexpr int kKv4MinUnits = 16;

// Floats of one partial result: o [NREP][D], m [NREP], l [NREP], in whole 16 bytes.
__host__ __device__ constexpr int kv4_part_floats(int nrep, int dim) { return (nrep * (dim + 2) + 3) / 4 * 4; }

template <int D, int NREP>
struct Kv4DecodeSmem {
    static constexpr int kWarps = kv4_warps(NREP);
    static constexpr int kStages = D == 128 ? 2 : 4;  // pairs of tiles a warp has in flight
    static constexpr int kParts = NREP > 4 ? 2 : 1;   // hi and lo queries as columns of one operand, or two operands
    static constexpr int kRow = D + 8;                // floats of a head's row of kO: two heads apart, other banks
    static constexpr size_t kRing = 0;
    static constexpr size_t kFrag = kRing + size_t(kWarps) * kStages * 2 * Kv4<D>::kTileBytes;  // [kParts][D/16][32] uint2
    static constexpr size_t kSum = kFrag + size_t(kParts) * (D / 16) * 32 * 8;                     // [kParts][D/32][8]
    static constexpr size_t kScale = kSum + size_t(kParts) * 8 * (D / 32) * 4;                     // [8]
    static constexpr size_t kQ = kScale + 8 * 4;
    static constexpr size_t kGamma = kQ + NREP * D * 4;  // norm weights of q and k
    static constexpr size_t kKn = kGamma + 2 * D * 4;
    static constexpr size_t kVn = kKn + D * 4;
    static constexpr size_t kCs = kVn + D * 4;
    static constexpr size_t kO = kCs + D / 2 * 8;                             // [warps][NREP][kRow]
    static constexpr size_t kM = kO + size_t(kWarps) * NREP * kRow * 4;  // [warps + 1][NREP]
    static constexpr size_t kL = kM + (kWarps + 1) * NREP * 4;
    static constexpr size_t kF = kL + (kWarps + 1) * NREP * 4;           // [warps + 1][NREP] factors, [NREP] M, [NREP] l
    static constexpr size_t kJoin = (kF + (kWarps + 3) * NREP * 4 + 15) / 16 * 16;  // sums of a join's groups
    static constexpr size_t kBar = kJoin + size_t(kWarps) * 32 * 16;
    static constexpr size_t kMisc = kBar + kWarps * kStages * 8;
    static constexpr size_t kFactors = kMisc + 16;  // [NREP] 1 / sum, then [blocks][NREP]
    static constexpr size_t total(int blocks) { return kFactors + size_t(blocks + 1) * NREP * 4; }
};

// Visible cached tiles of a row at position p: tiles [0, ns) hold the sinks, [tw, tw + nt - ns) the window.
struct Kv4Row {
    int pos, first, sinks;  // keys j < pos with j >= first or j < sinks
    int ns, tw, nt;
};
__device__ __forceinline__ Kv4Row kv4_row(const Kv4DecodeArgs& a, int pos) {
    Kv4Row r;
    r.pos = pos;
    r.first = a.window && pos >= a.window ? pos - a.window + 1 : 0;
    r.sinks = min(a.sinks, r.first);
    r.tw = r.first / kKv4Tile;
    r.ns = min((r.sinks + kKv4Tile - 1) / kKv4Tile, r.tw);
    r.nt = r.ns + (pos + kKv4Tile - 1) / kKv4Tile - min(r.tw, (pos + kKv4Tile - 1) / kKv4Tile);
    return r;
}
__device__ __forceinline__ int kv4_tile_of(const Kv4Row& r, int i) { return i < r.ns ? i : r.tw + (i - r.ns); }
// Units of one head of a row; none for an idle row.  (The launcher keeps the sum of all below 2^31.)
__device__ __forceinline__ int kv4_units(const Kv4DecodeArgs& a, int pos) {
    return pos < 0 || pos >= a.n_context ? 0 : kKv4ItemUnits + kv4_row(a, pos).nt + 1;
}

// The positions of a call.  Up to 32 rows: one load, a row a lane.
struct Kv4Positions {
    int mine;  // row `lane`, when there are at most 32
    __device__ __forceinline__ void load(const Kv4DecodeArgs& a, int lane) {
        mine = -1;
        if (a.pos_rows && a.n_rows <= 32 && lane < a.n_rows) mine = a.pos_rows[lane];
    }
    // Warp-uniform r.
    __device__ __forceinline__ int at(const Kv4DecodeArgs& a, int r) const {
        if (!a.pos_rows) return a.pos;
        if (a.n_rows <= 32) return __shfl_sync(0xffffffffu, mine, r);
        return a.pos_rows[r];
    }
    __device__ __forceinline__ int lane_at(const Kv4DecodeArgs& a, int r0, int lane) const {
        if (a.n_rows <= 32) return mine;
        return r0 + lane < a.n_rows ? a.pos_rows[r0 + lane] : -1;
    }
    // All units (warp-collective).
    __device__ __forceinline__ int total(const Kv4DecodeArgs& a, int lane) const {
        if (!a.pos_rows) return kv4_units(a, a.pos) * a.kv_heads * a.n_rows;
        int n = 0;
        for (int r0 = 0; r0 < a.n_rows; r0 += 32) n += kv4_units(a, lane_at(a, r0, lane));
        return __reduce_add_sync(0xffffffffu, n) * a.kv_heads;
    }
    // The row that holds unit u of the list, and the first of its units (warp-collective).
    __device__ __forceinline__ int find(const Kv4DecodeArgs& a, int u, int& start, int lane) const {
        if (!a.pos_rows) {
            const int per = kv4_units(a, a.pos) * a.kv_heads;
            start = u / per * per;
            return u / per;
        }
        int before = 0;
        for (int r0 = 0; r0 < a.n_rows; r0 += 32) {
            const int own = kv4_units(a, lane_at(a, r0, lane)) * a.kv_heads;
            int upto = own;  // inclusive scan
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > u);
            if (past) {
                const int w = __ffs(past) - 1;
                start = before + __shfl_sync(0xffffffffu, upto - own, w);
                return r0 + w;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        start = before;
        return a.n_rows - 1;
    }
};

// One head, 8 elements a lane (D/8 lanes, the other lanes the same again): norm and rotation of x; `dst`
// (shared, D floats) carries the exchange; the norm weights are in shared memory too.
template <int D>
__device__ __forceinline__ void kv4_head(float (&x)[8], const float* gamma, bool norm, float eps, const float2* cs,
                                         int pairs, int layout, float* dst, int lane) {
    constexpr int L = D / 8;
    const int l = lane % L;
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
        ss = head_sum<L>(ss);
        const float rs = rms_factor<D>(ss, eps);
        float gm[8];
        load8(gamma + l * 8, gm);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (x[i] * rs) * gm[i];
    }
    if (layout == LIGGUF_ROPE_ADJACENT) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * l + i < pairs) {
                const float2 w = cs[4 * l + i];
                const float x0 = x[2 * i], x1 = x[2 * i + 1];
                x[2 * i] = rope_first(x0, x1, w);
                x[2 * i + 1] = rope_second(x0, x1, w);
            }
    } else if (pairs) {
        if (lane < L) store8(dst + l * 8, x);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 8 * l + i;
            if (e < 2 * pairs) {
                const bool low = e < pairs;
                const float2 w = cs[low ? e : e - pairs];
                const float other = dst[low ? e + pairs : e - pairs];
                x[i] = low ? rope_first(x[i], other, w) : rope_second(other, x[i], w);
            }
        }
        __syncwarp();
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 x) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = x;
    } else {
        union {
            T h[4];
            uint2 v;
        } u;
        u.h[0] = KvTraits<T>::from_float(x.x), u.h[1] = KvTraits<T>::from_float(x.y);
        u.h[2] = KvTraits<T>::from_float(x.z), u.h[3] = KvTraits<T>::from_float(x.w);
        *reinterpret_cast<uint2*>(p) = u.v;
    }
}

__device__ __forceinline__ void store_rows8(void* rows, int type, long long at, const float (&y)[8]) {
    if (type == LIGGUF_KV_F32)
        store8(static_cast<float*>(rows) + at, y);
    else if (type == LIGGUF_KV_F16)
        store8(static_cast<__half*>(rows) + at, y);
    else
        store8(static_cast<__nv_bfloat16*>(rows) + at, y);
}

// D = A B + C: m16n8k16, fp16 operands, fp32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// n - 8 for the codes in bits 0-3 (code_low) or 4-7 (code_high) of both 16-bit halves, as halves.
__device__ __forceinline__ uint32_t code_low(uint32_t w) {
    const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), __floats2half2_rn(1032.f, 1032.f));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t code_high(uint32_t w) {
    const uint32_t x = (w & 0x00F000F0u) | 0x64006400u;
    const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&x), __floats2half2_rn(0.0625f, 0.0625f),
                              __floats2half2_rn(-72.f, -72.f));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint2 lds64(const void* p) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(smem_u32(p)));
    return r;
}

// One query head (8 elements a lane, D/8 lanes, the others the same again), times scale * log2(e), as B
// operands: column `head` of the hi parts and of the lo parts (column 4 + head, or a second operand).
// Column k = 2t + b + 8c of k-step j is element 16j + 4t + 2b + c, and meets codes * 2^-24 (c = 0) or
// * 2^-20 (c = 1).  sums: -8 * 2^-24 * the sum of a group's elements; scales: what the scores are short of.
template <int D, int NREP>
__device__ __forceinline__ void kv4_query_operands(const float (&x)[8], int head, uint2* frag, float* sums, float* scales,
                                                   int lane) {
    constexpr bool kWide = NREP > 4;
    constexpr int L = D / 8, G = D / 32;
    const int l = lane % L;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
    for (int o = 1; o < L; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // A power of two that brings the head's largest element to [2^10, 2^11): hi is then a normal half and lo
    // loses nothing either.
    const int e = min(100, max(-100, ((__float_as_int(top) >> 23) & 255) - 127));
    const float up = __int_as_float((127 + 10 - e) << 23);
    float sh = 0.f, sl = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        // hi: whole numbers, so that every product with a code and every sum of a group's is exact; lo: what is
        // left, at most a half.
        const float v0 = x[4 * u] * up, v1 = x[4 * u + 1] * up, v2 = x[4 * u + 2] * up, v3 = x[4 * u + 3] * up;
        const float w0 = rintf(v0), w1 = rintf(v1), w2 = rintf(v2), w3 = rintf(v3);
        const uint2 hi = make_uint2(pack_f16(w0, w2), pack_f16(w1 * 0.0625f, w3 * 0.0625f));
        const uint2 lo = make_uint2(pack_f16(v0 - w0, v2 - w2), pack_f16((v1 - w1) * 0.0625f, (v3 - w3) * 0.0625f));
        const float2 h0 = make_float2(w0, w2), h1 = make_float2(w1 * 0.0625f, w3 * 0.0625f);
        const float2 r0 = unpack_f16(lo.x), r1 = unpack_f16(lo.y);
        sh += (h0.x + h0.y) + 16.f * (h1.x + h1.y);
        sl += (r0.x + r0.y) + 16.f * (r1.x + r1.y);
        const int at = (l >> 1) * 32 + 2 * (l & 1) + u;
        if (lane < L) {
            frag[at + head * 4] = hi;
            frag[at + (kWide ? D / 16 * 32 + head * 4 : (4 + head) * 4)] = lo;
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        sh += __shfl_xor_sync(0xffffffffu, sh, o);
        sl += __shfl_xor_sync(0xffffffffu, sl, o);
    }
    constexpr float k8 = -8.f / 16777216.f;
    if (lane < L && (l & 3) == 0) {
        sums[(l >> 2) * 8 + head] = k8 * sh;
        sums[(kWide ? 8 * G : 4) + (l >> 2) * 8 + head] = k8 * sl;
    }
    if (lane == 0) {
        const float down = __int_as_float((127 + e + 14) << 23);  // 2^(e - 10) * 2^24
        scales[head] = down;
        if (!kWide) scales[4 + head] = down;
    }
}

// Sums of V values over the lanes that differ in bits 4..16 (the row groups) and, with kPairs, 2: each lane
// is left with the sum of one value, number value_of(lane).
template <int V, bool kPairs>
__device__ __forceinline__ float rows_sum(float (&v)[V], int lane) {
    static_assert(V == 2 || V == 4 || V == 8, "");
    int bit = 16;
#pragma unroll
    for (int n = V / 2; n >= 1; n /= 2, bit /= 2) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = up ? v[i] : v[n + i], keep = up ? v[n + i] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
        }
    }
#pragma unroll
    for (; bit >= (kPairs ? 2 : 4); bit /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
    return v[0];
}
template <int V>
__device__ __forceinline__ int rows_value(int lane) {
    return (lane >> 2) / (8 / V);
}

// One warp's running sums over the tiles it takes of an item.
template <int D, int NREP>
struct Kv4Warp {
    static constexpr bool kWide = NREP > 4;  // hi and lo parts as two products
    static constexpr int KS = D / 16, G = D / 32;
    // Queries as B operands, and -8 times the sums of their groups, stay in shared memory: two loads a pair of tiles
    // and k-step cost less than the registers.
    const uint2* b;   // this lane's, of k-step 0
    const float2* c;  // this lane's two columns, of group 0
    float sx[2];      // scales of the scores of this lane's two heads
    float m[2], l[2];                  // running maxima and sums of weights
    float o[KS][4];

    // From what kv4_query_operands left in shared memory.
    __device__ __forceinline__ void start(const uint2* frag, const float* sums, const float* scales, int lane) {
        const int t = lane & 3;
        b = frag + lane;
        c = reinterpret_cast<const float2*>(sums) + t;
        sx[0] = scales[2 * t], sx[1] = scales[2 * t + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) m[i] = -1e30f, l[i] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }

    // Raw scores of kTiles tiles' positions g (x[0], x[1]) and g + 8 (x[2], x[3]) with this lane's columns.
    template <int kTiles>
    __device__ __forceinline__ void scores(const uint8_t* tp, int lane, float (&x)[kTiles][4]) const {
        constexpr int TB = Kv4<D>::kTileBytes;
#pragma unroll
        for (int n = 0; n < kTiles; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
            uint4 w4[kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) w4[n] = lds128(tp + n * TB + ch * 512 + lane * 16);
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const int i = ch * 2 + gr;
                // (lo parts of eight heads in sums of their own: added to those of the hi parts they would be cut off)
                float s[kTiles][4] = {}, s2[kTiles][4] = {};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint2 q = b[(2 * i + u) * 32], r = kWide ? b[(KS + 2 * i + u) * 32] : make_uint2(0, 0);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const uint32_t lo = gr ? (u ? w4[n].w : w4[n].z) : (u ? w4[n].y : w4[n].x), hi = lo >> 8;
                        const uint32_t a0 = lo & 0x000F000Fu, a2 = lo & 0x00F000F0u, a1 = hi & 0x000F000Fu, a3 = hi & 0x00F000F0u;
                        mma_f16(s[n], a0, a1, a2, a3, q.x, q.y, s[n][0], s[n][1], s[n][2], s[n][3]);
                        if constexpr (kWide) mma_f16(s2[n], a0, a1, a2, a3, r.x, r.y, s2[n][0], s2[n][1], s2[n][2], s2[n][3]);
                    }
                }
                const float2 c0 = c[4 * i];
                float2 c1 = make_float2(0.f, 0.f);
                if constexpr (kWide) c1 = c[4 * (G + i)];
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    const __half* ks = reinterpret_cast<const __half*>(tp + n * TB + Kv4<D>::kKeyScales) + (lane >> 2) * G + i;
                    const float k0 = __half2float(ks[0]), k1 = __half2float(ks[8 * G]);
                    float* y = s[n];
                    if constexpr (kWide)
                        y[0] += s2[n][0] + c1.x, y[1] += s2[n][1] + c1.y, y[2] += s2[n][2] + c1.x, y[3] += s2[n][3] + c1.y;
                    x[n][0] = fmaf(y[0] + c0.x, k0, x[n][0]);
                    x[n][1] = fmaf(y[1] + c0.y, k0, x[n][1]);
                    x[n][2] = fmaf(y[2] + c0.x, k1, x[n][2]);
                    x[n][3] = fmaf(y[3] + c0.y, k1, x[n][3]);
                }
            }
        }
    }
    // Softmax weights of a tile's positions k0 + g, k0 + g + 8 from their raw scores; vs: their value scales.
    // masked: some position of the tile (or of the pair's other tile) is unseen.
    __device__ __forceinline__ void weights(const uint8_t* tp, const Kv4Row& r, int k0, bool masked, bool there, int lane,
                                            float (&x)[4], float (&p)[4], float (&vs)[2][G]) {
        const int g = lane >> 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= sx[i & 1];
        const float2 ex = load_value_scales(tp + Kv4<D>::kValueScales, g, vs);
        if (masked) {
            const int j0 = k0 + g, j1 = j0 + 8;
            const bool s0 = there && j0 < r.pos && (j0 >= r.first || j0 < r.sinks);
            const bool s1 = there && j1 < r.pos && (j1 >= r.first || j1 < r.sinks);
            if (!s0) x[0] = x[1] = -INFINITY;
            if (!s1) x[2] = x[3] = -INFINITY;
#pragma unroll
            for (int i = 0; i < G; ++i) {  // an unseen row's scales may be anything: 0 * NaN is NaN
                if (!s0) vs[0][i] = 0.f;
                if (!s1) vs[1][i] = 0.f;
            }
        }
        const float t0 = fmaxf(x[0] + ex.x, x[2] + ex.y), t1 = fmaxf(x[1] + ex.x, x[3] + ex.y);
        if (__any_sync(0xffffffffu, t0 > m[0] + 8.f || t1 > m[1] + 8.f)) move_max(t0, t1);
        const float m0 = m[0] - 7.f, m1 = m[1] - 7.f;
        p[0] = ex2(x[0] - m0), p[1] = ex2(x[1] - m1), p[2] = ex2(x[2] - m0), p[3] = ex2(x[3] - m1);
        l[0] += p[0] + p[2];
        l[1] += p[1] + p[3];
    }
    // O += V^T W for one word of the value codes (16 elements of the head).
    __device__ __forceinline__ void values(uint32_t lo, int j, uint32_t b0, uint32_t b1) {
        const uint32_t hi = lo >> 8;
        mma_f16(o[j], code_low(lo), code_high(lo), code_low(hi), code_high(hi), b0, b1, o[j][0], o[j][1], o[j][2], o[j][3]);
    }
    __device__ __forceinline__ static bool edge(const Kv4Row& r, int k0) { return k0 + kKv4Tile > r.pos || k0 < r.first; }

    // Two tiles in shared memory, of positions k0.. and k1.. (k1 < 0: only the first is there).
    __device__ __forceinline__ void pair(const uint8_t* tp, const Kv4Row& r, int k0, int k1, int lane) {
        constexpr int TB = Kv4<D>::kTileBytes;
        if constexpr (kWide) {
#pragma unroll 1
            for (int n = 0; n < 2; ++n, tp += TB, k0 = k1) {
                if (k0 < 0) return;
                float x[1][4], p[4], vs[2][G];
                scores<1>(tp, lane, x);
                weights(tp, r, k0, edge(r, k0), true, lane, x[0], p, vs);
#pragma unroll
                for (int ch = 0; ch < D / 64; ++ch) {
                    const uint4 w4 = lds128(tp + Kv4<D>::kCodes + ch * 512 + lane * 16);
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int gr = 0; gr < 2; ++gr) {
                        const int i = ch * 2 + gr;
                        uint32_t h0, h1, l0, l1;
                        split(i, p, vs, h0, h1, l0, l1);
                        h0 = movmatrix(h0), h1 = movmatrix(h1), l0 = movmatrix(l0), l1 = movmatrix(l1);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            values(w[2 * gr + u], 2 * i + u, h0, h1);
                            values(w[2 * gr + u], 2 * i + u, l0, l1);
                        }
                    }
                }
            }
        } else {
            const bool second = lane & 2;  // lanes of the lo columns take the second tile
            float x[4], p[4], vs[2][G];
            {
                float xs[2][4];
                scores<2>(tp, lane, xs);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[i] = (second ? xs[1][i] : xs[0][i]) + __shfl_xor_sync(0xffffffffu, second ? xs[0][i] : xs[1][i], 2);
            }
            // (k1 > k0, so these two are the first's lower and the second's upper edge; a tile of first tokens, below the
            // window, counts as an edge)
            const bool masked = k1 < 0 || k0 < r.first || k1 + kKv4Tile > r.pos;
            weights(second ? tp + TB : tp, r, second ? k1 : k0, masked, !second || k1 >= 0, lane, x, p, vs);
#pragma unroll
            for (int ch = 0; ch < D / 64; ++ch) {
                const uint4 wa4 = lds128(tp + Kv4<D>::kCodes + ch * 512 + lane * 16);
                const uint4 wb4 = lds128(tp + TB + Kv4<D>::kCodes + ch * 512 + lane * 16);
                const uint32_t wa[4] = {wa4.x, wa4.y, wa4.z, wa4.w}, wb[4] = {wb4.x, wb4.y, wb4.z, wb4.w};
#pragma unroll
                for (int gr = 0; gr < 2; ++gr) {
                    const int i = ch * 2 + gr;
                    uint32_t h0, h1, l0, l1;
                    split(i, p, vs, h0, h1, l0, l1);
                    // This lane's tile's other part goes two lanes over, the other tile's comes back.
                    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, second ? h0 : l0, 2);
                    const uint32_t r1 = __shfl_xor_sync(0xffffffffu, second ? h1 : l1, 2);
                    const uint32_t a0 = movmatrix(second ? r0 : h0), a1 = movmatrix(second ? r1 : h1);
                    const uint32_t b0 = movmatrix(second ? l0 : r0), b1 = movmatrix(second ? l1 : r1);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        values(wa[2 * gr + u], 2 * i + u, a0, a1);
                        values(wb[2 * gr + u], 2 * i + u, b0, b1);
                    }
                }
            }
        }
    }
    // Weights times the value scales of group i, as hi and lo halves of rows g (0) and g + 8 (1).
    __device__ __forceinline__ void split(int i, const float (&p)[4], const float (&vs)[2][G], uint32_t& h0, uint32_t& h1,
                                          uint32_t& l0, uint32_t& l1) {
        const float v0 = p[0] * vs[0][i], v1 = p[1] * vs[0][i], v2 = p[2] * vs[1][i], v3 = p[3] * vs[1][i];
        h0 = pack_f16(v0, v1);
        h1 = pack_f16(v2, v3);
        const float2 f0 = unpack_f16(h0), f1 = unpack_f16(h1);
        l0 = pack_f16(v0 - f0.x, v1 - f0.y);
        l1 = pack_f16(v2 - f1.x, v3 - f1.y);
    }

    // Moves the running maxima to those of all rows and rescales the sums.
    __device__ __forceinline__ void move_max(float t0, float t1) {
#pragma unroll
        for (int s = kWide ? 4 : 2; s < 32; s <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, s));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, s));
        }
        const float n0 = fmaxf(m[0], t0), n1 = fmaxf(m[1], t1);
        const float f0 = ex2(m[0] - n0), f1 = ex2(m[1] - n1);
        m[0] = n0, m[1] = n1;
        l[0] *= f0, l[1] *= f1;
#pragma unroll
        for (int j = 0; j < KS; ++j) o[j][0] *= f0, o[j][1] *= f1, o[j][2] *= f0, o[j][3] *= f1;
    }

    // The value scales, and for both rows an exponent E with |scale| < 2^E for every group.
    __device__ __forceinline__ static float2 load_value_scales(const uint8_t* s, int g, float (&out)[2][G]) {
        float e[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            uint32_t top;
            if constexpr (G == 4) {
                const uint2 u = lds64(s + (g + 8 * r) * 8);
                const float2 x = unpack_f16(u.x), y = unpack_f16(u.y);
                out[r][0] = x.x, out[r][1] = x.y, out[r][2] = y.x, out[r][3] = y.y;
                top = __vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu);
            } else {
                const uint32_t u = *reinterpret_cast<const uint32_t*>(s + (g + 8 * r) * 4);
                const float2 x = unpack_f16(u);
                out[r][0] = x.x, out[r][1] = x.y;
                top = u & 0x7FFF7FFFu;
            }
            top = max(top & 0xFFFFu, top >> 16);
            e[r] = static_cast<float>(static_cast<int>(top >> 10) - 14);
        }
        return make_float2(e[0], e[1]);
    }

    // Sums over the warp's rows, to shared memory: o [NREP][kRow], m and l [NREP]; all relative to 2^m.
    __device__ __forceinline__ void finish(float* so, float* sm, float* sl, int lane) {
        constexpr int kRow = Kv4DecodeSmem<D, NREP>::kRow;
        const int g = lane >> 2, t = lane & 3;
        const int h0 = kWide ? 2 * t : 2 * (t & 1);  // this lane's columns are heads h0, h0 + 1
        const bool first = kWide || t < 2;
        float lv[2] = {l[0], l[1]};
        const float ls = rows_sum<2, !kWide>(lv, lane);
        const int li = rows_value<2>(lane);
        if (first && h0 + li < NREP) sl[h0 + li] = ls, sm[h0 + li] = (li ? m[1] : m[0]) - 7.f;
        // Rows g and g + 8 of k-step j are elements 16j + 2g, 16j + 2g + 1.
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            float* at = so + h0 * kRow + 16 * j + 2 * g;
            if constexpr (kWide) {
                *reinterpret_cast<float2*>(at) = make_float2(o[j][0], o[j][2]);
                *reinterpret_cast<float2*>(at + kRow) = make_float2(o[j][1], o[j][3]);
            } else {  // hi and lo columns lie two lanes apart: one lane adds rows g, the other rows g + 8
                const float y0 = (first ? o[j][0] : o[j][2]) + __shfl_xor_sync(0xffffffffu, first ? o[j][2] : o[j][0], 2);
                const float y1 = (first ? o[j][1] : o[j][3]) + __shfl_xor_sync(0xffffffffu, first ? o[j][3] : o[j][1], 2);
                if (h0 < NREP) at[first ? 0 : 1] = y0;
                if (h0 + 1 < NREP) at[kRow + (first ? 0 : 1)] = y1;
            }
        }
    }
};

template <typename In, int D, int NREP>
__global__ void __launch_bounds__(32 * kv4_warps(NREP), kv4_blocks_per_sm(NREP)) kv4_decode_kernel(const Kv4DecodeArgs a) {
    using Sm = Kv4DecodeSmem<D, NREP>;
    constexpr int L = D / 8, TB = Kv4<D>::kTileBytes, PF = kv4_part_floats(NREP, D);
    constexpr unsigned S = Sm::kStages;
    constexpr int kWarps = Sm::kWarps, kThreads = 32 * kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    uint2* frag = reinterpret_cast<uint2*>(smem + Sm::kFrag);
    float* sums = reinterpret_cast<float*>(smem + Sm::kSum);
    float* scales = reinterpret_cast<float*>(smem + Sm::kScale);
    float* qs = reinterpret_cast<float*>(smem + Sm::kQ);
    float* kn = reinterpret_cast<float*>(smem + Sm::kKn);
    float* vn = reinterpret_cast<float*>(smem + Sm::kVn);
    float2* cs = reinterpret_cast<float2*>(smem + Sm::kCs);
    float* so = reinterpret_cast<float*>(smem + Sm::kO);
    float* sm = reinterpret_cast<float*>(smem + Sm::kM);
    float* sl = reinterpret_cast<float*>(smem + Sm::kL);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + Sm::kMisc);
    int* last = reinterpret_cast<int*>(smem + Sm::kMisc + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sm::kBar) + warp * S;
    uint8_t* ring = smem + Sm::kRing + size_t(warp) * S * 2 * TB;
    if (lane == 0) {
        for (unsigned s = 0; s < S; ++s) mbar_init(&bars[s], 1);
        fence_mbar_init();
    }
    if (threadIdx.x == 0) *abort = 0;
    if (NREP < 4) {  // columns without a head
        for (int i = threadIdx.x; i < D / 16 * 32; i += kThreads) frag[i] = make_uint2(0, 0);
        for (int i = threadIdx.x; i < 8 * (D / 32); i += kThreads) sums[i] = 0.f;
        if (threadIdx.x < 8) scales[threadIdx.x] = 1.f;
    }
    // The norm weights, which no kernel writes.
    float* gammas = reinterpret_cast<float*>(smem + Sm::kGamma);
    if (a.norm && threadIdx.x < 2 * D) gammas[threadIdx.x] = threadIdx.x < D ? a.q_gamma[threadIdx.x] : a.k_gamma[threadIdx.x - D];
    __syncthreads();
    // Everything before touched only this block's shared memory and what the host wrote; the previous kernel
    // of the stream (which may have written the cache, the positions or the rows) has completed after this.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Kv4Positions where;
    where.load(a, lane);
    const int total = where.total(a, lane);
    // At least total / gridDim.x, by a product: the conversion rounds up, and one in 2^20 covers the factor's error.
    const int share = max(kKv4MinUnits, __float2int_ru(static_cast<float>(total) * a.per_block) + (total >> 20));
    const int bx = blockIdx.x;
    // Idle rows: zeros.
    if (a.pos_rows) {
        for (int r = bx; r < a.n_rows; r += gridDim.x) {
            const int pos = where.at(a, r);
            if (pos >= 0 && pos < a.n_context) continue;
            if (pos >= 0 && threadIdx.x == 0) reinterpret_cast<volatile int*>(a.err)[kKv4ErrPosition] = 1;
            const float z[8] = {};
            for (int u = threadIdx.x; u < a.q_heads * L; u += kThreads)
                store8(static_cast<In*>(a.out) + (static_cast<long long>(r) * a.q_heads * L + u) * 8, z);
            for (int u = threadIdx.x; u < a.kv_heads * L; u += kThreads) {
                const long long at = (static_cast<long long>(r) * a.kv_heads * L + u) * 8;
                if (a.k_rows) store_rows8(a.k_rows, a.rows_type, at, z);
                if (a.v_rows) store_rows8(a.v_rows, a.rows_type, at, z);
            }
        }
    }
    const long long from = static_cast<long long>(bx) * share;
    if (from >= total) return;
    const int u0 = static_cast<int>(from), u1 = static_cast<int>(min(static_cast<long long>(total), from + share));
    const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;

    // Two cursors walk the share's items: the copies', ahead, and the sums'.
    struct Cursor {
        int row, head, t, t1;    // next pair of tiles of this warp in the item's share, and the share's end
        int start, units, next;  // first unit and units of the row's head; first unit of the next head
        Kv4Row r;
        const uint8_t* tiles;    // the head's first
    };
    auto enter = [&](Cursor& c, int u) {  // at unit u >= u0 of row c.row, whose heads start at c.start
        c.r = kv4_row(a, where.at(a, c.row));
        c.units = kKv4ItemUnits + c.r.nt + 1;
        // The head: heads whose units end at or before u.
        c.head = a.kv_heads <= 32 ? __popc(__ballot_sync(0xffffffffu, lane < a.kv_heads && (lane + 1) * c.units <= u - c.start))
                                  : (u - c.start) / c.units;
        const int h0 = c.start + c.head * c.units;
        c.next = h0 + c.units;
        c.t = max(0, u - h0 - kKv4ItemUnits) + 2 * warp;
        c.t1 = min(c.r.nt, u1 - h0 - kKv4ItemUnits);
        c.tiles = a.tiles + (static_cast<long long>(c.row) * a.kv_heads + c.head) * a.tiles_per_head * TB;
    };
    auto advance = [&](Cursor& c) {  // to the next item of the share; false at its end
        if (c.next + kKv4ItemUnits >= u1) return false;  // nothing but an item's first units is left
        if (c.head + 1 == a.kv_heads) {
            c.start = c.next;
            do {
                ++c.row;
            } while (c.row + 1 < a.n_rows && kv4_units(a, where.at(a, c.row)) == 0);
        }
        enter(c, c.next);
        return true;
    };
    Cursor in;
    in.row = where.find(a, u0, in.start, lane);
    enter(in, u0);
    if (in.t1 <= 0 && in.next > u1) return;  // the share ends before the item's first tile
    Cursor at = in;
    // The rows of an item that this warp prepares: heads, then (with the item's last unit) the token's key and value.
    constexpr int kRounds = (NREP + 2 + kWarps - 1) / kWarps;
    auto load_rows = [&](const Cursor& c, float (&x)[8], int job) {
        if (job >= NREP + (c.next <= u1 ? 2 : 0)) return;
        const In* src = job < NREP    ? static_cast<const In*>(a.q) + c.row * a.q_stride + (c.head * NREP + job) * D
                        : job == NREP ? static_cast<const In*>(a.k) + c.row * a.k_stride + c.head * D
                                      : static_cast<const In*>(a.v) + c.row * a.v_stride + c.head * D;
        load8(src + lane % L * 8, x);
    };
    float x[8] = {};
    load_rows(at, x, warp);  // on their way while the copies are requested
    const double turn = threadIdx.x < a.pairs ? a.turns[threadIdx.x] : 0.0;
    unsigned issued = 0, taken = 0;
    bool more = true;
    auto request = [&]() {  // the next pair of this warp, if there is one
        while (in.t >= in.t1) {
            more = more && advance(in);
            if (!more) return;
        }
        if (lane == 0) {
            const unsigned s = issued % S;
            uint8_t* dst = ring + s * 2 * TB;
            const int first = kv4_tile_of(in.r, in.t);
            const uint8_t* src = in.tiles + static_cast<long long>(first) * TB;
            const int bytes = in.t + 1 < in.t1 ? 2 * TB : TB;
            mbar_arrive_expect_tx(&bars[s], bytes);
            if (in.t + 1 != in.r.ns || bytes == TB) {  // neighbours
                bulk_copy_g2s(dst, src, bytes, &bars[s]);
            } else {
                bulk_copy_g2s(dst, src, TB, &bars[s]);
                bulk_copy_g2s(dst + TB, in.tiles + static_cast<long long>(in.r.tw) * TB, TB, &bars[s]);
            }
        }
        ++issued;
        in.t += 2 * kWarps;
    };
#pragma unroll 1
    for (unsigned s = 0; s < S; ++s) request();

    Kv4Warp<D, NREP> acc;
    int seg0 = u0;  // first unit of the current item in this share
    int turned = -1;  // the row whose rotations are in shared memory
    // Items shared with other blocks: at most the share's first and its last.  They are joined at the end, when the
    // tickets have long come back.
    struct Shared {
        long long item;
        int first, parts, lead, ticket;  // blocks that have parts, the slot of the first block's
    } lead_item = {0, 0, 0, 0, -1}, last_item = {0, 0, 0, 0, -1};
    for (int seg = 0;; ++seg) {
        const int pos = at.r.pos, g = at.head;
        const int item0 = at.next - at.units + kKv4ItemUnits;  // the item's first tile
        const bool own = at.next <= u1;  // the item's last unit, the token itself, is in this share
        const long long item = static_cast<long long>(at.row) * a.kv_heads + g;
        // Queries (and the token's own key and value) of the item.
        if (at.row != turned) {  // (a row's heads follow one another)
            if (threadIdx.x < a.pairs) cs[threadIdx.x] = rope_turn(turn, pos, a.magnitude);
            turned = at.row;
            __syncthreads();
        }
#pragma unroll
        for (int round = 0; round < kRounds; ++round) {
            const int job = warp + round * kWarps;
            const bool on = job < NREP + (own ? 2 : 0), isq = job < NREP, isk = job == NREP;
            if (round) load_rows(at, x, job);
            if (!on) continue;
            float* dst = isq ? qs + job * D : isk ? kn : vn;
            const bool rot = isq || isk;
            kv4_head<D>(x, gammas + (isq ? 0 : D), rot && a.norm, a.eps, cs, rot ? a.pairs : 0, a.layout, dst, lane);
            if (!isq) {
                uint32_t codes;
                const __half d = kv4_quantize8(x, codes);
                if (lane < L) {
                    uint8_t* tile = const_cast<uint8_t*>(at.tiles) + static_cast<long long>(pos / kKv4Tile) * TB;
                    if (isk)
                        kv4_store8<D, false>(tile, pos % kKv4Tile, lane, codes, d);
                    else
                        kv4_store8<D, true>(tile, pos % kKv4Tile, lane, codes, d);
                    void* rows = isk ? a.k_rows : a.v_rows;
                    if (rows) {
                        float y[8];
                        kv4_values8(codes, d, y);
                        store_rows8(rows, a.rows_type, item * D + lane * 8, y);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= a.scale_log2;
                kv4_query_operands<D, NREP>(x, job, frag, sums, scales, lane);
            }
            if (lane < L) store8(dst + lane * 8, x);
        }
        __syncthreads();
        acc.start(frag, sums, scales, lane);
        for (; at.t < at.t1; at.t += 2 * kWarps) {
            const unsigned s = taken % S;
            if (!mbar_try_wait(&bars[s], (taken / S) & 1) && !mbar_wait_bounded(&bars[s], (taken / S) & 1, deadline, abort)) {
                // (the tile is worked on as it is; the block stops at the next barrier)
                *abort = 1;
                reinterpret_cast<volatile int*>(a.err)[kKv4ErrWait] = KERR_TIMEOUT_FULL;
            }
            const int k0 = kv4_tile_of(at.r, at.t) * kKv4Tile;
            const int k1 = at.t + 1 == at.r.ns ? at.r.tw * kKv4Tile : k0 + kKv4Tile;
            acc.pair(ring + s * 2 * TB, at.r, k0, at.t + 1 < at.t1 ? k1 : -1, lane);
            __syncwarp();
            ++taken;
            request();
        }
        const int next = at.next, begin = at.next - at.units;
        const bool more_items = advance(at);
        if (more_items) load_rows(at, x, warp);  // of the next item, while this one is joined
        acc.finish(so + warp * NREP * Sm::kRow, sm + warp * NREP, sl + warp * NREP, lane);
        if (own)  // the token itself: one key whose weight is 1 relative to its own score
            for (int h = warp; h < NREP; h += kWarps) {
                float y = 0.f;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) y = fmaf(qs[h * D + lane + 32 * i], kn[lane + 32 * i], y);
                y = warp_sum(y);
                if (lane == 0) sm[kWarps * NREP + h] = y, sl[kWarps * NREP + h] = 1.f;
            }
        __syncthreads();
        if (*abort) break;  // raised before the barrier: every thread sees it
        // Join the warps: their factors, a head a warp, then the sums.
        float* fac = reinterpret_cast<float*>(smem + Sm::kF);
        for (int h = warp; h < NREP; h += kWarps) {
            const bool on = lane < kWarps + (own ? 1 : 0);
            const float m = on ? sm[lane * NREP + h] : -1e30f;
            const float M = warp_max(m), f = ex2(m - M);
            const float l = warp_sum(on ? sl[lane * NREP + h] * f : 0.f);
            if (on) fac[lane * NREP + h] = f;
            if (lane == 0) fac[(kWarps + 1) * NREP + h] = M, fac[(kWarps + 2) * NREP + h] = l;
        }
        __syncthreads();
        const bool whole = own && seg0 <= item0;  // no other block has a part of this item
        In* out = static_cast<In*>(a.out) + item * NREP * D;
        float* mine = a.parts + (static_cast<long long>(bx) * 2 + (seg ? 1 : 0)) * PF;
        for (int i = threadIdx.x; i < NREP * D; i += kThreads) {
            const int h = i / D, d = i % D;
            float osum = own ? fac[kWarps * NREP + h] * vn[d] : 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) osum = fmaf(so[(w * NREP + h) * Sm::kRow + d], fac[w * NREP + h], osum);
            const float M = fac[(kWarps + 1) * NREP + h], l = fac[(kWarps + 2) * NREP + h];
            if (whole) {
                out[i] = KvTraits<In>::from_float(osum / l);
            } else {
                mine[i] = osum;
                if (d == 0) mine[NREP * D + h] = M, mine[NREP * D + NREP + h] = l;
            }
        }
        __syncthreads();
        if (!whole) {
            // Blocks b0..b1 have parts of the item: those whose shares meet [item0, next).  Block b0's lies in its
            // second slot when the item is not the first of its share.
            const int b0 = item0 / share, b1 = (next - 1) / share;
            Shared e = {item, b0, b1 - b0 + 1, b0 * share < begin ? 1 : 0, -1};
            if (threadIdx.x == 0)
                // The block's part, ordered before this by the barrier, is out before the ticket; what the
                // other blocks put out before theirs is seen after it.
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(e.ticket) : "l"(a.tickets + item) : "memory");
            if (seg)
                last_item = e;
            else
                lead_item = e;
        }
        seg0 = next;
        if (!more_items) break;
    }
    // Joins the parts of an item that other blocks share, in the last of them to be done.
    auto join = [&](const Shared& e) {
        if (e.parts == 0) return;
        __syncthreads();
        if (threadIdx.x == 0) {
            *last = e.ticket == e.parts - 1;
            if (*last) a.tickets[e.item] = 0;
        }
        __syncthreads();
        if (!*last) return;
        const float* parts = a.parts + static_cast<long long>(e.first) * 2 * PF;
        auto part = [&](int w) { return parts + (w ? w * 2 : e.lead) * PF; };
        // Threads in groups, one 16-byte column a thread; a group takes every kGroups-th part.  All loads leave at
        // once, for up to kGroups * kAhead parts: one trip to the L2 instead of several.
        constexpr int kCols = NREP * D / 4, kGroups = kThreads / kCols, kAhead = 20;
        const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
        float4 y8[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (grp + u * kGroups < e.parts) y8[u] = __ldcg(reinterpret_cast<const float4*>(part(grp + u * kGroups)) + col);
        float* inv = reinterpret_cast<float*>(smem + Sm::kFactors);
        float* fac = inv + NREP;
        for (int h = warp; h < NREP; h += kWarps) {  // the parts' factors, a head a warp
            float m2[2], l2[2], M = -1e30f;  // of parts `lane` and `lane` + 32, which is all of them up to 64
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int w = lane + 32 * u;
                m2[u] = w < e.parts ? __ldcg(part(w) + NREP * D + h) : -1e30f;
                l2[u] = w < e.parts ? __ldcg(part(w) + NREP * D + NREP + h) : 0.f;
            }
            for (int w = lane + 64; w < e.parts; w += 32) M = fmaxf(M, __ldcg(part(w) + NREP * D + h));
            M = warp_max(fmaxf(M, fmaxf(m2[0], m2[1])));
            float l = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float f = ex2(m2[u] - M);
                if (lane + 32 * u < e.parts) fac[(lane + 32 * u) * NREP + h] = f;
                l = fmaf(l2[u], f, l);
            }
            for (int w = lane + 64; w < e.parts; w += 32) {
                const float f = ex2(__ldcg(part(w) + NREP * D + h) - M);
                fac[w * NREP + h] = f;
                l = fmaf(__ldcg(part(w) + NREP * D + NREP + h), f, l);
            }
            l = warp_sum(l);
            if (lane == 0) inv[h] = 1.f / l;
        }
        __syncthreads();
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        const int h = col * 4 / D;
        for (int w0 = grp; w0 < e.parts; w0 += kGroups * kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int w = w0 + u * kGroups;
                if (w >= e.parts) continue;
                const float f = fac[w * NREP + h];
                const float4 z = w0 == grp ? y8[u] : __ldcg(reinterpret_cast<const float4*>(part(w)) + col);
                y.x = fmaf(z.x, f, y.x), y.y = fmaf(z.y, f, y.y), y.z = fmaf(z.z, f, y.z), y.w = fmaf(z.w, f, y.w);
            }
        }
        float4* sums4 = reinterpret_cast<float4*>(smem + Sm::kJoin);
        sums4[threadIdx.x] = y;
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int i = 1; i < kGroups; ++i) {
                const float4 z = sums4[i * kCols + col];
                y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
            }
            const float f = inv[h];
            store4(static_cast<In*>(a.out) + e.item * NREP * D + col * 4, make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
        }
    };
    if (!*abort) {  // (the same for every thread: raised before a barrier that all have passed)
        join(lead_item);
        join(last_item);
    }
    // After a wait that gave up, the copies in flight land before the block ends.
    for (; taken < issued; ++taken)
        while (!mbar_try_wait(&bars[taken % S], (taken / S) & 1) && globaltimer_ns() < deadline + kWaitLimitNs / 2) {
        }
}

}  // namespace lg
