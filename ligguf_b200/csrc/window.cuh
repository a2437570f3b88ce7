// window.cuh - causal attention with a sliding window and first tokens that stay visible.
#pragma once

#include "common.cuh"
#include "flash_tc.cuh"

namespace lg {

struct WindowArgs {
    const void *q, *k, *v;
    void* out;
    long long q_stride, k_stride, v_stride, q_batch, k_batch, v_batch;
    const int *pos0, *lens;
    int batch, n, m, q_heads, kv_heads, window, sinks;
    float scale_log2;  // of the scores, times log2(e)
};

// ---------------------------------------------------------------------------- few query rows
// The rows of one KV head's queries (tokens x n_heads/n_kv_heads heads, at most 64) against long runs of keys: bound
// by the bytes of K and V, which every CTA reads once for all of its rows.  More tokens go in chunks of at most 64
// rows, each over its own visible tiles (then bound by the matrix instructions).
//
// Grid (split, KV head and chunk, batch entry): a CTA takes an equal run of its visible key tiles (64 keys; the run
// is worked out from pos0 and lens, which lie in device memory) and leaves its rows' unnormalised sums, maxima and
// row sums; window_join_kernel adds the splits up, in order.  The four warps are row groups of 16 rows x parts of
// the tile's keys.  K and V tiles come by TMA into a ring of two (SWIZZLE_128B rows of 64 columns), S = Q K^T and
// O += P V run on mma.m16n8k16 with ldmatrix reading the swizzled rows; S of a warp is P's operand without any
// exchange.  (tcgen05 wants 128 rows; with 16 of them in use its tiles would be mostly padding, and the kernel is
// bound by memory either way.)
constexpr int kFewKeys = 64, kFewWarps = 4, kFewStages = 2, kFewRows = 64;

struct WindowFewArgs {
    WindowArgs w;
    int splits, tokens, chunks;  // tokens of a chunk
    float* parts;  // [entry][chunk][KV head][split][rows][D + 2]: o, then m, then l (m in log2 units)
    int* err;
};

// The visible key tiles of tokens [i0, i0 + n) of an entry: tiles [0, ns) of the first tokens, then [tw, tw + nt - ns).
struct FewSpan {
    int p0, lo, hi, ns, tw, nt;
};
__device__ __forceinline__ FewSpan few_span(const WindowArgs& a, int b, int i0, int n) {
    FewSpan f;
    const int len = a.lens ? max(0, min(a.lens[b], a.m)) : a.m;
    // (bounded as in tc_window_item: positions beyond every key and window are all alike)
    f.p0 = max(-a.n, min(a.pos0 ? a.pos0[b] : len - a.n, a.m + a.window)) + i0;
    f.hi = max(0, min(len, f.p0 + n));
    f.lo = a.window ? max(0, min(f.p0 - a.window + 1, f.hi)) : 0;
    const int te = (f.hi + kFewKeys - 1) / kFewKeys, sinks = a.window ? min(a.sinks, f.hi) : 0;
    f.tw = min(f.lo / kFewKeys, te);
    f.ns = min((sinks + kFewKeys - 1) / kFewKeys, f.tw);
    f.nt = f.ns + (f.lo < f.hi ? te - f.tw : sinks > f.ns * kFewKeys ? 1 : 0);
    return f;
}

template <int D>
struct FewSmem {
    static constexpr int kTile = kFewKeys * D * 2;
    static constexpr int kChunk = kFewKeys * 128;  // one 64-column chunk of a tile
    static constexpr int kRow = D + 4;
    static constexpr size_t kRing = 0;
    static constexpr size_t kO = size_t(kFewStages) * 2 * kTile;
    static constexpr size_t kM = kO + size_t(kFewWarps) * 16 * kRow * 4;
    static constexpr size_t kL = kM + kFewWarps * 16 * 4;
    static constexpr size_t kBar = kL + kFewWarps * 16 * 4;
    static constexpr size_t kTotal = kBar + kFewStages * 8 + 16 + 1024;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma_16bit(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (KvTraits<T>::kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// kGroups row groups; the other factor of the four warps is parts of a tile's keys.  kTwo: weights as two numbers.
// Up to 32 rows the second product is not seen (4 tokens over 16448 keys: 20 to 22 us both ways); with 33 to 64, or
// in chunks, it takes up to a fifth (17 tokens, 32768 keys: 91.5 us against 76.7), and round_weights leaves it out.
template <typename T, typename Out, int D, int kGroups, bool kTwo>
__global__ void __launch_bounds__(32 * kFewWarps, 2)
    window_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const WindowFewArgs f) {
    using Sm = FewSmem<D>;
    constexpr int KS = D / 16, kParts = kFewWarps / kGroups, kMine = kFewKeys / kParts;  // keys of a warp
    extern __shared__ uint8_t few_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sm::kBar);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + Sm::kBar + kFewStages * 8);
    float* so = reinterpret_cast<float*>(smem + Sm::kO);
    float* sm = reinterpret_cast<float*>(smem + Sm::kM);
    float* sl = reinterpret_cast<float*>(smem + Sm::kL);
    const WindowArgs& a = f.w;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = warp % kGroups, part = warp / kGroups;
    const int split = blockIdx.x, head = blockIdx.y % a.kv_heads, chunk = blockIdx.y / a.kv_heads, b = blockIdx.z;
    const int i0 = chunk * f.tokens, n = min(f.tokens, a.n - i0), nrep = a.q_heads / a.kv_heads, rows = n * nrep;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) mbar_init(&full[s], 1);
        *abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint64_t deadline = globaltimer_ns() + kWaitLimitNs;
    const FewSpan sp = few_span(a, b, i0, n);
    const int t0 = static_cast<int>(static_cast<long long>(sp.nt) * split / f.splits);
    const int t1 = static_cast<int>(static_cast<long long>(sp.nt) * (split + 1) / f.splits);
    auto key0 = [&](int i) { return (i < sp.ns ? i : sp.tw + (i - sp.ns)) * kFewKeys; };
    auto fetch = [&](int i) {  // tile t0 + i into its stage (one thread)
        const int s = i % kFewStages, k0 = key0(t0 + i);
        uint8_t* dst = smem + Sm::kRing + s * 2 * Sm::kTile;
        mbar_arrive_expect_tx(&full[s], 2 * Sm::kTile);
        for (int c = 0; c < D / 64; ++c) {
            tma_load_4d(dst + c * Sm::kChunk, &tm_k, &full[s], 64 * c, head, k0, b);
            tma_load_4d(dst + Sm::kTile + c * Sm::kChunk, &tm_v, &full[s], 64 * c, head, k0, b);
        }
    };
    if (threadIdx.x == 0)
        for (int i = 0; i < min(kFewStages, t1 - t0); ++i) fetch(i);
    // Queries as A operands: rows g, g + 8 of the group; row r is token r / nrep, head r % nrep.
    uint32_t qa[KS][4];
    int p[2];  // positions of the two rows
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = group * 16 + g + 8 * u, i = r / nrep;
        p[u] = r < rows ? sp.p0 + i : -1;  // a row that is not there sees nothing
        const T* q = static_cast<const T*>(a.q) + b * a.q_batch + static_cast<long long>(i0 + i) * a.q_stride + (head * nrep + r % nrep) * D;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            qa[j][u] = r < rows ? *reinterpret_cast<const uint32_t*>(q + 16 * j + 2 * t) : 0u;
            qa[j][2 + u] = r < rows ? *reinterpret_cast<const uint32_t*>(q + 16 * j + 2 * t + 8) : 0u;
        }
    }
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    int taken = 0;
    for (; taken < t1 - t0; ++taken) {
        const int s = taken % kFewStages, k0 = key0(t0 + taken);
        if (!mbar_wait_bounded(&full[s], (taken / kFewStages) & 1, deadline, abort)) {
            *abort = 1;
            *reinterpret_cast<volatile int*>(f.err) = KERR_TIMEOUT_FULL;
        }
        uint8_t* tile = smem + Sm::kRing + s * 2 * Sm::kTile;
        const bool edge = k0 + kFewKeys > sp.p0 + 1 || k0 + kFewKeys > sp.hi || (k0 < sp.lo + n && a.window);
        if (k0 + kFewKeys > sp.hi || (k0 < sp.lo && k0 + kFewKeys > a.sinks)) {
            // Rows of V that no query sees may hold anything, and 0 * NaN is NaN.
            for (int r = threadIdx.x >> 3; r < kFewKeys; r += 4 * kFewWarps) {
                if (k0 + r < sp.hi && (k0 + r >= sp.lo || k0 + r < a.sinks)) continue;
                for (int c = 0; c < D / 64; ++c)
                    *reinterpret_cast<uint4*>(tile + Sm::kTile + c * Sm::kChunk + r * 128 + (threadIdx.x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();  // before a later copy into these rows
            __syncthreads();
        }
        const uint32_t kb = smem_u32(tile), vb = kb + Sm::kTile;
#pragma unroll
        for (int kk = 0; kk < kMine / 16; ++kk) {
            const int kr = part * kMine + kk * 16;  // first of 16 keys of the tile
            float c[2][4] = {};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const int key = kr + (lane >> 4) * 8 + (lane & 7), ch = 2 * j + ((lane >> 3) & 1);
                uint32_t r[4];
                ldmatrix4(r, kb + (ch >> 3) * Sm::kChunk + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
                mma_16bit<T>(c[0], qa[j], r[0], r[1]);
                mma_16bit<T>(c[1], qa[j], r[2], r[3]);
            }
            if (edge) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + kr + 8 * n + 2 * t + (e & 1), pr = p[e >> 1];
                        const bool seen = key <= pr && key < sp.hi && (!a.window || key > pr - a.window || key < a.sinks);
                        if (!seen) c[n][e] = -INFINITY;
                    }
            }
            float mx[2], ms[2], fac[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                mx[u] = fmaxf(fmaxf(c[0][2 * u], c[0][2 * u + 1]), fmaxf(c[1][2 * u], c[1][2 * u + 1])) * a.scale_log2;
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
                mx[u] = fmaxf(mx[u], m[u]);
                ms[u] = mx[u] == -INFINITY ? 0.f : mx[u];
                fac[u] = m[u] == mx[u] ? 1.f : exp2f(m[u] - ms[u]);
                m[u] = mx[u];
                l[u] *= fac[u];
            }
            // Weights as two numbers, hi + lo (TcWindow says why).  Those of fp16 lie in [0, 2^15], so that small ones keep
            // their bits.
            uint32_t pa[4], pb[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float up = KvTraits<T>::kBf16 ? ms[u] : ms[u] - 15.f;
                    const float e0 = exp2f(fmaf(c[n][2 * u], a.scale_log2, -up)), e1 = exp2f(fmaf(c[n][2 * u + 1], a.scale_log2, -up));
                    l[u] += e0 + e1;
                    pa[2 * n + u] = pack_16bit<T>(e0, e1);
                    if constexpr (kTwo) {
                        const float2 hi = unpack_16bit<T>(pa[2 * n + u]);
                        pb[2 * n + u] = pack_16bit<T>(e0 - hi.x, e1 - hi.y);
                    }
                }
            if (__any_sync(0xffffffffu, fac[0] != 1.f || fac[1] != 1.f))
#pragma unroll
                for (int j = 0; j < D / 8; ++j) o[j][0] *= fac[0], o[j][1] *= fac[0], o[j][2] *= fac[1], o[j][3] *= fac[1];
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const int key = kr + ((lane >> 3) & 1) * 8 + (lane & 7), ch = 2 * j + (lane >> 4);
                uint32_t r[4];
                ldmatrix4_trans(r, vb + (ch >> 3) * Sm::kChunk + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
                mma_16bit<T>(o[2 * j], pa, r[0], r[1]);
                mma_16bit<T>(o[2 * j + 1], pa, r[2], r[3]);
                if constexpr (kTwo) {
                    mma_16bit<T>(o[2 * j], pb, r[0], r[1]);
                    mma_16bit<T>(o[2 * j + 1], pb, r[2], r[3]);
                }
            }
        }
        __syncthreads();
        if (*abort) break;  // raised before the barrier: every thread sees it
        if (threadIdx.x == 0 && taken + kFewStages < t1 - t0) fetch(taken + kFewStages);
    }
    if (*abort) {  // the copies in flight land before the block ends (every stage rests on its last phase)
        if (threadIdx.x == 0)
            for (int i = taken; i < min(taken + kFewStages, t1 - t0); ++i)
                while (!mbar_try_wait(&full[i % kFewStages], (i / kFewStages) & 1) && globaltimer_ns() < deadline + kWaitLimitNs / 2) {
                }
        __syncthreads();
        return;
    }
    // The warps' sums to shared memory; the key parts of a row group are added up.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        float* row = so + (warp * 16 + g + 8 * u) * Sm::kRow;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(row + 8 * j + 2 * t) = make_float2(o[j][2 * u], o[j][2 * u + 1]);
        if (t == 0) sm[warp * 16 + g + 8 * u] = m[u], sl[warp * 16 + g + 8 * u] = l[u];
    }
    __syncthreads();
    const long long item = ((static_cast<long long>(b) * f.chunks + chunk) * a.kv_heads + head) * f.splits + split;
    float* parts = f.parts + item * (f.tokens * nrep) * (D + 2);
    for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * kFewWarps) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, w0 = r / 16, rr = r % 16;
        float M = -INFINITY, ls = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kParts; ++k) M = fmaxf(M, sm[(w0 + k * kGroups) * 16 + rr]);
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            const int w = (w0 + k * kGroups) * 16 + rr;
            const float e = M == -INFINITY ? 0.f : exp2f(sm[w] - M);
            const float4 y = *reinterpret_cast<const float4*>(so + w * Sm::kRow + d);
            ls = fmaf(sl[w], e, ls);
            x.x = fmaf(y.x, e, x.x), x.y = fmaf(y.y, e, x.y), x.z = fmaf(y.z, e, x.z), x.w = fmaf(y.w, e, x.w);
        }
        if (f.splits == 1) {
            const float inv = ls != 0.f ? 1.f / ls : 0.f;
            Out* out = static_cast<Out*>(a.out) + ((static_cast<long long>(b) * a.n + i0 + r / nrep) * a.q_heads + head * nrep + r % nrep) * D + d;
            tc_store4(out, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        } else {
            float* row = parts + r * (D + 2);
            *reinterpret_cast<float2*>(row + d) = make_float2(x.x, x.y);
            *reinterpret_cast<float2*>(row + d + 2) = make_float2(x.z, x.w);
            if (d == 0) row[D] = M, row[D + 1] = ls;
        }
    }
}

// Block (row, KV head, entry): adds up the row's splits, in order.
template <typename Out, int D>
__global__ void __launch_bounds__(D) window_join_kernel(const WindowFewArgs f) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const WindowArgs& a = f.w;
    const int r = blockIdx.x, head = blockIdx.y, b = blockIdx.z, nrep = a.q_heads / a.kv_heads, rows = f.tokens * nrep;
    const float* row = f.parts + (((static_cast<long long>(b) * f.chunks + r / rows) * a.kv_heads + head) * f.splits * rows + r % rows) * (D + 2);
    const long long step = static_cast<long long>(rows) * (D + 2);
    float M = -INFINITY, l = 0.f, o = 0.f;
    // Eight splits at a time, all loads of them in flight together.
    for (int s0 = 0; s0 < f.splits; s0 += 8) {
        float x[8], m[8], ls[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < f.splits) {
                const float* q = row + (s0 + k) * step;
                x[k] = __ldcg(q + threadIdx.x), m[k] = __ldcg(q + D), ls[k] = __ldcg(q + D + 1);
            } else {
                x[k] = 0.f, m[k] = -INFINITY, ls[k] = 0.f;
            }
        float top = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, m[k]);
        if (top == -INFINITY) continue;
        const float fac = exp2f(M - top);
        l *= fac, o *= fac, M = top;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float e = exp2f(m[k] - top);
            l = fmaf(ls[k], e, l);
            o = fmaf(x[k], e, o);
        }
    }
    Out* out = static_cast<Out*>(a.out) + ((static_cast<long long>(b) * a.n + r / nrep) * a.q_heads + head * nrep + r % nrep) * D;
    out[threadIdx.x] = KvTraits<Out>::from_float(l != 0.f ? o / l : 0.f);
}

}  // namespace lg
