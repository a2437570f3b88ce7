// longctx_api.cu - C ABI of the long-context operators (include/ligguf_cuda_attn.h): rotary positions
// and norms in one pass, the 4-bit cache, windowed attention.  Handles, argument checks, dispatch.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "ligguf_cuda_attn.h"
#include "api_util.h"
#include "common.cuh"
#include "flash_tc.cuh"
#include "kv4.cuh"
#include "kv4_decode.cuh"
#include "rope_rows.cuh"
#include "window.cuh"

using lgapi::DeviceGuard;
using lgapi::fail;

namespace {

// Longest windows, prompts and key ranges of the windowed attention: sums of a few of them stay below 2^31.
constexpr int kWindowMost = 1 << 28;
constexpr double kTwoPi = 6.283185307179586476925286766559;

bool type_ok(int t) { return t >= LIGGUF_KV_F32 && t <= LIGGUF_KV_BF16; }
size_t type_size(int t) { return t == LIGGUF_KV_F32 ? 4 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A row stride of `elems`-wide rows of `type` (0 = packed): at least the row, and 16-byte aligned.
int check_stride(long long* stride, long long elems, int type, const char* what) {
    if (*stride == 0) *stride = elems;
    if (*stride < elems) return fail(LIGGUF_ATTN_EINVAL, "%s %lld is less than a row's %lld elements", what, *stride, elems);
    if (*stride * static_cast<long long>(type_size(type)) % 16)
        return fail(LIGGUF_ATTN_EINVAL, "%s %lld is not a multiple of 16 bytes", what, *stride);
    return LIGGUF_ATTN_OK;
}

int check_device(int device) {
    int n = 0;
    LG_CUDA(cudaGetDeviceCount(&n));
    if (device < 0 || device >= n) return fail(LIGGUF_ATTN_EINVAL, "device %d of %d", device, n);
    return LIGGUF_ATTN_OK;
}

int check_heads(int n_heads, int n_kv_heads) {
    if (n_heads < 1 || n_kv_heads < 1) return fail(LIGGUF_ATTN_EINVAL, "n_heads and n_kv_heads must be positive");
    if (n_heads % n_kv_heads)
        return fail(LIGGUF_ATTN_EINVAL, "n_heads %d is not a multiple of n_kv_heads %d", n_heads, n_kv_heads);
    if (n_heads > 4096) return fail(LIGGUF_ATTN_EINVAL, "n_heads %d (at most 4096)", n_heads);
    return LIGGUF_ATTN_OK;
}

int check_rope(const ligguf_rope_cfg& r) {
    if (r.head_dim != 64 && r.head_dim != 128)
        return fail(LIGGUF_ATTN_EUNSUPPORTED, "head_dim %d (supported: 64, 128)", r.head_dim);
    if (r.rope_dim < 0 || r.rope_dim > r.head_dim || (r.rope_dim & 1))
        return fail(LIGGUF_ATTN_EINVAL, "rope_dim %d is not an even number in [0, %d]", r.rope_dim, r.head_dim);
    if (r.layout != LIGGUF_ROPE_ADJACENT && r.layout != LIGGUF_ROPE_HALVES)
        return fail(LIGGUF_ATTN_EINVAL, "rope layout %d", r.layout);
    if (r.scaling < LIGGUF_ROPE_SCALE_NONE || r.scaling > LIGGUF_ROPE_SCALE_BLEND)
        return fail(LIGGUF_ATTN_EINVAL, "rope scaling %d", r.scaling);
    if (!(r.magnitude >= 0.f) || std::isinf(r.magnitude)) return fail(LIGGUF_ATTN_EINVAL, "rope magnitude %g", r.magnitude);
    if (r.freq || r.rope_dim == 0) return LIGGUF_ATTN_OK;
    if (!(r.base > 0.f) || std::isinf(r.base)) return fail(LIGGUF_ATTN_EINVAL, "rope base %g", r.base);
    if (r.scaling != LIGGUF_ROPE_SCALE_NONE && (!(r.factor >= 1.f) || std::isinf(r.factor)))
        return fail(LIGGUF_ATTN_EINVAL, "rope scaling factor %g is not at least 1", r.factor);
    if (r.scaling == LIGGUF_ROPE_SCALE_BLEND && (r.orig_context < 1 || !(r.low < r.high)))
        return fail(LIGGUF_ATTN_EINVAL, "rope blend needs orig_context > 0 and low < high (%d, %g, %g)", r.orig_context,
                    r.low, r.high);
    return LIGGUF_ATTN_OK;
}

// Waits for what the set-up calls put on the legacy stream (copies from pageable memory, which return when they are
// staged, and memsets): the callers' streams may be non-blocking ones, which do not wait for that stream.
int set_up_done() {
    LG_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
    return LIGGUF_ATTN_OK;
}

// Turns per position of every pair, in device memory.
int make_turns(const ligguf_rope_cfg& r, double** out) {
    double t[64];
    const int pairs = r.rope_dim / 2;
    for (int i = 0; i < pairs; ++i) {
        double f = 0.0;
        if (r.freq) {
            f = r.freq[i];
        } else {
            f = std::pow(static_cast<double>(r.base), -2.0 * i / r.rope_dim);
            if (r.scaling == LIGGUF_ROPE_SCALE_LINEAR) {
                f /= r.factor;
            } else if (r.scaling == LIGGUF_ROPE_SCALE_BLEND) {
                const double turns = r.orig_context * f / kTwoPi;
                const double g = std::min(1.0, std::max(0.0, (turns - r.low) / (double(r.high) - r.low)));
                f *= g + (1.0 - g) / r.factor;
            }
        }
        t[i] = f / kTwoPi;
    }
    if (cudaMalloc(reinterpret_cast<void**>(out), sizeof(t)) != cudaSuccess)
        return fail(LIGGUF_ATTN_ENOMEM, "rotation table");
    LG_CUDA(cudaMemcpy(*out, t, pairs * sizeof(double), cudaMemcpyHostToDevice));
    return set_up_done();
}

int rope_layout(const ligguf_rope_cfg& r) {
    if (r.layout == LIGGUF_ROPE_ADJACENT) return lg::kRopeAdjacent;
    return r.rope_dim % 16 == 0 ? lg::kRopeHalves : lg::kRopeHalvesOdd;
}

template <typename In, typename Out, int D, int kLayout, int kTake>
int launch_rope_pairs(lg::RopeRowsArgs& a, cudaStream_t st) {
    const int items = ((a.q_heads + kTake - 1) / kTake + (a.kv_heads + kTake - 1) / kTake) * (D / 16);
    a.parts = (items + 255) / 256;
    const int threads = std::max(64, ((items + a.parts - 1) / a.parts + 31) / 32 * 32);
    const long long blocks = static_cast<long long>(a.n) * a.parts;
    if (blocks > INT32_MAX) return fail(LIGGUF_ATTN_EUNSUPPORTED, "%d tokens in one call", a.n);
    lg::rope_pairs_kernel<In, Out, D, kLayout, kTake><<<static_cast<unsigned>(blocks), threads, 0, st>>>(a);
    LG_CUDA(cudaGetLastError());
    return LIGGUF_ATTN_OK;
}
template <typename In, typename Out, int D, int kLayout>
int launch_rope_layout(lg::RopeRowsArgs& a, cudaStream_t st) {
    if constexpr (kLayout != lg::kRopeHalvesOdd)
        if (!a.tiles && a.n >= 32) return launch_rope_pairs<In, Out, D, kLayout, sizeof(In) == 4 ? 1 : 2>(a, st);
    // Few tokens: their heads over several blocks, which take less time than a large one.
    const int units = ((a.q ? a.q_heads : 0) + a.kv_heads * (a.v ? 2 : 1)) * (D / 8);
    const int threads = a.n >= 128 ? 256 : 128;
    a.units_per_block = a.n >= 128 ? (units + 31) / 32 * 32 : threads;
    a.parts = (units + a.units_per_block - 1) / a.units_per_block;
    const long long blocks = static_cast<long long>(a.n) * a.parts;
    if (blocks > INT32_MAX) return fail(LIGGUF_ATTN_EUNSUPPORTED, "%d tokens in one call", a.n);
    lg::rope_units_kernel<In, Out, D, kLayout><<<static_cast<unsigned>(blocks), threads, 0, st>>>(a);
    LG_CUDA(cudaGetLastError());
    return LIGGUF_ATTN_OK;
}
template <typename In, typename Out, int D>
int launch_rope_rows(lg::RopeRowsArgs& a, int layout, cudaStream_t st) {
    if (layout == lg::kRopeHalvesOdd) return launch_rope_layout<In, Out, D, lg::kRopeHalvesOdd>(a, st);
    return layout == lg::kRopeAdjacent ? launch_rope_layout<In, Out, D, lg::kRopeAdjacent>(a, st)
                                       : launch_rope_layout<In, Out, D, lg::kRopeHalves>(a, st);
}
template <typename In, typename Out>
int launch_rope_rows_d(lg::RopeRowsArgs& a, const ligguf_rope_cfg& r, cudaStream_t st) {
    return r.head_dim == 64 ? launch_rope_rows<In, Out, 64>(a, rope_layout(r), st)
                            : launch_rope_rows<In, Out, 128>(a, rope_layout(r), st);
}
template <typename In>
int launch_rope_rows_o(lg::RopeRowsArgs& a, const ligguf_rope_cfg& r, int out_type, cudaStream_t st) {
    switch (out_type) {
        case LIGGUF_KV_F32: return launch_rope_rows_d<In, float>(a, r, st);
        case LIGGUF_KV_F16: return launch_rope_rows_d<In, __half>(a, r, st);
        default: return launch_rope_rows_d<In, __nv_bfloat16>(a, r, st);
    }
}
int launch_rope_rows_any(lg::RopeRowsArgs& a, const ligguf_rope_cfg& r, int in_type, int out_type, cudaStream_t st) {
    switch (in_type) {
        case LIGGUF_KV_F32: return launch_rope_rows_o<float>(a, r, out_type, st);
        case LIGGUF_KV_F16: return launch_rope_rows_o<__half>(a, r, out_type, st);
        default: return launch_rope_rows_o<__nv_bfloat16>(a, r, out_type, st);
    }
}

int make_err_words(int** h_err, int** d_err) {
    if (cudaHostAlloc(reinterpret_cast<void**>(h_err), 64, cudaHostAllocMapped) != cudaSuccess)
        return fail(LIGGUF_ATTN_ENOMEM, "mapped error words");
    std::memset(*h_err, 0, 64);
    LG_CUDA(cudaHostGetDevicePointer(reinterpret_cast<void**>(d_err), *h_err, 0));
    return LIGGUF_ATTN_OK;
}

}  // namespace

struct ligguf_qk_rope {
    ligguf_qk_rope_cfg cfg;
    double* turns = nullptr;
};

struct ligguf_kv4 {
    ligguf_kv4_cfg cfg;
    int nrep = 0;
    long long tiles_per_head = 0;
    size_t tile_bytes = 0;
    uint8_t* tiles = nullptr;
    double* turns = nullptr;
    float* gammas = nullptr;          // [n_layers][2][head_dim]
    unsigned char* norm_set = nullptr;  // [n_layers], host
    float* parts = nullptr;  // decode: partial results of items that several blocks share
    int* tickets = nullptr;  // decode: [n_seqs * n_kv_heads] blocks done with such an item; zero between calls
    int num_sms = 0;
    int *h_err = nullptr, *d_err = nullptr;
    uint8_t* seq_tiles(int layer, int seq) const {
        return tiles + (static_cast<size_t>(layer) * cfg.n_seqs + seq) * cfg.n_kv_heads * tiles_per_head * tile_bytes;
    }
};

struct ligguf_window {
    ligguf_window_cfg cfg;
    float* parts = nullptr;  // few rows: partial sums of the splits
    int num_sms = 0;
    int *h_err = nullptr, *d_err = nullptr;
};

namespace {

int kv4_check(const ligguf_kv4* h, int layer, int seq, int n_seqs, int pos0, int n) {
    if (!h) return fail(LIGGUF_ATTN_EINVAL, "null handle");
    const ligguf_kv4_cfg& c = h->cfg;
    if (layer < 0 || layer >= c.n_layers) return fail(LIGGUF_ATTN_EINVAL, "layer %d out of range", layer);
    if (seq < 0 || n_seqs < 0 || n_seqs > c.n_seqs || seq > c.n_seqs - n_seqs)
        return fail(LIGGUF_ATTN_EINVAL, "sequences [%d, %d + %d) outside [0, %d)", seq, seq, n_seqs, c.n_seqs);
    if (n < 0 || pos0 < 0 || n > c.n_context || pos0 > c.n_context - n)
        return fail(LIGGUF_ATTN_EINVAL, "positions [%d, %d + %d) outside [0, %d)", pos0, pos0, n, c.n_context);
    return LIGGUF_ATTN_OK;
}

template <typename In, int D, int NREP>
int launch_kv4_decode(const ligguf_kv4* h, lg::Kv4DecodeArgs& a, cudaStream_t st) {
    using Sm = lg::Kv4DecodeSmem<D, NREP>;
    auto kern = lg::kv4_decode_kernel<In, D, NREP>;
    static bool attr_done[64] = {};
    const int device = h->cfg.device;
    if (device >= 64 || !attr_done[device]) {
        LG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Sm::total(h->num_sms * lg::kv4_blocks_per_sm(NREP)))));
        if (device < 64) attr_done[device] = true;
    }
    // As many blocks as fit at once, fewer when the longest visible contexts do not fill them.
    const long long keys = std::min<long long>(h->cfg.n_context, a.window ? 2ll * lg::kKv4Tile + a.window + a.sinks : INT32_MAX);
    const long long units = (keys / lg::kKv4Tile + 2 + lg::kKv4ItemUnits) * a.kv_heads * a.n_rows;
    const int slots = h->num_sms * lg::kv4_blocks_per_sm(NREP);
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(std::min<long long>(slots, std::max<long long>(1, units / lg::kKv4MinUnits))));
    a.per_block = 1.0f / static_cast<float>(lc.gridDim.x);
    lc.blockDim = dim3(32 * Sm::kWarps);
    lc.dynamicSmemBytes = Sm::total(slots);
    lc.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    LG_CUDA(cudaLaunchKernelEx(&lc, kern, a));
    return LIGGUF_ATTN_OK;
}
template <typename In, int D>
int launch_kv4_decode_n(const ligguf_kv4* h, lg::Kv4DecodeArgs& a, cudaStream_t st) {
    switch (h->nrep) {
        case 1: return launch_kv4_decode<In, D, 1>(h, a, st);
        case 2: return launch_kv4_decode<In, D, 2>(h, a, st);
        case 4: return launch_kv4_decode<In, D, 4>(h, a, st);
        default: return launch_kv4_decode<In, D, 8>(h, a, st);
    }
}
template <typename In>
int launch_kv4_decode_d(const ligguf_kv4* h, lg::Kv4DecodeArgs& a, cudaStream_t st) {
    return h->cfg.rope.head_dim == 64 ? launch_kv4_decode_n<In, 64>(h, a, st) : launch_kv4_decode_n<In, 128>(h, a, st);
}

lg::Kv4IoArgs kv4_io(const ligguf_kv4* h, int layer, int seq, int n_seqs, int pos0, int n, void* k, void* v) {
    lg::Kv4IoArgs a = {};
    a.tiles = h->seq_tiles(layer, seq);
    a.tiles_per_head = h->tiles_per_head;
    a.kv_heads = h->cfg.n_kv_heads;
    a.n_seqs = n_seqs;
    a.pos0 = pos0;
    a.n = n;
    a.k = k;
    a.v = v;
    return a;
}

// Blocks of 256 threads for `work` items; the grid's x limit is 2^31 - 1.
int io_grid(long long work, dim3* grid) {
    const long long blocks = (work + 255) / 256;
    if (blocks > INT32_MAX) return fail(LIGGUF_ATTN_EUNSUPPORTED, "%lld items in one call", work);
    *grid = dim3(static_cast<unsigned>(blocks), 2);
    return LIGGUF_ATTN_OK;
}

template <bool kLoad>
int kv4_blocks(ligguf_kv4* h, int layer, int seq0, int n_seqs, int pos0, int n, void* k, void* v, void* stream) {
    int rc = kv4_check(h, layer, seq0, n_seqs, pos0, n);
    if (rc || n == 0 || n_seqs == 0) return rc;
    if (!k || !v) return fail(LIGGUF_ATTN_EINVAL, "null block pointer");
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1)
        return fail(LIGGUF_ATTN_EINVAL, "blocks must be 2-byte aligned");
    const ligguf_kv4_cfg& c = h->cfg;
    DeviceGuard dg(c.device);
    const int D = c.rope.head_dim;
    dim3 grid;
    if ((rc = io_grid(static_cast<long long>(n_seqs) * n * c.n_kv_heads * (D / 32), &grid))) return rc;
    const lg::Kv4IoArgs a = kv4_io(h, layer, seq0, n_seqs, pos0, n, k, v);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (D == 64)
        lg::kv4_blocks_kernel<64, kLoad><<<grid, 256, 0, st>>>(a);
    else
        lg::kv4_blocks_kernel<128, kLoad><<<grid, 256, 0, st>>>(a);
    LG_CUDA(cudaGetLastError());
    return LIGGUF_ATTN_OK;
}

// [batch][rows][heads][D] of 16-bit elements; boxes of 64 columns x box_rows rows of one head.
int make_rows_tmap(CUtensorMap* m, const void* base, bool bf16, int D, int heads, long long stride, int rows, int batch,
                   long long batch_stride, int box_rows) {
    auto enc = lgapi::tensor_map_encoder();
    if (!enc) return fail(LIGGUF_ATTN_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(rows), cuuint64_t(batch)};
    cuuint64_t strides[3] = {cuuint64_t(D) * 2, cuuint64_t(stride) * 2, cuuint64_t(batch_stride) * 2};
    cuuint32_t box[4] = {64u, 1u, cuuint32_t(box_rows), 1u};
    cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
    const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                           dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LIGGUF_ATTN_EINVAL, "no tensor map for %d rows of stride %lld (%d)", rows, stride, int(r));
    return LIGGUF_ATTN_OK;
}

template <typename T, typename Out, int D, bool kTwo>
int launch_window_tc(const ligguf_window* h, const lg::WindowArgs& w, cudaStream_t st) {
    constexpr bool bf16 = lg::KvTraits<T>::kBf16;
    const int device = h->cfg.device;
    alignas(64) CUtensorMap tq, tk, tv;
    int rc;
    if ((rc = make_rows_tmap(&tq, w.q, bf16, D, w.q_heads, w.q_stride, w.n, w.batch, w.q_batch, lg::kTcRows)) ||
        (rc = make_rows_tmap(&tk, w.k, bf16, D, w.kv_heads, w.k_stride, w.m, w.batch, w.k_batch, lg::kTcKeys)) ||
        (rc = make_rows_tmap(&tv, w.v, bf16, D, w.kv_heads, w.v_stride, w.m, w.batch, w.v_batch, lg::kTcKeys)))
        return rc;
    auto kern = lg::flash_tc_kernel<D, lg::TcWindow<T, Out, kTwo>>;
    static int resident[64] = {};
    int slots = device < 64 ? resident[device] : 0;
    if (slots == 0) {
        LG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lg::TcSmem<D>::kTotal)));
        // The warpgroups' register shares (setmaxnreg) come out of the registers the CTA launched with.
        cudaFuncAttributes fa{};
        LG_CUDA(cudaFuncGetAttributes(&fa, kern));
        constexpr int need = lg::kTcRegsIssue + 2 * lg::kTcRegsSoftmax + lg::kTcRegsEpilogue;
        if (fa.numRegs * 4 < need)
            return fail(LIGGUF_ATTN_ECUDA, "windowed attention kernel built with %d registers per thread, %d needed", fa.numRegs,
                        (need + 3) / 4);
        int sms = 0, per_sm = 0;
        LG_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        LG_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, lg::kTcThreads, lg::TcSmem<D>::kTotal));
        if (per_sm < 1) return fail(LIGGUF_ATTN_ECUDA, "the windowed attention kernel does not fit on an SM");
        slots = sms * per_sm;
        if (device < 64) resident[device] = slots;
    }
    lg::TcArgs a = {};
    a.q_heads = w.q_heads;
    a.kv_heads = w.kv_heads;
    a.batch = w.batch;
    a.q_seq = w.n;
    a.kv_seq = w.m;
    a.lens = w.lens;
    a.causal = 1;
    a.nrep = w.q_heads / w.kv_heads;
    a.scale_log2 = w.scale_log2;
    a.err = h->d_err;
    a.pos0 = w.pos0;
    a.window = w.window;
    a.sinks = w.sinks;
    a.wout = w.out;
    const long long items = static_cast<long long>(w.q_heads) * ((w.n + lg::kTcRows - 1) / lg::kTcRows) * w.batch;
    if (items > INT32_MAX) return fail(LIGGUF_ATTN_EUNSUPPORTED, "%d x %d rows of %d heads in one call", w.batch, w.n, w.q_heads);
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(std::min<long long>(items, slots)));
    lc.blockDim = dim3(lg::kTcThreads);
    lc.dynamicSmemBytes = lg::TcSmem<D>::kTotal;
    lc.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    LG_CUDA(cudaLaunchKernelEx(&lc, kern, tq, tk, tv, a));
    return LIGGUF_ATTN_OK;
}
// CTAs of the few-rows form that leave partial sums: one wave of two an SM at most.
long long few_most_items(int sms) { return 2ll * sms; }

template <typename T, typename Out, int D, int kGroups, bool kTwo>
int launch_window_few(const ligguf_window* h, const lg::WindowArgs& w, cudaStream_t st) {
    constexpr bool bf16 = lg::KvTraits<T>::kBf16;
    const int device = h->cfg.device;
    alignas(64) CUtensorMap tk, tv;
    int rc;
    if ((rc = make_rows_tmap(&tk, w.k, bf16, D, w.kv_heads, w.k_stride, w.m, w.batch, w.k_batch, lg::kFewKeys)) ||
        (rc = make_rows_tmap(&tv, w.v, bf16, D, w.kv_heads, w.v_stride, w.m, w.batch, w.v_batch, lg::kFewKeys)))
        return rc;
    auto kern = lg::window_few_kernel<T, Out, D, kGroups, kTwo>;
    static bool attr_done[64] = {};
    if (device >= 64 || !attr_done[device]) {
        LG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lg::FewSmem<D>::kTotal)));
        if (device < 64) attr_done[device] = true;
    }
    lg::WindowFewArgs f = {};
    f.w = w;
    f.tokens = std::min(w.n, lg::kFewRows / (w.q_heads / w.kv_heads));
    f.chunks = (w.n + f.tokens - 1) / f.tokens;
    f.parts = h->parts;
    f.err = h->d_err;
    // Splits: one wave of two CTAs an SM, at least two tiles each (4 tokens over 16448 keys: 19.2 us; with one CTA
    // an SM 20.8, or 22.1 with a ring of three tiles; with 1.5 20.1).
    const long long pairs = static_cast<long long>(w.batch) * f.chunks * w.kv_heads;
    const long long keys = w.window ? std::min<long long>(w.m, static_cast<long long>(w.window) + w.n + w.sinks + 2 * lg::kFewKeys) : w.m;
    const long long tiles = (keys + lg::kFewKeys - 1) / lg::kFewKeys;
    f.splits = static_cast<int>(std::max(1ll, std::min(few_most_items(h->num_sms) / pairs, (tiles + 1) / 2)));
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(f.splits, w.kv_heads * f.chunks, w.batch);
    lc.blockDim = dim3(32 * lg::kFewWarps);
    lc.dynamicSmemBytes = lg::FewSmem<D>::kTotal;
    lc.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    LG_CUDA(cudaLaunchKernelEx(&lc, kern, tk, tv, f));
    if (f.splits == 1) return LIGGUF_ATTN_OK;
    lc.gridDim = dim3(w.n * (w.q_heads / w.kv_heads), w.kv_heads, w.batch);
    lc.blockDim = dim3(D);
    lc.dynamicSmemBytes = 0;
    LG_CUDA(cudaLaunchKernelEx(&lc, lg::window_join_kernel<Out, D>, f));
    return LIGGUF_ATTN_OK;
}

template <typename T, typename Out, int D>
int launch_window_d(const ligguf_window* h, const lg::WindowArgs& a, cudaStream_t st) {
    // Few rows a KV head: all of them against each key tile once, the keys split over the SMs.  Up to 64 rows this
    // is bound by K and V; the tensor-core form reads them once a head and gives a head's keys to one SM.  More rows
    // go in chunks of 64 where the tensor-core form would leave most SMs without work: one of its SMs takes about
    // 10 us for 1024 keys of a head, a chunk 24 us of one SM's time, and there is a join.  Hence the bounds of a
    // quarter as many chunks as SMs and of 1024 keys.  Measured, one sequence, head_dim 128, us in chunks / on the
    // tensor cores with 1024, 4096 and 32768 keys:
    //   32 and 8 heads   17 tokens  12.0 / 17.3   24.4 / 49.3   91.5 / 344     (rounded 11.5 / 15.2, 22.5 / 42.1, 76.9 / 297)
    //                    64 tokens  16.2 / 17.4   34.9 / 49.5   165 / 344
    //   16 and 16       100 tokens  15.7 / 17.4   34.1 / 50.1   164 / 346
    //    8 and 2        288 tokens  16.6 / 18.0   33.6 / 49.4   182 / 342
    //   16 and 2        288 tokens  18.3 / 18.3   49.6 / 49.9   345 / 344     (rounded 16.1 / 16.1, 42.0 / 42.0, 290 / 289)
    //    4 and 1        288 tokens  14.8 / 17.9   23.5 / 49.2   98 / 342
    // Never more than 2 % slower at 9 to 288 tokens of seven such layouts.  With 512 keys it would be (64 tokens of 32
    // and 8 heads, rounded: 12.7 / 10.7), and so it can be where entries are that short under a large m: their lengths
    // lie in device memory.
    const int nrep = a.q_heads / a.kv_heads;
    const long long rows = static_cast<long long>(a.n) * nrep;
    const long long keys = a.window ? std::min<long long>(a.m, static_cast<long long>(a.window) + a.n + a.sinks) : a.m;
    bool few = rows <= lg::kFewRows;
    if (!few && nrep <= lg::kFewRows && keys >= 1024) {
        const long long tokens = lg::kFewRows / nrep, chunks = (a.n + tokens - 1) / tokens;
        few = chunks * a.batch * a.kv_heads <= h->num_sms / 4;
    }
    if (few && a.batch <= 65535 && a.kv_heads <= 65535) {
        if (rows <= 16) return launch_window_few<T, Out, D, 1, true>(h, a, st);
        if (rows <= 32) return launch_window_few<T, Out, D, 2, true>(h, a, st);
        return h->cfg.round_weights ? launch_window_few<T, Out, D, 4, false>(h, a, st) : launch_window_few<T, Out, D, 4, true>(h, a, st);
    }
    return h->cfg.round_weights ? launch_window_tc<T, Out, D, false>(h, a, st) : launch_window_tc<T, Out, D, true>(h, a, st);
}
template <typename T, typename Out>
int launch_window(const ligguf_window* h, const lg::WindowArgs& a, cudaStream_t st) {
    return h->cfg.head_dim == 64 ? launch_window_d<T, Out, 64>(h, a, st) : launch_window_d<T, Out, 128>(h, a, st);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------ norms and rotation
int ligguf_cuda_qk_rope_free(ligguf_qk_rope* h) {
    if (!h) return LIGGUF_ATTN_OK;
    DeviceGuard dg(h->cfg.device);
    cudaFree(h->turns);
    delete h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_qk_rope_init(const ligguf_qk_rope_cfg* cfg, ligguf_qk_rope** out) {
    if (!cfg || !out) return fail(LIGGUF_ATTN_EINVAL, "null argument");
    *out = nullptr;
    ligguf_qk_rope_cfg c = *cfg;
    int rc;
    if ((rc = check_rope(c.rope))) return rc;
    if (c.n_heads < 1 || c.n_kv_heads < 0 || c.n_heads > 4096 || c.n_kv_heads > 4096)
        return fail(LIGGUF_ATTN_EINVAL, "%d query and %d key heads", c.n_heads, c.n_kv_heads);
    if (!type_ok(c.in_type) || !type_ok(c.out_type)) return fail(LIGGUF_ATTN_EINVAL, "types %d, %d", c.in_type, c.out_type);
    if (c.qk_norm && !(c.rms_epsilon >= 0.f)) return fail(LIGGUF_ATTN_EINVAL, "rms_epsilon %g", c.rms_epsilon);
    const long long qw = static_cast<long long>(c.n_heads) * c.rope.head_dim, kw = static_cast<long long>(c.n_kv_heads) * c.rope.head_dim;
    if ((rc = check_stride(&c.q_stride, qw, c.in_type, "q_stride")) || (rc = check_stride(&c.k_stride, kw, c.in_type, "k_stride")) ||
        (rc = check_stride(&c.q_out_stride, qw, c.out_type, "q_out_stride")) ||
        (rc = check_stride(&c.k_out_stride, kw, c.out_type, "k_out_stride")) || (rc = check_device(c.device)))
        return rc;
    DeviceGuard dg(c.device);
    ligguf_qk_rope* h = new (std::nothrow) ligguf_qk_rope();
    if (!h) return fail(LIGGUF_ATTN_ENOMEM, "host memory");
    h->cfg = c;
    h->cfg.rope.freq = nullptr;
    if ((rc = make_turns(c.rope, &h->turns))) {
        ligguf_cuda_qk_rope_free(h);
        return rc;
    }
    *out = h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_qk_rope_async(ligguf_qk_rope* h, int n, int pos0, const int* d_pos, const void* d_q, const void* d_k,
                              const float* d_q_gamma, const float* d_k_gamma, void* d_q_out, void* d_k_out,
                              void* stream) {
    if (!h) return fail(LIGGUF_ATTN_EINVAL, "null handle");
    const ligguf_qk_rope_cfg& c = h->cfg;
    if (n < 0 || (!d_pos && (pos0 < 0 || pos0 > INT32_MAX - n)))
        return fail(LIGGUF_ATTN_EINVAL, "%d tokens from position %d", n, pos0);
    if (n == 0) return LIGGUF_ATTN_OK;
    if (!d_q || !d_q_out || (c.n_kv_heads && (!d_k || !d_k_out))) return fail(LIGGUF_ATTN_EINVAL, "null tensor pointer");
    if (c.qk_norm && (!d_q_gamma || (c.n_kv_heads && !d_k_gamma))) return fail(LIGGUF_ATTN_EINVAL, "null norm weights");
    if (!aligned16(d_q) || !aligned16(d_q_out) || !aligned16(d_k) || !aligned16(d_k_out) || !aligned16(d_q_gamma) ||
        !aligned16(d_k_gamma))
        return fail(LIGGUF_ATTN_EINVAL, "rows and norm weights must be 16-byte aligned");
    DeviceGuard dg(c.device);
    lg::RopeRowsArgs a = {};
    a.q = d_q;
    a.k = d_k;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.q_out = d_q_out;
    a.k_out = d_k_out;
    a.q_out_stride = c.q_out_stride;
    a.k_out_stride = c.k_out_stride;
    a.q_gamma = d_q_gamma;
    a.k_gamma = d_k_gamma;
    a.turns = h->turns;
    a.pos = d_pos;
    a.n = n;
    a.pos0 = pos0;
    a.q_heads = c.n_heads;
    a.kv_heads = c.n_kv_heads;
    a.pairs = c.rope.rope_dim / 2;
    a.norm = c.qk_norm;
    a.eps = c.rms_epsilon;
    a.magnitude = c.rope.magnitude > 0.f ? c.rope.magnitude : 1.f;
    return launch_rope_rows_any(a, c.rope, c.in_type, c.out_type, static_cast<cudaStream_t>(stream));
}

// ------------------------------------------------------------------------------ 4-bit cache
int ligguf_cuda_kv4_free(ligguf_kv4* h) {
    if (!h) return LIGGUF_ATTN_OK;
    DeviceGuard dg(h->cfg.device);
    cudaFree(h->tiles);
    cudaFree(h->turns);
    cudaFree(h->gammas);
    cudaFree(h->parts);
    cudaFree(h->tickets);
    if (h->h_err) cudaFreeHost(h->h_err);
    delete[] h->norm_set;
    delete h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_kv4_init(const ligguf_kv4_cfg* cfg, ligguf_kv4** out) {
    if (!cfg || !out) return fail(LIGGUF_ATTN_EINVAL, "null argument");
    *out = nullptr;
    ligguf_kv4_cfg c = *cfg;
    int rc;
    if ((rc = check_rope(c.rope)) || (rc = check_heads(c.n_heads, c.n_kv_heads))) return rc;
    const int nrep = c.n_heads / c.n_kv_heads;
    if (nrep != 1 && nrep != 2 && nrep != 4 && nrep != 8)
        return fail(LIGGUF_ATTN_EUNSUPPORTED, "n_heads/n_kv_heads = %d (supported: 1, 2, 4, 8)", nrep);
    if (c.n_layers < 1 || c.n_seqs < 1 || c.n_context < 1)
        return fail(LIGGUF_ATTN_EINVAL, "n_layers, n_seqs and n_context must be positive");
    if (c.n_seqs > 65535) return fail(LIGGUF_ATTN_EINVAL, "n_seqs %d (at most 65535)", c.n_seqs);
    if (c.n_context > (1 << 30)) return fail(LIGGUF_ATTN_EINVAL, "n_context %d (at most 2^30)", c.n_context);
    if (c.window < 0 || c.sinks < 0 || (c.sinks && !c.window))
        return fail(LIGGUF_ATTN_EINVAL, "window %d with %d sinks", c.window, c.sinks);
    if (!(c.scale >= 0.f) || std::isinf(c.scale)) return fail(LIGGUF_ATTN_EINVAL, "scale %g", c.scale);
    if (!type_ok(c.in_type) || !type_ok(c.rows_type)) return fail(LIGGUF_ATTN_EINVAL, "types %d, %d", c.in_type, c.rows_type);
    if (c.qk_norm && !(c.rms_epsilon >= 0.f)) return fail(LIGGUF_ATTN_EINVAL, "rms_epsilon %g", c.rms_epsilon);
    const int D = c.rope.head_dim;
    const long long kw = static_cast<long long>(c.n_kv_heads) * D;
    if ((rc = check_stride(&c.q_stride, kw * nrep, c.in_type, "q_stride")) ||
        (rc = check_stride(&c.k_stride, kw, c.in_type, "k_stride")) ||
        (rc = check_stride(&c.v_stride, kw, c.in_type, "v_stride")) || (rc = check_device(c.device)))
        return rc;
    if (c.scale == 0.f) c.scale = 1.0f / sqrtf(static_cast<float>(D));
    DeviceGuard dg(c.device);
    ligguf_kv4* h = new (std::nothrow) ligguf_kv4();
    if (!h) return fail(LIGGUF_ATTN_ENOMEM, "host memory");
    h->cfg = c;
    h->cfg.rope.freq = nullptr;
    h->nrep = nrep;
    h->tiles_per_head = (c.n_context + lg::kKv4Tile - 1) / lg::kKv4Tile;
    h->tile_bytes = 18 * static_cast<size_t>(D);
    auto bail = [&](int code) {
        ligguf_cuda_kv4_free(h);
        return code;
    };
    if ((h->tiles_per_head + 2 + lg::kKv4ItemUnits) * c.n_kv_heads * static_cast<long long>(c.n_seqs) > INT32_MAX)
        return bail(fail(LIGGUF_ATTN_EUNSUPPORTED, "%d sequences x %d heads x %d positions in one cache", c.n_seqs, c.n_kv_heads, c.n_context));
    // The product in double first: a cache beyond any memory must not wrap around.
    const double want = double(c.n_layers) * c.n_seqs * c.n_kv_heads * double(h->tiles_per_head) * double(h->tile_bytes);
    if (want > 1e15) return bail(fail(LIGGUF_ATTN_ENOMEM, "4-bit cache of %.3g bytes does not fit", want));
    const size_t bytes = size_t(c.n_layers) * c.n_seqs * c.n_kv_heads * h->tiles_per_head * h->tile_bytes;
    const size_t gbytes = size_t(c.n_layers) * 2 * D * sizeof(float);
    h->norm_set = new (std::nothrow) unsigned char[c.n_layers]();
    if (!h->norm_set) return bail(fail(LIGGUF_ATTN_ENOMEM, "host memory"));
    if (cudaMalloc(&h->tiles, bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        return bail(fail(LIGGUF_ATTN_ENOMEM, "4-bit cache of %zu bytes does not fit", bytes));
    }
    if (cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, c.device) != cudaSuccess)
        return bail(fail(LIGGUF_ATTN_ECUDA, "cudaDeviceGetAttribute failed"));
    const size_t part_bytes = size_t(h->num_sms) * lg::kv4_blocks_per_sm(nrep) * 2 * lg::kv4_part_floats(nrep, D) * sizeof(float);
    const size_t ticket_bytes = size_t(c.n_seqs) * c.n_kv_heads * sizeof(int);
    if (cudaMalloc(&h->gammas, gbytes) != cudaSuccess || cudaMalloc(&h->parts, part_bytes) != cudaSuccess ||
        cudaMalloc(&h->tickets, ticket_bytes) != cudaSuccess) {
        (void)cudaGetLastError();
        return bail(fail(LIGGUF_ATTN_ENOMEM, "handle buffers"));
    }
    if (cudaMemset(h->tickets, 0, ticket_bytes) != cudaSuccess) return bail(fail(LIGGUF_ATTN_ECUDA, "cudaMemset of the tickets failed"));
    // Zeroed like the engine's cache: unwritten positions are zeros, not whatever lay there.
    if (cudaMemset(h->tiles, 0, bytes) != cudaSuccess) return bail(fail(LIGGUF_ATTN_ECUDA, "cudaMemset of the cache failed"));
    if ((rc = make_turns(c.rope, &h->turns)) || (rc = make_err_words(&h->h_err, &h->d_err)) || (rc = set_up_done())) return bail(rc);
    *out = h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_kv4_set_qk_norm(ligguf_kv4* h, int layer, const float* q_gamma, const float* k_gamma) {
    if (!h || !q_gamma || !k_gamma) return fail(LIGGUF_ATTN_EINVAL, "null argument");
    if (layer < 0 || layer >= h->cfg.n_layers) return fail(LIGGUF_ATTN_EINVAL, "layer %d out of range", layer);
    DeviceGuard dg(h->cfg.device);
    const int D = h->cfg.rope.head_dim;
    float* g = h->gammas + size_t(layer) * 2 * D;
    LG_CUDA(cudaMemcpy(g, q_gamma, D * sizeof(float), cudaMemcpyHostToDevice));
    LG_CUDA(cudaMemcpy(g + D, k_gamma, D * sizeof(float), cudaMemcpyHostToDevice));
    if (const int rc = set_up_done()) return rc;
    h->norm_set[layer] = 1;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_kv4_append_async(ligguf_kv4* h, int layer, int seq, int pos0, int n, const void* d_q, const void* d_k,
                                 const void* d_v, void* d_q_out, void* d_k_rows, void* d_v_rows, void* stream) {
    int rc = kv4_check(h, layer, seq, 1, pos0, n);
    if (rc || n == 0) return rc;
    const ligguf_kv4_cfg& c = h->cfg;
    if (!d_k || !d_v || (d_q_out && !d_q)) return fail(LIGGUF_ATTN_EINVAL, "null tensor pointer");
    if (!aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_q_out) || !aligned16(d_k_rows) ||
        !aligned16(d_v_rows))
        return fail(LIGGUF_ATTN_EINVAL, "rows must be 16-byte aligned");
    if (c.qk_norm && !h->norm_set[layer])
        return fail(LIGGUF_ATTN_ESTATE, "QK-norm weights of layer %d were not set", layer);
    DeviceGuard dg(c.device);
    const int D = c.rope.head_dim;
    lg::RopeRowsArgs a = {};
    a.q = d_q_out ? d_q : nullptr;
    a.k = d_k;
    a.v = d_v;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.v_stride = c.v_stride;
    a.q_out = d_q_out;
    a.q_out_stride = static_cast<long long>(c.n_heads) * D;
    a.q_gamma = h->gammas + size_t(layer) * 2 * D;
    a.k_gamma = a.q_gamma + D;
    a.turns = h->turns;
    a.n = n;
    a.pos0 = pos0;
    a.q_heads = c.n_heads;
    a.kv_heads = c.n_kv_heads;
    a.pairs = c.rope.rope_dim / 2;
    a.norm = c.qk_norm;
    a.eps = c.rms_epsilon;
    a.magnitude = c.rope.magnitude > 0.f ? c.rope.magnitude : 1.f;
    a.tiles = h->seq_tiles(layer, seq);
    a.tiles_per_head = h->tiles_per_head;
    a.k_rows = d_k_rows;
    a.v_rows = d_v_rows;
    return launch_rope_rows_any(a, c.rope, c.in_type, c.rows_type, static_cast<cudaStream_t>(stream));
}

int ligguf_cuda_kv4_decode_async(ligguf_kv4* h, int layer, int n_rows, int pos, const int* d_pos, const void* d_q,
                                 const void* d_k, const void* d_v, void* d_out, void* d_k_rows, void* d_v_rows,
                                 void* stream) {
    int rc = kv4_check(h, layer, 0, n_rows, 0, 0);
    if (rc || n_rows == 0) return rc;
    const ligguf_kv4_cfg& c = h->cfg;
    if (!d_pos && (pos < 0 || pos >= c.n_context)) return fail(LIGGUF_ATTN_EINVAL, "pos %d out of range [0, %d)", pos, c.n_context);
    if (!d_q || !d_k || !d_v || !d_out) return fail(LIGGUF_ATTN_EINVAL, "null tensor pointer");
    if (!aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_out) || !aligned16(d_k_rows) ||
        !aligned16(d_v_rows))
        return fail(LIGGUF_ATTN_EINVAL, "rows must be 16-byte aligned");
    if (c.qk_norm && !h->norm_set[layer])
        return fail(LIGGUF_ATTN_ESTATE, "QK-norm weights of layer %d were not set", layer);
    DeviceGuard dg(c.device);
    const int D = c.rope.head_dim;
    lg::Kv4DecodeArgs a = {};
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.v_stride = c.v_stride;
    a.out = d_out;
    a.k_rows = d_k_rows;
    a.v_rows = d_v_rows;
    a.q_gamma = h->gammas + size_t(layer) * 2 * D;
    a.k_gamma = a.q_gamma + D;
    a.turns = h->turns;
    a.pos_rows = d_pos;
    a.pos = pos;
    a.n_rows = n_rows;
    a.q_heads = c.n_heads;
    a.kv_heads = c.n_kv_heads;
    a.pairs = c.rope.rope_dim / 2;
    a.norm = c.qk_norm;
    a.n_context = c.n_context;
    a.layout = c.rope.layout;
    a.rows_type = c.rows_type;
    a.eps = c.rms_epsilon;
    a.magnitude = c.rope.magnitude > 0.f ? c.rope.magnitude : 1.f;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    a.window = c.window;
    a.sinks = c.sinks;
    a.tiles = h->seq_tiles(layer, 0);
    a.tiles_per_head = h->tiles_per_head;
    a.parts = h->parts;
    a.tickets = h->tickets;
    a.err = h->d_err;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (c.in_type) {
        case LIGGUF_KV_F32: return launch_kv4_decode_d<float>(h, a, st);
        case LIGGUF_KV_F16: return launch_kv4_decode_d<__half>(h, a, st);
        default: return launch_kv4_decode_d<__nv_bfloat16>(h, a, st);
    }
}

int ligguf_cuda_kv4_read_async(ligguf_kv4* h, int layer, int seq, int pos0, int n, void* d_k_rows, void* d_v_rows,
                               void* stream) {
    int rc = kv4_check(h, layer, seq, 1, pos0, n);
    if (rc || n == 0 || (!d_k_rows && !d_v_rows)) return rc;
    if (!aligned16(d_k_rows) || !aligned16(d_v_rows)) return fail(LIGGUF_ATTN_EINVAL, "rows must be 16-byte aligned");
    const ligguf_kv4_cfg& c = h->cfg;
    DeviceGuard dg(c.device);
    const int D = c.rope.head_dim;
    dim3 grid;
    if ((rc = io_grid(static_cast<long long>(n) * c.n_kv_heads * (D / 8), &grid))) return rc;
    const lg::Kv4IoArgs a = kv4_io(h, layer, seq, 1, pos0, n, d_k_rows, d_v_rows);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (D == 64) {
        switch (c.rows_type) {
            case LIGGUF_KV_F32: lg::kv4_read_kernel<float, 64><<<grid, 256, 0, st>>>(a); break;
            case LIGGUF_KV_F16: lg::kv4_read_kernel<__half, 64><<<grid, 256, 0, st>>>(a); break;
            default: lg::kv4_read_kernel<__nv_bfloat16, 64><<<grid, 256, 0, st>>>(a); break;
        }
    } else {
        switch (c.rows_type) {
            case LIGGUF_KV_F32: lg::kv4_read_kernel<float, 128><<<grid, 256, 0, st>>>(a); break;
            case LIGGUF_KV_F16: lg::kv4_read_kernel<__half, 128><<<grid, 256, 0, st>>>(a); break;
            default: lg::kv4_read_kernel<__nv_bfloat16, 128><<<grid, 256, 0, st>>>(a); break;
        }
    }
    LG_CUDA(cudaGetLastError());
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_kv4_load_async(ligguf_kv4* h, int layer, int seq0, int n_seqs, int pos0, int n, const void* d_k_blocks,
                               const void* d_v_blocks, void* stream) {
    return kv4_blocks<true>(h, layer, seq0, n_seqs, pos0, n, const_cast<void*>(d_k_blocks),
                            const_cast<void*>(d_v_blocks), stream);
}

int ligguf_cuda_kv4_store_async(ligguf_kv4* h, int layer, int seq0, int n_seqs, int pos0, int n, void* d_k_blocks,
                                void* d_v_blocks, void* stream) {
    return kv4_blocks<false>(h, layer, seq0, n_seqs, pos0, n, d_k_blocks, d_v_blocks, stream);
}

int ligguf_cuda_kv4_status(ligguf_kv4* h, void* stream) {
    if (!h) return fail(LIGGUF_ATTN_EINVAL, "null handle");
    DeviceGuard dg(h->cfg.device);
    LG_CUDA(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)));
    volatile int* words = h->h_err;
    const int code = words[lg::kKv4ErrWait], beyond = words[lg::kKv4ErrPosition];
    words[lg::kKv4ErrWait] = words[lg::kKv4ErrPosition] = 0;
    if (code) {  // blocks that gave up left tickets behind
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        LG_CUDA(cudaMemsetAsync(h->tickets, 0, size_t(h->cfg.n_seqs) * h->cfg.n_kv_heads * sizeof(int), st));
        LG_CUDA(cudaStreamSynchronize(st));
        return fail(LIGGUF_ATTN_ETIMEDOUT, "a bounded in-kernel wait gave up (kernel error code %d)%s", code,
                    beyond ? "; a decode row's position was beyond n_context too" : "");
    }
    if (beyond) return fail(LIGGUF_ATTN_EINVAL, "a decode row's position is beyond n_context %d", h->cfg.n_context);
    return LIGGUF_ATTN_OK;
}

// ------------------------------------------------------------------------------ windowed attention
int ligguf_cuda_window_free(ligguf_window* h) {
    if (!h) return LIGGUF_ATTN_OK;
    DeviceGuard dg(h->cfg.device);
    cudaFree(h->parts);
    if (h->h_err) cudaFreeHost(h->h_err);
    delete h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_window_init(const ligguf_window_cfg* cfg, ligguf_window** out) {
    if (!cfg || !out) return fail(LIGGUF_ATTN_EINVAL, "null argument");
    *out = nullptr;
    ligguf_window_cfg c = *cfg;
    int rc;
    if ((rc = check_heads(c.n_heads, c.n_kv_heads))) return rc;
    if (c.head_dim != 64 && c.head_dim != 128)
        return fail(LIGGUF_ATTN_EUNSUPPORTED, "head_dim %d (supported: 64, 128)", c.head_dim);
    if (c.window < 0 || c.sinks < 0 || c.window > kWindowMost || c.sinks > kWindowMost || (c.sinks && !c.window))
        return fail(LIGGUF_ATTN_EINVAL, "window %d with %d sinks", c.window, c.sinks);
    if (!(c.scale >= 0.f) || std::isinf(c.scale)) return fail(LIGGUF_ATTN_EINVAL, "scale %g", c.scale);
    if (c.round_weights != 0 && c.round_weights != 1) return fail(LIGGUF_ATTN_EINVAL, "round_weights %d", c.round_weights);
    if (c.in_type != LIGGUF_KV_F16 && c.in_type != LIGGUF_KV_BF16)
        return fail(LIGGUF_ATTN_EUNSUPPORTED, "in_type %d (supported: F16, BF16)", c.in_type);
    if (c.out_type != c.in_type && c.out_type != LIGGUF_KV_F32)
        return fail(LIGGUF_ATTN_EUNSUPPORTED, "out_type %d (supported: in_type, F32)", c.out_type);
    const long long qw = static_cast<long long>(c.n_heads) * c.head_dim, kw = static_cast<long long>(c.n_kv_heads) * c.head_dim;
    if ((rc = check_stride(&c.q_stride, qw, c.in_type, "q_stride")) || (rc = check_stride(&c.k_stride, kw, c.in_type, "k_stride")) ||
        (rc = check_stride(&c.v_stride, kw, c.in_type, "v_stride")))
        return rc;
    for (long long s : {c.q_batch_stride, c.k_batch_stride, c.v_batch_stride})
        if (s < 0 || s % 8) return fail(LIGGUF_ATTN_EINVAL, "batch stride %lld is not a multiple of 16 bytes", s);
    if ((rc = check_device(c.device))) return rc;
    if (c.scale == 0.f) c.scale = 1.0f / sqrtf(static_cast<float>(c.head_dim));
    DeviceGuard dg(c.device);
    ligguf_window* h = new (std::nothrow) ligguf_window();
    if (!h) return fail(LIGGUF_ATTN_ENOMEM, "host memory");
    h->cfg = c;
    auto bail = [&](int code) {
        ligguf_cuda_window_free(h);
        return code;
    };
    if (cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, c.device) != cudaSuccess)
        return bail(fail(LIGGUF_ATTN_ECUDA, "cudaDeviceGetAttribute failed"));
    if (cudaMalloc(&h->parts, few_most_items(h->num_sms) * lg::kFewRows * (c.head_dim + 2) * sizeof(float)) != cudaSuccess) {
        (void)cudaGetLastError();
        return bail(fail(LIGGUF_ATTN_ENOMEM, "handle buffers"));
    }
    if ((rc = make_err_words(&h->h_err, &h->d_err))) return bail(rc);
    *out = h;
    return LIGGUF_ATTN_OK;
}

int ligguf_cuda_window_attn_async(ligguf_window* h, int batch, int n, int m, const void* d_q, const void* d_k,
                                  const void* d_v, const int* d_pos0, const int* d_lens, void* d_out, void* stream) {
    if (!h) return fail(LIGGUF_ATTN_EINVAL, "null handle");
    const ligguf_window_cfg& c = h->cfg;
    if (batch < 0 || n < 0 || m < 0 || n > kWindowMost || m > kWindowMost)
        return fail(LIGGUF_ATTN_EINVAL, "batch %d, n %d, m %d", batch, n, m);
    if (batch == 0 || n == 0) return LIGGUF_ATTN_OK;
    if (!d_q || !d_out || (m && (!d_k || !d_v))) return fail(LIGGUF_ATTN_EINVAL, "null tensor pointer");
    if (!aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_out))
        return fail(LIGGUF_ATTN_EINVAL, "rows must be 16-byte aligned");
    DeviceGuard dg(c.device);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (m == 0) {  // no key to see
        LG_CUDA(cudaMemsetAsync(d_out, 0, size_t(batch) * n * c.n_heads * c.head_dim * type_size(c.out_type), st));
        return LIGGUF_ATTN_OK;
    }
    lg::WindowArgs a = {};
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.out = d_out;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.v_stride = c.v_stride;
    a.q_batch = c.q_batch_stride ? c.q_batch_stride : c.q_stride * n;
    a.k_batch = c.k_batch_stride ? c.k_batch_stride : c.k_stride * m;
    a.v_batch = c.v_batch_stride ? c.v_batch_stride : c.v_stride * m;
    a.pos0 = d_pos0;
    a.lens = d_lens;
    a.batch = batch;
    a.n = n;
    a.m = m;
    a.q_heads = c.n_heads;
    a.kv_heads = c.n_kv_heads;
    a.window = c.window;
    a.sinks = c.sinks;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    if (c.in_type == LIGGUF_KV_F16)
        return c.out_type == LIGGUF_KV_F32 ? launch_window<__half, float>(h, a, st)
                                           : launch_window<__half, __half>(h, a, st);
    return c.out_type == LIGGUF_KV_F32 ? launch_window<__nv_bfloat16, float>(h, a, st)
                                       : launch_window<__nv_bfloat16, __nv_bfloat16>(h, a, st);
}

int ligguf_cuda_window_status(ligguf_window* h, void* stream) {
    if (!h) return fail(LIGGUF_ATTN_EINVAL, "null handle");
    DeviceGuard dg(h->cfg.device);
    LG_CUDA(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)));
    const int code = *reinterpret_cast<volatile int*>(h->h_err);
    *reinterpret_cast<volatile int*>(h->h_err) = 0;
    if (code) return fail(LIGGUF_ATTN_ETIMEDOUT, "a bounded in-kernel wait gave up (kernel error code %d)", code);
    return LIGGUF_ATTN_OK;
}

}  // extern "C"
