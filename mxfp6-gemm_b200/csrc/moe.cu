// Mixture-of-experts layer for a few tokens: validation, workspace and launches (kernels in moe.cuh).
#include "moe.cuh"

#include <cstdio>
#include <mutex>

#include "host.hpp"
#include "mxfp6_gemm.h"
#include "route.hpp"

namespace mxfp6 {

void note_launch();  // launch counter (gemm.cu)

namespace {

constexpr int kMaxDevices = 64;

bool aligned(const void* p, uintptr_t a) {
    return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// Tokens of one expert that a product takes at a time (the width of its MMA and of its shared-memory
// stages). An expert with more is read again for the next ones, so the width leaves room above the mean.
int tile_tokens(int tokens, int top_k, int experts) {
    const int mean = (tokens * top_k + experts - 1) / experts;
    const int want = tokens < 2 * mean + 16 ? tokens : 2 * mean + 16;
    return want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : 128;
}

struct Layout {
    int nmax, slots, max_entries;
    size_t n_entries, entries, slot_of, slot_w, xq, sx, hq, sh, y, total;
};

Layout layout_of(const mxfp6_moe_layer& l, int tokens, int top_k) {
    Layout w;
    w.nmax = tile_tokens(tokens, top_k, l.experts);
    w.slots = tokens * top_k;
    w.max_entries = (l.experts < w.slots ? l.experts : w.slots) + w.slots / w.nmax;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    w.n_entries = take(sizeof(int));
    w.entries = take((size_t)w.max_entries * sizeof(moe::Entry));
    w.slot_of = take((size_t)w.slots * sizeof(int));
    w.slot_w = take((size_t)w.slots * sizeof(float));
    w.xq = take((size_t)w.slots * l.hidden);
    w.sx = take((size_t)w.max_entries * (l.hidden / 128) * 512);
    w.hq = take((size_t)w.slots * l.inter);
    w.sh = take((size_t)w.max_entries * (l.inter / 128) * 512);
    w.y = take((size_t)w.slots * l.hidden * sizeof(float));
    w.total = at;
    return w;
}

bool valid_layer(const mxfp6_moe_layer* l) {
    return l && l->experts > 0 && l->experts <= moe::MAX_EXPERTS && l->hidden > 0 && l->hidden % 128 == 0 &&
           l->inter > 0 && l->inter % 128 == 0 && (long long)l->experts * 2 * l->inter <= 0x7fffffff &&
           (long long)l->experts * l->hidden <= 0x7fffffff;
}

// Programmatic stream serialization: each kernel of the chain sets up while the one before it finishes. moe_prep and the up
// product touch global memory only after griddepcontrol.wait. The down product reads the list of entries and its first weights
// before its wait, and moe_combine the choices' places and weights before its own: both rest on moe_product letting its
// dependents start only after its own wait, when moe_prep, and whatever wrote the weights, is complete.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int cluster, int threads, size_t smem, cudaStream_t stream,
                   Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <int KIND, int NMAX>
cudaError_t launch_product(const CUtensorMap& tmW, const CUtensorMap& tmB, const moe::ProductParams& p, long long items,
                           cudaStream_t stream) {
    using C = moe::ProductConfig<KIND, NMAX>;
    auto kernel = moe::moe_product<KIND, NMAX>;
    static std::once_flag once[kMaxDevices];
    static cudaError_t attr_err[kMaxDevices];
    const int dev = host::device();
    std::call_once(once[dev], [&] {
        attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    });
    if (attr_err[dev] != cudaSuccess) return attr_err[dev];
    const long long slots = (long long)host::sm_count() * C::CTAS;
    return launch(kernel, dim3((unsigned)(items < slots ? items : slots)), 1, C::THREADS, C::SMEM_BYTES, stream, tmW, tmB, p);
}

template <int KIND>
cudaError_t launch_product_for(int nmax, const CUtensorMap& tmW, const CUtensorMap& tmB, const moe::ProductParams& p,
                               long long items, cudaStream_t stream) {
    switch (nmax) {
        case 16: return launch_product<KIND, 16>(tmW, tmB, p, items, stream);
        case 32: return launch_product<KIND, 32>(tmW, tmB, p, items, stream);
        case 64: return launch_product<KIND, 64>(tmW, tmB, p, items, stream);
        default: return launch_product<KIND, 128>(tmW, tmB, p, items, stream);
    }
}

}  // namespace

bool take_moe_status(unsigned int* bits) {
    unsigned int zero = 0;
    return cudaMemcpyFromSymbol(bits, g_moe_status, sizeof(*bits)) == cudaSuccess &&
           cudaMemcpyToSymbol(g_moe_status, &zero, sizeof(zero)) == cudaSuccess;
}

}  // namespace mxfp6

extern "C" size_t mxfp6_moe_workspace_size(const mxfp6_moe_layer* layer, int tokens, int top_k) {
    using namespace mxfp6;
    if (!valid_layer(layer) || tokens <= 0 || tokens > moe::MAX_TOKENS || top_k <= 0 || top_k > moe::MAX_TOPK) return 0;
    return layout_of(*layer, tokens, top_k).total;
}

extern "C" int mxfp6_moe(const mxfp6_moe_layer* layer, int ot, int tokens, int top_k, const void* x, int x_type,
                         long long ldx, const float* logits, int renormalize, int* ids, float* weights,
                         const void* residual, long long ld_residual, void* out, long long ldo, void* ws,
                         size_t ws_bytes, void* stream) {
    using namespace mxfp6;
    host::clear();
    char msg[256];
    if (!layer) return host::fail(MXFP6_ERR_NULL_POINTER, "moe: null layer");
    if (!valid_layer(layer)) {
        std::snprintf(msg, sizeof(msg),
                      "moe: %d experts (1..%d), hidden %d and inter %d (positive multiples of 128) with at most 2^31 "
                      "weight rows in all",
                      layer->experts, moe::MAX_EXPERTS, layer->hidden, layer->inter);
        return host::fail(MXFP6_ERR_INVALID_SHAPE, msg);
    }
    if (tokens < 0 || tokens > moe::MAX_TOKENS || top_k < 1 || top_k > moe::MAX_TOPK ||
        (logits && top_k > layer->experts)) {
        std::snprintf(msg, sizeof(msg), "moe: %d tokens (0..%d), %d of %d experts a token (1..%d)", tokens,
                      moe::MAX_TOKENS, top_k, layer->experts, moe::MAX_TOPK);
        return host::fail(MXFP6_ERR_INVALID_SHAPE, msg);
    }
    if (layer->activation < MXFP6_ACT_NONE || layer->activation > MXFP6_ACT_SILU) {
        std::snprintf(msg, sizeof(msg), "moe: activation %d", layer->activation);
        return host::fail(MXFP6_ERR_UNSUPPORTED, msg);
    }
    if (ot < MXFP6_OUT_F32 || ot > MXFP6_OUT_BF16 || x_type < MXFP6_OUT_F32 || x_type > MXFP6_OUT_BF16) {
        std::snprintf(msg, sizeof(msg), "moe: invalid output type %d or input type %d", ot, x_type);
        return host::fail(MXFP6_ERR_INVALID_OUT_TYPE, msg);
    }
    if (tokens == 0) return MXFP6_OK;
    if (!layer->w1 || !layer->s1 || !layer->w2 || !layer->s2 || !x || !out || (!logits && (!ids || !weights)))
        return host::fail(MXFP6_ERR_NULL_POINTER,
                          "moe: null weights, input or output, or neither logits nor ids and weights");
    if (ldx < layer->hidden || ldo < layer->hidden || (residual && ld_residual < layer->hidden)) {
        std::snprintf(msg, sizeof(msg), "moe: a row stride (x %lld, out %lld, residual %lld) is below hidden = %d", ldx,
                      ldo, ld_residual, layer->hidden);
        return host::fail(MXFP6_ERR_INVALID_STRIDE, msg);
    }
    const uintptr_t xe = x_type == MXFP6_OUT_F32 ? 4 : 2, oe = ot == MXFP6_OUT_F32 ? 4 : 2;
    if (!aligned(layer->w1, 32) || !aligned(layer->w2, 32) || !aligned(layer->s1, 16) || !aligned(layer->s2, 16) ||
        !aligned(x, xe) || !aligned(out, oe) || !aligned(residual, oe) || !aligned(logits, 4) || !aligned(ids, 4) ||
        !aligned(weights, 4))
        return host::fail(MXFP6_ERR_MISALIGNED,
                          "moe: weights need 32-byte, their scales 16-byte alignment, the rest that of their elements");
    const Layout w = layout_of(*layer, tokens, top_k);
    if (!ws || ws_bytes < w.total || !aligned(ws, 256)) {
        std::snprintf(msg, sizeof(msg), "moe: workspace %zu bytes, need %zu (256-byte aligned)", ws_bytes, w.total);
        return host::fail(MXFP6_ERR_WORKSPACE, msg);
    }
    const int dev = host::device();
    if (dev < 0 || dev >= kMaxDevices) return host::fail(MXFP6_ERR_CUDA, "moe: no CUDA device");

    const int H = layer->hidden, I = layer->inter, R1 = layer->gated ? 2 * I : I;
    uint8_t* b = static_cast<uint8_t*>(ws);
    CUtensorMap tmW1, tmX, tmW2, tmH;
    if (!host::fp6_tmap(&tmW1, layer->w1, layer->experts * R1, H, H / 4 * 3, layer->gated ? 64 : 128) ||
        !host::fp6_tmap(&tmW2, layer->w2, layer->experts * H, I, I / 4 * 3, 128) ||
        !host::bytes_tmap(&tmX, b + w.xq, w.slots, H, 16) || !host::bytes_tmap(&tmH, b + w.hq, w.slots, I, 16))
        return host::fail(MXFP6_ERR_CUDA, "moe: cuTensorMapEncodeTiled failed");
    cudaStream_t st = static_cast<cudaStream_t>(stream);

    moe::PrepParams pp;
    pp.x = x;
    pp.ldx = ldx;
    pp.x_type = x_type;
    pp.logits = logits;
    pp.renormalize = renormalize;
    pp.ids = ids;
    pp.weights = weights;
    pp.tokens = tokens;
    pp.experts = layer->experts;
    pp.top_k = top_k;
    pp.hidden = H;
    pp.nmax = w.nmax;
    pp.n_entries = reinterpret_cast<int*>(b + w.n_entries);
    pp.entries = reinterpret_cast<moe::Entry*>(b + w.entries);
    pp.slot_of = reinterpret_cast<int*>(b + w.slot_of);
    pp.slot_w = reinterpret_cast<float*>(b + w.slot_w);
    pp.xq = b + w.xq;
    pp.sx = b + w.sx;
    // eight 512-column chunks a CTA: more would wait for one another's issue slots, and the routing that every CTA
    // repeats takes its full width anyway
    int prep_grid = (tokens * ((H + 511) / 512) + 7) / 8;
    if (prep_grid > 32) prep_grid = 32;
    const int cluster = logits && tokens > 16 ? 8 : 1;
    prep_grid = (prep_grid + cluster - 1) / cluster * cluster;

    moe::ProductParams up;
    up.sW = layer->s1;
    up.sB = pp.sx;
    up.n_entries = pp.n_entries;
    up.entries = pp.entries;
    up.k_slabs = up.segment = H / 128;
    up.tiles = layer->gated ? I / 64 : I / 128;
    up.rows_per_expert = R1;
    up.inter = I;
    up.hidden = H;
    up.act = layer->activation;
    up.hq = b + w.hq;
    up.sh = b + w.sh;
    up.y = nullptr;
    up.wait_budget = host::wait_budget();
    moe::ProductParams down = up;
    down.sW = layer->s2;
    down.sB = up.sh;
    down.k_slabs = I / 128;
    down.tiles = H / 128;
    // An accumulator's error grows with the slabs it takes: an FP32 output's stay within FP32_SEGMENT_K (route.hpp). The hidden
    // values and 16-bit outputs are rounded far more coarsely.
    const int segments = ot == MXFP6_OUT_F32 ? (I + FP32_SEGMENT_K - 1) / FP32_SEGMENT_K : 1;
    down.segment = (down.k_slabs + segments - 1) / segments;
    down.rows_per_expert = H;
    down.y = reinterpret_cast<float*>(b + w.y);

    moe::CombineParams cp;
    cp.y = down.y;
    cp.slot_of = pp.slot_of;
    cp.slot_w = pp.slot_w;
    cp.residual = residual;
    cp.ld_residual = ld_residual;
    cp.out = out;
    cp.ldo = ldo;
    cp.type = ot;
    cp.top_k = top_k;
    cp.hidden = H;
    cp.out_vec = aligned(out, 16) && (tokens == 1 || ldo * (long long)oe % 16 == 0);

    const long long max_up = (long long)w.max_entries * up.tiles, max_down = (long long)w.max_entries * down.tiles;
    const int E = layer->experts;
    const bool few = w.slots <= moe::FEW && (!logits || moe::route_by_rank(tokens, E, renormalize));
    auto prep = few ? moe::moe_prep_few : E <= 64 ? moe::moe_prep<2> : E <= 128 ? moe::moe_prep<4> : E <= 256 ? moe::moe_prep<8> : moe::moe_prep<16>;
    cudaError_t e = launch(prep, dim3(prep_grid), cluster, moe::PREP_THREADS, 0, st, pp);
    if (e == cudaSuccess)
        e = layer->gated ? launch_product_for<moe::KIND_UP_GATED>(w.nmax, tmW1, tmX, up, max_up, st)
                         : launch_product_for<moe::KIND_UP>(w.nmax, tmW1, tmX, up, max_up, st);
    if (e == cudaSuccess)
        e = segments > 1 ? launch_product_for<moe::KIND_DOWN_LONG>(w.nmax, tmW2, tmH, down, max_down, st)
                         : launch_product_for<moe::KIND_DOWN>(w.nmax, tmW2, tmH, down, max_down, st);
    if (e == cudaSuccess) e = launch(moe::moe_combine, dim3((H + 1023) / 1024, tokens), 1, 256, 0, st, cp);
    if (e != cudaSuccess) {
        cudaGetLastError();
        std::snprintf(msg, sizeof(msg), "moe launch failed: %s", cudaGetErrorString(e));
        return host::fail(MXFP6_ERR_CUDA, msg);
    }
    return MXFP6_OK;
}
