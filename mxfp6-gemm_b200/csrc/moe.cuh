#pragma once
// Mixture-of-experts layer for a few tokens (at most 128): kernels.
//
//   out[t] = [residual[t] +] sum_j w[t][j] * down_e( q( act(gate_e(q(x[t]))) * up_e(q(x[t])) ) ),  e = ids[t][j]
//
// q() is MXFP6 quantisation (quant.cuh); gate, up and down are products with MXFP6 weights in the layout the
// GEMM reads (packed rows, tiled scales). Each chosen expert's weights are read once, whatever the number of
// its tokens, and everything else is small: the layer is bound by reading 0.78 bytes a weight.
//
//   moe_prep     routing (top-k and softmax of the logits), the list of (expert, its tokens), and x quantised
//                into one row per (token, choice), sorted by expert, so that an expert's tokens are consecutive
//                rows and the products need no gather.
//   moe_product  the two products, weights as the 128-row MMA operand (tcgen05.mma kind::mxf8f6f4, M = 128) and
//                the expert's tokens as the N = 16..128 one: up (gate and up rows interleaved 64 + 64 in a tile, so
//                that one CTA holds both halves of each hidden value and quantises them) and down.
//   moe_combine  the weighted sum over each token's choices, in their order.
//
// All FP32 sums are in tensor memory or registers, in a fixed order: results do not depend on timing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "epilogue.cuh"
#include "sm100_ptx.cuh"

namespace mxfp6 {

// Sticky status bits of the kernels below (MXFP6_DEV_*). This header is compiled into moe.cu only.
__device__ unsigned int g_moe_status = 0;

namespace moe {

constexpr int MAX_TOKENS = 128, MAX_TOPK = 16, MAX_EXPERTS = 512;
constexpr int MAX_SLOTS = MAX_TOKENS * MAX_TOPK;

// Up to NMAX tokens of one expert: rows [start, start + n) of the sorted slots.
struct Entry {
    int expert, start, n, pad;
};

// ---- routing and quantisation -------------------------------------------------------------------------

struct PrepParams {
    const void* x;
    long long ldx;
    int x_type;
    const float* logits;  // [tokens][experts]; null: ids and weights are inputs
    int renormalize;
    int* ids;        // [tokens][top_k]
    float* weights;  // [tokens][top_k]
    int tokens, experts, top_k, hidden, nmax;
    int* n_entries;   // workspace from here on
    Entry* entries;
    int* slot_of;     // [tokens][top_k]: sorted row, or -1
    float* slot_w;    // [tokens][top_k]
    uint8_t* xq;      // [slots][hidden]: 16 codes in the first 12 bytes of each 16
    uint8_t* sx;      // scale atoms [entries][hidden / 128][512]
};

// Floats as unsigned integers of the same order (-0 equal to +0); NaN and -inf (never chosen) are 0.
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// Its inverse, with +inf taken as the largest finite value.
__device__ __forceinline__ float key_logit(uint32_t k) {
    const float v = __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
    return fminf(v, 3.402823466e38f);
}

constexpr int PREP_THREADS = 1024;

// Every CTA routes all tokens for itself (a warp per token; at most 4 rounds of MAX_TOPK warp reductions) and
// sorts the choices by expert in shared memory; no CTA waits for another. Then the grid's warps share out the
// 512-column chunks of x. CTA 0 writes the tables and the chosen ids and weights.
__global__ void __launch_bounds__(PREP_THREADS) moe_prep(const PrepParams p) {
    __shared__ short s_id[MAX_SLOTS];
    __shared__ float s_w[MAX_SLOTS];
    __shared__ short s_rank[MAX_SLOTS];
    __shared__ int s_count[MAX_EXPERTS], s_start[MAX_EXPERTS], s_entry[MAX_EXPERTS];
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int WARPS = PREP_THREADS / 32;
    const int T = p.tokens, K = p.top_k, E = p.experts, slots = T * K;

    if (p.logits) {
        constexpr int PER = MAX_EXPERTS / 32;
        for (int t = warp; t < T; t += WARPS) {
            uint32_t key[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane + 32 * i;
                key[i] = e < E ? logit_key(p.logits[(size_t)t * E + e]) : 0u;
            }
            float top = 0.0f, sum = 0.0f, mine = 0.0f;  // lane j keeps choice j's exponential
            int chosen = -1;
            for (int j = 0; j < K; j++) {
                uint32_t best = 0;
                int at = 0;
#pragma unroll
                for (int i = 0; i < PER; i++)
                    if (key[i] > best) {
                        best = key[i];
                        at = i;
                    }
                const uint32_t all = __reduce_max_sync(0xffffffffu, best);
                if (all == 0) break;  // nothing left to choose
                const int e = __reduce_min_sync(0xffffffffu, best == all ? lane + 32 * at : 0x7fffffff);
                if (j == 0) {
                    top = key_logit(all);
                    if (!p.renormalize) {  // softmax over every expert
                        float s = 0.0f;
#pragma unroll
                        for (int i = 0; i < PER; i++)
                            if (key[i]) s += expf(key_logit(key[i]) - top);
#pragma unroll
                        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
                        sum = s;
                    }
                }
                const float ex = expf(key_logit(all) - top);
                if (p.renormalize) sum += ex;
                if (lane == j) {
                    mine = ex;
                    chosen = e;
                }
#pragma unroll
                for (int i = 0; i < PER; i++)
                    if (lane + 32 * i == e) key[i] = 0;
            }
            if (lane < K) {
                s_id[t * K + lane] = (short)chosen;
                s_w[t * K + lane] = chosen >= 0 ? mine / sum : 0.0f;
            }
        }
    } else {
        for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
            const int e = p.ids[i];
            s_id[i] = (short)(e >= 0 && e < E ? e : -1);
            s_w[i] = p.weights[i];
        }
    }
    __syncthreads();
    // count and rank each expert's choices in (token, choice) order: a warp per expert
    for (int e = warp; e < E; e += WARPS) {
        int n = 0;
        for (int i0 = 0; i0 < slots; i0 += 32) {
            const bool hit = i0 + lane < slots && s_id[i0 + lane] == e;
            const uint32_t b = __ballot_sync(0xffffffffu, hit);
            if (hit) s_rank[i0 + lane] = (short)(n + __popc(b & ((1u << lane) - 1u)));
            n += __popc(b);
        }
        if (lane == 0) s_count[e] = n;
    }
    __syncthreads();
    if (warp == 0) {  // first row and first entry of each expert
        int start = 0, entry = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int n = e0 + lane < E ? s_count[e0 + lane] : 0;
            const int m = (n + p.nmax - 1) / p.nmax;
            int sn = n, se = m;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int a = __shfl_up_sync(0xffffffffu, sn, d), b = __shfl_up_sync(0xffffffffu, se, d);
                if (lane >= d) {
                    sn += a;
                    se += b;
                }
            }
            if (e0 + lane < E) {
                s_start[e0 + lane] = start + sn - n;
                s_entry[e0 + lane] = entry + se - m;
                if (blockIdx.x == 0)
                    for (int c = 0; c < m; c++)
                        p.entries[entry + se - m + c] =
                            Entry{e0 + lane, start + sn - n + c * p.nmax, min(n - c * p.nmax, p.nmax), 0};
            }
            start += __shfl_sync(0xffffffffu, sn, 31);
            entry += __shfl_sync(0xffffffffu, se, 31);
        }
        if (blockIdx.x == 0 && lane == 0) *p.n_entries = entry;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
            const int e = s_id[i];
            p.slot_of[i] = e < 0 ? -1 : s_start[e] + s_rank[i];
            p.slot_w[i] = s_w[i];
            if (p.logits) {
                if (p.ids) p.ids[i] = e;
                if (p.weights) p.weights[i] = s_w[i];
            }
        }
    }
    // x, in chunks of 512 columns: a lane quantises 16 values (one block per lane pair) and writes them to
    // each of its token's rows
    const int chunks = (p.hidden + 511) / 512, k_slabs = p.hidden / 128;
    for (int u = blockIdx.x * WARPS + warp; u < T * chunks; u += gridDim.x * WARPS) {
        const int t = u / chunks, col = (u - t * chunks) * 512 + 16 * lane;
        const bool live = col < p.hidden;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = 0.0f;
        const int esize = p.x_type == kern::T_F32 ? 4 : 2;
        const bool vec = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * esize)) & 15) == 0;
        if (live) kern::load_elems<16>(p.x, p.x_type, (size_t)t * (size_t)p.ldx + (size_t)col, 16, vec, v);
        bool nan;
        float m = max_abs16(v, nan);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t code = scale_code(m);
        uint32_t w0, w1, w2;
        quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
        if (!live) continue;
        for (int j = 0; j < K; j++) {
            const int i = t * K + j, e = s_id[i];
            if (e < 0) continue;
            const int rank = s_rank[i], row = s_start[e] + rank, r = rank % p.nmax;
            *reinterpret_cast<uint4*>(p.xq + (size_t)row * p.hidden + col) = make_uint4(w0, w1, w2, 0u);
            if ((lane & 1) == 0) {
                const size_t atom = (size_t)(s_entry[e] + rank / p.nmax) * k_slabs + col / 128;
                p.sx[atom * 512 + (r % 32) * 16 + (r / 32) * 4 + (col / 32) % 4] = (uint8_t)code;
            }
        }
    }
}

// ---- the two products -----------------------------------------------------------------------------------

struct ProductParams {
    const uint8_t* sW;       // weight scale atoms
    const uint8_t* sB;       // token scale atoms [entries][k_slabs][512]
    const int* n_entries;
    const Entry* entries;
    int k_slabs;             // K / 128
    int tiles;               // row tiles of one expert
    int rows_per_expert;     // rows of W per expert
    int inter, hidden, act;
    uint8_t* hq;             // up: hidden values, quantised [slots][inter], 16 bytes per 16 codes
    uint8_t* sh;             // up: their scale atoms [entries][inter / 128][512]
    float* y;                // down: [slots][hidden]
    long long wait_budget;
};

// Cycles the abort path waits for copies and MMAs in flight (a quarter of the default wait budget).
constexpr long long DRAIN_BUDGET = 1000000000LL;

constexpr int KIND_UP_GATED = 0, KIND_UP = 1, KIND_DOWN = 2;

template <int KIND, int NMAX>
struct ProductConfig {
    static constexpr bool GATED = KIND == KIND_UP_GATED;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = NMAX * 128, SF_BYTES = 1024;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int CHUNK = NMAX < 32 ? NMAX : 32;  // tokens the epilogue takes at a time
    static constexpr int STG_PITCH = 132;
    static constexpr int STG_BYTES = KIND == KIND_DOWN ? 0 : CHUNK * STG_PITCH * 4;
    static constexpr int BAR_BYTES = 256;
    static constexpr int CTAS = NMAX <= 64 ? 2 : 1;  // per SM
    static constexpr int BUDGET = (CTAS == 2 ? 113 : 226) * 1024 - 1024 - STG_BYTES - BAR_BYTES;
    static constexpr int STAGES_FIT = BUDGET / (STAGE + SF_BYTES);
    static constexpr int STAGES = STAGES_FIT < 10 ? STAGES_FIT : 10;
    static constexpr int SMEM_BYTES = 1024 + STAGES * (STAGE + SF_BYTES) + STG_BYTES + BAR_BYTES;
    // tensor memory: two accumulators of NMAX columns, weight scales, token scales
    static constexpr int TMEM_SFA = 2 * NMAX, TMEM_SFB = 2 * NMAX + 4;
    static constexpr int TMEM_NEED = 2 * NMAX + 8;
    static constexpr int TMEM_COLS = TMEM_NEED <= 64 ? 64 : TMEM_NEED <= 128 ? 128 : TMEM_NEED <= 256 ? 256 : 512;
    static constexpr int THREADS = GATED ? 224 : 192;
    static_assert(STAGES >= 3 && SMEM_BYTES <= 227 * 1024, "shared memory budget");
    static_assert(8 * (2 * STAGES + 5) + 16 <= BAR_BYTES, "barrier area");
};

__device__ __forceinline__ void epilogue_sync() {
    asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
}

// Warp 0 loads, warp 1 issues the MMAs, warps 2..5 take the accumulators; for the gated product warp 6 loads the
// weight scales. Items (entry, row tile) go round-robin over a persistent grid. Waits are bounded as in the GEMM
// kernels: a timeout sets a status bit, ends every role, lets copies and MMAs settle and frees tensor memory.
template <int KIND, int NMAX>
__global__ void __launch_bounds__(ProductConfig<KIND, NMAX>::THREADS, ProductConfig<KIND, NMAX>::CTAS)
    moe_product(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmB, const ProductParams p) {
    using C = ProductConfig<KIND, NMAX>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw_u32 = sm100::smem_u32(smem_raw);
    const uint32_t base = (raw_u32 + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_u32);
    const uint32_t sf_base = base + C::STAGES * C::STAGE;
    const uint32_t stg_off = C::STAGES * (C::STAGE + C::SF_BYTES);
    float* stg = reinterpret_cast<float*>(base_ptr + stg_off);
    const uint32_t bar_base = base + stg_off + C::STG_BYTES;
    uint8_t* bar_ptr = base_ptr + stg_off + C::STG_BYTES;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (C::STAGES + s); };
    const uint32_t acc_full0 = bar_base + 8u * (2 * C::STAGES);
    const uint32_t acc_empty0 = acc_full0 + 16u;
    const uint32_t drain_bar = acc_full0 + 32u;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_ptr + 8 * (2 * C::STAGES + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_ptr + 8 * (2 * C::STAGES + 5) + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto raise = [&](unsigned int bit) {
        if (!*abort_flag) atomicOr(&g_moe_status, bit);
        *abort_flag = 1;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            sm100::mbar_init(full_bar(s), C::GATED ? 33 : 1);  // the loader, and the scale warp's lanes
            sm100::mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            sm100::mbar_init(acc_full0 + 8u * b, 1);
            sm100::mbar_init(acc_empty0 + 8u * b, 128);
        }
        sm100::mbar_init(drain_bar, 1);
        *abort_flag = 0;
        sm100::fence_mbar_init();
        sm100::fence_async_shared();
        sm100::prefetch_tmap(&tmW);
        sm100::prefetch_tmap(&tmB);
    }
    if (warp == 1) {
        sm100::tmem_alloc(sm100::smem_u32(tmem_slot), C::TMEM_COLS);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    sm100::griddep_wait();
    sm100::griddep_launch_dependents();

    const int total = *p.n_entries * p.tiles;
    uint32_t issued_mask = 0, issued_phase = 0;
    bool mma_issued = false;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
                const int a = it / p.tiles, tile = it - a * p.tiles;
                const Entry en = p.entries[a];
                const int boxes = (en.n + 15) / 16;
                const int row0 = en.expert * p.rows_per_expert + tile * (C::GATED ? 64 : 128);
                const uint32_t tx = 128u * 96u + 2048u * boxes + (C::GATED ? 512u : 1024u);
                for (int kb = 0; kb < p.k_slabs; kb++) {
                    if (!sm100::wait_parity_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget)) {
                        raise(0x1u);
                        ok = false;
                        break;
                    }
                    const uint32_t fb = full_bar(stage), a_dst = base + stage * C::STAGE;
                    sm100::mbar_arrive_expect_tx(fb, tx);
                    sm100::tma_load_2d(a_dst, &tmW, fb, kb * 128, row0);
                    if (C::GATED) sm100::tma_load_2d(a_dst + 64 * 128, &tmW, fb, kb * 128, row0 + p.inter);
                    for (int b = 0; b < boxes; b++)
                        sm100::tma_load_2d(a_dst + C::A_BYTES + 2048 * b, &tmB, fb, kb * 128, en.start + 16 * b);
                    const uint32_t sf = sf_base + stage * C::SF_BYTES;
                    if (!C::GATED) sm100::bulk_load(sf, p.sW + ((size_t)(row0 / 128) * p.k_slabs + kb) * 512, 512, fb);
                    sm100::bulk_load(sf + 512, p.sB + ((size_t)a * p.k_slabs + kb) * 512, 512, fb);
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, local = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < total && ok; it += gridDim.x, local++) {
                const int n = p.entries[it / p.tiles].n;
                const uint32_t idesc = sm100::make_idesc_e2m3(128, (n + 15) / 16 * 16);
                const int b = local & 1;
                const uint32_t d_taddr = tmem_base + b * NMAX;
                if (!sm100::wait_parity_bounded(acc_empty0 + 8u * b, ((local >> 1) & 1) ^ 1u, abort_flag, p.wait_budget)) {
                    raise(0x2u);
                    break;
                }
                sm100::tc_fence_after();
                for (int kb = 0; kb < p.k_slabs; kb++) {
                    if (!sm100::wait_parity_bounded(full_bar(stage), phase, abort_flag, p.wait_budget)) {
                        raise(0x2u);
                        ok = false;
                        break;
                    }
                    sm100::tc_fence_after();
                    const uint32_t sf = sf_base + stage * C::SF_BYTES;
                    sm100::tc_cp_32x128b_warpx4(tmem_base + C::TMEM_SFA, sm100::make_sf_desc(sf));
                    sm100::tc_cp_32x128b_warpx4(tmem_base + C::TMEM_SFB, sm100::make_sf_desc(sf + 512));
                    const uint32_t a_src = base + stage * C::STAGE, b_src = a_src + C::A_BYTES;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        sm100::tc_mma_mxf8f6f4(d_taddr, sm100::make_kmajor_sw128_desc(a_src + 32 * k),
                                               sm100::make_kmajor_sw128_desc(b_src + 32 * k),
                                               sm100::idesc_with_sf_ids(idesc, k, k),
                                               (tmem_base + C::TMEM_SFA) | ((uint32_t)k << 30),
                                               (tmem_base + C::TMEM_SFB) | ((uint32_t)k << 30), kb > 0 || k > 0 ? 1u : 0u);
                    mma_issued = true;
                    sm100::tc_commit(empty_bar(stage));
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) sm100::tc_commit(acc_full0 + 8u * b);
            }
        }
    } else if (warp < 6) {
        const int quarter = warp & 3;
        int local = 0;
        for (int it = blockIdx.x; it < total; it += gridDim.x, local++) {
            const int a = it / p.tiles, tile = it - a * p.tiles;
            const Entry en = p.entries[a];
            const int b = local & 1;
            // all four warps leave together on a timeout (they share a barrier below)
            const bool got = sm100::wait_parity_bounded(acc_full0 + 8u * b, (local >> 1) & 1, abort_flag, p.wait_budget);
            int lost;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.eq.u32 p, %1, 0;\n\t"
                "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                : "=r"(lost)
                : "r"((uint32_t)got)
                : "memory");
            if (lost) {
                raise(0x4u);
                break;
            }
            sm100::tc_fence_after();
            const uint32_t t_acc = tmem_base + ((uint32_t)(32 * quarter) << 16) + b * NMAX;
            const int tid = threadIdx.x - 64;
#pragma unroll 1
            for (int c0 = 0; c0 < en.n; c0 += C::CHUNK) {
                uint32_t r[C::CHUNK];
                sm100::tmem_ld_cols(t_acc + c0, r);
                if constexpr (KIND == KIND_DOWN) {
#pragma unroll
                    for (int j = 0; j < C::CHUNK; j++)
                        if (c0 + j < en.n)
                            p.y[(size_t)(en.start + c0 + j) * p.hidden + tile * 128 + 32 * quarter + lane] =
                                __uint_as_float(r[j]);
                } else {
                    // token-major through shared memory: a thread then holds 16 hidden values of a token
#pragma unroll
                    for (int j = 0; j < C::CHUNK; j++)
                        stg[j * C::STG_PITCH + 32 * quarter + lane] = __uint_as_float(r[j]);
                    epilogue_sync();
                    constexpr int ROWS = C::GATED ? 64 : 128, GROUPS = ROWS / 16;
#pragma unroll 1
                    for (int task = tid; task < C::CHUNK * GROUPS; task += 128) {
                        const int c = task / GROUPS, g = task % GROUPS;
                        const float* src = stg + c * C::STG_PITCH + 16 * g;
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float4 q = reinterpret_cast<const float4*>(src)[i];
                            v[4 * i] = q.x;
                            v[4 * i + 1] = q.y;
                            v[4 * i + 2] = q.z;
                            v[4 * i + 3] = q.w;
                        }
                        kern::activate_all<16>(p.act, v);
                        if (C::GATED) {
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float4 q = reinterpret_cast<const float4*>(src + 64)[i];
                                v[4 * i] *= q.x;
                                v[4 * i + 1] *= q.y;
                                v[4 * i + 2] *= q.z;
                                v[4 * i + 3] *= q.w;
                            }
                        }
                        bool nan;
                        float m = max_abs16(v, nan);
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        const uint32_t code = scale_code(m);
                        uint32_t w0, w1, w2;
                        quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
                        const int rk = c0 + c, col = tile * ROWS + 16 * g;
                        if (rk < en.n) {
                            *reinterpret_cast<uint4*>(p.hq + (size_t)(en.start + rk) * p.inter + col) =
                                make_uint4(w0, w1, w2, 0u);
                            if ((g & 1) == 0)
                                p.sh[((size_t)a * (p.inter / 128) + col / 128) * 512 + (rk % 32) * 16 + (rk / 32) * 4 +
                                     (col / 32) % 4] = (uint8_t)code;
                        }
                    }
                    epilogue_sync();
                }
            }
            sm100::tc_fence_before();
            sm100::mbar_arrive(acc_empty0 + 8u * b);
        }
    } else {
        // gated: rows 0..63 of a tile are gate rows, 64..127 up rows, so its scale atom takes 8 of the 16 bytes
        // of each line from either half's atom
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
            const int a = it / p.tiles, tile = it - a * p.tiles;
            const int row0 = p.entries[a].expert * p.rows_per_expert + tile * 64;
            const uint8_t* gate = p.sW + (size_t)(row0 / 128) * p.k_slabs * 512 + lane * 16 + (row0 % 128) / 32 * 4;
            const uint8_t* up = gate + (size_t)(p.inter / 128) * p.k_slabs * 512;
            for (int kb = 0; kb < p.k_slabs; kb++) {
                const bool got = sm100::wait_parity_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0) raise(0x1u);
                    ok = false;
                    break;
                }
                const uint32_t dst = sf_base + stage * C::SF_BYTES + lane * 16;
                sm100::cp_async_8(dst, gate + (size_t)kb * 512);
                sm100::cp_async_8(dst + 8, up + (size_t)kb * 512);
                sm100::cp_async_mbar_arrive_noinc(full_bar(stage));
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        sm100::cp_async_wait_all();
    }

    sm100::tc_fence_before();
    const int aborted = __syncthreads_or(*abort_flag != 0);
    if (aborted) {
        const int zero = 0;
        if (warp == 0 && lane == 0 && issued_mask) {
            if (C::GATED) {
                sm100::settle_ns(200000);  // a full barrier may lack arrivals that never come
            } else {
                for (int s = 0; s < C::STAGES; s++)
                    if ((issued_mask >> s) & 1u)
                        if (!sm100::wait_parity_bounded(full_bar(s), (issued_phase >> s) & 1u, &zero, DRAIN_BUDGET))
                            atomicOr(&g_moe_status, 0x8u);
            }
        }
        if (warp == 1 && lane == 0 && mma_issued) {
            sm100::tc_commit(drain_bar);
            if (!sm100::wait_parity_bounded(drain_bar, 0, &zero, DRAIN_BUDGET)) atomicOr(&g_moe_status, 0x8u);
        }
        sm100::tc_fence_before();
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// ---- weighted sum ------------------------------------------------------------------------------------------

struct CombineParams {
    const float* y;
    const int* slot_of;
    const float* slot_w;
    const void* residual;
    long long ld_residual;
    void* out;
    long long ldo;
    int type, top_k, hidden;
    int out_vec;  // rows of out are 16-byte aligned
};

// Four columns of one token per thread; hidden % 128 == 0.
__global__ void __launch_bounds__(256) moe_combine(const CombineParams p) {
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();
    const int t = blockIdx.y, col = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (col >= p.hidden) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = 0; j < p.top_k; j++) {
        const int s = p.slot_of[t * p.top_k + j];
        if (s < 0) continue;
        const float w = p.slot_w[t * p.top_k + j];
        const float4 q = *reinterpret_cast<const float4*>(p.y + (size_t)s * p.hidden + col);
        v[0] += w * q.x;
        v[1] += w * q.y;
        v[2] += w * q.z;
        v[3] += w * q.w;
    }
    if (p.residual)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] += kern::load_elem(p.residual, p.type, (size_t)t * p.ld_residual + col + i);
    const size_t at = (size_t)t * p.ldo + col;
    if (p.out_vec) {
        if (p.type == kern::T_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
                make_uint2(kern::pack2(v[0], v[1], p.type), kern::pack2(v[2], v[3], p.type));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) kern::store_elem(p.out, p.type, at + i, v[i]);
    }
}

}  // namespace moe
}  // namespace mxfp6
