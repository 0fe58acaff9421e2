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
//                the expert's tokens as the N = 16..128 one: up (64 gate and 64 up rows in a tile, so that one CTA
//                holds both halves of each hidden value and quantises them) and down.
//   moe_combine  the weighted sum over each token's choices, in their order.
//
// All FP32 sums are in tensor memory or registers, in a fixed order (a long down product's segments in y, by the thread that
// wrote them): results do not depend on timing.
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
struct __align__(16) Entry {
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

// Routing by counting: a thread per (token, expert) counts the experts that come before its own (larger logit, or equal
// and lower index), which is its place in the choice. E comparisons a thread, but no chain of reductions. For one token
// of 64 experts with 8 choices 1.6 us less than a warp's eight rounds of moe_prep; with a thread's work growing with E and
// every thread busy it no longer is (61 tokens of 64 experts: 0.9 us more).
constexpr int RANK_KEYS = PREP_THREADS;
inline bool route_by_rank(int tokens, int experts, int renormalize) {
    return renormalize && tokens * experts <= RANK_KEYS && experts <= 128;
}
// s_id [T][K] gets the choices, s_ex [T][K] their exponentials. Ends with a barrier.
__device__ __forceinline__ void choose_by_rank(const PrepParams& p, uint32_t* s_key, short* s_id, float* s_ex) {
    const int E = p.experts, K = p.top_k, t = threadIdx.x / E, e = threadIdx.x - t * E;
    const uint32_t key = t < p.tokens ? logit_key(p.logits[(size_t)t * E + e]) : 0u;
    s_key[threadIdx.x] = key;
    if (threadIdx.x < p.tokens * K) {
        s_id[threadIdx.x] = -1;
        s_ex[threadIdx.x] = 0.0f;
    }
    __syncthreads();
    if (key) {
        const uint32_t* row = s_key + t * E;
        int before = 0;
        uint32_t top = 0;
#pragma unroll 8
        for (int i = 0; i < E; i++) {
            const uint32_t other = row[i];
            before += other > key || (other == key && i < e) ? 1 : 0;
            top = max(top, other);
        }
        if (before < K) {
            s_id[t * K + before] = (short)e;
            s_ex[t * K + before] = expf(key_logit(key) - key_logit(top));
        }
    }
    __syncthreads();
}
// Their softmax, in the order of the choices, to the workspace and the caller's ids and weights: a warp per token.
__device__ __forceinline__ void write_by_rank(const PrepParams& p, const short* s_id, const float* s_ex) {
    const int K = p.top_k, lane = threadIdx.x & 31;
    for (int t = threadIdx.x >> 5; t < p.tokens; t += PREP_THREADS / 32) {
        const float x = lane < K ? s_ex[t * K + lane] : 0.0f;
        float sum = x;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane < K) {
            const int id = s_id[t * K + lane];
            const float w = id >= 0 ? x / sum : 0.0f;
            p.slot_w[t * K + lane] = w;
            if (p.ids) p.ids[t * K + lane] = id;
            if (p.weights) p.weights[t * K + lane] = w;
        }
    }
}

// 16 columns of a unit (token, 512-column chunk) of x per lane; zeros past the last unit and column.
__device__ __forceinline__ void load_unit(const PrepParams& p, int u, int units, int chunks, bool vec, float (&v)[16]) {
    const int t = u / chunks, col = (u - t * chunks) * 512 + 16 * (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = 0.0f;
    if (u < units && col < p.hidden)
        kern::load_elems<16>(p.x, p.x_type, (size_t)t * (size_t)p.ldx + (size_t)col, 16, vec, v);
}
__device__ __forceinline__ bool wide_rows(const PrepParams& p) {
    return ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * (p.x_type == kern::T_F32 ? 4 : 2))) & 15) == 0;
}
// Write 16 codes and (even lanes) their block's scale to sorted row `row`, row `r` of entry `entry`.
__device__ __forceinline__ void store_unit(const PrepParams& p, int row, int entry, int r, int col, uint4 codes,
                                           uint32_t scale) {
    *reinterpret_cast<uint4*>(p.xq + (size_t)row * p.hidden + col) = codes;
    if ((threadIdx.x & 1) == 0)
        p.sx[((size_t)entry * (p.hidden / 128) + col / 128) * 512 + (r % 32) * 16 + (r / 32) * 4 + (col / 32) % 4] =
            (uint8_t)scale;
}

constexpr int FEW = 32;
// At most FEW choices in all, given or routed by rank (a decoding step of one to a few tokens, where latency is all):
// every warp keeps the sorted list in its lanes, a lane per choice, and no barrier follows the choice.
__global__ void __launch_bounds__(PREP_THREADS) moe_prep_few(const PrepParams p) {
    __shared__ uint32_t s_key[RANK_KEYS];
    __shared__ float s_ex[FEW];
    __shared__ short s_id[FEW];
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int T = p.tokens, K = p.top_k, E = p.experts, slots = T * K, nmax_log = 31 - __clz(p.nmax);
    const int chunks = (p.hidden + 511) / 512, units = T * chunks;
    const bool vec = wide_rows(p);
    float v[16];
    int u = warp * gridDim.x + blockIdx.x;
    load_unit(p, u, units, chunks, vec, v);
    if (p.logits) {
        choose_by_rank(p, s_key, s_id, s_ex);
        if (blockIdx.x == 0) write_by_rank(p, s_id, s_ex);
    } else {
        if (threadIdx.x < slots) {
            const int e = p.ids[threadIdx.x];
            s_id[threadIdx.x] = (short)(e >= 0 && e < E ? e : -1);
            if (blockIdx.x == 0) p.slot_w[threadIdx.x] = p.weights[threadIdx.x];
        }
        __syncthreads();
    }
    // lane i holds choice i: its rank among its expert's, the first row and the first entry of that expert
    const int e = lane < slots ? s_id[lane] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u)), n = __popc(same);
    const int m = e >= 0 && rank == 0 ? (n + p.nmax - 1) >> nmax_log : 0;  // entries, at the expert's first choice
    int start = 0, entry = 0, total = 0;
    for (int i = 0; i < slots; i++) {
        const int ei = __shfl_sync(0xffffffffu, e, i), mi = __shfl_sync(0xffffffffu, m, i);
        total += mi;
        if (ei >= 0 && ei < e) {
            start++;
            entry += mi;
        }
    }
    if (blockIdx.x == 0 && warp == 0) {
        if (lane == 0) *p.n_entries = total;
        for (int c = 0; c < m; c++) p.entries[entry + c] = Entry{e, start + (c << nmax_log), min(n - (c << nmax_log), p.nmax), 0};
        if (lane < slots) p.slot_of[lane] = e < 0 ? -1 : start + rank;
    }
    const int row = e < 0 ? -1 : start + rank;
    entry += rank >> nmax_log;
    for (; u < units; u += gridDim.x * (PREP_THREADS / 32)) {
        const int t = u / chunks, col = (u - t * chunks) * 512 + 16 * lane;
        bool nan;
        float top = max_abs16(v, nan);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const uint32_t code = scale_code(top);
        uint32_t w0, w1, w2;
        quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
        load_unit(p, u + gridDim.x * (PREP_THREADS / 32), units, chunks, vec, v);
        for (int j = 0; j < K; j++) {
            const int to = __shfl_sync(0xffffffffu, row, t * K + j), en = __shfl_sync(0xffffffffu, entry, t * K + j);
            const int r = __shfl_sync(0xffffffffu, rank, t * K + j) & (p.nmax - 1);
            if (to >= 0 && col < p.hidden) store_unit(p, to, en, r, col, make_uint4(w0, w1, w2, 0u), code);
        }
    }
}

// Every cluster of CTAs (one CTA, or eight for many tokens) routes all tokens for itself, a warp per token, and every CTA
// sorts the choices by expert in shared memory; no cluster waits for another. Then the grid's warps share out the 512-column chunks of x, whose
// loads were issued first. CTA 0 writes the tables and the chosen ids and weights. PER: experts per lane (2, 4, 8, 16).
template <int PER>
__global__ void __launch_bounds__(PREP_THREADS) moe_prep(const PrepParams p) {
    __shared__ short s_id[MAX_SLOTS], s_rank[MAX_SLOTS];
    __shared__ int s_count[MAX_EXPERTS], s_start[MAX_EXPERTS], s_entry[MAX_EXPERTS];
    __shared__ __align__(4) uint8_t s_hits[MAX_SLOTS / 32 * MAX_EXPERTS];  // choices of an expert among 32 slots
    int* s_place = reinterpret_cast<int*>(s_hits);  // then, per slot: entry * 128 + row inside the entry
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int WARPS = PREP_THREADS / 32;
    const int T = p.tokens, K = p.top_k, E = p.experts, slots = T * K, nmax_log = 31 - __clz(p.nmax);
    const int chunks = (p.hidden + 511) / 512, units = T * chunks;
    const bool vec = wide_rows(p);
    float v[16];
    int u = warp * gridDim.x + blockIdx.x;
    load_unit(p, u, units, chunks, vec, v);

    const int groups = (slots + 31) / 32;
    const int ctas = (int)sm100::cluster_nctarank(), rank = (int)sm100::cluster_ctarank(), first = rank + ctas * warp;
    for (int i = threadIdx.x; i < (groups * E + 3) / 4; i += PREP_THREADS) reinterpret_cast<uint32_t*>(s_hits)[i] = 0;
    if (p.logits) {
        uint32_t next[PER];
        auto load_keys = [&](int t) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane + 32 * i;
                next[i] = t < T && e < E ? logit_key(p.logits[(size_t)t * E + e]) : 0u;
            }
        };
        load_keys(first);
        for (int t = first; t < T; t += ctas * WARPS) {
            uint32_t key[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) key[i] = next[i];
            load_keys(t + ctas * WARPS);
            short* ids = s_id + t * K;
            if (lane < K) ids[lane] = -1;
            __syncwarp();
            uint32_t top = 0, mine = 0;  // lane j keeps choice j
            float sum = 0.0f;
            for (int j = 0; j < K; j++) {
                uint32_t best = 0;
                int e = lane;
#pragma unroll
                for (int i = 0; i < PER; i++)
                    if (key[i] > best) {
                        best = key[i];
                        e = lane + 32 * i;
                    }
                const uint32_t all = __reduce_max_sync(0xffffffffu, best);
                if (all == 0) break;  // nothing left to choose
                bool win = best == all;
                const uint32_t ties = __ballot_sync(0xffffffffu, win);
                if (ties & (ties - 1)) {  // equal logits in several lanes: the lowest index (every lane takes part)
                    const int lowest = __reduce_min_sync(0xffffffffu, win ? e : 0x7fffffff);
                    win = win && e == lowest;
                }
                if (j == 0) {
                    top = all;
                    if (!p.renormalize) {  // softmax over every expert
#pragma unroll
                        for (int i = 0; i < PER; i++)
                            if (key[i]) sum += expf(key_logit(key[i]) - key_logit(top));
#pragma unroll
                        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    }
                }
                if (lane == j) mine = all;
                if (win) ids[j] = (short)e;
#pragma unroll
                for (int i = 0; i < PER; i++)
                    if (win && lane + 32 * i == e) key[i] = 0;
            }
            if ((int)blockIdx.x < ctas) {
                const float x = mine ? expf(key_logit(mine) - key_logit(top)) : 0.0f;
                if (p.renormalize) {
                    sum = x;
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                }
                __syncwarp();
                if (lane < K) {
                    const float w = mine ? x / sum : 0.0f;
                    p.slot_w[t * K + lane] = w;
                    if (p.ids) p.ids[t * K + lane] = ids[lane];
                    if (p.weights) p.weights[t * K + lane] = w;
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
            const int e = p.ids[i];
            s_id[i] = (short)(e >= 0 && e < E ? e : -1);
            if (blockIdx.x == 0) p.slot_w[i] = p.weights[i];
        }
    }
    if (p.logits && ctas > 1) {  // the other CTAs' tokens
        __syncwarp();
        sm100::cluster_sync();
        for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
            const uint32_t owner = (uint32_t)((i / K) % ctas);
            if ((int)owner == rank) continue;
            uint16_t id;
            asm volatile("ld.shared::cluster.u16 %0, [%1];"
                         : "=h"(id)
                         : "r"(sm100::mapa_shared(sm100::smem_u32(s_id + i), owner))
                         : "memory");
            s_id[i] = (short)id;
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    }
    __syncthreads();
    // rank of each choice among its expert's, in (token, choice) order: within 32 slots, then over those before
    for (int g = warp; g < groups; g += WARPS) {
        const int i = 32 * g + lane, e = i < slots ? s_id[i] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int before = __popc(same & ((1u << lane) - 1u));
        if (e >= 0) {
            s_rank[i] = (short)before;
            if (before == 0) s_hits[g * E + e] = (uint8_t)__popc(same);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += PREP_THREADS) {
        int n = 0;
        for (int g = 0; g < groups; g++) n += s_hits[g * E + e];
        s_count[e] = n;
    }
    for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
        const int e = s_id[i];
        int n = s_rank[i];
        if (e >= 0)
            for (int g = 0; g < i / 32; g++) n += s_hits[g * E + e];
        s_rank[i] = (short)n;
    }
    __syncthreads();
    if (warp == 0) {  // first row and first entry of each expert: PER consecutive experts a lane, then over the lanes
        int n[PER], sn = 0, se = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane * PER + i;
            n[i] = e < E ? s_count[e] : 0;
            sn += n[i];
            se += (n[i] + p.nmax - 1) >> nmax_log;
        }
        int start = sn, entry = se;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int a = __shfl_up_sync(0xffffffffu, start, d), b = __shfl_up_sync(0xffffffffu, entry, d);
            if (lane >= d) {
                start += a;
                entry += b;
            }
        }
        if (blockIdx.x == 0 && lane == 31) *p.n_entries = entry;
        start -= sn;
        entry -= se;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane * PER + i;
            if (e < E) {
                s_start[e] = start;
                s_entry[e] = entry;
            }
            if (blockIdx.x == 0)
                for (int c = 0; c < n[i]; c += p.nmax, entry++)
                    p.entries[entry] = Entry{e, start + c, min(n[i] - c, p.nmax), 0};
            else
                entry += (n[i] + p.nmax - 1) >> nmax_log;
            start += n[i];
        }
    }
    __syncthreads();
    if (p.logits && ctas > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // s_id was read
    for (int i = threadIdx.x; i < slots; i += PREP_THREADS) {
        const int e = s_id[i], at = s_rank[i];
        const int row = e < 0 ? -1 : s_start[e] + at;
        if (blockIdx.x == 0) p.slot_of[i] = row;
        s_id[i] = (short)row;  // from here on the sorted row, and the entry with the row inside it
        s_place[i] = e < 0 ? 0 : (s_entry[e] + (at >> nmax_log)) * 128 + (at & (p.nmax - 1));
    }
    __syncthreads();
    // a lane quantises its 16 values (one block per lane pair) and writes them to each of its token's rows
    for (; u < units; u += gridDim.x * WARPS) {
        const int t = u / chunks, col = (u - t * chunks) * 512 + 16 * lane;
        bool nan;
        float m = max_abs16(v, nan);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t code = scale_code(m);
        uint32_t w0, w1, w2;
        quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
        load_unit(p, u + gridDim.x * WARPS, units, chunks, vec, v);
        if (col >= p.hidden) continue;
#pragma unroll 4
        for (int j = 0; j < K; j++) {
            const int row = s_id[t * K + j], place = s_place[t * K + j], r = place & 127;
            if (row < 0) continue;
            store_unit(p, row, place >> 7, r, col, make_uint4(w0, w1, w2, 0u), code);
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
    int segment;             // down, long: slabs of one accumulator; an item's segments are added in FP32 in y
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

// KIND_DOWN_LONG: a down product whose K is summed in segments, an accumulator each. It is an instantiation of its own because
// the others took 1-4% longer with the segments' control flow.
constexpr int KIND_UP_GATED = 0, KIND_UP = 1, KIND_DOWN = 2, KIND_DOWN_LONG = 3;

template <int KIND, int NMAX>
struct ProductConfig {
    static constexpr bool GATED = KIND == KIND_UP_GATED, DOWN = KIND >= KIND_DOWN, LONG = KIND == KIND_DOWN_LONG;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = NMAX * 128, SF_BYTES = 1024;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int CHUNK = NMAX < 32 ? NMAX : 32;  // tokens the epilogue takes at a time
    static constexpr int STG_PITCH = 132;
    static constexpr int STG_BYTES = DOWN ? 0 : CHUNK * STG_PITCH * 4;
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
    // The up product lets the down product start only after its own griddepcontrol.wait, that is once the list of
    // entries, and whatever wrote the weights, is complete. So the down product reads the list, and loads its first weight
    // tiles, while the up product still runs; its tokens (the hidden values) and outputs wait. Tokens go with the wait
    // in warp 0, outputs in warps 2..5.
    constexpr bool EARLY = C::DOWN;
    if (!EARLY) sm100::griddep_wait();
    // An entry, past L1: its lines are only sure to be newer than the list after the wait.
    auto entry = [&](int a) {
        const int4 q = sm100::ld_l2_s32x4(reinterpret_cast<const int4*>(p.entries) + a);
        return Entry{q.x, q.y, q.z, q.w};
    };
    // the first item's entry is read beside the count (it exists in the workspace whatever the count is)
    const Entry first = entry((int)blockIdx.x / p.tiles);
    const int total = sm100::ld_l2_s32(p.n_entries) * p.tiles;
    if (EARLY && warp != 0) sm100::griddep_wait();
    // Never before this thread's wait (see moe.cu): the next kernel reads what moe_prep wrote without waiting for it.
    if (!EARLY || warp != 0) sm100::griddep_launch_dependents();
    // the entry of item `it`, read an item ahead of its use
    auto entry_at = [&](int it) { return it < total ? entry(it / p.tiles) : Entry{0, 0, 0, 0}; };
    uint32_t issued_mask = 0, issued_phase = 0;
    bool mma_issued = false;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            Entry next = first;
            // Before the wait (EARLY): the weights of this many of the first item's slabs; their tokens follow it.
            const int ahead = EARLY && (int)blockIdx.x < total ? min(C::STAGES, p.k_slabs) : 0;
            auto load_weights = [&](int st, int row0, int kb) {
                const uint32_t fb = full_bar(st), dst = base + st * C::STAGE;
                sm100::tma_load_2d(dst, &tmW, fb, kb * 128, row0);
                if (C::GATED) sm100::tma_load_2d(dst + 64 * 128, &tmW, fb, kb * 128, row0 + p.inter);
                if (!C::GATED)
                    sm100::bulk_load(sf_base + st * C::SF_BYTES, p.sW + ((size_t)(row0 / 128) * p.k_slabs + kb) * 512, 512, fb);
            };
            for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
                const int a = it / p.tiles, tile = it - a * p.tiles;
                const Entry en = next;
                next = entry_at(it + gridDim.x);
                const int boxes = (en.n + 15) / 16;
                const int row0 = en.expert * p.rows_per_expert + tile * (C::GATED ? 64 : 128);
                const uint32_t tx = 128u * 96u + 2048u * boxes + (C::GATED ? 512u : 1024u);
                const int done = it == (int)blockIdx.x ? ahead : 0;
                if (EARLY && it == (int)blockIdx.x) {
                    for (int kb = 0; kb < ahead; kb++) {  // the ring is empty: no wait
                        sm100::mbar_arrive_expect_tx(full_bar(kb), tx);
                        load_weights(kb, row0, kb);
                        issued_mask |= 1u << kb;
                    }
                    sm100::griddep_wait();
                    sm100::griddep_launch_dependents();  // after the wait, as above
                }
                for (int kb = 0; kb < p.k_slabs; kb++) {
                    const uint32_t fb = full_bar(stage);
                    if (kb >= done) {
                        if (!sm100::wait_parity_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget)) {
                            raise(0x1u);
                            ok = false;
                            break;
                        }
                        sm100::mbar_arrive_expect_tx(fb, tx);
                        load_weights(stage, row0, kb);
                    }
                    for (int b = 0; b < boxes; b++)
                        sm100::tma_load_2d(base + stage * C::STAGE + C::A_BYTES + 2048 * b, &tmB, fb, kb * 128,
                                           en.start + 16 * b);
                    sm100::bulk_load(sf_base + stage * C::SF_BYTES + 512, p.sB + ((size_t)a * p.k_slabs + kb) * 512, 512, fb);
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
        // a down product without items still ends after the up product
        if (EARLY && (lane != 0 || (int)blockIdx.x >= total)) {
            sm100::griddep_wait();
            sm100::griddep_launch_dependents();
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, local = 0;
            uint32_t phase = 0;
            bool ok = true;
            Entry next = first;
            // the next slab's barrier is polled right after a slab's MMAs are issued: the pipe's queue is short
            bool ready = false;
            for (int it = blockIdx.x; it < total && ok; it += gridDim.x, local++) {
                const int n = next.n;
                next = entry_at(it + gridDim.x);
                const uint32_t idesc = sm100::make_idesc_e2m3(128, (n + 15) / 16 * 16);
                uint32_t d_taddr = 0;
                auto next_accumulator = [&] {
                    if (!sm100::wait_parity_bounded(acc_empty0 + 8u * (local & 1), ((local >> 1) & 1) ^ 1u, abort_flag,
                                                    p.wait_budget)) {
                        raise(0x2u);
                        return false;
                    }
                    sm100::tc_fence_after();
                    d_taddr = tmem_base + (local & 1) * NMAX;
                    return true;
                };
                if (!next_accumulator()) break;
                int kb0 = 0;  // the segment's first slab
                for (int kb = 0; kb < p.k_slabs; kb++) {
                    if (C::LONG && kb == kb0 + p.segment) {
                        sm100::tc_commit(acc_full0 + 8u * (local & 1));
                        local++;
                        kb0 = kb;
                        if (!next_accumulator()) {
                            ok = false;
                            break;
                        }
                    }
                    if (!ready && !sm100::wait_parity_bounded(full_bar(stage), phase, abort_flag, p.wait_budget)) {
                        raise(0x2u);
                        ok = false;
                        break;
                    }
                    // the scale warp's cp.async writes are generic-proxy writes; tcgen05.cp reads through the async proxy
                    if constexpr (C::GATED) sm100::fence_async_shared();
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
                                               (tmem_base + C::TMEM_SFB) | ((uint32_t)k << 30), kb > kb0 || k > 0 ? 1u : 0u);
                    mma_issued = true;
                    sm100::tc_commit(empty_bar(stage));
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    ready = sm100::mbar_test_wait(full_bar(stage), phase);
                }
                if (ok) sm100::tc_commit(acc_full0 + 8u * (local & 1));
            }
        }
    } else if (warp < 6) {
        const int quarter = warp & 3;
        int local = 0;
        Entry next = first;
        Entry en{};
        int a = 0, tile = 0, kb0 = 0;  // kb0: the segment's first slab
        for (int it = blockIdx.x; it < total; local++) {
            if (!C::LONG || kb0 == 0) {
                a = it / p.tiles, tile = it - a * p.tiles;
                en = next;
                next = entry_at(it + gridDim.x);
            }
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
                if constexpr (C::DOWN) {
#pragma unroll
                    for (int j = 0; j < C::CHUNK; j++)
                        if (c0 + j < en.n) {
                            float* y = p.y + (size_t)(en.start + c0 + j) * p.hidden + tile * 128 + 32 * quarter + lane;
                            *y = C::LONG && kb0 > 0 ? *y + __uint_as_float(r[j]) : __uint_as_float(r[j]);
                        }
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
            if constexpr (C::LONG) kb0 = kb0 + p.segment < p.k_slabs ? kb0 + p.segment : 0;
            if (!C::LONG || kb0 == 0) it += gridDim.x;
        }
    } else {
        // gated: rows 0..63 of a tile are gate rows, 64..127 up rows, so its scale atom takes 8 of the 16 bytes
        // of each line from either half's atom
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        Entry next = first;
        for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
            const int a = it / p.tiles, tile = it - a * p.tiles;
            const int row0 = next.expert * p.rows_per_expert + tile * 64;
            next = entry_at(it + gridDim.x);
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
    // the places and weights were complete when the down product let this kernel start (see moe_product): read them
    // before the wait, past L1
    const int t = blockIdx.y, col = (blockIdx.x * blockDim.x + threadIdx.x) * 4, lane = threadIdx.x & 31;
    const int slot = lane < p.top_k ? sm100::ld_l2_s32(p.slot_of + t * p.top_k + lane) : -1;
    const float weight = lane < p.top_k ? sm100::ld_l2_f32(p.slot_w + t * p.top_k + lane) : 0.0f;
    sm100::griddep_wait();
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool in = col < p.hidden;
#pragma unroll 4
    for (int j = 0; j < p.top_k; j++) {
        const int s = __shfl_sync(0xffffffffu, slot, j);
        const float w = __shfl_sync(0xffffffffu, weight, j);
        if (s < 0 || !in) continue;
        const float4 q = *reinterpret_cast<const float4*>(p.y + (size_t)s * p.hidden + col);
        v[0] += w * q.x;
        v[1] += w * q.y;
        v[2] += w * q.z;
        v[3] += w * q.w;
    }
    if (!in) return;
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
