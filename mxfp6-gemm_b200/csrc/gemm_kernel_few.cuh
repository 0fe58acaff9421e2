#pragma once
// The GEMM with a fused epilogue for few rows (M <= 64): one wave of CTAs, K split over a cluster.
//
// A cluster of S = 1..8 CTAs computes one 128 x BN tile, each over its own K segment, with the operand stages, scale
// copies and MMAs of gemm_mxfp6_sm100 (gemm_kernel.cuh). Such a GEMM reads every weight once and is over in a few
// microseconds, so what counts is the latency from the first load to the last store:
//   * every SM gets weights to read (S is the largest that one wave of two CTAs per SM holds), and the K segments' sums meet in shared
//     memory of the cluster instead of global memory and a second kernel: each CTA leaves its FP32 accumulator in its own
//     shared memory (over the operand ring, which is idle by then) and, after a cluster barrier, sums a share of the
//     tile's (row, 32 columns) groups over the S CTAs, in segment order;
//   * the epilogue runs on those groups with a lane per column, or per four columns of a row, spread over all warps of
//     all CTAs. In the tensor-memory layout (a lane per row) 16 rows would leave every warp but one idle.
// Rows past M come from whatever follows A's rows in shared memory (any bytes are valid codes) and end in accumulator
// lanes nobody reads. Waits are bounded (gemm_kernel.cuh); after a timeout every thread still takes both cluster barriers.
#include "gemm_kernel.cuh"

namespace mxfp6 {
namespace kern {

constexpr int FEW_ROWS = 64;       // rows at most
constexpr int FEW_CLUSTER = 8;     // K segments at most
constexpr int FEW_THREADS = 256;
// Rows of a column that a warp finishes together: one up to FEW_SINGLE rows, where there are more warps than groups of
// four, else four.
constexpr int FEW_BATCH = 4, FEW_SINGLE = 16;

template <int BN>
struct FewConfig {
    static constexpr int W_BYTES = BN * 128, SF_BYTES = 512 + BN / 128 * 512;
    static constexpr int PITCH = BN + 4;  // floats between the rows of the accumulator in shared memory
    static constexpr int TMEM_SFA = BN, TMEM_SFB = BN + 4, TMEM_COLS = BN == 256 ? 512 : 256;
    static constexpr int BAR_BYTES = 256, MAX_STAGES = 12;
    // A stages of `rows` (16, 32 or 64) rows. Two CTAs of the narrow tile share an SM: the next call's CTAs then set up, and
    // wait for this one, beside it (1 x 4096 x 4096 back to back: 12.3 us with the whole SM, 7.5 us with half).
    static constexpr int stage_bytes(int rows) { return rows * 128 + W_BYTES + SF_BYTES; }
    static constexpr int stages(int rows) {
        const int fit = ((BN == 256 ? 227 : 113) * 1024 - 1024 - BAR_BYTES) / stage_bytes(rows);
        return fit < MAX_STAGES ? fit : MAX_STAGES;
    }
    static constexpr int smem_bytes(int rows) { return 1024 + stages(rows) * stage_bytes(rows) + BAR_BYTES; }
    static_assert(8 * (2 * MAX_STAGES + 2) + 16 <= BAR_BYTES, "barrier area");
    static_assert(stages(64) >= 3 && stages(64) * stage_bytes(64) >= FEW_ROWS * PITCH * 4, "the accumulator fits the ring");
    static_assert(stages(16) * stage_bytes(16) >= 16 * PITCH * 4 && 16 * 128 + stages(16) * W_BYTES >= 128 * 128, "ring");
};

// Bias and aux values of a task: of R rows of a lane's column, or of four columns of a row (few_quad).
struct FewOperands {
    float bias[4], aux[FEW_BATCH];
};
// `in`: the column is inside D.
template <int R>
__device__ __forceinline__ void few_load(const Epi& e, int row0, int M, int n, bool in, FewOperands& o) {
    o.bias[0] = e.bias && in ? load_elem(e.bias, e.bias_type, (size_t)n) : 0.0f;
    if (e.aux_op != AUX_NONE) {
#pragma unroll
        for (int i = 0; i < R; i++)
            o.aux[i] = in && row0 + i < M ? load_elem(e.aux, e.aux_type, (size_t)(row0 + i) * (size_t)e.ld_aux + (size_t)n) : 0.0f;
    }
}

// R rows of 32 columns: lane l has the sums of column n.
template <int R>
__device__ __forceinline__ void few_store(const Epi& e, int row0, int M, int n, bool in, float (&v)[R], const FewOperands& o) {
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < R; i++) v[i] += o.bias[0];
    }
    activate_all<R, true>(e.act, v);
    if (e.aux_op != AUX_NONE) {
#pragma unroll
        for (int i = 0; i < R; i++) epi_join(e.aux_op, v[i], o.aux[i]);
    }
#pragma unroll
    for (int i = 0; i < R; i++)
        if (in && row0 + i < M) store_elem(e.out, e.out_type, (size_t)(row0 + i) * (size_t)e.ldd + (size_t)n, v[i]);
}

// The first task of this warp (few_finish).
template <int BN, int R>
__device__ __forceinline__ void few_load_first(const FusedParams& p, int tile, int rank, int S, FewOperands& o) {
    constexpr int G = BN / 32;
    const int t = rank + S * (int)(threadIdx.x >> 5), n = tile * BN + t % G * 32 + (int)(threadIdx.x & 31);
    if (t < (p.M + R - 1) / R * G) few_load<R>(p.epi, t / G * R, p.M, n, n < p.N, o);
}

// This CTA's share of the tile: tasks of 32 columns of R rows, summed over the cluster's accumulators at `here` in segment
// order. All of a task's loads are in flight together; `o` has the first task's bias and aux values.
template <int BN, int R>
__device__ __forceinline__ void few_finish(const FusedParams& p, int tile, int rank, int S, uint32_t here, FewOperands& o) {
    using C = FewConfig<BN>;
    constexpr int G = BN / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t part[FEW_CLUSTER];
#pragma unroll
    for (int s = 0; s < FEW_CLUSTER; s++) part[s] = s < S ? sm100::mapa_shared(here, (uint32_t)s) : 0u;
    const int tasks = (p.M + R - 1) / R * G;
    for (int t = rank + S * warp; t < tasks; t += S * (FEW_THREADS / 32)) {
        const int row0 = t / G * R, c = t % G * 32 + lane, n = tile * BN + c;
        if (t >= S * (FEW_THREADS / 32)) few_load<R>(p.epi, row0, p.M, n, n < p.N, o);
        if (n - lane >= p.N) continue;
        const uint32_t at = (uint32_t)(row0 * C::PITCH + c) * 4u;
        float q[FEW_CLUSTER][R], v[R];
#pragma unroll
        for (int s = 0; s < FEW_CLUSTER; s++)
#pragma unroll
            for (int i = 0; i < R; i++)
                q[s][i] = s < S && row0 + i < p.M ? sm100::ld_cluster_f32(part[s] + at + (uint32_t)(i * C::PITCH * 4)) : 0.0f;
#pragma unroll
        for (int i = 0; i < R; i++) {
            v[i] = q[0][i];
#pragma unroll
            for (int s = 1; s < FEW_CLUSTER; s++)
                if (s < S) v[i] += q[s][i];
        }
        few_store<R>(p.epi, row0, p.M, n, n < p.N, v, o);
    }
}

// The same for aligned rows and MXFP6, in tasks of four rows of 32 columns with four columns of a row per lane: a fourth of
// the exchange's loads, wide stores, and a block's maximum and codes in eight lanes (64 x 8192 x 2048 into MXFP6 11.6
// against 9.2 us, 36 x 3328 x 1408 with residual 8.7 / 7.3, 16 x 8192 x 2048 7.2 / 6.8; one row 6.98 / 7.08, so it keeps
// the other form).
__device__ __forceinline__ void few_quad_load(const Epi& e, int row, int M, int n, int valid, FewOperands& o) {
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++) o.bias[i] = i < valid ? load_elem(e.bias, e.bias_type, (size_t)(n + i)) : 0.0f;
    }
    if (e.aux_op == AUX_NONE) return;
    const size_t at = (size_t)row * (size_t)e.ld_aux + (size_t)n;
    if (!e.aux_vec || valid < 4 || row >= M) {
#pragma unroll
        for (int i = 0; i < 4; i++) o.aux[i] = i < valid && row < M ? load_elem(e.aux, e.aux_type, at + i) : 0.0f;
    } else if (e.aux_type == T_F32) {
        const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(e.aux) + at);
        o.aux[0] = q.x;
        o.aux[1] = q.y;
        o.aux[2] = q.z;
        o.aux[3] = q.w;
    } else {
        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(e.aux) + at);
        unpack2(q.x, e.aux_type, o.aux[0], o.aux[1]);
        unpack2(q.y, e.aux_type, o.aux[2], o.aux[3]);
    }
}

template <int BN>
__device__ __forceinline__ void few_quad(const FusedParams& p, int tile, int rank, int S, uint32_t here, FewOperands& o) {
    using C = FewConfig<BN>;
    constexpr int G = BN / 32;
    const Epi& e = p.epi;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t part[FEW_CLUSTER];
#pragma unroll
    for (int s = 0; s < FEW_CLUSTER; s++) part[s] = s < S ? sm100::mapa_shared(here, (uint32_t)s) : 0u;
    const int tasks = (p.M + 3) / 4 * G;
    for (int t = rank + S * warp; t < tasks; t += S * (FEW_THREADS / 32)) {
        const int row = t / G * 4 + lane / 8, c = t % G * 32 + lane % 8 * 4, n = tile * BN + c;
        if (t >= S * (FEW_THREADS / 32)) few_quad_load(e, row, p.M, n, p.N - n, o);
        if (tile * BN + t % G * 32 >= p.N) continue;
        const uint32_t at = (uint32_t)(row * C::PITCH + c) * 4u;
        float4 q[FEW_CLUSTER];
#pragma unroll
        for (int s = 0; s < FEW_CLUSTER; s++)
            q[s] = s < S && row < p.M ? sm100::ld_cluster_f32x4(part[s] + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float v[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
        for (int s = 1; s < FEW_CLUSTER; s++)
            if (s < S) {
                v[0] += q[s].x;
                v[1] += q[s].y;
                v[2] += q[s].z;
                v[3] += q[s].w;
            }
        if (e.bias) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += o.bias[i];
        }
        activate_all<4>(e.act, v);
        if (e.aux_op != AUX_NONE) {
#pragma unroll
            for (int i = 0; i < 4; i++) epi_join(e.aux_op, v[i], o.aux[i]);
        }
        if (e.out_type != T_MXFP6) {
            if (row < p.M && n < p.N) store_elems4(e, row, n, p.N - n, v);
            continue;
        }
        // magnitudes order like their bits (NaN does not count)
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) mag = max(mag, v[i] != v[i] ? 0u : __float_as_uint(fabsf(v[i])));
#pragma unroll
        for (int x = 1; x < 8; x *= 2) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, x));
        const uint32_t code = scale_code(__uint_as_float(mag));
        const float inv = e8m0_reciprocal(code);
        const uint32_t c4 = __byte_perm(to_e2m3x2(v[1] * inv, v[0] * inv), to_e2m3x2(v[3] * inv, v[2] * inv), 0x5410) & 0x3F3F3F3Fu;
        const uint32_t c24 = __dp4a(c4, 0x00004001u, 0u) + (__dp4a(c4, 0x40010000u, 0u) << 12);
        // lane j of the block's eight: bytes [3j, 3j + 3); words 0..5 from lanes 4j/3 and the next one
        const int j = lane % 8, first = (lane & 24) + j * 4 / 3;
        const uint32_t lo = __shfl_sync(0xffffffffu, c24, first), hi = __shfl_sync(0xffffffffu, c24, first + 1);
        const uint32_t w = j % 3 == 0 ? lo | (hi << 24) : j % 3 == 1 ? (lo >> 8) | (hi << 16) : (lo >> 16) | (hi << 8);
        if (row >= p.M) continue;
        uint8_t* d = static_cast<uint8_t*>(e.out) + (size_t)row * (size_t)e.ldd + (size_t)((n - 4 * j) / 4 * 3);
        if (j < 6) reinterpret_cast<uint32_t*>(d)[j] = w;
        if (j == 6) e.scales[scale_atom_offset(row, (n - 4 * j) / 32, e.k_atoms)] = (uint8_t)code;
    }
}

// `rows`: A's rows in a stage (the tensor map's box). The cluster's rank is the K segment.
template <int BN>
__global__ void __launch_bounds__(FEW_THREADS, 1)
    gemm_mxfp6_few(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const FusedParams p,
                   const int rows) {
    using C = FewConfig<BN>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw_u32 = sm100::smem_u32(smem_raw);
    const uint32_t base = (raw_u32 + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_u32);
    const int stages = C::stages(rows), x_bytes = rows * 128;
    const uint32_t w_base = base + stages * x_bytes, sf_base = w_base + stages * C::W_BYTES;
    const uint32_t bar_base = base + stages * C::stage_bytes(rows);
    uint8_t* bar_ptr = base_ptr + stages * C::stage_bytes(rows);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (C::MAX_STAGES + s); };
    const uint32_t acc_full = bar_base + 8u * (2 * C::MAX_STAGES);
    const uint32_t drain_bar = acc_full + 8u;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_ptr + 8 * (2 * C::MAX_STAGES + 2));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_ptr + 8 * (2 * C::MAX_STAGES + 2) + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (int)sm100::cluster_nctarank(), rank = (int)sm100::cluster_ctarank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            sm100::mbar_init(full_bar(s), 1);
            sm100::mbar_init(empty_bar(s), 1);
        }
        sm100::mbar_init(acc_full, 1);
        sm100::mbar_init(drain_bar, 1);
        *abort_flag = 0;
        sm100::fence_mbar_init();
        sm100::fence_async_shared();
        sm100::prefetch_tmap(&tmA);
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
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();

    const int tile = (int)blockIdx.x / S;
    const int kb0 = (int)((long long)p.k_slabs * rank / S), kb1 = (int)((long long)p.k_slabs * (rank + 1) / S);
    const int atoms = min(BN / 128, (p.N - tile * BN + 127) / 128);  // B's scale atoms inside the matrix
    bool loads_issued = false, mma_issued = false;
    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        const uint32_t tx = (uint32_t)(rows * 96 + BN * 96 + 512 * (1 + atoms));
        for (int kb = kb0; kb < kb1; kb++) {
            if (!sm100::wait_parity_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget)) {
                if (!*abort_flag) raise_status(0x1u, abort_flag);
                break;
            }
            const uint32_t fb = full_bar(stage), sf = sf_base + stage * C::SF_BYTES;
            sm100::mbar_arrive_expect_tx(fb, tx);
            sm100::tma_load_2d(w_base + stage * C::W_BYTES, &tmB, fb, kb * BK, tile * BN);
            for (int j = 0; j < atoms; j++)
                sm100::bulk_load(sf + 512 + 512 * j, p.sfB + ((size_t)(tile * (BN / 128) + j) * p.k_slabs + kb) * 512, 512, fb);
            sm100::tma_load_2d(base + stage * x_bytes, &tmA, fb, kb * BK, 0);
            sm100::bulk_load(sf, p.sfA + (size_t)kb * 512, 512, fb);
            loads_issued = true;
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = sm100::make_idesc_e2m3(BM, BN);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!sm100::wait_parity_bounded(full_bar(stage), phase, abort_flag, p.wait_budget)) {
                if (!*abort_flag) raise_status(0x2u, abort_flag);
                ok = false;
                break;
            }
            const uint32_t sf = sf_base + stage * C::SF_BYTES;
            sm100::tc_cp_32x128b_warpx4(tmem_base + C::TMEM_SFA, sm100::make_sf_desc(sf));
#pragma unroll
            for (int j = 0; j < BN / 128; j++)
                sm100::tc_cp_32x128b_warpx4(tmem_base + C::TMEM_SFB + 4 * j, sm100::make_sf_desc(sf + 512 + 512 * j));
            const uint32_t a_src = base + stage * x_bytes, b_src = w_base + stage * C::W_BYTES;
#pragma unroll
            for (int k = 0; k < BK / 32; k++) {
                const uint32_t sel = (uint32_t)k << 30;
                sm100::tc_mma_mxf8f6f4(tmem_base, sm100::make_kmajor_sw128_desc(a_src + 32 * k),
                                       sm100::make_kmajor_sw128_desc(b_src + 32 * k), sm100::idesc_with_sf_ids(idesc, k, k),
                                       (tmem_base + C::TMEM_SFA) | sel, (tmem_base + C::TMEM_SFB) | sel,
                                       kb > kb0 || k > 0 ? 1u : 0u);
            }
            mma_issued = true;
            sm100::tc_commit(empty_bar(stage));
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (ok) sm100::tc_commit(acc_full);
    }
    __syncwarp();
    // The first task's bias and aux values are on their way while the last MMAs run.
    FewOperands first = {};
    const bool quad = p.epi.out_type == T_MXFP6 || (p.epi.out_vec && p.M > 1);
    if (quad) {
        const int t = rank + S * warp, row = t / (BN / 32) * 4 + lane / 8, n = tile * BN + t % (BN / 32) * 32 + lane % 8 * 4;
        if (t < (p.M + 3) / 4 * (BN / 32)) few_quad_load(p.epi, row, p.M, n, p.N - n, first);
    } else if (p.M <= FEW_SINGLE)
        few_load_first<BN, 1>(p, tile, rank, S, first);
    else
        few_load_first<BN, FEW_BATCH>(p, tile, rank, S, first);
    // The accumulator to shared memory: a lane per row, half of the columns per warp.
    const bool got = sm100::wait_parity_bounded(acc_full, 0, abort_flag, p.wait_budget);
    if (!got && !*abort_flag) raise_status(0x4u, abort_flag);
    const int aborted = __syncthreads_or(!got);
    float* acc = reinterpret_cast<float*>(base_ptr);
    if (!aborted) {
        sm100::tc_fence_after();
        const int quarter = warp & 3, row = 32 * quarter + lane;
        if (32 * quarter < p.M) {
#pragma unroll 1
            for (int c = (warp >> 2) * (BN / 2); c < (warp >> 2) * (BN / 2) + BN / 2; c += 32) {
                uint32_t r[32];
                sm100::tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(32 * quarter) << 16) + (uint32_t)c, r);
                sm100::tmem_ld_wait(r);
                if (row < p.M) {
                    uint4* d = reinterpret_cast<uint4*>(acc + row * C::PITCH + c);
#pragma unroll
                    for (int i = 0; i < 8; i++) d[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                }
            }
        }
        sm100::tc_fence_before();
    } else {
        // the other CTAs read whatever is here: let loads in flight land, and the MMAs finish, first
        const int zero = 0;
        if (loads_issued) sm100::settle_ns(200000);
        if (mma_issued) {
            sm100::tc_commit(drain_bar);
            if (!sm100::wait_parity_bounded(drain_bar, 0, &zero, WAIT_BUDGET / 4)) atomicOr(&g_device_status, 0x8u);
        }
        sm100::tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if (S > 1) sm100::cluster_sync();
    if (quad)
        few_quad<BN>(p, tile, rank, S, sm100::smem_u32(acc), first);
    else if (p.M <= FEW_SINGLE)
        few_finish<BN, 1>(p, tile, rank, S, sm100::smem_u32(acc), first);
    else
        few_finish<BN, FEW_BATCH>(p, tile, rank, S, sm100::smem_u32(acc), first);
    if (S > 1) sm100::cluster_sync();  // no CTA leaves while another may read its accumulator
}

}  // namespace kern
}  // namespace mxfp6
