#pragma once
// Fused epilogue of the GEMM kernels: D = op(act(A·B + bias), aux), written as FP32, FP16, BF16 or
// quantised to MXFP6 (packed rows and tiled scales: the A operand of a following GEMM).
//
// A lane of an epilogue warp holds 32 consecutive columns of one output row, which is exactly one
// MXFP6 block: its maximum, scale and codes need no other thread. Everything is computed on the FP32
// accumulator and rounded once, to the output type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "quant.cuh"

namespace mxfp6 {
namespace kern {

// Element types (values of mxfp6_out_type) and, for `out_type`, MXFP6.
constexpr int T_F32 = 0, T_F16 = 1, T_BF16 = 2, T_MXFP6 = 3;
// Values of mxfp6_activation and mxfp6_aux_op.
constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4;
constexpr int AUX_NONE = 0, AUX_ADD = 1, AUX_MUL = 2;

struct Epi {
    const void* bias;   // [N] or null
    const void* aux;    // [M][ld_aux]
    void* out;          // [M][ldd] of out_type; MXFP6: packed rows of ldd bytes
    uint8_t* scales;    // MXFP6: tiled scales
    long long ld_aux, ldd;
    int bias_type, act, aux_op, aux_type, out_type;
    int aux_vec;            // 16-byte (1) or 32-byte (2) loads of whole aux chunks are aligned
    int out_vec;            // so are 16-byte (1) or 32-byte (2) stores; 0: neither, or aux is not
    int k_atoms;                     // MXFP6: N / 128
};

// 2^x and 1/x by the hardware approximations (2 and 1 ulp), which flush subnormal results to 0: without .ftz each carries
// instructions that rescale its argument.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LOG2E = 1.4426950408889634f;

// The activations work on two values at a time. What bounds an exposed epilogue is the special-function unit (16 results
// per clock and SM) about as much as issue slots: the packed arithmetic halves the latter, and two values share one
// reciprocal (1.5 special-function results per value, not 2). 2048 x 6144 x 2048 with residual, FP16: GELU 37.1 -> 33.7
// us (35.4 against 34.5 with the longer polynomial it has now), tanh GELU 36.7 -> 33.5, SiLU 34.6 -> 33.4; packed
// arithmetic with a reciprocal per value 35.1 / 35.6 / 34.8.
__device__ __forceinline__ F2 ex2(F2 x) {
    float a, b;
    split(x, a, b);
    return pair(ex2(a), ex2(b));
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN stays NaN
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 1/a and 1/b. SHARE: with one reciprocal, from 1/(ab), for a and b in [1, 2^63].
template <bool SHARE>
__device__ __forceinline__ F2 rcp(float a, float b) {
    if constexpr (!SHARE) return pair(rcp(a), rcp(b));
    return both(rcp(a * b)) * pair(b, a);
}

// v / (1 + 2^y) for two values, y <= 62 or NaN where v is.
template <bool SHARE>
__device__ __forceinline__ F2 over_one_plus_ex2(F2 v, F2 y) {
    float a, b;
    split(ex2(y) + both(1.0f), a, b);
    if constexpr (!SHARE) return v * rcp<false>(a, b);
    return v * rcp<true>(fminf(a, 0x1p63f), fminf(b, 0x1p63f));  // a NaN must not reach the other value
}

// v Phi(v) = max(v, 0) - |v| erfc(|v| / sqrt(2)) / 2, and erfc(u / sqrt(2)) / 2 = (a1 t + ... + a8 t^8) e^(-u^2 / 2),
// t = 1 / (1 + p u). The polynomial is a fit of this header's own: the quotient of the two sides is within 7.8e-8 of 1 for
// u in [0, 13.3] (least largest relative error, at this p), so that the negative tail keeps its digits, which a form with an
// absolute bound does not (with the five coefficients of Abramowitz and Stegun 7.1.26 it was 2e-3 off at -5, 1e-2 at -8).
// e^(-u^2 / 2) = 2^(-u^2 log2(e) / 2) adds its argument's rounding, 2^-23 u^2; from u = 13.3 on it is 0. In all the relative
// error is below 2^-19 + 2^-23 v^2: t is off by 5 half steps at most, which count 3.4 times at u = 0.
template <bool SHARE>
__device__ __forceinline__ F2 gelu_erf(float v0, float v1) {
    const float u0 = fminf(fabsf(v0), 16.0f), u1 = fminf(fabsf(v1), 16.0f);
    const F2 u = pair(u0, u1);
    float a, b;
    split(fma(u, both(0.233f), both(1.0f)), a, b);
    const F2 t = rcp<SHARE>(a, b);
    F2 q = fma(t, both(-0.0687599108f), both(0.235863566f));
    q = fma(q, t, both(-0.184671089f));
    q = fma(q, t, both(0.212113991f));
    q = fma(q, t, both(0.0195844453f));
    q = fma(q, t, both(0.101660840f));
    q = fma(q, t, both(0.0911546126f));
    q = fma(q, t, both(0.0930535197f));
    const F2 half_erfc = q * t * ex2(u * u * both(-0.5f * LOG2E));
    return fma(pair(-u0, -u1), half_erfc, pair(max_nan(v0, 0.0f), max_nan(v1, 0.0f)));
}

// The quotients have no cancellation anywhere: a few FP32 ulp, and on the negative side the rounding of the exponent, 2^-23 |v|
// for SiLU (2^-20 + 2^-23 |v| in all) and 2^-21 |v| (1 + 0.0447 v^2) for the tanh form of GELU (2^-20 more in all). Below -43
// (-7.5) SiLU (the tanh form) is the value there, -9e-18 (-4e-18), instead of one even nearer to 0: 1 + e^43 is what the
// shared reciprocal takes.
template <int ACT, bool SHARE>
__device__ __forceinline__ F2 activate(float v0, float v1) {
    if constexpr (ACT == ACT_RELU) return pair(max_nan(v0, 0.0f), max_nan(v1, 0.0f));
    if constexpr (ACT == ACT_GELU) return gelu_erf<SHARE>(v0, v1);
    if constexpr (ACT == ACT_GELU_TANH) {
        // 0.5 v (1 + tanh(u)) = v / (1 + e^(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
        const F2 v = pair(max_nan(v0, -7.5f), max_nan(v1, -7.5f));
        constexpr float c = -LOG2E * 1.5957691216057308f;
        return over_one_plus_ex2<SHARE>(v, v * fma(v * v, both(c * 0.044715f), both(c)));
    }
    const F2 v = pair(max_nan(v0, -43.0f), max_nan(v1, -43.0f));
    return over_one_plus_ex2<SHARE>(v, v * both(-LOG2E));
}

// Values of one row in pairs; a pair's shared reciprocal makes the last bit of one depend on the other. EACH: values of
// different rows, each with its own, so that no row's result depends on another row.
template <int N, bool EACH = false>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
    static_assert(N % 2 == 0 || (N == 1 && EACH), "pairs");
    switch (act) {
#define MXFP6_ACT_CASE(A)                                                  \
    case A:                                                                \
        _Pragma("unroll") for (int i = 0; i < N; i += 2) {                 \
            float a, b;                                                    \
            split(activate<A, !EACH>(v[i], v[N > 1 ? i + 1 : i]), a, b);   \
            v[i] = a;                                                      \
            if (N > 1) v[N > 1 ? i + 1 : i] = b;                           \
        }                                                                  \
        break;
        MXFP6_ACT_CASE(ACT_RELU)
        MXFP6_ACT_CASE(ACT_GELU)
        MXFP6_ACT_CASE(ACT_GELU_TANH)
        MXFP6_ACT_CASE(ACT_SILU)
#undef MXFP6_ACT_CASE
        default: break;
    }
}

__device__ __forceinline__ float load_elem(const void* p, int type, size_t i) {
    if (type == T_F32) return static_cast<const float*>(p)[i];
    if (type == T_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int type, size_t i, float v) {
    if (type == T_F32)
        static_cast<float*>(p)[i] = v;
    else if (type == T_F16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void unpack2(uint32_t w, int type, float& a, float& b) {
    if (type == T_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x;
        b = f.y;
    } else {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {
    if (type == T_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// N consecutive elements (N % 8 == 0) from element `i` on: 16-byte loads where `vec`, else one by one
// below `valid`; the rest are 0.
template <int N>
__device__ __forceinline__ void load_elems(const void* p, int type, size_t i, int valid, bool vec, float (&v)[N]) {
    if (vec && valid >= N) {
        if (type == T_F32) {
            const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
            for (int k = 0; k < N / 4; k++) {
                const float4 q = s[k];
                v[4 * k] = q.x;
                v[4 * k + 1] = q.y;
                v[4 * k + 2] = q.z;
                v[4 * k + 3] = q.w;
            }
        } else {
            const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
            for (int k = 0; k < N / 8; k++) {
                const uint4 q = s[k];
                unpack2(q.x, type, v[8 * k], v[8 * k + 1]);
                unpack2(q.y, type, v[8 * k + 2], v[8 * k + 3]);
                unpack2(q.z, type, v[8 * k + 4], v[8 * k + 5]);
                unpack2(q.w, type, v[8 * k + 6], v[8 * k + 7]);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = k < valid ? load_elem(p, type, i + k) : 0.0f;
    }
}

// bias, activation and aux on four columns (col % 4 == 0), and their store, for the split-K second stage.
__device__ __forceinline__ void epi_apply4(const Epi& e, int row, int col, int valid, float (&v)[4]) {
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < valid) v[i] += load_elem(e.bias, e.bias_type, (size_t)(col + i));
    }
    activate_all<4>(e.act, v);
    if (e.aux_op != AUX_NONE) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < valid) {
                const float a = load_elem(e.aux, e.aux_type, (size_t)row * (size_t)e.ld_aux + (size_t)(col + i));
                v[i] = e.aux_op == AUX_ADD ? v[i] + a : v[i] * a;
            }
    }
}
__device__ __forceinline__ void store_elems4(const Epi& e, int row, int col, int valid, const float (&v)[4]) {
    const size_t i = (size_t)row * (size_t)e.ldd + (size_t)col;
    if (e.out_vec && valid >= 4) {
        if (e.out_type == T_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(e.out) + i) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(e.out) + i) =
                make_uint2(pack2(v[0], v[1], e.out_type), pack2(v[2], v[3], e.out_type));
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < valid) store_elem(e.out, e.out_type, i + k, v[k]);
    }
}

// A warp's copy of a tile's bias in shared memory, CHUNKS chunks of 32 columns `step` columns apart from
// `col` on: it is loaded while the warp waits for the accumulator, and read back as broadcasts. Loading
// it from global memory chunk by chunk cost 2.5 us (no activation) to 6 us of 2048 x 6144 x 2048.
template <int CHUNKS>
__device__ __forceinline__ void epi_load_bias(const Epi& e, int col, int step, int N, float* bias) {
    const int lane = threadIdx.x & 31;
    float v[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
        const int c = col + i * step + lane;
        v[i] = e.bias && c < N ? load_elem(e.bias, e.bias_type, (size_t)c) : 0.0f;
    }
    __syncwarp();  // the previous tile's reads
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) bias[32 * i + lane] = v[i];
    __syncwarp();
}

// 8 words as one 32-byte store (full L2 sectors).
__device__ __forceinline__ void st_v8(void* dst, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// NWORDS consecutive words of one row: 256-bit stores where the row is 32-byte aligned, else 128-bit.
template <int NWORDS>
__device__ __forceinline__ void store_words(void* dst, const uint32_t* w, bool align32) {
    if (align32) {
#pragma unroll
        for (int i = 0; i < NWORDS / 8; i++) st_v8(static_cast<uint8_t*>(dst) + 32 * i, w + 8 * i);
    } else {
        uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
        for (int i = 0; i < NWORDS / 4; i++) d[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
}

// One lane's aux operand of a chunk as loaded. It is loaded a chunk ahead of its use: the loads of the next chunk are in
// flight while this one is computed and stored. Row layout (lane = row): 32 columns (FP32: 32 words, else 16). Column
// layout (lane = column): a word for each of 32 rows, 16-bit elements in its low half.
template <bool COLUMNS>
struct AuxRaw;
template <>
struct AuxRaw<false> {
    uint4 q[8];
};
template <>
struct AuxRaw<true> {
    uint32_t w[32];
};
__device__ __forceinline__ void epi_load_aux(const Epi& e, int row0, int M, int col, int N, AuxRaw<true>& a) {
    const int c = col + (threadIdx.x & 31), rows = M - row0;
    if (e.aux_op == AUX_NONE || rows <= 0 || col < 0 || c >= N) return;
    const size_t i = (size_t)row0 * (size_t)e.ld_aux + (size_t)c;
    if (e.aux_type == T_F32) {
        const uint32_t* s = static_cast<const uint32_t*>(e.aux) + i;
#pragma unroll
        for (int k = 0; k < 32; k++) {
            if (k < rows) a.w[k] = *s;
            s += e.ld_aux;
        }
    } else {
        const uint16_t* s = static_cast<const uint16_t*>(e.aux) + i;
#pragma unroll
        for (int k = 0; k < 32; k++) {
            if (k < rows) a.w[k] = *s;
            s += e.ld_aux;
        }
    }
}
// 32 bytes in one load: with a lane per row, a load costs the cache one look-up per lane whatever its width.
__device__ __forceinline__ void ld_v8(const uint4* s, uint4& a, uint4& b) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(s)
                 : "memory");
}
__device__ __forceinline__ void epi_load_aux(const Epi& e, int row0, int M, int col, int N, AuxRaw<false>& a) {
    const int row = row0 + (threadIdx.x & 31);
    const bool live = row < M && col >= 0 && col + 32 <= N;
    if (e.aux_op == AUX_NONE || !e.aux_vec || !live) return;
    const size_t i = (size_t)row * (size_t)e.ld_aux + (size_t)col;
    const uint4* s = e.aux_type == T_F32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(e.aux) + i)
                                         : reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.aux) + i);
    if (e.aux_vec == 2) {
        ld_v8(s, a.q[0], a.q[1]);
        ld_v8(s + 2, a.q[2], a.q[3]);
        if (e.aux_type == T_F32) {
            ld_v8(s + 4, a.q[4], a.q[5]);
            ld_v8(s + 6, a.q[6], a.q[7]);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) a.q[k] = s[k];
    if (e.aux_type == T_F32) {
#pragma unroll
        for (int k = 4; k < 8; k++) a.q[k] = s[k];
    }
}

__device__ __forceinline__ void epi_join(int op, float& v, float a) {
    v = op == AUX_ADD ? v + a : v * a;
}

// Per epilogue warp: a 32 x 32 FP32 tile of shared memory, rows 36 words apart (16-byte row writes and
// column reads both spread over all banks).
constexpr int EPI_TILE_PITCH = 36;
constexpr int EPI_TILE_BYTES = 32 * EPI_TILE_PITCH * 4;

// The warp's rows of the last, partial chunk from its shared-memory tile, lane = column, four rows at a time (the
// code of eight, inlined into the chunk loop, costs whole chunks 1.5 us of 2048 x 6144 x 2048 with residual).
// `in`: the lane's column is inside D.
template <int OT>
__device__ __forceinline__ void epi_rows(const Epi& e, int row0, int rows, int col, bool in, float bias,
                                         const float* tile) {
    using Out = std::conditional_t<OT == T_F32, float, std::conditional_t<OT == T_F16, __half, __nv_bfloat16>>;
    Out* out = static_cast<Out*>(e.out) + (size_t)row0 * (size_t)e.ldd + (size_t)col;
    size_t ai = (size_t)row0 * (size_t)e.ld_aux + (size_t)col;
#pragma unroll 1
    for (int q = 0; q < rows; q += 4) {
        float v[4], a[4];
#pragma unroll
        for (int k = 0; k < 4; k++) a[k] = 0.0f;
        if (e.aux_op != AUX_NONE) {
            if (e.aux_type == T_F32) {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (in && q + k < rows) a[k] = load_elem(e.aux, T_F32, ai + (size_t)k * (size_t)e.ld_aux);
            } else if (e.aux_type == T_F16) {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (in && q + k < rows) a[k] = load_elem(e.aux, T_F16, ai + (size_t)k * (size_t)e.ld_aux);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (in && q + k < rows) a[k] = load_elem(e.aux, T_BF16, ai + (size_t)k * (size_t)e.ld_aux);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = tile[(q + k) * EPI_TILE_PITCH] + bias;
        activate_all<4, true>(e.act, v);
        if (e.aux_op != AUX_NONE) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = e.aux_op == AUX_ADD ? v[k] + a[k] : v[k] * a[k];
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (in && q + k < rows) store_elem(out + (size_t)k * (size_t)e.ldd, OT, 0, v[k]);
        out += (size_t)4 * (size_t)e.ldd;
        ai += (size_t)4 * (size_t)e.ld_aux;
    }
}

// bias and activation of a lane's row of a chunk, `bias` the chunk's 32 values in shared memory (zeros without a bias).
__device__ __forceinline__ void epi_activate(const Epi& e, const uint32_t (&r)[32], const float* bias, float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float4 q = reinterpret_cast<const float4*>(bias)[i];
            split(pair(v[4 * i], v[4 * i + 1]) + pair(q.x, q.y), v[4 * i], v[4 * i + 1]);
            split(pair(v[4 * i + 2], v[4 * i + 3]) + pair(q.z, q.w), v[4 * i + 2], v[4 * i + 3]);
        }
    }
    activate_all<32>(e.act, v);
}

// The warp's activated rows from its shared-memory tile, lane = column: aux, and a store of consecutive addresses of one
// row at a time. AT: aux type, or -1 for none.
template <int OT, int AT>
__device__ __forceinline__ void epi_columns(const Epi& e, int row0, int rows, int col, bool in, const AuxRaw<true>& a,
                                            const float* tile) {
    using Out = std::conditional_t<OT == T_F32, float, std::conditional_t<OT == T_F16, __half, __nv_bfloat16>>;
    Out* out = static_cast<Out*>(e.out) + (size_t)row0 * (size_t)e.ldd + (size_t)col;
#pragma unroll
    for (int k = 0; k < 32; k++) {
        float v = tile[k * EPI_TILE_PITCH];
        if constexpr (AT >= 0) {
            uint32_t w = a.w[k];
            asm volatile("" : "+r"(w));  // convert here: hoisted to the load, the conversion would wait for it
            epi_join(e.aux_op, v, AT == T_F32 ? __uint_as_float(w)
                                  : AT == T_F16 ? __half2float(__ushort_as_half((unsigned short)w)) : __uint_as_float(w << 16));
        }
        if (in && k < rows) store_elem(out, OT, 0, v);
        out += e.ldd;
    }
}
template <int OT>
__device__ __forceinline__ void epi_columns(const Epi& e, int row0, int rows, int col, bool in, const AuxRaw<true>& a,
                                            const float* tile) {
    if (e.aux_op == AUX_NONE)
        epi_columns<OT, -1>(e, row0, rows, col, in, a, tile);
    else if (e.aux_type == T_F32)
        epi_columns<OT, T_F32>(e, row0, rows, col, in, a, tile);
    else if (e.aux_type == T_F16)
        epi_columns<OT, T_F16>(e, row0, rows, col, in, a, tile);
    else
        epi_columns<OT, T_BF16>(e, row0, rows, col, in, a, tile);
}

// The epilogue of a warp's chunk, in the column layout: for outputs whose rows are not 16-byte aligned (odd N, odd pitch),
// or whose aux operand's are not. Lane l holds the accumulators of columns [col, col + 32) of row row0 + l; after the
// activation the chunk goes through `tile`, this warp's shared-memory tile, to lane = column, because a lane per row would
// touch 32 sectors with each 2- or 4-byte access. `valid` = N - col (> 0, the same in every lane).
__device__ __forceinline__ void epi_chunk(const Epi& e, int row0, int M, int col, int valid, const uint32_t (&r)[32],
                                          const AuxRaw<true>& aux, const float* bias, float* tile) {
    const int lane = threadIdx.x & 31, rows = M - row0;
    if (rows <= 0) return;
    float v[32];
    epi_activate(e, r, bias, v);
    float4* mine = reinterpret_cast<float4*>(tile + lane * EPI_TILE_PITCH);
#pragma unroll
    for (int i = 0; i < 8; i++) mine[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
    if (e.out_type == T_F32)
        epi_columns<T_F32>(e, row0, rows, col + lane, lane < valid, aux, tile + lane);
    else if (e.out_type == T_F16)
        epi_columns<T_F16>(e, row0, rows, col + lane, lane < valid, aux, tile + lane);
    else
        epi_columns<T_BF16>(e, row0, rows, col + lane, lane < valid, aux, tile + lane);
    __syncwarp();  // the tile is rewritten by the next chunk
}

// The same in the row layout: every lane stores its row's 32 columns with wide accesses, and of an MXFP6 output
// quantises them, since they are one block. The last chunk of a width that is no multiple of 32 goes through `tile`.
__device__ __forceinline__ void epi_chunk(const Epi& e, int row0, int M, int col, int valid, const uint32_t (&r)[32],
                                          const AuxRaw<false>& aux, const float* bias, float* tile) {
    const int lane = threadIdx.x & 31, row = row0 + lane;
    if (e.out_type != T_MXFP6 && valid < 32) {
        const int rows = M - row0 < 32 ? M - row0 : 32;
        if (rows <= 0) return;
        uint4* mine = reinterpret_cast<uint4*>(tile + lane * EPI_TILE_PITCH);
#pragma unroll
        for (int i = 0; i < 8; i++) mine[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        __syncwarp();
        const bool in = lane < valid;
        if (e.out_type == T_F32)
            epi_rows<T_F32>(e, row0, rows, col + lane, in, bias[lane], tile + lane);
        else if (e.out_type == T_F16)
            epi_rows<T_F16>(e, row0, rows, col + lane, in, bias[lane], tile + lane);
        else
            epi_rows<T_BF16>(e, row0, rows, col + lane, in, bias[lane], tile + lane);
        __syncwarp();  // the tile is rewritten by the next chunk
        return;
    }
    if (row >= M) return;
    float v[32];
    epi_activate(e, r, bias, v);
    if (e.aux_op != AUX_NONE) {
        if (!e.aux_vec) {  // MXFP6 output only
#pragma unroll
            for (int i = 0; i < 32; i++)
                epi_join(e.aux_op, v[i], load_elem(e.aux, e.aux_type, (size_t)row * (size_t)e.ld_aux + (size_t)(col + i)));
        } else if (e.aux_type == T_F32) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                epi_join(e.aux_op, v[4 * k], __uint_as_float(aux.q[k].x));
                epi_join(e.aux_op, v[4 * k + 1], __uint_as_float(aux.q[k].y));
                epi_join(e.aux_op, v[4 * k + 2], __uint_as_float(aux.q[k].z));
                epi_join(e.aux_op, v[4 * k + 3], __uint_as_float(aux.q[k].w));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t w[4] = {aux.q[k].x, aux.q[k].y, aux.q[k].z, aux.q[k].w};
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    float a, b;
                    unpack2(w[h], e.aux_type, a, b);
                    epi_join(e.aux_op, v[8 * k + 2 * h], a);
                    epi_join(e.aux_op, v[8 * k + 2 * h + 1], b);
                }
            }
        }
    }
    if (e.out_type == T_F32) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; i++) w[i] = __float_as_uint(v[i]);
        store_words<32>(static_cast<float*>(e.out) + (size_t)row * (size_t)e.ldd + (size_t)col, w, e.out_vec == 2);
        return;
    }
    if (e.out_type != T_MXFP6) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = pack2(v[2 * i], v[2 * i + 1], e.out_type);
        store_words<16>(static_cast<uint16_t*>(e.out) + (size_t)row * (size_t)e.ldd + (size_t)col, w, e.out_vec == 2);
        return;
    }
    bool nan0, nan1;
    const float m0 = max_abs16(v, nan0), m1 = max_abs16(v + 16, nan1);
    const uint32_t code = scale_code(fmaxf(m0, m1));
    const float inv = e8m0_reciprocal(code);
    uint32_t w[6];
    quantize16(v, inv, nan0, w[0], w[1], w[2]);
    quantize16(v + 16, inv, nan1, w[3], w[4], w[5]);
    uint8_t* d = static_cast<uint8_t*>(e.out) + (size_t)row * (size_t)e.ldd + (size_t)(col / 4 * 3);
    if (col & 32) {  // 24 bytes from an odd multiple of 8 on, else from a multiple of 16
        *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint4*>(d + 8) = make_uint4(w[2], w[3], w[4], w[5]);
    } else {
        *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint2*>(d + 16) = make_uint2(w[4], w[5]);
    }
    e.scales[scale_atom_offset(row, col / 32, e.k_atoms)] = (uint8_t)code;
}

}  // namespace kern
}  // namespace mxfp6
