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
    int bias_vec, aux_vec, out_vec;  // 16-byte accesses of whole chunks are aligned
    int k_atoms;                     // MXFP6: N / 128
};

// Logistic sigmoid times v: v / (1 + e^-x). The quotient has no cancellation anywhere, and the
// hardware exponential and division keep it within a few FP32 ulp.
__device__ __forceinline__ float times_sigmoid(float v, float x) {
    return __fdividef(v, 1.0f + __expf(-x));
}

__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
        case ACT_RELU: return v < 0.0f ? 0.0f : v;  // NaN stays NaN
        case ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        // 0.5 v (1 + tanh(u)) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3)
        case ACT_GELU_TANH: return times_sigmoid(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
        case ACT_SILU: return times_sigmoid(v, v);
        default: return v;
    }
}

template <int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
    switch (act) {
#define MXFP6_ACT_CASE(A)                                        \
    case A:                                                      \
        _Pragma("unroll") for (int i = 0; i < N; i++) v[i] = activate(A, v[i]); \
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

template <int N>
__device__ __forceinline__ void store_elems(void* p, int type, size_t i, int valid, bool vec, const float (&v)[N]) {
    if (vec && valid >= N) {
        if (type == T_F32) {
            float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
            for (int k = 0; k < N / 4; k++) d[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        } else {
            uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i);
#pragma unroll
            for (int k = 0; k < N / 8; k++)
                d[k] = make_uint4(pack2(v[8 * k], v[8 * k + 1], type), pack2(v[8 * k + 2], v[8 * k + 3], type),
                                  pack2(v[8 * k + 4], v[8 * k + 5], type), pack2(v[8 * k + 6], v[8 * k + 7], type));
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (k < valid) store_elem(p, type, i + k, v[k]);
    }
}

// bias, activation and aux on N consecutive accumulators of (row, col..), `valid` of them inside D.
template <int N>
__device__ __forceinline__ void epi_apply(const Epi& e, int row, int col, int valid, float (&v)[N]) {
    if (e.bias) {
        float b[N];
        load_elems<N>(e.bias, e.bias_type, (size_t)col, valid, e.bias_vec != 0, b);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += b[i];
    }
    activate_all<N>(e.act, v);
    if (e.aux_op != AUX_NONE) {
        float a[N];
        load_elems<N>(e.aux, e.aux_type, (size_t)row * (size_t)e.ld_aux + (size_t)col, valid, e.aux_vec != 0, a);
        if (e.aux_op == AUX_ADD) {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += a[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] *= a[i];
        }
    }
}

// The same on four columns (col % 4 == 0) and their store, for the split-K second stage.
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

// The whole epilogue of one lane's chunk: accumulators of columns [col, col + 32) of row `row`.
// `valid` = N - col (> 0); MXFP6 output has N % 128 == 0, so its chunks are whole.
__device__ __forceinline__ void epi_chunk(const Epi& e, int row, int col, int valid, const uint32_t (&r)[32]) {
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
    epi_apply<32>(e, row, col, valid, v);
    if (e.out_type != T_MXFP6) {
        store_elems<32>(e.out, e.out_type, (size_t)row * (size_t)e.ldd + (size_t)col, valid, e.out_vec != 0, v);
        return;
    }
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) m = fmaxf(m, fabsf(v[i]));
    const uint32_t code = scale_code(m);
    const float inv = e8m0_reciprocal(code);
    uint32_t w[6];
    quantize16(v, inv, w[0], w[1], w[2]);
    quantize16(v + 16, inv, w[3], w[4], w[5]);
    uint2* d = reinterpret_cast<uint2*>(static_cast<uint8_t*>(e.out) + (size_t)row * (size_t)e.ldd + (size_t)(col / 4 * 3));
    d[0] = make_uint2(w[0], w[1]);
    d[1] = make_uint2(w[2], w[3]);
    d[2] = make_uint2(w[4], w[5]);
    e.scales[scale_atom_offset(row, col / 32, e.k_atoms)] = (uint8_t)code;
}

}  // namespace kern
}  // namespace mxfp6
