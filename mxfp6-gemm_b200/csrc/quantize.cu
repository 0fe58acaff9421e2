// Device-side MXFP6 quantiser: the reference's host quantize_to_mxfp6
// (include/mxfp6/preprocess.hpp:51-97 of eeezio/mxfp6-gemm) run on the GPU, bit for bit:
//   per row, per 32-element block: scale = smallest power of two >= max|x| / 7.5 (E8M0 code,
//   127 for an all-zero block, NaN inputs ignored by the max), codes = nearest E2M3 of x/scale
//   (ties to even, saturating at 7.5; NaN -> 0x18, as the reference's conversion gives on x86-64),
//   packed four codes per three bytes, least significant bits first.
// It is the step before the GEMM for activations (the FFN's A operand), so it writes the scales
// either raw [rows][cols/32] or directly in the GEMM's 128x4 atom layout.
//
// Traffic: each element reads 4 bytes and writes 0.75 + 1/32. A warp quantises a 512-element
// chunk: 16 consecutive values per lane (four float4 loads), a 32-value block per lane pair, and
// each lane writes its own 12 packed bytes as three aligned words (quantize_kernel).
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>

#include "mxfp6_gemm.h"
#include "epilogue.cuh"
#include "host.hpp"
#include "quant.cuh"
#include "sm100_ptx.cuh"

namespace mxfp6 {
void note_launch();  // launch counter (gemm.cu)

namespace {

template <typename T>
struct TypeOf;
template <>
struct TypeOf<__half> {
    static constexpr int value = kern::T_F16;
};
template <>
struct TypeOf<__nv_bfloat16> {
    static constexpr int value = kern::T_BF16;
};

// One warp quantises a 512-element chunk of a row: lane l owns the 16 consecutive values
// [16 l, 16 l + 16), so each 32-value block spans the lane pair (2b, 2b + 1) (one shuffle for its
// max) and each lane packs its own 16 codes into 12 bytes = 3 words (bytes [12 l, 12 l + 12) of
// the chunk's 384): no packing shuffles, and a warp's stores cover 384 contiguous bytes.
// Grid: x covers the chunks of a row (8 warps per block), y the rows.
__global__ void __launch_bounds__(256) quantize_kernel(const float* __restrict__ in, int rows, int cols,
                                                       uint8_t* __restrict__ packed, int out_row_bytes,
                                                       uint8_t* __restrict__ scales, int scale_cols, int tiled) {
    const int lane = threadIdx.x & 31;
    const int chunk = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = blockIdx.y;
    if (chunk * 512 >= cols || row >= rows) return;
    const int col = chunk * 512 + 16 * lane;  // first of this lane's 16 values
    const bool live = col < cols;             // cols % 32 == 0: a lane's 16 values are all in or all out
    float v[16];
    if (live) {
        const float4* src = reinterpret_cast<const float4*>(in + (size_t)row * cols + col);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 q = __ldg(src + i);
            v[4 * i] = q.x;
            v[4 * i + 1] = q.y;
            v[4 * i + 2] = q.z;
            v[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = 0.0f;
    }
    bool nan;
    float m = max_abs16(v, nan);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t code = scale_code(m);
    uint32_t w0, w1, w2;
    quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
    if (live) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(packed + (size_t)row * out_row_bytes + (size_t)col / 4 * 3);
        dst[0] = w0;
        dst[1] = w1;
        dst[2] = w2;
        if ((lane & 1) == 0) {
            const int j = col / 32;  // block index in the row
            size_t off;
            if (tiled) {
                const size_t atom = (size_t)(row / 128) * (size_t)(scale_cols / 4) + (size_t)(j / 4);
                off = atom * 512 + (size_t)((row % 32) * 16 + ((row % 128) / 32) * 4 + (j % 4));
            } else {
                off = (size_t)row * scale_cols + j;
            }
            scales[off] = (uint8_t)code;
        }
    }
}

// A lane's 16 values as loaded.
template <typename In>
struct Raw16 {
    uint4 q[sizeof(In)];  // 16 * sizeof(In) bytes
};
template <typename In, bool VEC>
__device__ __forceinline__ void load_raw(const In* src, Raw16<In>& r) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(In); i++) r.q[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
        In* d = reinterpret_cast<In*>(r.q);
#pragma unroll
        for (int i = 0; i < 16; i++) d[i] = src[i];
    }
}
__device__ __forceinline__ void raw_values(const Raw16<float>& r, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[4 * i] = __uint_as_float(r.q[i].x);
        v[4 * i + 1] = __uint_as_float(r.q[i].y);
        v[4 * i + 2] = __uint_as_float(r.q[i].z);
        v[4 * i + 3] = __uint_as_float(r.q[i].w);
    }
}
template <typename In>
__device__ __forceinline__ void raw_values(const Raw16<In>& r, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        kern::unpack2(r.q[i].x, TypeOf<In>::value, v[8 * i], v[8 * i + 1]);
        kern::unpack2(r.q[i].y, TypeOf<In>::value, v[8 * i + 2], v[8 * i + 3]);
        kern::unpack2(r.q[i].z, TypeOf<In>::value, v[8 * i + 4], v[8 * i + 5]);
        kern::unpack2(r.q[i].w, TypeOf<In>::value, v[8 * i + 6], v[8 * i + 7]);
    }
}

// The quantiser for any input type and row stride, padding in the same pass: the lane layout of
// quantize_kernel, with the tail [cols, padded_cols) written as zero codes with the finite scale 127. A
// BF16 element reads 2 bytes and writes 0.78, so the instructions per element count as much as the bytes: a warp
// takes its 512 columns of ROWS consecutive rows, all loads first, and sets up its addresses once.
// VEC: 16-byte aligned rows (ld and base), so a lane's 16 values are two (four for FP32) wide loads. They are plain loads of
// a plain pointer: the kernel before may still be writing `in` when this one starts (griddep_wait), so it is not constant
// for the kernel's life.
template <typename In, bool VEC, int ROWS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const In* in, int rows, int cols, long long ld,
                                                            int padded_cols, uint8_t* __restrict__ packed,
                                                            uint8_t* __restrict__ scales, int tiled) {
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();  // launched with programmatic stream serialization
    const int lane = threadIdx.x & 31;
    const int chunk = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if ((long long)chunk * 512 >= padded_cols) return;
    const int col = chunk * 512 + 16 * lane;
    const bool live = col < cols;  // cols % 32 == 0: a lane's 16 values are all in or all out
    const bool kept = col < padded_cols;
    const size_t out_row_bytes = (size_t)(padded_cols / 4 * 3);
    const int j = col / 32;
    for (int row0 = blockIdx.y * ROWS; row0 < rows; row0 += gridDim.y * ROWS) {
        const In* src = in + (size_t)row0 * (size_t)ld + (size_t)col;
        Raw16<In> raw[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(In); k++) raw[i].q[k] = make_uint4(0u, 0u, 0u, 0u);
            if (live && row0 + i < rows) load_raw<In, VEC>(src, raw[i]);
            src += ld;
        }
        uint8_t* dst = packed + (size_t)row0 * out_row_bytes + (size_t)(col / 4 * 3);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            float v[16];
            raw_values(raw[i], v);
            bool nan;
            float m = max_abs16(v, nan);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            const uint32_t code = scale_code(m);
            uint32_t w0, w1, w2;
            quantize16(v, e8m0_reciprocal(code), nan, w0, w1, w2);
            if (kept && row0 + i < rows) {
                reinterpret_cast<uint32_t*>(dst)[0] = w0;
                reinterpret_cast<uint32_t*>(dst)[1] = w1;
                reinterpret_cast<uint32_t*>(dst)[2] = w2;
                if ((lane & 1) == 0) {
                    const size_t off = tiled ? scale_atom_offset(row0 + i, j, padded_cols / 128)
                                             : (size_t)(row0 + i) * (size_t)(padded_cols / 32) + (size_t)j;
                    scales[off] = (uint8_t)code;
                }
            }
            dst += out_row_bytes;
        }
    }
}

// Padded rows: zero bytes [row_bytes, out_row_bytes) of each row, and give the scale blocks past
// the data the finite code 127 (a zero K-tail then contributes 0, never NaN).
__global__ void pad_tail_kernel(int rows, int row_bytes, uint8_t* __restrict__ packed, int out_row_bytes,
                                uint8_t* __restrict__ scales, int data_blocks, int scale_cols, int tiled) {
    const int row = blockIdx.x;
    if (row >= rows) return;
    uint8_t* dst = packed + (size_t)row * out_row_bytes;
    for (int i = row_bytes + threadIdx.x; i < out_row_bytes; i += blockDim.x) dst[i] = 0;
    for (int j = data_blocks + threadIdx.x; j < scale_cols; j += blockDim.x) {
        size_t off;
        if (tiled) {
            const size_t atom = (size_t)(row / 128) * (size_t)(scale_cols / 4) + (size_t)(j / 4);
            off = atom * 512 + (size_t)((row % 32) * 16 + ((row % 128) / 32) * 4 + (j % 4));
        } else {
            off = (size_t)row * scale_cols + j;
        }
        scales[off] = 127;
    }
}

// Loads of data that is read once, kept after the griddep_wait() before them (14.4 us against 16.2 with plain loads for
// 8192 rows of 6120 bytes).
__device__ __forceinline__ uint8_t ld_stream(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.cs.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return (uint8_t)v;
}
__device__ __forceinline__ uint32_t ld_stream(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.cs.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 ld_stream(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.cs.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// Copy rows between strides, zero-filling each destination row past bytes_used (re-padding
// compact operand rows for the tensor-memory accelerator). One block per row, in units of U
// bytes: the largest of 16, 8, 4, 1 that divides both bases, both strides and bytes_used, so
// that a compact stride of 3K/4 (a multiple of 8) still moves 8-byte words. HBM bound.
template <typename U>
__global__ void __launch_bounds__(256) repad_kernel(const uint8_t* src, int rows, int src_row_bytes,
                                                    int bytes_used, uint8_t* __restrict__ dst, int dst_row_bytes) {
    sm100::griddep_launch_dependents();
    sm100::griddep_wait();  // launched with programmatic stream serialization (launch_repad)
    const int row = blockIdx.x;
    if (row >= rows) return;
    const U* s = reinterpret_cast<const U*>(src + (size_t)row * src_row_bytes);
    U* d = reinterpret_cast<U*>(dst + (size_t)row * dst_row_bytes);
    const int used = bytes_used / (int)sizeof(U), total = dst_row_bytes / (int)sizeof(U);
    const int bd = blockDim.x;
    // four loads in flight per thread before their stores
    for (int base = threadIdx.x; base < used; base += 4 * bd) {
        U r[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (base + k * bd < used) r[k] = ld_stream(s + base + k * bd);
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (base + k * bd < used) d[base + k * bd] = r[k];
    }
    U zero;
    memset(&zero, 0, sizeof(U));
    for (int i = used + threadIdx.x; i < total; i += bd) d[i] = zero;
}

}  // namespace

template <typename In, int ROWS>
cudaError_t launch_quantize_rows_of(const In* in, int rows, int cols, long long ld, int padded_cols, uint8_t* packed,
                                    uint8_t* scales, int tiled, cudaStream_t stream) {
    const bool vec = (reinterpret_cast<uintptr_t>(in) & 15) == 0 && (rows == 1 || ld * (long long)sizeof(In) % 16 == 0);
    const int groups = (rows + ROWS - 1) / ROWS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((padded_cols + 4095) / 4096), (unsigned)(groups < 65535 ? groups : 65535), 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return vec ? cudaLaunchKernelEx(&cfg, quantize_rows_kernel<In, true, ROWS>, in, rows, cols, ld, padded_cols, packed,
                                    scales, tiled)
               : cudaLaunchKernelEx(&cfg, quantize_rows_kernel<In, false, ROWS>, in, rows, cols, ld, padded_cols, packed,
                                    scales, tiled);
}

// Rows per warp: four (two of FP32: the same registers) once that still fills the GPU's warps, else one.
template <typename In>
cudaError_t launch_quantize_rows(const In* in, int rows, int cols, long long ld, int padded_cols, uint8_t* packed,
                                 uint8_t* scales, int tiled, cudaStream_t stream) {
    constexpr int MANY = sizeof(In) == 4 ? 2 : 4;
    const long long warps = (long long)rows * ((padded_cols + 511) / 512);
    if (warps >= (long long)host::sm_count() * 48 * MANY)
        return launch_quantize_rows_of<In, MANY>(in, rows, cols, ld, padded_cols, packed, scales, tiled, stream);
    return launch_quantize_rows_of<In, 1>(in, rows, cols, ld, padded_cols, packed, scales, tiled, stream);
}

// Launch the re-pad copy with the widest unit the pointers and strides allow (used by
// mxfp6_repad_rows_device and by gemm() for compact A with a large enough workspace).
cudaError_t launch_repad(const uint8_t* src, int rows, int src_row_bytes, int bytes_used, uint8_t* dst,
                         int dst_row_bytes, cudaStream_t stream) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) |
                        (uintptr_t)src_row_bytes | (uintptr_t)dst_row_bytes | (uintptr_t)bytes_used;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((a & 15) == 0)
        return cudaLaunchKernelEx(&cfg, repad_kernel<uint4>, src, rows, src_row_bytes, bytes_used, dst, dst_row_bytes);
    if ((a & 7) == 0)
        return cudaLaunchKernelEx(&cfg, repad_kernel<uint2>, src, rows, src_row_bytes, bytes_used, dst, dst_row_bytes);
    if ((a & 3) == 0)
        return cudaLaunchKernelEx(&cfg, repad_kernel<uint32_t>, src, rows, src_row_bytes, bytes_used, dst,
                                  dst_row_bytes);
    return cudaLaunchKernelEx(&cfg, repad_kernel<uint8_t>, src, rows, src_row_bytes, bytes_used, dst, dst_row_bytes);
}

}  // namespace mxfp6

extern "C" int mxfp6_quantize_device_padded(const float* d_mat, int rows, int cols, int padded_cols, uint8_t* d_packed,
                                            uint8_t* d_scales, int scale_layout, void* stream) {
    using namespace mxfp6;
    if (!d_mat || !d_packed || !d_scales || rows <= 0 || cols <= 0 || cols % 32 || padded_cols < cols ||
        padded_cols % 32 || (scale_layout != 0 && scale_layout != 1) || (scale_layout == 1 && padded_cols % 128)) {
        std::fprintf(stderr, "[mxfp6] quantize_device: invalid arguments (%d x %d padded to %d, layout %d)\n", rows,
                     cols, padded_cols, scale_layout);
        return MXFP6_ERR_INVALID_SHAPE;
    }
    const int out_row_bytes = padded_cols / 4 * 3;
    if ((reinterpret_cast<uintptr_t>(d_mat) & 15) || (reinterpret_cast<uintptr_t>(d_packed) & 3) || (cols % 4) ||
        (out_row_bytes % 4)) {
        std::fprintf(stderr, "[mxfp6] quantize_device: input must be 16-byte and output 4-byte aligned\n");
        return MXFP6_ERR_MISALIGNED;
    }
    if (rows > 65535) {
        std::fprintf(stderr, "[mxfp6] quantize_device: at most 65535 rows per call\n");
        return MXFP6_ERR_INVALID_SHAPE;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int chunks = (cols + 511) / 512;
    dim3 grid((chunks + 7) / 8, rows);
    quantize_kernel<<<grid, 256, 0, st>>>(d_mat, rows, cols, d_packed, out_row_bytes, d_scales, padded_cols / 32,
                                          scale_layout);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && padded_cols > cols) {
        pad_tail_kernel<<<rows, 128, 0, st>>>(rows, cols / 4 * 3, d_packed, out_row_bytes, d_scales, cols / 32,
                                             padded_cols / 32, scale_layout);
        e = cudaGetLastError();
        if (e == cudaSuccess) note_launch();
    }
    if (e != cudaSuccess) {
        std::fprintf(stderr, "[mxfp6] quantize_device launch failed: %s\n", cudaGetErrorString(e));
        return MXFP6_ERR_CUDA;
    }
    note_launch();
    return MXFP6_OK;
}

extern "C" int mxfp6_quantize_device_typed(const void* d_mat, int in_type, int rows, int cols, long long ld,
                                           int padded_cols, uint8_t* d_packed, uint8_t* d_scales, int scale_layout,
                                           void* stream) {
    using namespace mxfp6;
    if (in_type < MXFP6_OUT_F32 || in_type > MXFP6_OUT_BF16) {
        std::fprintf(stderr, "[mxfp6] quantize_device_typed: invalid input type %d\n", in_type);
        return MXFP6_ERR_INVALID_OUT_TYPE;
    }
    if (rows < 0 || cols <= 0 || cols % 32 || padded_cols < cols || padded_cols % 32 ||
        (scale_layout != 0 && scale_layout != 1) || (scale_layout == 1 && padded_cols % 128)) {
        std::fprintf(stderr, "[mxfp6] quantize_device_typed: invalid arguments (%d x %d padded to %d, layout %d)\n", rows,
                     cols, padded_cols, scale_layout);
        return MXFP6_ERR_INVALID_SHAPE;
    }
    if (rows == 0) return MXFP6_OK;
    if (!d_mat || !d_packed || !d_scales) {
        std::fprintf(stderr, "[mxfp6] quantize_device_typed: null device pointer\n");
        return MXFP6_ERR_NULL_POINTER;
    }
    if (ld < cols) {
        std::fprintf(stderr, "[mxfp6] quantize_device_typed: row stride %lld is below cols = %d\n", ld, cols);
        return MXFP6_ERR_INVALID_STRIDE;
    }
    const uintptr_t esize = in_type == MXFP6_OUT_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(d_mat) & (esize - 1)) || (reinterpret_cast<uintptr_t>(d_packed) & 3)) {
        std::fprintf(stderr, "[mxfp6] quantize_device_typed: input must be aligned to its element, output to 4 bytes\n");
        return MXFP6_ERR_MISALIGNED;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e =
        in_type == MXFP6_OUT_F32
            ? launch_quantize_rows(static_cast<const float*>(d_mat), rows, cols, ld, padded_cols, d_packed, d_scales,
                                   scale_layout, st)
        : in_type == MXFP6_OUT_F16
            ? launch_quantize_rows(static_cast<const __half*>(d_mat), rows, cols, ld, padded_cols, d_packed, d_scales,
                                   scale_layout, st)
            : launch_quantize_rows(static_cast<const __nv_bfloat16*>(d_mat), rows, cols, ld, padded_cols, d_packed,
                                   d_scales, scale_layout, st);
    if (e != cudaSuccess) {
        cudaGetLastError();
        std::fprintf(stderr, "[mxfp6] quantize_device_typed launch failed: %s\n", cudaGetErrorString(e));
        return MXFP6_ERR_CUDA;
    }
    note_launch();
    return MXFP6_OK;
}

extern "C" int mxfp6_quantize_device(const float* d_mat, int rows, int cols, uint8_t* d_packed, uint8_t* d_scales,
                                     int scale_layout, void* stream) {
    return mxfp6_quantize_device_padded(d_mat, rows, cols, cols, d_packed, d_scales, scale_layout, stream);
}

extern "C" int mxfp6_repad_rows_device(const void* d_src, int rows, int src_row_bytes, int bytes_used, void* d_dst,
                                       int dst_row_bytes, void* stream) {
    using namespace mxfp6;
    if (!d_src || !d_dst || rows <= 0 || bytes_used <= 0 || bytes_used > src_row_bytes ||
        bytes_used > dst_row_bytes) {
        std::fprintf(stderr, "[mxfp6] repad_rows_device: invalid arguments\n");
        return MXFP6_ERR_INVALID_STRIDE;
    }
    const cudaError_t le = launch_repad(static_cast<const uint8_t*>(d_src), rows, src_row_bytes, bytes_used,
                                        static_cast<uint8_t*>(d_dst), dst_row_bytes,
                                        static_cast<cudaStream_t>(stream));
    cudaError_t e = le;
    if (e != cudaSuccess) {
        std::fprintf(stderr, "[mxfp6] repad_rows_device launch failed: %s\n", cudaGetErrorString(e));
        return MXFP6_ERR_CUDA;
    }
    note_launch();
    return MXFP6_OK;
}
