#pragma once
// Device pieces of MXFP6 quantisation shared by the quantisers (quantize.cu) and the kernels that
// write MXFP6 themselves (epilogue.cuh, moe.cu). Per 32 values: scale = smallest power of two
// >= max|x| / 7.5 (E8M0 code, 127 for a block of zeros, NaN ignored by the max), codes = nearest
// E2M3 of x / scale, packed four codes per three bytes, least significant bits first.
#include <cstdint>

namespace mxfp6 {

// Two floats in one 64-bit register: multiply, add and multiply-add take one instruction for both.
struct F2 {
    unsigned long long w;
};
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1,%2};" : "=l"(r.w) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 both(float a) { return pair(a, a); }
__device__ __forceinline__ void split(F2 x, float& a, float& b) { asm("mov.b64 {%0,%1}, %2;" : "=f"(a), "=f"(b) : "l"(x.w)); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
    return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
    return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w));
    return r;
}
// E8M0 code of the smallest power of two >= v (v > 0, finite or +Inf): from the float bits,
// the same result as frexp-based rounding up (a power of two maps to itself).
__device__ __forceinline__ uint32_t ceil_pow2_code(float v) {
    const uint32_t b = __float_as_uint(v);
    if (b >= 0x7F800000u) return 127;  // +Inf: the reference's frexp reports exponent 0
    int e;                              // v = m * 2^e with m in [1, 2)
    uint32_t man;
    if (b >= 0x00800000u) {
        e = (int)(b >> 23) - 127;
        man = b & 0x7FFFFFu;
    } else {  // subnormal: normalise the mantissa
        const int lz = __clz(b) - 8;    // leading zeros within the 24-bit significand field
        e = -126 - lz;
        man = (b << lz) & 0x7FFFFFu;
    }
    const int code = e + (man != 0 ? 1 : 0) + 127;
    return (uint32_t)(code < 0 ? 0 : (code > 254 ? 254 : code));
}

// E8M0 code of the reference's block scale for block max m >= 0: the smallest power of two
// >= RN(m / 7.5), 127 for m == 0. For P = 2^e >= 2^-125, RN(m / 7.5) <= P exactly when
// m <= 7.5 * P (the rounding boundary P + ulp(P)/2 lies below the next float above 7.5 * P), so
// with m = 1.f * 2^E the code is E - 2, plus 1 when the mantissa exceeds 1.875, plus the bias.
// Subnormal quotients, an infinite max and m == 0 take the division.
__device__ __forceinline__ uint32_t scale_code(float m) {
    const uint32_t mb = __float_as_uint(m);
    const int e = (int)(mb >> 23) - 129 + ((mb & 0x7FFFFFu) > 0x700000u ? 1 : 0);
    if (mb < 0x7F800000u && (mb >> 23) != 0u && e >= -125) return (uint32_t)(e + 127);
    return m == 0.0f ? 127u : ceil_pow2_code(__fdiv_rn(m, 7.5f));
}

// Nearest E2M3 codes of two values (round to nearest even, saturating at 7.5) with the
// hardware conversion cvt.rn.satfinite.e2m3x2.f32, which writes a's code to the upper byte and
// b's to the lower one. Two inputs are first replaced so that the codes equal the reference's
// conversion (include/mxfp6/types.hpp:26-72): NaN -> 4.0 (code 0x18, what the reference yields on
// x86-64) and -0.0 -> +0.0 (code 0; other negatives that round to zero keep the sign, 0x20).
// Returns code(b) | code(a) << 8.
__device__ __forceinline__ uint32_t to_e2m3x2(float a, float b) {
    a = a != a ? 4.0f : __fadd_rn(a, 0.0f);  // never joined with the multiplication before it (quantize16)
    b = b != b ? 4.0f : __fadd_rn(b, 0.0f);
    uint16_t d;
    asm("cvt.rn.satfinite.e2m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(a), "f"(b));
    return d;
}

// 1 / 2^(code - 127) = 2^(127 - code), exact for every code the quantiser produces (0..254):
// multiplying by it rounds exactly like dividing by the scale.
__device__ __forceinline__ float e8m0_reciprocal(uint32_t code) {
    const int e = 254 - (int)code;  // biased exponent of 2^(127 - code)
    return e > 0 ? __int_as_float(e << 23) : __int_as_float(0x00400000 >> (-e));
}

// Largest magnitude of 16 values, NaN ignored; `nan` tells whether there is one.
__device__ __forceinline__ float max_abs16(const float* v, bool& nan) {
    float m = 0.0f;  // the NaN-propagating maximum needs no second pass unless there is a NaN
#pragma unroll
    for (int i = 0; i < 16; i++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[i])));
    nan = m != m;
    if (nan) {
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) m = fmaxf(m, fabsf(v[i]));
    }
    return m;
}

// 16 values times `inv`, as 16 codes in three words (bits 6k of 96). Adding +0 to the rounded product makes a -0 product
// +0 (to_e2m3x2's other replacement, NaN, is only made where max_abs16 saw one). The multiply-add alone would not: a
// negative product too small for FP32, as of -1e-30 beside 1e24, is not zero before its rounding, which then gives -0. The
// product is a multiply-add because a packed multiplication and the packed addition after it were joined into one: the
// bytes showed it. Four codes in four bytes become 24 bits with two byte dot products (weights 1 and 64) and a multiply-add.
__device__ __forceinline__ void quantize16(const float* v, float inv, bool nan, uint32_t& w0, uint32_t& w1,
                                           uint32_t& w2) {
    uint32_t q[8], g[4];  // q[i] = code(v[2i]) | code(v[2i + 1]) << 8
    if (nan) {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = to_e2m3x2(v[2 * i + 1] * inv, v[2 * i] * inv);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint16_t d;
            float lo, hi;
            split(fma(pair(v[2 * i], v[2 * i + 1]), both(inv), both(0.0f)) + both(0.0f), lo, hi);
            asm("cvt.rn.satfinite.e2m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
            q[i] = d;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t c = __byte_perm(q[2 * i], q[2 * i + 1], 0x5410) & 0x3F3F3F3Fu;
        g[i] = __dp4a(c, 0x00004001u, 0u) + (__dp4a(c, 0x40010000u, 0u) << 12);
    }
    w0 = g[0] | (g[1] << 24);
    w1 = (g[1] >> 8) | (g[2] << 16);
    w2 = (g[2] >> 16) | (g[3] << 8);
}

// Byte offset of the scale of (row, 32-column block j) in the GEMM's atoms of 128 rows x 4 blocks;
// k_atoms = columns / 128.
__device__ __forceinline__ size_t scale_atom_offset(int row, int j, int k_atoms) {
    const size_t atom = (size_t)(row / 128) * (size_t)k_atoms + (size_t)(j / 4);
    return atom * 512 + (size_t)((row % 32) * 16 + ((row % 128) / 32) * 4 + (j % 4));
}

}  // namespace mxfp6
