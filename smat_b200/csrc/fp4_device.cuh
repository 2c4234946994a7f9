// Conversions between e2m1, e4m3, e8m0 and wider types, shared by the kernels for matrices in 4 bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "fp4_format.h"

namespace smat {
namespace {

// ---- scales -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float scale_e4m3(uint32_t code) {
    uint32_t h2;
    const uint16_t c = (uint16_t)code;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(c));
    return __low2float(*reinterpret_cast<__half2*>(&h2));
}
// 2^(code - 127); 255: NaN.  Exponent bits of an fp32, but for code 0, which is below the normal numbers.
__device__ __forceinline__ float scale_e8m0(uint32_t code) {
    const uint32_t bits = code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23;
    return __uint_as_float(bits);
}
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t code) {
    return FMT == SMAT_FP4_NV ? scale_e4m3(code) : scale_e8m0(code);
}
// Byte offset of the scale of (row r, columns from k) in the scales of a dense matrix.
template <int FMT>
__device__ __forceinline__ size_t dense_scale_at(size_t r, size_t k, size_t quads) {
    return ((r >> 7) * quads + (k >> 6)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (FMT == SMAT_FP4_NV ? (k >> 4) & 3 : (k >> 5) & 1);
}

// ---- codes ------------------------------------------------------------------------------------------------------------------
// Eight codes -> four pairs of fp16, exact; pair i holds codes 2i (low) and 2i + 1.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// Four codes, the same.
__device__ __forceinline__ void e2m1x4_to_f16(uint16_t w, uint32_t& h0, uint32_t& h1) {
    asm("{\n\t.reg .b8 b0, b1;\n\tmov.b16 {b0, b1}, %2;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t}"
        : "=r"(h0), "=r"(h1) : "h"(w));
}
// Product of two pairs.
template <int DT>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    if constexpr (DT == SMAT_F16) {
        const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
// A pair of fp16 that came from e2m1 -> the same pair in bf16.  The magnitude shifted down by the three bits that the exponent field is
// wider reads as the value times 2^-112 (0 stays 0, all others are normal); the factor 2^112 (0x7780) takes that back, a smaller one
// gives the pair times a power of two.
__device__ __forceinline__ uint32_t f16_code_to_bf16(uint32_t h2, uint32_t factor = 0x77807780u) {
    return mul2<SMAT_BF16>((h2 & 0x80008000u) | ((h2 & 0x7fff7fffu) >> 3), factor);
}
// Eight fp32 -> eight codes, to nearest, ties to even, saturating at 6 (no NaN comes here).
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float* v) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}

// ---- 16-bit and fp32 values ---------------------------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<SMAT_F16> { using T = __half; };
template <> struct Elem<SMAT_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<SMAT_F32> { using T = float; };

// 16 consecutive values (16-byte aligned) as they lie in memory.
template <int DT>
struct Raw {
    uint4 v[DT == SMAT_F32 ? 4 : 2];
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p) {
#pragma unroll
        for (int i = 0; i < (DT == SMAT_F32 ? 4 : 2); i++) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (DT == SMAT_F32 ? 4 : 2); i++) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void unpack(float (&f)[16]) const {
#pragma unroll
        for (int i = 0; i < (DT == SMAT_F32 ? 4 : 2); i++) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (DT == SMAT_F32) {
                    f[4 * i + j] = __uint_as_float(w[j]);
                } else if constexpr (DT == SMAT_F16) {
                    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                    f[8 * i + 2 * j] = t.x; f[8 * i + 2 * j + 1] = t.y;
                } else {
                    f[8 * i + 2 * j] = __uint_as_float(w[j] << 16); f[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
        }
    }
    // Largest magnitude among the finite values; bad: there are others.  Magnitudes compare like their bits.
    __device__ __forceinline__ float amax(bool& bad) const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < (DT == SMAT_F32 ? 4 : 2); i++) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) m = DT == SMAT_F32 ? max(m, w[j] & 0x7fffffffu) : __vmaxu2(m, w[j] & 0x7fff7fffu);
        }
        if (DT != SMAT_F32) m = max(m & 0xffffu, m >> 16);
        bad = m >= (DT == SMAT_F32 ? 0x7f800000u : DT == SMAT_F16 ? 0x7c00u : 0x7f80u);
        if (bad) {
            float f[16], a = 0.f;
            unpack(f);
#pragma unroll
            for (int i = 0; i < 16; i++) a = fmaxf(a, (__float_as_uint(f[i]) & 0x7f800000u) != 0x7f800000u ? fabsf(f[i]) : 0.f);
            return a;
        }
        if constexpr (DT == SMAT_F32) return __uint_as_float(m);
        else if constexpr (DT == SMAT_F16) return __half2float(__ushort_as_half((unsigned short)m));
        else return __uint_as_float(m << 16);
    }
};
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == SMAT_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ void store_c(void* C, int dtype, size_t at, float v) {
    if (dtype == SMAT_F16) static_cast<__half*>(C)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
}

}  // namespace
}  // namespace smat
