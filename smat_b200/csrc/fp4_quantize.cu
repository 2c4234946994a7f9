// Quantisation to 4 bits and back, of dense matrices and of the blocks of a block-sparse matrix.
//
// Mathematics.  A group is divided by its scale s and every quotient rounded to the nearest e2m1 value, ties to even:
//   SMAT_FP4_MX  s = 2^e, e = floor(log2 gmax) - 2: the division is exact
//   SMAT_FP4_NV  s = e4m3(gmax / 6 / p) * p with p the least power of two >= amax(row) / 2688 (2688 = 6 * 448, so e4m3 does not
//                overflow): s has four significant bits, the scale and the products of codes and scales are exact in 16 bits.
// The codes are those of exact arithmetic: quotients that an fp32 division would round onto a tie are moved off it again.
// A group that holds a NaN or an infinity gets the scale NaN and codes 0; row maxima are taken over finite values.
//
// What bounds it: HBM.  The row maximum is taken by the CTA that quantises the row right after it: the second reading comes out of
// L2 (or L1), so a value crosses HBM once and no launch waits for another.
#include "fp4_device.cuh"

namespace smat {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Least power of two p >= amax / 2688 with exponent >= -100; 1 for 0.  amax = f * 2^e with f in [1, 2); 2688 = 1.3125 * 2^11.
__device__ __forceinline__ float pow2_of_row(float amax) {
    if (amax == 0.f) return 1.f;
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7fffffu) > 0x280000u ? 1 : 0);  // subnormal amax ends at the bound below
    return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// x / d for a later rounding to a few bits.  q = RN(x / d) by a reciprocal and one corrective step (Markstein 1990: with the
// correctly rounded reciprocal, q1 = RN(q0 + (x - q0 d) y) is the correctly rounded quotient).  That q may be a tie of the coarse
// rounding although x / d is not: then it is moved to the neighbour on the side of x / d.  EXACT16: x has at most 11 significant
// bits and d four, so a quotient that is no tie is at least 2^-13 away from one and q is already on its side.
template <bool EXACT16>
__device__ __forceinline__ float divide_for_rounding(float x, float d, float y) {
    float q = x * y;
    q = fmaf(fmaf(-q, d, x), y, q);
    if (!EXACT16) {
        const float r = fmaf(-q, d, x);
        if (r != 0.f && (__float_as_uint(q) & 0x3ffffu) == 0 && q != 0.f)
            q = __uint_as_float(__float_as_uint(q) + ((r > 0.f) == (q > 0.f) ? 1 : -1));
    }
    return q;
}

// Scale byte of a group with largest magnitude gmax (bad: it holds a NaN or an infinity), and what its values are divided by.
// The quotients are formed from values times `up`, a power of two that keeps them and the divisor inside the normal numbers.
template <int FMT>
__device__ __forceinline__ uint32_t group_scale(float gmax, bool bad, float inv_p, float& d, float& up) {
    if constexpr (FMT == SMAT_FP4_NV) {
        up = inv_p;
        const float g = divide_for_rounding<false>(gmax * inv_p, 6.f, 1.f / 6.f);
        uint16_t c;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(0.f), "f"(g));
        d = scale_e4m3(c & 0x7fu);
        return bad ? 0x7fu : c & 0x7fu;
    } else {
        const int e = max((int)(__float_as_uint(gmax) >> 23) - 127 - 2, -127);  // of a subnormal gmax: the bound
        up = __uint_as_float((uint32_t)min(127 - e, 254) << 23);  // 2^-e; e <= 125
        d = 1.f;
        return bad ? 0xffu : (uint32_t)(e + 127);
    }
}

// 16 values with the largest magnitude of their group -> 8 bytes of codes and the scale byte.
template <int FMT, int DT>
__device__ __forceinline__ uint2 quantize16(const float (&v)[16], float gmax, bool bad, float inv_p, uint32_t& scale) {
    float d, up;
    scale = group_scale<FMT>(gmax, bad, inv_p, d, up);
    if (bad || d == 0.f) return make_uint2(0, 0);
    float q[16];
    if constexpr (FMT == SMAT_FP4_NV) {
        const float y = __frcp_rn(d);
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] = divide_for_rounding<DT != SMAT_F32>(v[i] * up, d, y);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] = v[i] * up;
    }
    return make_uint2(f32x8_to_e2m1(q), f32x8_to_e2m1(q + 8));
}

// Largest magnitude among the finite values; bad: there are others.
__device__ __forceinline__ float amax16(const float (&v)[16], bool& bad) {
    float m = 0.f;
    bad = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const bool f = finite_bits(v[i]);
        bad |= !f;
        m = fmaxf(m, f ? fabsf(v[i]) : 0.f);
    }
    return m;
}

// ---- dense ----------------------------------------------------------------------------------------------------------------------
template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const typename Elem<DT>::T* __restrict__ X, size_t N, size_t K, size_t ldx,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                float* __restrict__ row_scale) {
    const size_t r = blockIdx.x, quads = (K + 63) / 64;
    const auto* x = X + r * ldx;
    float v[16];
    bool bad;
    __shared__ float s_max[kThreads / 32];
    float inv_p = 1.f;
    if constexpr (FMT == SMAT_FP4_NV) {
        float m = 0.f;
        for (size_t j = threadIdx.x; j * 16 < K; j += kThreads) {
            load16<DT>(x + j * 16, v);
            m = fmaxf(m, amax16(v, bad));
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (threadIdx.x % 32 == 0) s_max[threadIdx.x / 32] = m;
        __syncthreads();
        m = s_max[0];
        for (int w = 1; w < kThreads / 32; w++) m = fmaxf(m, s_max[w]);
        const float p = pow2_of_row(m);
        inv_p = 1.f / p;
        if (threadIdx.x == 0) row_scale[r] = p;
    }
    const size_t groups = quads * 4, up = (groups + kThreads - 1) / kThreads * kThreads;  // whole warps: lanes exchange below
    for (size_t j = threadIdx.x; j < up; j += kThreads) {
        const bool in = j * 16 < K;
        if (in) {
            load16<DT>(x + j * 16, v);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = 0.f;
        }
        float g = amax16(v, bad);
        if constexpr (FMT == SMAT_FP4_MX) {
            g = fmaxf(g, __shfl_xor_sync(~0u, g, 1));
            bad = __shfl_xor_sync(~0u, bad ? 1 : 0, 1) || bad;
        }
        if (j >= groups) continue;
        uint32_t s;
        const uint2 c = quantize16<FMT, DT>(v, g, bad, inv_p, s);
        *reinterpret_cast<uint2*>(codes + r * quads * 32 + j * 8) = c;
        const size_t at = dense_scale_at<SMAT_FP4_NV>(r, j * 16, quads);
        if constexpr (FMT == SMAT_FP4_NV) scales[at] = in ? s : 0;
        else scales[at - (j & 3) + ((j & 1) ? 2 : 0) + ((j & 3) >> 1)] = (j & 1) || !in ? 0 : s;
    }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                  const float* __restrict__ row_scale, size_t K,
                                                                  typename Elem<DT>::T* __restrict__ Y, size_t ldy) {
    const size_t r = blockIdx.x, quads = (K + 63) / 64;
    const float p = row_scale ? __ldg(row_scale + r) : 1.f;
    for (size_t j = threadIdx.x; j * 16 < K; j += kThreads) {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + r * quads * 32) + j);
        const float s = scale_value<FMT>(__ldg(scales + dense_scale_at<FMT>(r, j * 16, quads))) * p;
        uint32_t h[2][4];
        e2m1x8_to_f16(c.x, h[0]);
        e2m1x8_to_f16(c.y, h[1]);
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i / 4][i % 4]));
            v[2 * i] = f.x * s; v[2 * i + 1] = f.y * s;
        }
        store16<DT>(Y + r * ldy + j * 16, v);
    }
}

// ---- blocks ---------------------------------------------------------------------------------------------------------------------
// The blocks of block-row r, or none where the row pointers are inconsistent (which is reported).
__device__ __forceinline__ int2 blocks_of_row(const int* rowptr, size_t r, size_t nnzb, int* status) {
    int lo = __ldg(rowptr + r), hi = __ldg(rowptr + r + 1);
    if (lo < 0 || hi < lo || (size_t)hi > nnzb) {
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusBadRowptr);
        lo = hi = 0;
    }
    return make_int2(lo, hi);
}

// A CTA takes a block-row, a thread a row of a block.
template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_quantize_blocks_kernel(const typename Elem<DT>::T* __restrict__ vals,
                                                                       const int* __restrict__ rowptr, const int* __restrict__ colidx,
                                                                       size_t nnzb, uint8_t* __restrict__ codes,
                                                                       uint8_t* __restrict__ scales, float* __restrict__ row_scale,
                                                                       int* status) {
    const int2 range = blocks_of_row(rowptr, blockIdx.x, nnzb, status);
    const int i = threadIdx.x % 16;
    float v[16];
    bool bad;
    float inv_p = 1.f;
    if constexpr (FMT == SMAT_FP4_NV) {
        __shared__ unsigned s_max[16];  // magnitudes of floats compare like their bits
        if (threadIdx.x < 16) s_max[threadIdx.x] = 0;
        __syncthreads();
        float m = 0.f;
        for (int b = range.x + threadIdx.x / 16; b < range.y; b += kThreads / 16) {
            load16<DT>(vals + (size_t)b * 256 + i * 16, v);
            m = fmaxf(m, amax16(v, bad));
        }
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
        if (threadIdx.x % 32 < 16) atomicMax(&s_max[i], __float_as_uint(m));
        __syncthreads();
        const float p = pow2_of_row(__uint_as_float(s_max[i]));
        inv_p = 1.f / p;
        if (threadIdx.x < 16) row_scale[(size_t)blockIdx.x * 16 + i] = p;
    }
    for (int b = range.x + threadIdx.x / 16; b < range.y; b += kThreads / 16) {
        load16<DT>(vals + (size_t)b * 256 + i * 16, v);
        float g = amax16(v, bad);
        if constexpr (FMT == SMAT_FP4_MX) {
            const int col = __ldg(colidx + b);
            const int other = col & 16 ? b - 1 : b + 1;  // where the other block of the pair would be
            if (other >= range.x && other < range.y && __ldg(colidx + other) == (col ^ 16)) {
                float w[16];
                bool bad2;
                load16<DT>(vals + (size_t)other * 256 + i * 16, w);
                g = fmaxf(g, amax16(w, bad2));
                bad |= bad2;
            }
        }
        uint32_t s;
        const uint2 c = quantize16<FMT, DT>(v, g, bad, inv_p, s);
        *reinterpret_cast<uint2*>(codes + (size_t)b * 128 + i * 8) = c;
        scales[(size_t)b * 16 + i] = s;
    }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_blocks_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                         const float* __restrict__ row_scale, const int* __restrict__ rowptr,
                                                                         size_t nnzb, typename Elem<DT>::T* __restrict__ vals, int* status) {
    const int2 range = blocks_of_row(rowptr, blockIdx.x, nnzb, status);
    const int i = threadIdx.x % 16;
    const float p = row_scale ? __ldg(row_scale + (size_t)blockIdx.x * 16 + i) : 1.f;
    for (int b = range.x + threadIdx.x / 16; b < range.y; b += kThreads / 16) {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + (size_t)b * 128) + i);
        const float s = scale_value<FMT>(__ldg(scales + (size_t)b * 16 + i)) * p;
        uint32_t h[2][4];
        e2m1x8_to_f16(c.x, h[0]);
        e2m1x8_to_f16(c.y, h[1]);
        float v[16];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[j / 4][j % 4]));
            v[2 * j] = f.x * s; v[2 * j + 1] = f.y * s;
        }
        store16<DT>(vals + (size_t)b * 256 + i * 16, v);
    }
}

// Calls f<FMT, DT>() for run-time values of both.
template <class F>
cudaError_t with_types(int fmt, int dtype, F f) {
    auto of = [&](auto fm) {
        if (dtype == SMAT_F16) return f(fm, std::integral_constant<int, SMAT_F16>());
        if (dtype == SMAT_BF16) return f(fm, std::integral_constant<int, SMAT_BF16>());
        return f(fm, std::integral_constant<int, SMAT_F32>());
    };
    return fmt == SMAT_FP4_NV ? of(std::integral_constant<int, SMAT_FP4_NV>()) : of(std::integral_constant<int, SMAT_FP4_MX>());
}

int check_types(int fmt, int dtype) {
    if (fmt != SMAT_FP4_NV && fmt != SMAT_FP4_MX) return fail(SMAT_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (dtype != SMAT_F16 && dtype != SMAT_BF16 && dtype != SMAT_F32) return fail(SMAT_ERR_BAD_ARG, "unknown element type %d", dtype);
    return SMAT_OK;
}
size_t size_of(int dtype) { return dtype == SMAT_F32 ? 4 : 2; }

int check_dense(const void* X, int dtype, size_t N, size_t K, size_t ld, int fmt, const void* codes, const void* scales) {
    if (int rc = check_types(fmt, dtype)) return rc;
    if (K % 16) return fail(SMAT_ERR_BAD_ARG, "K (%zu) must be a multiple of 16", K);
    if (N >= ((size_t)1 << 31) || K >= ((size_t)1 << 31)) return fail(SMAT_ERR_RANGE, "dimension beyond 2^31");
    if (N && K && (!X || !codes || !scales)) return fail(SMAT_ERR_BAD_ARG, "NULL argument");
    if (ld < K || ld * size_of(dtype) % 16) return fail(SMAT_ERR_BAD_ARG, "rows must be at least K elements and a multiple of 16 bytes apart");
    if (((uintptr_t)X | (uintptr_t)codes | (uintptr_t)scales) & 15) return fail(SMAT_ERR_BAD_ARG, "arrays must be 16-byte aligned");
    return SMAT_OK;
}
int check_blocks(const void* vals, int dtype, const int* rowptr, size_t M, size_t nnzb, int fmt, const void* codes, const void* scales) {
    if (int rc = check_types(fmt, dtype)) return rc;
    if (M % 16) return fail(SMAT_ERR_BAD_ARG, "M (%zu) must be a multiple of 16", M);
    if (M / 16 >= ((size_t)1 << 31) || nnzb * 16 >= ((size_t)1 << 31)) return fail(SMAT_ERR_RANGE, "size beyond the index range");
    if (!rowptr || (nnzb && (!vals || !codes || !scales))) return fail(SMAT_ERR_BAD_ARG, "NULL argument");
    if (((uintptr_t)vals | (uintptr_t)codes | (uintptr_t)scales) & 15) return fail(SMAT_ERR_BAD_ARG, "arrays must be 16-byte aligned");
    return SMAT_OK;
}

}  // namespace
}  // namespace smat

using namespace smat;

extern "C" {

size_t smat_fp4_codes_bytes(size_t N, size_t K) { return N * fp4_pitch(K); }
size_t smat_fp4_scales_bytes(size_t N, size_t K) { return (N + 127) / 128 * fp4_quads(K) * 512; }

int smat_fp4_quantize(const void* X, int dtype, size_t N, size_t K, size_t ldx, int fmt, void* codes, void* scales, float* row_scale,
                      void* stream) {
    clear_error();
    if (int rc = check_dense(X, dtype, N, K, ldx, fmt, codes, scales)) return rc;
    if (fmt == SMAT_FP4_NV && N && !row_scale) return fail(SMAT_ERR_BAD_ARG, "row_scale is NULL");
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    if (!N || (!K && fmt == SMAT_FP4_MX)) return SMAT_OK;
    SMAT_CUDA_TRY(with_types(fmt, dtype, [&](auto f, auto d) {
        constexpr int F = decltype(f)::value, D = decltype(d)::value;
        fp4_quantize_kernel<F, D><<<(unsigned)N, kThreads, 0, (cudaStream_t)stream>>>(
            static_cast<const typename Elem<D>::T*>(X), N, K, ldx, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), row_scale);
        return cudaGetLastError();
    }));
    count_launch();
    return SMAT_OK;
}

int smat_fp4_dequantize(const void* codes, const void* scales, const float* row_scale, int fmt, size_t N, size_t K, void* Y, int dtype,
                        size_t ldy, void* stream) {
    clear_error();
    if (int rc = check_dense(Y, dtype, N, K, ldy, fmt, codes, scales)) return rc;
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    if (!N || !K) return SMAT_OK;
    SMAT_CUDA_TRY(with_types(fmt, dtype, [&](auto f, auto d) {
        constexpr int F = decltype(f)::value, D = decltype(d)::value;
        fp4_dequantize_kernel<F, D><<<(unsigned)N, kThreads, 0, (cudaStream_t)stream>>>(
            static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), row_scale, K, static_cast<typename Elem<D>::T*>(Y), ldy);
        return cudaGetLastError();
    }));
    count_launch();
    return SMAT_OK;
}

int smat_fp4_quantize_blocks(const void* vals, int dtype, const int* rowptr, const int* colidx, size_t M, size_t nnzb, int fmt, void* codes,
                             void* scales, float* row_scale, void* stream) {
    clear_error();
    if (int rc = check_blocks(vals, dtype, rowptr, M, nnzb, fmt, codes, scales)) return rc;
    if (fmt == SMAT_FP4_NV && M && !row_scale) return fail(SMAT_ERR_BAD_ARG, "row_scale is NULL");
    if (nnzb && !colidx) return fail(SMAT_ERR_BAD_ARG, "bcsrColIdxA is NULL");
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    if (!M) return SMAT_OK;
    SMAT_CUDA_TRY(with_types(fmt, dtype, [&](auto f, auto d) {
        constexpr int F = decltype(f)::value, D = decltype(d)::value;
        fp4_quantize_blocks_kernel<F, D><<<(unsigned)(M / 16), kThreads, 0, (cudaStream_t)stream>>>(
            static_cast<const typename Elem<D>::T*>(vals), rowptr, colidx, nnzb, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
            row_scale, ctx->d_status);
        return cudaGetLastError();
    }));
    count_launch();
    return SMAT_OK;
}

int smat_fp4_dequantize_blocks(const void* codes, const void* scales, const float* row_scale, int fmt, const int* rowptr, size_t M,
                               size_t nnzb, void* vals, int dtype, void* stream) {
    clear_error();
    if (int rc = check_blocks(vals, dtype, rowptr, M, nnzb, fmt, codes, scales)) return rc;
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    if (!M) return SMAT_OK;
    SMAT_CUDA_TRY(with_types(fmt, dtype, [&](auto f, auto d) {
        constexpr int F = decltype(f)::value, D = decltype(d)::value;
        fp4_dequantize_blocks_kernel<F, D><<<(unsigned)(M / 16), kThreads, 0, (cudaStream_t)stream>>>(
            static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), row_scale, rowptr, nnzb,
            static_cast<typename Elem<D>::T*>(vals), ctx->d_status);
        return cudaGetLastError();
    }));
    count_launch();
    return SMAT_OK;
}

}  // extern "C"
