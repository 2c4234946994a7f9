// Quantisation to 4 bits and back, of dense matrices and of the blocks of a block-sparse matrix.
//
// Mathematics.  A group is divided by its scale s and every quotient rounded to the nearest e2m1 value, ties to even:
//   SMAT_FP4_MX  s = 2^e, e = floor(log2 gmax) - 2: the division is exact
//   SMAT_FP4_NV  s = e4m3(gmax / 6 / p) * p with p the least power of two >= amax(row) / 2688 (2688 = 6 * 448, so e4m3 does not
//                overflow): s has four significant bits, the scale and the products of codes and scales are exact in 16 bits.
// The codes are those of exact arithmetic: quotients that an fp32 division would round onto a tie are moved off it again.
// A group that holds a NaN or an infinity gets the scale NaN and codes 0; row maxima are taken over finite values.
//
// What bounds it: HBM and some seven instructions a value, of which neither is full (issue slots 53 %, HBM 38 % for 2048 x 14336): a row
// is loaded, waited for, and converted once its maximum is known.  (Half a group a lane, which lays loads side by side as the way back
// does with its stores, has each scale worked out twice: 125 us instead of 75.)  Prompt of 4096 x 28672 bf16: 75 us, 0.61 of HBM's rate; back 50,
// 0.92.  Blocks of the layer 8192 x 28672 at 20 %: 30 and 24 us.  A row of a dense matrix stays in the registers of its CTA between the maximum
// and the codes (up to 128 values a thread; longer ones are read again, from L2); so do not the blocks of a block-row, whose second
// reading comes out of L2.  Loads are issued several groups at a time.
#include <algorithm>
#include <type_traits>

#include "fp4_device.cuh"

namespace smat {
namespace {

constexpr int kThreads = 256;

// Least power of two p >= amax / 2688 with exponent >= -100; 1 for 0.  amax = f * 2^e with f in [1, 2); 2688 = 1.3125 * 2^11.
__device__ __forceinline__ float pow2_of_row(float amax) {
    if (amax == 0.f) return 1.f;
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7fffffu) > 0x280000u ? 1 : 0);  // subnormal amax ends at the bound below
    return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// x / d for a later rounding to a few bits, y = RN(1 / d).  One corrective step makes the quotient the correctly rounded one (Markstein
// 1990: q1 = RN(q0 + (x - q0 d) y)).  That may be a tie of the coarse rounding although x / d is not: then it is moved to the neighbour
// on the side of x / d.  EXACT16: x has at most 11 significant bits, and d and the ties so few that a quotient that is no tie is at
// least 2^-13 of itself away from one; the correctly rounded one is on its side then.
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
// The same for a code of a value with at most 11 significant bits, in two instructions: the quotient rounded to a multiple of 2^-16.  It
// is below 9 in size (6 times 1 + 2^-4 where the scale is a normal e4m3, 6 times 1.5 where it is the least subnormal), so that the sum
// with 192 stays in [128, 256), whose step is 2^-16.  x y is within 2^-20 of it; ties are multiples of 1/4, and what is no tie is at
// least 2^-13 away from one.
__device__ __forceinline__ float divide_for_code(float x, float y) { return fmaf(x, y, 192.f) - 192.f; }

// Scale byte of a group with largest magnitude gmax (bad: it holds a NaN or an infinity); values are divided by d, whose correctly
// rounded reciprocal is y.  p: the row's power of two.
template <int FMT, bool EXACT16>
__device__ __forceinline__ uint32_t group_scale(float gmax, bool bad, float p, float inv_p, float& d, float& y) {
    if constexpr (FMT == SMAT_FP4_NV) {
        const float g = divide_for_rounding<EXACT16>(gmax * inv_p, 6.f, 1.f / 6.f);
        uint16_t c;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(0.f), "f"(g));
        const float s = scale_e4m3(c & 0x7fu);
        d = s * p;  // exact: four bits, and powers of two that stay inside the normal numbers (2^-9 2^-100 to 2^9 2^117)
        y = __frcp_rn(s) * inv_p;
        return bad ? 0x7fu : c & 0x7fu;
    } else {
        const int e = max((int)(__float_as_uint(gmax) >> 23) - 127 - 2, -127);  // of a subnormal gmax: the bound
        d = 1.f;
        y = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e; e is -127 to 125
        return bad ? 0xffu : (uint32_t)(e + 127);
    }
}

// 16 values with the largest magnitude of their group -> 8 bytes of codes and the scale byte.
template <int FMT, int DT>
__device__ __forceinline__ uint2 quantize16(const Raw<DT>& raw, float gmax, bool bad, float p, float inv_p, uint32_t& scale) {
    float d, y, q[16];
    scale = group_scale<FMT, DT != SMAT_F32>(gmax, bad, p, inv_p, d, y);
    if (bad || d == 0.f) return make_uint2(0, 0);
    raw.unpack(q);
#pragma unroll
    for (int i = 0; i < 16; i++)
        q[i] = FMT == SMAT_FP4_MX ? q[i] * y : DT == SMAT_F32 ? divide_for_rounding<false>(q[i], d, y) : divide_for_code(q[i], y);
    return make_uint2(f32x8_to_e2m1(q), f32x8_to_e2m1(q + 8));
}
// Eight codes to values: half a group a lane, so that a warp's 16-byte stores lie side by side (a group a lane, each store filled half
// of 32 sectors: 72 us instead of 50 for 4096 x 28672 bf16).  Code times scale is exact; the row scale p, which may be any number, comes
// last, so that fp32 rounds once and nothing overflows or ends at zero on the way.
template <int FMT, int DT>
__device__ __forceinline__ void dequantize8(uint32_t c, float s, float p, typename Elem<DT>::T* to) {
    uint32_t h[4];
    e2m1x8_to_f16(c, h);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
        v[2 * i] = f.x * s; v[2 * i + 1] = f.y * s;
        if constexpr (FMT == SMAT_FP4_NV) { v[2 * i] *= p; v[2 * i + 1] *= p; }
    }
    if constexpr (DT == SMAT_F32) {
        reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
    }
}

// ---- dense ----------------------------------------------------------------------------------------------------------------------
// Codes and scale of group j of row r; lanes j & 3 of a warp hold the groups of 64 columns and write their scales together.
template <int FMT, int DT>
__device__ __forceinline__ void quantize_group(const Raw<DT>& raw, size_t r, int j, bool in, int quads, float p, float inv_p, uint8_t* codes, uint8_t* scales) {
    bool bad;
    float g = raw.amax(bad);
    if constexpr (FMT == SMAT_FP4_MX) {
        g = fmaxf(g, __shfl_xor_sync(~0u, g, 1));
        bad = __shfl_xor_sync(~0u, bad ? 1 : 0, 1) || bad;
    }
    uint32_t s;
    const uint2 c = quantize16<FMT, DT>(raw, g, bad, p, inv_p, s);
    if (!in) s = 0;
    uint32_t word = FMT == SMAT_FP4_NV ? s << (j & 3) * 8 : j & 1 ? 0 : s << (j & 3) * 4;
    word |= __shfl_xor_sync(~0u, word, 1);
    word |= __shfl_xor_sync(~0u, word, 2);
    if (j >= quads * 4) return;
    *reinterpret_cast<uint2*>(codes + r * quads * 32 + (size_t)j * 8) = c;
    if ((j & 3) == 0) *reinterpret_cast<uint32_t*>(scales + dense_scale_at<SMAT_FP4_NV>(r, (size_t)j * 16, quads)) = word;
}

// A CTA a row; G groups of 16 a thread in registers, or 0: the row is read twice.
template <int FMT, int DT, int G>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const typename Elem<DT>::T* __restrict__ X, int K, size_t ldx,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                float* __restrict__ row_scale) {
    const size_t r = blockIdx.x;
    const int quads = (K + 63) / 64, threads = blockDim.x;
    const auto* x = X + r * ldx;
    Raw<DT> raw[G ? G : 1];
    float p = 1.f, inv_p = 1.f;
    if constexpr (G > 0) {
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int j = (int)threadIdx.x + i * threads;
            if (j * 16 < K) raw[i].load(x + (size_t)j * 16);
            else raw[i].zero();
        }
    }
    if constexpr (FMT == SMAT_FP4_NV) {
        __shared__ float s_max[kThreads / 32];
        float m = 0.f;
        bool bad;
        if constexpr (G > 0) {
#pragma unroll
            for (int i = 0; i < G; i++) m = fmaxf(m, raw[i].amax(bad));
        } else {
            for (int j = threadIdx.x; j * 16 < K; j += threads) {
                raw[0].load(x + (size_t)j * 16);
                m = fmaxf(m, raw[0].amax(bad));
            }
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (threadIdx.x % 32 == 0) s_max[threadIdx.x / 32] = m;
        __syncthreads();
        m = s_max[0];
        for (int w = 1; w < threads / 32; w++) m = fmaxf(m, s_max[w]);
        p = pow2_of_row(m);
        inv_p = 1.f / p;
        if (threadIdx.x == 0) row_scale[r] = p;
    }
    if constexpr (G > 0) {
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int j = (int)threadIdx.x + i * threads;
            quantize_group<FMT, DT>(raw[i], r, j, j * 16 < K, quads, p, inv_p, codes, scales);
        }
    } else {
        for (int j = threadIdx.x; j - (int)threadIdx.x < quads * 4; j += threads) {  // whole warps: lanes exchange
            if (j * 16 < K) raw[0].load(x + (size_t)j * 16);
            else raw[0].zero();
            quantize_group<FMT, DT>(raw[0], r, j, j * 16 < K, quads, p, inv_p, codes, scales);
        }
    }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                  const float* __restrict__ row_scale, int K,
                                                                  typename Elem<DT>::T* __restrict__ Y, size_t ldy) {
    constexpr int U = 8;
    const size_t r = blockIdx.x;
    const int quads = (K + 63) / 64, halves = K / 8, threads = blockDim.x;
    const float p = row_scale ? __ldg(row_scale + r) : 1.f;
    for (int j0 = threadIdx.x; j0 < halves; j0 += U * threads) {
        uint32_t c[U], s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = min(j0 + u * threads, halves - 1);
            c[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + r * quads * 32) + j);
            s[u] = __ldg(scales + dense_scale_at<FMT>(r, (size_t)j * 8, quads));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = j0 + u * threads;
            if (j < halves) dequantize8<FMT, DT>(c[u], scale_value<FMT>(s[u]), p, Y + r * ldy + (size_t)j * 8);
        }
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
    constexpr int U = DT == SMAT_F32 ? 2 : 4, STEP = kThreads / 16;  // blocks a thread has on their way, blocks of the CTA at a time
    const int2 range = blocks_of_row(rowptr, blockIdx.x, nnzb, status);
    const int i = threadIdx.x % 16;
    Raw<DT> raw[U];
    bool bad;
    float p = 1.f, inv_p = 1.f;
    if constexpr (FMT == SMAT_FP4_NV) {
        __shared__ unsigned s_max[16];  // magnitudes of floats compare like their bits
        if (threadIdx.x < 16) s_max[threadIdx.x] = 0;
        __syncthreads();
        float m = 0.f;
        for (int b0 = range.x + threadIdx.x / 16; b0 < range.y; b0 += U * STEP) {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u].load(vals + (size_t)min(b0 + u * STEP, range.y - 1) * 256 + i * 16);
#pragma unroll
            for (int u = 0; u < U; u++) m = fmaxf(m, raw[u].amax(bad));
        }
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
        if (threadIdx.x % 32 < 16) atomicMax(&s_max[i], __float_as_uint(m));
        __syncthreads();
        p = pow2_of_row(__uint_as_float(s_max[i]));
        inv_p = 1.f / p;
        if (threadIdx.x < 16) row_scale[(size_t)blockIdx.x * 16 + i] = p;
    }
    for (int b0 = range.x + threadIdx.x / 16; b0 < range.y; b0 += U * STEP) {
        Raw<DT> pair[FMT == SMAT_FP4_MX ? U : 1];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = min(b0 + u * STEP, range.y - 1);
            raw[u].load(vals + (size_t)b * 256 + i * 16);
            if constexpr (FMT == SMAT_FP4_MX) {
                const int col = __ldg(colidx + b), other = col & 16 ? b - 1 : b + 1;  // where the other block of the pair would be
                if (other >= range.x && other < range.y && __ldg(colidx + other) == (col ^ 16)) pair[u].load(vals + (size_t)other * 256 + i * 16);
                else pair[u].zero();
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = b0 + u * STEP;
            if (b >= range.y) break;
            float g = raw[u].amax(bad);
            if constexpr (FMT == SMAT_FP4_MX) {
                bool bad2;
                g = fmaxf(g, pair[u].amax(bad2));
                bad |= bad2;
            }
            uint32_t s;
            const uint2 c = quantize16<FMT, DT>(raw[u], g, bad, p, inv_p, s);
            *reinterpret_cast<uint2*>(codes + (size_t)b * 128 + i * 8) = c;
            scales[(size_t)b * 16 + i] = s;
        }
    }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_blocks_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                         const float* __restrict__ row_scale, const int* __restrict__ rowptr,
                                                                         size_t nnzb, typename Elem<DT>::T* __restrict__ vals, int* status) {
    // A warp a block, half a row of it a lane.
    constexpr int U = 8, STEP = kThreads / 32;
    const int2 range = blocks_of_row(rowptr, blockIdx.x, nnzb, status);
    const int lane = threadIdx.x % 32;
    const float p = row_scale ? __ldg(row_scale + (size_t)blockIdx.x * 16 + lane / 2) : 1.f;
    for (int b0 = range.x + threadIdx.x / 32; b0 < range.y; b0 += U * STEP) {
        uint32_t c[U], s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = min(b0 + u * STEP, range.y - 1);
            c[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + (size_t)b * 128) + lane);
            s[u] = __ldg(scales + (size_t)b * 16 + lane / 2);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = b0 + u * STEP;
            if (b < range.y) dequantize8<FMT, DT>(c[u], scale_value<FMT>(s[u]), p, vals + (size_t)b * 256 + lane * 8);
        }
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
    if (N >= ((size_t)1 << 31) || K >= ((size_t)1 << 30)) return fail(SMAT_ERR_RANGE, "N beyond 2^31 - 1 or K beyond 2^30 - 1");
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
        const int groups = (int)fp4_quads(K) * 4, threads = std::max(32, std::min(kThreads, (groups + 31) / 32 * 32));
        const auto* x = static_cast<const typename Elem<D>::T*>(X);
        auto *c = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
        auto launch = [&](auto kernel) { kernel<<<(unsigned)N, threads, 0, (cudaStream_t)stream>>>(x, (int)K, ldx, c, s, row_scale); };
        const int per = (groups + threads - 1) / threads;
        if (per <= 1) launch(fp4_quantize_kernel<F, D, 1>);
        else if (per <= 2) launch(fp4_quantize_kernel<F, D, 2>);
        else if (per <= 4) launch(fp4_quantize_kernel<F, D, 4>);
        else if (per <= 8 && D != SMAT_F32) launch(fp4_quantize_kernel<F, D, D == SMAT_F32 ? 4 : 8>);
        else launch(fp4_quantize_kernel<F, D, 0>);
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
        const int threads = std::max(32, std::min(kThreads, ((int)K / 8 + 31) / 32 * 32));
        fp4_dequantize_kernel<F, D><<<(unsigned)N, threads, 0, (cudaStream_t)stream>>>(
            static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), row_scale, (int)K, static_cast<typename Elem<D>::T*>(Y), ldy);
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
        fp4_quantize_blocks_kernel<F, D><<<(unsigned)(M / 16), kThreads, 0, (cudaStream_t)stream>>>(static_cast<const typename Elem<D>::T*>(vals), rowptr, colidx, nnzb, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
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
        fp4_dequantize_blocks_kernel<F, D><<<(unsigned)(M / 16), kThreads, 0, (cudaStream_t)stream>>>(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), row_scale, rowptr, nnzb,
            static_cast<typename Elem<D>::T*>(vals), ctx->d_status);
        return cudaGetLastError();
    }));
    count_launch();
    return SMAT_OK;
}

}  // extern "C"
