// Plans for products of a block-sparse matrix in 4 bits (smat_fp4_plan_*).
#include <new>

#include "fp4_format.h"
#include "smat_internal.h"

struct smat_fp4_plan {
    smat::Fp4View v;
    int device = -1;
    void* buffer = nullptr;
};

namespace smat {
namespace {

constexpr int kThreads = 256;

// Looks a block-row's pointers and columns over (a CTA a block-row): they have to lie in the arrays and the matrix, the columns in
// ascending order.  An inconsistent block-row is left out (empty) and reported.  totals: blocks, longest block-row.
__global__ void __launch_bounds__(kThreads) fp4_ranges_kernel(const int* __restrict__ rowptr, const int* __restrict__ colidx, size_t K, size_t nnzb,
                                                              int2* __restrict__ range, unsigned long long* __restrict__ totals, int* status) {
    const size_t r = blockIdx.x;
    const int lo = __ldg(rowptr + r), hi = __ldg(rowptr + r + 1);
    int bad = lo < 0 || hi < lo || (size_t)hi > nnzb ? kStatusBadRowptr : 0;
    bool wrong = false;
    if (!bad) {
        for (long long p = (long long)lo + threadIdx.x; p < hi; p += kThreads) {
            const int c = __ldg(colidx + p);
            wrong |= c < 0 || (size_t)c + 16 > K || c % 16 || (p > lo && __ldg(colidx + p - 1) >= c);
        }
    }
    if (__syncthreads_or(wrong)) bad = kStatusBadColumns;
    if (threadIdx.x == 0) {
        if (bad) atomicCAS(status, 0, bad);
        range[r] = bad ? make_int2(0, 0) : make_int2(lo, hi);
        if (!bad) {
            atomicAdd(totals, (unsigned long long)(hi - lo));
            atomicMax(totals + 1, (unsigned long long)(hi - lo));
        }
    }
}

int check_product(const smat_fp4_plan* plan, const void* B, const void* C, int c_dtype, size_t N) {
    if (!plan) return fail(SMAT_ERR_BAD_ARG, "plan is NULL");
    if (N >= ((size_t)1 << 31)) return fail(SMAT_ERR_RANGE, "N beyond 2^31");
    if (c_dtype != SMAT_F16 && c_dtype != SMAT_BF16) return fail(SMAT_ERR_BAD_ARG, "C must be fp16 or bf16");
    if (plan->v.block_rows && N && (!C || (plan->v.K && !B))) return fail(SMAT_ERR_BAD_ARG, "B or C is NULL");
    if (((uintptr_t)B | (uintptr_t)C) & 15) return fail(SMAT_ERR_BAD_ARG, "B and C must be 16-byte aligned");
    int dev = -1;
    SMAT_CUDA_TRY(cudaGetDevice(&dev));
    if (dev != plan->device) return fail(SMAT_ERR_BAD_ARG, "the plan belongs to device %d, the current device is %d", plan->device, dev);
    return SMAT_OK;
}

}  // namespace
}  // namespace smat

using namespace smat;

extern "C" {

int smat_fp4_plan_create(smat_fp4_plan** out, const void* codes, const void* scales, const float* row_scale, int fmt, const int* rowptr,
                         const int* colidx, size_t M, size_t K, size_t nnzb, size_t brow_begin, size_t brow_end, void* stream) {
    clear_error();
    if (!out || !rowptr || (nnzb && (!codes || !scales || !colidx))) return fail(SMAT_ERR_BAD_ARG, "NULL argument");
    *out = nullptr;
    if (fmt != SMAT_FP4_NV && fmt != SMAT_FP4_MX) return fail(SMAT_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (M % 16 || K % 16) return fail(SMAT_ERR_BAD_ARG, "M (%zu) and K (%zu) must be multiples of 16", M, K);
    if (((uintptr_t)codes | (uintptr_t)scales) & 15) return fail(SMAT_ERR_BAD_ARG, "codes and scales must be 16-byte aligned");
    if (brow_begin > brow_end || brow_end > M / 16)
        return fail(SMAT_ERR_BAD_ARG, "block-row range [%zu, %zu) outside [0, %zu]", brow_begin, brow_end, M / 16);
    if (nnzb * 16 >= ((size_t)1 << 31) || K >= ((size_t)1 << 31) || M / 16 >= ((size_t)1 << 31)) return fail(SMAT_ERR_RANGE, "size beyond 2^31");
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    smat_fp4_plan* p = new (std::nothrow) smat_fp4_plan();
    if (!p) return fail(SMAT_ERR_NOMEM, "out of host memory");
    p->device = ctx->device;
    Fp4View& v = p->v;
    v.codes = static_cast<const uint8_t*>(codes);
    v.scales = static_cast<const uint8_t*>(scales);
    v.row_scale = row_scale;
    v.colidx = colidx;
    v.fmt = fmt;
    v.K = K;
    v.brow_begin = brow_begin;
    v.block_rows = brow_end - brow_begin;
    cudaError_t e = cudaSuccess;
    if (v.block_rows) {
        const size_t bytes = 16 + v.block_rows * sizeof(int2);
        unsigned long long totals[2] = {0, 0};
        e = cudaMalloc(&p->buffer, bytes);
        if (e == cudaSuccess) e = cudaMemsetAsync(p->buffer, 0, 16, (cudaStream_t)stream);
        if (e == cudaSuccess) {
            int2* range = reinterpret_cast<int2*>(static_cast<char*>(p->buffer) + 16);
            v.range = range;
            fp4_ranges_kernel<<<(unsigned)v.block_rows, kThreads, 0, (cudaStream_t)stream>>>(
                rowptr + brow_begin, colidx, K, nnzb, range, static_cast<unsigned long long*>(p->buffer), ctx->d_status);
            count_launch();
            e = cudaGetLastError();
        }
        if (e == cudaSuccess) e = cudaMemcpyAsync(totals, p->buffer, 16, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
        v.blocks = totals[0];
        v.longest = totals[1];
    }
    if (e != cudaSuccess) {
        cudaFree(p->buffer);
        delete p;
        return fail(SMAT_ERR_CUDA, "plan build failed: %s", cudaGetErrorString(e));
    }
    *out = p;
    return SMAT_OK;
}

int smat_fp4_plan_spmm(const smat_fp4_plan* plan, const void* B, int dtype, void* C, size_t N, void* stream) {
    clear_error();
    if (dtype != SMAT_F16 && dtype != SMAT_BF16) return fail(SMAT_ERR_BAD_ARG, "B must be fp16 or bf16");
    if (int rc = check_product(plan, B, C, dtype, N)) return rc;
    if (!plan->v.block_rows || !N) return SMAT_OK;
    Fp4Rhs rhs;
    rhs.data = B;
    rhs.dtype = dtype;
    return launch_fp4_stream(plan->v, rhs, C, dtype, N, (cudaStream_t)stream);
}

int smat_fp4_plan_spmm_fp4(const smat_fp4_plan* plan, const void* codes, const void* scales, const float* row_scale, int fmt, void* C,
                           int c_dtype, size_t N, void* stream) {
    clear_error();
    if (int rc = check_product(plan, codes, C, c_dtype, N)) return rc;
    if (fmt != plan->v.fmt) return fail(SMAT_ERR_BAD_ARG, "B must be in the format of A");
    if (!plan->v.block_rows || !N) return SMAT_OK;
    if ((plan->v.K && !scales) || ((uintptr_t)scales & 15)) return fail(SMAT_ERR_BAD_ARG, "scales is NULL or not 16-byte aligned");
    Fp4Rhs rhs;
    rhs.data = codes;
    rhs.scales = static_cast<const uint8_t*>(scales);
    rhs.row_scale = row_scale;
    rhs.dtype = kFp4Rhs;
    return launch_fp4_stream(plan->v, rhs, C, c_dtype, N, (cudaStream_t)stream);
}

int smat_fp4_plan_destroy(smat_fp4_plan* plan) {
    clear_error();
    if (!plan) return SMAT_OK;
    const cudaError_t e = plan->buffer ? cudaFree(plan->buffer) : cudaSuccess;
    delete plan;
    if (e != cudaSuccess) return fail(SMAT_ERR_CUDA, "cudaFree failed: %s", cudaGetErrorString(e));
    return SMAT_OK;
}

}  // extern "C"
