// Plans for products of a block-sparse matrix in 4 bits (smat_fp4_plan_*).
#include <algorithm>
#include <new>

#include "fp4_format.h"
#include "smat_internal.h"

struct smat_fp4_plan {
    smat::Fp4View v;
    int device = -1;
    void* buffer = nullptr;  // totals, block ranges, rows and first steps
    const int2* range = nullptr;
    const int* four_first = nullptr;
    smat::Fp4Row* rows = nullptr;
    void* fours = nullptr;
    void* steps = nullptr;   // steps and what their tiles are made of
    smat::Fp4Where* where = nullptr;
    void* tiles = nullptr;
    int* gsp = nullptr;  // first steps on the host
};

namespace smat {
namespace {

constexpr int kThreads = 256;
// Tiles are made where a step of 256 x 256 holds so many blocks (of 256) on average; they take 36 KB a step.  For wide products they are
// faster at any fill (8192 x 8192, N = 512, tiles against warp-level MMAs: 31 and 55 us with 2 blocks a step, 33 and 77 with 4, 33 and
// 211 with 16), so this bounds the memory: 9 KB a block, 64 times what is stored.
constexpr size_t kFp4TileFill = 4;
// With so few columns and blocks the warp-level kernel is faster all the same.  Measured, us, warp-level and tiles, 8 columns: 8192 x 8192
// 6.7 and 13.9 with 5 200 blocks, 7.4 and 14.8 with 26 200, 11.3 and 14.8 with 52 400; 28672 x 8192 18.2 and 30.0 with 91 700;
// 8192 x 28672 16.2 and 31.2 with 91 700, 27.1 and 31.1 with 183 500.  16 columns: 9.4 and 13.9, 10.3 and 14.8, 16.2 and 14.9; 27.1 and
// 30.0; 23.8 and 31.3, 40.4 and 30.8.  So both bounds are on the tiles' side: with more blocks, or a few more columns of few blocks,
// the warp-level kernel would still be the faster one.
constexpr size_t kFp4NarrowColumns = 8, kFp4NarrowBlocks = 50000;

// Looks a block-row's pointers and columns over (a CTA a block-row): they have to lie in the arrays and the matrix, the columns in
// ascending order.  An inconsistent block-row is left out (empty) and reported.  totals: blocks, longest block-row.
__global__ void __launch_bounds__(kThreads) fp4_ranges_kernel(const int* __restrict__ rowptr, const int* __restrict__ colidx, size_t K, size_t nnzb,
                                                              int2* __restrict__ range, int* __restrict__ fours,
                                                              unsigned long long* __restrict__ totals, int* status) {
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
        fours[r + 1] = bad ? 0 : (hi - lo + 3) / 4;
        if (!bad) {
            atomicAdd(totals, (unsigned long long)(hi - lo));
            atomicMax(totals + 1, (unsigned long long)(hi - lo));
        }
    }
}

// Fours of a block-row (a CTA a block-row, a warp a four); `first` is scanned.  Of SMAT_FP4_MX, a block-row in which the blocks of a
// pair have different scales is left out (empty) and reported: an MMA takes one scale for both.
template <int FMT>
__global__ void __launch_bounds__(kThreads) fp4_fours_kernel(const int2* __restrict__ range, const int* __restrict__ first, const int* __restrict__ colidx,
                                                             const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             Fp4Row* __restrict__ rows, uint8_t* __restrict__ fours, int* status) {
    const int2 mine = range[blockIdx.x];
    const int f0 = first[blockIdx.x], lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    bool wrong = false;
    if constexpr (FMT == SMAT_FP4_MX) {
        for (int p = mine.x + (int)threadIdx.x; p + 1 < mine.y; p += kThreads) {
            const int c = __ldg(colidx + p);
            if (c & 16 || __ldg(colidx + p + 1) != c + 16) continue;
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(scales) + p), y = __ldg(reinterpret_cast<const uint4*>(scales) + p + 1);
            wrong |= x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w;
        }
        wrong = __syncthreads_or(wrong);
    }
    if (threadIdx.x == 0) {
        rows[blockIdx.x] = {f0, wrong ? 0 : mine.y - mine.x};
        if (wrong) atomicCAS(status, 0, kStatusBadScales);
    }
    for (int f = threadIdx.x / 32; f * 4 < mine.y - mine.x; f += kThreads / 32) {
        uint8_t* const to = fours + (size_t)(f0 + f) * kFp4FourBytes;
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int p = mine.x + 4 * f + u;
            const uint16_t* row = reinterpret_cast<const uint16_t*>(codes + (size_t)p * 128 + g * 16);  // rows 2g and 2g + 1, four codes an element
            w[u] = p < mine.y ? __ldg(row + t) | (uint32_t)__ldg(row + 4 + t) << 16 : 0;
        }
        *reinterpret_cast<uint4*>(to + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        const int p = mine.x + 4 * f + t;  // lane (g, t): scales of rows 2g and 2g + 1 of block t
        *reinterpret_cast<uint16_t*>(to + 512 + g * 8 + t * 2) = p < mine.y ? __ldg(reinterpret_cast<const uint16_t*>(scales + (size_t)p * 16) + g) : 0;
        if (lane < 4) *reinterpret_cast<int*>(to + 576 + lane * 4) = __ldg(colidx + min(mine.x + 4 * f + lane, mine.y - 1));
    }
}

// The steps of a group (a CTA a group, a warp a block-row): a bitmap of the 256-column ranges that hold a block, counted (FILL false)
// or turned into records.  Shared memory: `words` words of bitmap and, to fill, as many prefix counts.
constexpr int kStepThreads = 32 * (int)kFp4GroupRows;
constexpr size_t kFp4MostColumns = (size_t)1 << 26;  // K lies below
constexpr int kStepWords = (int)(kFp4MostColumns / (32 * kFp4StepColumns));  // words of a bitmap, at most
template <bool FILL>
__global__ void __launch_bounds__(kStepThreads) fp4_steps_kernel(const int2* __restrict__ range, const int* __restrict__ colidx, int block_rows,
                                                                 int words, int* __restrict__ gsp, uint32_t* __restrict__ steps,
                                                                 Fp4Where* __restrict__ where) {
    extern __shared__ uint32_t sm[];
    uint32_t *bitmap = sm, *prefix = sm + words;
    __shared__ int sums[kStepThreads];
    const int tid = threadIdx.x, e = tid / 32, row = (int)(blockIdx.x * kFp4GroupRows) + e;
    const int2 mine = row < block_rows ? range[row] : make_int2(0, 0);
    for (int w = tid; w < words; w += kStepThreads) bitmap[w] = 0;
    __syncthreads();
    for (int p = mine.x + tid % 32; p < mine.y; p += 32) {
        const int k = __ldg(colidx + p) >> 8;
        atomicOr(&bitmap[k >> 5], 1u << (k & 31));
    }
    __syncthreads();
    const int per = (words + kStepThreads - 1) / kStepThreads, w0 = min(words, tid * per), w1 = min(words, w0 + per);
    int n = 0;
    for (int w = w0; w < w1; w++) n += __popc(bitmap[w]);
    sums[tid] = n;
    __syncthreads();
    for (int d = 1; d < kStepThreads; d *= 2) {
        const int v = tid >= d ? sums[tid - d] : 0;
        __syncthreads();
        sums[tid] += v;
        __syncthreads();
    }
    if (!FILL) {
        if (tid == 0) gsp[blockIdx.x + 1] = max(1, sums[kStepThreads - 1]);
        return;
    }
    int before = sums[tid] - n;
    for (int w = w0; w < w1; w++) {
        prefix[w] = before;
        before += __popc(bitmap[w]);
    }
    __syncthreads();
    const int first = gsp[blockIdx.x];
    for (int p = mine.x + tid % 32; p < mine.y; p += 32) {
        const int k = __ldg(colidx + p) >> 8;
        if (p > mine.x && __ldg(colidx + p - 1) >> 8 == k) continue;  // the first block of these columns speaks for all
        uint32_t blocks = 0, mask = 0;
        for (int q = p, c; q < mine.y && (c = __ldg(colidx + q)) >> 8 == k; q++) {
            blocks |= 1u << (c >> 4 & 15);
            mask |= 1u << (c >> 6 & 3);
        }
        const int at = first + (int)prefix[k >> 5] + __popc(bitmap[k >> 5] & ((1u << (k & 31)) - 1));
        where[at].group = blockIdx.x;  // the same from all block-rows
        where[at].begin[e] = p;
        where[at].blocks[e] = (uint16_t)blocks;
        atomicOr(&steps[at], (uint32_t)k << 8 | mask << (e / 8 * 4));
    }
}

// Lays the blocks of a step out into its two tiles: a warp a block-row, a lane half a row (eight block-columns).  Block-rows that `rows`
// says to be empty are.
template <int FMT>
__global__ void __launch_bounds__(kStepThreads) fp4_tiles_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 const Fp4Row* __restrict__ rows, const Fp4Where* __restrict__ where,
                                                                 uint8_t* __restrict__ tiles) {
    const uint32_t e = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane & 15, h = lane >> 4;
    const Fp4Where& w = where[blockIdx.x];
    const bool left_out = w.blocks[e] && rows[w.group * (int)kFp4GroupRows + (int)e].blocks == 0;
    const uint32_t blocks = left_out ? 0 : w.blocks[e], mine = blocks >> (8 * h) & 0xff;
    size_t p = (size_t)w.begin[e] + (h ? __popc(blocks & 0xff) : 0);
    uint2 v[8];
    uint32_t s[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) {
        v[j] = make_uint2(0, 0);
        s[j] = 0;
        if (mine >> j & 1) {
            v[j] = __ldg(reinterpret_cast<const uint2*>(codes + p * 128) + r);
            s[j] = __ldg(scales + p * 16 + r);
            p++;
        }
    }
    const uint32_t row = (e & 7) * 16 + r;
    uint8_t* const tile = tiles + ((size_t)blockIdx.x * 2 + e / 8) * kFp4TileBytes;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
        *reinterpret_cast<uint4*>(tile + row * 128 + (((4 * h + j) ^ (r & 7)) << 4)) = make_uint4(v[2 * j].x, v[2 * j].y, v[2 * j + 1].x, v[2 * j + 1].y);
#pragma unroll
    for (uint32_t j = 0; j < 2; j++) {
        const uint32_t* q = s + 4 * j;
        *reinterpret_cast<uint32_t*>(tile + kFp4TileCodes + (2 * h + j) * 512 + (row & 31) * 16 + (row >> 5) * 4) =
            FMT == SMAT_FP4_NV ? q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24 : (q[0] | q[1]) | (q[2] | q[3]) << 8;  // mxfp4: the blocks of a pair have equal scales
    }
}

// What a plan holds of codes and scales.
int fill_values(const smat_fp4_plan* p, const DeviceCtx* ctx, cudaStream_t stream) {
    const Fp4View& v = p->v;
    if (!v.block_rows) return SMAT_OK;
    const auto fours = v.fmt == SMAT_FP4_NV ? fp4_fours_kernel<SMAT_FP4_NV> : fp4_fours_kernel<SMAT_FP4_MX>;
    fours<<<(unsigned)v.block_rows, kThreads, 0, stream>>>(p->range, p->four_first, v.colidx, v.codes, v.scales, p->rows,
                                                           static_cast<uint8_t*>(p->fours), ctx->d_status);
    count_launch();
    SMAT_CUDA_TRY(cudaGetLastError());
    if (!v.tiles || !v.blocks) return SMAT_OK;
    uint8_t* tiles = static_cast<uint8_t*>(p->tiles);
    const auto lay_out = v.fmt == SMAT_FP4_NV ? fp4_tiles_kernel<SMAT_FP4_NV> : fp4_tiles_kernel<SMAT_FP4_MX>;
    lay_out<<<(unsigned)v.total_steps, kStepThreads, 0, stream>>>(v.codes, v.scales, p->rows, p->where, tiles);
    count_launch();
    SMAT_CUDA_TRY(cudaGetLastError());
    return SMAT_OK;
}

// Ranges and totals of a plan, and the steps and tiles for products with B in 4 bits.  Synchronises the stream.
int build_plan(smat_fp4_plan* p, const int* rowptr, const int* colidx, size_t nnzb, bool with_tiles, const DeviceCtx* ctx, cudaStream_t stream) {
    Fp4View& v = p->v;
    const size_t groups = (v.block_rows + kFp4GroupRows - 1) / kFp4GroupRows;
    // totals, ranges and rows of block-rows, first fours of block-rows, first steps of groups
    const size_t bytes = 16 + v.block_rows * (sizeof(int2) + sizeof(Fp4Row)) + (v.block_rows + 1 + groups + 1) * sizeof(int);
    SMAT_CUDA_TRY(cudaMalloc(&p->buffer, bytes));
    unsigned long long* totals = static_cast<unsigned long long*>(p->buffer);
    int2* range = reinterpret_cast<int2*>(totals + 2);
    p->rows = reinterpret_cast<Fp4Row*>(range + v.block_rows);
    int* fours = reinterpret_cast<int*>(p->rows + v.block_rows);
    int* gsp = fours + v.block_rows + 1;
    SMAT_CUDA_TRY(cudaMemsetAsync(p->buffer, 0, bytes, stream));
    fp4_ranges_kernel<<<(unsigned)v.block_rows, kThreads, 0, stream>>>(rowptr + v.brow_begin, colidx, v.K, nnzb, range, fours, totals, ctx->d_status);
    count_launch();
    SMAT_CUDA_TRY(cudaGetLastError());
    if (int rc = scan_inplace_async(fours, (int)v.block_rows + 1, stream)) return rc;
    const int words = (int)((v.K + 32 * kFp4StepColumns - 1) / (32 * kFp4StepColumns));
    if (with_tiles) {
        fp4_steps_kernel<false><<<(unsigned)groups, kStepThreads, words * 4, stream>>>(range, colidx, (int)v.block_rows, words, gsp, nullptr, nullptr);
        count_launch();
        SMAT_CUDA_TRY(cudaGetLastError());
        if (int rc = scan_inplace_async(gsp, (int)groups + 1, stream)) return rc;
    }
    unsigned long long h_totals[2] = {0, 0};
    int h_steps = 0, h_fours = 0;
    SMAT_CUDA_TRY(cudaMemcpyAsync(h_totals, totals, sizeof(h_totals), cudaMemcpyDeviceToHost, stream));
    SMAT_CUDA_TRY(cudaMemcpyAsync(&h_fours, fours + v.block_rows, sizeof(int), cudaMemcpyDeviceToHost, stream));
    SMAT_CUDA_TRY(cudaMemcpyAsync(&h_steps, gsp + groups, sizeof(int), cudaMemcpyDeviceToHost, stream));
    SMAT_CUDA_TRY(cudaStreamSynchronize(stream));
    if (h_totals[0] > nnzb) {
        // Block-rows overlap, so row pointers run backwards somewhere, which is reported.  The 32-bit sums may have wrapped (16384 row
        // pointers in turn 0 and 2^20 are enough), so nothing is laid out by them: all block-rows count as empty.
        SMAT_CUDA_TRY(cudaMemsetAsync(p->buffer, 0, bytes, stream));
        h_totals[0] = h_totals[1] = 0;
        h_steps = h_fours = 0;
        with_tiles = false;
    }
    p->range = range;
    p->four_first = fours;
    v.rows = p->rows;
    v.blocks = h_totals[0];
    v.longest = h_totals[1];
    SMAT_CUDA_TRY(cudaMalloc(&p->fours, std::max<size_t>(h_fours, 1) * kFp4FourBytes));
    v.fours = static_cast<const uint8_t*>(p->fours);
    const size_t steps = (size_t)h_steps;
    if (with_tiles && v.blocks >= kFp4TileFill * steps) {
        SMAT_CUDA_TRY(cudaMalloc(&p->steps, steps * (sizeof(uint32_t) + sizeof(Fp4Where))));
        uint32_t* step = static_cast<uint32_t*>(p->steps);
        p->where = reinterpret_cast<Fp4Where*>(step + steps);
        SMAT_CUDA_TRY(cudaMalloc(&p->tiles, steps * 2 * kFp4TileBytes));
        SMAT_CUDA_TRY(cudaMemsetAsync(p->steps, 0, steps * (sizeof(uint32_t) + sizeof(Fp4Where)), stream));
        // The limit is the function's on this device, not this launch's: one for all plans, which may be made by several threads.
        SMAT_CUDA_TRY(cudaFuncSetAttribute(fp4_steps_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStepWords * 8));
        fp4_steps_kernel<true><<<(unsigned)groups, kStepThreads, words * 8, stream>>>(range, colidx, (int)v.block_rows, words, gsp, step, p->where);
        count_launch();
        SMAT_CUDA_TRY(cudaGetLastError());
        p->gsp = new (std::nothrow) int[groups + 1];
        if (!p->gsp) return fail(SMAT_ERR_NOMEM, "out of host memory");
        SMAT_CUDA_TRY(cudaMemcpyAsync(p->gsp, gsp, (groups + 1) * sizeof(int), cudaMemcpyDeviceToHost, stream));
        v.gsp = gsp;
        v.h_gsp = p->gsp;
        v.total_steps = steps;
        v.steps = step;
        v.tiles = static_cast<const uint8_t*>(p->tiles);
    }
    if (int rc = fill_values(p, ctx, stream)) return rc;
    SMAT_CUDA_TRY(cudaStreamSynchronize(stream));
    return SMAT_OK;
}

cudaError_t free_plan(smat_fp4_plan* p) {
    cudaError_t e = cudaSuccess;
    for (void* m : {p->buffer, p->fours, p->steps, p->tiles}) {
        const cudaError_t f = cudaFree(m);
        if (e == cudaSuccess) e = f;
    }
    delete[] p->gsp;
    delete p;
    return e;
}

int check_plan_device(const smat_fp4_plan* plan) {
    int dev = -1;
    SMAT_CUDA_TRY(cudaGetDevice(&dev));
    if (dev != plan->device)
        return fail(SMAT_ERR_BAD_ARG, "the plan belongs to device %d but device %d is current", plan->device, dev);
    return SMAT_OK;
}

int check_product(const smat_fp4_plan* plan, const void* B, const void* C, int c_dtype, size_t N) {
    // The kernels count columns in 32 bits and add offsets of up to two tiles of 256 to the first column of the last tile.
    if (N >= ((size_t)1 << 31) - 512) return fail(SMAT_ERR_RANGE, "N (%zu) beyond 2^31 - 513", N);
    if (!plan) return fail(SMAT_ERR_BAD_ARG, "plan is NULL");
    if (c_dtype != SMAT_F16 && c_dtype != SMAT_BF16) return fail(SMAT_ERR_BAD_ARG, "C must be fp16 or bf16");
    if (plan->v.block_rows && N && (!C || (plan->v.K && !B))) return fail(SMAT_ERR_BAD_ARG, "B or C is NULL");
    if (((uintptr_t)B | (uintptr_t)C) & 15) return fail(SMAT_ERR_BAD_ARG, "B and C must be 16-byte aligned");
    return check_plan_device(plan);
}

}  // namespace
}  // namespace smat

using namespace smat;

extern "C" {

int smat_fp4_plan_create(smat_fp4_plan** out, const void* codes, const void* scales, const float* row_scale, int fmt, const int* rowptr,
                         const int* colidx, size_t M, size_t K, size_t nnzb, size_t brow_begin, size_t brow_end, int with_tiles,
                         void* stream) {
    clear_error();
    if (!out || !rowptr || (nnzb && (!codes || !scales || !colidx))) return fail(SMAT_ERR_BAD_ARG, "NULL argument");
    *out = nullptr;
    if (fmt != SMAT_FP4_NV && fmt != SMAT_FP4_MX) return fail(SMAT_ERR_BAD_ARG, "unknown 4-bit format %d", fmt);
    if (M % 16 || K % 16) return fail(SMAT_ERR_BAD_ARG, "M (%zu) and K (%zu) must be multiples of 16", M, K);
    if (((uintptr_t)codes | (uintptr_t)scales) & 15) return fail(SMAT_ERR_BAD_ARG, "codes and scales must be 16-byte aligned");
    if (brow_begin > brow_end || brow_end > M / 16)
        return fail(SMAT_ERR_BAD_ARG, "block-row range [%zu, %zu) outside [0, %zu]", brow_begin, brow_end, M / 16);
    if (nnzb * 16 >= ((size_t)1 << 31) || M / 16 >= ((size_t)1 << 30)) return fail(SMAT_ERR_RANGE, "nonzeroBlocks beyond 2^27 - 1 or M beyond 2^34 - 16");
    if (K >= kFp4MostColumns) return fail(SMAT_ERR_RANGE, "K (%zu) beyond 2^26 - 1", K);  // a bitmap of steps in shared memory
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
    if (v.block_rows) {
        if (int rc = build_plan(p, rowptr, colidx, nnzb, with_tiles != 0, ctx, (cudaStream_t)stream)) {
            free_plan(p);
            return rc;
        }
    }
    *out = p;
    return SMAT_OK;
}

int smat_fp4_plan_set_values(smat_fp4_plan* plan, void* stream) {
    clear_error();
    if (!plan) return fail(SMAT_ERR_BAD_ARG, "plan is NULL");
    if (int rc = check_plan_device(plan)) return rc;
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    return fill_values(plan, ctx, (cudaStream_t)stream);
}

static int spmm_fp4(const smat_fp4_plan* plan, const void* codes, const void* scales, const float* row_scale, int fmt, void* C, int c_dtype,
                    size_t N, void* stream, bool selftest) {
    clear_error();
    if (int rc = check_product(plan, codes, C, c_dtype, N)) return rc;
    if (fmt != plan->v.fmt) return fail(SMAT_ERR_BAD_ARG, "B must be in the format of A");
    if (selftest && (!plan->v.tiles || !plan->v.blocks || !N)) return fail(SMAT_ERR_BAD_ARG, "this product's kernel has no such self-test");
    if (!plan->v.block_rows || !N) return SMAT_OK;
    if ((plan->v.K && !scales) || ((uintptr_t)scales & 15)) return fail(SMAT_ERR_BAD_ARG, "scales is NULL or not 16-byte aligned");
    if (!plan->v.blocks) {
        SMAT_CUDA_TRY(cudaMemsetAsync(C, 0, plan->v.block_rows * 16 * N * 2, (cudaStream_t)stream));
        return SMAT_OK;
    }
    Fp4Rhs rhs;
    rhs.data = codes;
    rhs.scales = static_cast<const uint8_t*>(scales);
    rhs.row_scale = row_scale;
    rhs.dtype = kFp4Rhs;
    const bool narrow = N <= kFp4NarrowColumns && plan->v.blocks <= kFp4NarrowBlocks && !selftest;
    if (plan->v.tiles && !narrow) return launch_fp4_tile(plan->v, rhs, C, c_dtype, N, (cudaStream_t)stream, selftest);
    return launch_fp4_stream(plan->v, rhs, C, c_dtype, N, (cudaStream_t)stream);
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
    return spmm_fp4(plan, codes, scales, row_scale, fmt, C, c_dtype, N, stream, false);
}

int smat_selftest_fp4_plan_wait_timeout(const smat_fp4_plan* plan, const void* codes, const void* scales, const float* row_scale, int fmt,
                                        void* C, int c_dtype, size_t N, void* stream) {
    return spmm_fp4(plan, codes, scales, row_scale, fmt, C, c_dtype, N, stream, true);
}

int smat_fp4_plan_destroy(smat_fp4_plan* plan) {
    clear_error();
    if (!plan) return SMAT_OK;
    const cudaError_t e = free_plan(plan);
    if (e != cudaSuccess) return fail(SMAT_ERR_CUDA, "cudaFree failed: %s", cudaGetErrorString(e));
    return SMAT_OK;
}

}  // extern "C"
