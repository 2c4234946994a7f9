// C = A x B with A in 4-bit blocks and few columns of B: warps walk the blocks of a block-row.
//
// Mathematics.  A block is 16 x 16 and a scale covers a whole row of it, so the block's product P = codes(A) x B is formed with the
// codes as they are (exact in fp16 and bf16) by one m16n8k16 MMA per 8 columns, and C += scale(row) * P is one fp32 FMA per
// element: any scale format, nothing rounded on the way in.  B in 4 bits has one scale for the block's 16 rows as well.
//
// Layout.  The 128 bytes of a block are read as they lie, one word per lane.  Word l holds half of row l / 2; MMA rows g and g + 8
// stand for rows 2g and 2g + 1 of the block, which lie in the words of lanes 4g .. 4g + 3, so one exchange with lane l ^ 2 gives
// each lane four columns of both rows.  The k order inside a block is permuted by that, in the same way for A and B.
#include "fp4_device.cuh"
#include "smat_internal.h"

#include <cooperative_groups.h>

namespace smat {
namespace {

constexpr int kWarps = 8;

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

struct StreamArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scale;  // first of the range, or null
    const int* colidx;
    const int2* range;
    const void* B;
    const uint8_t* b_scales;
    const float* b_row_scale;
    void* C;
    int c_dtype;
    int block_rows, N;
    size_t K;
};

// BT: SMAT_F16, SMAT_BF16 or kFp4Rhs.  NT: 8-column tiles of C per warp.  WR warps of a CTA (times the CTAs of a cluster) share a
// block-row; a CTA holds kWarps / WR block-rows.
template <int BT, int FMT, int NT, int U>
__global__ void __launch_bounds__(kWarps * 32) fp4_stream_kernel(const StreamArgs a, int wr) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int cl = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int rows_per_cta = kWarps / wr;
    const int row_ctas = (a.block_rows + rows_per_cta - 1) / rows_per_cta;
    const int r0 = (int)(blockIdx.x / cl % row_ctas) * rows_per_cta, r = r0 + warp / wr;
    const int n0 = (int)(blockIdx.x / cl / row_ctas) * NT * 8;
    const int kbase = (t & 1) * 8 + (t >> 1) * 4;
    const size_t quads = (a.K + 63) / 64;

    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[j][e] = 0.f;

    if (r < a.block_rows) {
        const int2 range = a.range[r];
        const int n = range.y - range.x, parts = wr * cl, part = rank * wr + warp % wr;
        const int lo = range.x + (int)((long long)n * part / parts), hi = range.x + (int)((long long)n * (part + 1) / parts);
        for (int p0 = lo; p0 < hi; p0 += 32) {
            const int mine = p0 + lane < hi ? __ldg(a.colidx + p0 + lane) : 0;
            const int cnt = min(32, hi - p0);
            for (int u0 = 0; u0 < cnt; u0 += U) {
                uint32_t w[U], sc[U], b[U][NT][2];
                uint32_t bs[U][NT][2];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int col = __shfl_sync(~0u, mine, (u0 + u) & 31);
                    const bool in = u0 + u < cnt;
                    const size_t p = (size_t)(p0 + u0 + u);
                    w[u] = in ? __ldg(reinterpret_cast<const uint32_t*>(a.codes + p * 128) + lane) : 0;
                    sc[u] = in ? __ldg(reinterpret_cast<const uint16_t*>(a.scales + p * 16) + g) : 0;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const int c = n0 + j * 8 + g;
                        const bool ok = in && c < a.N;
                        if constexpr (BT == kFp4Rhs) {
                            b[u][j][0] = ok ? __ldg(reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(a.B) + c * (quads * 32) + (col + kbase) / 2)) : 0;
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int cc = n0 + j * 8 + 2 * t + e;
                                bs[u][j][e] = in && cc < a.N ? __ldg(a.b_scales + dense_scale_at<FMT>(cc, col, quads)) : 0;
                            }
                        } else {
                            const uint2 v = ok ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.B) + (size_t)c * a.K + col + kbase)) : make_uint2(0, 0);
                            b[u][j][0] = v.x;
                            b[u][j][1] = v.y;
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (u0 + u >= cnt) break;
                    const uint32_t got = __shfl_xor_sync(~0u, t < 2 ? w[u] >> 16 : w[u] & 0xffffu, 2);
                    const uint32_t both = t < 2 ? (w[u] & 0xffffu) | got << 16 : got | (w[u] & 0xffff0000u);
                    uint32_t h[4];
                    e2m1x8_to_f16(both, h);
                    uint32_t am[4] = {h[0], h[2], h[1], h[3]};
                    if constexpr (BT == SMAT_BF16) {
#pragma unroll
                        for (int e = 0; e < 4; e++) am[e] = f16_code_to_bf16(am[e]);
                    }
                    const float s0 = scale_value<FMT>(sc[u] & 0xff), s1 = scale_value<FMT>(sc[u] >> 8);
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        float d[4];
                        if constexpr (BT == kFp4Rhs) {
                            uint32_t b0, b1;
                            e2m1x4_to_f16((uint16_t)b[u][j][0], b0, b1);
                            mma_16816<false>(d, am, b0, b1);
                            const float q0 = scale_value<FMT>(bs[u][j][0]), q1 = scale_value<FMT>(bs[u][j][1]);
                            d[0] *= q0; d[1] *= q1; d[2] *= q0; d[3] *= q1;
                        } else {
                            mma_16816<BT == SMAT_BF16>(d, am, b[u][j][0], b[u][j][1]);
                        }
                        acc[j][0] = fmaf(s0, d[0], acc[j][0]);
                        acc[j][1] = fmaf(s0, d[1], acc[j][1]);
                        acc[j][2] = fmaf(s1, d[2], acc[j][2]);
                        acc[j][3] = fmaf(s1, d[3], acc[j][3]);
                    }
                }
            }
        }
    }

    // Parts of a block-row are added in a fixed order: the warps of a CTA, then the CTAs of the cluster.
    constexpr int W = NT * 8, ROW = W + 4;  // floats of a row of a warp's tile; padded against bank conflicts
    __shared__ float part_sum[kWarps][16 * ROW];
    float* my = part_sum[warp];
#pragma unroll
    for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int e = 0; e < 4; e++) my[(2 * g + e / 2) * ROW + j * 8 + 2 * t + e % 2] = acc[j][e];
    }
    __syncthreads();
    if (cl > 1) {  // wr == kWarps
        for (int i = threadIdx.x; i < 16 * W; i += kWarps * 32) {
            float v = 0.f;
            for (int k = 0; k < kWarps; k++) v += part_sum[k][i / W * ROW + i % W];
            part_sum[0][i / W * ROW + i % W] = v;
        }
        cluster.sync();
    }
    if (rank == 0) {
        for (int i = threadIdx.x; i < rows_per_cta * 16 * W; i += kWarps * 32) {
            const int br = i / (16 * W), row = i / W % 16, c = i % W;
            const int gr = r0 + br;
            if (gr >= a.block_rows || n0 + c >= a.N) continue;
            float v = 0.f;
            if (cl > 1) {
                for (int k = 0; k < cl; k++) v += cluster.map_shared_rank(&part_sum[0][0], k)[row * ROW + c];
            } else {
                for (int k = 0; k < wr; k++) v += part_sum[br * wr + k][row * ROW + c];
            }
            const size_t m = (size_t)gr * 16 + row;
            if (a.row_scale) v *= __ldg(a.row_scale + m);
            if (a.b_row_scale) v *= __ldg(a.b_row_scale + n0 + c);
            store_c(a.C, a.c_dtype, m * a.N + n0 + c, v);
        }
    }
    if (cl > 1) cluster.sync();  // shared memory is read from rank 0 until here
}

template <int BT, int FMT, int NT, int U>
cudaError_t launch(const StreamArgs& a, int wr, int cl, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    const size_t ctas = ((size_t)a.block_rows + kWarps / wr - 1) / (kWarps / wr) * cl * (((size_t)a.N + NT * 8 - 1) / (NT * 8));
    if (ctas >= ((size_t)1 << 31)) return cudaErrorInvalidConfiguration;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fp4_stream_kernel<BT, FMT, NT, U>, a, wr);
}

template <int BT, int FMT>
cudaError_t launch_width(const StreamArgs& a, int wr, int cl, cudaStream_t stream) {
    if (a.N <= 8) return launch<BT, FMT, 1, 8>(a, wr, cl, stream);
    if (a.N <= 16) return launch<BT, FMT, 2, 4>(a, wr, cl, stream);
    if (a.N <= 32) return launch<BT, FMT, 4, 2>(a, wr, cl, stream);
    return launch<BT, FMT, 8, 2>(a, wr, cl, stream);
}
template <int BT>
cudaError_t launch_format(int fmt, const StreamArgs& a, int wr, int cl, cudaStream_t stream) {
    return fmt == SMAT_FP4_NV ? launch_width<BT, SMAT_FP4_NV>(a, wr, cl, stream) : launch_width<BT, SMAT_FP4_MX>(a, wr, cl, stream);
}

}  // namespace

int launch_fp4_stream(const Fp4View& A, const Fp4Rhs& B, void* C, int c_dtype, size_t N, cudaStream_t stream) {
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    StreamArgs a = {};
    a.codes = A.codes;
    a.scales = A.scales;
    a.row_scale = A.row_scale ? A.row_scale + A.brow_begin * 16 : nullptr;
    a.colidx = A.colidx;
    a.range = A.range;
    a.B = B.data;
    a.b_scales = B.scales;
    a.b_row_scale = B.row_scale;
    a.C = C;
    a.c_dtype = c_dtype;
    a.block_rows = (int)A.block_rows;
    a.N = (int)N;
    a.K = A.K;
    // Warps of a block-row: so many that the SMs hold about 32 warps each, but not below 8 blocks a warp.
    const size_t tiles = (N + 63) / 64, want = (size_t)ctx->sm_count * 32;
    const size_t per_row = A.blocks / A.block_rows + 1;
    size_t parts = 1;
    while (parts < 64 && A.block_rows * tiles * parts * 2 <= want && per_row / (parts * 2) >= 8) parts *= 2;
    const int wr = (int)(parts < kWarps ? parts : kWarps), cl = (int)(parts / wr);
    cudaError_t e;
    if (B.dtype == SMAT_F16) e = launch_format<SMAT_F16>(A.fmt, a, wr, cl, stream);
    else if (B.dtype == SMAT_BF16) e = launch_format<SMAT_BF16>(A.fmt, a, wr, cl, stream);
    else e = launch_format<kFp4Rhs>(A.fmt, a, wr, cl, stream);
    count_launch();
    SMAT_CUDA_TRY(e);
    return SMAT_OK;
}

}  // namespace smat
