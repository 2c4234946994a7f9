// C = A x B with A in 4-bit blocks and few columns of B: warps walk the blocks of a block-row.
//
// Mathematics.  A block is 16 x 16 and a scale covers a whole row of it.  e2m1 times e4m3 has at most six significant bits and fits
// fp16 and bf16, and e2m1 times 2^e fits bf16, so the scaled values go into m16n8k16 MMAs that accumulate in fp32, nothing rounded on
// the way in.  Powers of two beyond the range of fp16 (SMAT_FP4_MX and fp16) and scales of B in 4 bits are applied to a block's product
// instead, one fp32 FMA per element.  Of SMAT_FP4_MX, where scales go up to 2^127, all sums are kept times a power of two that lets
// nothing overflow on the way to a result that fp32 holds: values of A in bf16 are at most 6 * 2^127 (kept times 2^-3), a block's
// product with a scale of B in 4 bits at most 16 * 36 * 2^127 (kept times 2^-12).  Downwards both stay exact.
//
// Layout.  Plans keep the blocks in fours in the order in which a warp's lanes take them (fp4_format.h): read as they are stored, a
// word a lane and block, they cost twice the instructions.  MMA rows g and g + 8 stand for rows 2g and 2g + 1 of the block, the k
// order inside a block is permuted in the same way for A and B.
//
// What bounds it: instructions (some 20 a block and 8 columns) and, from 16 columns on, the rows of B that every block gathers through
// L2.  The next four are on their way while a four is multiplied, without branches: a load behind one is waited for before the next
// is issued.  One token, layer 8192 x 28672 at 20 % (fp16, nvfp4): 31 us with branches, 22 without, 12.2 in fours (2.2 TB/s; an empty
// product takes 3.6); 16 tokens (bf16, mxfp4): 21, of which the rows of B alone, 2.9 million sectors, take 10.  More warps a block-row
// or an SM than now are slower or equal (64 instead of 32 an SM: 16 us).
#include "fp4_device.cuh"
#include "smat_internal.h"

#include <cooperative_groups.h>

namespace smat {
namespace {

constexpr int kWarps = 8;

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

struct StreamArgs {
    const uint8_t* fours;
    const Fp4Row* rows;
    const float* row_scale;  // first of the range, or null
    const void* B;
    const uint8_t* b_scales;
    const float* b_row_scale;
    void* C;
    int c_dtype;
    int block_rows, N;
    size_t K;
};

// Four blocks, and U of them with their rows of B.
struct Four {
    uint4 w;     // codes
    uint2 s;     // scales
    int4 col;
};
template <int BT, int NT, int U>
struct Panel {
    uint2 b[U][NT];                            // 16 bits: four values; 4 bits: four codes in x
    uint16_t q[BT == kFp4Rhs ? U : 1][NT][2];  // 4 bits: scales of columns 2t and 2t + 1
};

// BT: SMAT_F16, SMAT_BF16 or kFp4Rhs.  NT: 8-column tiles of C per warp.  WR warps of a CTA (times the CTAs of a cluster) share a
// block-row; a CTA holds kWarps / WR block-rows.
template <int BT, int FMT, int NT, int U>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) fp4_stream_kernel(const StreamArgs a, int wr) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int cl = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int rows_per_cta = kWarps / wr;
    const int row_ctas = (a.block_rows + rows_per_cta - 1) / rows_per_cta;
    const int r0 = (int)(blockIdx.x / cl % row_ctas) * rows_per_cta, r = r0 + warp / wr;
    const int n0 = (int)(blockIdx.x / cl / row_ctas) * NT * 8;
    const size_t quads = (a.K + 63) / 64;
    constexpr bool DOWN = FMT == SMAT_FP4_MX && BT != SMAT_F16;                         // sums are kept times 1 / UP
    constexpr float UP = !DOWN ? 1.f : BT == SMAT_BF16 ? 8.f : 4096.f;
    constexpr bool FOLD = BT == SMAT_BF16 || (BT == SMAT_F16 && FMT == SMAT_FP4_NV);  // scales go into the values of A

    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[j][e] = 0.f;

    if (r < a.block_rows) {
        const Fp4Row row = a.rows[r];
        const int n = (row.blocks + 3) / 4, parts = wr * cl, part = rank * wr + warp % wr;
        const int lo = (int)((long long)n * part / parts), hi = (int)((long long)n * (part + 1) / parts);
        const uint8_t* at = a.fours + (size_t)(row.first + lo) * kFp4FourBytes;
        const uint8_t* b0[NT];  // this lane's columns of C; those beyond N are computed from the last one and not stored
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const size_t c = (size_t)min(n0 + j * 8 + g, a.N - 1);
            b0[j] = static_cast<const uint8_t*>(a.B) + (BT == kFp4Rhs ? c * (quads * 32) + 2 * t : (c * a.K + 4 * t) * 2);
        }
        auto load = [&](Four& x) {
            x.w = __ldg(reinterpret_cast<const uint4*>(at) + lane);
            x.s = __ldg(reinterpret_cast<const uint2*>(at + 512) + g);
            x.col = __ldg(reinterpret_cast<const int4*>(at + 576));
            at += kFp4FourBytes;
        };
        auto panel = [&](const Four& x, Panel<BT, NT, U>& y, int u0) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = u0 + u, col = k == 0 ? x.col.x : k == 1 ? x.col.y : k == 2 ? x.col.z : x.col.w;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if constexpr (BT == kFp4Rhs) {
                        y.b[u][j].x = __ldg(reinterpret_cast<const uint16_t*>(b0[j] + col / 2));
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            y.q[u][j][e] = __ldg(a.b_scales + dense_scale_at<FMT>((size_t)min(n0 + j * 8 + 2 * t + e, a.N - 1), col, quads));
                    } else {
                        y.b[u][j] = __ldg(reinterpret_cast<const uint2*>(b0[j] + (size_t)col * 2));
                    }
                }
            }
        };
        // `left`: blocks of this four that exist; what stands in the places of the others is zeros, but B may hold anything there.
        auto multiply = [&](const Four& x, Panel<BT, NT, U>& y, int u0, int left) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = u0 + u;
                const uint32_t w = k == 0 ? x.w.x : k == 1 ? x.w.y : k == 2 ? x.w.z : x.w.w, sc = (k < 2 ? x.s.x : x.s.y) >> (k % 2 * 16) & 0xffff;
                uint32_t h[4];
                e2m1x8_to_f16(w, h);
                uint32_t am[4] = {h[0], h[2], h[1], h[3]};
                float s0 = 1.f, s1 = 1.f;
                if constexpr (FOLD) {
                    // the pair of scales of rows 2g and 2g + 1, each in both halves of a word
                    uint32_t s2;
                    if constexpr (FMT == SMAT_FP4_NV) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(s2) : "h"((uint16_t)sc));
                    else asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(s2) : "h"((uint16_t)sc));
                    uint32_t both[2] = {__byte_perm(s2, s2, 0x1010), __byte_perm(s2, s2, 0x3232)};
                    if constexpr (FMT == SMAT_FP4_NV && BT == SMAT_BF16) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&s2));
                        both[0] = pack2<SMAT_BF16>(f.x, f.x);
                        both[1] = pack2<SMAT_BF16>(f.y, f.y);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) am[e] = BT == SMAT_F16 ? mul2<SMAT_F16>(am[e], both[e % 2]) : mul2<SMAT_BF16>(f16_code_to_bf16(am[e], DOWN ? 0x76007600u : 0x77807780u), both[e % 2]);  // 2^109, 2^112
                } else {
                    s0 = scale_value<FMT>(sc & 0xff);
                    s1 = scale_value<FMT>(sc >> 8);
                    if constexpr (DOWN) {
#pragma unroll
                        for (int e = 0; e < 4; e++) am[e] = mul2<SMAT_F16>(am[e], 0x0c000c00u);  // 2^-12
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    uint32_t bx = k < left ? y.b[u][j].x : 0, by = k < left ? y.b[u][j].y : 0;
                    if constexpr (BT == kFp4Rhs) e2m1x4_to_f16((uint16_t)bx, bx, by);
                    if constexpr (FOLD) {
                        mma_16816<BT == SMAT_BF16>(acc[j], am, bx, by, acc[j]);
                    } else {
                        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
                        float d[4];
                        mma_16816<BT == SMAT_BF16>(d, am, bx, by, zero);
                        if constexpr (BT == kFp4Rhs) {
                            const float q0 = k < left ? scale_value<FMT>(y.q[u][j][0]) : 0.f, q1 = k < left ? scale_value<FMT>(y.q[u][j][1]) : 0.f;
                            d[0] *= q0; d[1] *= q1; d[2] *= q0; d[3] *= q1;
                        }
                        acc[j][0] = fmaf(s0, d[0], acc[j][0]);
                        acc[j][1] = fmaf(s0, d[1], acc[j][1]);
                        acc[j][2] = fmaf(s1, d[2], acc[j][2]);
                        acc[j][3] = fmaf(s1, d[3], acc[j][3]);
                    }
                }
            }
        };
        if (hi > lo) {
            // Codes a four ahead (two where the registers hold it), rows of B, which need the columns, a panel ahead.
            constexpr bool DEEP = NT <= 4;
            Four x, y, z;
            load(x);
            if (lo + 1 < hi) load(y); else y = x;
            Panel<BT, NT, U> p[2];
            panel(x, p[0], 0);
            auto four = [&](int i, int left) {
                if (DEEP) {
                    if (i + 2 < hi) load(z); else z = y;
                }
#pragma unroll
                for (int u0 = 0; u0 < 4; u0 += U) {
                    const int cur = u0 / U % 2;
                    if (u0 + U < 4) panel(x, p[cur ^ 1], u0 + U);
                    else panel(y, p[cur ^ 1], 0);
                    multiply(x, p[cur], u0, left);
                }
                if (4 / U % 2) p[0] = p[1];
                x = y;
                if (DEEP) y = z;
                else if (i + 2 < hi) load(y);
            };
            for (int i = lo; i < hi - 1; i++) four(i, 4);
            four(hi - 1, min(4, row.blocks - 4 * (hi - 1)));
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
            if constexpr (DOWN) v *= UP;
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

// Columns in tiles of equal width: 64 at most, 32 of B in 4 bits, whose scales take registers too; as many blocks in a panel as the
// registers hold.
template <int BT, int FMT>
cudaError_t launch_width(const StreamArgs& a, int wr, int cl, cudaStream_t stream) {
    constexpr int most = BT == kFp4Rhs ? 32 : 64;
    const int tiles = (int)(((long long)a.N + most - 1) / most), width = (int)(((long long)a.N + tiles - 1) / tiles);
    switch ((width + 7) / 8) {
        case 1: return launch<BT, FMT, 1, 4>(a, wr, cl, stream);
        case 2: return launch<BT, FMT, 2, 4>(a, wr, cl, stream);
        case 3: return launch<BT, FMT, 3, 2>(a, wr, cl, stream);
        case 4: return launch<BT, FMT, 4, 2>(a, wr, cl, stream);
    }
    if constexpr (BT != kFp4Rhs) {
        switch ((width + 7) / 8) {
            case 5: return launch<BT, FMT, 5, 1>(a, wr, cl, stream);
            case 6: return launch<BT, FMT, 6, 1>(a, wr, cl, stream);
            case 7: return launch<BT, FMT, 7, 1>(a, wr, cl, stream);
            default: return launch<BT, FMT, 8, 1>(a, wr, cl, stream);
        }
    }
    return cudaErrorInvalidValue;  // not reached
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
    a.fours = A.fours;
    a.rows = A.rows;
    a.row_scale = A.row_scale ? A.row_scale + A.brow_begin * 16 : nullptr;
    a.B = B.data;
    a.b_scales = B.scales;
    a.b_row_scale = B.row_scale;
    a.C = C;
    a.c_dtype = c_dtype;
    a.block_rows = (int)A.block_rows;
    a.N = (int)N;
    a.K = A.K;
    // Warps of a block-row: so many that the SMs hold about 32 warps each, but not below 8 blocks a warp.  Measured with B in 16 bits,
    // whose tiles are up to 64 columns wide; of B in 4 bits, with tiles of 32, it counts half the tiles from 33 columns on, and was not
    // measured.
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
