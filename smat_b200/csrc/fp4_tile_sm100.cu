// C = A x B with both in 4 bits, on block-scaled tensor-core MMAs (tcgen05, kind::mxf4nvf4 / kind::mxf4).
//
// Mathematics.  An MMA of M 128, N up to 256 and K 64 multiplies codes, each group of 16 or 32 along k times its scales, into fp32
// accumulators; the fp32 scales of rows and columns are applied to the sums.
//
// Why tiles.  The MMA takes 64 columns at a time and reads a panel of 128 rows of B in 32 cycles whatever it is multiplied with, so
// single 16-row blocks (8 cycles of work) cannot feed it.  Eight block-rows form a tile of 128 rows, laid out by the plan: where
// blocks are absent zeros are multiplied, which costs less than their absence would from a fill of 1/4 of the quads (16 x 64) on.
// Steps of 256 columns in which a group of two tiles holds no block are left out, and so are MMAs of 64 columns without one.  (Laying
// the blocks out in shared memory instead, from the 144 bytes each, was measured first: 950 us for the layer 8192 x 28672 at 20 %,
// N = 4096; the hand-overs between copying, laying out and multiplying warps took 700 cycles a step alone.)
//
// Roles.  One thread fetches the tiles (bulk copies), B (tiled TMA copies with 128-byte swizzle) and its scales; one thread moves the
// scales to tensor memory and issues the MMAs; four warps store finished tiles of C.  The (tile of C, step) pairs are dealt out in
// equal contiguous ranges, one per CTA; tiles that a range boundary falls into are joined from fp32 parts in a fixed order by a
// second kernel.  All waits are bounded.
#include "fp4_device.cuh"
#include "ptx_sm100.cuh"
#include "smat_internal.h"
#include "spmm_sched.cuh"

namespace smat {
namespace {

using namespace ptx;

// ---- tcgen05 with block scales --------------------------------------------------------------------------------------------------
// Instruction descriptor: e2m1 A and B (format 1 in bits [7,10) and [10,13)), N >> 3 in [17,23), bit 23: e8m0 scales (else e4m3),
// M >> 4 in [24,29); bytes 0.. of the scale words are used (scale ids 0).
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n, bool e8m0) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((e8m0 ? 1u : 0u) << 23) | ((uint32_t)(m >> 4) << 24);
}
template <int FMT>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == SMAT_FP4_NV)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}
// 32 rows of 16 bytes (a scale tile of 512 bytes) to four columns of tensor memory, the same in all four lane quarters.
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Descriptor of such a tile: no swizzle, groups of 8 rows x 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t desc_scales(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}
// ---- schedule -------------------------------------------------------------------------------------------------------------------
// Positions: the steps of a tile of C after one another, tiles of a group of block-rows after one another, groups after one another.
struct Work {
    const int* gsp;
    int groups, tiles, parts;
    long long total;
    __device__ __forceinline__ long long first(int g) const { return (long long)__ldg(gsp + g) * tiles; }
    __device__ __forceinline__ int group_of(long long p) const {
        int lo = 0, hi = groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first(mid) <= p) lo = mid; else hi = mid - 1;
        }
        return lo;
    }
    // First position of CTA c's range.  Where a CTA has eight tiles or more its range begins with one: a cut tile goes through
    // memory in fp32, which costs more than being off the equal share by half a tile.
    __device__ __forceinline__ long long begin(int c) const {
        if (c >= parts) return total;
        const long long p = total * c / parts;
        const int g = group_of(p), ns = __ldg(gsp + g + 1) - __ldg(gsp + g);
        if ((long long)ns * 8 * parts > total) return p;
        const long long off = (p - first(g)) % ns;
        return 2 * off <= ns ? p - off : p - off + ns;
    }
};
struct Piece {  // steps [k0, k1) of the ns steps of tile (g, t)
    int g, t, k0, k1, gs, ns, slot;
    bool cut;
};
struct Walk {
    Work w;
    long long p, p_begin, p_end;
    int g;
    __device__ __forceinline__ Walk(const Work& work, int c) : w(work) {
        p = p_begin = w.begin(c);
        p_end = w.begin(c + 1);
        g = p < p_end ? w.group_of(p) : 0;
    }
    __device__ __forceinline__ bool next(Piece& s) {
        if (p >= p_end) return false;
        while (w.first(g + 1) <= p) g++;
        s.g = g;
        s.gs = __ldg(w.gsp + g);
        s.ns = __ldg(w.gsp + g + 1) - s.gs;
        const long long off = p - w.first(g);
        s.t = (int)(off / s.ns);
        s.k0 = (int)(off - (long long)s.t * s.ns);
        const long long left = p_end - p;
        s.k1 = left < s.ns - s.k0 ? s.k0 + (int)left : s.ns;
        s.cut = s.k0 != 0 || s.k1 != s.ns;
        s.slot = 2 * (int)blockIdx.x + (p_begin < p - s.k0 ? 1 : 0);
        p += s.k1 - s.k0;
        return true;
    }
};

struct TileArgs {
    const Fp4Step* steps;
    const uint8_t* tiles;
    const uint8_t* b_scales;
    const float* row_scale;  // first of the range, or null
    const float* b_row_scale;
    void* C;
    float* scratch;
    int* status;
    int c_dtype, rows, N, quads, b_row_tiles, col_tiles;
};

// 16 values of row m from column n on (those below N), scaled, to C.
__device__ __forceinline__ void store_row16(const TileArgs& a, int m, int n, const float (&v)[16]) {
    float o[16];
    const float rs = a.row_scale ? __ldg(a.row_scale + m) : 1.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        o[i] = v[i] * rs;
        if (a.b_row_scale) o[i] *= n + i < a.N ? __ldg(a.b_row_scale + n + i) : 0.f;
    }
    const size_t at = (size_t)m * a.N + n;
    if (a.N % 8 == 0 && n + 16 <= a.N) {
        if (a.c_dtype == SMAT_F16) store16<SMAT_F16>(static_cast<__half*>(a.C) + at, o);
        else store16<SMAT_BF16>(static_cast<__nv_bfloat16*>(a.C) + at, o);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (n + i < a.N) store_c(a.C, a.c_dtype, at + i, o[i]);
    }
}

// NT columns of C per tile.
template <int NT>
struct Cfg {
    static constexpr uint32_t S = NT == 256 ? 4 : NT == 128 ? 6 : NT == 64 ? 7 : 9;  // stages
    static constexpr int BT = NT / 128 > 0 ? NT / 128 : 1;                           // scale tiles of B
    static constexpr uint32_t B_BYTES = NT * 128, SFB_BYTES = 2048 * BT;
    static constexpr uint32_t OFF_SFA = kFp4TileCodes, OFF_B = kFp4TileBytes, OFF_SFB = OFF_B + B_BYTES;
    static constexpr uint32_t STAGE = OFF_SFB + SFB_BYTES;
    static constexpr uint32_t OFF_BAR = S * STAGE;
    static constexpr uint32_t OFF_MASK = OFF_BAR + 8 * (2 * S + 2);
    static constexpr uint32_t OFF_MISC = OFF_MASK + 4 * S;
    static constexpr uint32_t SMEM = OFF_MISC + 12 + 1024;
    static_assert(STAGE % 1024 == 0 && SMEM <= 232448, "shared memory");
};
constexpr int kTileThreads = 8 * 32;

template <int NT, int FMT>
__global__ void __launch_bounds__(kTileThreads, 1) fp4_tile_kernel(const __grid_constant__ CUtensorMap mapB, const TileArgs a, const Work work) {
    using G = Cfg<NT>;
    constexpr uint32_t S = G::S;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto full = [&](uint32_t s) { return base + G::OFF_BAR + 8 * s; };
    auto empty = [&](uint32_t s) { return base + G::OFF_BAR + 8 * (S + s); };
    const uint32_t acc_full = base + G::OFF_BAR + 16 * S, acc_empty = acc_full + 8;
    const uint32_t tmem_slot = base + G::OFF_MISC, abort_addr = tmem_slot + 4, any_addr = tmem_slot + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < S; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        mbar_init(acc_full, 2);
        mbar_init(acc_empty, 4);
        st_shared_u32(abort_addr, 0);
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tensormap(&mapB);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ld_shared_u32(tmem_slot);

    Walk walk(work, (int)blockIdx.x);
    Piece s;
    uint32_t i = 0;  // steps so far

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            while (ok && walk.next(s)) {
                const int half = s.t / a.col_tiles, t = s.t - half * a.col_tiles, rt = t * G::BT;
                const uint32_t b_tiles = (uint32_t)min(G::BT, a.b_row_tiles - rt);
                const uint2* rec = reinterpret_cast<const uint2*>(a.steps + s.gs);
                uint2 next = __ldg(rec + s.k0);
                for (int k = s.k0; k < s.k1; k++, i++) {
                    const uint32_t st = i % S, stage = base + st * G::STAGE, ks = next.x, m = next.y >> (4 * half) & 15;
                    if (k + 1 < s.k1) next = __ldg(rec + k + 1);
                    if (!wait_bar(empty(st), ((i / S) & 1) ^ 1, abort_addr, a.status, 60)) { ok = false; break; }
                    st_shared_u32(base + G::OFF_MASK + 4 * st, m);
                    if (m == 0) { mbar_arrive(full(st)); continue; }  // nothing in this half
                    const uint32_t sf = (uint32_t)min(4, a.quads - (int)ks * 4) * 512;
                    mbar_arrive_expect_tx(full(st), kFp4TileBytes + G::B_BYTES + sf * b_tiles);
                    bulk_load(stage, a.tiles + ((size_t)(s.gs + k) * 2 + half) * kFp4TileBytes, kFp4TileBytes, full(st));
                    tma_load_2d(stage + G::OFF_B, &mapB, (int)ks * 128, t * NT, full(st));
                    for (uint32_t j = 0; j < b_tiles; j++)
                        bulk_load(stage + G::OFF_SFB + 2048 * j, a.b_scales + ((size_t)(rt + j) * a.quads + ks * 4) * 512, sf, full(st));
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp walks, so that what the MMAs are given is uniform; one lane issues.
        constexpr uint32_t idesc = idesc_fp4(128, NT, FMT == SMAT_FP4_MX);
        bool ok = true;
        for (uint32_t n = 0; ok && walk.next(s); n++) {
            ok = __all_sync(~0u, wait_bar(acc_empty, (n & 1) ^ 1, abort_addr, a.status, 61));
            tc_fence_after();
            uint32_t acc = 0;
            for (int k = s.k0; ok && k < s.k1; k++, i++) {
                const uint32_t st = i % S, stage = base + st * G::STAGE;
                ok = __all_sync(~0u, wait_bar(full(st), (i / S) & 1, abort_addr, a.status, 62));
                if (!ok) break;
                tc_fence_after();
                const uint32_t mask = uniform(ld_shared_u32(base + G::OFF_MASK + 4 * st));
                const uint32_t sf = tmem + 256 + (i & 1) * 48;
                const uint64_t da = smem_desc_k_sw128(stage), db = smem_desc_k_sw128(stage + G::OFF_B);
                const uint64_t dsa = desc_scales(stage + G::OFF_SFA), dsb = desc_scales(stage + G::OFF_SFB);
                if (elect_one()) {
                    uint32_t on = acc;
#pragma unroll
                    for (uint32_t q = 0; q < 4; q++) {
                        if (!(mask >> q & 1)) continue;
                        cp_scales(sf + q * 4, dsa + q * 32);
#pragma unroll
                        for (int j = 0; j < G::BT; j++) cp_scales(sf + 16 + q * 8 + j * 4, dsb + q * 32 + j * 128);
                        mma_fp4<FMT>(tmem, da + q * 2, db + q * 2, idesc, sf + q * 4, sf + 16 + q * 8, on);
                        on = 1;
                    }
                    tc_commit(empty(st));
                }
                acc |= mask;
                __syncwarp();
            }
            if (ok && elect_one()) {
                st_shared_u32(any_addr, acc);
                tc_commit(acc_full);
                mbar_arrive(acc_full);
            }
            __syncwarp();
        }
    } else if (warp >= 4 && warp < 8) {
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        const int row = (warp & 3) * 32 + lane;
        for (uint32_t n = 0; walk.next(s); n++) {
            int ok = 1;
            if (lane == 0) ok = wait_bar(acc_full, n & 1, abort_addr, a.status, 63);
            if (!__shfl_sync(~0u, ok, 0)) break;
            tc_fence_after();
            const bool none = ld_shared_u32(any_addr) == 0;  // no MMA wrote the accumulators
            const int half = s.t / a.col_tiles, m = s.g * 256 + half * 128 + row, n0 = (s.t - half * a.col_tiles) * NT, cols = min(NT, a.N - n0);
            float* part = a.scratch + (size_t)s.slot * (128 * NT) + row;
            for (int c = 0; c < cols; c += 16) {
                uint32_t u[16];
                float v[16];
                tmem_ld_x16(lanes + c, u);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = none ? 0.f : __uint_as_float(u[j]);
                if (s.cut) {
#pragma unroll
                    for (int j = 0; j < 16; j++) part[(size_t)(c + j) * 128] = v[j];
                } else if (m < a.rows) {
                    store_row16(a, m, n0 + c, v);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (ld_shared_u32(abort_addr)) {
        // a wait ran out somewhere: give copies still in flight time to land before the CTA retires
        for (int j = 0; j < 64; j++) __nanosleep(1000);
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Adds up the parts of the tiles that a range boundary falls into.  CTA (c - 1, j) looks at the boundary between the ranges of CTAs
// c - 1 and c: if it is the first inside a tile, the tile's 32 columns from 32 j on are summed, the parts in the order of the ranges.
template <int NT>
__global__ void __launch_bounds__(256) fp4_join_kernel(const TileArgs a, const Work work) {
    const int c = (int)blockIdx.x + 1, c0 = (int)blockIdx.y * 32;
    const long long b = work.begin(c);
    const int g = work.group_of(b < work.total ? b : work.total - 1);
    const int ns = __ldg(work.gsp + g + 1) - __ldg(work.gsp + g);
    const int t = (int)((b - work.first(g)) / ns);
    const long long u0 = work.first(g) + (long long)t * ns, u1 = u0 + ns;
    const long long before = work.begin(c - 1);
    if (b >= work.total || b == u0 || before > u0) return;
    const int row = threadIdx.x % 128, h = threadIdx.x / 128;
    const int half = t / a.col_tiles, n0 = (t - half * a.col_tiles) * NT + c0 + h * 16, m = g * 256 + half * 128 + row;
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = 0.f;
    long long p = before;
    for (int k = c - 1; p < u1; k++) {
        const float* part = a.scratch + (size_t)(2 * k + (p < u0 ? 1 : 0)) * (128 * NT) + (size_t)(c0 + h * 16) * 128 + row;
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (n0 + j < a.N) v[j] += __ldg(part + (size_t)j * 128);
        p = work.begin(k + 1);
    }
    if (m < a.rows && n0 < a.N) store_row16(a, m, n0, v);
}

template <int NT, int FMT>
int launch_tile(const TileArgs& args, const CUtensorMap& map, Work work, size_t total, const DeviceCtx* ctx, cudaStream_t stream) {
    using G = Cfg<NT>;
    TileArgs a = args;
    const cudaError_t attr = cudaFuncSetAttribute(fp4_tile_kernel<NT, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
    if (attr != cudaSuccess) return fail(SMAT_ERR_CUDA, "cudaFuncSetAttribute failed: %s", cudaGetErrorString(attr));
    a.col_tiles = (a.N + NT - 1) / NT;
    work.tiles = 2 * a.col_tiles;  // of each half of a group
    work.total = (long long)total * work.tiles;
    // a CTA for every SM, but not below four steps each
    work.parts = (int)(work.total / 4 < ctx->sm_count ? (work.total / 4 > 0 ? work.total / 4 : 1) : ctx->sm_count);
    void* scratch = nullptr;
    if (work.parts > 1) {
        SMAT_CUDA_TRY(cudaMallocFromPoolAsync(&scratch, (size_t)work.parts * 2 * 128 * NT * sizeof(float), ctx->pool, stream));
        a.scratch = static_cast<float*>(scratch);
    }
    fp4_tile_kernel<NT, FMT><<<work.parts, kTileThreads, G::SMEM, stream>>>(map, a, work);
    cudaError_t e = cudaGetLastError();
    count_launch();
    if (e == cudaSuccess && work.parts > 1) {
        fp4_join_kernel<NT><<<dim3(work.parts - 1, NT / 32), 256, 0, stream>>>(a, work);
        e = cudaGetLastError();
        count_launch();
    }
    const cudaError_t f = scratch ? cudaFreeAsync(scratch, stream) : cudaSuccess;
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return fail(SMAT_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return SMAT_OK;
}

template <int NT>
int launch_tile_format(int fmt, const TileArgs& a, const CUtensorMap& map, const Work& work, size_t total, const DeviceCtx* ctx, cudaStream_t stream) {
    return fmt == SMAT_FP4_NV ? launch_tile<NT, SMAT_FP4_NV>(a, map, work, total, ctx, stream)
                              : launch_tile<NT, SMAT_FP4_MX>(a, map, work, total, ctx, stream);
}

}  // namespace

int launch_fp4_tile(const Fp4View& A, const Fp4Rhs& B, void* C, int c_dtype, size_t N, cudaStream_t stream) {
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    const int nt = N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
    CUtensorMap map;
    const size_t pitch = fp4_pitch(A.K);
    if (int rc = encode_tensor_map_2d_u8(&map, B.data, pitch, N, pitch, 128, (uint32_t)nt)) return rc;
    TileArgs a = {};
    a.steps = A.steps;
    a.tiles = A.tiles;
    a.b_scales = B.scales;
    a.row_scale = A.row_scale ? A.row_scale + A.brow_begin * 16 : nullptr;
    a.b_row_scale = B.row_scale;
    a.C = C;
    a.status = ctx->d_status;
    a.c_dtype = c_dtype;
    a.rows = (int)(A.block_rows * 16);
    a.N = (int)N;
    a.quads = (int)fp4_quads(A.K);
    a.b_row_tiles = (int)((N + 127) / 128);
    Work work = {};
    work.gsp = A.gsp;
    work.groups = (int)((A.block_rows + kFp4GroupRows - 1) / kFp4GroupRows);
    switch (nt) {
        case 32: return launch_tile_format<32>(A.fmt, a, map, work, A.total_steps, ctx, stream);
        case 64: return launch_tile_format<64>(A.fmt, a, map, work, A.total_steps, ctx, stream);
        case 128: return launch_tile_format<128>(A.fmt, a, map, work, A.total_steps, ctx, stream);
        default: return launch_tile_format<256>(A.fmt, a, map, work, A.total_steps, ctx, stream);
    }
}

}  // namespace smat
