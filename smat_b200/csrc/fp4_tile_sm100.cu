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
// Beyond 128 columns of C two CTAs share a tile of 256 x 256 (cta_group::2): each holds 128 rows of A and 128 columns of B, so an SM
// fetches 38 KB a step of 512 cycles of MMAs instead of 54; L2 delivers about 70 bytes a cycle and SM.
//
// Roles.  One thread fetches tiles of A (bulk copies, of a pair tiled ones), B (tiled TMA copies with 128-byte swizzle) and its scales; four warps move the
// scales to tensor memory through registers (tcgen05.cp, 12 of them a step, took their issuer 24 cycles each in a CTA of its own and
// 140 in a pair); one thread issues the MMAs; eight warps store finished tiles of C through shared memory, whole 128-byte lines at a
// time.  Of a pair, the second CTA issues no MMAs.
//
// Measured: layer 8192 x 28672 at 20 %, N = 4096, 342 us, steps of 640 cycles (512 of MMAs) at 1.6 GHz, the power limit; that is 5.6
// PFLOP/s with the zeros, 1.12 without.  All waits are bounded.
#include <algorithm>
#include <type_traits>

#include "fp4_device.cuh"
#include "ptx_sm100.cuh"
#include "smat_internal.h"
#include "spmm_sched.cuh"

namespace smat {
namespace {

using namespace ptx;

// ---- tcgen05 with block scales; CG: CTAs of the group (cta_group::1 or ::2) -----------------------------------------------------
// Instruction descriptor: e2m1 A and B (format 1 in bits [7,10) and [10,13)), N >> 3 in [17,23), bit 23: e8m0 scales (else e4m3),
// M >> 4 in [24,29); bytes 0.. of the scale words are used (scale ids 0).
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n, bool e8m0) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((e8m0 ? 1u : 0u) << 23) | ((uint32_t)(m >> 4) << 24);
}
template <int FMT, int CG>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
#define SMAT_MMA_FP4(cg, kind)                                                                                  \
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"     \
                 "setp.ne.b32 p, %8, 0;\n\t"                                                                     \
                 "tcgen05.mma.cta_group::" cg ".kind::" kind " [%0], da, db, %5, [%6], [%7], p;\n\t}" ::"r"(d),  \
                 "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)     \
                 : "memory")
    if constexpr (FMT == SMAT_FP4_NV && CG == 1) SMAT_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (FMT == SMAT_FP4_NV) SMAT_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (CG == 1) SMAT_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
    else SMAT_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
#undef SMAT_MMA_FP4
}
// Arrives on this CTA's barrier, of a pair on that of both, once every tcgen05 operation issued so far by this thread has completed.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CG == 1) tc_commit(bar);
    else
        asm volatile(
            "{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void alloc_all(uint32_t dst_smem) {
    if constexpr (CG == 1) {
        tmem_alloc(dst_smem, 512);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst_smem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void dealloc_all(uint32_t taddr) {
    if constexpr (CG == 1) tmem_dealloc(taddr, 512);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}

// ---- the two CTAs of a pair -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// Arrives on the barrier at the same place of the first CTA's shared memory.  Only for what lies in tensor memory, which is ordered by the
// tcgen05 fences around arrival and wait and needs no release at cluster scope (700 to 900 cycles).  Shared memory of the second CTA is
// announced by the copies that fill it: they complete on the first CTA's barrier.
__device__ __forceinline__ void arrive_at_first(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, 0;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [r];\n\t}" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Stores under a predicate, without a branch.
__device__ __forceinline__ void store_if(bool on, uint16_t* p, uint32_t v) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.u32 [%0], %1;\n\t}" ::"l"(p), "r"(v), "r"((uint32_t)on) : "memory");
}
__device__ __forceinline__ void store_if(bool on, uint16_t* p, uint4 v) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t@q st.global.v4.u32 [%0], {%1, %2, %3, %4};\n\t}" ::"l"(p), "r"(v.x),
                 "r"(v.y), "r"(v.z), "r"(v.w), "r"((uint32_t)on)
                 : "memory");
}
__device__ __forceinline__ void store_if(bool on, uint16_t* p, uint16_t v) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.u16 [%0], %1;\n\t}" ::"l"(p), "h"(v), "r"((uint32_t)on) : "memory");
}
// Writes 16 consecutive columns of the calling thread's lane.
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint4* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w), "r"(v[2].x), "r"(v[2].y),
        "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w)
        : "memory");
}

// ---- schedule -------------------------------------------------------------------------------------------------------------------
// Units: tiles of C, those of a group of block-rows one after another.  The first `rounds` units of a part (a CTA or pair) are dealt out
// one by one, so that all parts walk the columns in step and L2 serves what several of them read (in contiguous ranges from the start,
// the layer 8192 x 28672 at 20 %, N = 4096, fetched everything from HBM: 830 us).  What is left is one contiguous range for each part,
// from one start to the next; units that a start falls into are joined from fp32 sums in a fixed order by a second kernel.  Worked out
// on the host and handed over as a kernel parameter: looked up on the device, five dependent loads at a time, it took 7 us of every
// launch and 18 us of the joining kernel.
struct Start {
    int g, t, k;  // group, unit of the group, step of the unit
};
constexpr int kMaxParts = 160;
struct Schedule {
    Start at[kMaxParts + 1];
    int parts, units, rounds;  // units: of a group
};
struct Piece {  // steps [k0, k1) of the ns steps of unit (g, t)
    int g, t, k0, k1, gs, ns, slot;
    bool cut;
};
struct Walk {
    const int* gsp;
    Start now, end;
    int units, parts, slot, unit, left;
    __device__ __forceinline__ Walk(const Schedule& s, const int* first_steps, int part)
        : gsp(first_steps), now(s.at[part]), end(s.at[part + 1]), units(s.units), parts(s.parts), slot(2 * part), unit(part), left(s.rounds) {}
    __device__ __forceinline__ void look_up(Piece& p, int g, int t) const {
        p.g = g;
        p.t = t;
        p.gs = __ldg(gsp + g);
        p.ns = __ldg(gsp + g + 1) - p.gs;
    }
    __device__ __forceinline__ bool next(Piece& p) {
        if (left) {
            look_up(p, unit / units, unit % units);
            p.k0 = 0;
            p.k1 = p.ns;
            p.cut = false;
            p.slot = 0;
            unit += parts;
            left--;
            return true;
        }
        const bool last = now.g == end.g && now.t == end.t;
        if (last && now.k == end.k) return false;
        look_up(p, now.g, now.t);
        p.k0 = now.k;
        p.k1 = last ? end.k : p.ns;
        p.cut = p.k0 != 0 || p.k1 != p.ns;
        p.slot = slot;
        slot |= 1;  // for a unit that begins inside the range
        now.k = last ? end.k : 0;
        if (!last && ++now.t == units) { now.t = 0; now.g++; }
        return true;
    }
};

// Step words, read by a warp 32 at a time and 32 ahead: one at a time, each iteration of a loop waited 800 cycles for its own.
struct Records {
    const uint32_t* p;
    int last, base;
    uint32_t cur, next;
    __device__ __forceinline__ Records(const uint32_t* steps, int n) : p(steps), last(n - 1), base(-64) {}
    __device__ __forceinline__ uint32_t load(int b) const { return __ldg(p + min(b + (int)(threadIdx.x & 31), last)); }
    __device__ __forceinline__ uint32_t get(int at) {  // by all lanes; uniform
        if ((unsigned)(at - base) >= 32) {
            if ((unsigned)(at - base) < 64) {
                cur = next;
                base += 32;
            } else {
                base = at;
                cur = load(base);
            }
            next = load(base + 32);
        }
        return uniform((int)(threadIdx.x & 31) == at - base ? cur : 0);
    }
};

struct TileArgs {
    const uint32_t* steps;
    const uint8_t* tiles;
    const int* gsp;
    const uint8_t* b_scales;
    const float* row_scale;  // first of the range, or null
    const float* b_row_scale;
    void* C;
    float* scratch;
    int* status;
    int c_dtype, rows, N, quads, b_row_tiles, col_tiles, total_steps;
    uint32_t lost_bytes;  // expected but not copied, by the self-test of giving up
    long long wait_cycles;
};

// NT columns of C per tile; a pair of CTAs (CG 2) for 256.
template <int NT>
struct Cfg {
    static constexpr int CG = NT == 256 ? 2 : 1;
    static constexpr uint32_t S = NT == 64 ? 6 : NT == 32 ? 7 : 5;  // stages of codes
    static constexpr uint32_t Q = NT == 256 ? 4 : 6;                // stages of scales on their way to tensor memory; see `arrived`
    static constexpr uint32_t NB = NT / CG;                         // columns of C whose part of B this CTA fetches
    static constexpr int BT = NT > 128 ? NT / 128 : 1;              // scale tiles of B
    static constexpr uint32_t OFF_B = kFp4TileCodes, STAGE = OFF_B + NB * 128;
    static constexpr uint32_t SF_STAGE = 2048 + 2048 * BT, SF_COLUMNS = 16 + 16 * BT;  // in shared and in tensor memory
    static constexpr uint32_t ACC = NT == 256 ? 1 : 2;              // accumulators
    static constexpr uint32_t OFF_SF = S * STAGE;
    static constexpr uint32_t OFF_OUT = OFF_SF + Q * SF_STAGE;      // 32 rows x 64 columns for each storing warp
    static constexpr uint32_t OFF_COL = OFF_OUT + 8 * 4096;         // and the scales of these columns
    static constexpr uint32_t OFF_BAR = OFF_COL + 8 * 256;
    static constexpr uint32_t OFF_MISC = OFF_BAR + 8 * (2 * S + 2 * Q + 4);
    static constexpr uint32_t SMEM = OFF_MISC + 16 + 1024;
    static_assert(STAGE % 1024 == 0 && Q % 2 == 0 && SMEM <= 232448, "shared memory");
    static_assert(ACC * NT <= 256 && 256 + S * SF_COLUMNS <= 512, "tensor memory");
};
constexpr int kTileThreads = 20 * 32;

template <int NT, int FMT>
__global__ void __launch_bounds__(kTileThreads, 1)
fp4_tile_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ TileArgs a,
                const __grid_constant__ Schedule plan) {
    using G = Cfg<NT>;
    constexpr uint32_t S = G::S;
    constexpr int CG = G::CG;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar = base + G::OFF_BAR;
    // A step's codes have arrived and its scales are in tensor memory, of both CTAs: one barrier, the first CTA's, since each wait takes
    // the MMAs' thread 130 cycles.  The second CTA's codes complete on it as well, which releases them at cluster scope; the MMAs' warp
    // acquires there.  (Layer 8192 x 28672 at 20 %, N = 4096: 342 us.  With a warp of the second CTA that waits for its codes and announces
    // them with a releasing arrival: 797.)
    auto ready = [&](uint32_t s) { return bar + 8 * s; };
    auto empty = [&](uint32_t s) { return bar + 8 * (S + s); };  // ... and have been used
    // Scales in shared memory.  Two sets of warps wait for them in turn, and each must see every phase of a barrier that it waits for
    // by parity, so the stages are an even number.
    auto arrived = [&](uint32_t s) { return bar + 8 * (2 * S + s); };
    auto taken = [&](uint32_t s) { return bar + 8 * (2 * S + G::Q + s); };
    auto acc_full = [&](uint32_t b) { return bar + 8 * (2 * S + 2 * G::Q + b); };
    auto acc_empty = [&](uint32_t b) { return bar + 8 * (2 * S + 2 * G::Q + 2 + b); };
    const uint32_t tmem_slot = base + G::OFF_MISC, abort_addr = tmem_slot + 4, any_addr = tmem_slot + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? uniform(cluster_rank()) : 0;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < S; s++) { mbar_init(ready(s), 1 + 4 * CG); mbar_init(empty(s), 1); }
        for (uint32_t s = 0; s < G::Q; s++) { mbar_init(arrived(s), 1); mbar_init(taken(s), 4); }
        for (uint32_t b = 0; b < 2; b++) { mbar_init(acc_full(b), CG == 1 ? 2 : 1); mbar_init(acc_empty(b), 8 * CG); }
        st_shared_u32(abort_addr, 0);
        fence_barrier_init();
        fence_proxy_async();
        if (CG == 2) prefetch_tensormap(&mapA);
        prefetch_tensormap(&mapB);
    }
    if (warp == 1) alloc_all<CG>(tmem_slot);
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = uniform(ld_shared_u32(tmem_slot));

    Walk walk(plan, a.gsp, (int)blockIdx.x / CG);
    Piece s;
    uint32_t i = 0;  // steps so far

    // Half of the group and tile column of a unit; a pair takes both halves.
    auto half_of = [&](int t) { return CG == 2 ? (int)rank : t / a.col_tiles; };
    auto column_of = [&](int t) { return CG == 2 ? t : t % a.col_tiles; };

    // Quads of a step that hold blocks, for a pair in either half.
    auto quads_of = [&](uint32_t rec, int half) { return CG == 2 ? (rec | rec >> 4) & 15 : rec >> (4 * half) & 15; };

    // What decides on addresses is made uniform, and one elected lane issues: otherwise every copy costs its warp 100 cycles for
    // bringing its operands into uniform registers lane by lane, and the loops below take 800 cycles a step.
    if (warp == 0) {
        // Codes.
        Records records(a.steps, a.total_steps);
        bool ok = true;
        uint32_t st = 0, phase = 1;
        while (ok && walk.next(s)) {
            const int half = (int)uniform(half_of(s.t)), gs = (int)uniform(s.gs), k1 = (int)uniform(s.k1);
            const int row = (int)uniform(column_of(s.t)) * NT + (CG == 2 ? (int)(rank * G::NB) : 0);
            const uint8_t* tile = a.tiles + ((size_t)(gs + (int)uniform(s.k0)) * 2 + half) * kFp4TileBytes;
            for (int k = (int)uniform(s.k0); k < k1; k++, tile += 2 * kFp4TileBytes) {
                const uint32_t rec = records.get(gs + k), stage = base + st * G::STAGE;
                ok = __all_sync(~0u, wait_bar(empty(st), phase, abort_addr, a.status, 60, a.wait_cycles));
                if (!ok) break;
                if (elect_one()) {
                    if (quads_of(rec, half) == 0) {  // no blocks here, of a pair in neither half
                        if (rank == 0) mbar_arrive(ready(st));
                    } else if constexpr (CG == 1) {
                        mbar_arrive_expect_tx(ready(st), G::STAGE + a.lost_bytes);
                        bulk_load(stage, tile, kFp4TileCodes, ready(st));
                        tma_load_2d(stage + G::OFF_B, &mapB, (int)(rec >> 8) * 128, row, ready(st));
                    } else {
                        // Copies of the second CTA may complete before the first expects them: the phase ends with the first one's arrival.
                        const uint32_t first = pair_bar(ready(st), 0);
                        if (rank == 0) mbar_arrive_expect_tx(ready(st), 2 * G::STAGE + a.lost_bytes);
                        tma_load_2d_pair(stage, &mapA, 0, ((gs + k) * 2 + half) * (int)(kFp4TileBytes / 128), first);
                        tma_load_2d_pair(stage + G::OFF_B, &mapB, (int)(rec >> 8) * 128, row, first);
                    }
                }
                __syncwarp();
                if (++st == S) { st = 0; phase ^= 1; }
            }
        }
    } else if (warp == 2) {
        // Scales.
        Records records(a.steps, a.total_steps);
        bool ok = true;
        uint32_t st = 0, phase = 1;
        while (ok && walk.next(s)) {
            const int half = (int)uniform(half_of(s.t)), gs = (int)uniform(s.gs), k1 = (int)uniform(s.k1), rt = (int)uniform(column_of(s.t)) * G::BT;
            const uint32_t b_tiles = (uint32_t)min(G::BT, a.b_row_tiles - rt);
            const uint8_t* tile = a.tiles + ((size_t)(gs + (int)uniform(s.k0)) * 2 + half) * kFp4TileBytes + kFp4TileCodes;
            const uint8_t* panel = a.b_scales + (size_t)rt * a.quads * 512;
            for (int k = (int)uniform(s.k0); k < k1; k++, tile += 2 * kFp4TileBytes) {
                const uint32_t rec = records.get(gs + k), stage = base + G::OFF_SF + st * G::SF_STAGE, quad = (rec >> 8) * 4;
                const uint32_t bytes = min(4u, (uint32_t)a.quads - quad) * 512;
                ok = __all_sync(~0u, wait_bar(taken(st), phase, abort_addr, a.status, 61, a.wait_cycles));
                if (!ok) break;
                if (elect_one()) {
                    if (quads_of(rec, half) == 0) {
                        mbar_arrive(arrived(st));
                    } else {
                        mbar_arrive_expect_tx(arrived(st), 2048 + bytes * b_tiles);
                        bulk_load(stage, tile, 2048, arrived(st));
                        bulk_load(stage + 2048, panel + (size_t)quad * 512, bytes, arrived(st));
                        if (G::BT == 2 && b_tiles == 2) bulk_load(stage + 4096, panel + ((size_t)a.quads + quad) * 512, bytes, arrived(st));
                    }
                }
                __syncwarp();
                if (++st == G::Q) { st = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1 && rank == 0) {
        // The whole warp walks, so that what the MMAs are given is uniform; one lane issues.
        constexpr uint32_t idesc = idesc_fp4(128 * CG, NT, FMT == SMAT_FP4_MX);
        const uint64_t da0 = smem_desc_k_sw128(base), db0 = smem_desc_k_sw128(base + G::OFF_B);
        const uint32_t da_hi = (uint32_t)(da0 >> 32), db_hi = (uint32_t)(db0 >> 32);
        Records records(a.steps, a.total_steps);
        bool ok = true;
        uint32_t st = 0, phase = 0, n = 0;
        for (; ok && walk.next(s); n++) {
            const uint32_t buf = n % G::ACC;
            const int half = (int)uniform(half_of(s.t)), gs = (int)uniform(s.gs), k1 = (int)uniform(s.k1);
            ok = __all_sync(~0u, wait_bar(acc_empty(buf), ((n / G::ACC) & 1) ^ 1, abort_addr, a.status, 62, a.wait_cycles));
            tc_fence_after();
            uint32_t acc = 0;
            for (int k = (int)uniform(s.k0); ok && k < k1; k++) {
                const uint32_t mask = quads_of(records.get(gs + k), half);
                const uint32_t sf = tmem + 256 + st * G::SF_COLUMNS;
                const uint32_t da = (uint32_t)da0 + st * (G::STAGE >> 4), db = (uint32_t)db0 + st * (G::STAGE >> 4);
                ok = __all_sync(~0u, wait_bar<CG == 2>(ready(st), phase, abort_addr, a.status, 63, a.wait_cycles));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    uint32_t on = acc;
#pragma unroll
                    for (uint32_t q = 0; q < 4; q++) {
                        if (!(mask >> q & 1)) continue;
                        mma_fp4<FMT, CG>(tmem + buf * NT, da + q * 2, da_hi, db + q * 2, db_hi, idesc, sf + q * 4, sf + 16 + q * 4 * G::BT, on);
                        on = 1;
                    }
                    commit<CG>(empty(st));
                }
                acc |= mask;
                if (++st == S) { st = 0; phase ^= 1; }
                __syncwarp();
            }
            if (ok && elect_one()) {
                if (CG == 1) st_shared_u32(any_addr + 4 * buf, acc);
                commit<CG>(acc_full(buf));
                if (CG == 1) mbar_arrive(acc_full(buf));
            }
            __syncwarp();
        }
    } else if (warp >= 12) {
        // Scales to tensor memory, as soon as the MMAs have used what is there: four words a lane and scale tile, the same in all lane
        // quarters.  A set of four warps takes every other step.
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21) + 256;
        uint32_t steps = 0;
        while (walk.next(s)) steps += (uint32_t)(s.k1 - s.k0);
        for (i = (uint32_t)(warp - 12) / 4; i < steps; i += 2) {
            const uint32_t st = i % S, from = base + G::OFF_SF + i % G::Q * G::SF_STAGE + lane * 16;
            if (!__all_sync(~0u, wait_bar(arrived(i % G::Q), (i / G::Q) & 1, abort_addr, a.status, 67, a.wait_cycles) &&
                                     wait_bar(empty(st), ((i / S) & 1) ^ 1, abort_addr, a.status, 68, a.wait_cycles)))
                break;
            tc_fence_after();
            uint4 v[4 + 4 * G::BT];
#pragma unroll
            for (int q = 0; q < 4; q++) v[q] = ld_shared_v4(from + q * 512);
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int j = 0; j < G::BT; j++) v[4 + q * G::BT + j] = ld_shared_v4(from + 2048 * (1 + j) + q * 512);
            const uint32_t to = lanes + st * G::SF_COLUMNS;
#pragma unroll
            for (int j = 0; j < 1 + G::BT; j++) tmem_st_x16(to + 16 * j, v + 4 * j);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2 && rank == 1) arrive_at_first(ready(st));
                else mbar_arrive(ready(st));
                mbar_arrive(taken(i % G::Q));
            }
        }
    } else if (warp >= 4) {
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), out = base + G::OFF_OUT + (uint32_t)(warp - 4) * 4096;
        const uint32_t col = base + G::OFF_COL + (uint32_t)(warp - 4) * 256;
        const int row0 = (warp & 3) * 32, c0 = (warp - 4) / 4 * 64;  // rows and first columns of this warp
        // What the next unit needs is looked up before this one is stored.
        Piece f = {};
        float rs, cs[NT == 256 ? 2 : 1][2];
        auto look_up = [&]() {
            const int m = f.g * 256 + half_of(f.t) * 128 + row0 + lane, n = column_of(f.t) * NT + c0 + lane;
            rs = a.row_scale && m < a.rows ? __ldg(a.row_scale + m) : 1.f;
#pragma unroll
            for (int j = 0; j < (NT == 256 ? 2 : 1); j++)
#pragma unroll
                for (int e = 0; e < 2; e++) cs[j][e] = a.b_row_scale && n + j * 128 + e * 32 < a.N ? __ldg(a.b_row_scale + n + j * 128 + e * 32) : 1.f;
            // of a pair, only the one step of an empty group has no MMA
            f.k0 = CG == 2 && f.ns == 1 && (__ldg(a.steps + f.gs) & 0xff) == 0;
        };
        bool more = walk.next(f);
        if (more) look_up();
        for (uint32_t n = 0; more; n++) {
            const uint32_t buf = n % G::ACC;
            s = f;
            const int m0 = s.g * 256 + half_of(s.t) * 128 + row0, n0 = column_of(s.t) * NT, cols = min(NT, a.N - n0);
            if (!__all_sync(~0u, wait_bar(acc_full(buf), (n / G::ACC) & 1, abort_addr, a.status, 69, a.wait_cycles))) break;
            tc_fence_after();
            const bool none = CG == 1 ? ld_shared_u32(any_addr + 4 * buf) == 0 : s.k0 != 0;  // no MMA wrote the accumulators
            auto release = [&]() {  // all of this warp's accumulators are read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2 && rank == 1) arrive_at_first(acc_empty(buf));
                    else mbar_arrive(acc_empty(buf));
                }
            };
            if (s.cut) {
                float* to = a.scratch + (size_t)s.slot * (128 * CG * NT) + (CG == 2 ? (int)rank * 128 : 0) + row0 + lane;
                for (int c = c0; c < cols; c += 128)
                    for (int j0 = c; j0 < min(c + 64, cols); j0 += 16) {
                        uint32_t u[16];
                        tmem_ld_x16(lanes + buf * NT + j0, u);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; j++) to[(size_t)(j0 + j) * (128 * CG)] = none ? 0.f : __uint_as_float(u[j]);
                    }
                release();
                more = walk.next(f);
                if (more) look_up();
                continue;
            }
            // 64 columns at a time: scaled, rounded, through shared memory and out.  Of 256 columns (one accumulator) the second half
            // is taken into registers before the first is stored, so that the next unit's MMAs need not wait for that.
            constexpr int W = NT < 64 ? NT : 64;
            auto take = [&](int jc, auto type, auto&& sink) {  // sink(j, words): columns j to j + 31 of the 64
                st_shared_u32(col + lane * 4, __float_as_uint(cs[jc][0]));
                st_shared_u32(col + lane * 4 + 128, __float_as_uint(cs[jc][1]));
                __syncwarp();
#pragma unroll
                for (int j0 = 0; j0 < W; j0 += 32) {
                    uint32_t u[2][16], w[16];
                    tmem_ld_x16(lanes + buf * NT + c0 + jc * 128 + j0, u[0]);
                    tmem_ld_x16(lanes + buf * NT + c0 + jc * 128 + j0 + 16, u[1]);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t* q = u[j / 4] + 4 * (j % 4);
                        const uint4 by = ld_shared_v4(col + (j0 + 4 * j) * 4);
                        w[2 * j] = pack2<decltype(type)::value>(__uint_as_float(q[0]) * rs * __uint_as_float(by.x), __uint_as_float(q[1]) * rs * __uint_as_float(by.y));
                        w[2 * j + 1] = pack2<decltype(type)::value>(__uint_as_float(q[2]) * rs * __uint_as_float(by.z), __uint_as_float(q[3]) * rs * __uint_as_float(by.w));
                    }
                    if (none) {
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = 0;
                    }
                    sink(j0, w);
                }
                __syncwarp();
            };
            auto put = [&](int j0, const uint32_t* w) {
#pragma unroll
                for (int j = 0; j < 4; j++) st_shared_v4(out + lane * 128 + (((j0 / 8 + j) ^ (lane & 7)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            };
            auto store = [&](int jc) {
                const int c = c0 + jc * 128;
                __syncwarp();
                const int width = min(64, cols - c);
                uint16_t* const to = static_cast<uint16_t*>(a.C) + (size_t)m0 * a.N + n0 + c;
                if (a.N % 8 == 0) {  // eight lanes a row
#pragma unroll
                    for (int r0 = 0; r0 < 32; r0 += 4) {
                        const int r = r0 + lane / 8, j = lane % 8;
                        const uint4 v = ld_shared_v4(out + r * 128 + ((j ^ (r & 7)) << 4));
                        store_if(m0 + r < a.rows && j * 8 < width, to + (size_t)r * a.N + j * 8, v);
                    }
                } else {
                    // Rows begin anywhere: a warp a row, two columns a lane from the first even address on.  (One column at a time took
                    // 20000 cycles a tile.)
                    for (int r0 = 0; r0 < 32; r0 += 8) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) w[i] = ld_shared_u32(out + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            uint16_t* const row = to + (size_t)(r0 + i) * a.N;
                            const int odd = (int)((uintptr_t)row >> 1 & 1), j = 2 * lane + odd;
                            const uint32_t after = __shfl_down_sync(~0u, w[i], 1), v = odd ? w[i] >> 16 | after << 16 : w[i];
                            const bool in = m0 + r0 + i < a.rows;
                            store_if(in && j + 1 < width, row + j, v);
                            store_if(in && j + 1 == width, row + j, (uint16_t)v);
                            store_if(in && odd && lane == 0, row, (uint16_t)w[i]);
                        }
                    }
                }
                __syncwarp();
            };
            uint32_t second[NT == 256 ? 32 : 1];
            auto take_all = [&](auto type) {
                if (NT == 256 && c0 + 128 < cols)
                    take(1, type, [&](int j0, const uint32_t* w) {
#pragma unroll
                        for (int j = 0; j < 16; j++) second[(j0 / 2 + j) % (NT == 256 ? 32 : 1)] = w[j];
                    });
                if (c0 < cols) take(0, type, put);
            };
            if (a.c_dtype == SMAT_F16) take_all(std::integral_constant<int, SMAT_F16>());
            else take_all(std::integral_constant<int, SMAT_BF16>());
            release();
            more = walk.next(f);
            if (more) look_up();
            if (c0 < cols) store(0);
            if (NT == 256 && c0 + 128 < cols) {
#pragma unroll
                for (int j0 = 0; j0 < 64; j0 += 32) put(j0, second + j0 / 2 % (NT == 256 ? 32 : 1));
                store(1);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (ld_shared_u32(abort_addr)) {
        // a wait ran out somewhere: give copies still in flight time to land before the CTA retires
        for (int j = 0; j < 64; j++) __nanosleep(1000);
    }
    if (CG == 2) cluster_sync();  // the MMAs read both CTAs' shared memory
    if (warp == 1) {
        tc_fence_after();
        dealloc_all<CG>(tmem);
    }
}

// Units that a start falls into, and the scratch slots of their parts in order.  Listed on the host: found on the device, from dozens of
// dependent reads of the schedule, they took the joining kernel 15 of its 19 us.
struct Joins {
    Start unit[kMaxParts];
    short first[kMaxParts + 1], slot[3 * kMaxParts];
    int n;
};
void list_joins(const Schedule& s, Joins& j) {
    j.n = 0;
    int used = 0;
    for (int c = 1; c < s.parts; c++) {
        const Start b = s.at[c], before = s.at[c - 1];
        const bool same = before.g == b.g && before.t == b.t;
        if (b.k == 0 || (same && before.k != 0)) continue;  // no cut, or not the first in this unit
        j.unit[j.n] = b;
        j.first[j.n++] = (short)used;
        j.slot[used++] = (short)(2 * (c - 1) + (same ? 0 : 1));
        int k = c;
        do {
            const Start from = s.at[k], to = s.at[k + 1];
            if (from.k != to.k || from.g != to.g || from.t != to.t) j.slot[used++] = (short)(2 * k);  // not an empty range
        } while (++k < s.parts && s.at[k].g == b.g && s.at[k].t == b.t);
    }
    j.first[j.n] = (short)used;
}

// Adds up the parts of cut units in the order of the ranges.  CTA (i, j): kJoinColumns columns of the i-th, a thread 16 of a row; the
// loads of a round are independent and under no condition (with one each, they came one after the other: 24 instead of 5 us).
template <int NT>
constexpr int kJoinColumns = 32 / Cfg<NT>::CG;
template <int NT>
__global__ void __launch_bounds__(256) fp4_join_kernel(const __grid_constant__ TileArgs a, const __grid_constant__ Joins joins) {
    constexpr int CG = Cfg<NT>::CG, ROWS = 128 * CG, COLS = kJoinColumns<NT>, PITCH = COLS * 2 + 16;  // bytes of a row in shared memory
    const Start b = joins.unit[blockIdx.x];
    const int k0 = joins.first[blockIdx.x], k1 = joins.first[blockIdx.x + 1];
    const int n0 = (CG == 2 ? b.t : b.t % a.col_tiles) * NT + (int)blockIdx.y * COLS, cols = min(COLS, a.N - n0);
    const int m0 = b.g * 256 + (CG == 2 ? 0 : b.t / a.col_tiles * 128), row = threadIdx.x % ROWS, c0 = threadIdx.x / ROWS * 16;
    if (cols <= 0) return;
    __shared__ alignas(16) uint8_t tile[ROWS * PITCH];
    float v[16], by[16];
    const float rs = a.row_scale && m0 + row < a.rows ? __ldg(a.row_scale + m0 + row) : 1.f;
#pragma unroll
    for (int j = 0; j < 16; j++) {
        v[j] = 0.f;
        by[j] = 1.f;
    }
    if (a.b_row_scale) {
#pragma unroll
        for (int j = 0; j < 16; j++) by[j] = __ldg(a.b_row_scale + min(n0 + c0 + j, a.N - 1));
    }
    const float* src = a.scratch + ((size_t)blockIdx.y * COLS + c0) * ROWS + row;
    for (int k = k0; k < k1; k++) {
        const float* p = src + (size_t)joins.slot[k] * (ROWS * NT);
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] += __ldg(p + j * ROWS);  // columns beyond N hold anything, and go nowhere
    }
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = v[2 * j] * rs * by[2 * j], y = v[2 * j + 1] * rs * by[2 * j + 1];
        w[j] = a.c_dtype == SMAT_F16 ? pack2<SMAT_F16>(x, y) : pack2<SMAT_BF16>(x, y);
    }
    *reinterpret_cast<uint4*>(tile + row * PITCH + c0 * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(tile + row * PITCH + c0 * 2 + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    __syncthreads();
    uint16_t* const to = static_cast<uint16_t*>(a.C) + (size_t)m0 * a.N + n0;
    if (a.N % 8 == 0) {
#pragma unroll
        for (int j = threadIdx.x; j < ROWS * COLS / 8; j += 256) {
            const int r = j / (COLS / 8), c = j % (COLS / 8) * 8;
            if (m0 + r < a.rows && c < cols) *reinterpret_cast<uint4*>(to + (size_t)r * a.N + c) = *reinterpret_cast<const uint4*>(tile + r * PITCH + c * 2);
        }
    } else {
#pragma unroll
        for (int j = threadIdx.x; j < ROWS * COLS; j += 256) {
            const int r = j / COLS, c = j % COLS;
            if (m0 + r < a.rows && c < cols) to[(size_t)r * a.N + c] = *reinterpret_cast<const uint16_t*>(tile + r * PITCH + c * 2);
        }
    }
}

// Returns whether any unit is cut.
bool make_schedule(const int* gsp, int groups, int units, int sms, Schedule& s) {
    constexpr long long kLeast = 8;  // steps of a range: below, joining costs more than the time saved
    constexpr long long kUnit = 6;   // what a unit takes beside its steps, in steps
    // What storing parts and joining them takes, in steps of tiles of 256 columns (8 to 10 us).  Narrower tiles have shorter steps; the
    // same rule is right for them or a little late to cut: us, cut and whole, 32, 64, 128 and 256 columns: layer 4096 x 14336 at 20 %
    // 13.7 and 22.3, 14.1 and 22.5, 15.5 and 23.3, 23.4 and 27.3 (it cuts); 8192 x 8192 at 5 % 13.0 and 14.6, 13.5 and 14.7, 15.4 and
    // 15.6, 23.1 and 19.2 (it does not).  kUnit between 1 and 12 makes no difference to the first of these.
    constexpr long long kJoin = 24;
    const long long total = (long long)gsp[groups] * units, all = (long long)groups * units;
    s.parts = (int)std::max<long long>(std::min<long long>(std::min(sms, kMaxParts), std::max(total / kLeast, all)), 1);
    s.units = units;
    s.rounds = (int)(all / s.parts);
    long long load[kMaxParts];
    int shortest = gsp[1], longest = 0;
    for (int g = 0; g < groups; g++) {
        shortest = std::min(shortest, gsp[g + 1] - gsp[g]);
        longest = std::max(longest, gsp[g + 1] - gsp[g]);
    }
    const long long cost = total + kUnit * all;
    auto deal = [&]() {
        long long most = 0;
        for (int c = 0; c < s.parts; c++) load[c] = shortest == longest ? s.rounds * (longest + kUnit) : 0;
        if (shortest != longest) {
            const long long dealt = (long long)s.rounds * s.parts;
            int c = 0;
            long long unit = 0;
            for (int g = 0; g < groups && unit < dealt; g++)
                for (int t = 0; t < units && unit < dealt; t++, unit++) {
                    load[c] += gsp[g + 1] - gsp[g] + kUnit;
                    if (++c == s.parts) c = 0;
                }
        }
        for (int c = 0; c < s.parts; c++) most = std::max(most, load[c]);
        return most;
    };
    // Units of very different lengths: everything in ranges.
    const bool uneven = s.rounds && deal() * s.parts > cost + cost / 4;
    if (uneven) s.rounds = 0;
    long long most = deal();
    const long long first = (long long)s.rounds * s.parts;  // the first unit of the ranges
    int g = (int)(first / units);
    const long long begin = (long long)gsp[g] * units + (first - (long long)g * units) * (g < groups ? gsp[g + 1] - gsp[g] : 0);
    const long long rest = total - begin;
    const long long left = all - first;  // units: fewer than parts, unless they are uneven
    bool may_cut = rest >= 2 * kLeast * left;
    int order[kMaxParts];
    if (!uneven) {
        // Whole units, one more for each of the parts with the least to do, or cut to equal shares?
        for (int c = 0; c < s.parts; c++) order[c] = c;
        std::sort(order, order + s.parts, [&](int x, int y) { return load[x] != load[y] ? load[x] < load[y] : x < y; });
        if (left) most = std::max(most, load[order[left - 1]] + longest + kUnit);
        if (most <= cost / s.parts + kJoin) may_cut = false;
        if (!may_cut && !s.rounds) {
            s.parts = (int)all;
            s.rounds = 1;
            for (int c = 0; c <= s.parts; c++) s.at[c] = {groups, 0, 0};
            return false;
        }
    }
    long long want[kMaxParts], sum = 0, given = 0;
    if (!uneven && !may_cut) {
        bool one[kMaxParts] = {};
        for (long long j = 0; j < left; j++) one[order[j]] = true;
        long long unit = first;
        for (int c = 0; c < s.parts; c++) {
            s.at[c] = {(int)(unit / units), (int)(unit % units), 0};
            unit += one[c];
        }
        s.at[s.parts] = {groups, 0, 0};
        return false;
    }
    // A part gets of the rest what it is short of an equal share; ranges of long units may cut them, others hold whole ones.
    for (int c = 0; c < s.parts; c++) {
        want[c] = std::max<long long>(cost / s.parts + 1 - load[c], 0);
        if (want[c] < kLeast && may_cut) want[c] = 0;
        sum += want[c];
    }
    if (!sum) { want[0] = sum = 1; }
    bool cut = false;
    for (int c = 0; c < s.parts; c++) {
        const long long p = begin + rest * given / sum;
        given += want[c];
        while (g < groups && (long long)gsp[g + 1] * units <= p) g++;
        Start b = {g, 0, 0};
        if (g < groups) {
            const int ns = gsp[g + 1] - gsp[g];
            const long long off = p - (long long)gsp[g] * units;
            b.t = (int)(off / ns);
            b.k = (int)(off % ns);
            if (b.k && !may_cut) {
                if (2 * b.k > ns && ++b.t == units) { b.t = 0; b.g++; }
                b.k = 0;
            }
        }
        cut |= b.k != 0;
        s.at[c] = b;
    }
    s.at[s.parts] = {groups, 0, 0};
    return cut;
}

template <int NT, int FMT>
int launch_tile(const TileArgs& args, const CUtensorMap& mapA, const CUtensorMap& map, const int* gsp, int groups, const DeviceCtx* ctx, cudaStream_t stream) {
    using G = Cfg<NT>;
    TileArgs a = args;
    SMAT_CUDA_TRY(cudaFuncSetAttribute(fp4_tile_kernel<NT, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
    a.col_tiles = (a.N + NT - 1) / NT;
    Schedule s;
    const bool cut = make_schedule(gsp, groups, (G::CG == 2 ? 1 : 2) * a.col_tiles, ctx->sm_count / G::CG, s);
    void* scratch = nullptr;
    if (cut) {
        SMAT_CUDA_TRY(cudaMallocFromPoolAsync(&scratch, (size_t)s.parts * 2 * 128 * G::CG * NT * sizeof(float), ctx->pool, stream));
        a.scratch = static_cast<float*>(scratch);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s.parts * G::CG));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = G::CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, fp4_tile_kernel<NT, FMT>, mapA, map, a, s);
    count_launch();
    if (e == cudaSuccess && cut) {
        Joins joins;
        list_joins(s, joins);
        fp4_join_kernel<NT><<<dim3(joins.n, NT / kJoinColumns<NT>), 256, 0, stream>>>(a, joins);
        e = cudaGetLastError();
        count_launch();
    }
    const cudaError_t f = scratch ? cudaFreeAsync(scratch, stream) : cudaSuccess;
    if (e == cudaSuccess) e = f;
    if (e != cudaSuccess) return fail(SMAT_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    return SMAT_OK;
}

template <int NT>
int launch_tile_format(int fmt, const TileArgs& a, const CUtensorMap& mapA, const CUtensorMap& map, const int* gsp, int groups, const DeviceCtx* ctx, cudaStream_t stream) {
    return fmt == SMAT_FP4_NV ? launch_tile<NT, SMAT_FP4_NV>(a, mapA, map, gsp, groups, ctx, stream)
                              : launch_tile<NT, SMAT_FP4_MX>(a, mapA, map, gsp, groups, ctx, stream);
}

}  // namespace

int launch_fp4_tile(const Fp4View& A, const Fp4Rhs& B, void* C, int c_dtype, size_t N, cudaStream_t stream, bool selftest) {
    DeviceCtx* ctx = nullptr;
    if (int rc = get_device_ctx(&ctx)) return rc;
    // The narrowest tile that holds N, or pairs.  Below 256 a tile has to hold all of N: its first column is looked for in the scales of
    // B by tiles of 128 rows.  us, tiles of 32, 64, 128 and 256 columns: layer 8192 x 28672 at 20 %, N = 8 30.9, 31.2, 42.0, 36.1; N = 32
    // 30.7, 30.2, 30.9, 33.9; N = 128 33.8 and 38.4 (the last two); layer 4096 x 14336, N = 8 13.5, 14.8, 16.5, 18.7; N = 32 13.7, 13.5,
    // 14.0, 18.1; N = 64 14.2, 14.4 and 19.0; N = 128 15.5 and 20.3.
    const int nt = N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
    CUtensorMap map, mapA = {};
    const size_t pitch = fp4_pitch(A.K);
    if (int rc = encode_tensor_map_2d_u8(&map, B.data, pitch, N, pitch, 128, (uint32_t)std::min(nt, 128), 128)) return rc;
    if (nt == 256) {  // pairs: A's tiles as rows of 128 bytes, 128 of codes and 16 of scales each, which lie in the order of shared memory
        constexpr uint32_t rows = kFp4TileBytes / 128;
        if (int rc = encode_tensor_map_2d_u8(&mapA, A.tiles, 128, A.total_steps * 2 * rows, 128, 128, kFp4TileCodes / 128, 0)) return rc;
    }
    TileArgs a = {};
    a.steps = A.steps;
    a.tiles = A.tiles;
    a.gsp = A.gsp;
    a.b_scales = B.scales;
    a.row_scale = A.row_scale ? A.row_scale + A.brow_begin * 16 : nullptr;
    a.b_row_scale = B.row_scale;
    a.C = C;
    a.status = ctx->d_status;
    a.wait_cycles = selftest ? kSelftestWaitCycles : kWaitCycles;
    a.lost_bytes = selftest ? 16 : 0;
    a.c_dtype = c_dtype;
    a.rows = (int)(A.block_rows * 16);
    a.N = (int)N;
    a.quads = (int)fp4_quads(A.K);
    a.total_steps = (int)A.total_steps;
    a.b_row_tiles = (int)((N + 127) / 128);
    const int groups = (int)((A.block_rows + kFp4GroupRows - 1) / kFp4GroupRows);
    switch (nt) {
        case 32: return launch_tile_format<32>(A.fmt, a, mapA, map, A.h_gsp, groups, ctx, stream);
        case 64: return launch_tile_format<64>(A.fmt, a, mapA, map, A.h_gsp, groups, ctx, stream);
        case 128: return launch_tile_format<128>(A.fmt, a, mapA, map, A.h_gsp, groups, ctx, stream);
        default: return launch_tile_format<256>(A.fmt, a, mapA, map, A.h_gsp, groups, ctx, stream);
    }
}

}  // namespace smat
