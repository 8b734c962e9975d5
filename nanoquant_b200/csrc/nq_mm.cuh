// Products of two dense matrices on the 5th-generation tensor cores, with the epilogue of the operator that needs them:
//
//     acc[m, n] = sum_k A[m, k] B[n, k]        16-bit floats with fp32 sums, or signed bytes with int32 sums
//
// Either operand may lie with k contiguous (rows of A or B) or with m / n contiguous (the product of a transposed matrix needs no copy).
//
// One CTA (CG = 1, 128 rows), or a pair on neighbouring SMs (CG = 2, 256 rows, each CTA holding its half of A and of B), takes tiles
// t, t + ctas, ... of `bn` columns:
//
//   warp 0       operands by TMA, 128 bytes of k per step, 128-byte swizzle
//   warp 1       MMAs (the pair's first CTA), four per step
//   warps 4-11   epilogue, two sets of four warps, 64 columns in turn; tensor memory holds two accumulators, so that the epilogue
//                of a tile runs beside the main loop of the next
//
// `bn` is a multiple of 16 up to 256 that the host chooses so that the tiles fill whole rounds of the SMs.  A product over a long k and
// few tiles is split: `splits` ranges of k are tiles of their own, whose partial sums the operator adds.
#pragma once

#include "nq_common.cuh"
#include "nq_tcgen05.cuh"

namespace nq {

constexpr int kMmThreads = 32 * 12, kMmEpilogueWarps = 8;
constexpr int kMmMaxStages = 24, kMmABytes = 128 * 128, kMmStageOut = 4096;   // (bytes of output staging per epilogue warp)
constexpr int kMmBarOff = 0, kMmFewOff = 512, kMmOutOff = 1024, kMmStageOff = kMmOutOff + kMmEpilogueWarps * kMmStageOut;
constexpr int kMmSmemMost = 226 * 1024;
constexpr int kMmAccCols = 256;

// How an operand's part of a step is fetched: `loads` boxes of its 3-d map, 64 of the first coordinate apart; the coordinates of k are (dx k, dy k), those
// of row r (m or n) are (r if x_rows, r if y_rows, r / 64 if z_rows).
struct MmLoad {
    int bytes;                     // of all of it
    int loads, dx, dy, x_rows, y_rows, z_rows;
};
struct MmShape {
    int M, N;                      // rows and columns of the result
    int m_tiles, n_tiles, bn;
    int ksteps, steps_per_split, splits;
    int kel, stages, stage_bytes, a_stage;  // elements of k per step; bytes of a stage, and of A in it
    int m_fast;                    // consecutive tiles share their columns
    int a_mn, b_mn;                // operand has m / n contiguous
    MmLoad a, b;
    int early_b;                   // B does not depend on the kernel before, which is one of the same call and has waited for all before it
    int release;                   // the kernel behind, one of the same call, may start early (but behind everything before this one)
    int few;                       // (kBuildA) bytes of A per step: 1024 for every eight rows
    const int* live;               // nullable: how many of the rows of A (live_k: of the steps' k) there are, known on the device alone
    int live_k, live_alt;          // (live_alt: A is map_alt's matrix where that is fewer than all)
    uint32_t idesc;
    unsigned wait_limit;
    unsigned* status;
};

// What a launch has to do: the host's numbers, or what the device knows better; in shared memory (registers are short in some epilogues).
struct MmDims {
    int rows, live;                // of A: that are taken (of a `live` number up to the next multiple of 64), and that count
    int ksteps, m_tiles, tiles;
};

template <class Epi>
struct alignas(64) MmParams {
    CUtensorMap map_a, map_b, map_alt;
    MmShape s;
    typename Epi::Params e;
};

// A split of the launch's registers between warpgroups (each call by all four warps of one).
template <int REGS>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }

// MN-major, 128-byte swizzle: 64 elements of m / n per 128-byte row, one row per k; 8-k groups 1024 bytes apart, the next 64 elements 8192.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr >> 4) & 0x3FFFu) | ((8192u >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
template <int CG, bool S8>
__device__ __forceinline__ void mm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define NQ_MM_ISSUE(cg, kind)                                                   \
    asm volatile("{\n\t.reg .pred p;\n\t"                                       \
                 "setp.ne.b32 p, %4, 0;\n\t"                                    \
                 "tcgen05.mma.cta_group::" cg ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory")
    if constexpr (CG == 2 && S8) NQ_MM_ISSUE("2", "i8");
    else if constexpr (CG == 2) NQ_MM_ISSUE("2", "f16");
    else if constexpr (S8) NQ_MM_ISSUE("1", "i8");
    else NQ_MM_ISSUE("1", "f16");
#undef NQ_MM_ISSUE
}
template <int CG>
__device__ __forceinline__ void mm_commit(uint32_t bar) {      // the barrier at this offset in every CTA of the group
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void mm_load(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// mbar_wait_warp for a thread of its own.
template <bool CLUSTER>
__device__ __forceinline__ bool mm_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned* status, unsigned limit) {
    auto done = [&]() { return CLUSTER ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity); };
    if (done()) return true;
    for (unsigned i = 0; i < limit; ++i) {
        if (done()) return true;
        if (*abort_flag != 0) return false;
    }
    *abort_flag = 1;
    atomicExch(status, (unsigned)(-NQ_ERR_TIMEOUT));
    return false;
}
// 32 columns of this warp's 32 rows: lane i has row i.
__device__ __forceinline__ void mm_tmem_start(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void mm_tmem_landed() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// (the registers are operands, so that no use moves above the wait in front of this)
__device__ __forceinline__ void mm_tmem_use(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
// 32 rows x 64 columns of 16-bit outputs through 4 KB of the warp's shared memory, so that eight lanes store a row's 128 bytes: lane i brings row i,
// 32 columns (`half` 0 or 1) as 16 words at a time.
__device__ __forceinline__ void mm_stage_row(unsigned char* stage, int half, const uint32_t (&w)[16]) {
    const int lane = threadIdx.x & 31;
    if (half == 0) __syncwarp();          // the stores before have read theirs
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * half + j) ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}
// `rows` / `cols` of them exist; `wide`: the rows start at 16-byte boundaries.
__device__ __forceinline__ void mm_store_rows(const unsigned char* stage, uint16_t* out, long long ld, int rows, int cols, bool wide) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (wide) {
        const int j = lane & 7;
        uint16_t* dst = out + (lane >> 3) * ld + 8 * j;
#pragma unroll
        for (int i = 0; i < 8; ++i, dst += 4 * ld) {
            const int r = 4 * i + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((j ^ (r & 7)) << 4));
            if (r < rows) store_rows(dst, v, cols - 8 * j, 8 * j + 8 <= cols);
        }
    } else {
        for (int c = lane; c < cols; c += 32)
            for (int r = 0; r < rows; ++r)
                out[r * ld + c] = *reinterpret_cast<const uint16_t*>(stage + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + 2 * (c & 7));
    }
}

// Epi: struct Params; kS8; kBuildA: the epilogue warps make A themselves, all of it before the first MMA (few rows: `build` writes its steps, each of
// whole 8-row groups in the layout of umma_desc, and may leave up to 512 bytes at `few` for the epilogue; the MMA reads rows beyond as they
// are, whose results nobody looks at); an object per epilogue thread with
//   Epi(const Params&, const MmShape&, few, dims)
//   begin(row, n0, m_tile, n_tile, split, ...)      a tile of this thread's row (row >= M: none)
//   chunk(r, c, cols, stage, half)                  32 columns from n0 + c, `cols` of which exist (all lanes call it, if any of their rows exists)
//   flush(c, cols, stage)                           behind both halves of 64 columns
//   end()
// kChunk: steps of k after which the accumulator is added to fp32 sums in registers (0: never).  The tensor cores cut an accumulator off, towards zero, with every
// instruction, so that the error of a long sum grows with its length, and has a sign: logits of 8 were 2.8e-5 low at 4096 columns, five times the
// rms error of fp32 additions.  A sum of C chunks is off by a C-th of that.
constexpr int kMmRegsLaunch = 168, kMmRegsIssue = 40, kMmRegsSums = 232;      // of a thread: at launch, and after the split with kChunk
static_assert(128 * kMmRegsIssue + 256 * kMmRegsSums <= kMmThreads * kMmRegsLaunch, "register split");
template <int CG, class Epi>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kMmThreads, 1) mm_kernel(const __grid_constant__ MmParams<Epi> P) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bars = sbase + kMmBarOff;
    const MmShape& S = P.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto bar_ready = [&](int s) { return bars + 8 * s; };                                  // used in the pair's first CTA
    auto bar_free = [&](int s) { return bars + 8 * (kMmMaxStages + s); };
    auto bar_acc_full = [&](int a) { return bars + 8 * (2 * kMmMaxStages + a); };
    auto bar_acc_empty = [&](int a) { return bars + 8 * (2 * kMmMaxStages + 2 + a); };     // used in the pair's first CTA
    const uint32_t bar_built = bars + 8 * (2 * kMmMaxStages + 4);
    constexpr int kMisc = kMmBarOff + 8 * (2 * kMmMaxStages + 5);
    static_assert(kMisc + 8 + (int)sizeof(MmDims) <= kMmFewOff, "shared memory map");
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + kMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kMisc + 4);
    volatile MmDims* dims = reinterpret_cast<volatile MmDims*>(smem + kMisc + 8);
    const int rank = CG == 2 ? (int)(blockIdx.x & 1) : 0;
    if (warp == 2) {
        if (lane < kMmMaxStages) {
            mbar_init(bar_ready(lane), 1);
            mbar_init(bar_free(lane), 1);
        }
        if (lane < 2) {
            mbar_init(bar_acc_full(lane), 1);
            mbar_init(bar_acc_empty(lane), CG * kMmEpilogueWarps);
        }
        if (lane == 0) {
            mbar_init(bar_built, kMmEpilogueWarps);
            *abort_flag = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(2u * kMmAccCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(2u * kMmAccCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    if (threadIdx.x == 0) {
        int rows = S.M, live = S.M, ksteps = S.ksteps, m_tiles = S.m_tiles;
        if (S.live) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            const int n = __ldcg(S.live), some = (max(n, 1) + 63) & ~63;      // (one step at least, of zeros)
            if (S.live_k) {
                ksteps = min(ksteps, some / 64);
            } else {
                live = n;
                rows = min(rows, some);
                m_tiles = (rows + 128 * CG - 1) / (128 * CG);
            }
        }
        dims->rows = rows;
        dims->live = live;
        dims->ksteps = ksteps;
        dims->m_tiles = m_tiles;
        dims->tiles = m_tiles * S.n_tiles * S.splits;
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    constexpr int kChunk = Epi::kChunk ? Epi::kChunk : 1 << 30;
    const int groups = (int)gridDim.x / CG, first = (int)blockIdx.x / CG, tiles = dims->tiles;
    struct Tile { int m, n, split, k0, k1; };
    auto tile_of = [&](int t) {
        const int m_tiles = dims->m_tiles, plane = m_tiles * S.n_tiles;
        Tile r;
        r.split = t / plane;
        const int u = t - r.split * plane;
        if (S.m_fast) { r.n = u / m_tiles; r.m = u - r.n * m_tiles; }
        else { r.m = u / S.n_tiles; r.n = u - r.m * S.n_tiles; }
        r.k0 = r.split * S.steps_per_split;
        r.k1 = min(dims->ksteps, r.k0 + S.steps_per_split);
        return r;
    };
    constexpr bool kBuildA = Epi::kBuildA;
    const uint32_t built = sbase + kMmStageOff, stage0 = built + (kBuildA ? (uint32_t)(S.few * S.ksteps) : 0u);
    const uint32_t a_stage = (uint32_t)S.a_stage;

    if (warp < 4) {
        if constexpr (Epi::kChunk > 0) regs_down<kMmRegsIssue>();
        // One thread each for the loads and for the MMAs: a step takes some 450 cycles, and votes of the warp, branches and look-ups in every one cost a tenth
        // of the tensor cores' time.
        if (warp == 0 && elect_one()) {
            // ------------------------------------------------------------ operands
            const uint32_t step_bytes = (uint32_t)CG * (uint32_t)((kBuildA ? 0 : S.a.bytes) + S.b.bytes), stage_bytes = (uint32_t)S.stage_bytes;
            const uint32_t ready0 = CG == 2 ? cluster_map(bar_ready(0), 0) : bar_ready(0);
            const CUtensorMap *map_a = &P.map_a, *map_b = &P.map_b;
            if (S.live_alt && dims->live < S.M) map_a = &P.map_alt;
            int ax, ay, az, bx, by, bz;                    // of the tile's rows
            auto tile_rows = [&](const Tile& T) {
                const int m = (T.m * CG + rank) * 128, n = T.n * S.bn + rank * (S.bn / CG);
                ax = S.a.x_rows ? m : 0; ay = S.a.y_rows ? m : 0; az = S.a.z_rows ? m >> 6 : 0;
                bx = S.b.x_rows ? n : 0; by = S.b.y_rows ? n : 0; bz = S.b.z_rows ? n >> 6 : 0;
            };
            const int adx = S.a.dx, ady = S.a.dy, bdx = S.b.dx, bdy = S.b.dy;
            auto load_a = [&](int k, uint32_t dst, uint32_t bar) {
                if constexpr (kBuildA) return;
                mm_load<CG>(dst, map_a, ax + k * adx, ay + k * ady, az, bar);
                for (int i = 1; i < S.a.loads; ++i) mm_load<CG>(dst + 8192u * i, map_a, ax + 64 * i, ay + k * ady, az, bar);
            };
            auto load_b = [&](int k, uint32_t dst, uint32_t bar) {
                mm_load<CG>(dst, map_b, bx + k * bdx, by + k * bdy, bz, bar);
                for (int i = 1; i < S.b.loads; ++i) mm_load<CG>(dst + 8192u * i, map_b, bx + 64 * i, by + k * bdy, bz, bar);
            };
            int s = 0, pre = 0;
            uint32_t ph = 0;
            bool ok = true;
            if (S.early_b && first < tiles) {      // the first tile's columns while the kernel before still writes the rows
                const Tile T = tile_of(first);
                tile_rows(T);
                pre = min(S.stages, T.k1 - T.k0);
                for (int i = 0; i < pre; ++i) {
                    if (rank == 0) mbar_expect_tx(bar_ready(i), step_bytes);
                    load_b(T.k0 + i, stage0 + (uint32_t)i * stage_bytes + a_stage, ready0 + 8 * i);
                }
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            if (S.release) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if (pre) {
                const int k0 = tile_of(first).k0;
                for (int i = 0; i < pre; ++i) load_a(k0 + i, stage0 + (uint32_t)i * stage_bytes, ready0 + 8 * i);
                s = pre;
                if (s == S.stages) { s = 0; ph = 1; }
            }
            for (int t = first; t < tiles && ok; t += groups) {
                const Tile T = tile_of(t);
                tile_rows(T);
                for (int k = T.k0 + pre; k < T.k1; ++k) {
                    ok = mm_wait<CG == 2>(bar_free(s), ph ^ 1, abort_flag, S.status, S.wait_limit);
                    if (!ok) break;
                    if (rank == 0) mbar_expect_tx(bar_ready(s), step_bytes);
                    const uint32_t dst = stage0 + (uint32_t)s * stage_bytes, bar = ready0 + 8 * s;
                    load_a(k, dst, bar);
                    load_b(k, dst + a_stage, bar);
                    if (++s == S.stages) { s = 0; ph ^= 1; }
                }
                pre = 0;
            }
        } else if (warp == 1 && rank == 0 && elect_one()) {
            // ------------------------------------------------------------ MMA issue
            const uint32_t a_step = S.a_mn ? 2048u >> 4 : 32u >> 4, b_step = S.b_mn ? 2048u >> 4 : 32u >> 4, idesc = S.idesc;
            const uint64_t a0 = S.a_mn ? umma_desc_mn(kBuildA ? built : stage0) : umma_desc(kBuildA ? built : stage0);
            const uint64_t b0 = S.b_mn ? umma_desc_mn(stage0 + a_stage) : umma_desc(stage0 + a_stage);
            const uint32_t stage_units = (uint32_t)S.stage_bytes >> 4, few_units = (uint32_t)S.few >> 4;
            int s = 0, a = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            if constexpr (kBuildA) {
                ok = mm_wait<false>(bar_built, 0, abort_flag, S.status, S.wait_limit);
                tc_fence_after();
            }
            for (int t = first; t < tiles && ok; t += groups) {
                const Tile T = tile_of(t);
                for (int c0 = T.k0; c0 < T.k1 && ok; c0 += kChunk) {
                    const int c1 = min(T.k1 - c0, kChunk) + c0;
                    const uint32_t d = tmem_base + (uint32_t)(a * kMmAccCols);
                    ok = mm_wait<CG == 2>(bar_acc_empty(a), aph ^ 1, abort_flag, S.status, S.wait_limit);
                    tc_fence_after();
                    for (int k = c0; k < c1 && ok; ++k) {
                        ok = mm_wait<CG == 2>(bar_ready(s), ph, abort_flag, S.status, S.wait_limit);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t ad = a0 + (uint64_t)(kBuildA ? (uint32_t)k * few_units : (uint32_t)s * stage_units), bd = b0 + (uint64_t)((uint32_t)s * stage_units);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mm_mma<CG, Epi::kS8>(d, ad + (uint64_t)(a_step * i), bd + (uint64_t)(b_step * i), idesc, k > c0 || i ? 1u : 0u);
                        mm_commit<CG>(bar_free(s));
                        if (++s == S.stages) { s = 0; ph ^= 1; }
                    }
                    if (ok) mm_commit<CG>(bar_acc_full(a));
                    if (++a == 2) { a = 0; aph ^= 1; }
                    if (T.k1 - c0 <= kChunk) break;
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- epilogue
        if constexpr (Epi::kChunk > 0) regs_up<kMmRegsSums>();
        const int ew = warp & 3, set = (warp - 4) >> 2;
        unsigned char* stage = smem + kMmOutOff + (warp - 4) * kMmStageOut;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if constexpr (kBuildA) {
            Epi::build(P.e, S, smem + kMmStageOff, smem + kMmFewOff);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_built);
        }
        Epi epi(P.e, S, smem + kMmFewOff, dims);
        int a = 0;
        uint32_t aph = 0;
        for (int t = first; t < tiles; t += groups) {
            const Tile T = tile_of(t);
            const int row = (T.m * CG + rank) * 128 + 32 * ew + lane, n0 = T.n * S.bn, live = min(S.bn, S.N - n0);
            auto full = [&]() {
                const bool ok = mbar_wait_warp<CG == 2>(bar_acc_full(a), aph, abort_flag, S.status, S.wait_limit);
                tc_fence_after();
                return ok;
            };
            auto empty = [&]() {                          // this warp has read the accumulator
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_map(bar_acc_empty(a), 0)) : "memory");
                    else mbar_arrive(bar_acc_empty(a));
                }
                if (++a == 2) { a = 0; aph ^= 1; }
            };
            const bool some = row - lane < dims->rows;    // of the warp's rows exist
            if constexpr (Epi::kChunk > 0) {
                float sum[kMmAccCols / 64][32] = {};
                bool ok = true;
                for (int c0 = T.k0; c0 < T.k1; c0 += kChunk) {
                    ok = full();
                    if (!ok) break;
                    const uint32_t d = tmem_base + (uint32_t)(a * kMmAccCols) + ((uint32_t)(32 * ew) << 16);
#pragma unroll
                    for (int j = 0; j < kMmAccCols / 64; j += 2) {        // (two loads under way)
                        if (64 * set + 64 * j < live && some) {
                            uint32_t r0[32], r1[32];
                            mm_tmem_start(d + (uint32_t)(64 * set + 64 * j), r0);
                            mm_tmem_start(d + (uint32_t)(64 * set + 64 * j + 32), r1);      // (within the accumulator, whatever the tile's width)
                            mm_tmem_landed();
                            mm_tmem_use(r0);
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[j][i] += __uint_as_float(r0[i]);
                            mm_tmem_use(r1);
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[j + 1][i] += __uint_as_float(r1[i]);
                        }
                    }
                    empty();
                }
                if (!ok) break;
                epi.begin(row, n0, set, T.n, T.split);
#pragma unroll
                for (int j = 0; j < kMmAccCols / 64; j += 2) {
                    const int c = 64 * set + 64 * j;
                    if (c < live && some) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            uint32_t r[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(sum[j + half][i]);
                            if (half == 0 || c + 32 < live) epi.chunk(r, c + 32 * half, min(32, live - c - 32 * half), stage, half);
                        }
                        epi.flush(c, min(64, live - c), stage);
                    }
                }
            } else {
                if (!full()) break;
                epi.begin(row, n0, set, T.n, T.split);
                const uint32_t d = tmem_base + (uint32_t)(a * kMmAccCols) + ((uint32_t)(32 * ew) << 16);
#pragma unroll 1
                for (int c = 64 * set; c < live && some; c += 128) {
                    uint32_t r0[32], r1[32];
                    mm_tmem_start(d + (uint32_t)c, r0);
                    mm_tmem_start(d + (uint32_t)c + 32u, r1);      // (within the accumulator, whatever the tile's width)
                    mm_tmem_landed();
                    mm_tmem_use(r0);
                    epi.chunk(r0, c, min(32, live - c), stage, 0);
                    mm_tmem_use(r1);
                    if (c + 32 < live) epi.chunk(r1, c + 32, min(32, live - c - 32), stage, 1);
                    epi.flush(c, min(64, live - c), stage);
                }
                empty();
            }
            epi.end();
        }
    }
    // On an expired wait, give the copies in flight a bounded time to land before shared memory is released.
    if (*abort_flag && threadIdx.x == 0) {
        for (unsigned i = 0; i < (1u << 20); ++i) __nanosleep(64);
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 2) {
        // the other CTA may still signal barriers here, and its MMAs and epilogue use the pair's tensor memory
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * kMmAccCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * kMmAccCols) : "memory");
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// One operand: a matrix of `rows` (m or n) and K columns, or its transpose (`mn`: rows of K, `rows` contiguous elements each).
struct MmOperand {
    const void* p;
    int64_t stride;       // bytes between its rows in memory
    int mn;
    int64_t extent = 0;   // (mn) `rows` that may be read, if more
};

// Width of the tiles: the multiple of `unit` up to 256 that takes least time, in columns of a k step.
// Pairs of CTAs: whole rounds of tiles over the pairs; a tile costs its columns and some 220 more, for its rows pass through L2 to the SMs as often as
// there are tiles.  us at 128 / 160 / 192 / 224 / 256 columns: int8 12288 x 4096, 512 tokens 32.1 / 34.3 / 30.6 / 31.6 / 33.2, 2048 tokens 111 / 93 / 85 / 86 (taken) /
// 97, 4096 tokens 172 / 157 / 146 / 141 / 139, 4096 x 12288, 2048 tokens 102 / 89 / 95 / 100 / 85; the loss of 2048 tokens at 128256 x 2048 895 / 792 / 731 / 704 / 681.
// Single CTAs have up to 128 rows and are bound by the memory that B streams from, as long as a step has enough of it: its four MMAs take as long for
// 16 columns as for some 100 (they fetch 128 rows of A all the same).  The last tile's latency is what narrow tiles save.  One token, int8, us at
// 32 / 64 / 96 / 128 / 176 / 208 / 256 columns: 128256 x 2048 94 / 52 / 46.4 / 44.5 / 50.5 / 51.6 / 48.6, 151936 x 4096 200 / 108 / 94.8 / 97.4 / 97.0 /
// 96.2 / 106, 12288 x 4096 22.1 / 17.0 / 13.1 / 13.3 / 16.3 / 17.4 / 20.2.
inline int mm_tile_cols(int N, int m_tiles, int cg, int least) {
    const int groups = sm_count() / cg, unit = 16 * cg;
    int best = 0;
    double best_cost = 0;
    for (int bn = 256; bn >= least; bn -= unit) {
        const int64_t tiles = (int64_t)((N + bn - 1) / bn) * m_tiles, rounds = (tiles + groups - 1) / groups;
        const double cost = cg == 2 ? (double)rounds * (bn + 220) : (double)rounds * (bn > 100 ? bn : 100) + 0.4 * bn;
        if (!best || cost < best_cost * 0.995) { best = bn; best_cost = cost; }
    }
    return best;
}

// Map and loads of an operand's `box` rows per step.
inline int mm_operand(CUtensorMap* map, MmLoad& L, const MmOperand& O, int type, int64_t rows, int64_t K, int kel, int box) {
    L = {box * 128, 1, 0, 0, 0, 0, 0};
    if (!O.mn) {
        L.dx = kel; L.y_rows = 1;
        return mm_encode(map, O.p, type, K, rows, O.stride, kel, box);
    }
    // All of an operand's columns of 64 by one load (by one load each, both operands' kept the loading thread busy longer than the MMAs take; the gradient of
    // 50688 x 4096 weights over 2048 tokens 612 us -> 524), where they are whole.
    L.dy = 64;
    if (rows % 64 == 0) {
        L.z_rows = 1;
        return mm_encode_columns(map, O.p, type, rows, K, O.stride, box / 64);
    }
    L.loads = box / 64; L.x_rows = 1;
    return mm_encode(map, O.p, type, rows, K, O.stride, 64, 64);
}
// P.s.live, live_k and live_alt (with P.map_alt) are the caller's, or zero.
template <int CG, class Epi>
int mm_launch(MmParams<Epi>& P, int type, const MmOperand& A, const MmOperand& B, int M, int N, int64_t K, int bn, int splits,
              int early_b, int release, unsigned* status, cudaStream_t stream) {
    static bool attr_set[64];
    int dev = 0;
    NQ_CUDA_TRY(cudaGetDevice(&dev));
    const void* fn = (const void*)mm_kernel<CG, Epi>;
    if (!attr_set[dev & 63]) {
        NQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMmSmemMost));
        attr_set[dev & 63] = true;
    }
    MmShape& S = P.s;
    const int esize = type == kMmS8 ? 1 : 2;
    S.M = M; S.N = N; S.bn = bn;
    S.m_tiles = (M + 128 * CG - 1) / (128 * CG);
    S.n_tiles = (N + bn - 1) / bn;
    S.m_fast = S.m_tiles <= S.n_tiles;
    S.kel = 128 / esize;                                     // elements of k per step
    S.ksteps = (int)((K + S.kel - 1) / S.kel);
    S.few = Epi::kBuildA ? (M + 7) / 8 * 1024 : 0;
    if (splits > S.ksteps) splits = S.ksteps;
    S.steps_per_split = (S.ksteps + splits - 1) / splits;
    S.splits = (S.ksteps + S.steps_per_split - 1) / S.steps_per_split;
    const int64_t am = A.extent > M ? A.extent : M, bm = B.extent > N ? B.extent : N;
    S.a_mn = A.mn; S.b_mn = B.mn;
    const int a_rows = A.mn || CG == 2 || M >= 128 ? 128 : (M + 7) / 8 * 8, b_rows = bn / CG;
    S.a_stage = Epi::kBuildA ? 0 : a_rows * 128;
    S.stage_bytes = S.a_stage + b_rows * 128;
    // (a step's MMAs read 128 rows of A; what lies behind fewer is read as it is, and nobody looks at these rows' results)
    const int fixed = 1024 + kMmStageOff + S.few * S.ksteps, slack = Epi::kBuildA || S.a_stage < kMmABytes ? kMmABytes : 0;
    S.stages = (kMmSmemMost - fixed - slack) / S.stage_bytes;
    if (S.stages > kMmMaxStages) S.stages = kMmMaxStages;
    S.early_b = early_b && !S.live;
    S.release = release;
    const uint32_t fmt = type == kMmF16 ? 0u : 1u;           // kind::f16: 1 = bf16; kind::i8: 1 = signed
    S.idesc = (type == kMmS8 ? 2u : 1u) << 4 | fmt << 7 | fmt << 10 | (uint32_t)A.mn << 15 | (uint32_t)B.mn << 16 |
              (uint32_t)(bn >> 3) << 17 | (uint32_t)(128 * CG >> 4) << 24;
    S.wait_limit = gemm_wait_limit();
    S.status = status;
    int st = Epi::kBuildA ? NQ_OK : mm_operand(&P.map_a, S.a, A, type, am, K, S.kel, a_rows);
    if (st != NQ_OK) return st;
    st = mm_operand(&P.map_b, S.b, B, type, bm, K, S.kel, b_rows);
    if (st != NQ_OK) return st;
    const int64_t tiles = (int64_t)S.m_tiles * S.n_tiles * S.splits, most = sm_count() / CG;
    if (tiles > 0x3fffffff) return NQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(CG * (tiles < most ? tiles : most)));
    cfg.blockDim = dim3(kMmThreads);
    cfg.dynamicSmemBytes = fixed + S.stages * S.stage_bytes + slack;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    return launch_dependent(cfg, attr, 0, fn, args);
}

}  // namespace nq
