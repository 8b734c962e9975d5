// Attention of whole prompts, packed, with grouped heads, on the 5th-generation tensor cores.
//
//     S = Q K^T,   P = 2^(scale log2(e) S - m),   O = P V,   o = O / sum P
//
// One pass over the keys with the running maximum and sum of a softmax.  Bound by the tensor cores and, as closely, by the exponentials: a tile of 128 queries x 128
// keys of 128 columns is 1024 clk of products and 16384 exponentials, 1024 clk of an SM's MUFU.  Two tiles of queries take turns so that one's products run
// beside the other's softmax.
//
// Work.  A tile's 128 rows are the query heads that share a key head, of as many tokens as fit (row = token x heads + head): keys and values pass from L2 once
// for all of them, and a causal block ends close to the diagonal.  A CTA has a block of two tiles (heads of up to 128 columns; one tile above) of one sequence and
// one key head; blocks of a sequence start with its last, the longest.
//
//   warp 0       queries, then keys and values in turn into a ring of stages, by TMA (128-byte swizzle), a box for each page of a cache
//   warp 1       products: S into tensor memory, then P (from tensor memory, over its S) times V into O, also there
//   warp 2       values behind a sequence's last token are set to zero in shared memory: their weights are zero, which a NaN would survive
//   warps 4-11   softmax, four warps to a tile, a row to a thread; the next S of a tile is ordered behind its P V, the other tile's products run meanwhile
//
// The maximum m is moved, and O multiplied accordingly, only when it grows by more than 2^8: P and its sum have room for that, and the result does not depend on m.
// The weights P are rounded to the operands' 16-bit type for the product with the values (what the tensor cores take): 2^-9 (bf16) or 2^-12 (fp16) of each, not
// enlarged by the average over tokens.
#include <type_traits>

#include "nq_attn.cuh"
#include "nq_mm.cuh"

namespace nq {

int attention_check(const nq_attention_desc& d);
int attention_cache_check(const nq_attention_desc& d);

struct alignas(64) PromptParams {
    CUtensorMap map_q, map_k, map_v;
    nq_attention_desc d;
    int rows, tokens;              // query heads to a key head; tokens of a tile
    int piece, shift;              // keys of one box; log2(page_size)
    int paged;
    float factor;                  // scale log2(e)
    uint32_t idesc_s, idesc_o;
    unsigned wait_limit;
    unsigned* status;
};

template <int DP> struct PromptShape {
    static constexpr int kTiles = DP <= 128 ? 2 : 1;
    static constexpr int kKeys = DP <= 128 ? 128 : 64;            // of a step
    static constexpr int kEarly = kTiles == 2 ? 3 : 2;            // 32s of keys whose weights are handed over first
    static constexpr int kColumns = DP / 64;                      // 128-byte columns of a row
    static constexpr int kTileBytes = 128 * DP * 2;               // queries
    static constexpr int kStageBytes = kKeys * DP * 2;
    static constexpr int kStages = DP == 64 ? 8 : 5;
    static constexpr int kThreads = 128 + 128 * kTiles;
    static constexpr int kQOff = 1024, kRingOff = kQOff + kTiles * kTileBytes;
    static constexpr int kSmem = 1024 + kRingOff + kStages * kStageBytes;
    static constexpr int kOCol = 256;                             // tensor memory: S at 0, O from here
    static_assert(kSmem <= 227 * 1024 && kOCol + kTiles * DP <= 512, "shared and tensor memory");
};
constexpr int kPromptRegsLaunch = 168, kPromptRegsIssue = 88, kPromptRegsSoftmax = 208;      // of a thread: at launch, and after the split
static_assert(128 * kPromptRegsIssue + 256 * kPromptRegsSoftmax <= 384 * kPromptRegsLaunch, "register split");
constexpr float kPromptSlack = 8.f;                               // powers of two by which a maximum may be behind

struct PromptBlock {
    int seq, first;                // first token of the block, within the sequence
    int q_len, k_len;
    int q_at, k_at;                // rows of the sequence's first tokens
    int bad;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// A [128 x 16] from tensor memory, B from shared memory.
__device__ __forceinline__ void prompt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The block that CTA `index` (of a key head) has, by one warp; false: none.
__device__ __forceinline__ bool prompt_block(const PromptParams& P, int index, int block_tokens, PromptBlock& B) {
    const nq_attention_desc& d = P.d;
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < d.seqs; s0 += 32) {
        const int s = s0 + lane;
        int begin = 0, end = 0;
        if (s < d.seqs) {
            begin = min(max(__ldcg(d.cu_seqlens + s), 0), (int)d.T);
            end = min(max(__ldcg(d.cu_seqlens + s + 1), begin), (int)d.T);
        }
        const int n = (end - begin + block_tokens - 1) / block_tokens;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        sum += before;
        const unsigned hit = __ballot_sync(0xffffffffu, index < sum);
        if (hit) {
            const int src = __ffs(hit) - 1;
            B.seq = s0 + src;
            B.q_at = __shfl_sync(0xffffffffu, begin, src);
            B.q_len = __shfl_sync(0xffffffffu, end, src) - B.q_at;
            const int last = __shfl_sync(0xffffffffu, sum, src);           // blocks up to this sequence's end
            B.first = (last - 1 - index) * block_tokens;
            B.bad = 0;
            B.k_at = B.q_at;
            B.k_len = B.q_len;
            if (P.paged) {
                B.k_at = 0;
                B.k_len = max(__ldcg(d.lengths + B.seq), 0);
                if ((long long)B.k_len > ((long long)d.max_pages << P.shift)) { B.bad = 1; B.k_len = 0; }
            } else if (d.cu_seqlens_k) {
                B.k_at = min(max(__ldcg(d.cu_seqlens_k + B.seq), 0), (int)d.Tk);
                B.k_len = min(max(__ldcg(d.cu_seqlens_k + B.seq + 1), B.k_at), (int)d.Tk) - B.k_at;
            } else {
                B.k_len = min(B.k_at + B.k_len, (int)d.Tk) - min(B.k_at, (int)d.Tk);      // (fewer keys than queries)
            }
            return true;
        }
        before = __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(PromptShape<DP>::kThreads, 1) prompt_kernel(const __grid_constant__ PromptParams P) {
    using Sh = PromptShape<DP>;
    constexpr int kTiles = Sh::kTiles, kKeys = Sh::kKeys, kStages = Sh::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const nq_attention_desc& d = P.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto bar_full = [&](int s) { return sbase + 8 * s; };
    auto bar_free = [&](int s) { return sbase + 8 * (kStages + s); };
    constexpr int kBars = 2 * kStages;
    const uint32_t bar_q = sbase + 8 * kBars, bar_tail = bar_q + 8;
    auto bar_s = [&](int i) { return bar_q + 16 + 8 * i; };           // S is there (by tile, or with one tile by buffer)
    auto bar_p = [&](int i) { return bar_q + 32 + 8 * i; };           // P is there
    auto bar_o = [&](int i) { return bar_q + 48 + 8 * i; };           // P V has been added (by tile)
    auto bar_h = [&](int i) { return bar_q + 64 + 8 * i; };           // the rest of P is there (two tiles)
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + 256);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 260);
    volatile int* bad_page = reinterpret_cast<volatile int*>(smem + 264);
    volatile int* have = reinterpret_cast<volatile int*>(smem + 268);
    volatile PromptBlock* block = reinterpret_cast<volatile PromptBlock*>(smem + 272);
    static_assert(8 * kBars + 80 <= 256, "shared memory map");

    const int kh = blockIdx.x % d.k_heads, index = blockIdx.x / d.k_heads, block_tokens = kTiles * P.tokens;
    if (warp == 2) {
        if (lane < kStages) {
            mbar_init(bar_full(lane), 1);
            mbar_init(bar_free(lane), 1);
        }
        if (lane < 2) {
            mbar_init(bar_s(lane), 1);
            mbar_init(bar_p(lane), 4);
            mbar_init(bar_o(lane), 1);
            mbar_init(bar_h(lane), 4);
        }
        if (lane == 0) {
            mbar_init(bar_q, 1);
            mbar_init(bar_tail, 1);
            *abort_flag = 0;
            *bad_page = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 3) {
        PromptBlock B;
        const bool some = prompt_block(P, index, block_tokens, B);
        if (lane == 0) {
            *have = some;
            if (some) {
                block->seq = B.seq; block->first = B.first; block->q_len = B.q_len; block->k_len = B.k_len;
                block->q_at = B.q_at; block->k_at = B.k_at; block->bad = B.bad;
            }
        }
        // rows of no sequence
        const int head = min(max(__ldcg(d.cu_seqlens), 0), (int)d.T), tail = min(max(__ldcg(d.cu_seqlens + d.seqs), head), (int)d.T);
        const long long per = (long long)d.q_heads * d.D / 8, missing = ((long long)head + (d.T - tail)) * per;
        for (long long i = (long long)blockIdx.x * 32 + lane; i < missing; i += (long long)gridDim.x * 32) {
            const long long at = i < head * per ? i : i - head * per + tail * per;
            static_cast<uint4*>(d.out)[at] = make_uint4(0, 0, 0, 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // what the block has to do
    const bool some = *have;
    const int first = some ? block->first : 0, q_len = some ? block->q_len : 0, k_len = some ? block->k_len : 0, q_at = block->q_at, k_at = block->k_at;
    const int behind = k_len - q_len;              // query t is at place t + behind
    auto sees_end = [&](int t) { return max(0, d.causal ? min(k_len, t + behind + 1) : k_len); };
    auto sees_begin = [&](int t) { return d.window > 0 ? max(0, t + behind + 1 - d.window) : 0; };
    // the first key, at the start of a page (or of a step)
    const int k_first = sees_begin(first) / P.piece * P.piece;
    int steps[kTiles], most = 0;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        const int t = first + i * P.tokens, last = min(t + P.tokens, q_len) - 1;
        steps[i] = t < q_len ? max(0, (sees_end(last) - k_first + kKeys - 1) / kKeys) : 0;
        most = max(most, steps[i]);
    }
    const int tail_rows = k_len - k_first - (most - 1) * kKeys;          // of the last step, that the sequence has
    const bool fix = most > 0 && tail_rows < kKeys;

    if (warp < 4) {
        if constexpr (kTiles == 2) regs_down<kPromptRegsIssue>();
        if (warp == 0) {
            // ------------------------------------------------------------ operands
            const int* table = d.block_table + (P.paged ? (long long)block->seq * d.table_stride : 0);
            if (most > 0 && elect_one()) {
                const uint32_t bytes = (uint32_t)(P.rows * P.tokens * 128 * Sh::kColumns);
                int tiles = 0;
                for (int i = 0; i < kTiles; ++i) tiles += steps[i] > 0;
                mbar_expect_tx(bar_q, tiles * bytes);
                for (int i = 0; i < kTiles; ++i) {
                    if (steps[i] == 0) continue;
                    for (int c = 0; c < Sh::kColumns; ++c)
                        tma_load_4d(sbase + Sh::kQOff + i * Sh::kTileBytes + c * 128 * 128, &P.map_q, 64 * c, kh * P.rows, q_at + first + i * P.tokens, 0, bar_q);
                }
            }
            __syncwarp();
            const int pieces = kKeys / P.piece;
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int j = 0; j < most && ok; ++j) {
                const int key = k_first + j * kKeys + lane * P.piece;       // this lane's box
                const int boxes = P.paged ? min(pieces, (k_len - (k_first + j * kKeys) + P.piece - 1) / P.piece) : 1;
                int page = 0, row = k_at + key;
                if (P.paged && lane < boxes) {
                    page = __ldcg(table + (key >> P.shift));
                    row = key & (d.page_size - 1);
                    if (page < 0 || page >= d.pages) { page = 0; *bad_page = 1; }
                }
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    ok = mbar_wait_warp(bar_free(s), ph ^ 1, abort_flag, P.status, P.wait_limit);
                    if (!ok) break;
                    const uint32_t bar = kv == 1 && fix && j == most - 1 ? bar_tail : bar_full(s);
                    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(boxes * P.piece * 128 * Sh::kColumns));
                    __syncwarp();
                    if (lane < boxes) {
                        const uint32_t dst = sbase + Sh::kRingOff + s * Sh::kStageBytes + lane * P.piece * 128;
                        for (int c = 0; c < Sh::kColumns; ++c) tma_load_4d(dst + c * kKeys * 128, kv ? &P.map_v : &P.map_k, 64 * c, row, kh, page, bar);
                    }
                    __syncwarp();
                    if (++s == kStages) { s = 0; ph ^= 1; }
                }
            }
        } else if (warp == 1) {
            if (most > 0 && elect_one()) {
                // -------------------------------------------------------- products
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    const bool ok = mm_wait<false>(bar, parity, abort_flag, P.status, P.wait_limit);
                    tc_fence_after();
                    return ok;
                };
                auto stage = [&](int n) { return sbase + Sh::kRingOff + (n % kStages) * Sh::kStageBytes; };
                auto parity = [&](int n) { return (uint32_t)(n / kStages) & 1u; };
                // S of tile i (one tile: into buffer b) with the keys at `kt`
                auto product_s = [&](int i, int b, uint32_t kt) {
                    const uint64_t qd = umma_desc(sbase + Sh::kQOff + i * Sh::kTileBytes), kd = umma_desc(kt);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mm_mma<1, false>(tmem + (i + b) * kKeys, qd + (uint64_t)(((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4),
                                         kd + (uint64_t)(((k >> 2) * kKeys * 128 + (k & 3) * 32) >> 4), P.idesc_s, k > 0);
                    mm_commit<1>(bar_s(i + b));
                };
                // with the keys [16 k0, 16 k1) of a step
                auto product_o = [&](int i, int b, uint32_t vt, int k0, int k1, bool more) {
                    // values: 64 columns to a 128-byte row, a row to a key; the next 64 columns kKeys rows on
                    const uint64_t vd = (umma_desc_mn(vt) & ~(0x3FFFull << 16)) | ((uint64_t)((kKeys * 128) >> 4) << 16);
#pragma unroll
                    for (int k = k0; k < k1; ++k)
                        prompt_mma_ts(tmem + Sh::kOCol + i * DP, tmem + (i + b) * kKeys + 8 * k, vd + (uint64_t)((k * 2048) >> 4), P.idesc_o, more || k > 0);
                };
                bool ok = wait(bar_q, 0) && wait(bar_full(0), 0);
                if (ok) {
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
                        if (steps[i] > 0) product_s(i, 0, stage(0));
                    mm_commit<1>(bar_free(0));
                }
                for (int j = 0; j < most && ok; ++j) {
                    const int nv = 2 * j + 1, nk = nv + 1;               // places of these values and of the next keys in the ring
                    const bool next = j + 1 < most;
                    if constexpr (kTiles == 1) {
                        // the next S before this P: two buffers
                        const int b = j & 1;
                        if (next) {
                            ok = wait(bar_full(nk % kStages), parity(nk));
                            if (!ok) break;
                            product_s(0, b ^ 1, stage(nk));
                            mm_commit<1>(bar_free(nk % kStages));
                        }
                        ok = wait(bar_full(nv % kStages), parity(nv)) && wait(bar_p(b), (uint32_t)(j >> 1) & 1u);
                        if (!ok) break;
                        product_o(0, b, stage(nv), 0, 2 * Sh::kEarly, j > 0);
                        mm_commit<1>(bar_o(0));
                    } else {
                        ok = wait(bar_full(nv % kStages), parity(nv));
                        bool keys = false;
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) {
                            if (!ok || j >= steps[i]) continue;
                            ok = wait(bar_p(i), (uint32_t)j & 1u);
                            if (!ok) continue;
                            product_o(i, 0, stage(nv), 0, 2 * Sh::kEarly, j > 0);
                            ok = wait(bar_h(i), (uint32_t)j & 1u);
                            if (!ok) continue;
                            product_o(i, 0, stage(nv), 2 * Sh::kEarly, kKeys / 16, true);
                            mm_commit<1>(bar_o(i));
                            if (j + 1 < steps[i]) {
                                if (!keys) ok = wait(bar_full(nk % kStages), parity(nk));
                                keys = true;
                                if (ok) product_s(i, 0, stage(nk));
                            }
                        }
                        if (!ok) break;
                        if (next) mm_commit<1>(bar_free(nk % kStages));
                    }
                    mm_commit<1>(bar_free(nv % kStages));
                }
            }
            __syncwarp();
        } else if (warp == 2 && fix) {
            // ------------------------------------------------------------ values behind the last token
            const int n = 2 * most - 1;
            if (mbar_wait_warp(bar_tail, 0, abort_flag, P.status, P.wait_limit)) {
                unsigned char* at = smem + Sh::kRingOff + (n % kStages) * Sh::kStageBytes;
                const int left = (kKeys - tail_rows) * 8;                 // 16-byte units of a column
                for (int i = lane; i < left * Sh::kColumns; i += 32) {
                    const int c = i / left;
                    *reinterpret_cast<uint4*>(at + c * kKeys * 128 + tail_rows * 128 + (i - c * left) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_full(n % kStages));
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax
        constexpr int kChunks = kKeys / 32, kEarly = Sh::kEarly;
        if constexpr (kTiles == 2) regs_up<kPromptRegsSoftmax>();
        const int i = (warp - 4) >> 2, row = 32 * (warp & 3) + lane;
        const int token = row / P.rows, t = first + i * P.tokens + token;
        const bool live = token < P.tokens && t < q_len;
        const int begin = sees_begin(t), end = live ? sees_end(t) : 0;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t o_at = tmem + lanes + Sh::kOCol + i * DP;
        float m = live ? -INFINITY : 0.f, l = 0.f;      // (rows that are not there hold nobody up)
        const int n = kTiles == 1 ? most : (i == 0 ? steps[0] : steps[kTiles - 1]);
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const int b = kTiles == 1 ? j & 1 : i;
            ok = mbar_wait_warp(bar_s(b), (uint32_t)(kTiles == 1 ? j >> 1 : j) & 1u, abort_flag, P.status, P.wait_limit);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = tmem + lanes + b * kKeys;
            const int key = k_first + j * kKeys;
            const bool masked = __any_sync(0xffffffffu, live && (key < begin || key + kKeys > end));
            uint32_t r[kChunks][32], w[16];
            uint64_t sum2[2] = {0, 0};
            const uint64_t factor2 = pair_of(P.factor, P.factor);
            auto peaks = [&](int c) {              // (NaN where there is one)
                float top[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) top[u] = __uint_as_float(r[c][u]);
#pragma unroll
                for (int e = 4; e < 28; e += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) top[u] = max3_or_nan(top[u], __uint_as_float(r[c][e + u]), __uint_as_float(r[c][e + 4 + u]));
#pragma unroll
                for (int u = 0; u < 4; ++u) top[u] = max_or_nan(top[u], __uint_as_float(r[c][28 + u]));
                return max_or_nan(max_or_nan(top[0], top[1]), max_or_nan(top[2], top[3]));
            };
            // The weights of 32 keys, pairs e0 .. e1 - 1.
            auto weights = [&](int c, int e0, int e1, uint64_t base2) {
#pragma unroll
                for (int e = e0; e < e1; ++e) {
                    float x, y;
                    pair_split(pair_fma(pair_of(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), factor2, base2), x, y);
                    x = exp2_approx(x);
                    y = exp2_approx(y);
                    sum2[e & 1] = pair_add(sum2[e & 1], pair_of(x, y));
                    w[e] = head_pack<BF16>(x, y);
                }
            };
            auto total = [&]() {
                float a0, a1, b0, b1;
                pair_split(sum2[0], a0, a1);
                pair_split(sum2[1], b0, b1);
                return (a0 + a1) + (b0 + b1);
            };
            auto stored = [&]() {
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
            };
            auto arrive = [&](uint32_t bar) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            // The last 32 keys' weights; the ones before are handed over when half of them are done, by when they have been stored.
            auto finish = [&](uint64_t base2) {
                constexpr int c = kChunks - 1;
                weights(c, 0, 8, base2);
                if (kEarly < kChunks) {
                    stored();
                    arrive(bar_p(b));
                }
                weights(c, 8, 16, base2);
                tmem_st16(s_at + 16 * c, w);
                stored();
                // (one tile: S(j) says nothing about the P V before this one, and two phases behind would look like none)
                if (kTiles == 1 && j > 0) ok = mbar_wait_warp(bar_o(i), (uint32_t)(j - 1) & 1u, abort_flag, P.status, P.wait_limit);
                if (ok) arrive(kEarly < kChunks ? bar_h(b) : bar_p(b));
            };
#pragma unroll
            for (int c = 0; c < kChunks; ++c) mm_tmem_start(s_at + 32 * c, r[c]);
            mm_tmem_landed();
#pragma unroll
            for (int c = 0; c < kChunks; ++c) mm_tmem_use(r[c]);
            bool done = false;
            if (!masked && __all_sync(0xffffffffu, m > -INFINITY)) {
                // With the maximum as it is, and without looking for this step's: as long as sums of weights stay below 2^12, so does every weight.  (Of the last
                // 32 keys, whose weights come when the others are gone, the maximum does it.)  Half of the instructions.
                const uint64_t base2 = pair_of(-m, -m);
#pragma unroll
                for (int c = 0; c + 1 < kChunks; ++c) {
                    weights(c, 0, 16, base2);
                    tmem_st16(s_at + 16 * c, w);
                }
                const bool fine = total() < 4096.f && peaks(kChunks - 1) * P.factor < m + 12.f;
                done = __all_sync(0xffffffffu, fine || !live);
                if (done) finish(base2);
                else sum2[0] = sum2[1] = 0;
            }
            if (!done) {
                float peak = -INFINITY;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    if (masked) {
                        const int lo = begin - key - 32 * c, hi = end - key - 32 * c;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e < lo || e >= hi) r[c][e] = 0xff800000u;
                    }
                    peak = max_or_nan(peak, peaks(c));
                }
                peak *= P.factor;
                const bool grow = peak > m + kPromptSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float to = grow ? peak : m, shrink = grow ? exp2_approx(m - to) : 1.f;
                    m = to;
                    if (j > 0) {
                        l *= shrink;
                        ok = mbar_wait_warp(bar_o(i), (uint32_t)(j - 1) & 1u, abort_flag, P.status, P.wait_limit);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DP; c += 32) {
                            uint32_t v[32];
                            mm_tmem_start(o_at + c, v);
                            mm_tmem_landed();
                            mm_tmem_use(v);
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * shrink);
                            tmem_st32(o_at + c, v);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                const uint64_t base2 = pair_of(-base, -base);
#pragma unroll
                for (int c = 0; c + 1 < kChunks; ++c) {
                    weights(c, 0, 16, base2);
                    tmem_st16(s_at + 16 * c, w);
                }
                finish(base2);
            }
            if (!ok) break;
            l += total();
        }
        if (ok && n > 0) ok = mbar_wait_warp(bar_o(i), (uint32_t)(n - 1) & 1u, abort_flag, P.status, P.wait_limit);
        tc_fence_after();
        const bool bad = (some && block->bad) || *bad_page;
        const float inv = bad ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : 1.f / l;
        // rows through this tile's queries, which nothing reads any more, 64 columns at a time
        unsigned char* stage = smem + Sh::kQOff + i * Sh::kTileBytes + (warp & 3) * kMmStageOut;
        for (int c = 0; c < d.D && ok; c += 64) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[32] = {}, w[16];
                if (n > 0) {
                    mm_tmem_start(o_at + c + 32 * half, v);
                    mm_tmem_landed();
                    mm_tmem_use(v);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = head_pack<BF16>(__uint_as_float(v[2 * e]) * inv, __uint_as_float(v[2 * e + 1]) * inv);
                mm_stage_row(stage, half, w);
            }
            __syncwarp();
            const int u = lane & 7;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int rr = 4 * k + (lane >> 3), full = 32 * (warp & 3) + rr, tok = full / P.rows, h = full - tok * P.rows;
                if (tok < P.tokens && first + i * P.tokens + tok < q_len && c + 8 * u < d.D) {
                    const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((u ^ (rr & 7)) << 4));
                    uint16_t* out = static_cast<uint16_t*>(d.out) + ((long long)(q_at + first + i * P.tokens + tok) * d.q_heads + kh * P.rows + h) * d.D;
                    *reinterpret_cast<uint4*>(out + c + 8 * u) = v;
                }
            }
        }
    }
    // On an expired wait, give the copies in flight a bounded time to land before shared memory is released.
    if (*abort_flag && threadIdx.x == 0) {
        for (unsigned k = 0; k < (1u << 20); ++k) __nanosleep(64);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int DP, bool BF16>
static int prompt_launch(PromptParams& P, cudaStream_t stream) {
    using Sh = PromptShape<DP>;
    static bool attr_set[64];
    int dev = 0;
    NQ_CUDA_TRY(cudaGetDevice(&dev));
    const void* fn = (const void*)prompt_kernel<DP, BF16>;
    if (!attr_set[dev & 63]) {
        // (the warps' shares of the registers are drawn from what the block is launched with)
        cudaFuncAttributes fa;
        NQ_CUDA_TRY(cudaFuncGetAttributes(&fa, fn));
        if (Sh::kTiles == 2 && fa.numRegs < kPromptRegsLaunch) return NQ_ERR_UNSUPPORTED;
        NQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
        attr_set[dev & 63] = true;
    }
    const nq_attention_desc& d = P.d;
    const int type = BF16 ? kMmBf16 : kMmF16;
    P.tokens = 128 / P.rows;
    P.piece = P.paged && d.page_size < Sh::kKeys ? d.page_size : Sh::kKeys;
    const uint32_t fmt = BF16 ? 1u : 0u, base = 1u << 4 | fmt << 7 | fmt << 10 | (uint32_t)(128 >> 4) << 24;
    P.idesc_s = base | (uint32_t)(Sh::kKeys >> 3) << 17;
    P.idesc_o = base | 1u << 16 | (uint32_t)(DP >> 3) << 17;
    int st = mm_encode_heads(&P.map_q, d.q, type, {d.D, d.q_heads, d.T, 1}, {d.q_head, d.q_token, 0}, {64, P.rows, P.tokens, 1});
    if (st != NQ_OK) return st;
    const int64_t rows = P.paged ? d.page_size : d.Tk, pages = P.paged ? d.pages : 1;
    st = mm_encode_heads(&P.map_k, d.k, type, {d.D, rows, d.k_heads, pages}, {d.k_slot, d.k_head, d.k_page}, {64, P.piece, 1, 1});
    if (st != NQ_OK) return st;
    st = mm_encode_heads(&P.map_v, d.v, type, {d.D, rows, d.k_heads, pages}, {d.v_slot, d.v_head, d.v_page}, {64, P.piece, 1, 1});
    if (st != NQ_OK) return st;
    const int64_t block = (int64_t)Sh::kTiles * P.tokens, ctas = ((d.T + block - 1) / block + d.seqs) * d.k_heads;
    if (ctas > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(Sh::kThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    return launch_dependent(cfg, attr, 0, fn, args);
}

}  // namespace nq

extern "C" int nq_prompt_attention_fwd(const nq_attention_desc* desc, void* status_word, nq_stream_t stream) {
    using namespace nq;
    if (!desc || !status_word) return NQ_ERR_NULL;
    const nq_attention_desc& d = *desc;
    int st = attention_check(d);
    if (st != NQ_OK) return st;
    if (!d.cu_seqlens) return NQ_ERR_NULL;
    if (d.T <= 0 || d.q_heads / d.k_heads > 128) return NQ_ERR_SHAPE;
    if (d.T > 0x3fffffff || d.Tk > 0x3fffffff) return NQ_ERR_TOO_LARGE;
    if (!aligned_to(4, (const char*)d.cu_seqlens, (const char*)d.cu_seqlens_k) || !aligned16(status_word)) return NQ_ERR_ALIGN;
    PromptParams P{};
    P.d = d;
    P.rows = d.q_heads / d.k_heads;
    P.paged = d.block_table != nullptr;
    P.factor = d.scale * 1.44269504088896340736f;
    P.wait_limit = gemm_wait_limit();
    P.status = static_cast<unsigned*>(status_word) + 2;
    if (P.paged) {
        st = attention_cache_check(d);
        if (st != NQ_OK) return st;
        if ((int64_t)d.max_pages * d.page_size > 0x3fffffff) return NQ_ERR_TOO_LARGE;
        P.shift = log2_of(d.page_size);
    } else if (d.Tk <= 0) {
        return NQ_ERR_SHAPE;
    }
    const bool bf = d.dtype == NQ_BF16;
    if (d.D <= 64) return bf ? prompt_launch<64, true>(P, as_stream(stream)) : prompt_launch<64, false>(P, as_stream(stream));
    if (d.D <= 128) return bf ? prompt_launch<128, true>(P, as_stream(stream)) : prompt_launch<128, false>(P, as_stream(stream));
    return bf ? prompt_launch<256, true>(P, as_stream(stream)) : prompt_launch<256, false>(P, as_stream(stream));
}
