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
//   warp 2       values that no query of the block sees, ahead of a window or behind the last token, are set to zero in shared memory: their weights are
//                zero, which a NaN would survive; and whether the cache has all pages of the sequence, also those that other blocks read: beside the products
//   warp 3       which block is next: the CTAs that fit the SMs take the grid's other blocks over one by one (cluster launch control), so that long and short
//                blocks fill the SMs evenly; asked for three steps ahead of a block's end (at its start, the first CTAs took blocks that other SMs were about
//                to start: 138 us instead of 113 for four pieces of 512 tokens behind up to 4096)
//   warps 4-11   softmax, four warps to a tile, a row to a thread; the next S of a tile is ordered behind its P V, the other tile's products run meanwhile
//
// The maximum m is moved, and O multiplied accordingly, only when it grows by more than 2^8: P and its sum have room for that, and the result does not depend on
// m.  Where no row of a warp has a mask in a step, its weights are formed with m as it is, without looking for the step's maximum, and only done again when their sum
// says that it has been left behind by more than 2^12 (half of the instructions of a step).  Results leave through shared memory, 128 bytes of a row at a time.
//
// Few tokens behind many keys are too few blocks for the SMs: a block's steps are then divided among up to 16 CTAs, whose sums a second launch joins.
//
// The weights P are rounded to the operands' 16-bit type for the product with the values (what the tensor cores take): 2^-9 (bf16) or 2^-12 (fp16) of each, not
// enlarged by the average over tokens.  fp16 has subnormals below 2^-14, where a rounding is 2^-25 whatever the weight, and nothing below 2^-25: its weights are formed 2^3
// times as large (m is kept that much below the maximum; 2^(12 + 3) is the most that fp16 holds), so that this is 2^-28 of the largest weight for each key (formed
// as they are, weights of 2^-25.2 are all lost, however many).  The sum l is of the weights ahead of this rounding.
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
    int splits, least;             // parts of a block's steps at most; steps of a part at least
    float factor;                  // scale log2(e)
    float* part;                   // (splits > 1) [block][key head][part][tile]: PromptShape::kPart floats
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
    static constexpr int kStages = DP == 64 ? 8 : 4;
    static constexpr int kThreads = 128 + 128 * kTiles;
    static constexpr int kQOff = 1024, kRingOff = kQOff + kTiles * kTileBytes, kOutOff = kRingOff + kStages * kStageBytes;
    static constexpr int kSmem = 1024 + kOutOff + 4 * kTiles * kMmStageOut;
    static constexpr int kOCol = 256;                             // tensor memory: S at 0, O from here
    static constexpr int kPart = 128 * (DP + 2);                  // of a tile: [columns of four][row][4], then maxima and sums of the rows
    static_assert(kSmem <= 227 * 1024 && kOCol + kTiles * DP <= 512, "shared and tensor memory");
};
constexpr int kPromptRegsLaunch = 168, kPromptRegsIssue = 104, kPromptRegsSoftmax = 200;      // (two tiles) of a thread: at launch, and after the split
static_assert(128 * kPromptRegsIssue + 256 * kPromptRegsSoftmax <= 384 * kPromptRegsLaunch, "register split");
constexpr int kPromptAsk = 3;                                     // steps before a block's end, in which the next one is looked up
constexpr int kPromptParts = 16;                                  // of a block at most
constexpr float kPromptSlack = 8.f;                               // powers of two by which a maximum may be behind
constexpr float kPromptMost = 12.f;                               // and by which weights may exceed 1 where it is not looked for

struct PromptBlock {
    int have;                      // 1; 0: nothing to do; -1: no more blocks
    int head;                      // key head
    int first;                     // first token of the block, within the sequence
    int q_len, k_len;
    int q_at, k_at;                // rows of the sequence's first tokens
    int seq, bad;
    int part, parts;               // of the block's steps
    int number;                    // of the block, in all of them of this key head
};
// What a block has to do.  Query t is at place t + behind.
template <int DP>
struct PromptWork : PromptBlock {
    int behind, k_first;           // (the first key: at the start of a page, or of a step)
    int steps[PromptShape<DP>::kTiles], most;
    int front_rows;                // of the first step, ahead of what any query of the block sees
    int tail_rows;                 // of the last step, that the sequence has
    __device__ __forceinline__ int sees_end(const PromptParams& P, int t) const { return max(0, P.d.causal ? min(k_len, t + behind + 1) : k_len); }
    __device__ __forceinline__ int sees_begin(const PromptParams& P, int t) const { return P.d.window > 0 ? max(0, t + behind + 1 - P.d.window) : 0; }
    __device__ __forceinline__ void read(const PromptParams& P, const volatile PromptBlock* b) {
        have = b->have; head = b->head; first = b->first; q_len = b->q_len; k_len = b->k_len; q_at = b->q_at; k_at = b->k_at; seq = b->seq; bad = b->bad;
        part = b->part; number = b->number;
        divide(P);
    }
    __device__ __forceinline__ void divide(const PromptParams& P) {
        behind = k_len - q_len;
        k_first = sees_begin(P, first) & ~(P.piece - 1);
        front_rows = sees_begin(P, first) - k_first;
        most = 0;
#pragma unroll
        for (int i = 0; i < PromptShape<DP>::kTiles; ++i) {
            const int t = first + i * P.tokens, last = min(t + P.tokens, q_len) - 1;
            steps[i] = have > 0 && t < q_len ? max(0, sees_end(P, last) - k_first + PromptShape<DP>::kKeys - 1) / PromptShape<DP>::kKeys : 0;
            most = max(most, steps[i]);
        }
        parts = 1;
        if (P.splits > 1 && most > P.least) {      // this part's steps
            const int size = max((most + P.splits - 1) / P.splits, P.least), from = part * size;
            parts = (most + size - 1) / size;
            if (part >= parts) have = 0;
            most = have > 0 ? min(most - from, size) : 0;
            k_first += from * PromptShape<DP>::kKeys;
            if (part > 0) front_rows = 0;
#pragma unroll
            for (int i = 0; i < PromptShape<DP>::kTiles; ++i) steps[i] = min(max(steps[i] - from, 0), most);
        } else if (part > 0) {
            have = min(have, 0);
            most = 0;
#pragma unroll
            for (int i = 0; i < PromptShape<DP>::kTiles; ++i) steps[i] = 0;
        }
        tail_rows = k_len - k_first - (most - 1) * PromptShape<DP>::kKeys;
    }
    __device__ __forceinline__ bool fix(int j) const { return (j == 0 && front_rows > 0) || (j == most - 1 && tail_rows < PromptShape<DP>::kKeys); }
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
            B.have = 1;
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

// The next block that has not been started takes this CTA's time instead of an SM's own (16 bytes of answer); whether there was one, and its number.
__device__ __forceinline__ void next_block_ask(uint32_t answer, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool next_block_get(uint32_t answer, int& block) {
    uint32_t some, x;
    asm volatile("{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t"
                 "ld.shared.b128 a, [%2];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}" : "=r"(some), "=r"(x) : "r"(answer) : "memory");
    block = (int)x;
    return some != 0;
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
    auto bar_fix = [&](int s) { return sbase + 8 * (2 * kStages + s); };      // values are there, some of which are to become zeros
    const uint32_t bars = sbase + 24 * kStages;
    const uint32_t bar_q = bars, bar_q_free = bars + 8, bar_answer = bars + 24;
    auto bar_s = [&](int i) { return bars + 32 + 8 * i; };            // S is there (by tile, or with one tile by buffer)
    auto bar_p = [&](int i) { return bars + 48 + 8 * i; };            // P is there, or the first of it
    auto bar_h = [&](int i) { return bars + 64 + 8 * i; };            // the rest of P is there (two tiles)
    auto bar_o = [&](int i) { return bars + 80 + 8 * i; };            // P V has been added (by tile)
    auto bar_info = [&](int i) { return bars + 96 + 8 * i; };         // the number and sequence of a block are there
    auto bar_info_free = [&](int i) { return bars + 112 + 8 * i; };
    const uint32_t bar_ask = bars + 128;                              // a block is nearly done
    // The pages of a block's sequence have been looked at.  Four in turn: warp 2 has at most two blocks more than the softmax warps, for a description waits until they
    // have read the last but one.
    auto bar_pages = [&](int n) { return bars + 136 + 8 * (n & 3); };
    static_assert(24 * kStages + 168 <= 368, "shared memory map");
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + 368);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 372);
    volatile int* bad_pages = reinterpret_cast<volatile int*>(smem + 376);          // four in turn: one of them lies outside the cache
    const uint32_t answer = sbase + 400;
    volatile PromptBlock* info = reinterpret_cast<volatile PromptBlock*>(smem + 416);
    static_assert(416 + 2 * sizeof(PromptBlock) <= 1024, "shared memory map");

    const int block_tokens = kTiles * P.tokens;
    if (warp == 2) {
        if (lane < kStages) {
            mbar_init(bar_full(lane), 1);
            mbar_init(bar_free(lane), 1);
            mbar_init(bar_fix(lane), 1);
        }
        if (lane < 2) {
            mbar_init(bar_s(lane), 1);
            mbar_init(bar_p(lane), 4);
            mbar_init(bar_h(lane), 4);
            mbar_init(bar_o(lane), 1);
            mbar_init(bar_info(lane), 1);
            mbar_init(bar_info_free(lane), 3 + 4 * kTiles);
        }
        if (lane < 4) mbar_init(bar_pages(lane), 1);
        if (lane == 0) {
            mbar_init(bar_q, 1);
            mbar_init(bar_q_free, 1);
            mbar_init(bar_answer, 1);
            mbar_init(bar_ask, 1);
            *abort_flag = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    PromptWork<DP> B;
    // The next block's description, for a warp that keeps it in registers; false: no more, or a wait has expired.  `n` counts blocks.
    auto next_info = [&](int n) {
        if (!mbar_wait_warp(bar_info(n & 1), (uint32_t)(n >> 1) & 1u, abort_flag, P.status, P.wait_limit)) return false;
        B.read(P, info + (n & 1));
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_info_free(n & 1));
        return B.have >= 0;
    };

    if (warp < 4) {
        if constexpr (kTiles == 2) regs_down<kPromptRegsIssue>();
        if (warp == 3) {
            // ------------------------------------------------------------ which blocks
            int index = blockIdx.x, lives = 0;
            bool more = true;
            for (int n = 0;; ++n) {
                PromptBlock next{};
                next.have = -1;
                if (more) {
                    const int unit = index / d.k_heads;
                    next.have = 0;
                    next.head = index - unit * d.k_heads;
                    next.number = unit / P.splits;
                    next.part = unit - next.number * P.splits;
                    prompt_block(P, next.number, block_tokens, next);
                    // rows of no sequence
                    const int head = min(max(__ldcg(d.cu_seqlens), 0), (int)d.T), tail = min(max(__ldcg(d.cu_seqlens + d.seqs), head), (int)d.T);
                    const long long per = (long long)d.q_heads * d.D / 8, missing = ((long long)head + (d.T - tail)) * per;
                    for (long long i = (long long)index * 32 + lane; i < missing; i += (long long)gridDim.x * 32) {
                        const long long at = i < head * per ? i : i - head * per + tail * per;
                        static_cast<uint4*>(d.out)[at] = make_uint4(0, 0, 0, 0);
                    }
                }
                if (!mbar_wait_warp(bar_info_free(n & 1), ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag, P.status, P.wait_limit)) break;
                if (lane == 0) {
                    volatile PromptBlock* to = info + (n & 1);
                    to->have = next.have; to->head = next.head; to->first = next.first; to->q_len = next.q_len; to->k_len = next.k_len;
                    to->q_at = next.q_at; to->k_at = next.k_at; to->seq = next.seq; to->bad = next.bad; to->part = next.part; to->number = next.number;
                    mbar_arrive(bar_info(n & 1));
                }
                __syncwarp();
                if (!more) break;
                // The next one is asked for near the end of this: at once, the first CTAs would take blocks that other SMs are about to start.
                B.read(P, info + (n & 1));
                if (B.most > 0 && !mbar_wait_warp(bar_ask, (uint32_t)lives++ & 1u, abort_flag, P.status, P.wait_limit)) break;
                if (lane == 0) {
                    mbar_expect_tx(bar_answer, 16);
                    next_block_ask(answer, bar_answer);
                }
                __syncwarp();
                if (!mbar_wait_warp(bar_answer, (uint32_t)n & 1u, abort_flag, P.status, P.wait_limit)) break;
                more = next_block_get(answer, index);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
        } else if (warp == 0) {
            // ------------------------------------------------------------ operands
            const int pieces = kKeys / P.piece;
            int s = 0, lives = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int n = 0; ok && next_info(n); ++n) {
                if (B.most == 0) continue;
                const int* table = d.block_table + (P.paged ? (long long)B.seq * d.table_stride : 0);
                for (int j = 0; j < B.most && ok; ++j) {
                    const int key = B.k_first + j * kKeys + lane * P.piece;       // this lane's box
                    const int boxes = P.paged ? min(pieces, (B.k_len - (B.k_first + j * kKeys) + P.piece - 1) / P.piece) : 1;
                    int page = 0, row = B.k_at + key;
                    if (P.paged && lane < boxes) {
                        page = __ldcg(table + (key >> P.shift));
                        row = key & (d.page_size - 1);
                        if (page < 0 || page >= d.pages) page = 0;                // (which warp 2 finds, too)
                    }
                    for (int kv = 0; kv < 2 && ok; ++kv) {
                        ok = mbar_wait_warp(bar_free(s), ph ^ 1, abort_flag, P.status, P.wait_limit);
                        if (!ok) break;
                        const uint32_t bar = kv == 1 && B.fix(j) ? bar_fix(s) : bar_full(s);
                        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(boxes * P.piece * 128 * Sh::kColumns));
                        __syncwarp();
                        if (lane < boxes) {
                            const uint32_t dst = sbase + Sh::kRingOff + s * Sh::kStageBytes + lane * P.piece * 128;
                            for (int c = 0; c < Sh::kColumns; ++c) tma_load_4d(dst + c * kKeys * 128, kv ? &P.map_v : &P.map_k, 64 * c, row, B.head, page, bar);
                        }
                        __syncwarp();
                        if (++s == kStages) { s = 0; ph ^= 1; }
                        if (j == 0 && kv == 0) {
                            // (the queries behind the first keys, which need not wait for the block before)
                            ok = mbar_wait_warp(bar_q_free, ((uint32_t)lives & 1u) ^ 1u, abort_flag, P.status, P.wait_limit);
                            ++lives;
                            if (ok && elect_one()) {
                                const uint32_t bytes = (uint32_t)(P.rows * P.tokens * 128 * Sh::kColumns);
                                int tiles = 0;
                                for (int i = 0; i < kTiles; ++i) tiles += B.steps[i] > 0;
                                mbar_expect_tx(bar_q, tiles * bytes);
                                for (int i = 0; i < kTiles; ++i) {
                                    if (B.steps[i] == 0) continue;
                                    for (int c = 0; c < Sh::kColumns; ++c)
                                        tma_load_4d(sbase + Sh::kQOff + i * Sh::kTileBytes + c * 128 * 128, &P.map_q, 64 * c, B.head * P.rows, B.q_at + B.first + i * P.tokens, 0, bar_q);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
            }
        } else if (warp == 1) {
            if (elect_one()) {
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
                int at = 0, lives = 0;             // places in the ring; blocks with keys
                int count[kTiles] = {};            // steps of a tile
                bool ok = true;
                for (int n = 0; ok; ++n) {
                    ok = wait(bar_info(n & 1), (uint32_t)(n >> 1) & 1u);
                    if (!ok) break;
                    B.read(P, info + (n & 1));
                    mbar_arrive(bar_info_free(n & 1));
                    if (B.have < 0) break;
                    if (B.most == 0) continue;
                    ok = wait(bar_q, (uint32_t)lives & 1u) && wait(bar_full(at % kStages), parity(at));
                    ++lives;
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
                        if (B.steps[i] > 0) product_s(i, kTiles == 1 ? count[0] & 1 : 0, stage(at));
                    mm_commit<1>(bar_free(at % kStages));
                    if (B.most == 1) mm_commit<1>(bar_q_free);
                    for (int j = 0; j < B.most && ok; ++j) {
                        const int nv = at + 2 * j + 1, nk = nv + 1;      // places of these values and of the next keys in the ring
                        if (j == max(0, B.most - kPromptAsk)) mbar_arrive(bar_ask);
                        const bool next = j + 1 < B.most;
                        if constexpr (kTiles == 1) {
                            // the next S before this P: two buffers
                            const int c = count[0], b = c & 1;
                            if (next) {
                                ok = wait(bar_full(nk % kStages), parity(nk));
                                if (!ok) break;
                                product_s(0, b ^ 1, stage(nk));
                                mm_commit<1>(bar_free(nk % kStages));
                                if (j + 2 == B.most) mm_commit<1>(bar_q_free);
                            }
                            ok = wait(bar_full(nv % kStages), parity(nv)) && wait(bar_p(b), (uint32_t)(c >> 1) & 1u);
                            if (!ok) break;
                            product_o(0, b, stage(nv), 0, 2 * Sh::kEarly, j > 0);
                            mm_commit<1>(bar_o(0));
                            ++count[0];
                        } else {
                            ok = wait(bar_full(nv % kStages), parity(nv));
                            bool keys = false;
#pragma unroll
                            for (int i = 0; i < kTiles; ++i) {
                                if (!ok || j >= B.steps[i]) continue;
                                ok = wait(bar_p(i), (uint32_t)count[i] & 1u);
                                if (!ok) continue;
                                product_o(i, 0, stage(nv), 0, 2 * Sh::kEarly, j > 0);
                                ok = wait(bar_h(i), (uint32_t)count[i] & 1u);
                                if (!ok) continue;
                                product_o(i, 0, stage(nv), 2 * Sh::kEarly, kKeys / 16, true);
                                mm_commit<1>(bar_o(i));
                                ++count[i];
                                if (j + 1 < B.steps[i]) {
                                    if (!keys) ok = wait(bar_full(nk % kStages), parity(nk));
                                    keys = true;
                                    if (ok) product_s(i, 0, stage(nk));
                                }
                            }
                            if (!ok) break;
                            if (next) mm_commit<1>(bar_free(nk % kStages));
                            if (j + 2 == B.most) mm_commit<1>(bar_q_free);
                        }
                        mm_commit<1>(bar_free(nv % kStages));
                    }
                    at += 2 * B.most;
                }
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------------ values that no query of a block sees, pages that are not there
            // (a part of a block looks at its share of the pages: the join behind sees all parts)
            auto look = [&](int n) {
                const int* table = d.block_table + (long long)B.seq * d.table_stride;
                const int page0 = B.sees_begin(P, 0) >> P.shift, pages = B.have > 0 ? ((B.k_len + d.page_size - 1) >> P.shift) - page0 : 0;
                const int to = page0 + (int)((long long)pages * (B.part + 1) / B.parts);
                bool bad = false;
#pragma unroll 8
                for (int i = page0 + (int)((long long)pages * B.part / B.parts) + lane; i < to; i += 32) {
                    const int page = __ldcg(table + i);
                    bad |= page < 0 || page >= d.pages;
                }
                bad = __any_sync(0xffffffffu, bad);
                if (lane == 0) {
                    bad_pages[n & 3] = bad;
                    mbar_arrive(bar_pages(n));
                }
                __syncwarp();
            };
            int at = 0;
            uint32_t phases = 0;                   // of the stages' barriers, a bit each
            bool ok = true;
            for (int n = 0; ok && next_info(n); ++n) {
                if (P.paged) look(n);              // (a description comes some steps before the block before it is done)
                for (int j = 0; j < B.most && ok; j = j == 0 && B.most > 1 ? B.most - 1 : B.most) {
                    if (!B.fix(j)) continue;
                    const int s = (at + 2 * j + 1) % kStages;
                    ok = mbar_wait_warp(bar_fix(s), phases >> s & 1u, abort_flag, P.status, P.wait_limit);
                    if (!ok) break;
                    phases ^= 1u << s;
                    unsigned char* to = smem + Sh::kRingOff + s * Sh::kStageBytes;
                    auto clear = [&](int row, int rows) {
                        for (int i = lane; i < 8 * rows * Sh::kColumns; i += 32) {           // 16 bytes each
                            const int c = i / (8 * rows);
                            *reinterpret_cast<uint4*>(to + c * kKeys * 128 + row * 128 + (i - c * 8 * rows) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    };
                    if (j == 0) clear(0, B.front_rows);
                    if (j == B.most - 1 && B.tail_rows < kKeys) clear(B.tail_rows, kKeys - B.tail_rows);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_full(s));
                }
                at += 2 * B.most;
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax
        if constexpr (kTiles == 2) regs_up<kPromptRegsSoftmax>();
        constexpr int kChunks = kKeys / 32, kEarly = Sh::kEarly;
        constexpr float kLift = BF16 ? 0.f : 3.f, kMostWeight = BF16 ? 4096.f : 32768.f;       // 2^(kPromptMost + kLift)
        const int i = (warp - 4) >> 2, row = 32 * (warp & 3) + lane;
        const int token = row / P.rows;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t o_at = tmem + lanes + Sh::kOCol + i * DP;
        const uint32_t out_stage = sbase + Sh::kOutOff + (warp - 4) * kMmStageOut;
        const int magic = (65536 + P.rows - 1) / P.rows;                 // (x / rows = x magic / 65536 for x < 128)
        int count = 0;                             // steps of this tile
        bool ok = true;
        for (int block = 0; ok && next_info(block); ++block) {
          if (B.have == 0) continue;
          const int first = B.first + i * P.tokens, t = first + token, left = B.q_len - first;       // (tokens of the sequence from the tile's first on)
          const bool live = token < P.tokens && token < left;
          const int begin = B.sees_begin(P, t), end = live ? B.sees_end(P, t) : 0, k_first = B.k_first;
          float m = live && begin < end ? -INFINITY : 0.f, l = 0.f;      // (rows that are not there, or see nothing, hold nobody up)
          const int n = kTiles == 1 ? B.most : (i == 0 ? B.steps[0] : B.steps[kTiles - 1]);
          for (int j = 0; j < n; ++j, ++count) {
            const int b = kTiles == 1 ? count & 1 : i;
            ok = mbar_wait_warp(bar_s(b), (uint32_t)(kTiles == 1 ? count >> 1 : count) & 1u, abort_flag, P.status, P.wait_limit);
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
                if (kTiles == 1 && j > 0) ok = mbar_wait_warp(bar_o(i), (uint32_t)(count - 1) & 1u, abort_flag, P.status, P.wait_limit);
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
                const bool fine = total() < kMostWeight && peaks(kChunks - 1) * P.factor < m + (kPromptMost + kLift);
                done = __all_sync(0xffffffffu, fine || !live);
                if (done) {
                    finish(base2);
                } else {                           // (the same columns are stored once more: nothing else orders two stores to tensor memory)
                    sum2[0] = sum2[1] = 0;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
            }
            if (!done) {
                float peak = -INFINITY;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    if (masked) {                  // (most 32s of a step are seen by all of a warp's rows, or end for them without a beginning)
                        const int lo = begin - key - 32 * c, hi = end - key - 32 * c;
                        if (__any_sync(0xffffffffu, hi < 32)) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e >= hi) r[c][e] = 0xff800000u;
                        }
                        if (__any_sync(0xffffffffu, lo > 0)) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e < lo) r[c][e] = 0xff800000u;
                        }
                    }
                    peak = max_or_nan(peak, peaks(c));
                }
                peak *= P.factor;
                const bool grow = peak > m + (kPromptSlack + kLift);
                if (__any_sync(0xffffffffu, grow)) {
                    const float to = grow ? peak - kLift : m, shrink = grow ? exp2_approx(m - to) : 1.f;
                    m = to;
                    if (j > 0) {
                        l *= shrink;
                        ok = mbar_wait_warp(bar_o(i), (uint32_t)(count - 1) & 1u, abort_flag, P.status, P.wait_limit);
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
          if (!ok) break;
          if (n > 0) ok = mbar_wait_warp(bar_o(i), (uint32_t)(count - 1) & 1u, abort_flag, P.status, P.wait_limit);
          tc_fence_after();
          if (ok && P.paged) ok = mbar_wait_warp(bar_pages(block), (uint32_t)(block >> 2) & 1u, abort_flag, P.status, P.wait_limit);
          const bool bad = B.bad || (P.paged && bad_pages[block & 3]);
          if (B.parts > 1) {
            // This part's sums, unnormalised, a row to a thread; joined with the others' by the kernel behind.
            float* const to = P.part + ((((long long)B.number * d.k_heads + B.head) * P.splits + B.part) * kTiles + i) * Sh::kPart + row * 4;
#pragma unroll 1
            for (int c = 0; c < d.D && n > 0 && ok; c += 32) {
                uint32_t v[32];
                mm_tmem_start(o_at + c, v);
                mm_tmem_landed();
                mm_tmem_use(v);
#pragma unroll
                for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(to + (long long)(c + e) * 128) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
            float* const numbers = to - row * 4 + 128 * DP + row;
            numbers[0] = l > 0.f || bad || l != l ? m : -INFINITY;
            numbers[128] = bad ? __int_as_float(0x7fffffff) : l;
            tc_fence_before();
            continue;
          }
          // (no sum: nothing is seen, or, without a maximum, only scores of minus infinity: 0 x infinity, as a softmax of these is)
          const float inv = bad ? __int_as_float(0x7fffffff) : l == 0.f && m > -INFINITY ? 0.f : 1.f / l;
          uint16_t* const out = static_cast<uint16_t*>(d.out) + ((long long)(B.q_at + first) * d.q_heads + B.head * P.rows) * d.D;
          // 64 columns at a time through shared memory, so that eight lanes store a row's 128 bytes (every thread its own row kept the load and store unit busy for 4000 clk);
          // the next block's first products run meanwhile.  (Places are computed here: kept from block to block they would take the registers that a step needs.)
          int ln = lane;
          asm volatile("" : "+r"(ln));
          const uint32_t mine = out_stage + ln * 128, u = ln & 7, r0 = ln >> 3, theirs = out_stage + r0 * 128;
          int place[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int full = 32 * (warp & 3) + 4 * k + r0, tok = (full * magic) >> 16;
            place[k] = tok < P.tokens && tok < left ? (tok * d.q_heads + full - tok * P.rows) * d.D + 8 * (int)u : -1;
          }
#pragma unroll
          for (int c = 0; c < DP; c += 64) {
            if (c >= d.D || !ok) break;
            uint32_t v[2][32] = {};
            if (n > 0) {
                mm_tmem_start(o_at + c, v[0]);
                mm_tmem_start(o_at + c + 32, v[1]);
                mm_tmem_landed();
                mm_tmem_use(v[0]);
                mm_tmem_use(v[1]);
            }
            __syncwarp();                          // (the stores before have read theirs)
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = head_pack<BF16>(__uint_as_float(v[q >> 2][8 * (q & 3) + 2 * e]) * inv, __uint_as_float(v[q >> 2][8 * (q & 3) + 2 * e + 1]) * inv);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(mine + ((q ^ u) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            }
            __syncwarp();
            const bool column = c + 8 * (int)u < d.D;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (place[k] >= 0 && column) {
                    uint4 x;
                    // (row 4 k + r0, unit u)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(theirs + k * 512 + ((u ^ ((4 * k + r0) & 7)) << 4)) : "memory");
                    *reinterpret_cast<uint4*>(out + place[k] + c) = x;
                }
            }
          }
          tc_fence_before();
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

// The parts of blocks that have several.  A CTA has a quarter of a tile's rows, 32, of one key head, and all columns or 32 of them: four threads to a row, eight
// columns at a time; everything a thread needs of up to eight parts is on its way at once (part after part it took 42 us instead of 6 for 16 parts of 64 rows and eight key heads).
template <int DP, bool BF16>
__global__ void __launch_bounds__(128) prompt_join_kernel(const __grid_constant__ PromptParams P) {
    using Sh = PromptShape<DP>;
    constexpr int kTiles = Sh::kTiles;
    const nq_attention_desc& d = P.d;
    const int number = blockIdx.x / d.k_heads, head = blockIdx.x - number * d.k_heads, i = blockIdx.y >> 2;
    const int row = 32 * (blockIdx.y & 3) + (threadIdx.x & 31), quarter = threadIdx.x >> 5;
    // (the lengths are older than the kernel before)
    PromptWork<DP> B;
    B.have = 0;
    prompt_block(P, number, kTiles * P.tokens, B);
    B.head = head;
    B.part = 0;
    B.number = number;
    B.divide(P);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int token = row / P.rows, h = row - token * P.rows, t = B.first + i * P.tokens + token;
    if (B.have <= 0 || B.parts <= 1 || token >= P.tokens || t >= B.q_len) return;
    const float* at = P.part + ((((long long)number * d.k_heads + head) * P.splits) * kTiles + i) * Sh::kPart + row * 4;
    const long long step = (long long)kTiles * Sh::kPart;
    auto number_of = [&](int p, int k) { return __ldcg(at + p * step - row * 4 + 128 * DP + 128 * k + row); };
    uint16_t* out = static_cast<uint16_t*>(d.out) + ((long long)(B.q_at + t) * d.q_heads + head * P.rows + h) * d.D;
    float w[kPromptParts], sums[kPromptParts], top = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < kPromptParts; ++p) {
        w[p] = p < B.parts ? number_of(p, 0) : -INFINITY;
        sums[p] = p < B.parts ? number_of(p, 1) : 0.f;
    }
    for (int c = 8 * (4 * blockIdx.z + quarter); c < d.D; c += 32 * gridDim.z) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll
        for (int p0 = 0; p0 < kPromptParts; p0 += 8) {
            if (p0 >= B.parts) break;
            float4 x[8], y[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                if (p0 + p >= B.parts) continue;
                x[p] = __ldcg(reinterpret_cast<const float4*>(at + (p0 + p) * step + (long long)c * 128));
                y[p] = __ldcg(reinterpret_cast<const float4*>(at + (p0 + p) * step + (long long)(c + 4) * 128));
            }
            if (p0 == 0 && c == 8 * (4 * (int)blockIdx.z + quarter)) {         // the parts' weights, while the sums are on their way
#pragma unroll
                for (int p = 0; p < kPromptParts; ++p) top = fmaxf(top, w[p]);
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int p = 0; p < kPromptParts; ++p) {
                    w[p] = exp2_approx(w[p] - base);
                    l += sums[p] * w[p];
                }
                const float inv = l == 0.f && B.sees_begin(P, t) >= B.sees_end(P, t) ? 0.f : 1.f / l;
#pragma unroll
                for (int p = 0; p < kPromptParts; ++p) w[p] *= inv;
            }
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                const float v = w[p0 + p];
                if (p0 + p >= B.parts || v == 0.f) continue;                   // (a part that saw nothing has left no sums)
                a.x += x[p].x * v; a.y += x[p].y * v; a.z += x[p].z * v; a.w += x[p].w * v;
                b.x += y[p].x * v; b.y += y[p].y * v; b.z += y[p].z * v; b.w += y[p].w * v;
            }
        }
        *reinterpret_cast<uint4*>(out + c) = make_uint4(head_pack<BF16>(a.x, a.y), head_pack<BF16>(a.z, a.w), head_pack<BF16>(b.x, b.y), head_pack<BF16>(b.z, b.w));
    }
}

// Parts of a block's steps.  Blocks are dealt out as CTAs become free; below 1.5 of them for an SM (`blocks` counts a block to each sequence more than there may be) they
// are cut to make two.  Cut by this rule and whole, us in a graph, 32 heads on 8 of 128, bf16, pages of 64: 128 tokens behind 2048 26 and 34, behind 8192 29 and 112; four times
// that 31 and 35, 82 and 122; eight times (128 blocks with work) 56 and 37, 155 and 139.  So parts that the SMs take all at once gain much, and a second turn of them
// costs more than it gains on short caches; which it is depends on the lengths, which the host does not have.  Above the line: four pieces of 512 tokens behind 4096, 126 whole and
// 155 in two; 8192 tokens over themselves, 489 and 630.  Sixteen parts at most (16 tokens behind 131072: 112 us, ten parts 172, eight 202).
// A part has eight steps at least of the keys that there may be (of a prompt over itself, whose blocks see half of it, sixteen: 2048 tokens whole 39 us, in two 59), and
// four of those that there are, where the table is wider than the sequences: of 2048 tokens and a table for 131072, 128 queries take 22 us in parts of four steps, 28 of eight, 38 of
// sixteen, and 16 queries 18, 23, 33.
template <int DP>
static int prompt_splits(const nq_attention_desc& d, int tokens) {
    using Sh = PromptShape<DP>;
    const int64_t block = (int64_t)Sh::kTiles * tokens, blocks = ((d.T + block - 1) / block + d.seqs) * d.k_heads;
    const int64_t keys = d.block_table ? (int64_t)d.max_pages * d.page_size : d.Tk, steps = keys / Sh::kKeys, wanted = 2 * (int64_t)sm_count();
    int64_t n = 4 * blocks >= 3 * wanted ? 1 : (wanted + blocks - 1) / blocks;
    const int64_t most = steps / (d.block_table || d.cu_seqlens_k ? 8 : 16);
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : n > kPromptParts ? kPromptParts : n);
}
template <int DP>
static size_t prompt_scratch(const nq_attention_desc& d) {
    using Sh = PromptShape<DP>;
    const int tokens = 128 / (d.q_heads / d.k_heads), splits = prompt_splits<DP>(d, tokens);
    const int64_t block = (int64_t)Sh::kTiles * tokens, blocks = ((d.T + block - 1) / block + d.seqs) * d.k_heads;
    return splits == 1 ? 0 : (size_t)(blocks * splits * Sh::kTiles) * Sh::kPart * sizeof(float);
}
static size_t prompt_scratch_of(const nq_attention_desc& d) { return d.D <= 64 ? prompt_scratch<64>(d) : d.D <= 128 ? prompt_scratch<128>(d) : prompt_scratch<256>(d); }

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
    P.splits = prompt_splits<DP>(d, P.tokens);
    P.least = 4;                   // (measured at prompt_splits)
    const int64_t block = (int64_t)Sh::kTiles * P.tokens, blocks = ((d.T + block - 1) / block + d.seqs) * d.k_heads, ctas = blocks * P.splits;
    if (ctas > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(Sh::kThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    st = launch_dependent(cfg, attr, 0, fn, args);
    if (st != NQ_OK || P.splits == 1) return st;
    // (32 columns to a CTA as long as the SMs take all CTAs at once)
    cfg.gridDim = dim3((unsigned)blocks, 4 * Sh::kTiles, blocks * 4 * Sh::kTiles * (DP / 32) <= 12 * sm_count() ? DP / 32 : 1);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    return launch_dependent(cfg, attr, 0, (const void*)prompt_join_kernel<DP, BF16>, args);
}

// What does not need a pointer that is followed.
static int prompt_check(const nq_attention_desc& d) {
    int st = attention_check(d);
    if (st != NQ_OK) return st;
    if (!d.cu_seqlens) return NQ_ERR_NULL;
    if (d.T <= 0 || d.q_heads / d.k_heads > 128) return NQ_ERR_SHAPE;
    if (d.T > 0x3fffffff || d.Tk > 0x3fffffff) return NQ_ERR_TOO_LARGE;
    if (!aligned_to(4, (const char*)d.cu_seqlens, (const char*)d.cu_seqlens_k)) return NQ_ERR_ALIGN;
    if (!d.block_table) return d.Tk <= 0 ? NQ_ERR_SHAPE : NQ_OK;
    st = attention_cache_check(d);
    if (st != NQ_OK) return st;
    return (int64_t)d.max_pages * d.page_size > 0x3fffffff ? NQ_ERR_TOO_LARGE : NQ_OK;
}

}  // namespace nq

extern "C" {

size_t nq_prompt_attention_scratch_bytes(const nq_attention_desc* desc) {
    return desc && nq::prompt_check(*desc) == NQ_OK ? nq::prompt_scratch_of(*desc) : 0;
}

int nq_prompt_attention_fwd(const nq_attention_desc* desc, void* scratch, size_t scratch_bytes, void* status_word, nq_stream_t stream) {
    using namespace nq;
    if (!desc || !status_word) return NQ_ERR_NULL;
    const nq_attention_desc& d = *desc;
    const int st = prompt_check(d);
    if (st != NQ_OK) return st;
    if (!aligned16(status_word)) return NQ_ERR_ALIGN;
    const size_t need = prompt_scratch_of(d);
    if (need) {
        if (!scratch) return NQ_ERR_NULL;
        if (!aligned16(scratch)) return NQ_ERR_ALIGN;
        if (scratch_bytes < need) return NQ_ERR_SCRATCH;
    }
    PromptParams P{};
    P.part = static_cast<float*>(scratch);
    P.d = d;
    P.rows = d.q_heads / d.k_heads;
    P.paged = d.block_table != nullptr;
    P.factor = d.scale * 1.44269504088896340736f;
    P.wait_limit = gemm_wait_limit();
    P.status = static_cast<unsigned*>(status_word) + 2;
    if (P.paged) P.shift = log2_of(d.page_size);
    const bool bf = d.dtype == NQ_BF16;
    if (d.D <= 64) return bf ? prompt_launch<64, true>(P, as_stream(stream)) : prompt_launch<64, false>(P, as_stream(stream));
    if (d.D <= 128) return bf ? prompt_launch<128, true>(P, as_stream(stream)) : prompt_launch<128, false>(P, as_stream(stream));
    return bf ? prompt_launch<256, true>(P, as_stream(stream)) : prompt_launch<256, false>(P, as_stream(stream));
}

}  // extern "C"
