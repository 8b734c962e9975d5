// Attention of one new token per sequence over a paged cache.
//
//     o[h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q[h] . k_j - m),   m the largest of these exponents so far, less 8 at most (fp16: less 7 to 15)
//
// Bound by memory: keys and values are read once, for all the query heads that share them: 4 D bytes for 4 D G operations.  Those G heads are the rows of
// mma.sync.m16n8k16 (up to 16; the instruction's rate is far above what memory delivers, and few rows would leave tcgen05's 128 idle).
//
// Work.  The tokens that a sequence's query sees are cut into steps of 16 (heads of up to 64 columns: 32).  An item is a sequence, a key head and up to
// 16 of its query heads.  The steps of all sequences lie one behind the other; a group of warps, one for each key head, takes the same number of them as
// every other group, found from the lengths on the device: batches of any lengths fill the SMs evenly, and a captured graph follows the lengths.  (What
// the heads of a token have in the cache lies side by side and is read at the same time; with one head's steps after the other's, 32 heads on 8 of 64
// columns ran at 5.8 TB/s instead of 6.5, and 64 on 8 of 128 at 6.4 instead of 6.65: eight sequences of 131072 tokens.)  A warp has a ring of steps of its own in shared memory (TMA
// boxes of a page's tokens x 64 columns; it runs on into the next sequence), its own running maximum, sum and accumulators: nothing in the loop waits
// for another warp.  (Copied by cp.async, 16 bytes a lane, the same steps were as fast, but of 650 instructions each instead of 370; bulk copies of 256-byte rows took
// 206 us where these take 153.)  An item that lies in several groups leaves fp32 results (m, sum, unnormalised o) in the scratch, which a second,
// overlapped launch joins in their order.  Where the table has room for short sequences only, a CTA takes an item, its steps divided among the four warps
// and their results joined through shared memory: one launch.
//
// Measured: 32 sequences of up to 4096 tokens, 32 heads of 128, fp16: 107 us, 5.9 TB/s; 4 of up to 131072, 64 heads on 8, bf16: 154 us, 5.9 TB/s, of
// which some 10 us are start, join and the uneven end; one of 1000, 32 heads on 8: 8.7 us, two launches.
//
// The weights p are rounded to the operands' type for the product with the values: 2^-9 (bf16) or 2^-12 (fp16) of each, which the average over
// tokens does not enlarge.  fp16 has subnormals below 2^-14, where a rounding is 2^-25 whatever the weight, and nothing below 2^-25: its weights are formed 2^7 times as
// large (m is kept that much below the maximum; 2^(8 + 7) is the most that fp16 holds), so that this is 2^-32 of the largest weight for each token.  Sums of p are
// fp32 sums of the rounded values.
#include <algorithm>

#include "nq_attn.cuh"
#include "nq_stage.h"
#include "nq_tcgen05.cuh"

namespace nq {

constexpr int kPagedWarps = 4, kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedWhole = 1024;               // tokens of a sequence that a single CTA takes at most
constexpr int kPagedRows = 16;                  // query heads of an item at most

struct alignas(64) PagedParams {
    CUtensorMap map_k, map_v;
    nq_attention_desc d;
    int shift;                                  // log2(page_size)
    int step, box;                              // tokens of a step, and of a box of it (a page's at most)
    int rows, chunks;                           // query heads to a key head; items of 16 of them
    int groups;                                 // of the split kernel: a warp for each key head and 16 of its query heads (`per_seq` of them)
    int piece;                                  // floats of an item's result
    int items;                                  // (of all sequences)
    float factor;                               // scale log2(e)
    unsigned wait_limit;
    unsigned* status;
    float* part;                                // [groups][per_seq][2][query heads of an item][DP + 2]
};

// Steps of a sequence's items, and what they cover.
struct PagedRange {
    int begin, end;                             // tokens seen
    int first, steps;                           // of PagedParams::step tokens; one at least, so that somebody writes the result
    int bad;                                    // the table does not hold the sequence
};
__device__ __forceinline__ PagedRange paged_range(const PagedParams& P, int s) {
    const nq_attention_desc& d = P.d;
    PagedRange r;
    const int n = __ldcg(d.lengths + s);
    r.end = max(n, 0);
    r.bad = (long long)r.end > ((long long)d.max_pages << P.shift);
    if (r.bad) r.end = 0;
    r.begin = d.window > 0 ? max(r.end - d.window, 0) : 0;
    r.first = r.begin / P.step;
    r.steps = max((r.end + P.step - 1) / P.step - r.first, 1);
    return r;
}

// Where a step of all steps lies.
struct PagedPlace {
    long long before;                           // steps ahead of the sequence
    int seq;
    PagedRange range;
};
struct PagedPlan {
    PagedPlace place[kPagedWarps];
    long long sums[32];
};
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {       // inclusive
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();                            // (the sums before have been read)
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    total = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        if (w < warp) v += warp_sums[w];
        total += warp_sums[w];
    }
    return v;
}
// Steps of all sequences.  By the whole CTA.  n, sum and range: of this thread's sequence, for batches of up to as many.
__device__ __forceinline__ long long paged_total(const PagedParams& P, PagedPlan& plan, long long& n, long long& sum, PagedRange& range) {
    long long total = 0;
    for (int s0 = 0; s0 < P.d.seqs; s0 += blockDim.x) {
        const int s = s0 + threadIdx.x;
        n = 0;
        if (s < P.d.seqs) {
            range = paged_range(P, s);
            n = range.steps;
        }
        long long some;
        sum = block_scan(n, plan.sums, some) + total;
        total += some;
    }
    return total;
}
// The sequences that the steps unit(0) .. unit(COUNT - 1) lie in (those that are below the total).
template <int COUNT, class Unit>
__device__ __forceinline__ void paged_find(const PagedParams& P, PagedPlan& plan, long long n, long long sum, PagedRange range, Unit unit) {
    auto look = [&](int s) {
#pragma unroll
        for (int w = 0; w < COUNT; ++w)
            if (n > 0 && sum - n <= unit(w) && unit(w) < sum) plan.place[w] = {sum - n, s, range};
    };
    if (P.d.seqs <= (int)blockDim.x) {
        look(threadIdx.x);
    } else {
        long long before = 0;
        for (int s0 = 0; s0 < P.d.seqs; s0 += blockDim.x) {
            const int s = s0 + threadIdx.x;
            n = 0;
            if (s < P.d.seqs) {
                range = paged_range(P, s);
                n = range.steps;
            }
            long long some;
            sum = block_scan(n, plan.sums, some) + before;
            before += some;
            look(s);
        }
    }
    __syncthreads();
}

template <bool BF16>
__device__ __forceinline__ void paged_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void paged_box(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// A warp's step is bound by its own latency, so what counts is how many warps an SM has, each with one step on its way while it works on another:
// three CTAs of rings of 2 (columns up to 128) took 106 us for 32 sequences of up to 4096 tokens and 32 heads of 128, two of rings of 3 108.5; with heads of 64,
// 8 x 131072 tokens, 369 us and 390 (one CTA: 783).  Of 64 columns a step has 32 tokens: with 16 and four CTAs an SM, 387.  (All before the heads were read side by side.)
template <int DP> struct PagedShape {
    static constexpr int kColumns = DP / 64;                      // boxes of 64 columns: rows of 128 bytes, 128-byte swizzle
    static constexpr int kStep = DP == 64 ? 32 : 16;              // tokens of a step
    static constexpr int kColumnBytes = kStep * 128;
    static constexpr int kTileBytes = kColumns * kColumnBytes;    // of keys, or of values
    static constexpr int kStages = DP <= 128 ? 2 : 3;
    static constexpr int kWarpBytes = 2 * kStages * kTileBytes;
    static constexpr int kBarOff = kPagedWarps * kWarpBytes;
    static constexpr int kSmem = 1024 + kBarOff + 8 * kPagedWarps * kStages;
    static constexpr int kRow = DP + 2;                           // floats of a head's result: o, m, sum
    static constexpr int kPart = kPagedRows * kRow;
    static constexpr int kCtasPerSm = DP <= 128 ? 3 : 1;
    static_assert(kPagedWarps * kPart * 4 <= kBarOff, "the warps' results fit the rings");
    static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "shared memory");
};
// A barrier for every stage of a CTA's warps.
template <int DP>
__device__ __forceinline__ void paged_rings(uint32_t smem) {
    using S = PagedShape<DP>;
    if (threadIdx.x < kPagedWarps * S::kStages) mbar_init(smem + S::kBarOff + 8 * threadIdx.x, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
}
// Waits for a stage by a whole warp; false after `limit` more attempts of some 4 us, which sets the status word.
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, unsigned* status, unsigned limit) {
    for (unsigned i = 0; i <= limit; ++i)
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
    if ((threadIdx.x & 31) == 0) atomicExch(status, (unsigned)(-NQ_ERR_TIMEOUT));
    // (the copies in flight get a bounded time to land before shared memory is released)
    for (unsigned i = 0; i < (1u << 20); ++i) __nanosleep(64);
    return false;
}

// The pages of 32 boxes of an item, one after the other, held by the lanes of a warp.
struct PagedPages {
    int page, from, until;                      // until: the step behind the last whose pages are here
    // From step s on; `to`: steps from there on are not wanted.  False: a page outside the cache.
    template <int STEP>
    __device__ __forceinline__ bool look(const PagedParams& P, int seq, const PagedRange& R, int s, int to) {
        const nq_attention_desc& d = P.d;
        const int boxes = STEP / P.box, lane = threadIdx.x & 31;
        until = s + 32 / boxes;
        from = s;
        const int token = (R.first + s) * STEP + lane * P.box;
        // (only pages that hold a token that is seen)
        page = 0;
        bool bad = false;
        if (s + lane / boxes < to && token < R.end && token + P.box > R.begin) {
            const int p = __ldcg(d.block_table + (long long)seq * d.table_stride + (token >> P.shift));
            if (p < 0 || p >= d.pages) bad = true;
            else page = p;
        }
        return !__any_sync(0xffffffffu, bad);
    }
};
// Keys and values of step s into a stage: boxes of a page's tokens and 64 columns.
template <int DP>
__device__ __forceinline__ void paged_load(const PagedParams& P, const PagedRange& R, const PagedPages& pages, int kh, int s, uint32_t kt, uint32_t bar) {
    using S = PagedShape<DP>;
    const nq_attention_desc& d = P.d;
    const int boxes = S::kStep / P.box, lane = threadIdx.x & 31, token = (R.first + s) * S::kStep + lane * P.box;
    const int page = __shfl_sync(0xffffffffu, pages.page, ((s - pages.from) * boxes + lane) & 31);
    // (a page that holds nothing that is seen is not looked at; of no tokens at all the first box is, so that something arrives)
    const bool mine = lane < boxes && ((token < R.end && token + P.box > R.begin) || (lane == 0 && R.end <= token));
    const unsigned all = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(all) * P.box * 256 * S::kColumns));
    __syncwarp();
    if (mine) {
        const uint32_t dst = kt + lane * P.box * 128;
        const int slot = token & (d.page_size - 1);
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) {
            paged_box(dst + c * S::kColumnBytes, &P.map_k, 64 * c, slot, kh, page, bar);
            paged_box(dst + S::kTileBytes + c * S::kColumnBytes, &P.map_v, 64 * c, slot, kh, page, bar);
        }
    }
    __syncwarp();
}
// Values of a landed step's tokens that are not seen: zeros, for their weights are, which a NaN would survive.
template <int DP>
__device__ __forceinline__ void paged_clear(const PagedRange& R, int s, uint32_t kt) {
    using S = PagedShape<DP>;
    const int lane = threadIdx.x & 31, token0 = (R.first + s) * S::kStep;
    if (token0 >= R.begin && token0 + S::kStep <= R.end) return;
    for (int r = lane; r < S::kStep * S::kColumns; r += 32) {
        const int token = token0 + r % S::kStep;
        if (token < R.begin || token >= R.end)
            for (int u = 0; u < 8; ++u)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(kt + S::kTileBytes + r / S::kStep * S::kColumnBytes + r % S::kStep * 128 + 16 * u), "r"(0) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // (before a later copy to the same place)
    __syncwarp();
}
// Up to 16 heads' queries, accumulators, maxima and sums, as MMA fragments: lane (g, q) has the heads g and g + 8.
template <int DP, bool BF16>
struct PagedHeads {
    uint32_t a[DP / 16][4];
    float o[DP / 8][4], m[2], l[2];

    __device__ __forceinline__ void start(const nq_attention_desc& d, int seq, int h0, int rows) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
        const uint16_t* qp = static_cast<const uint16_t*>(d.q) + (long long)seq * d.q_token + (long long)h0 * d.q_head;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = g + 8 * (i & 1), col = 16 * k + 2 * q + 8 * (i >> 1);
                a[k][i] = row < rows && col < d.D ? __ldcg(reinterpret_cast<const unsigned*>(qp + (long long)row * d.q_head + col)) : 0u;
            }
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
    __device__ __forceinline__ void step(const PagedRange& R, int s, float factor, uint32_t kt) {
        using S = PagedShape<DP>;
        constexpr int kSub = S::kStep / 16;
        const int lane = threadIdx.x & 31, q = lane & 3;
        // 16 bytes number u of row r are at u ^ (r & 7)
        const uint32_t k_at = kt + ((lane & 7) + ((lane >> 4) << 3)) * 128, k_unit = (((lane >> 3) & 1) ^ (lane & 7)) << 4;
        const uint32_t v_at = kt + S::kTileBytes + ((lane & 7) + (((lane >> 3) & 1) << 3)) * 128, v_unit = ((lane >> 4) ^ (lane & 7)) << 4;
        float c[2 * kSub][4] = {};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
            for (int t = 0; t < kSub; ++t) {
                uint32_t b[4];
                // matrices: keys 0-7 and 8-15 (lanes 8-15 / 24-31: the second 8 columns)
                ldmatrix4(b, k_at + 2048 * t + (k >> 2) * S::kColumnBytes + (k_unit ^ (32 * (k & 3))));
                paged_mma<BF16>(c[2 * t], a[k], b[0], b[1]);
                paged_mma<BF16>(c[2 * t + 1], a[k], b[2], b[3]);
            }
        }
        // lane: heads g (c[.][0..1]) and g + 8 (c[.][2..3]), tokens 8 n + 2 q + (i & 1)
        const int token0 = (R.first + s) * S::kStep;
        if (token0 < R.begin || token0 + S::kStep > R.end) {
#pragma unroll
            for (int i = 0; i < 8 * kSub; ++i) {
                const int token = token0 + 8 * (i >> 2) + 2 * q + (i & 1);
                if (token < R.begin || token >= R.end) c[i >> 2][i & 3] = -INFINITY;
            }
        }
        float top[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(c[0][2 * r], c[0][2 * r + 1]);
#pragma unroll
            for (int n = 1; n < 2 * kSub; ++n) top[r] = fmaxf(top[r], fmaxf(c[n][2 * r], c[n][2 * r + 1]));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2)) * factor;
        }
        // The maximum is moved, and o multiplied, only when it grows by more than 2^8: weights and sums have room for that.
        constexpr float kLift = BF16 ? 0.f : 7.f, kBehind = 8.f + kLift;
        if (__any_sync(0xffffffffu, top[0] > m[0] + kBehind || top[1] > m[1] + kBehind)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (!(top[r] > m[r] + kBehind)) continue;
                const float to = top[r] - kLift, shrink = exp2_approx(m[r] - to);      // (0 at first)
                m[r] = to;
                l[r] *= shrink;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][2 * r] *= shrink;
                    o[n][2 * r + 1] *= shrink;
                }
            }
        }
        uint32_t p[kSub][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int t = 0; t < kSub; ++t) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = exp2_approx(fmaf(c[2 * t + (i >> 1)][2 * r + (i & 1)], factor, -base));
                p[t][r] = head_pack<BF16>(e[0], e[1]);
                p[t][2 + r] = head_pack<BF16>(e[2], e[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) l[r] += head_float<BF16>(i < 2 ? p[t][r] : p[t][2 + r], i & 1);
            }
        }
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
#pragma unroll
            for (int t = 0; t < kSub; ++t) {
                uint32_t b[4];
                // matrices (transposed): tokens 0-7 and 8-15 of columns 16 n .., then of 16 n + 8 ..
                ldmatrix4_trans(b, v_at + 2048 * t + (n >> 2) * S::kColumnBytes + (v_unit ^ (32 * (n & 3))));
                paged_mma<BF16>(o[2 * n], p[t], b[0], b[1]);
                paged_mma<BF16>(o[2 * n + 1], p[t], b[2], b[3]);
            }
        }
    }
    // The sums over the lanes of a row; NaN for a sequence that is not there.
    __device__ __forceinline__ void finish(bool bad) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (bad) l[r] = __int_as_float(0x7fffffff);
        }
    }
    __device__ __forceinline__ void save(float* box, int rows) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            float* at = box + row * PagedShape<DP>::kRow;
            if (row < rows) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(at + 8 * n + 2 * q) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if (q == 0) *reinterpret_cast<float2*>(at + DP) = make_float2(m[r], l[r]);
            }
        }
    }
    // (no sum: there is no token, or only scores of minus infinity: 0 x infinity, as a softmax of these is)
    __device__ __forceinline__ void store(const nq_attention_desc& d, int seq, int h0, int rows, bool tokens) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            const float inv = l[r] == 0.f && !tokens ? 0.f : 1.f / l[r];
            uint16_t* at = static_cast<uint16_t*>(d.out) + ((long long)seq * d.q_heads + h0 + row) * d.D;
            if (row < rows) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
                    if (8 * n < d.D) *reinterpret_cast<uint32_t*>(at + 8 * n + 2 * q) = head_pack<BF16>(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
            }
        }
    }
};

// Long caches: the warps of group g have the steps [share g, share (g + 1)) of all sequences' steps, each for its key head: what lies side by side in the cache is
// read at the same time.
template <int DP, bool BF16>
__global__ void __launch_bounds__(kPagedThreads, PagedShape<DP>::kCtasPerSm) paged_split_kernel(const __grid_constant__ PagedParams P) {
    using S = PagedShape<DP>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ PagedPlan plan;
    const nq_attention_desc& d = P.d;
    const int warp = threadIdx.x >> 5;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = smem + warp * S::kWarpBytes, bars = smem + S::kBarOff + 8 * warp * S::kStages;
    paged_rings<DP>(smem);
    const int per_seq = d.k_heads * P.chunks, W = blockIdx.x * kPagedWarps + warp, group = W / per_seq, item = W - group * per_seq;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    long long n, sum;
    PagedRange range;
    const long long total = paged_total(P, plan, n, sum, range), share = (total + P.groups - 1) / P.groups;
    paged_find<kPagedWarps>(P, plan, n, sum, range, [&](int w) { return share * ((blockIdx.x * kPagedWarps + w) / per_seq); });
    const long long unit = share * group;
    if (unit >= total) return;                  // (no barrier behind this)
    const int count = (int)min(share, total - unit);

    const int kh = item / P.chunks, chunk = item - kh * P.chunks;
    const int h0 = kh * P.rows + chunk * kPagedRows, rows = min(kPagedRows, P.rows - chunk * kPagedRows);
    struct Cursor {
        PagedRange R;
        int seq, s;                             // the next step of the sequence
    } load{plan.place[warp].range, plan.place[warp].seq, (int)(unit - plan.place[warp].before)}, at = load;
    auto advance = [&](Cursor& c) {             // (true: behind the last step of a sequence)
        if (++c.s < c.R.steps) return false;
        c.s = 0;
        if (++c.seq < d.seqs) c.R = paged_range(P, c.seq);
        return true;
    };
    PagedPages pages{};
    bool fresh = true;
    unsigned bad_items = 0, load_items = 0;     // (bit i: the i-th item from here on, modulo 32, has a page outside the cache; a ring holds far fewer)
    auto load_next = [&](int i, int stage) {    // step i of this warp's
        if (fresh || load.s >= pages.until) {
            const bool ok = pages.look<S::kStep>(P, load.seq, load.R, load.s, min(load.R.steps, load.s + (count - i)));
            if (!ok) bad_items |= 1u << (load_items & 31);
            fresh = false;
        }
        paged_load<DP>(P, load.R, pages, kh, load.s, ring + stage * 2 * S::kTileBytes, bars + 8 * stage);
        if (advance(load)) {
            fresh = true;
            ++load_items;
            bad_items &= ~(1u << (load_items & 31));
        }
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i)
        if (i < count) load_next(i, i);
    PagedHeads<DP, BF16> heads;
    unsigned at_items = 0;
    uint32_t phase = 0;
    bool begin = true;                          // of an item, here
    int from = at.s;
    for (int i = 0, stage = 0; i < count; ++i) {
        if (begin) {
            heads.start(d, at.seq, h0, rows);
            from = at.s;
            begin = false;
        }
        if (i + S::kStages - 1 < count) load_next(i + S::kStages - 1, stage == 0 ? S::kStages - 1 : stage - 1);
        if (!paged_wait(bars + 8 * stage, phase, P.status, P.wait_limit)) return;
        paged_clear<DP>(at.R, at.s, ring + stage * 2 * S::kTileBytes);
        heads.step(at.R, at.s, P.factor, ring + stage * 2 * S::kTileBytes);
        __syncwarp();                           // the stage may be filled again
        if (++stage == S::kStages) { stage = 0; phase ^= 1; }
        const int seq = at.seq;
        const bool seq_bad = at.R.bad != 0, tokens = at.R.end > 0, last = at.s + 1 == at.R.steps;
        if (last || i + 1 == count) {
            heads.finish(seq_bad || (bad_items >> (at_items & 31) & 1u));
            if (from == 0 && last) heads.store(d, seq, h0, rows, tokens);
            else heads.save(P.part + ((long long)W * 2 + (from == 0 ? 1 : 0)) * P.piece, rows);
            ++at_items;
            begin = true;
        }
        advance(at);
    }
}

// Short caches: a CTA per item, a quarter of its steps to a warp.
template <int DP, bool BF16>
__global__ void __launch_bounds__(kPagedThreads, PagedShape<DP>::kCtasPerSm) paged_whole_kernel(const __grid_constant__ PagedParams P) {
    using S = PagedShape<DP>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const boxes = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const nq_attention_desc& d = P.d;
    const int warp = threadIdx.x >> 5;
    const uint32_t smem = smem_u32(boxes), ring = smem + warp * S::kWarpBytes, bars = smem + S::kBarOff + 8 * warp * S::kStages;
    paged_rings<DP>(smem);
    const int per_seq = d.k_heads * P.chunks, seq = blockIdx.x / per_seq, item = blockIdx.x - seq * per_seq;
    const int kh = item / P.chunks, chunk = item - kh * P.chunks;
    const int h0 = kh * P.rows + chunk * kPagedRows, rows = min(kPagedRows, P.rows - chunk * kPagedRows);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    PagedHeads<DP, BF16> heads;
    heads.start(d, seq, h0, rows);
    const PagedRange R = paged_range(P, seq);
    const int mine = (R.steps + kPagedWarps - 1) / kPagedWarps, s0 = warp * mine, s1 = min(s0 + mine, R.steps);
    static_assert(kPagedWhole / 8 / kPagedWarps <= 32, "one look at the table");
    PagedPages pages{};
    bool bad = R.bad != 0;
    if (!pages.look<S::kStep>(P, seq, R, s0, s1)) bad = true;
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i)
        if (s0 + i < s1) paged_load<DP>(P, R, pages, kh, s0 + i, ring + i * 2 * S::kTileBytes, bars + 8 * i);
    uint32_t phase = 0;
    for (int s = s0, stage = 0; s < s1; ++s) {
        const int ahead = s + S::kStages - 1, to = stage == 0 ? S::kStages - 1 : stage - 1;
        if (ahead < s1) paged_load<DP>(P, R, pages, kh, ahead, ring + to * 2 * S::kTileBytes, bars + 8 * to);
        if (!paged_wait(bars + 8 * stage, phase, P.status, P.wait_limit)) break;
        paged_clear<DP>(R, s, ring + stage * 2 * S::kTileBytes);
        heads.step(R, s, P.factor, ring + stage * 2 * S::kTileBytes);
        __syncwarp();
        if (++stage == S::kStages) { stage = 0; phase ^= 1; }
    }
    heads.finish(__syncthreads_or(bad));
    heads.save(reinterpret_cast<float*>(boxes) + warp * S::kPart, rows);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (DP / 2); i += kPagedThreads) {
        const int row = i / (DP / 2), col = 2 * (i - row * (DP / 2));
        const float* at = reinterpret_cast<const float*>(boxes) + row * S::kRow;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) top = fmaxf(top, at[w * S::kPart + DP]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
            const float e = exp2_approx(at[w * S::kPart + DP] - base);
            const float2 u = *reinterpret_cast<const float2*>(at + w * S::kPart + col);
            sum += at[w * S::kPart + DP + 1] * e;
            v.x += u.x * e;
            v.y += u.y * e;
        }
        const float inv = sum == 0.f && R.end == 0 ? 0.f : 1.f / sum;
        if (col < d.D)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(d.out) + ((long long)seq * d.q_heads + h0 + row) * d.D + col) = head_pack<BF16>(v.x * inv, v.y * inv);
    }
}

// The results of items that lie in several warps of the split kernel.  A CTA has one such item (of few items: the one of its number; of many: the one whose first
// part is at the end of the warp of its number), all of its heads or (gridDim.y) one of them.  The pieces' weights 2^(m - largest m) first, while
// the first pieces are already on their way, then sums over the pieces, column by column, by groups of threads that take turns and add up in their order.
template <int DP, bool BF16, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_join_kernel(const __grid_constant__ PagedParams P) {
    using S = PagedShape<DP>;
    constexpr int kPairs = DP / 2, kGroups = THREADS / kPairs, kWarps = THREADS / 32, kAhead = 8;
    extern __shared__ float weight[];            // of the pieces
    __shared__ PagedPlan plan;
    __shared__ float top_of[kWarps], sum_of[kWarps];
    __shared__ float2 partial[THREADS];
    const nq_attention_desc& d = P.d;
    const int per_seq = d.k_heads * P.chunks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // (the lengths are older than the kernel above, which has waited for what wrote them before it let this one start)
    long long n, sum;
    PagedRange range;
    const long long total = paged_total(P, plan, n, sum, range), share = (total + P.groups - 1) / P.groups;
    int seq;
    const bool by_item = d.seqs <= P.groups;
    const int number = blockIdx.x / per_seq, item = blockIdx.x - number * per_seq;       // of a sequence, or of a group
    if (by_item) {
        seq = number;
        if (d.seqs <= THREADS) {
            if ((int)threadIdx.x == seq) plan.place[0] = {sum - n, seq, range};
        } else {
            long long before = 0;
            for (int s0 = 0; s0 < seq; s0 += THREADS) {
                const int s = s0 + threadIdx.x;
                long long some;
                block_scan(s < seq ? (long long)paged_range(P, s).steps : 0, plan.sums, some);
                before += some;
            }
            if (threadIdx.x == 0) plan.place[0] = {before, seq, paged_range(P, seq)};
        }
        __syncthreads();
    } else {
        paged_find<1>(P, plan, n, sum, range, [&](int) { return share * (number + 1) - 1; });
        if (share * (number + 1) - 1 >= total) {          // (the group has none, or not all, of its steps: nothing of an item behind it)
            asm volatile("griddepcontrol.wait;" ::: "memory");
            return;
        }
        seq = plan.place[0].seq;
    }
    const long long begin = plan.place[0].before, end = begin + plan.place[0].range.steps;
    const long long first = begin / share, last = (end - 1) / share;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (first == last || (!by_item && first != number)) return;
    const int count = (int)(last - first) + 1;
    const int kh = item / P.chunks, chunk = item - kh * P.chunks;
    const int h0 = kh * P.rows + chunk * kPagedRows, rows = min(kPagedRows, P.rows - chunk * kPagedRows);
    const int col = 2 * (threadIdx.x % kPairs), group = threadIdx.x / kPairs;
    for (int row = blockIdx.y; row < rows; row += gridDim.y) {
        // the first piece is its warp's second result, the others are their warps' first
        auto piece = [&](int i) { return P.part + (((first + i) * per_seq + item) * 2 + (i == 0)) * P.piece + row * S::kRow; };
        auto numbers = [&](int k) { return k < count ? __ldcg(reinterpret_cast<const float2*>(piece(k) + DP)) : make_float2(-INFINITY, 0.f); };
        const float2 mine = numbers(threadIdx.x);
        float2 u[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int k = group + i * kGroups;
            u[i] = k < count ? __ldcg(reinterpret_cast<const float2*>(piece(k) + col)) : make_float2(0.f, 0.f);
        }
        float top = mine.x;
        for (int k = threadIdx.x + THREADS; k < count; k += THREADS) top = fmaxf(top, numbers(k).x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        __syncthreads();                         // (the row before is done)
        if (lane == 0) top_of[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, top_of[w]);
        const float base = top == -INFINITY ? 0.f : top;
        float l = 0.f;
        for (int k = threadIdx.x; k < count; k += THREADS) {
            const float2 ml = k == (int)threadIdx.x ? mine : numbers(k);
            const float e = exp2_approx(ml.x - base);
            weight[k] = e;
            l += ml.y * e;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) sum_of[warp] = l;
        __syncthreads();
        l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) l += sum_of[w];
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int k = group + i * kGroups;
            if (k < count) {
                v.x += u[i].x * weight[k];
                v.y += u[i].y * weight[k];
            }
        }
#pragma unroll 8
        for (int k = group + kAhead * kGroups; k < count; k += kGroups) {
            const float2 w = __ldcg(reinterpret_cast<const float2*>(piece(k) + col));
            v.x += w.x * weight[k];
            v.y += w.y * weight[k];
        }
        if constexpr (kGroups > 1) {
            partial[threadIdx.x] = v;
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int k = 1; k < kGroups; ++k) {
                    v.x += partial[threadIdx.x + k * kPairs].x;
                    v.y += partial[threadIdx.x + k * kPairs].y;
                }
        }
        const float inv = 1.f / l;               // (an item of several groups has tokens; no sum: only scores of minus infinity, 0 x infinity)
        if (group == 0 && col < d.D)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(d.out) + ((long long)seq * d.q_heads + h0 + row) * d.D + col) = head_pack<BF16>(v.x * inv, v.y * inv);
    }
}

static int padded_columns(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
static int paged_ctas(int dp) { return sm_count() * (dp == 64 ? PagedShape<64>::kCtasPerSm : dp == 128 ? PagedShape<128>::kCtasPerSm : PagedShape<256>::kCtasPerSm); }

// Whether the table has room for short sequences only: a CTA per item and one launch instead of two, but nothing evens out the lengths.  Heads of 128, 32 on 8, all
// sequences of one length, us whole and split: 1 x 100 tokens 5.0 and 7.3; 1 x 250 7.1 and 7.5; 1 x 500 10.8 and 7.9; 16 x 500 10.8 and 14.4; 16 x 1000 17.8 and 17.3;
// 32 x 1000 25.2 and 31.2; 128 x 1000 89.5 and 98; 16 x 2000 33 and 30; 64 x 2000 100 and 97.
static bool paged_whole(int64_t items, int64_t most) { return most <= 256 || (most <= kPagedWhole && 8 * items >= most); }
// Groups of warps: as many as fit the SMs at once, or, of so many heads that this would leave warps over, four times as many.
static int64_t paged_groups(int dp, int64_t per_seq) {
    const int64_t warps = (int64_t)paged_ctas(dp) * kPagedWarps;
    return 16 * per_seq <= warps ? warps / per_seq : (4 * warps + per_seq - 1) / per_seq;
}
static int paged_piece(int q_heads, int k_heads, int dp) { return std::min(q_heads / k_heads, kPagedRows) * (dp + 2); }
static int64_t paged_items(int64_t seqs, int q_heads, int k_heads) { return seqs * k_heads * ((q_heads / k_heads + kPagedRows - 1) / kPagedRows); }
// What paged_groups and the like can count: the sizes of every description that is taken.
static bool paged_sizes_ok(int seqs, int q_heads, int k_heads, int D, int64_t max_tokens) {
    return seqs > 0 && q_heads > 0 && k_heads > 0 && q_heads % k_heads == 0 && q_heads <= 1 << 16 && D > 0 && D % 8 == 0 && D <= kHeadMaxCols && max_tokens > 0 && max_tokens <= 0x3fffffff &&
           paged_items(seqs, q_heads, k_heads) <= 0x3fffffff;
}
template <int DP, bool BF16>
static int paged_launch(PagedParams& P, bool whole, cudaStream_t stream) {
    static bool attr_set[64];
    int dev = 0;
    NQ_CUDA_TRY(cudaGetDevice(&dev));
    const void *split_fn = (const void*)paged_split_kernel<DP, BF16>, *whole_fn = (const void*)paged_whole_kernel<DP, BF16>;
    if (!attr_set[dev & 63]) {
        NQ_CUDA_TRY(cudaFuncSetAttribute(split_fn, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedShape<DP>::kSmem));
        NQ_CUDA_TRY(cudaFuncSetAttribute(whole_fn, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedShape<DP>::kSmem));
        attr_set[dev & 63] = true;
    }
    const int per_seq = P.d.k_heads * P.chunks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(whole ? P.items : (P.groups * per_seq + kPagedWarps - 1) / kPagedWarps));
    cfg.blockDim = dim3(kPagedThreads);
    cfg.dynamicSmemBytes = PagedShape<DP>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    const int st = launch_dependent(cfg, attr, 0, whole ? whole_fn : split_fn, args);
    if (st != NQ_OK || whole) return st;
    // A CTA for each head while that makes no more of them than the SMs take at once; more threads where an item has many pieces (sequences of 1000 tokens, 32 heads on 8:
    // one of them 8.7 us, with 128 threads 10.8; sixteen 17.4 with 128 and 21.8 with 512).
    const int joins = P.d.seqs <= P.groups ? P.items : P.groups * per_seq, rows = P.rows < kPagedRows ? P.rows : kPagedRows;
    const bool many = (int64_t)P.d.seqs * 32 <= P.groups;
    cfg.gridDim = dim3((unsigned)joins, (unsigned)((int64_t)joins * rows <= 8 * sm_count() ? rows : 1));
    cfg.blockDim = dim3(many ? 512 : 128);
    cfg.dynamicSmemBytes = P.groups * sizeof(float);
    return launch_dependent(cfg, attr, 0, many ? (const void*)paged_join_kernel<DP, BF16, 512> : (const void*)paged_join_kernel<DP, BF16, 128>, args);
}

// What both attention entry points ask of their cache; 0: fine.
int attention_cache_check(const nq_attention_desc& d) {
    if (!d.block_table || !d.lengths) return NQ_ERR_NULL;
    if (d.max_pages <= 0 || d.pages <= 0 || !page_size_ok(d.page_size) || d.table_stride < 0 || !multiple_of_8({d.k_page, d.v_page})) return NQ_ERR_SHAPE;
    if (d.pages > 0x7fffffff || d.page_size > 1 << 20) return NQ_ERR_TOO_LARGE;
    if (!aligned_to(4, (const char*)d.block_table, (const char*)d.lengths)) return NQ_ERR_ALIGN;
    return NQ_OK;
}
int attention_check(const nq_attention_desc& d) {
    if (!d.q || !d.k || !d.v || !d.out) return NQ_ERR_NULL;
    if (d.dtype != NQ_F16 && d.dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (d.seqs <= 0 || d.q_heads <= 0 || d.k_heads <= 0 || d.q_heads % d.k_heads != 0 || d.D <= 0 || d.D % 8 != 0 || d.window < 0 || !(d.scale > 0.f) || d.scale > 1e30f ||
        !multiple_of_8({d.q_token, d.q_head, d.k_slot, d.k_head, d.v_slot, d.v_head}))
        return NQ_ERR_SHAPE;
    if (d.D > kHeadMaxCols || d.q_heads > 1 << 16) return NQ_ERR_TOO_LARGE;
    if (!aligned_to(16, (const char*)d.q, (const char*)d.k, (const char*)d.v, (const char*)d.out)) return NQ_ERR_ALIGN;
    return NQ_OK;
}

}  // namespace nq

extern "C" {

size_t nq_paged_attention_scratch_bytes(int seqs, int q_heads, int k_heads, int D, int64_t max_tokens) {
    using namespace nq;
    if (!paged_sizes_ok(seqs, q_heads, k_heads, D, max_tokens) || paged_whole(paged_items(seqs, q_heads, k_heads), max_tokens)) return 0;
    const int dp = padded_columns(D);
    const int64_t per_seq = paged_items(1, q_heads, k_heads);
    return (size_t)(paged_groups(dp, per_seq) * per_seq) * 2 * paged_piece(q_heads, k_heads, dp) * sizeof(float);
}

int nq_paged_attention_fwd(const nq_attention_desc* desc, void* scratch, size_t scratch_bytes, void* status_word, nq_stream_t stream) {
    using namespace nq;
    if (!desc || !status_word) return NQ_ERR_NULL;
    const nq_attention_desc& d = *desc;
    int st = attention_check(d);
    if (st == NQ_OK) st = attention_cache_check(d);
    if (st != NQ_OK) return st;
    if (!aligned16(status_word)) return NQ_ERR_ALIGN;
    PagedParams P{};
    P.d = d;
    P.shift = log2_of(d.page_size);
    P.rows = d.q_heads / d.k_heads;
    P.factor = d.scale * 1.44269504088896340736f;
    P.wait_limit = gemm_wait_limit();
    P.status = static_cast<unsigned*>(status_word) + 2;
    P.part = static_cast<float*>(scratch);
    P.chunks = (P.rows + kPagedRows - 1) / kPagedRows;
    const int64_t most = (int64_t)d.max_pages * d.page_size, items = paged_items(d.seqs, d.q_heads, d.k_heads);
    if (!paged_sizes_ok(d.seqs, d.q_heads, d.k_heads, d.D, most)) return NQ_ERR_TOO_LARGE;      // (what else it asks for has been checked)
    const size_t need = nq_paged_attention_scratch_bytes(d.seqs, d.q_heads, d.k_heads, d.D, most);
    if (need) {
        if (!scratch) return NQ_ERR_NULL;
        if (!aligned16(scratch)) return NQ_ERR_ALIGN;
        if (scratch_bytes < need) return NQ_ERR_SCRATCH;
    }
    P.items = (int)items;
    const bool whole = need == 0;
    const bool bf = d.dtype == NQ_BF16;
    const int type = bf ? kMmBf16 : kMmF16;
    P.step = padded_columns(d.D) == 64 ? PagedShape<64>::kStep : PagedShape<128>::kStep;
    P.box = d.page_size < P.step ? d.page_size : P.step;
    st = mm_encode_heads(&P.map_k, d.k, type, {d.D, d.page_size, d.k_heads, d.pages}, {d.k_slot, d.k_head, d.k_page}, {64, P.box, 1, 1});
    if (st == NQ_OK) st = mm_encode_heads(&P.map_v, d.v, type, {d.D, d.page_size, d.k_heads, d.pages}, {d.v_slot, d.v_head, d.v_page}, {64, P.box, 1, 1});
    if (st != NQ_OK) return st;
    // (no more groups than the table has steps for: one sequence of 1000 tokens takes 63 of the 222)
    const int dp = padded_columns(d.D);
    P.groups = (int)std::min<int64_t>(paged_groups(dp, (int64_t)d.k_heads * P.chunks), d.seqs * ((most + P.step - 1) / P.step));
    P.piece = paged_piece(d.q_heads, d.k_heads, dp);
    switch (dp) {
        case 64: return bf ? paged_launch<64, true>(P, whole, as_stream(stream)) : paged_launch<64, false>(P, whole, as_stream(stream));
        case 128: return bf ? paged_launch<128, true>(P, whole, as_stream(stream)) : paged_launch<128, false>(P, whole, as_stream(stream));
        default: return bf ? paged_launch<256, true>(P, whole, as_stream(stream)) : paged_launch<256, false>(P, whole, as_stream(stream));
    }
}

}  // extern "C"
