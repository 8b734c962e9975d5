// Attention of one new token per sequence over a paged cache.
//
//     o[h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q[h] . k_j - m),   m the largest of these exponents so far
//
// Bound by memory: keys and values are read once, for all the query heads that share them: 4 D bytes for 4 D G operations.  Those G heads are the rows of
// mma.sync.m16n8k16 (up to 16; the instruction's rate is far above what memory delivers, and few rows would leave tcgen05's 128 idle).
//
// Work.  The tokens that a sequence's query sees are cut into steps of 16.  An item is a sequence, a key head and up to 16 of its query heads; the steps of all
// items lie one behind the other, and every CTA takes the same number of them, found from the lengths on the device: batches of any lengths fill the
// SMs evenly, and a captured graph follows the lengths.  Within a CTA each of the four warps takes a contiguous quarter of the CTA's part of an item,
// with a ring of steps of its own in shared memory (cp.async), its own running maximum, sum and accumulators: no barrier in the loop.  The warps' results are
// joined through shared memory.  An item that lies in several CTAs leaves fp32 results (m, sum, unnormalised o) in the scratch, which a
// second, overlapped launch joins in the order of the CTAs.  Batches without long sequences take whole items and need no second launch.
//
// The weights p are rounded to the operands' type for the product with the values: 2^-9 (bf16) or 2^-12 (fp16) of each, which the average over
// tokens does not enlarge.  Sums of p are fp32 sums of the rounded values.
#include "nq_attn.cuh"

namespace nq {

constexpr int kPagedWarps = 4, kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedStep = 16;                  // tokens
constexpr int kPagedRows = 16;                  // query heads of an item at most
constexpr int kPagedWhole = 256;                // caches of up to so many tokens a sequence: whole items

struct PagedParams {
    nq_attention_desc d;
    int shift;                                  // log2(page_size)
    int rows, chunks;                           // query heads to a key head; items of 16 of them
    int whole;                                  // every CTA takes whole items
    float factor;                               // scale log2(e)
    float* part;                                // [CTAs][2][16][DP + 2]
};

// Steps of a sequence's items, and what a step covers.
struct PagedRange {
    int begin, end;                             // tokens seen
    int first, steps;                           // steps of 16 tokens; one at least, so that somebody writes the result
    bool bad;                                   // the table does not hold the sequence
};
__device__ __forceinline__ PagedRange paged_range(const nq_attention_desc& d, int s, int shift) {
    PagedRange r;
    const int n = __ldcg(d.lengths + s);
    r.end = max(n, 0);
    r.bad = (long long)r.end > ((long long)d.max_pages << shift);
    if (r.bad) r.end = 0;
    r.begin = d.window > 0 ? max(r.end - d.window, 0) : 0;
    r.first = r.begin / kPagedStep;
    r.steps = max((r.end + kPagedStep - 1) / kPagedStep - r.first, 1);
    return r;
}

// The sequence that step `at` of all steps lies in, and the steps ahead of it; all steps where `at` is negative.  By the whole CTA.
struct PagedPlace {
    int seq;
    long long before, total;
};
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums) {       // inclusive
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += warp_sums[w];
    __syncthreads();
    return v;
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
// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    const int n = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

template <int DP> struct PagedShape {
    static constexpr int kChunks = DP / 8;                        // 16-byte chunks of a row
    static constexpr int kRowBytes = 2 * DP;
    static constexpr int kTileBytes = kPagedStep * kRowBytes;     // of keys, or of values
    static constexpr int kStages = DP == 64 ? 4 : 3;
    static constexpr int kWarpBytes = 2 * kStages * kTileBytes;
    static constexpr int kSmem = kPagedWarps * kWarpBytes;
    static constexpr int kPart = kPagedRows * (DP + 2);           // floats of a partial result
    static constexpr int kCtasPerSm = DP == 64 ? 3 : DP == 128 ? 2 : 1;
    static_assert(kPagedWarps * kPart * 4 <= kSmem, "the warps' results fit the rings");
};
// Chunk c of row r: eight rows' same chunk lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t paged_at(uint32_t base, int r, int c) { return base + r * PagedShape<DP>::kRowBytes + ((c ^ (r & 7)) << 4); }

template <int DP, bool BF16>
__global__ void __launch_bounds__(kPagedThreads, PagedShape<DP>::kCtasPerSm) paged_kernel(const __grid_constant__ PagedParams P) {
    using S = PagedShape<DP>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan[kPagedWarps];
    __shared__ long long place[2];
    const nq_attention_desc& d = P.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
    const int per_seq = d.k_heads * P.chunks;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // this CTA's steps: [unit, unit_end) of all items' steps
    long long unit, unit_end, seq_before;          // (seq_before: steps ahead of the sequence, of one of its items' kind)
    int seq;
    if (P.whole) {
        seq = blockIdx.x / per_seq;
        const int steps = paged_range(d, seq, P.shift).steps;
        seq_before = 0;
        unit = (long long)(blockIdx.x - seq * per_seq) * steps;
        unit_end = unit + steps;
    } else {
        long long total = 0;
        for (int s0 = 0; s0 < d.seqs; s0 += kPagedThreads) {
            const int s = s0 + threadIdx.x;
            const long long sum = block_scan(s < d.seqs ? (long long)paged_range(d, s, P.shift).steps * per_seq : 0, scan);
            if (threadIdx.x == kPagedThreads - 1) place[0] = sum;
            __syncthreads();
            total += place[0];
            __syncthreads();
        }
        long long share = (total + gridDim.x - 1) / gridDim.x;
        share = max(share, (long long)kPagedWarps);
        unit = share * blockIdx.x;
        unit_end = min(unit + share, total);
        if (unit >= unit_end) return;
        long long before = 0;
        seq = 0;
        seq_before = 0;
        for (int s0 = 0; s0 < d.seqs; s0 += kPagedThreads) {
            const int s = s0 + threadIdx.x;
            const long long n = s < d.seqs ? (long long)paged_range(d, s, P.shift).steps * per_seq : 0, sum = block_scan(n, scan) + before;
            if (n > 0 && sum - n <= unit && unit < sum) {
                place[0] = s;
                place[1] = sum - n;
            }
            if (threadIdx.x == kPagedThreads - 1) scan[0] = sum;
            __syncthreads();
            before = scan[0];
            if (before > unit) {
                seq = (int)place[0];
                seq_before = place[1];
                break;
            }
            __syncthreads();
        }
        __syncthreads();
    }

    while (unit < unit_end) {
        const PagedRange R = paged_range(d, seq, P.shift);
        const long long seq_steps = (long long)R.steps * per_seq;
        if (unit >= seq_before + seq_steps) {      // (whole: never)
            seq_before += seq_steps;
            ++seq;
            continue;
        }
        const int item = (int)((unit - seq_before) / R.steps), from = (int)(unit - seq_before - (long long)item * R.steps);
        const int to = (int)min((long long)R.steps, from + (unit_end - unit));
        const int kh = item / P.chunks, chunk = item - kh * P.chunks;
        const int h0 = kh * P.rows + chunk * kPagedRows, rows = min(kPagedRows, P.rows - chunk * kPagedRows);

        // this warp's steps
        const int mine = (to - from + kPagedWarps - 1) / kPagedWarps;
        const int s0 = from + warp * mine, s1 = min(s0 + mine, to);
        const int* table = d.block_table + (long long)seq * d.table_stride;
        const uint16_t* kbase = static_cast<const uint16_t*>(d.k) + (long long)kh * d.k_head;
        const uint16_t* vbase = static_cast<const uint16_t*>(d.v) + (long long)kh * d.v_head;
        bool bad = R.bad;

        // pages of the next 32 steps' first and (pages of 8) second halves: lane i those of step i
        int page0 = 0, page1 = 0;
        auto pages = [&](int s) {                  // steps s .. s + 31
            const int t = (R.first + s + lane) * kPagedStep;
            auto look = [&](int token) {
                // (only pages that hold a token that is seen)
                if (s + lane >= s1 || token >= R.end || token + min(d.page_size, kPagedStep) <= R.begin) return 0;
                const int p = __ldcg(table + (token >> P.shift));
                if (p < 0 || p >= d.pages) { bad = true; return 0; }
                return p;
            };
            page0 = look(t);
            page1 = d.page_size < kPagedStep ? look(t + 8) : page0;
        };
        auto load = [&](int s, int stage) {        // step s, whose page is held by lane (s - s0) % 32
            const int src = (s - s0) & 31;
            const int pa = __shfl_sync(0xffffffffu, page0, src), pb = __shfl_sync(0xffffffffu, page1, src);
            const uint32_t kt = ring + stage * 2 * S::kTileBytes, vt = kt + S::kTileBytes;
            constexpr int kRowsAtOnce = 32 / S::kChunks > 0 ? 32 / S::kChunks : 1;
            const int c = lane % S::kChunks, r0 = lane / S::kChunks;
            const int token0 = (R.first + s) * kPagedStep;
#pragma unroll
            for (int i = 0; i < kPagedStep; i += kRowsAtOnce) {
                const int r = r0 + i, token = token0 + r;
                const bool live = token >= R.begin && token < R.end && 8 * c < d.D;
                const long long page = r < 8 ? pa : pb, slot = token & (d.page_size - 1);
                copy16(paged_at<DP>(kt, r, c), live ? kbase + page * d.k_page + slot * d.k_slot + 8 * c : kbase, live);
            }
#pragma unroll
            for (int i = 0; i < kPagedStep; i += kRowsAtOnce) {
                const int r = r0 + i, token = token0 + r;
                const bool live = token >= R.begin && token < R.end && 8 * c < d.D;
                const long long page = r < 8 ? pa : pb, slot = token & (d.page_size - 1);
                copy16(paged_at<DP>(vt, r, c), live ? vbase + page * d.v_page + slot * d.v_slot + 8 * c : vbase, live);
            }
        };
        if (s0 < s1) pages(s0);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            if (s0 + i < s1) load(s0 + i, i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }

        // queries: rows g and g + 8 of the MMA
        uint32_t a[DP / 16][4];
        {
            const uint16_t* qp = static_cast<const uint16_t*>(d.q) + (long long)seq * d.q_token + (long long)h0 * d.q_head;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = g + 8 * (i & 1), col = 16 * k + 2 * q + 8 * (i >> 1);
                    a[k][i] = row < rows && col < d.D ? __ldcg(reinterpret_cast<const unsigned*>(qp + (long long)row * d.q_head + col)) : 0u;
                }
            }
        }
        float o[DP / 8][4] = {};
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        for (int s = s0, stage = 0; s < s1; ++s) {
            const int ahead = s + S::kStages - 1;
            if (ahead < s1) {
                if (((ahead - s0) & 31) == 0) pages(ahead);
                load(ahead, stage == 0 ? S::kStages - 1 : stage - 1);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();
            const uint32_t kt = ring + stage * 2 * S::kTileBytes, vt = kt + S::kTileBytes;
            float c[2][4] = {};
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t b[4];
                // matrices: keys 0-7 and 8-15 (lanes 8-15 / 24-31: the second 8 columns)
                ldmatrix4(b, paged_at<DP>(kt, (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                paged_mma<BF16>(c[0], a[k], b[0], b[1]);
                paged_mma<BF16>(c[1], a[k], b[2], b[3]);
            }
            // lane: heads g (c[.][0..1]) and g + 8 (c[.][2..3]), tokens 8 n + 2 q + (i & 1)
            const int token0 = (R.first + s) * kPagedStep;
            if (token0 < R.begin || token0 + kPagedStep > R.end) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int token = token0 + 8 * (i >> 2) + 2 * q + (i & 1);
                    if (token < R.begin || token >= R.end) c[i >> 2][i & 3] = -INFINITY;
                }
            }
            uint32_t p[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = fmaxf(fmaxf(c[0][2 * r], c[0][2 * r + 1]), fmaxf(c[1][2 * r], c[1][2 * r + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float to_m = fmaxf(m[r], top * P.factor), base = to_m == -INFINITY ? 0.f : to_m;
                const float shrink = exp2_approx(m[r] - base);          // (0 at first, exactly 1 where m stays)
                m[r] = to_m;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = exp2_approx(fmaf(c[i >> 1][2 * r + (i & 1)], P.factor, -base));
                p[r] = head_pack<BF16>(e[0], e[1]);
                p[2 + r] = head_pack<BF16>(e[2], e[3]);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += head_float<BF16>(i < 2 ? p[r] : p[2 + r], i & 1);
                l[r] = l[r] * shrink + sum;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][2 * r] *= shrink;
                    o[n][2 * r + 1] *= shrink;
                }
            }
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                // matrices (transposed): tokens 0-7 and 8-15 of columns 16 n .., then of 16 n + 8 ..
                ldmatrix4_trans(b, paged_at<DP>(vt, (lane & 7) + (((lane >> 3) & 1) << 3), 2 * n + (lane >> 4)));
                paged_mma<BF16>(o[2 * n], p, b[0], b[1]);
                paged_mma<BF16>(o[2 * n + 1], p, b[2], b[3]);
            }
            __syncwarp();                          // the stage may be filled again
            if (++stage == S::kStages) stage = 0;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        // a page outside the cache: NaN from here on
        if (__syncthreads_or(bad)) l[0] = l[1] = __int_as_float(0x7fffffff);
        // the warps' results through their rings
        float* box = reinterpret_cast<float*>(smem) + warp * S::kPart;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            float* at = box + row * (DP + 2);
            if (row < rows) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(at + 8 * n + 2 * q) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if (q == 0) *reinterpret_cast<float2*>(at + DP) = make_float2(m[r], l[r]);
            }
        }
        __syncthreads();
        const bool all = from == 0 && to == R.steps;
        float* part = P.part + ((long long)blockIdx.x * 2 + (from == 0 ? 1 : 0)) * S::kPart;
        const float* boxes = reinterpret_cast<const float*>(smem);
        for (int i = threadIdx.x; i < rows * (DP / 2); i += kPagedThreads) {
            const int row = i / (DP / 2), col = 2 * (i - row * (DP / 2));
            const float* at = boxes + row * (DP + 2);
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
            if (all) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                if (col < d.D)
                    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(d.out) + ((long long)seq * d.q_heads + h0 + row) * d.D + col) = head_pack<BF16>(v.x * inv, v.y * inv);
            } else {
                *reinterpret_cast<float2*>(part + row * (DP + 2) + col) = v;
                if (col == 0) *reinterpret_cast<float2*>(part + row * (DP + 2) + DP) = make_float2(top, sum);
            }
        }
        __syncthreads();                           // the rings are filled again
        unit += to - from;
    }
}

// The results of an item that lies in several CTAs of the kernel above, by the CTA of the same number as the first of them.
template <int DP, bool BF16>
__global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(const __grid_constant__ PagedParams P) {
    using S = PagedShape<DP>;
    __shared__ long long scan[kPagedWarps];
    __shared__ long long place[2];
    const nq_attention_desc& d = P.d;
    const int per_seq = d.k_heads * P.chunks;
    // (the lengths are older than the kernel above, which has waited for what wrote them before it let this one start)
    long long total = 0;
    for (int s0 = 0; s0 < d.seqs; s0 += kPagedThreads) {
        const int s = s0 + threadIdx.x;
        const long long sum = block_scan(s < d.seqs ? (long long)paged_range(d, s, P.shift).steps * per_seq : 0, scan);
        if (threadIdx.x == kPagedThreads - 1) place[0] = sum;
        __syncthreads();
        total += place[0];
        __syncthreads();
    }
    long long share = (total + gridDim.x - 1) / gridDim.x;
    share = max(share, (long long)kPagedWarps);
    const long long last = share * (blockIdx.x + 1) - 1;       // this CTA's last step
    bool split = last < total - 1;
    long long begin = 0, end = 0;
    int seq = 0, item = 0;
    if (split) {
        long long before = 0, seq_before = 0;
        for (int s0 = 0; s0 < d.seqs; s0 += kPagedThreads) {
            const int s = s0 + threadIdx.x;
            const long long n = s < d.seqs ? (long long)paged_range(d, s, P.shift).steps * per_seq : 0, sum = block_scan(n, scan) + before;
            if (n > 0 && sum - n <= last && last < sum) {
                place[0] = s;
                place[1] = sum - n;
            }
            if (threadIdx.x == kPagedThreads - 1) scan[0] = sum;
            __syncthreads();
            before = scan[0];
            if (before > last) {
                seq = (int)place[0];
                seq_before = place[1];
                break;
            }
            __syncthreads();
        }
        const int steps = paged_range(d, seq, P.shift).steps;
        item = (int)((last - seq_before) / steps);
        begin = seq_before + (long long)item * steps;
        end = begin + steps;
        split = end > last + 1 && begin >= share * blockIdx.x;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!split) return;
    const int count = (int)((end - 1) / share) - (int)blockIdx.x + 1;
    const int kh = item / P.chunks, chunk = item - kh * P.chunks;
    const int h0 = kh * P.rows + chunk * kPagedRows, rows = min(kPagedRows, P.rows - chunk * kPagedRows);
    // the first piece is its CTA's second result, the others are their CTAs' first
    auto piece = [&](int i) { return P.part + ((long long)(blockIdx.x + i) * 2 + (i == 0)) * S::kPart; };
    for (int i = threadIdx.x; i < rows * (DP / 2); i += kPagedThreads) {
        const int row = i / (DP / 2), col = 2 * (i - row * (DP / 2));
        float top = -INFINITY;
        for (int k = 0; k < count; ++k) top = fmaxf(top, __ldcg(piece(k) + row * (DP + 2) + DP));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float2 v = make_float2(0.f, 0.f);
        for (int k = 0; k < count; ++k) {
            const float* at = piece(k) + row * (DP + 2);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(at + DP)), u = __ldcg(reinterpret_cast<const float2*>(at + col));
            const float e = exp2_approx(ml.x - base);
            sum += ml.y * e;
            v.x += u.x * e;
            v.y += u.y * e;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (col < d.D)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(d.out) + ((long long)seq * d.q_heads + h0 + row) * d.D + col) = head_pack<BF16>(v.x * inv, v.y * inv);
    }
}

static int padded_columns(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
static int paged_ctas(int dp) { return sm_count() * (dp == 64 ? PagedShape<64>::kCtasPerSm : dp == 128 ? PagedShape<128>::kCtasPerSm : PagedShape<256>::kCtasPerSm); }

template <int DP, bool BF16>
static int paged_launch(PagedParams& P, int items, cudaStream_t stream) {
    static bool attr_set[64];
    int dev = 0;
    NQ_CUDA_TRY(cudaGetDevice(&dev));
    const void* fn = (const void*)paged_kernel<DP, BF16>;
    if (!attr_set[dev & 63]) {
        NQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedShape<DP>::kSmem));
        attr_set[dev & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(P.whole ? items : paged_ctas(DP)));
    cfg.blockDim = dim3(kPagedThreads);
    cfg.dynamicSmemBytes = PagedShape<DP>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    const int st = launch_dependent(cfg, attr, 0, fn, args);
    if (st != NQ_OK || P.whole) return st;
    cfg.dynamicSmemBytes = 0;
    return launch_dependent(cfg, attr, 0, (const void*)paged_join_kernel<DP, BF16>, args);
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
    if (seqs <= 0 || q_heads <= 0 || k_heads <= 0 || D <= 0 || D > kHeadMaxCols || max_tokens <= kPagedWhole) return 0;
    const int dp = padded_columns(D);
    return (size_t)paged_ctas(dp) * 2 * kPagedRows * (dp + 2) * sizeof(float);
}

int nq_paged_attention_fwd(const nq_attention_desc* desc, void* scratch, size_t scratch_bytes, nq_stream_t stream) {
    using namespace nq;
    if (!desc) return NQ_ERR_NULL;
    const nq_attention_desc& d = *desc;
    int st = attention_check(d);
    if (st == NQ_OK) st = attention_cache_check(d);
    if (st != NQ_OK) return st;
    PagedParams P{d, log2_of(d.page_size), d.q_heads / d.k_heads, 0, 0, d.scale * 1.44269504088896340736f, static_cast<float*>(scratch)};
    P.chunks = (P.rows + kPagedRows - 1) / kPagedRows;
    const int64_t most = (int64_t)d.max_pages * d.page_size, items = (int64_t)d.seqs * d.k_heads * P.chunks;
    if (most > 0x7fffff00 || items > 0x3fffffff) return NQ_ERR_TOO_LARGE;
    const size_t need = nq_paged_attention_scratch_bytes(d.seqs, d.q_heads, d.k_heads, d.D, most);
    if (need) {
        if (!scratch) return NQ_ERR_NULL;
        if (!aligned16(scratch)) return NQ_ERR_ALIGN;
        if (scratch_bytes < need) return NQ_ERR_SCRATCH;
    }
    P.whole = need == 0;
    const bool bf = d.dtype == NQ_BF16;
    switch (padded_columns(d.D)) {
        case 64: return bf ? paged_launch<64, true>(P, (int)items, as_stream(stream)) : paged_launch<64, false>(P, (int)items, as_stream(stream));
        case 128: return bf ? paged_launch<128, true>(P, (int)items, as_stream(stream)) : paged_launch<128, false>(P, (int)items, as_stream(stream));
        default: return bf ? paged_launch<256, true>(P, (int)items, as_stream(stream)) : paged_launch<256, false>(P, (int)items, as_stream(stream));
    }
}

}  // extern "C"
