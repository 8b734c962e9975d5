// Softmax cross entropy over the un-quantised head, without the logits:
//
//     l[t, v] = h[t] . w[v]        lse[t] = log sum_v exp(l[t, v])        loss[t] = lse[t] - l[t, target[t]]
//     d[t, v] = g[t] (exp(l[t, v] - lse[t]) - [v = target[t]])            dh = d w        dw = d^T h
//
// Forward: one product whose epilogue keeps, for each token and each tile's half of the columns, the largest logit and the sum of exponentials
// relative to it (fp32), and picks the target's logit; a second kernel joins the pieces of a token in a fixed order.
//
// Backward, over pieces of the vocabulary whose d fits the scratch (kLossPieceBytes): the logits of the piece once more, d from them and
// the kept lse, rounded to the type of the operands (what the tensor cores multiply), then dw of the piece, complete, and the piece's part of
// dh, added in fp32.  So four products in all, 8 T N V operations (T: the tokens that have a target, in larger calls), and no more memory than a piece.  The
// logits in fp32 would save the fourth product, and take 4 T V bytes: 1.2 GB for 2048 tokens and 151936 words.
//
// Bound by the tensor cores from some 300 tokens on, below by reading w (each product once).  2048 tokens, 51200 x 4096, all with a target, us: logits and
// their sums 521, d 560, dw 535, dh 571, the tensor cores busy for 98, 90, 94 and 98 % of the cycles; packing 7, joining 11, preparing 13, adding dh 17.
#include <type_traits>

#include "nq_common.cuh"
#include "nq_mm.cuh"

namespace nq {

// Bytes of d of a piece.  Three products of the backward pass, us at 64 / 128 / 256 / 512 MB: 2048 tokens, 151936 x 4096 6224 / 6079 / 6091 / 5967, 8192 tokens 25478 /
// 25419 / 24933 / 24271, 16384 tokens, 32000 x 4096 11319 / 10386 / 11144 / 11167, 1000 tokens, 128256 x 8192 5357 / 5245 / 5155 / 5170.
constexpr int64_t kLossPieceBytes = 256ll << 20;
constexpr int kLossPieceUnit = 256;
// Steps of 64 products after which a sum leaves the tensor cores, which cut it off towards zero with every instruction (nq_mm.cuh).  Logits: the same in both
// passes, so that the backward's are the numbers that lse came from.  (With whole sums there, p - 1 of a target with p = 0.999 was off by 6 to 19 % at 4096 columns and
// by up to 38 % at 8192.)  Forward level with whole sums, with 256 columns 5 % slower; the backward's logits and d 6 % (4096 columns) to 15 % (2048)
// slower, 2 to 6 % of the pass: a tile's outputs all come at its end.  Sums over tokens and words: of 2048 products, whose error of 1.2e-5
// is far below the outputs' rounding and does not grow with their number (65536 tokens: 4.2e-4 of a whole sum); level with whole sums, with 512 products 9 %
// slower.
constexpr int kLossLogitsChunk = 8, kLossSumsChunk = 32;
constexpr int kLossRows = 16384;           // tokens of a forward product: the scratch holds 8 bytes for each and every 64 to 128 words
constexpr int kLossJoinHere = 8192;        // pieces of all tokens that one CTA joins
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// fp16 holds d as multiples of this fraction of the largest |g|: probabilities down to 4e-9 of it are normal numbers.  (bf16 has the exponents of fp32.)
constexpr float kLossHalfScale = 16384.f;

__device__ __forceinline__ float exp2_fast(float x) {      // 2 ulp, zero below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
struct LossTargets {
    const void* p;
    int wide;            // int64, not int32
    long long ignore;
};
// (through L2, as h: whatever wrote them may have released this kernel early, which the non-coherent path does not allow)
__device__ __forceinline__ long long loss_target(const LossTargets& t, int row) {
    return t.wide ? __ldcg(static_cast<const long long*>(t.p) + row) : (long long)__ldcg(static_cast<const int*>(t.p) + row);
}

// ---------------------------------------------------------------------------
// tokens without a target
// ---------------------------------------------------------------------------
// They need no logits.  Larger calls (loss_packs) pack the rows of the others, so that prompts and padding in a batch cost no products; how many there are
// is known on the device alone, and the products' kernels read it there.
struct LossRows {
    LossTargets targets;
    const uint4* h;
    uint4* out;
    long long ldh;                 // 16-byte units
    int *pos, *words, *live;       // nullable (no packing): [T] a token's row, -1 without a target; [rows] their targets, -1: no word of the vocabulary; number of rows
    int T, V, packs;
    int skip_all;                  // nothing to copy where all tokens have a target
};
__device__ __forceinline__ bool loss_has_target(const LossTargets& t, int row) { return loss_target(t, row) != t.ignore; }
// One CTA of 512 threads takes the tokens first .. first + count - 1 (at most 512).  `each(token, row)` is called by one thread for each of them (row -1: none).
// Every CTA counts the targets in front of its tokens and all of them for itself: no launch, and no wait, for a list.
template <class Each>
__device__ __forceinline__ void loss_copy_rows(const LossRows& R, int first, int count, Each each) {
    __shared__ int sums[16], before[16], rows[512];
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int n = 0;                     // rows of all tokens
    if (R.pos) {
        int ahead = 0;
#pragma unroll 4
        for (int t = tid; t < R.T; t += 512) {
            const int has = loss_has_target(R.targets, t);
            n += has;
            ahead += t < first ? has : 0;
        }
        n = __reduce_add_sync(0xffffffffu, n);
        ahead = __reduce_add_sync(0xffffffffu, ahead);
        if (lane == 0) { sums[warp] = n; before[warp] = ahead; }
        __syncthreads();
        n = ahead = 0;
        for (int i = 0; i < 16; ++i) { n += sums[i]; ahead += before[i]; }
        __syncthreads();
        const bool has = tid < count && loss_has_target(R.targets, first + tid);
        const unsigned mask = __ballot_sync(0xffffffffu, has);
        if (lane == 0) sums[warp] = __popc(mask);
        __syncthreads();
        for (int i = 0; i < warp; ++i) ahead += sums[i];
        const int row = has ? ahead + __popc(mask & ((1u << lane) - 1)) : -1;
        rows[tid] = row;
        if (tid < count) {
            R.pos[first + tid] = row;
            if (has) {
                const long long word = loss_target(R.targets, first + tid);
                R.words[row] = word >= 0 && word < R.V ? (int)word : -1;
            }
            each(first + tid, row);
        }
        if (first == 0 && tid == 0) *R.live = n;
    } else {
        rows[tid] = tid < count && loss_has_target(R.targets, first + tid) ? first + tid : -1;
        if (tid < count) each(first + tid, first + tid);
    }
    __syncthreads();
    if (!R.out || (R.pos && R.skip_all && n == R.T)) return;
    // Rows of the products.  Without packing a token's row is its own, zeros for one without a target, whatever it holds (its d is zero, but zero times a NaN
    // is not); behind packed ones zeros up to a multiple of 64, which a step of the product over tokens reads.
    const int zeros = (max(n, 1) + 63) & ~63;
    for (int i = tid; i < count * R.packs; i += 512) {
        const int k = i / R.packs, c = i - k * R.packs, t = first + k, row = rows[k];
        if (row >= 0) R.out[(long long)row * R.packs + c] = __ldcg(R.h + t * R.ldh + c);
        if (R.pos ? t >= n && t < zeros : row < 0) R.out[(long long)t * R.packs + c] = make_uint4(0, 0, 0, 0);
    }
}
__global__ void __launch_bounds__(512) loss_pack_kernel(const LossRows R, int per_cta) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // (behind the wait: what starts early may rely on everything before)
    const int first = (int)blockIdx.x * per_cta;
    loss_copy_rows(R, first, min(per_cta, R.T - first), [](int, int) {});
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
struct LseEpilogue {
    static constexpr bool kS8 = false, kBuildA = false;
    static constexpr int kChunk = kLossLogitsChunk;
    struct Params {
        LossTargets targets;
        const int* words;          // nullable: the rows' targets (-1: none of the vocabulary's), else `targets` has them
        float2* part;              // [2 n_tiles][T]: largest logit (times log2 e), sum
        float* target_logit;       // [T]
    };
    const Params& p;
    const MmShape& s;
    const volatile MmDims* dims;
    int row, n0, slot;
    long long target;
    float top, sum;
    __device__ LseEpilogue(const Params& p_, const MmShape& s_, const unsigned char*, const volatile MmDims* dims_) : p(p_), s(s_), dims(dims_) {}
    __device__ __forceinline__ void begin(int row_, int n0_, int set, int n_tile, int) {
        row = row_;
        n0 = n0_;
        slot = 2 * n_tile + set;
        target = row >= dims->live ? -1 : p.words ? (long long)__ldcg(p.words + row) : loss_target(p.targets, row);
        top = -INFINITY;
        sum = 0.f;
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int cols, unsigned char*, int) {
        float cm = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < cols) cm = fmaxf(cm, __uint_as_float(r[i]));
        const float m = fmaxf(top, cm * kLog2e), base = m == -INFINITY ? 0.f : m;
        sum *= exp2_fast(top - base);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float a = exp2_fast(fmaf(__uint_as_float(r[i]), kLog2e, -base)), b = exp2_fast(fmaf(__uint_as_float(r[i + 1]), kLog2e, -base));
            if (i < cols) s0 += a;
            if (i + 1 < cols) s1 += b;
        }
        sum += s0 + s1;
        top = m;
        const long long at = target - (n0 + c);
        if (at >= 0 && at < cols) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (at == i) p.target_logit[row] = __uint_as_float(r[i]);
        }
    }
    __device__ __forceinline__ void flush(int, int, const unsigned char*) {}
    __device__ __forceinline__ void end() {
        if (row < dims->live) p.part[(long long)slot * s.M + row] = make_float2(top, sum);
    }
};

__device__ __forceinline__ float2 lse_join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), base = m == -INFINITY ? 0.f : m;
    return make_float2(m, a.y * exp2_fast(a.x - base) + b.y * exp2_fast(b.x - base));
}
__device__ __forceinline__ float2 lse_warp_join(float2 a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = lse_join(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
    return a;
}
// Loss and lse of token r, whose logits are row `at`'s, from its joined pieces.  A target that is no word of the vocabulary (and not `ignore`) makes both NaN.
__device__ __forceinline__ float lse_finish(float2 v, int r, int at, const float* target_logit, const LossTargets& targets, int V, float* lse) {
    const long long t = loss_target(targets, r);
    float l = v.x * kLn2 + logf(v.y), loss = 0.f;
    if (t != targets.ignore) {
        if (t >= 0 && t < V) loss = l - __ldcg(target_logit + at);
        else loss = l = __int_as_float(0x7fffffff);
    }
    lse[r] = l;
    return loss;
}
// ROWS tokens a CTA of 256 threads (so that the CTAs are there before the product's have left): eight, whose pieces lie side by side, or for few tokens
// one, with all threads on its pieces (151936 words have some 1600).
template <int ROWS>
__global__ void __launch_bounds__(256) lse_join_kernel(const float2* part, const float* target_logit, LossTargets targets, float* row_loss, float* lse, const int* pos, int slots, int T, int V, int release) {
    constexpr int kPieces = 256 / ROWS;            // threads of a token
    __shared__ float2 red[ROWS][kPieces / 32 > 1 ? kPieces / 32 : 33];
    const int sub = threadIdx.x % ROWS, piece = threadIdx.x / ROWS, row = blockIdx.x * ROWS + sub, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (release) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float2 v = make_float2(-INFINITY, 0.f);
    const int from = row >= T ? -1 : pos ? __ldcg(pos + row) : row;      // row of the logits (pos: -1 without a target)
    if (from >= 0) {
        int i = piece;
        for (; i + 7 * kPieces < slots; i += 8 * kPieces) {      // eight loads in flight
            float2 p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = __ldcg(part + (long long)(i + kPieces * k) * T + from);
#pragma unroll
            for (int k = 0; k < 8; ++k) v = lse_join(v, p[k]);
        }
        for (; i < slots; i += kPieces) v = lse_join(v, __ldcg(part + (long long)i * T + from));
    }
    int r = blockIdx.x;
    if constexpr (ROWS == 1) {
        v = lse_warp_join(v);
        if (lane == 0) red[0][warp] = v;
        __syncthreads();
        if (warp > 0) return;
        v = lse_warp_join(lane < 8 ? red[0][lane] : make_float2(-INFINITY, 0.f));
    } else {
        red[sub][piece] = v;
        __syncthreads();
        r = blockIdx.x * ROWS + warp;
        v = lse_warp_join(red[warp][lane]);
    }
    if (lane == 0 && r < T) {
        const int at = pos ? __ldcg(pos + r) : r;
        if (at < 0) row_loss[r] = lse[r] = 0.f;
        else row_loss[r] = lse_finish(v, r, at, target_logit, targets, V, lse);
    }
}

// Sum (mean: of the tokens with a target) of the tokens' losses and the number of these tokens; one CTA, a fixed order, 64-bit sums.  With `part` the pieces
// are joined here as well (a warp per token, few of them: one launch less).
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float2* part, const float* target_logit, float* row_loss, float* lse, LossTargets targets, float* out, float* count,
                                                        int slots, int T, int V, int mean) {
    __shared__ double sums[32];
    __shared__ int counts[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    double s = 0;
    int n = 0;
    if (part) {
        for (int r = warp; r < T; r += 32) {
            float2 v = make_float2(-INFINITY, 0.f);
            for (int i = lane; i < slots; i += 32) v = lse_join(v, __ldcg(part + (long long)i * T + r));
            v = lse_warp_join(v);
            if (lane == 0) {
                s += lse_finish(v, r, r, target_logit, targets, V, lse);
                n += loss_target(targets, r) != targets.ignore;
            }
        }
    } else {
        for (int i = threadIdx.x; i < T; i += 1024) {
            s += __ldcg(row_loss + i);
            n += loss_target(targets, i) != targets.ignore;
        }
    }
    auto reduce = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
        }
    };
    reduce();
    if (lane == 0) { sums[warp] = s; counts[warp] = n; }
    __syncthreads();
    if (warp == 0) {
        s = sums[lane];
        n = counts[lane];
        reduce();
        if (lane == 0) {
            *count = (float)n;
            *out = mean ? (float)(s / n) : (float)s;
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// Backward: what the products need, in one launch: the rows of h; row_scale, what d of a row is multiplied by before it is rounded, and (with packing) its lse;
// final_scale, what the products' sums are multiplied by.
struct LossPrepare {
    LossRows rows;
    const float *grad, *count, *lse;
    long long grad_stride;
    float *row_scale, *final_scale, *row_lse;
    int reduction;
    float unit;
};
__global__ void __launch_bounds__(512) loss_prepare_kernel(const LossPrepare P, int per_cta) {
    __shared__ float red[16];
    const LossRows& R = P.rows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, T = R.T, first = (int)blockIdx.x * per_cta;
    const bool none = P.reduction == NQ_REDUCE_NONE;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // (behind the wait, as above)
    float top = 1.f;                       // the largest |grad|, which fp16 is relative to
    if (none && P.unit != 1.f) {
        top = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < T; i += 512)
            if (loss_has_target(R.targets, i)) top = fmaxf(top, fabsf(P.grad[i * P.grad_stride]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) red[warp] = top;
        __syncthreads();
        for (int i = 0; i < 16; ++i) top = fmaxf(top, red[i]);
        if (top == 0.f || top == INFINITY) top = 1.f;
    }
    if (first == 0 && threadIdx.x == 0) {
        float f = none ? top : P.grad[0];
        if (P.reduction == NQ_REDUCE_MEAN) f = *P.count > 0.f ? f / *P.count : 0.f;
        *P.final_scale = f / P.unit;
    }
    loss_copy_rows(R, first, min(per_cta, T - first), [&](int t, int row) {
        if (row < 0) return;
        P.row_scale[row] = !loss_has_target(R.targets, t) ? 0.f : none ? P.grad[t * P.grad_stride] / top * P.unit : P.unit;
        if (R.pos) P.row_lse[row] = __ldcg(P.lse + t);
    });
}

// d of a piece of the vocabulary.
template <int OUT, bool LONG>
struct GradEpilogue {
    static constexpr bool kS8 = false, kBuildA = false;
    static constexpr int kChunk = LONG ? kLossLogitsChunk : 0;
    struct Params {
        LossTargets targets;
        const int* words;          // as in LseEpilogue; then all rows below `live` count
        const float *lse, *row_scale;
        uint16_t* d;
        long long ldd;
        int v0;                    // first word of the piece
    };
    const Params& p;
    const MmShape& s;
    const volatile MmDims* dims;
    int row, n0, at;
    float base, scale;
    bool live;
    __device__ GradEpilogue(const Params& p_, const MmShape& s_, const unsigned char*, const volatile MmDims* dims_) : p(p_), s(s_), dims(dims_) {}
    __device__ __forceinline__ void begin(int row_, int n0_, int, int, int) {
        row = row_;
        n0 = n0_;
        live = false;
        at = -1;
        base = scale = 0.f;
        if (row < dims->live) {
            const long long t = p.words ? (long long)__ldcg(p.words + row) : loss_target(p.targets, row);
            live = p.words || t != p.targets.ignore;
            const long long rel = t - p.v0 - n0;
            at = rel >= 0 && rel < kMmAccCols ? (int)rel : -1;
            base = __ldcg(p.lse + row) * kLog2e;
            scale = __ldcg(p.row_scale + row);
        }
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int, unsigned char* stage, int half) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float d[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float e = exp2_fast(fmaf(__uint_as_float(r[i + k]), kLog2e, -base));
                if (at == c + i + k) e -= 1.f;
                d[k] = live ? e * scale : 0.f;
            }
            w[i / 2] = pack_outputs<OUT>(d[0], d[1], 0);
        }
        mm_stage_row(stage, half, w);
    }
    __device__ __forceinline__ void flush(int c, int cols, const unsigned char* stage) {
        const int row0 = row & ~31;
        mm_store_rows(stage, p.d + row0 * p.ldd + n0 + c, p.ldd, min(32, dims->rows - row0), cols, true);
    }
    __device__ __forceinline__ void end() {}
};

// dw of a piece (or dh): rows of words, times the final scale.
template <int OUT, bool LONG>
struct RowsEpilogue {
    static constexpr bool kS8 = false, kBuildA = false;
    static constexpr int kChunk = LONG ? kLossSumsChunk : 0;
    struct Params {
        const float* final_scale;
        uint16_t* out;
        long long ld;
    };
    const Params& p;
    const MmShape& s;
    int row0, n0;
    float f;
    __device__ RowsEpilogue(const Params& p_, const MmShape& s_, const unsigned char*, const volatile MmDims*) : p(p_), s(s_), f(__ldcg(p_.final_scale)) {}
    __device__ __forceinline__ void begin(int row, int n0_, int, int, int) {
        row0 = row & ~31;
        n0 = n0_;
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int, unsigned char* stage, int half) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack_outputs<OUT>(__uint_as_float(r[2 * i]) * f, __uint_as_float(r[2 * i + 1]) * f, 0);
        mm_stage_row(stage, half, w);
    }
    __device__ __forceinline__ void flush(int c, int cols, const unsigned char* stage) {
        mm_store_rows(stage, p.out + row0 * p.ld + n0 + c, p.ld, min(32, s.M - row0), cols, true);
    }
    __device__ __forceinline__ void end() {}
};

// Partial sums of dh in fp32: [split][128 rows][4 columns][row], so that a warp's stores are whole lines.
template <bool LONG>
struct SumEpilogue {
    static constexpr bool kS8 = false, kBuildA = false;
    static constexpr int kChunk = LONG ? kLossSumsChunk : 0;
    struct Params {
        float4* sums;
        int blocks, quads;         // of 128 rows; of 4 columns, padded to whole tiles
        int add;                   // to what an earlier piece left
    };
    const Params& p;
    const MmShape& s;
    int n0;
    float4* dst;
    __device__ SumEpilogue(const Params& p_, const MmShape& s_, const unsigned char*, const volatile MmDims*) : p(p_), s(s_) {}
    __device__ __forceinline__ void begin(int row, int n0_, int, int, int split) {
        n0 = n0_;
        dst = p.sums + (((long long)split * p.blocks + (row >> 7)) * p.quads + (n0 >> 2)) * 128 + (row & 127);
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int, unsigned char*, int) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float4* q = dst + (long long)((c >> 2) + i) * 128;
            float4 v = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
            if (p.add) {
                const float4 o = __ldcg(q);
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            *q = v;
        }
    }
    __device__ __forceinline__ void flush(int, int, const unsigned char*) {}
    __device__ __forceinline__ void end() {}
};

// dh: the splits' sums, added in order, times the final scale.  32 tokens x 64 columns a CTA.
template <int OUT>
__global__ void __launch_bounds__(256) dh_kernel(const float4* sums, const float* final_scale, uint16_t* dh, long long ld, const int* pos, int T, int N, int blocks, int quads, int splits) {
    __shared__ uint32_t tile[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row0 = blockIdx.x * 32, col0 = blockIdx.y * 64;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float f = __ldcg(final_scale);
    const int from = row0 + lane >= T ? -1 : pos ? __ldcg(pos + row0 + lane) : row0 + lane;      // the token's row, -1: zeros
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int qd = 2 * warp + k, quad = (col0 >> 2) + qd;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (quad < quads && from >= 0) {
#pragma unroll 4
            for (int sp = 0; sp < splits; ++sp) {
                const float4 o = __ldcg(sums + (((long long)sp * blocks + (from >> 7)) * quads + quad) * 128 + (from & 127));
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
        }
        tile[lane][2 * qd] = pack_outputs<OUT>(v.x * f, v.y * f, 0);
        tile[lane][2 * qd + 1] = pack_outputs<OUT>(v.z * f, v.w * f, 0);
    }
    __syncthreads();
    const int r = threadIdx.x >> 3, j = threadIdx.x & 7;
    if (row0 + r < T && col0 + 8 * j < N)               // (N is a multiple of 8)
        *reinterpret_cast<uint4*>(dh + (long long)(row0 + r) * ld + col0 + 8 * j) = make_uint4(tile[r][4 * j], tile[r][4 * j + 1], tile[r][4 * j + 2], tile[r][4 * j + 3]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
static int launch_plain(const void* fn, dim3 grid, int threads, void** args, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    return launch_dependent(cfg, attr, 0, fn, args);
}
static bool loss_pairs(int64_t T) { return T > 128; }
// Whether a call packs the rows that have a target: forward a launch and a copy of h (where rows fall away), some 8 us, against products that take 150 us
// and more and have several tiles of 256 rows.
static bool loss_packs(int64_t T, int64_t N, int64_t V) { return T > 512 && 2.0 * (double)T * (double)N * (double)V > 2e11; }

// Forward: columns of a tile, pieces of a token's logits.
struct LossTiles { int bn, slots; };
static LossTiles loss_tiles(int64_t T, int64_t V) {
    const int cg = loss_pairs(T) ? 2 : 1, bn = mm_tile_cols((int)V, (int)((T + 128 * cg - 1) / (128 * cg)), cg, 64);
    return {bn, 2 * (int)((V + bn - 1) / bn)};
}
// Backward.
struct LossPlan {
    int64_t piece;                       // words
    int d_bn, w_bn, h_bn, h_splits, h_blocks, h_quads;
    bool h_direct;                       // one piece, one split: dh as the product writes it
};
static LossPlan plan_loss(int64_t T, int64_t N, int64_t V) {
    LossPlan p;
    const int cg = loss_pairs(T) ? 2 : 1, groups = sm_count() / cg, m_tiles = (int)((T + 128 * cg - 1) / (128 * cg));
    p.piece = kLossPieceBytes / 2 / T / kLossPieceUnit * kLossPieceUnit;
    if (p.piece < kLossPieceUnit) p.piece = kLossPieceUnit;
    const int64_t all = up(V, kLossPieceUnit);
    if (p.piece > all) p.piece = all;
    else {
        const int64_t pieces = (V + p.piece - 1) / p.piece;      // of equal size
        p.piece = up((V + pieces - 1) / pieces, kLossPieceUnit);
    }
    p.d_bn = mm_tile_cols((int)(p.piece < V ? p.piece : V), m_tiles, cg, 64);
    p.w_bn = N <= 128 ? 128 : 256;
    // dh: few tiles over a long k, in us: rounds of the longest tile (a step takes 0.27, a tile's start and end as much as 8), the launch that adds the
    // splits' sums, and what writing (with several pieces, also reading) and adding them moves.
    // dh alone (the logits' product included), us with 1 / 2 / 4 / 8 splits and as chosen: 128 tokens, 32000 x 2048 212 / 128 / 86 / 68, 66; 512 tokens, 128256 x 2048
    // 779 / 600 / 512 / 501, 499; 1024 tokens 1161 / 927 / 930 / 956, 939; 2048 tokens, 51200 x 4096 1411 / 1427 / 1404 / 1446, 1402; 8192 tokens, 32000 x 2048 1815 /
    // 1814 / 1852 / 1998, 1794 (large ones run at the power limit, where idle SMs leave the others a higher clock).
    p.h_bn = cg == 2 ? (N <= 128 ? 128 : 256) : (N <= 64 ? 64 : N <= 128 ? 128 : 256);
    const int64_t tiles = (int64_t)m_tiles * ((N + p.h_bn - 1) / p.h_bn), steps = ((p.piece < V ? p.piece : V) + 63) / 64;
    const bool one = p.piece >= V && !loss_packs(T, N, V);
    p.h_splits = 1;
    p.h_direct = one;
    double best = 0;
    for (int s = 1; s <= 32 && s <= steps; ++s) {
        const int64_t bytes = s * tiles * p.h_bn * 128 * cg * 4;
        if (s > 1 && bytes > kLossPieceBytes) break;
        const double cost = 0.27 * (double)((tiles * s + groups - 1) / groups) * (double)((steps + s - 1) / s + 8) + (one && s == 1 ? 0. : 5. + (one ? 2 : 4) * (double)bytes * 1e-6 / 5.);
        if (s == 1 || cost < best) { best = cost; p.h_splits = s; p.h_direct = one && s == 1; }
    }
    p.h_blocks = m_tiles * cg;
    p.h_quads = (int)(up(N, p.h_bn) / 4);
    return p;
}
struct LossScratch { int64_t d, h, sums, row_scale, final_scale, pos, words, row_lse, live, bytes; };
static LossScratch loss_scratch(const LossPlan& p, int64_t T, int64_t N, bool packs) {
    LossScratch s;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at += up(bytes, 256); return here; };
    s.d = take(T * p.piece * 2);
    s.h = take(T * N * 2);
    s.sums = take(p.h_direct ? 0 : (int64_t)p.h_splits * p.h_blocks * p.h_quads * 128 * 16);
    s.row_scale = take(T * 4);
    s.final_scale = take(4);
    s.pos = take(packs ? T * 4 : 0);
    s.words = take(packs ? T * 4 : 0);
    s.row_lse = take(packs ? T * 4 : 0);
    s.live = take(packs ? 4 : 0);
    s.bytes = at;
    return s;
}
// Forward: the pieces and the targets' logits of kLossRows tokens, their packed rows, the losses of all.
struct LossFwdScratch { int64_t target_logit, row_loss, h, pos, words, live, bytes; };
static LossFwdScratch loss_fwd_scratch(int64_t T, int64_t N, int64_t V) {
    LossFwdScratch s;
    int64_t part = 0;
    for (int64_t t : {T < kLossRows ? T : (int64_t)kLossRows, T % kLossRows}) {      // (the last product may be another one)
        const int64_t bytes = t > 0 ? loss_tiles(t, V).slots * t * 8 : 0;
        if (bytes > part) part = bytes;
    }
    const int64_t most = T < kLossRows ? T : (int64_t)kLossRows;
    const bool packs = loss_packs(most, N, V);
    s.target_logit = up(part, 256);
    s.row_loss = s.target_logit + up(most * 4, 256);
    s.h = s.row_loss + up(T * 4, 256);
    s.pos = s.h + (packs ? up(most * N * 2, 256) : 0);
    s.words = s.pos + (packs ? up(most * 4, 256) : 0);
    s.live = s.words + (packs ? up(most * 4, 256) : 0);
    s.bytes = s.live + (packs ? 256 : 0);
    return s;
}
static int check_loss(int64_t T, int64_t N, int64_t V, int64_t ldh, int64_t ldw, int dtype, int reduction, int target_bits) {
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (target_bits != 32 && target_bits != 64) return NQ_ERR_DTYPE;
    if (reduction < NQ_REDUCE_NONE || reduction > NQ_REDUCE_MEAN) return NQ_ERR_UNSUPPORTED;
    if (T < 1 || N < 1 || V < 1 || N % 8 || ldh < N || ldh % 8 || ldw < N || ldw % 8) return NQ_ERR_SHAPE;
    if (T > (1 << 22) || N > (1 << 20) || V > (1 << 24)) return NQ_ERR_TOO_LARGE;
    return NQ_OK;
}

// Tokens of a CTA that copies rows: so many CTAs that a copy takes microseconds, no more than four to an SM.
static int rows_per_cta(int64_t T) {
    int64_t per = (T + 4 * sm_count() - 1) / (4 * sm_count());
    return (int)(per < 4 ? 4 : per > 512 ? 512 : per);
}

// `packed` (with `live`): the rows of h that have a target, read where they are fewer than all.
template <int CG>
static int launch_lse(const void* h, const void* packed, const int* live, const void* w, const LseEpilogue::Params& e, int T, int N, int V, int64_t ldh, int64_t ldw,
                      int type, int bn, unsigned* status, cudaStream_t stream) {
    MmParams<LseEpilogue> P = {};
    P.e = e;
    if (live) {
        P.s.live = live;
        P.s.live_alt = 1;
        const int st = mm_encode(&P.map_alt, packed, type, N, T, (int64_t)N * 2, 64, CG == 2 || T >= 128 ? 128 : (T + 7) / 8 * 8);
        if (st != NQ_OK) return st;
    }
    return mm_launch<CG>(P, type, {h, ldh * 2, 0}, {w, ldw * 2, 0}, T, V, N, bn, 1, 0, 1, status, stream);
}

// `run` with the kernels that add a sum of k products up by chunks of `steps`, or, where one chunk is all of it, with those that keep no sums in registers and
// write outputs as they are loaded (logits and dw of one token, 151936 x 4096, 490 us instead of 600).
template <class Run>
static int by_length(int64_t k, int steps, Run run) {
    return k > 64 * steps ? run(std::true_type()) : run(std::false_type());
}

template <int CG, int OUT>
static int launch_backward(const void* h, const void* w, const LossTargets& targets, const float* lse, void* dh, void* dw, char* scratch,
                           const LossPlan& p, const LossScratch& at, int T, int N, int V, int64_t ldh, int64_t ldw, int64_t lddh, int64_t lddw,
                           unsigned* status, cudaStream_t stream) {
    const int type = OUT == kOutFp16 ? kMmF16 : kMmBf16;
    uint16_t* d = reinterpret_cast<uint16_t*>(scratch + at.d);
    const float* final_scale = reinterpret_cast<float*>(scratch + at.final_scale);
    const bool packs = loss_packs(T, N, V);
    const int *pos = packs ? reinterpret_cast<int*>(scratch + at.pos) : nullptr, *live = packs ? reinterpret_cast<int*>(scratch + at.live) : nullptr;
    const int* words = packs ? reinterpret_cast<int*>(scratch + at.words) : nullptr;
    const void* rows = packs ? scratch + at.h : h;      // of the logits
    const int64_t ld_rows = packs ? N : ldh;
    if (packs) lse = reinterpret_cast<float*>(scratch + at.row_lse);
    int splits = p.h_splits;
    for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
        const int vc = (int)(V - v0 < p.piece ? V - v0 : p.piece);
        const char* wp = static_cast<const char*>(w) + v0 * ldw * 2;
        int st = by_length(N, kLossLogitsChunk, [&](auto is_long) {
            MmParams<GradEpilogue<OUT, is_long>> P = {};
            const typename GradEpilogue<OUT, is_long>::Params e = {targets, words, lse, reinterpret_cast<float*>(scratch + at.row_scale), d, p.piece, (int)v0};
            P.e = e;
            P.s.live = live;
            return mm_launch<CG>(P, type, {rows, ld_rows * 2, 0}, {wp, ldw * 2, 0}, T, vc, N, p.d_bn, 1, 1, 1, status, stream);
        });
        if (st != NQ_OK) return st;
        if (dw) {
            st = by_length(T, kLossSumsChunk, [&](auto is_long) {
                MmParams<RowsEpilogue<OUT, is_long>> P = {};
                P.e = {final_scale, static_cast<uint16_t*>(dw) + v0 * lddw, lddw};
                P.s.live = live;
                P.s.live_k = 1;
                return mm_launch<2>(P, type, {d, p.piece * 2, 1, up(vc, 64)}, {scratch + at.h, (int64_t)N * 2, 1}, vc, N, T, p.w_bn, 1, 0, dh || v0 + p.piece < V, status, stream);
            });
            if (st != NQ_OK) return st;
        }
        if (dh && p.h_direct)
            return by_length(vc, kLossSumsChunk, [&](auto is_long) {
                MmParams<RowsEpilogue<OUT, is_long>> P = {};
                P.e = {final_scale, static_cast<uint16_t*>(dh), lddh};
                return mm_launch<CG>(P, type, {d, p.piece * 2, 0}, {wp, ldw * 2, 1}, T, N, vc, p.h_bn, 1, 1, 0, status, stream);
            });
        if (dh) {
            int made = 0;
            st = by_length((vc + splits - 1) / splits, kLossSumsChunk, [&](auto is_long) {
                MmParams<SumEpilogue<is_long>> P = {};
                P.e = {reinterpret_cast<float4*>(scratch + at.sums), p.h_blocks, p.h_quads, v0 > 0};
                P.s.live = live;
                const int r = mm_launch<CG>(P, type, {d, p.piece * 2, 0}, {wp, ldw * 2, 1}, T, N, vc, p.h_bn, splits, 1, 1, status, stream);
                made = P.s.splits;
                return r;
            });
            if (st != NQ_OK) return st;
            if (v0 == 0) splits = made;                        // (the last piece may be shorter and have fewer)
        }
    }
    if (dh) {
        const void* fn = (const void*)dh_kernel<OUT>;
        const float4* sums = reinterpret_cast<const float4*>(scratch + at.sums);
        long long ld = lddh;
        int blocks = p.h_blocks, quads = p.h_quads;
        void* args[] = {&sums, &final_scale, &dh, &ld, &pos, &T, &N, &blocks, &quads, &splits};
        return launch_plain(fn, dim3((T + 31) / 32, (N + 63) / 64), 256, args, stream);
    }
    return NQ_OK;
}

}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_linear_ce_fwd_scratch_bytes(int64_t T, int64_t N, int64_t V) {
    if (check_loss(T, N, V, N, N, NQ_F16, NQ_REDUCE_NONE, 64) != NQ_OK) return 0;
    return (size_t)loss_fwd_scratch(T, N, V).bytes;
}

int nq_linear_ce_fwd(const void* h, const void* w, const void* targets, int target_bits, int64_t ignore_index, float* loss, float* lse,
                     float* count, void* scratch, size_t scratch_bytes, void* status_word, int64_t T, int64_t N, int64_t V, int64_t ldh,
                     int64_t ldw, int reduction, int dtype, nq_stream_t stream) {
    if (!h || !w || !targets || !loss || !lse || !count || !scratch || !status_word) return NQ_ERR_NULL;
    int st = check_loss(T, N, V, ldh, ldw, dtype, reduction, target_bits);
    if (st != NQ_OK) return st;
    if (!aligned16(h) || !aligned16(w) || !aligned16(scratch) || !aligned16(status_word)) return NQ_ERR_ALIGN;
    if (!aligned_to(target_bits / 8, targets) || !aligned_to(4, loss, lse, count)) return NQ_ERR_ALIGN;
    const LossFwdScratch at = loss_fwd_scratch(T, N, V);
    if (scratch_bytes < (size_t)at.bytes) return NQ_ERR_SCRATCH;
    cudaStream_t s = as_stream(stream);
    unsigned* status = static_cast<unsigned*>(status_word) + 2;
    char* base = static_cast<char*>(scratch);
    float2* part = reinterpret_cast<float2*>(base);
    float* target_logit = reinterpret_cast<float*>(base + at.target_logit);
    float* row_loss = reduction == NQ_REDUCE_NONE ? loss : reinterpret_cast<float*>(base + at.row_loss);
    const int type = dtype == NQ_BF16 ? kMmBf16 : kMmF16;
    LossTargets all = {targets, target_bits == 64, ignore_index};
    const float2* joined = nullptr;
    int slots = 0, v = (int)V, mean = reduction == NQ_REDUCE_MEAN, all_t = (int)T;
    for (int64_t t0 = 0; t0 < T; t0 += kLossRows) {
        int t = (int)(T - t0 < kLossRows ? T - t0 : kLossRows), release = reduction != NQ_REDUCE_NONE || t0 + t < T;
        const LossTiles tiles = loss_tiles(t, V);
        slots = tiles.slots;
        const char* rows = static_cast<const char*>(h) + t0 * ldh * 2;
        LossTargets tg = {static_cast<const char*>(targets) + t0 * (target_bits / 8), all.wide, ignore_index};
        int *pos = nullptr, *words = nullptr, *live = nullptr;
        char* packed = base + at.h;
        if (loss_packs(t, N, V)) {
            pos = reinterpret_cast<int*>(base + at.pos);
            words = reinterpret_cast<int*>(base + at.words);
            live = reinterpret_cast<int*>(base + at.live);
            LossRows R = {tg, reinterpret_cast<const uint4*>(rows), reinterpret_cast<uint4*>(packed), ldh / 8, pos, words, live, t, v, (int)(N / 8), 1};
            int per_cta = rows_per_cta(t);
            void* pack_args[] = {&R, &per_cta};
            st = launch_plain((const void*)loss_pack_kernel, dim3((unsigned)((t + per_cta - 1) / per_cta)), 512, pack_args, s);
            if (st != NQ_OK) return st;
        }
        const LseEpilogue::Params e = {tg, words, part, target_logit};
        st = loss_pairs(t) ? launch_lse<2>(rows, packed, live, w, e, t, (int)N, v, ldh, ldw, type, tiles.bn, status, s)
                           : launch_lse<1>(rows, packed, live, w, e, t, (int)N, v, ldh, ldw, type, tiles.bn, status, s);
        if (st != NQ_OK) return st;
        if (reduction != NQ_REDUCE_NONE && !pos && T <= 1024 && T * slots <= kLossJoinHere) {
            joined = part;
            break;
        }
        float *loss_out = row_loss + t0, *lse_out = lse + t0;
        void* join_args[] = {&part, &target_logit, &tg, &loss_out, &lse_out, &pos, &slots, &t, &v, &release};
        st = t <= 8 * sm_count() ? launch_plain((const void*)lse_join_kernel<1>, dim3((unsigned)t), 256, join_args, s)
                                 : launch_plain((const void*)lse_join_kernel<8>, dim3((unsigned)((t + 7) / 8)), 256, join_args, s);
        if (st != NQ_OK) return st;
    }
    if (reduction == NQ_REDUCE_NONE) return NQ_OK;
    void* sum_args[] = {&joined, &target_logit, &row_loss, &lse, &all, &loss, &count, &slots, &all_t, &v, &mean};
    return launch_plain((const void*)loss_sum_kernel, dim3(1), 1024, sum_args, s);
}

size_t nq_linear_ce_bwd_scratch_bytes(int64_t T, int64_t N, int64_t V) {
    if (check_loss(T, N, V, N, N, NQ_F16, NQ_REDUCE_NONE, 64) != NQ_OK) return 0;
    return (size_t)loss_scratch(plan_loss(T, N, V), T, N, loss_packs(T, N, V)).bytes;
}

int nq_linear_ce_bwd(const void* h, const void* w, const void* targets, int target_bits, int64_t ignore_index, const float* lse,
                     const float* count, const float* grad_loss, int64_t grad_stride, void* dh, void* dw, void* scratch, size_t scratch_bytes,
                     void* status_word, int64_t T, int64_t N, int64_t V, int64_t ldh, int64_t ldw, int64_t lddh, int64_t lddw, int reduction,
                     int dtype, nq_stream_t stream) {
    if (!h || !w || !targets || !lse || !count || !grad_loss || !scratch || !status_word) return NQ_ERR_NULL;
    int st = check_loss(T, N, V, ldh, ldw, dtype, reduction, target_bits);
    if (st != NQ_OK) return st;
    if ((dh && (lddh < N || lddh % 8)) || (dw && (lddw < N || lddw % 8))) return NQ_ERR_SHAPE;
    if (!aligned16(h) || !aligned16(w) || !aligned16(dh) || !aligned16(dw) || !aligned16(scratch) || !aligned16(status_word)) return NQ_ERR_ALIGN;
    if (!aligned_to(target_bits / 8, targets) || !aligned_to(4, lse, count, grad_loss)) return NQ_ERR_ALIGN;
    const LossPlan p = plan_loss(T, N, V);
    const bool packs = loss_packs(T, N, V);
    const LossScratch at = loss_scratch(p, T, N, packs);
    if (scratch_bytes < (size_t)at.bytes) return NQ_ERR_SCRATCH;
    if (!dh && !dw) return NQ_OK;
    cudaStream_t s = as_stream(stream);
    unsigned* status = static_cast<unsigned*>(status_word) + 2;
    char* base = static_cast<char*>(scratch);
    LossTargets tg = {targets, target_bits == 64, ignore_index};
    LossRows R = {tg, static_cast<const uint4*>(h), dw || packs ? reinterpret_cast<uint4*>(base + at.h) : nullptr, ldh / 8, nullptr, nullptr, nullptr, (int)T, (int)V,
                  (int)(N / 8), 0};
    if (packs) {
        R.pos = reinterpret_cast<int*>(base + at.pos);
        R.words = reinterpret_cast<int*>(base + at.words);
        R.live = reinterpret_cast<int*>(base + at.live);
    }
    LossPrepare prep = {R, grad_loss, count, lse, grad_stride, reinterpret_cast<float*>(base + at.row_scale), reinterpret_cast<float*>(base + at.final_scale),
                        reinterpret_cast<float*>(base + at.row_lse), reduction, dtype == NQ_F16 ? kLossHalfScale : 1.f};
    int per_cta = rows_per_cta(T);
    void* prepare_args[] = {&prep, &per_cta};
    st = launch_plain((const void*)loss_prepare_kernel, dim3((unsigned)((T + per_cta - 1) / per_cta)), 512, prepare_args, s);
    if (st != NQ_OK) return st;
#define NQ_LOSS_BACKWARD(cg, out) launch_backward<cg, out>(h, w, tg, lse, dh, dw, base, p, at, (int)T, (int)N, (int)V, ldh, ldw, lddh, lddw, status, s)
    if (dtype == NQ_BF16) return loss_pairs(T) ? NQ_LOSS_BACKWARD(2, kOutBf16) : NQ_LOSS_BACKWARD(1, kOutBf16);
    return loss_pairs(T) ? NQ_LOSS_BACKWARD(2, kOutFp16) : NQ_LOSS_BACKWARD(1, kOutFp16);
#undef NQ_LOSS_BACKWARD
}

}  // extern "C"
