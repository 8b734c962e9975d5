// Layer norm and RMS norm of 16-bit activations, forward and backward:
//
//     y = (x - m) r w + b        m = mean(x), or 0 (RMS)        r = 1 / sqrt(mean((x - m)^2) + eps)
//     dx = r (g - mean(g) - xhat mean(g xhat))                  g = dy w, xhat = (x - m) r (mean(g) only where m is subtracted)
//     dw = sum_rows dy xhat        db = sum_rows dy
//
// Bound by memory: forward 2 bytes in and 2 out per element, backward 4 in and 2 out.  Every element is read once: a group of warps
// holds a row in registers (the mean, then the sum of squares of the differences, all in fp32, cost no second read).
//
//   stream kernels   many rows at 16-byte boundaries.  As many CTAs as fit the SMs, each of one group or more; a group takes rows first, first +
//                    groups, ...  A thread has the same columns of every row and copies the next rows' into its own part of shared memory
//                    (cp.async), so that loads stay in flight across the reductions of a row, and no thread waits for another's copies.
//   ragged kernels   the same for rows at any address.
//   direct kernels   few rows: a CTA each, one load a thread (latency).
//
// Backward: a thread adds dy xhat and dy of its columns to fp32 sums in registers.  One row of partial sums per CTA goes to the scratch; a
// second kernel adds these in a fixed order, so results do not depend on timing.
#include <atomic>

#include "nq_common.cuh"

namespace nq {

constexpr int kNormMaxCols = 16384;
// CTAs of a backward kernel to an SM at most: rows of partial sums.
static int norm_ctas_per_sm(int64_t N) { return N <= 2048 ? 8 : N <= 4096 ? 4 : 2; }

struct NormParams {
    const void *x, *w, *b, *dy;
    void *y;                               // forward: y; backward: dx
    float2* stats;                         // (mean, 1 / sigma) of a row; forward: nullable
    float *part_w, *part_b;                // backward: [CTAs][N] or nullptr
    long long rows, ldx, ldy, lddy;
    int N, w32;
    float eps, inv_n;
};

template <bool BF16>
__device__ __forceinline__ float norm_float(uint16_t h) {
    if constexpr (BF16) return __uint_as_float((uint32_t)h << 16);
    else return __half2float(__ushort_as_half(h));
}
template <bool BF16>
__device__ __forceinline__ uint32_t norm_pack(float a, float b) {
    uint32_t r;
    if constexpr (BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        r = *reinterpret_cast<const uint32_t*>(&h);
    }
    return r;
}
// VEC consecutive elements (one 16-byte load, or a single element) as they are, and as floats.  Nothing here is read by the non-coherent path: these kernels
// may be on their SMs while a kernel that released them early still writes.  Rows come through L2, weights, which all rows read, through L1.
template <int VEC> struct NormVec { uint32_t w[VEC / 2]; };
template <> struct NormVec<1> { uint16_t h; };
template <int VEC>
__device__ __forceinline__ NormVec<VEC> norm_load(const void* p, long long i, bool live) {
    NormVec<VEC> v = {};
    if (live) {
        if constexpr (VEC == 1) v.h = __ldcg(static_cast<const unsigned short*>(p) + i);
        else {
            const uint4 u = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
            v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
        }
    }
    return v;
}
template <int VEC, bool BF16>
__device__ __forceinline__ float norm_at(const NormVec<VEC>& v, int e) {
    if constexpr (VEC == 1) return norm_float<BF16>(v.h);
    else return norm_float<BF16>((uint16_t)(v.w[e >> 1] >> (16 * (e & 1))));
}
template <int VEC, bool BF16>
__device__ __forceinline__ void norm_store(void* p, long long i, const float (&f)[VEC]) {
    if constexpr (VEC == 1) static_cast<uint16_t*>(p)[i] = (uint16_t)norm_pack<BF16>(f[0], 0.f);
    else *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(norm_pack<BF16>(f[0], f[1]), norm_pack<BF16>(f[2], f[3]), norm_pack<BF16>(f[4], f[5]), norm_pack<BF16>(f[6], f[7]));
}
// Weights of VEC columns: 16-bit like the activations, or fp32.
template <int VEC, bool BF16>
__device__ __forceinline__ void norm_weights(const void* p, int w32, int c, float (&f)[VEC]) {
    if (w32) {
        const float* q = static_cast<const float*>(p) + c;
        if constexpr (VEC == 1) f[0] = *q;
        else {
            const float4 a = reinterpret_cast<const float4*>(q)[0], b = reinterpret_cast<const float4*>(q)[1];
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        }
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + c;
        if constexpr (VEC == 1) f[0] = norm_float<BF16>(*q);
        else {
            const uint4 u = *reinterpret_cast<const uint4*>(q);
            const NormVec<VEC> v = {{u.x, u.y, u.z, u.w}};
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = norm_at<VEC, BF16>(v, e);
        }
    }
}
__device__ __forceinline__ float2 warp_sum2(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}
// Sums over the WARPS warps of a row's group (the whole CTA, or one warp); `red` is used alternately, so one barrier a call is enough.
template <int WARPS>
__device__ __forceinline__ float2 group_sum2(float2 v, float2* red, int& turn) {
    v = warp_sum2(v);
    if constexpr (WARPS > 1) {
        float2* buf = red + 32 * (turn & 1);
        ++turn;
        if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        const int lane = threadIdx.x & 31;
        v = warp_sum2(lane < WARPS ? buf[lane] : make_float2(0.f, 0.f));
    }
    return v;
}

template <int WARPS>
constexpr int norm_rows_per_cta() { return WARPS == 1 ? 4 : 1; }

template <int VEC, int PACKS, int WARPS, bool BF16, bool CENTER>
__global__ void __launch_bounds__(32 * WARPS * norm_rows_per_cta<WARPS>()) norm_fwd_kernel(const NormParams P) {
    constexpr int G = 32 * WARPS, RPC = norm_rows_per_cta<WARPS>();
    __shared__ float2 red[64];
    int turn = 0;
    const int tid = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
    const long long row = (long long)blockIdx.x * RPC + (WARPS == 1 ? threadIdx.x >> 5 : 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= P.rows) return;             // (whole warps, and groups of one warp only: no barrier is missed)
    NormVec<VEC> v[PACKS];
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
        const int c = (p * G + tid) * VEC;
        v[p] = norm_load<VEC>(P.x, row * P.ldx + c, c < P.N);
    }
    float mean = 0.f;
    if constexpr (CENTER) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int p = 0; p < PACKS; ++p)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s.x += norm_at<VEC, BF16>(v[p], e);
        mean = group_sum2<WARPS>(s, red, turn).x / P.N;      // (exact where the sum is: a constant row's differences are zero)
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
        const bool live = (p * G + tid) * VEC < P.N;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = live ? norm_at<VEC, BF16>(v[p], e) - mean : 0.f;
            s.x = fmaf(d, d, s.x);
        }
    }
    const float rstd = 1.f / sqrtf(group_sum2<WARPS>(s, red, turn).x * P.inv_n + P.eps);
    if (tid == 0 && P.stats) P.stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
        const int c = (p * G + tid) * VEC;
        if (c < P.N) {
            float f[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = (norm_at<VEC, BF16>(v[p], e) - mean) * rstd;
            if (P.w) {
                float w[VEC];
                norm_weights<VEC, BF16>(P.w, P.w32, c, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] *= w[e];
            }
            if (P.b) {
                float b[VEC];
                norm_weights<VEC, BF16>(P.b, P.w32, c, b);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] += b[e];
            }
            norm_store<VEC, BF16>(P.y, row * P.ldy + c, f);
        }
    }
}

template <int VEC, int PACKS, int WARPS, bool BF16, bool CENTER>
__global__ void __launch_bounds__(32 * WARPS * norm_rows_per_cta<WARPS>()) norm_bwd_kernel(const NormParams P) {
    constexpr int G = 32 * WARPS, RPC = norm_rows_per_cta<WARPS>();
    __shared__ float2 red[64];
    int turn = 0;
    const int tid = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x, sub = WARPS == 1 ? threadIdx.x >> 5 : 0;
    float aw[PACKS][VEC], ab[PACKS][VEC];
#pragma unroll
    for (int p = 0; p < PACKS; ++p)
#pragma unroll
        for (int e = 0; e < VEC; ++e) aw[p][e] = ab[p][e] = 0.f;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (long long row = (long long)blockIdx.x * RPC + sub; row < P.rows; row += (long long)gridDim.x * RPC) {
        NormVec<VEC> x[PACKS], dy[PACKS];
        const float2 st = __ldcg(P.stats + row);
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int c = (p * G + tid) * VEC;
            x[p] = norm_load<VEC>(P.x, row * P.ldx + c, c < P.N);
            dy[p] = norm_load<VEC>(P.dy, row * P.lddy + c, c < P.N);
        }
        float2 s = make_float2(0.f, 0.f);  // sums of g xhat and of g
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int c = (p * G + tid) * VEC;
            if (c < P.N) {
                float w[VEC];
                if (P.w) norm_weights<VEC, BF16>(P.w, P.w32, c, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xh = (norm_at<VEC, BF16>(x[p], e) - st.x) * st.y, d = norm_at<VEC, BF16>(dy[p], e);
                    const float g = P.w ? d * w[e] : d;
                    s.x = fmaf(g, xh, s.x);
                    s.y += g;
                    aw[p][e] = fmaf(d, xh, aw[p][e]);
                    ab[p][e] += d;
                }
            }
        }
        if (P.y) {
            s = group_sum2<WARPS>(s, red, turn);
            const float c1 = s.x * P.inv_n, c2 = CENTER ? s.y * P.inv_n : 0.f;
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                const int c = (p * G + tid) * VEC;
                if (c < P.N) {
                    float w[VEC], f[VEC];
                    if (P.w) norm_weights<VEC, BF16>(P.w, P.w32, c, w);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float xh = (norm_at<VEC, BF16>(x[p], e) - st.x) * st.y, d = norm_at<VEC, BF16>(dy[p], e);
                        f[e] = st.y * ((P.w ? d * w[e] : d) - c2 - xh * c1);
                    }
                    norm_store<VEC, BF16>(P.y, row * P.ldy + c, f);
                }
            }
        }
    }
    // One row of partial sums per CTA; the rows of one-warp groups are added in the order of the warps.
    auto put = [&](float* part, const float (&a)[PACKS][VEC]) {
        float* dst = part + (size_t)blockIdx.x * P.N;
        for (int r = 0; r < RPC; ++r) {
            if (sub == r) {
#pragma unroll
                for (int p = 0; p < PACKS; ++p) {
                    const int c = (p * G + tid) * VEC;
                    if (c < P.N)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) dst[c + e] = (r ? dst[c + e] : 0.f) + a[p][e];
                }
            }
            if (RPC > 1) __syncthreads();
        }
    };
    if (P.part_w) put(P.part_w, aw);
    if (P.part_b) put(P.part_b, ab);
}

// ---------------------------------------------------------------------------
// stream kernels
// ---------------------------------------------------------------------------
__device__ __forceinline__ void norm_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void norm_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void norm_copies_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ uint4 norm_shared(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void norm_clear(uint32_t addr) { asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory"); }
// Two fp32 numbers in one 64-bit register, and the instructions that work on both: with one element at a time the stream kernels were bound by
// instruction issue (16384 x 5120: 28 instructions per element forward, 34 backward).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// (x - m) r of two elements, from -m and r.  The difference first: x r - m r would round twice to the size of m r, many times the result's in rows far from zero.
template <bool CENTER>
__device__ __forceinline__ f32x2 norm_hat(f32x2 x, f32x2 shift, f32x2 r) { return mul2(CENTER ? add2(x, shift) : x, r); }
template <bool BF16>
__device__ __forceinline__ f32x2 unpack2(uint32_t w) {
    if constexpr (BF16) return pair2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair2(f.x, f.y);
}
template <bool BF16>
__device__ __forceinline__ uint32_t repack2(f32x2 v) {
    const float2 f = split2(v);
    return norm_pack<BF16>(f.x, f.y);
}
// Weights of eight columns.
template <bool BF16>
__device__ __forceinline__ void weights2(const void* p, int w32, int c, f32x2 (&w)[4]) {
    if (w32) {
        const float4 *q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c), a = q[0], b = q[1];
        w[0] = pair2(a.x, a.y); w[1] = pair2(a.z, a.w); w[2] = pair2(b.x, b.y); w[3] = pair2(b.z, b.w);
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + c);
        w[0] = unpack2<BF16>(v.x); w[1] = unpack2<BF16>(v.y); w[2] = unpack2<BF16>(v.z); w[3] = unpack2<BF16>(v.w);
    }
}
// A group of G threads (whole warps) per batch of a few rows.  A batch's rows are all read for their sums, one exchange between the group's
// warps serves all of them, and they are read again for the outputs; each time from shared memory, by the thread that copied them (cp.async).  The next
// batch is on its way meanwhile.  16384 x 5120, layer norm, us: a row at a time 97 forward and 200 backward (waiting for reductions); batches with
// addresses computed for every access 78 and 105 (20 and 30 instructions per element); rows PITCH bytes apart in shared memory, PITCH a constant, and
// sums of several rows in one butterfly 59 and 91; with the difference from the mean taken first (norm_hat) 61 and 93; without branches for the columns beyond N
// 59 and 92.5 (5.7 and 5.4 TB/s; RMS 60 and 84).
template <int PITCH, bool BWD>
struct NormShape {
    static constexpr int kPacks = PITCH <= 4096 || (BWD && PITCH <= 10240) ? 1 : PITCH <= 16384 ? 2 : 4;      // times eight columns a thread
    static constexpr int kRows = BWD ? (PITCH <= 10240 ? 4 : PITCH <= 16384 ? 2 : 1) : PITCH <= 16384 ? 4 : 2;
    static constexpr int kThreads = PITCH <= 4096 ? 256 : PITCH / 16 / kPacks;                               // of a CTA at most
    static constexpr int kCtas = BWD ? (PITCH <= 4096 ? 3 : 1) : PITCH <= 8192 ? 3 : PITCH <= 10240 ? 2 : 1;  // to an SM at least (registers)
    static constexpr int kSlot = (BWD ? 2 : 1) * PITCH;                                                        // bytes of a row (x, then dy)
    static constexpr int kGroupBytes = 2 * kRows * kSlot;
};
// Sums over the warp of NUM numbers, a power of two up to 8; lane i has number i / (32 / NUM).
template <int NUM>
__device__ __forceinline__ float warp_sums(const float (&v)[NUM]) {
    const int lane = threadIdx.x & 31;
    float t[NUM];
#pragma unroll
    for (int i = 0; i < NUM; ++i) t[i] = v[i];
    int o = 16;
#pragma unroll
    for (int n = NUM; n > 1; n >>= 1, o >>= 1) {          // half of the numbers to either half of the lanes
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float keep = upper ? t[i + n / 2] : t[i], give = upper ? t[i] : t[i + n / 2];
            t[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (; o > 0; o >>= 1) t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
    return t[0];
}
struct NormGroup {
    int G, id, tid, lane, warps;
    float* red;
    __device__ NormGroup(float (*red_)[2][8], int G_) : G(G_) {
        id = threadIdx.x / G;
        tid = threadIdx.x - id * G;
        lane = threadIdx.x & 31;
        warps = G >> 5;
        red = &red_[id * warps][0][0];
    }
    // NUM numbers of every warp (as warp_sums leaves them) at OFF for all of the group to read, those of warp i at 16 i.
    template <int NUM>
    __device__ __forceinline__ void put(float v, int off, int parity) {
        if ((lane & (32 / NUM - 1)) == 0) red[(tid >> 5) * 16 + 8 * parity + off + lane / (32 / NUM)] = v;
    }
    __device__ __forceinline__ void sync() { asm volatile("bar.sync %0, %1;" ::"r"(1 + id), "r"(G) : "memory"); }
};
// Mean and squares of a batch's rows from those of the group's warps, which have warp_sums' lanes; `count`: columns of a warp.
template <int ROWS, bool CENTER, class Count>
__device__ __forceinline__ void group_moments(NormGroup& g, int parity, Count count, float inv_n, float& mean, float& squares) {
    g.put<ROWS>(squares, 0, parity);
    if constexpr (CENTER) g.put<ROWS>(mean, ROWS, parity);
    g.sync();
    const float* all = g.red + 8 * parity + g.lane / (32 / ROWS);      // of the lane's row; its lanes share the warps
    auto join = [](float t) {
#pragma unroll
        for (int o = 16 / ROWS; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        return t;
    };
    mean = squares = 0.f;
    const int i0 = g.lane & (32 / ROWS - 1);
    if constexpr (CENTER) {
        // (by the distances from the first warp's: rounded once to the size of the mean, whose rounding counts 1 / sigma times)
        const float start = all[ROWS];
        for (int i = i0; i < g.warps; i += 32 / ROWS) mean = fmaf(count(i), all[16 * i + ROWS] - start, mean);
        mean = fmaf(join(mean), inv_n, start);
        for (int i = i0; i < g.warps; i += 32 / ROWS) {
            const float d = all[16 * i + ROWS] - mean;
            squares += fmaf(count(i) * d, d, all[16 * i]);
        }
    } else {
        for (int i = i0; i < g.warps; i += 32 / ROWS) squares += all[16 * i];
    }
    squares = join(squares);
}
// Sums over the group of what the warps have, number lane / (32 / NUM) as warp_sums leaves it.
template <int NUM>
__device__ __forceinline__ float group_totals(NormGroup& g, int parity, float total) {
    if (g.warps > 1) {
        g.put<NUM>(total, 0, parity);
        g.sync();
        const float* all = g.red + 8 * parity + g.lane / (32 / NUM);
        total = 0.f;
        for (int i = g.lane & (32 / NUM - 1); i < g.warps; i += 32 / NUM) total += all[16 * i];
#pragma unroll
        for (int o = 16 / NUM; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    return total;
}
__device__ __forceinline__ void unpack8(const uint4& v, uint32_t (&w)[4]) { w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }

template <int PITCH, bool BF16, bool CENTER>
__global__ void __launch_bounds__(NormShape<PITCH, false>::kThreads, NormShape<PITCH, false>::kCtas) norm_fwd_stream_kernel(const NormParams P, int G) {
    using Shape = NormShape<PITCH, false>;
    constexpr int PACKS = Shape::kPacks, ROWS = Shape::kRows;
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float red[Shape::kThreads / 32][2][8];     // (two halves in turn, so that one barrier a batch is enough)
    NormGroup g(red, G);
    const int packs = P.N >> 3, groups = blockDim.x / G;
    const long long batches = (P.rows + ROWS - 1) / ROWS, step = (long long)gridDim.x * groups, first = (long long)blockIdx.x * groups + g.id;
    const uint32_t mine = smem_u32(norm_smem) + (uint32_t)(g.id * Shape::kGroupBytes + g.tid * 16);
    auto live = [&](int p) { return p * G + g.tid < packs; };
    const long long ldx = 2 * P.ldx, ldy = 2 * P.ldy, next_x = step * ROWS * ldx, next_y = step * ROWS * ldy;     // bytes
    const char* x = static_cast<const char*>(P.x) + first * ROWS * ldx + g.tid * 16;          // of the next batch to be copied
    char* y = static_cast<char*>(P.y) + first * ROWS * ldy + g.tid * 16;
    long long ahead = first;                              // that batch
    auto copy = [&](int stage) {
        if (ahead < batches) {
            const char* src = x;
            const uint32_t dst = mine + (uint32_t)(stage * ROWS * PITCH);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (r == 0 || ahead * ROWS + r < P.rows) {
#pragma unroll
                    for (int p = 0; p < PACKS; ++p)
                        if (live(p)) norm_copy16(dst + (uint32_t)(p * G * 16) + r * PITCH, src + p * G * 16);
                }
                src += ldx;
            }
        }
        x += next_x;
        ahead += step;
        norm_commit();
    };
    auto count = [&](int warp) {                          // columns of a warp of the group (eight at least)
        int n = 0;
#pragma unroll
        for (int p = 0; p < PACKS; ++p) n += max(0, min(32, packs - p * G - 32 * warp));
        return 8.f * n;
    };
    const float own_columns = count(g.tid >> 5);
    // Slots of columns beyond N hold zeros, so that the loops below need no branches for them.
#pragma unroll
    for (int p = 0; p < PACKS; ++p)
        if (!live(p))
            for (int i = 0; i < 2 * ROWS; ++i) norm_clear(mine + (uint32_t)(p * G * 16 + i * PITCH));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    copy(0);
    copy(1);
    f32x2 w[PACKS][4], b[PACKS][4];                       // of the thread's columns, for all rows
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[p][k] = pair2(1.f, 1.f);
            b[p][k] = 0;
        }
        if (live(p) && P.w) weights2<BF16>(P.w, P.w32, (p * G + g.tid) * 8, w[p]);
        if (CENTER && live(p) && P.b) weights2<BF16>(P.b, P.w32, (p * G + g.tid) * 8, b[p]);
    }
    int stage = 0;
    for (long long batch = first; batch < batches; batch += step, y += next_y) {
        const int rows = (int)min((long long)ROWS, P.rows - batch * ROWS);
        uint32_t at[PACKS];
#pragma unroll
        for (int p = 0; p < PACKS; ++p) at[p] = mine + (uint32_t)(stage * ROWS * PITCH + p * G * 16);
        norm_copies_landed<1>();
        // Layer norm: each warp's own mean and squares of the differences from it, then those of all warps, so that one exchange is enough and no
        // small difference of large sums is taken: sum (x - m)^2 = sum_w [sum (x - m_w)^2 + n_w (m_w - m)^2].
        float v[ROWS], own = 0.f;                         // own: of row lane / (32 / ROWS)
        if constexpr (CENTER) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                f32x2 s = 0;
#pragma unroll
                for (int p = 0; p < PACKS; ++p) {
                    uint32_t xw[4];
                    unpack8(norm_shared(at[p] + r * PITCH), xw);
                    s = add2(s, add2(add2(unpack2<BF16>(xw[0]), unpack2<BF16>(xw[1])), add2(unpack2<BF16>(xw[2]), unpack2<BF16>(xw[3]))));
                }
                v[r] = split2(s).x + split2(s).y;
            }
            own = warp_sums(v) / own_columns;
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            f32x2 s = 0, shift = 0;
            if constexpr (CENTER) {
                const float m = -__shfl_sync(0xffffffffu, own, r * (32 / ROWS));
                shift = pair2(m, m);
            }
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                uint32_t xw[4];
                unpack8(norm_shared(at[p] + r * PITCH), xw);
                const f32x2 own_shift = live(p) ? shift : 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x2 d = CENTER ? add2(unpack2<BF16>(xw[k]), own_shift) : unpack2<BF16>(xw[k]);
                    s = fma2(d, d, s);
                }
            }
            v[r] = split2(s).x + split2(s).y;
        }
        float squares = warp_sums(v), mean = own;
        if (g.warps > 1) group_moments<ROWS, CENTER>(g, stage, count, P.inv_n, mean, squares);
        const float rstd = 1.f / sqrtf(squares * P.inv_n + P.eps);
        if (P.stats && g.tid < 32 && (g.lane & (32 / ROWS - 1)) == 0 && g.lane / (32 / ROWS) < rows)
            P.stats[batch * ROWS + g.lane / (32 / ROWS)] = make_float2(mean, rstd);
        char* dst = y;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float rs = __shfl_sync(0xffffffffu, rstd, r * (32 / ROWS)), ms = CENTER ? -__shfl_sync(0xffffffffu, mean, r * (32 / ROWS)) : 0.f;
            const f32x2 r2 = pair2(rs, rs), shift = pair2(ms, ms);
#pragma unroll
            for (int p = 0; p < PACKS; ++p) {
                uint32_t xw[4];
                unpack8(norm_shared(at[p] + r * PITCH), xw);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    xw[k] = repack2<BF16>(CENTER ? fma2(norm_hat<true>(unpack2<BF16>(xw[k]), shift, r2), w[p][k], b[p][k]) : mul2(mul2(unpack2<BF16>(xw[k]), r2), w[p][k]));
                if (r < rows && live(p)) *reinterpret_cast<uint4*>(dst + p * G * 16) = make_uint4(xw[0], xw[1], xw[2], xw[3]);
            }
            dst += ldy;
        }
        copy(stage);
        stage ^= 1;
    }
}

template <int PITCH, bool BF16, bool CENTER>
__global__ void __launch_bounds__(NormShape<PITCH, true>::kThreads, NormShape<PITCH, true>::kCtas) norm_bwd_stream_kernel(const NormParams P, int G) {
    using Shape = NormShape<PITCH, true>;
    constexpr int PACKS = Shape::kPacks, ROWS = Shape::kRows, kSlot = Shape::kSlot;
    constexpr int kSums = CENTER ? 2 * ROWS : ROWS;       // of g xhat, and of g
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float red[Shape::kThreads / 32][2][8];     // (two halves in turn, so that one barrier a batch is enough)
    NormGroup g(red, G);
    const int packs = P.N >> 3, groups = blockDim.x / G, tid = g.tid, lane = g.lane;
    const long long batches = (P.rows + ROWS - 1) / ROWS, step = (long long)gridDim.x * groups, first = (long long)blockIdx.x * groups + g.id;
    const uint32_t mine = smem_u32(norm_smem) + (uint32_t)(g.id * Shape::kGroupBytes + tid * 16);
    auto live = [&](int p) { return p * G + tid < packs; };
    const long long ldx = 2 * P.ldx, lddy = 2 * P.lddy, lddx = 2 * P.ldy, next_x = step * ROWS * ldx, next_dy = step * ROWS * lddy, next_dx = step * ROWS * lddx;
    const char *x = static_cast<const char*>(P.x) + first * ROWS * ldx + tid * 16, *dy = static_cast<const char*>(P.dy) + first * ROWS * lddy + tid * 16;
    char* dx = static_cast<char*>(P.y) + first * ROWS * lddx + tid * 16;
    long long ahead = first;                              // the next batch to be copied
    auto copy = [&](int stage) {
        if (ahead < batches) {
            const char *sx = x, *sd = dy;
            const uint32_t dst = mine + (uint32_t)(stage * ROWS * kSlot);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (r == 0 || ahead * ROWS + r < P.rows) {
#pragma unroll
                    for (int p = 0; p < PACKS; ++p)
                        if (live(p)) {
                            norm_copy16(dst + (uint32_t)(p * G * 16) + r * kSlot, sx + p * G * 16);
                            norm_copy16(dst + (uint32_t)(p * G * 16) + r * kSlot + PITCH, sd + p * G * 16);
                        }
                }
                sx += ldx;
                sd += lddy;
            }
        }
        x += next_x;
        dy += next_dy;
        ahead += step;
        norm_commit();
    };
    // mean and 1 / sigma of row `lane` of a batch
    auto load_stats = [&](long long batch) {
        return lane < ROWS && batch * ROWS + lane < P.rows ? __ldcg(P.stats + batch * ROWS + lane) : make_float2(0.f, 0.f);
    };
    f32x2 aw[PACKS][4], ab[PACKS][4], w[PACKS][4];
#pragma unroll
    for (int p = 0; p < PACKS; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            aw[p][k] = ab[p][k] = 0;
            w[p][k] = pair2(1.f, 1.f);
        }
    // Slots of columns beyond N hold zeros, so that the loops below need no branches for them.
#pragma unroll
    for (int p = 0; p < PACKS; ++p)
        if (!live(p))
            for (int i = 0; i < 4 * ROWS; ++i) norm_clear(mine + (uint32_t)(p * G * 16 + i * PITCH));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    copy(0);
    copy(1);
    float2 next = load_stats(first);
#pragma unroll
    for (int p = 0; p < PACKS; ++p)
        if (P.w && live(p)) weights2<BF16>(P.w, P.w32, (p * G + tid) * 8, w[p]);
    int stage = 0;
    for (long long batch = first; batch < batches; batch += step, dx += next_dx) {
        const int rows = (int)min((long long)ROWS, P.rows - batch * ROWS);
        const float rstd = next.y, shift = -next.x;                // of row `lane`
        next = load_stats(batch + step);
        uint32_t at[PACKS];
#pragma unroll
        for (int p = 0; p < PACKS; ++p) at[p] = mine + (uint32_t)(stage * ROWS * kSlot + p * G * 16);
        norm_copies_landed<1>();
        float sums[kSums];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float r1 = __shfl_sync(0xffffffffu, rstd, r), s1 = __shfl_sync(0xffffffffu, shift, r);
            const f32x2 r2 = pair2(r1, r1), s2 = pair2(s1, s1);
            f32x2 sx = 0, sg = 0;
            if (r < rows) {
#pragma unroll
                for (int p = 0; p < PACKS; ++p) {
                    uint32_t xw[4], dw[4];
                    unpack8(norm_shared(at[p] + r * kSlot), xw);
                    unpack8(norm_shared(at[p] + r * kSlot + PITCH), dw);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f32x2 xh = norm_hat<CENTER>(unpack2<BF16>(xw[k]), s2, r2), d = unpack2<BF16>(dw[k]), gr = mul2(d, w[p][k]);
                        sx = fma2(gr, xh, sx);
                        aw[p][k] = fma2(d, xh, aw[p][k]);
                        if constexpr (CENTER) {
                            sg = add2(sg, gr);
                            ab[p][k] = add2(ab[p][k], d);
                        }
                    }
                }
            }
            sums[r] = split2(sx).x + split2(sx).y;
            if constexpr (CENTER) sums[ROWS + r] = split2(sg).x + split2(sg).y;
        }
        if (P.y) {
            const float total = -P.inv_n * group_totals<kSums>(g, stage, warp_sums(sums));
            char* dst = dx;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float r1 = __shfl_sync(0xffffffffu, rstd, r), s1 = __shfl_sync(0xffffffffu, shift, r);
                // dx = r g - (r mean(g)) - xhat (r mean(g xhat))
                const float c1 = r1 * __shfl_sync(0xffffffffu, total, r * (32 / kSums)), c2 = CENTER ? r1 * __shfl_sync(0xffffffffu, total, (ROWS + r) * (32 / kSums)) : 0.f;
                const f32x2 r2 = pair2(r1, r1), s2 = pair2(s1, s1), c1p = pair2(c1, c1), c2p = pair2(c2, c2);
                if (r < rows) {
#pragma unroll
                    for (int p = 0; p < PACKS; ++p) {
                        uint32_t xw[4], dw[4];
                        unpack8(norm_shared(at[p] + r * kSlot), xw);
                        unpack8(norm_shared(at[p] + r * kSlot + PITCH), dw);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const f32x2 xh = norm_hat<CENTER>(unpack2<BF16>(xw[k]), s2, r2);
                            xw[k] = repack2<BF16>(fma2(mul2(unpack2<BF16>(dw[k]), w[p][k]), r2, fma2(xh, c1p, c2p)));
                        }
                        if (live(p)) *reinterpret_cast<uint4*>(dst + p * G * 16) = make_uint4(xw[0], xw[1], xw[2], xw[3]);
                    }
                }
                dst += lddx;
            }
        }
        copy(stage);
        stage ^= 1;
    }
    // One row of partial sums per CTA: the groups' in turn, in shared memory over the copies' (which have all landed and been read).
    norm_copies_landed<0>();
    float* sums = reinterpret_cast<float*>(norm_smem);
    auto put = [&](float* part, const f32x2 (&a)[PACKS][4]) {
        float* dst = part + (size_t)blockIdx.x * P.N;
        for (int r = 0; r < groups; ++r) {
            __syncthreads();
            if (g.id == r) {
#pragma unroll
                for (int p = 0; p < PACKS; ++p) {
                    const int c = (p * G + tid) * 8;
                    if (live(p)) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const f32x2 v = r ? add2(a[p][k], *reinterpret_cast<const f32x2*>(sums + c + 2 * k)) : a[p][k];
                            *reinterpret_cast<f32x2*>((r + 1 < groups ? sums : dst) + c + 2 * k) = v;
                        }
                    }
                }
            }
        }
    };
    if (P.part_w) put(P.part_w, aw);
    if (P.part_b) put(P.part_b, ab);
}

// ---------------------------------------------------------------------------
// the same for rows at any address
// ---------------------------------------------------------------------------
// A row's 16-byte units (the first and the last hold elements of its neighbours, or what lies around the tensor in these units, which is ignored) are
// copied as they are, and a thread takes the columns tid, tid + G, ...: single elements, but out of shared memory, and stores side by side.  A row is
// read by others than copied it: one more barrier a batch, behind which the batch after this one is requested.  8000 x 5001, us: layer norm forward
// 147 -> 107, backward 322 -> 119 against the direct kernels; bound by the loads of single elements from shared memory.
__device__ __forceinline__ uint16_t ragged_shared(uint32_t addr) {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr) : "memory");
    return h;
}
// Copies a row's units, G threads; the row then starts ragged_shift(src) bytes into `dst`.
__device__ __forceinline__ uint32_t ragged_shift(const void* src) { return (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15u); }
__device__ __forceinline__ void ragged_copy(uint32_t dst, const char* src, int N, int tid, int G) {
    const uint32_t shift = ragged_shift(src), bytes = shift + 2u * (uint32_t)N;
    for (uint32_t at = 16u * (uint32_t)tid; at < bytes; at += 16u * (uint32_t)G) {
        const uint32_t left = bytes - at;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + at), "l"(src - shift + at), "r"(left < 16u ? left : 16u) : "memory");
    }
}
template <bool BF16>
__device__ __forceinline__ f32x2 ragged_pair(uint32_t a, uint32_t b) { return pair2(norm_float<BF16>(ragged_shared(a)), norm_float<BF16>(ragged_shared(b))); }
template <bool BF16>
__device__ __forceinline__ float ragged_weight(const void* p, int w32, int c) {
    return w32 ? static_cast<const float*>(p)[c] : norm_float<BF16>(static_cast<const uint16_t*>(p)[c]);
}

// COLS columns a thread; dead ones (beyond N) read the row's first element and count for nothing.
template <int COLS, int ROWS, bool BF16, bool CENTER>
__global__ void __launch_bounds__(512, 1) norm_fwd_ragged_kernel(const NormParams P, int G, int pitch) {
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float red[16][2][8];
    NormGroup g(red, G);
    const int groups = blockDim.x / G, tid = g.tid, N = P.N;
    const long long batches = (P.rows + ROWS - 1) / ROWS, step = (long long)gridDim.x * groups, first = (long long)blockIdx.x * groups + g.id;
    const uint32_t mine = smem_u32(norm_smem) + (uint32_t)(g.id * 2 * ROWS * pitch);
    const char* x0 = static_cast<const char*>(P.x);
    auto row_at = [&](long long batch, int r) { return x0 + 2 * min(batch * ROWS + r, P.rows - 1) * P.ldx; };
    auto copy = [&](long long batch, int stage) {
        if (batch < batches)
            for (int r = 0; r < ROWS; ++r) ragged_copy(mine + (uint32_t)((stage * ROWS + r) * pitch), row_at(batch, r), N, tid, G);
        norm_commit();
    };
    auto live = [&](int e) { return e * G + tid < N; };
    auto count = [&](int warp) {
        int n = 0;
#pragma unroll
        for (int e = 0; e < COLS; ++e) n += max(0, min(32, N - e * G - 32 * warp));
        return (float)n;
    };
    const float own_columns = count(tid >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    copy(first, 0);
    uint32_t off[COLS];                    // bytes of the thread's columns
    f32x2 w[COLS / 2], b[COLS / 2];
#pragma unroll
    for (int e = 0; e < COLS; e += 2) {
        off[e] = live(e) ? 2u * (uint32_t)(e * G + tid) : 0u;
        off[e + 1] = live(e + 1) ? 2u * (uint32_t)((e + 1) * G + tid) : 0u;
        w[e / 2] = P.w ? pair2(ragged_weight<BF16>(P.w, P.w32, off[e] >> 1), ragged_weight<BF16>(P.w, P.w32, off[e + 1] >> 1)) : pair2(1.f, 1.f);
        b[e / 2] = CENTER && P.b ? pair2(ragged_weight<BF16>(P.b, P.w32, off[e] >> 1), ragged_weight<BF16>(P.b, P.w32, off[e + 1] >> 1)) : 0;
    }
    int stage = 0;
    for (long long batch = first; batch < batches; batch += step) {
        const int rows = (int)min((long long)ROWS, P.rows - batch * ROWS);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        g.sync();                          // this batch is there for all, and all have left the one before
        copy(batch + step, stage ^ 1);
        uint32_t at[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) at[r] = mine + (uint32_t)((stage * ROWS + r) * pitch) + ragged_shift(row_at(batch, r));
        float v[ROWS], own = 0.f;
        if constexpr (CENTER) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                v[r] = 0.f;
#pragma unroll
                for (int e = 0; e < COLS; ++e) v[r] += live(e) ? norm_float<BF16>(ragged_shared(at[r] + off[e])) : 0.f;
            }
            own = warp_sums(v) / own_columns;
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float m = CENTER ? __shfl_sync(0xffffffffu, own, r * (32 / ROWS)) : 0.f;
            v[r] = 0.f;
#pragma unroll
            for (int e = 0; e < COLS; ++e) {
                const float d = live(e) ? norm_float<BF16>(ragged_shared(at[r] + off[e])) - m : 0.f;
                v[r] = fmaf(d, d, v[r]);
            }
        }
        float squares = warp_sums(v), mean = own;
        if (g.warps > 1) group_moments<ROWS, CENTER>(g, stage, count, P.inv_n, mean, squares);
        const float rstd = 1.f / sqrtf(squares * P.inv_n + P.eps);
        if (P.stats && tid < 32 && (g.lane & (32 / ROWS - 1)) == 0 && g.lane / (32 / ROWS) < rows)
            P.stats[batch * ROWS + g.lane / (32 / ROWS)] = make_float2(mean, rstd);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float rs = __shfl_sync(0xffffffffu, rstd, r * (32 / ROWS)), ms = CENTER ? -__shfl_sync(0xffffffffu, mean, r * (32 / ROWS)) : 0.f;
            const f32x2 r2 = pair2(rs, rs), shift = pair2(ms, ms);
            if (r < rows) {
                char* dst = static_cast<char*>(P.y) + 2 * (batch * ROWS + r) * P.ldy;
#pragma unroll
                for (int e = 0; e < COLS; e += 2) {
                    const f32x2 xv = ragged_pair<BF16>(at[r] + off[e], at[r] + off[e + 1]);
                    const uint32_t o = repack2<BF16>(CENTER ? fma2(norm_hat<true>(xv, shift, r2), w[e / 2], b[e / 2]) : mul2(mul2(xv, r2), w[e / 2]));
                    if (live(e)) *reinterpret_cast<uint16_t*>(dst + off[e]) = (uint16_t)o;
                    if (live(e + 1)) *reinterpret_cast<uint16_t*>(dst + off[e + 1]) = (uint16_t)(o >> 16);
                }
            }
        }
        stage ^= 1;
    }
}

template <int COLS, int ROWS, bool BF16, bool CENTER>
__global__ void __launch_bounds__(512, 1) norm_bwd_ragged_kernel(const NormParams P, int G, int pitch) {
    constexpr int kSums = CENTER ? 2 * ROWS : ROWS;
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float red[16][2][8];
    NormGroup g(red, G);
    const int groups = blockDim.x / G, tid = g.tid, lane = g.lane, N = P.N;
    const long long batches = (P.rows + ROWS - 1) / ROWS, step = (long long)gridDim.x * groups, first = (long long)blockIdx.x * groups + g.id;
    const uint32_t mine = smem_u32(norm_smem) + (uint32_t)(g.id * 4 * ROWS * pitch);
    auto row_at = [&](const void* p, long long ld, long long batch, int r) { return static_cast<const char*>(p) + 2 * min(batch * ROWS + r, P.rows - 1) * ld; };
    auto copy = [&](long long batch, int stage) {
        if (batch < batches)
            for (int r = 0; r < ROWS; ++r) {
                const uint32_t dst = mine + (uint32_t)((stage * ROWS + r) * 2 * pitch);
                ragged_copy(dst, row_at(P.x, P.ldx, batch, r), N, tid, G);
                ragged_copy(dst + (uint32_t)pitch, row_at(P.dy, P.lddy, batch, r), N, tid, G);
            }
        norm_commit();
    };
    auto live = [&](int e) { return e * G + tid < N; };
    f32x2 aw[COLS / 2], ab[COLS / 2], w[COLS / 2];
    uint32_t off[COLS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    copy(first, 0);
#pragma unroll
    for (int e = 0; e < COLS; e += 2) {
        off[e] = live(e) ? 2u * (uint32_t)(e * G + tid) : 0u;
        off[e + 1] = live(e + 1) ? 2u * (uint32_t)((e + 1) * G + tid) : 0u;
        // (a dead column has weight 0, so that it adds nothing to the sums; what it adds up for dw and db is not stored)
        w[e / 2] = pair2(!live(e) ? 0.f : P.w ? ragged_weight<BF16>(P.w, P.w32, off[e] >> 1) : 1.f, !live(e + 1) ? 0.f : P.w ? ragged_weight<BF16>(P.w, P.w32, off[e + 1] >> 1) : 1.f);
        aw[e / 2] = ab[e / 2] = 0;
    }
    int stage = 0;
    for (long long batch = first; batch < batches; batch += step) {
        const int rows = (int)min((long long)ROWS, P.rows - batch * ROWS);
        const float2 st = lane < rows ? __ldcg(P.stats + batch * ROWS + lane) : make_float2(0.f, 0.f);
        const float rstd = st.y, shift = -st.x;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        g.sync();                          // this batch is there for all, and all have left the one before
        copy(batch + step, stage ^ 1);
        uint32_t ax[ROWS], ad[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const uint32_t base = mine + (uint32_t)((stage * ROWS + r) * 2 * pitch);
            ax[r] = base + ragged_shift(row_at(P.x, P.ldx, batch, r));
            ad[r] = base + (uint32_t)pitch + ragged_shift(row_at(P.dy, P.lddy, batch, r));
        }
        float sums[kSums];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float r1 = __shfl_sync(0xffffffffu, rstd, r), s1 = __shfl_sync(0xffffffffu, shift, r);
            const f32x2 r2 = pair2(r1, r1), s2 = pair2(s1, s1);
            f32x2 sx = 0, sg = 0;
            if (r < rows) {
#pragma unroll
                for (int e = 0; e < COLS; e += 2) {
                    const f32x2 xh = norm_hat<CENTER>(ragged_pair<BF16>(ax[r] + off[e], ax[r] + off[e + 1]), s2, r2), d = ragged_pair<BF16>(ad[r] + off[e], ad[r] + off[e + 1]);
                    const f32x2 gr = mul2(d, w[e / 2]);
                    sx = fma2(gr, xh, sx);
                    aw[e / 2] = fma2(d, xh, aw[e / 2]);
                    if constexpr (CENTER) {
                        sg = add2(sg, gr);
                        ab[e / 2] = add2(ab[e / 2], d);
                    }
                }
            }
            sums[r] = split2(sx).x + split2(sx).y;
            if constexpr (CENTER) sums[ROWS + r] = split2(sg).x + split2(sg).y;
        }
        if (P.y) {
            const float total = -P.inv_n * group_totals<kSums>(g, stage, warp_sums(sums));
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const float r1 = __shfl_sync(0xffffffffu, rstd, r), s1 = __shfl_sync(0xffffffffu, shift, r);
                const float c1 = r1 * __shfl_sync(0xffffffffu, total, r * (32 / kSums)), c2 = CENTER ? r1 * __shfl_sync(0xffffffffu, total, (ROWS + r) * (32 / kSums)) : 0.f;
                const f32x2 r2 = pair2(r1, r1), s2 = pair2(s1, s1), c1p = pair2(c1, c1), c2p = pair2(c2, c2);
                if (r < rows) {
                    char* dst = static_cast<char*>(P.y) + 2 * (batch * ROWS + r) * P.ldy;
#pragma unroll
                    for (int e = 0; e < COLS; e += 2) {
                        const f32x2 xh = norm_hat<CENTER>(ragged_pair<BF16>(ax[r] + off[e], ax[r] + off[e + 1]), s2, r2), d = ragged_pair<BF16>(ad[r] + off[e], ad[r] + off[e + 1]);
                        const uint32_t o = repack2<BF16>(fma2(mul2(d, w[e / 2]), r2, fma2(xh, c1p, c2p)));
                        if (live(e)) *reinterpret_cast<uint16_t*>(dst + off[e]) = (uint16_t)o;
                        if (live(e + 1)) *reinterpret_cast<uint16_t*>(dst + off[e + 1]) = (uint16_t)(o >> 16);
                    }
                }
            }
        }
        stage ^= 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float* sums = reinterpret_cast<float*>(norm_smem);     // (4 N bytes: a batch of the group's own is more)
    auto put = [&](float* part, const f32x2 (&a)[COLS / 2]) {
        float* dst = part + (size_t)blockIdx.x * N;
        for (int r = 0; r < groups; ++r) {
            __syncthreads();
            if (g.id == r) {
#pragma unroll
                for (int e = 0; e < COLS; ++e)
                    if (live(e)) {
                        const int c = off[e] >> 1;
                        const float v = (r ? sums[c] : 0.f) + (e & 1 ? split2(a[e / 2]).y : split2(a[e / 2]).x);
                        if (r + 1 < groups) sums[c] = v;
                        else dst[c] = v;
                    }
            }
        }
    };
    if (P.part_w) put(P.part_w, aw);
    if (P.part_b) put(P.part_b, ab);
}

// out[c] = sum over the CTAs of part[i][c]: 32 columns a CTA, 32 warps over the rows (so that a warp's few loads are one round trip), then over the warps.
template <bool BF16>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* part_w, const float* part_b, void* dw, void* db, int ctas, int N, int w32) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* part = blockIdx.y ? part_b : part_w;
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    float s = 0.f;
    if (c < N) {
#pragma unroll 8
        for (int i = warp; i < ctas; i += 32) s += __ldcg(part + (size_t)i * N + c);
    }
    red[warp][lane] = s;
    __syncthreads();
    s = red[lane][warp];                   // warp w: column w
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int col = blockIdx.x * 32 + warp;
    if (lane == 0 && col < N) {
        if (w32) static_cast<float*>(out)[col] = s;
        else static_cast<uint16_t*>(out)[col] = (uint16_t)norm_pack<BF16>(s, 0.f);
    }
}

using NormKernel = void (*)(NormParams);
struct NormVariant {
    NormKernel fn;
    int threads, rows_per_cta;
};
template <int VEC, int PACKS, int WARPS>
NormVariant norm_variant(bool bwd, bool bf16, bool center) {
    NormKernel k;
    if (bwd) k = bf16 ? (center ? norm_bwd_kernel<VEC, PACKS, WARPS, true, true> : norm_bwd_kernel<VEC, PACKS, WARPS, true, false>)
                      : (center ? norm_bwd_kernel<VEC, PACKS, WARPS, false, true> : norm_bwd_kernel<VEC, PACKS, WARPS, false, false>);
    else k = bf16 ? (center ? norm_fwd_kernel<VEC, PACKS, WARPS, true, true> : norm_fwd_kernel<VEC, PACKS, WARPS, true, false>)
                  : (center ? norm_fwd_kernel<VEC, PACKS, WARPS, false, true> : norm_fwd_kernel<VEC, PACKS, WARPS, false, false>);
    return {k, 32 * WARPS * norm_rows_per_cta<WARPS>(), norm_rows_per_cta<WARPS>()};
}
// Direct kernels: the smallest group that holds a row.  16-byte loads where every row starts at a 16-byte boundary, single elements otherwise.
// (vec: at most 2 sm_count() rows, more are streamed)
NormVariant choose_norm(bool bwd, bool bf16, bool center, bool vec, int N) {
    if (vec) {
        const int packs = (N + 7) / 8;
        if (packs <= 64) return norm_variant<8, 2, 1>(bwd, bf16, center);
        if (packs <= 128) return norm_variant<8, 1, 4>(bwd, bf16, center);
        if (packs <= 512) return norm_variant<8, 1, 16>(bwd, bf16, center);
        if (packs <= 1024) return norm_variant<8, 2, 16>(bwd, bf16, center);
        return norm_variant<8, 4, 16>(bwd, bf16, center);
    }
    // (wider than 1024: few rows only)
    if (N <= 128) return norm_variant<1, 4, 1>(bwd, bf16, center);
    if (N <= 1024) return norm_variant<1, 8, 4>(bwd, bf16, center);
    if (N <= 4096) return norm_variant<1, 8, 16>(bwd, bf16, center);
    return norm_variant<1, 32, 16>(bwd, bf16, center);
}
// How a stream kernel is launched.
struct NormStream {
    const void* fn;
    std::atomic<unsigned long long>* ready;      // devices on which the kernel may use kNormSmemMost
    int threads, smem, G, rows, pitch;
    int64_t ctas;
};
// Shared memory of any of them at most.  A kernel's limit is set once per device and to this, not to a call's own size: it belongs to the process, and a
// smaller call in another thread would lower it between a call's setting and its launch.
constexpr int kNormSmemMost = 160 * 1024;
template <int PITCH>
NormStream norm_stream(bool bwd, bool bf16, bool center, int N) {
    static std::atomic<unsigned long long> ready[8];
    static_assert(NormShape<PITCH, true>::kGroupBytes * (PITCH <= 4096 ? 4096 / PITCH : 1) <= kNormSmemMost, "shared memory");
    NormStream v = {};
    v.ready = &ready[4 * bwd + 2 * bf16 + center];
    if (bwd) v.fn = bf16 ? (center ? (const void*)norm_bwd_stream_kernel<PITCH, true, true> : (const void*)norm_bwd_stream_kernel<PITCH, true, false>)
                         : (center ? (const void*)norm_bwd_stream_kernel<PITCH, false, true> : (const void*)norm_bwd_stream_kernel<PITCH, false, false>);
    else v.fn = bf16 ? (center ? (const void*)norm_fwd_stream_kernel<PITCH, true, true> : (const void*)norm_fwd_stream_kernel<PITCH, true, false>)
                     : (center ? (const void*)norm_fwd_stream_kernel<PITCH, false, true> : (const void*)norm_fwd_stream_kernel<PITCH, false, false>);
    const int per = bwd ? NormShape<PITCH, true>::kPacks : NormShape<PITCH, false>::kPacks;
    v.G = (N / 8 + 32 * per - 1) / (32 * per) * 32;
    const int groups = v.G >= 256 ? 1 : 256 / v.G;
    v.threads = groups * v.G;
    v.smem = groups * (bwd ? NormShape<PITCH, true>::kGroupBytes : NormShape<PITCH, false>::kGroupBytes);
    v.rows = groups * (bwd ? NormShape<PITCH, true>::kRows : NormShape<PITCH, false>::kRows);
    return v;
}
template <int COLS, int ROWS>
NormStream norm_ragged(bool bwd, bool bf16, bool center, int N) {
    static std::atomic<unsigned long long> ready[8];
    NormStream v = {};
    v.ready = &ready[4 * bwd + 2 * bf16 + center];
    if (bwd) v.fn = bf16 ? (center ? (const void*)norm_bwd_ragged_kernel<COLS, ROWS, true, true> : (const void*)norm_bwd_ragged_kernel<COLS, ROWS, true, false>)
                         : (center ? (const void*)norm_bwd_ragged_kernel<COLS, ROWS, false, true> : (const void*)norm_bwd_ragged_kernel<COLS, ROWS, false, false>);
    else v.fn = bf16 ? (center ? (const void*)norm_fwd_ragged_kernel<COLS, ROWS, true, true> : (const void*)norm_fwd_ragged_kernel<COLS, ROWS, true, false>)
                     : (center ? (const void*)norm_fwd_ragged_kernel<COLS, ROWS, false, true> : (const void*)norm_fwd_ragged_kernel<COLS, ROWS, false, false>);
    v.G = (N + 32 * COLS - 1) / (32 * COLS) * 32;
    v.pitch = (2 * N + 14 + 15) / 16 * 16;
    const int groups = v.G >= 256 ? 1 : 256 / v.G;
    v.threads = groups * v.G;
    v.smem = groups * 2 * ROWS * (bwd ? 2 : 1) * v.pitch;
    v.rows = groups * ROWS;
    return v;
}
// A class of its own for 4104 to 5120 columns, us with it and in the class of 8192 (16384 rows of layer norm): 4352 51.6 and 64.5 forward, 87.8 and 99.8 backward, 5120
// 57.6 and 67.7, 93.1 and 103.4.  6144 and 7168 reach 5.3 to 5.5 TB/s in that class, as 5120 does in its own (5.8 and 5.4).
int choose_stream(bool bwd, bool bf16, bool center, bool vec, const NormParams& P, NormStream& v) {
    const int N = P.N;
    if (!vec) v = N <= 4096 ? norm_ragged<16, 4>(bwd, bf16, center, N) : N <= 8192 ? norm_ragged<16, 2>(bwd, bf16, center, N) : norm_ragged<32, 1>(bwd, bf16, center, N);
    else v = N <= 256    ? norm_stream<512>(bwd, bf16, center, N)
        : N <= 512  ? norm_stream<1024>(bwd, bf16, center, N)
        : N <= 1024 ? norm_stream<2048>(bwd, bf16, center, N)
        : N <= 2048 ? norm_stream<4096>(bwd, bf16, center, N)
        : N <= 4096 ? norm_stream<8192>(bwd, bf16, center, N)
        : N <= 5120 ? norm_stream<10240>(bwd, bf16, center, N)
        : N <= 8192 ? norm_stream<16384>(bwd, bf16, center, N)
                    : norm_stream<32768>(bwd, bf16, center, N);
    int dev = 0, per_sm = 1;
    NQ_CUDA_TRY(cudaGetDevice(&dev));
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(*v.ready & bit)) {
        NQ_CUDA_TRY(cudaFuncSetAttribute(v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmemMost));
        *v.ready |= bit;
    }
    NQ_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, v.fn, v.threads, v.smem));
    const int most = bwd ? norm_ctas_per_sm(N) : 8;
    per_sm = per_sm < 1 ? 1 : per_sm > most ? most : per_sm;
    const int64_t units = (P.rows + v.rows - 1) / v.rows;
    v.ctas = units < (int64_t)per_sm * sm_count() ? units : (int64_t)per_sm * sm_count();
    return NQ_OK;
}
int launch_stream(const NormStream& v, const NormParams& P, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)v.ctas);
    cfg.blockDim = dim3(v.threads);
    cfg.dynamicSmemBytes = v.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    NormParams p = P;
    int G = v.G, pitch = v.pitch;
    void* args[] = {&p, &G, &pitch};       // (the last one for the ragged kernels)
    return launch_dependent(cfg, attr, 0, v.fn, args);
}
int launch_norm(const NormVariant& v, long long ctas, const NormParams& P, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(v.threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    NormParams p = P;
    void* args[] = {&p};
    return launch_dependent(cfg, attr, 0, (const void*)v.fn, args);
}
bool norm_rows_aligned(const void* p, long long ld) { return aligned16(p) && ld % 8 == 0; }
// Direct kernels for few rows, and for short rows at any address (8192 x 1003 of layer norm, us: forward 14.2 and 21.1 ragged, backward 24.8 and 37.4;
// 8000 x 5001: 147 and 107, 322 and 119).
bool norm_streamed(bool vec, int64_t rows, int64_t N) { return rows > 2 * sm_count() && (vec || N > 1024); }

}  // namespace nq

using namespace nq;

extern "C" {

int nq_norm_max_columns(void) { return kNormMaxCols; }

int nq_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats, int64_t rows, int64_t N,
                int64_t ldx, int64_t ldy, float eps, int center, int dtype, int weight_dtype, nq_stream_t stream) {
    if (!x || !y) return NQ_ERR_NULL;
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (weight_dtype != dtype && weight_dtype != NQ_F32) return NQ_ERR_DTYPE;
    if (rows < 1 || N < 1 || ldx < 0 || ldy < N) return NQ_ERR_SHAPE;
    if (N > kNormMaxCols || rows > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    if (bias && !center) return NQ_ERR_UNSUPPORTED;
    if (!aligned_to(2, x, y) || !aligned_to(weight_dtype == NQ_F32 ? 4 : 2, weight, bias) || !aligned_to(8, stats)) return NQ_ERR_ALIGN;
    NormParams P = {};
    P.x = x; P.w = weight; P.b = bias; P.y = y; P.stats = reinterpret_cast<float2*>(stats);
    P.rows = rows; P.ldx = ldx; P.ldy = ldy; P.N = (int)N; P.w32 = weight_dtype == NQ_F32;
    P.eps = eps; P.inv_n = 1.f / (float)N;
    const bool vec = N % 8 == 0 && norm_rows_aligned(x, ldx) && norm_rows_aligned(y, ldy) && aligned16(weight) && aligned16(bias);
    if (norm_streamed(vec, rows, N)) {
        NormStream v = {};
        const int st = choose_stream(false, dtype == NQ_BF16, center != 0, vec, P, v);
        return st != NQ_OK ? st : launch_stream(v, P, as_stream(stream));
    }
    const NormVariant v = choose_norm(false, dtype == NQ_BF16, center != 0, vec, (int)N);
    return launch_norm(v, (rows + v.rows_per_cta - 1) / v.rows_per_cta, P, as_stream(stream));
}

size_t nq_norm_bwd_scratch_bytes(int64_t rows, int64_t N) {
    if (rows < 1 || N < 1 || N > kNormMaxCols) return 0;
    const int64_t most = (int64_t)norm_ctas_per_sm(N) * sm_count(), ctas = rows < most ? rows : most;
    return (size_t)(ctas * N * 2 * 4);
}

int nq_norm_bwd(const void* dy, const void* x, const void* weight, const float* stats, void* dx, void* dweight, void* dbias,
                void* scratch, size_t scratch_bytes, int64_t rows, int64_t N, int64_t lddy, int64_t ldx, int64_t lddx,
                int center, int dtype, int weight_dtype, nq_stream_t stream) {
    if (!dy || !x || !stats) return NQ_ERR_NULL;
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (weight_dtype != dtype && weight_dtype != NQ_F32) return NQ_ERR_DTYPE;
    if (rows < 1 || N < 1 || ldx < 0 || lddy < 0 || (dx && lddx < N)) return NQ_ERR_SHAPE;
    if (N > kNormMaxCols || rows > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    if (dbias && !center) return NQ_ERR_UNSUPPORTED;
    if (!aligned_to(2, dy, x, dx) || !aligned_to(weight_dtype == NQ_F32 ? 4 : 2, weight, dweight, dbias) || !aligned_to(8, stats)) return NQ_ERR_ALIGN;
    if (!dx && !dweight && !dbias) return NQ_OK;
    const bool sums = dweight || dbias;
    if (sums && !scratch) return NQ_ERR_NULL;
    if (sums && scratch_bytes < nq_norm_bwd_scratch_bytes(rows, N)) return NQ_ERR_SCRATCH;
    if (sums && !aligned16(scratch)) return NQ_ERR_ALIGN;
    const bool bf16 = dtype == NQ_BF16;
    const bool vec = N % 8 == 0 && norm_rows_aligned(x, ldx) && norm_rows_aligned(dy, lddy) && (!dx || norm_rows_aligned(dx, lddx)) &&
                     aligned16(weight);
    const bool streamed = norm_streamed(vec, rows, N);
    NormParams P = {};
    P.x = x; P.w = weight; P.dy = dy; P.y = dx; P.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    P.rows = rows; P.ldx = ldx; P.lddy = lddy; P.ldy = lddx; P.N = (int)N; P.w32 = weight_dtype == NQ_F32;
    NormVariant v = {};
    NormStream sv = {};
    int64_t ctas = 0;
    if (streamed) {
        const int st = choose_stream(true, bf16, center != 0, vec, P, sv);
        if (st != NQ_OK) return st;
        ctas = sv.ctas;
    } else {
        v = choose_norm(true, bf16, center != 0, vec, (int)N);
        int per_sm = 0;
        NQ_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, (const void*)v.fn, v.threads, 0));
        const int most = norm_ctas_per_sm(N);
        per_sm = per_sm < 1 ? 1 : per_sm > most ? most : per_sm;
        ctas = (rows + v.rows_per_cta - 1) / v.rows_per_cta;
        if (ctas > (int64_t)per_sm * sm_count()) ctas = (int64_t)per_sm * sm_count();
    }
    P.part_w = dweight ? static_cast<float*>(scratch) : nullptr;
    P.part_b = dbias ? static_cast<float*>(scratch) + (size_t)ctas * N : nullptr;
    P.inv_n = 1.f / (float)N;
    const int st = streamed ? launch_stream(sv, P, as_stream(stream)) : launch_norm(v, ctas, P, as_stream(stream));
    if (st != NQ_OK || !sums) return st;
    const void* fn = bf16 ? (const void*)norm_reduce_kernel<true> : (const void*)norm_reduce_kernel<false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((N + 31) / 32), dbias ? 2 : 1);
    cfg.blockDim = dim3(1024);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    int n_ctas = (int)ctas, cols = (int)N;
    void* args[] = {&P.part_w, &P.part_b, &dweight, &dbias, &n_ctas, &cols, &P.w32};
    return launch_dependent(cfg, attr, 0, fn, args);
}

}  // extern "C"
