// Layer norm and RMS norm of 16-bit activations, forward and backward:
//
//     y = (x - m) r w + b        m = mean(x), or 0 (RMS)        r = 1 / sqrt(mean((x - m)^2) + eps)
//     dx = r (g - mean(g) - xhat mean(g xhat))                  g = dy w, xhat = (x - m) r (mean(g) only where m is subtracted)
//     dw = sum_rows dy xhat        db = sum_rows dy
//
// Bound by memory: forward 2 bytes in and 2 out per element, backward 4 in and 2 out.  Every element is read once: a group of warps
// holds a row in registers (the mean, then the sum of squares of the differences, all in fp32, cost no second read).  Groups are sized by
// the row, and for few rows a thread takes fewer columns, so that one token's row is a single load per thread.
//
// Backward.  A group takes rows `first, first + groups, ...`; a thread has the same columns of each and adds dy xhat and dy to fp32 sums
// in registers.  One row of partial sums per CTA goes to the scratch; a second kernel adds these in a fixed order, so results do not
// depend on timing.
#include "nq_common.cuh"

namespace nq {

constexpr int kNormMaxCols = 16384;
constexpr int kNormCtasPerSm = 4;          // of the backward kernel at most: rows of partial sums per SM

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
// VEC consecutive elements (one 16-byte load, or a single element) as they are, and as floats.
template <int VEC> struct NormVec { uint32_t w[VEC / 2]; };
template <> struct NormVec<1> { uint16_t h; };
template <int VEC>
__device__ __forceinline__ NormVec<VEC> norm_load(const void* p, long long i, bool live) {
    NormVec<VEC> v = {};
    if (live) {
        if constexpr (VEC == 1) v.h = __ldg(static_cast<const uint16_t*>(p) + i);
        else {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
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
        if constexpr (VEC == 1) f[0] = __ldg(q);
        else {
            const float4 a = __ldg(reinterpret_cast<const float4*>(q)), b = __ldg(reinterpret_cast<const float4*>(q) + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        }
    } else {
        const NormVec<VEC> v = norm_load<VEC>(p, c, true);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = norm_at<VEC, BF16>(v, e);
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
        mean = group_sum2<WARPS>(s, red, turn).x * P.inv_n;
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
        const float2 st = __ldg(P.stats + row);
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

// out[c] = sum over the CTAs of part[i][c]: 32 columns a CTA, eight warps over the rows, then over the warps.
template <bool BF16>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* part_w, const float* part_b, void* dw, void* db, int ctas, int N, int w32) {
    __shared__ float red[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* part = blockIdx.y ? part_b : part_w;
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    float s = 0.f;
    if (c < N) {
#pragma unroll 4
        for (int i = warp; i < ctas; i += 8) s += part[(size_t)i * N + c];
    }
    red[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < N) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[k][lane];
        if (w32) static_cast<float*>(out)[c] = s;
        else static_cast<uint16_t*>(out)[c] = (uint16_t)norm_pack<BF16>(s, 0.f);
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
// The smallest group that holds a row.  16-byte loads where every row starts at a 16-byte boundary, single elements otherwise.
NormVariant choose_norm(bool bwd, bool bf16, bool center, bool vec, long long rows, int N) {
    if (vec) {
        const int packs = (N + 7) / 8;
        if (packs <= 64) return norm_variant<8, 2, 1>(bwd, bf16, center);
        if (rows <= 2 * sm_count() && packs <= 512)      // few rows: one load a thread
            return packs <= 128 ? norm_variant<8, 1, 4>(bwd, bf16, center) : norm_variant<8, 1, 16>(bwd, bf16, center);
        if (packs <= 256) return norm_variant<8, 2, 4>(bwd, bf16, center);
        if (packs <= 512) return norm_variant<8, 2, 8>(bwd, bf16, center);
        if (packs <= 1024) return norm_variant<8, 2, 16>(bwd, bf16, center);
        return norm_variant<8, 4, 16>(bwd, bf16, center);
    }
    if (N <= 128) return norm_variant<1, 4, 1>(bwd, bf16, center);
    if (N <= 1024) return norm_variant<1, 8, 4>(bwd, bf16, center);
    if (N <= 4096) return norm_variant<1, 8, 16>(bwd, bf16, center);
    return norm_variant<1, 32, 16>(bwd, bf16, center);
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
    NormParams P = {};
    P.x = x; P.w = weight; P.b = bias; P.y = y; P.stats = reinterpret_cast<float2*>(stats);
    P.rows = rows; P.ldx = ldx; P.ldy = ldy; P.N = (int)N; P.w32 = weight_dtype == NQ_F32;
    P.eps = eps; P.inv_n = 1.f / (float)N;
    const bool vec = N % 8 == 0 && norm_rows_aligned(x, ldx) && norm_rows_aligned(y, ldy) && aligned16(weight) && aligned16(bias);
    const NormVariant v = choose_norm(false, dtype == NQ_BF16, center != 0, vec, rows, (int)N);
    return launch_norm(v, (rows + v.rows_per_cta - 1) / v.rows_per_cta, P, as_stream(stream));
}

size_t nq_norm_bwd_scratch_bytes(int64_t rows, int64_t N) {
    if (rows < 1 || N < 1 || N > kNormMaxCols) return 0;
    const int64_t most = (int64_t)kNormCtasPerSm * sm_count(), ctas = rows < most ? rows : most;
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
    if (!dx && !dweight && !dbias) return NQ_OK;
    const bool sums = dweight || dbias;
    if (sums && !scratch) return NQ_ERR_NULL;
    if (sums && scratch_bytes < nq_norm_bwd_scratch_bytes(rows, N)) return NQ_ERR_SCRATCH;
    if (sums && !aligned16(scratch)) return NQ_ERR_ALIGN;
    const bool bf16 = dtype == NQ_BF16;
    const bool vec = N % 8 == 0 && norm_rows_aligned(x, ldx) && norm_rows_aligned(dy, lddy) && (!dx || norm_rows_aligned(dx, lddx)) &&
                     aligned16(weight);
    const NormVariant v = choose_norm(true, bf16, center != 0, vec, rows, (int)N);
    int per_sm = 0;
    NQ_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, (const void*)v.fn, v.threads, 0));
    per_sm = per_sm < 1 ? 1 : per_sm > kNormCtasPerSm ? kNormCtasPerSm : per_sm;
    int64_t ctas = (rows + v.rows_per_cta - 1) / v.rows_per_cta;
    if (ctas > (int64_t)per_sm * sm_count()) ctas = (int64_t)per_sm * sm_count();
    NormParams P = {};
    P.x = x; P.w = weight; P.dy = dy; P.y = dx; P.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    P.part_w = dweight ? static_cast<float*>(scratch) : nullptr;
    P.part_b = dbias ? static_cast<float*>(scratch) + (size_t)ctas * N : nullptr;
    P.rows = rows; P.ldx = ldx; P.lddy = lddy; P.ldy = lddx; P.N = (int)N; P.w32 = weight_dtype == NQ_F32;
    P.inv_n = 1.f / (float)N;
    const int st = launch_norm(v, ctas, P, as_stream(stream));
    if (st != NQ_OK || !sums) return st;
    const void* fn = bf16 ? (const void*)norm_reduce_kernel<true> : (const void*)norm_reduce_kernel<false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((N + 31) / 32), dbias ? 2 : 1);
    cfg.blockDim = dim3(256);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    int n_ctas = (int)ctas, cols = (int)N;
    void* args[] = {&P.part_w, &P.part_b, &dweight, &dbias, &n_ctas, &cols, &P.w32};
    return launch_dependent(cfg, attr, 0, fn, args);
}

}  // extern "C"
