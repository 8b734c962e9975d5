// Linear with 8-bit weights and activations:
//
//     y[t, v] = s_x[t] s_w[v] sum_k q_x[t, k] q_w[v, k] (+ bias[v])
//
// s = max|x| / 127 of the token (or, for weights, of the output channel) and q = rint(127 x / max|x|).  The activations are quantised in a kernel
// of its own, one CTA per token; the product's CTAs load their first weights meanwhile.  Sums of products are exact (int32, K up to
// 2^31 / 127^2); the two scales are multiplied and applied in fp32.
//
// Few tokens are bound by the memory that the weights stream from: K V bytes, half of the 16-bit head.  The tokens are the MMA's 128
// rows and the output channels its columns, so any number of tokens up to 128 costs the same reads.  Prompts are bound by the tensor
// cores, pairs of CTAs on 256 x 256 tiles.
#include "nq_common.cuh"
#include "nq_mm.cuh"

namespace nq {

constexpr int kInt8MaxCols = 131072;      // 127^2 * 2^17 < 2^31

template <bool BF16>
__device__ __forceinline__ float q8_float(uint32_t w, int half) {
    const uint16_t h = (uint16_t)(w >> (16 * half));
    return io_float(h, BF16);
}
// 127 x is exact and the division IEEE, so that the result is that of the definition: 16-bit x and max|x| have at most 11 significant bits, and
// 127 x / max|x| is half a whole number exactly (x = max|x| / 2 is: 63.5, to 64) or further from it than the quotient's rounding.  (x / s in fp32
// would decide such halves by the rounding of s.)
__device__ __forceinline__ int q8_round(float x, float top) { return (int)rintf(127.f * x / top); }

// VEC: elements per load (8: 16 bytes in, 8 out; 1: any alignment).
template <bool BF16, int VEC>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const uint16_t* x, int8_t* q, float* scale, int N, long long ldx, long long ldq, int release) {
    __shared__ float red[16];
    const long long row = blockIdx.x;
    const uint16_t* xr = x + row * ldx;
    int8_t* qr = q + row * ldq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (behind the wait: what starts early may rely on everything before this kernel)
    if (release) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float top = 0.f;
#pragma unroll 2
    for (int c = tid * VEC; c < N; c += blockDim.x * VEC) {
        if constexpr (VEC == 8) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(xr + c));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max_or_nan(top, fabsf(q8_float<BF16>(w[e >> 1], e & 1)));
        } else {
            top = max_or_nan(top, fabsf(q8_float<BF16>(__ldg(xr + c), 0)));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) top = max_or_nan(top, red[i]);
    // a NaN or an infinity makes every output of the row NaN: a NaN scale, and zeros
    const float s = top <= 3.4e38f ? top / 127.f : __int_as_float(0x7fffffff);
    if (tid == 0) scale[row] = s;
    const bool live = s > 0.f;
#pragma unroll 2
    for (int c = tid * VEC; c < N; c += blockDim.x * VEC) {
        if constexpr (VEC == 8) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(xr + c));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            uint32_t o[2] = {0u, 0u};
            if (live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e >> 2] |= (uint32_t)(q8_round(q8_float<BF16>(w[e >> 1], e & 1), top) & 0xff) << (8 * (e & 3));
            }
            *reinterpret_cast<uint2*>(qr + c) = make_uint2(o[0], o[1]);
        } else {
            qr[c] = live ? (int8_t)q8_round(q8_float<BF16>(__ldg(xr + c), 0), top) : (int8_t)0;
        }
    }
}

static int launch_quantize(const void* x, int8_t* q, float* scale, int64_t rows, int64_t N, int64_t ldx, int64_t ldq, int bf16, int release, cudaStream_t stream) {
    const bool vec = aligned16(x) && ldx % 8 == 0 && N % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
    const int64_t per = vec ? 8 : 1;
    int threads = (int)((N + per * 32 - 1) / (per * 32) * 32);
    if (threads > 512) threads = 512;
    const void* fn = vec ? (bf16 ? (const void*)quantize_rows_kernel<true, 8> : (const void*)quantize_rows_kernel<false, 8>)
                         : (bf16 ? (const void*)quantize_rows_kernel<true, 1> : (const void*)quantize_rows_kernel<false, 1>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    int n = (int)N;
    long long lx = ldx, lq = ldq;
    void* args[] = {&x, &q, &scale, &n, &lx, &lq, &release};
    return launch_dependent(cfg, attr, 0, fn, args);
}

template <int OUT>
struct Int8Epilogue {
    static constexpr bool kS8 = true;
    struct Params {
        const float *xs, *ws;
        const uint16_t* bias;
        uint16_t* y;
        long long ldy;
        int wide;
    };
    const Params& p;
    const MmShape& s;
    float sx;
    int n0, row0;
    __device__ Int8Epilogue(const Params& p_, const MmShape& s_) : p(p_), s(s_) {}
    __device__ __forceinline__ void begin(int row, int n0_, int, int, int) {
        n0 = n0_;
        row0 = row & ~31;
        sx = row < s.M ? __ldcg(p.xs + row) : 0.f;
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int cols, unsigned char* stage) {
        if (row0 >= s.M) return;                        // (the whole warp)
        const float* ws = p.ws + n0 + c;
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            float f[4];
            if (i + 4 <= cols) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(ws + i));
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = i + k < cols ? __ldg(ws + i + k) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = (float)(int)r[i + k] * (sx * f[k]);
            if (p.bias) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k < cols) f[k] += io_float(__ldg(p.bias + n0 + c + i + k), OUT != kOutFp16);
            }
            w[i / 2] = pack_outputs<OUT>(f[0], f[1], 0);
            w[i / 2 + 1] = pack_outputs<OUT>(f[2], f[3], 0);
        }
        mm_store_rows(stage, w, p.y + row0 * p.ldy + n0 + c, p.ldy, min(32, s.M - row0), cols, p.wide);
    }
    __device__ __forceinline__ void end() {}
};

template <int CG, int OUT>
static int launch_int8(const int8_t* xq, int64_t ldq, const int8_t* w, int64_t ldw, const typename Int8Epilogue<OUT>::Params& e, int T, int N, int V,
                       unsigned* status, cudaStream_t stream) {
    MmParams<Int8Epilogue<OUT>> P = {};
    P.e = e;
    const int m_tiles = (T + 128 * CG - 1) / (128 * CG);
    const int bn = mm_tile_cols(V, m_tiles, sm_count() / CG, 16 * CG, 16 * CG);
    return mm_launch<CG>(P, kMmS8, {xq, ldq, 0}, {w, ldw, 0}, T, V, N, bn, 1, 1, status, stream);
}

}  // namespace nq

using namespace nq;

extern "C" {

int nq_quantize_rows_s8(const void* x, int8_t* q, float* scale, int64_t rows, int64_t N, int64_t ldx, int64_t ldq, int dtype,
                        nq_stream_t stream) {
    if (!x || !q || !scale) return NQ_ERR_NULL;
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (rows < 1 || N < 1 || ldx < 0 || ldq < N) return NQ_ERR_SHAPE;
    if (rows > 0x7fffffff || N > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    return launch_quantize(x, q, scale, rows, N, ldx, ldq, dtype == NQ_BF16, 0, as_stream(stream));
}

size_t nq_int8_linear_scratch_bytes(int64_t T, int64_t N) {
    if (T < 1 || N < 1) return 0;
    return (size_t)((T * 4 + 255) / 256 * 256 + T * ((N + 15) / 16 * 16));
}

int nq_int8_linear_fwd(const void* x, const int8_t* w, const float* w_scale, const void* bias, void* y, void* scratch, size_t scratch_bytes,
                       void* status_word, int64_t T, int64_t N, int64_t V, int64_t ldx, int64_t ldw, int64_t ldy, int dtype,
                       nq_stream_t stream) {
    if (!x || !w || !w_scale || !y || !scratch || !status_word) return NQ_ERR_NULL;
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (T < 1 || N < 1 || V < 1 || ldx < 0 || ldw < N || ldw % 16 || ldy < V) return NQ_ERR_SHAPE;
    if (N > kInt8MaxCols || T > 0x1fffffff || V > 0x1fffffff) return NQ_ERR_TOO_LARGE;
    if (!aligned16(w) || !aligned16(w_scale) || !aligned16(scratch) || !aligned16(status_word)) return NQ_ERR_ALIGN;
    if (scratch_bytes < nq_int8_linear_scratch_bytes(T, N)) return NQ_ERR_SCRATCH;
    const bool bf16 = dtype == NQ_BF16;
    float* xs = static_cast<float*>(scratch);
    int8_t* xq = static_cast<int8_t*>(scratch) + (T * 4 + 255) / 256 * 256;
    const int64_t ldq = (N + 15) / 16 * 16;
    cudaStream_t s = as_stream(stream);
    unsigned* status = static_cast<unsigned*>(status_word) + 2;
    const int st = launch_quantize(x, xq, xs, T, N, ldx, ldq, bf16, 1, s);
    if (st != NQ_OK) return st;
    auto params = [&](auto& e) {
        e.xs = xs; e.ws = w_scale; e.bias = static_cast<const uint16_t*>(bias); e.y = static_cast<uint16_t*>(y); e.ldy = ldy;
        e.wide = aligned16(y) && ldy % 8 == 0;
    };
    if (bf16) {
        Int8Epilogue<kOutBf16>::Params e;
        params(e);
        return T <= 128 ? launch_int8<1, kOutBf16>(xq, ldq, w, ldw, e, (int)T, (int)N, (int)V, status, s)
                        : launch_int8<2, kOutBf16>(xq, ldq, w, ldw, e, (int)T, (int)N, (int)V, status, s);
    }
    Int8Epilogue<kOutFp16>::Params e;
    params(e);
    return T <= 128 ? launch_int8<1, kOutFp16>(xq, ldq, w, ldw, e, (int)T, (int)N, (int)V, status, s)
                    : launch_int8<2, kOutFp16>(xq, ldq, w, ldw, e, (int)T, (int)N, (int)V, status, s);
}

}  // extern "C"
