// Linear with 8-bit weights and activations:
//
//     y[t, v] = s_x[t] s_w[v] sum_k q_x[t, k] q_w[v, k] (+ bias[v])
//
// s = max|x| / 127 of the token (or, for weights, of the output channel) and q = rint(127 x / max|x|).  The activations are quantised in a kernel
// of its own, one CTA per token; the product's CTAs load their first weights meanwhile.  Sums of products are exact (int32, K up to
// 2^31 / 127^2); the two scales are applied in fp32, the channel's first.
//
// Few tokens are bound by the memory that the weights stream from: K V bytes, half of the 16-bit head.  The tokens are the MMA's 128
// rows and the output channels its columns, so any number of tokens up to 128 costs the same reads.  Prompts are bound by the tensor
// cores, pairs of CTAs on tiles of 256 rows and up to 256 columns.
#include "nq_common.cuh"
#include "nq_mm.cuh"

namespace nq {

constexpr int kInt8MaxCols = 131072;      // 127^2 * 2^17 < 2^31

__device__ __forceinline__ float q8_nan() { return __int_as_float(0x7fffffff); }
// The largest |x| of a row is found on the bits: without the sign, those of both types are ordered like their values, a NaN above an infinity above
// the numbers.
__device__ __forceinline__ uint32_t q8_top(const uint4& u, uint32_t top) {
    const uint32_t mask = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(__vmaxu2(u.x & mask, u.y & mask), __vmaxu2(u.z & mask, u.w & mask)), top);
}
__device__ __forceinline__ uint32_t warp_top(uint32_t top) {      // of both halves
    top = max(top & 0xffffu, top >> 16);
    return __reduce_max_sync(0xffffffffu, top);
}
// What a row is quantised by, from the bits of its largest |x|: a NaN or an infinity makes every output of the row NaN (a NaN scale, and zeros).
struct Q8Row {
    float top, inv, scale;
    bool live;
};
template <bool BF16>
__device__ __forceinline__ Q8Row q8_row(uint32_t top_bits) {
    Q8Row r;
    r.top = io_float((uint16_t)top_bits, BF16);
    r.scale = r.top <= 3.4e38f ? r.top / 127.f : q8_nan();
    r.inv = 127.f / r.top;
    r.live = r.scale > 0.f;
    return r;
}
// 127 x is exact and the division IEEE, so that the result is that of the definition: 16-bit x and max|x| have at most 11 significant bits, and
// 127 x / max|x| is half a whole number exactly (x = max|x| / 2 is: 63.5, to 64) or further from it than the quotient's rounding.  (x / s in fp32
// would decide such halves by the rounding of s.)  Both times 2^-8, exactly (bf16 has no unit below 2^-133), where 127 x could leave fp32.
__device__ __forceinline__ int q8_exact(float x, float top) {
    const float unit = top > 1e36f ? 0.00390625f : 1.f;
    return (int)rintf(127.f * (x * unit) / (top * unit));
}
// Eight values, as bytes.  The products with `inv` are off by 2^-16 at most, so that only quotients within 2^-14 of a half need the division (or where
// `inv` has overflowed); adding 1.5 2^23 leaves a whole number in the low bits.
template <bool BF16>
__device__ __forceinline__ uint2 q8_pack(const uint4& u, const Q8Row& q) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t r[8];
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = io_float((uint16_t)(w[e >> 1] >> (16 * (e & 1))), BF16) * q.inv, m = t + 12582912.f;
        off = max_or_nan(off, fabsf(t - (m - 12582912.f)));
        r[e] = __float_as_uint(m);
    }
    if (!(off <= 0.49993896484375f)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (uint32_t)q8_exact(io_float((uint16_t)(w[e >> 1] >> (16 * (e & 1))), BF16), q.top);
    }
    uint2 o;
    o.x = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
    return q.live ? o : make_uint2(0u, 0u);
}
template <bool BF16>
__device__ __forceinline__ int8_t q8_one(uint16_t x, const Q8Row& q) { return q.live ? (int8_t)q8_exact(io_float(x, BF16), q.top) : (int8_t)0; }

// (As in all kernels here, nothing is read by the non-coherent path: the kernel that writes the activations may have released this one early.)
// A row per CTA.  PACKS > 0: 16-byte loads, PACKS of eight values a thread, kept in registers; 0: single values at any address, read twice.
template <bool BF16, int PACKS>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const uint16_t* x, int8_t* q, float* scale, int N, long long ldx, long long ldq, int release) {
    __shared__ uint32_t red[16];
    const long long row = blockIdx.x;
    const uint16_t* xr = x + row * ldx;
    int8_t* qr = q + row * ldq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (behind the wait: what starts early may rely on everything before this kernel)
    if (release) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t top = 0;
    uint4 v[PACKS > 0 ? PACKS : 1];
    if constexpr (PACKS > 0) {
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int c = (p * (int)blockDim.x + tid) * 8;
            v[p] = c < N ? __ldcg(reinterpret_cast<const uint4*>(xr + c)) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int p = 0; p < PACKS; ++p) top = q8_top(v[p], top);
    } else {
#pragma unroll 4
        for (int c = tid; c < N; c += blockDim.x) top = max(top, (uint32_t)(__ldca(xr + c) & 0x7fff));
    }
    top = warp_top(top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) top = max(top, red[i]);
    const Q8Row by = q8_row<BF16>(top);
    if (tid == 0) scale[row] = by.scale;
    if constexpr (PACKS > 0) {
#pragma unroll
        for (int p = 0; p < PACKS; ++p) {
            const int c = (p * (int)blockDim.x + tid) * 8;
            if (c < N) *reinterpret_cast<uint2*>(qr + c) = q8_pack<BF16>(v[p], by);
        }
    } else {
#pragma unroll 4
        for (int c = tid; c < N; c += blockDim.x) qr[c] = q8_one<BF16>(__ldca(xr + c), by);
    }
}
template <int PACKS>
static const void* quantize_fn(int bf16) {
    return bf16 ? (const void*)quantize_rows_kernel<true, PACKS> : (const void*)quantize_rows_kernel<false, PACKS>;
}

static int launch_quantize(const void* x, int8_t* q, float* scale, int64_t rows, int64_t N, int64_t ldx, int64_t ldq, int bf16, int release, cudaStream_t stream) {
    // Many rows: four packs a thread, so that all rows' CTAs are there at once (2048 x 4096: 8.8 us); few: one.
    const bool vec = aligned16(x) && ldx % 8 == 0 && N % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0 && N <= 8 * 8 * 512;
    const int64_t packs = (N + 7) / 8;
    const int per = !vec ? 0 : packs > 4 * 512 ? 8 : packs > 512 || (rows > 2 * sm_count() && packs >= 128) ? 4 : 1;
    const int64_t need = vec ? (packs + per - 1) / per : N;
    const int threads = (int)(need > 512 ? 512 : (need + 31) / 32 * 32);
    const void* fn = per == 8 ? quantize_fn<8>(bf16) : per == 4 ? quantize_fn<4>(bf16) : per == 1 ? quantize_fn<1>(bf16) : quantize_fn<0>(bf16);
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

// FEW: up to kInt8Few tokens, quantised by every CTA for itself, beside its first weights' loads (one launch, no copy of the quantised
// activations); otherwise their bytes and scales are in memory.  us with and without: one token 97.6 and 102.5 (151936 x 4096), 8.0 and 11.7 (512 x
// 2048); two 100.3 and 102.6; four 104.1 and 103.3, sixteen 32.7 and 16.6 (12288 x 4096: every SM reads and converts all tokens).
constexpr int kInt8Few = 2, kInt8FewBytes = 96 * 1024;       // tokens; bytes of A in shared memory
template <int OUT, bool FEW>
struct Int8Epilogue {
    static constexpr bool kS8 = true, kBuildA = FEW;
    static constexpr int kChunk = 0;
    struct Params {
        const float *xs, *ws;
        const uint16_t* bias;
        uint16_t* y;
        long long ldy;
        int wide;
        const uint16_t* x;         // FEW
        long long ldx;
        int N, vec;
    };
    // `few`: scales of the tokens, then the warps' maxima
    static __device__ __forceinline__ void build(const Params& p, const MmShape& s, unsigned char* a, unsigned char* few) {
        constexpr bool BF16 = OUT != kOutFp16;
        float* scales = reinterpret_cast<float*>(few);
        uint32_t* tops = reinterpret_cast<uint32_t*>(few) + kInt8Few;
        const int warp = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31, T = s.M;
        const int share = kMmEpilogueWarps / T;                             // warps of a token
        {
            const int t = warp / share, part = warp % share;
            const uint16_t* x = p.x + (long long)t * p.ldx;
            uint32_t top = 0;
            if (p.vec) {
#pragma unroll 8
                for (int c = (part * 32 + lane) * 8; c < p.N; c += share * 256) top = q8_top(__ldca(reinterpret_cast<const uint4*>(x + c)), top);
            } else {
#pragma unroll 8
                for (int c = part * 32 + lane; c < p.N; c += share * 32) top = max(top, (uint32_t)(__ldca(x + c) & 0x7fff));
            }
            top = warp_top(top);
            if (lane == 0) tops[warp] = top;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kMmEpilogueWarps) : "memory");
            for (int i = 0; i < share; ++i) top = max(top, tops[warp - part + i]);
            const Q8Row by = q8_row<BF16>(top);
            if (part == 0 && lane == 0) scales[t] = by.scale;
            // row t: step c / 128, 16-byte unit (c / 16) mod 8 swizzled by the row
            unsigned char* row = a + t * 128;
            auto at = [&](int c) { return row + (c >> 7) * s.few + ((((c >> 4) & 7) ^ t) << 4) + (c & 15); };
            if (p.vec) {
#pragma unroll 8
                for (int c = (part * 32 + lane) * 8; c < p.N; c += share * 256)
                    *reinterpret_cast<uint2*>(at(c)) = q8_pack<BF16>(__ldca(reinterpret_cast<const uint4*>(x + c)), by);
            } else {
                for (int c = part * 32 + lane; c < p.N; c += share * 32) *at(c) = (unsigned char)q8_one<BF16>(__ldca(x + c), by);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kMmEpilogueWarps) : "memory");      // (the scales)
    }
    const float* few;
    const Params& p;
    const MmShape& s;
    float sx;
    int n0, row0;
    __device__ Int8Epilogue(const Params& p_, const MmShape& s_, const unsigned char* few_, const volatile MmDims*) : few(reinterpret_cast<const float*>(few_)), p(p_), s(s_) {}
    __device__ __forceinline__ void begin(int row, int n0_, int, int, int) {
        n0 = n0_;
        row0 = row & ~31;
        sx = row < s.M ? (FEW ? few[row] : __ldcg(p.xs + row)) : 0.f;
    }
    __device__ __forceinline__ void chunk(const uint32_t (&r)[32], int c, int cols, unsigned char* stage, int half) {
        const float* ws = p.ws + n0 + c;
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            float f[4];
            if (i + 4 <= cols) {
                const float4 v = __ldca(reinterpret_cast<const float4*>(ws + i));
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = i + k < cols ? __ldca(ws + i + k) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = (float)(int)r[i + k] * f[k] * sx;      // (s_x s_w may leave fp32 where the result does not)
            if (p.bias) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k < cols) f[k] += io_float(__ldca(p.bias + n0 + c + i + k), OUT != kOutFp16);
            }
            w[i / 2] = pack_outputs<OUT>(f[0], f[1], 0);
            w[i / 2 + 1] = pack_outputs<OUT>(f[2], f[3], 0);
        }
        mm_stage_row(stage, half, w);
    }
    __device__ __forceinline__ void flush(int c, int cols, const unsigned char* stage) {
        mm_store_rows(stage, p.y + row0 * p.ldy + n0 + c, p.ldy, min(32, s.M - row0), cols, p.wide);
    }
    __device__ __forceinline__ void end() {}
};

template <int CG, int OUT, bool FEW>
static int launch_int8(const typename Int8Epilogue<OUT, FEW>::Params& e, const int8_t* xq, int64_t ldq, const int8_t* w, int64_t ldw, int T, int V,
                       unsigned* status, cudaStream_t stream) {
    MmParams<Int8Epilogue<OUT, FEW>> P = {};
    P.e = e;
    const int m_tiles = (T + 128 * CG - 1) / (128 * CG);
    const int bn = mm_tile_cols(V, m_tiles, CG, 16 * CG);
    return mm_launch<CG>(P, kMmS8, {xq, ldq, 0}, {w, ldw, 0}, T, V, e.N, bn, 1, !FEW, 0, status, stream);
}
static bool int8_few(int64_t T, int64_t N) { return T <= kInt8Few && 1024 * ((N + 127) / 128) <= kInt8FewBytes; }
template <int OUT>
static int int8_linear(const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const float* ws, const void* bias, void* y, int64_t ldy, void* scratch,
                       int T, int N, int V, unsigned* status, cudaStream_t stream) {
    auto fill = [&](auto& e) {
        e.ws = ws; e.bias = static_cast<const uint16_t*>(bias); e.y = static_cast<uint16_t*>(y); e.ldy = ldy;
        e.wide = aligned16(y) && ldy % 8 == 0;
        e.x = static_cast<const uint16_t*>(x); e.ldx = ldx; e.N = N;
        e.vec = aligned16(x) && ldx % 8 == 0 && N % 8 == 0;
    };
    if (int8_few(T, N)) {
        typename Int8Epilogue<OUT, true>::Params e = {};
        fill(e);
        return launch_int8<1, OUT, true>(e, nullptr, 0, w, ldw, T, V, status, stream);
    }
    typename Int8Epilogue<OUT, false>::Params e = {};
    fill(e);
    float* xs = static_cast<float*>(scratch);
    int8_t* xq = static_cast<int8_t*>(scratch) + ((int64_t)T * 4 + 255) / 256 * 256;
    const int64_t ldq = (N + 15) / 16 * 16;
    e.xs = xs;
    const int st = launch_quantize(x, xq, xs, T, N, ldx, ldq, OUT != kOutFp16, 1, stream);
    if (st != NQ_OK) return st;
    return T <= 128 ? launch_int8<1, OUT, false>(e, xq, ldq, w, ldw, T, V, status, stream) : launch_int8<2, OUT, false>(e, xq, ldq, w, ldw, T, V, status, stream);
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
    if (!aligned_to(2, x) || !aligned_to(4, scale)) return NQ_ERR_ALIGN;
    return launch_quantize(x, q, scale, rows, N, ldx, ldq, dtype == NQ_BF16, 0, as_stream(stream));
}

size_t nq_int8_linear_scratch_bytes(int64_t T, int64_t N) {
    if (T < 1 || N < 1 || int8_few(T, N)) return 0;
    return (size_t)((T * 4 + 255) / 256 * 256 + T * ((N + 15) / 16 * 16));
}

int nq_int8_linear_fwd(const void* x, const int8_t* w, const float* w_scale, const void* bias, void* y, void* scratch, size_t scratch_bytes,
                       void* status_word, int64_t T, int64_t N, int64_t V, int64_t ldx, int64_t ldw, int64_t ldy, int dtype,
                       nq_stream_t stream) {
    if (!x || !w || !w_scale || !y || !status_word) return NQ_ERR_NULL;
    if (dtype != NQ_F16 && dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if (T < 1 || N < 1 || V < 1 || ldx < 0 || ldw < N || ldw % 16 || ldy < V) return NQ_ERR_SHAPE;
    if (N > kInt8MaxCols || T > 0x1fffffff || V > 0x1fffffff) return NQ_ERR_TOO_LARGE;
    if (!aligned16(w) || !aligned16(w_scale) || !aligned16(scratch) || !aligned16(status_word) || !aligned_to(2, x, bias, y)) return NQ_ERR_ALIGN;
    const size_t need = nq_int8_linear_scratch_bytes(T, N);
    if (need && !scratch) return NQ_ERR_NULL;
    if (scratch_bytes < need) return NQ_ERR_SCRATCH;
    unsigned* status = static_cast<unsigned*>(status_word) + 2;
    auto run = dtype == NQ_BF16 ? int8_linear<kOutBf16> : int8_linear<kOutFp16>;
    return run(x, ldx, w, ldw, w_scale, bias, y, ldy, scratch, (int)T, (int)N, (int)V, status, as_stream(stream));
}

}  // extern "C"
