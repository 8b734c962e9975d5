// Queries and keys behind their projections: RMS norm of each head, rotation by the token's position, and keys and values into the paged cache.
//
//     x^ = x / sqrt(mean(x^2) + eps) w        (a, b) -> (a cos - b sin, b cos + a sin) scaling,   angle = p f_i
//
// Bound by memory: 2 bytes in and 2 out per element, everything read once.  A head belongs to a group of 4, 8 or 16 lanes with
// 16 elements each, so that a norm is a few shuffles; the two elements of a pair are in one lane (chunks of 8 that are R/2 apart, or neighbours).
// A CTA takes a range of tokens and a group the same head of each: its addresses move by a stride (407 instructions per 16
// elements a lane with heads in turn, which bound the kernel; packed fp32 pairs for the same reason).  The angles and places in the cache of eight tokens are computed
// at a time, by the CTA's threads side by side, and shared by all heads; a group has its next head under way while it works on one.
//
// Angles.  p f leaves the precision of fp32 for far positions (131072 x 1: an angle is known to 2^-7).  It is formed in 64 bits, where the product of a position
// below 2^29 and an fp32 frequency is exact, divided by 2 pi and reduced to half a turn there; cospi and sinpi take the rest in fp32.
#include <type_traits>

#include "nq_attn.cuh"

namespace nq {

struct HeadsParams {
    nq_heads_desc d;
    int shift;               // log2(page_size)
    int group;               // lanes of a head
    int w32;
    int tokens, heads;       // of a CTA
};
constexpr int kHeadsBatch = 8;        // tokens whose angles are in shared memory

enum : int { kHalves = 0, kNeighbours = 1, kHalvesAnywhere = 2 };      // pairs: R/2 apart (whole chunks of 8), neighbours, R/2 apart

template <bool BF16>
__device__ __forceinline__ float head_weight(const void* w, int w32, int c) {
    if (w32) return static_cast<const float*>(w)[c];
    return head_float<BF16>(static_cast<const uint16_t*>(w)[c], 0);
}

template <bool BF16, int PAIRS, bool cached>
__global__ void __launch_bounds__(512, 2) heads_kernel(const __grid_constant__ HeadsParams P) {
    extern __shared__ float4 all_turns[];             // of a token: (cos, cos, sin, sin) of two pairs each, pair 8 g + j at [j / 2][g]
    __shared__ long long place[kHeadsBatch];          // page and slot of a token (-1: nowhere; -2: padding)
    __shared__ ulonglong2 weights[2][4][16];          // of queries and of keys: four elements each, lane g's at [.][g]
    const nq_heads_desc& d = P.d;
    const int lanes = P.group, g = threadIdx.x & (lanes - 1), h = blockIdx.y * P.heads + threadIdx.x / lanes;
    const int chunks = d.D >> 3, half = d.R >> 4, heads = d.q_heads + d.k_heads * (cached ? 2 : 1);
    const bool mine = (int)threadIdx.x < P.heads * lanes && h < heads;
    // this lane's two chunks of 8 elements
    int c0 = 2 * g, c1 = 2 * g + 1;
    if (PAIRS == kHalves) {
        c0 = g < half ? g : 2 * g;
        c1 = g < half ? g + half : 2 * g + 1;
    }
    const bool live0 = mine && c0 < chunks, live1 = mine && c1 < chunks;
    const int columns = (d.R / 2 + 7) / 8;            // of `turns`
    const bool is_q = h < d.q_heads, is_v = h >= d.q_heads + d.k_heads;
    const long long from = (long long)blockIdx.x * P.tokens, to = min(from + P.tokens, (long long)d.T);

    // the head's first token in and (where it does not go to the cache) out; how far the next one is
    const uint16_t* src;
    uint16_t* dst;
    int src_step, dst_step = 0;
    if (is_q) {
        src_step = (int)d.q_token;
        src = static_cast<const uint16_t*>(d.q) + (long long)h * d.q_head;
        dst_step = d.q_heads * d.D;
        dst = static_cast<uint16_t*>(d.q_out) + (long long)h * d.D;
    } else if (!is_v) {
        const int k = h - d.q_heads;
        src_step = (int)d.k_token;
        src = static_cast<const uint16_t*>(d.k) + (long long)k * d.k_head;
        if (!cached) dst_step = d.k_heads * d.D;
        dst = cached ? static_cast<uint16_t*>(d.k_cache) + k * d.kc_head : static_cast<uint16_t*>(d.k_out) + (long long)k * d.D;
    } else {
        const int k = h - d.q_heads - d.k_heads;
        src_step = (int)d.v_token;
        src = static_cast<const uint16_t*>(d.v) + (long long)k * d.v_head;
        dst = static_cast<uint16_t*>(d.v_cache) + k * d.vc_head;
    }
    src += from * src_step;
    dst += from * dst_step;
    const bool to_cache = cached && !is_q;
    auto fetch = [&](const uint16_t* p, bool more, uint4& a, uint4& b) {
        a = b = make_uint4(0, 0, 0, 0);
        if (live0 && more) a = __ldcg(reinterpret_cast<const uint4*>(p) + c0);
        if (live1 && more) b = __ldcg(reinterpret_cast<const uint4*>(p) + c1);
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint4 r0, r1;                                     // of this token
    fetch(src, from < to, r0, r1);
    // (in shared memory for the registers' sake: with 64 of them three CTAs of 320 threads share an SM)
    const bool normed = is_q ? d.q_weight != nullptr : !is_v && d.k_weight != nullptr;
    if (threadIdx.x < 2 * lanes) {
        const int kind = (int)threadIdx.x >= lanes;
        const void* w = kind ? d.k_weight : d.q_weight;
        if (w) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int chunk = e < 4 ? c0 : c1, c = 8 * chunk + 2 * (e & 3);
                const uint64_t v = chunk < chunks ? pair_of(head_weight<BF16>(w, P.w32, c), head_weight<BF16>(w, P.w32, c + 1)) : 0;
                (e & 1 ? weights[kind][e >> 1][g].y : weights[kind][e >> 1][g].x) = v;
            }
        }
    }
    const float inv_d = 1.f / (float)d.D;
    const unsigned group_mask = ((1u << (lanes - 1)) * 2u - 1u) << (threadIdx.x & 31 & ~(lanes - 1));

    for (long long base = from; base < to; base += kHeadsBatch) {
        const int batch = (int)min((long long)kHeadsBatch, to - base);
        auto position = [&](long long at) -> long long {
            return d.position_bits == 64 ? __ldcg(static_cast<const long long*>(d.positions) + at) : __ldcg(static_cast<const int*>(d.positions) + at);
        };
        if (base > from) __syncthreads();             // (the angles before are not needed any more)
        if (cached && (int)threadIdx.x < batch) {
            const long long at = base + threadIdx.x, pos = position(at);
            long long page = -1;
            if (pos >= 0) {
                const long long seq = d.sequences ? __ldcg(d.sequences + at) : at, n = pos >> P.shift;
                if (seq >= 0 && seq < d.seqs && n < d.max_pages) page = __ldcg(d.block_table + seq * d.table_stride + n);
                if (page >= d.pages) page = -1;
            }
            place[threadIdx.x] = pos < 0 ? -2 : page < 0 ? -1 : page << P.shift | (pos & (d.page_size - 1));
        }
        for (int i = threadIdx.x; i < batch * (d.R / 2); i += blockDim.x) {
            const int b = i / (d.R / 2), k = i - b * (d.R / 2);
            const double turn = (double)position(base + b) * (double)d.inv_freq[k] * 0.15915494309189533577;      // 1 / (2 pi)
            float sn, cs;
            sincospif(2.f * (float)(turn - rint(turn)), &sn, &cs);
            float* at = reinterpret_cast<float*>(all_turns + (b * 4 + ((k & 7) >> 1)) * columns + (k >> 3)) + (k & 1);
            at[0] = cs * d.scaling;
            at[2] = sn * d.scaling;
        }
        __syncthreads();
        if (!mine) continue;

        for (int b = 0; b < batch; ++b) {
            uint4 n0, n1;                             // of the next one, under way
            fetch(src + src_step, base + b + 1 < to, n0, n1);
            const float4* turns = all_turns + b * 4 * columns;
            const long long where = cached ? place[b] : 0;
            if (!is_v) {
                const uint32_t raw[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
                uint64_t x[8];                        // (two elements each)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = pair_of(head_float<BF16>(raw[e], 0), head_float<BF16>(raw[e], 1));
                float rstd = 1.f;
                if (normed) {
                    uint64_t sum2 = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum2 = pair_fma(x[e], x[e], sum2);
                    float lo, hi;
                    pair_split(sum2, lo, hi);
                    float sum = lo + hi;
                    for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(group_mask, sum, o);
                    rstd = rsqrtf(fmaf(sum, inv_d, d.eps));
                    const uint64_t r2 = pair_of(rstd, rstd);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const ulonglong2 f = weights[is_q ? 0 : 1][e][g];
                        x[2 * e] = pair_mul(pair_mul(x[2 * e], r2), f.x);
                        x[2 * e + 1] = pair_mul(pair_mul(x[2 * e + 1], r2), f.y);
                    }
                }
                if constexpr (PAIRS == kHalves) {
                    if (g < half) {
                        const uint64_t minus = pair_of(-1.f, -1.f);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float4 u = turns[j * columns + g];
                            const uint64_t cs = pair_of(u.x, u.y), sn = pair_of(u.z, u.w), a = x[j], c = x[4 + j];
                            x[j] = pair_fma(pair_mul(c, sn), minus, pair_mul(a, cs));
                            x[4 + j] = pair_fma(a, sn, pair_mul(c, cs));
                        }
                    }
                } else if constexpr (PAIRS == kNeighbours) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (8 * g + 2 * j < d.R / 2) {
                            const float4 u = turns[j * columns + g];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                float a, c;
                                pair_split(x[2 * j + k], a, c);
                                const float cs = k ? u.y : u.x, sn = k ? u.w : u.z;
                                if (8 * g + 2 * j + k < d.R / 2) x[2 * j + k] = pair_of(a * cs - c * sn, c * cs + a * sn);
                            }
                        }
                    }
                } else {
                    // an element's partner lies anywhere in the head: read again, from L1 or L2
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float y[2];
                        pair_split(x[e], y[0], y[1]);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int c = 16 * g + 2 * e + k;
                            if (c < d.R) {
                                const int i = c < d.R / 2 ? c : c - d.R / 2, other = c < d.R / 2 ? c + d.R / 2 : i;
                                float v = head_float<BF16>(__ldcg(src + other), 0);
                                if (normed) v = v * rstd * head_weight<BF16>(is_q ? d.q_weight : d.k_weight, P.w32, other);
                                const float* u = reinterpret_cast<const float*>(turns + ((i & 7) >> 1) * columns + (i >> 3)) + (i & 1);
                                y[k] = c < d.R / 2 ? y[k] * u[0] - v * u[2] : y[k] * u[0] + v * u[2];
                            }
                        }
                        x[e] = pair_of(y[0], y[1]);
                    }
                }
                uint32_t packed[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float lo, hi;
                    pair_split(x[e], lo, hi);
                    packed[e] = where == -2 ? 0u : head_pack<BF16>(lo, hi);
                }
                r0 = make_uint4(packed[0], packed[1], packed[2], packed[3]);
                r1 = make_uint4(packed[4], packed[5], packed[6], packed[7]);
            }
            uint16_t* out = dst;
            if (to_cache) out += (where >> P.shift) * (is_v ? d.vc_page : d.kc_page) + ((int)where & (d.page_size - 1)) * (is_v ? d.vc_slot : d.kc_slot);
            if (!to_cache || where >= 0) {
                if (live0) reinterpret_cast<uint4*>(out)[c0] = r0;
                if (live1) reinterpret_cast<uint4*>(out)[c1] = r1;
            }
            if (!to_cache) dst += dst_step;
            src += src_step;
            r0 = n0;
            r1 = n1;
        }
    }
}

}  // namespace nq

extern "C" {

int nq_head_max_columns(void) { return nq::kHeadMaxCols; }

int nq_heads_fwd(const nq_heads_desc* desc, nq_stream_t stream) {
    using namespace nq;
    if (!desc) return NQ_ERR_NULL;
    const nq_heads_desc& d = *desc;
    const bool cached = d.k_cache || d.v_cache;
    if (!d.positions || (d.q_heads > 0 && (!d.q || !d.q_out)) || (d.k_heads > 0 && !d.k) || (d.R > 0 && !d.inv_freq)) return NQ_ERR_NULL;
    if (cached ? !d.k_cache || !d.v_cache || !d.v || !d.block_table : d.k_heads > 0 && !d.k_out) return NQ_ERR_NULL;
    if (d.dtype != NQ_F16 && d.dtype != NQ_BF16) return NQ_ERR_DTYPE;
    if ((d.weight_dtype != d.dtype && d.weight_dtype != NQ_F32) || (d.position_bits != 32 && d.position_bits != 64)) return NQ_ERR_DTYPE;
    if (d.T <= 0 || d.q_heads < 0 || d.k_heads < 0 || d.q_heads + d.k_heads <= 0 || (cached && d.k_heads <= 0) || d.D <= 0 || d.D % 8 != 0 || d.R < 0 || d.R > d.D ||
        d.R % 2 != 0)
        return NQ_ERR_SHAPE;
    if (!multiple_of_8({d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head})) return NQ_ERR_SHAPE;
    if (d.D > kHeadMaxCols || d.q_heads > 1 << 16 || d.k_heads > 1 << 16 || d.T > 0x7fffffff || d.q_token > 0x7fffffff || d.k_token > 0x7fffffff || d.v_token > 0x7fffffff)
        return NQ_ERR_TOO_LARGE;
    if (cached && (d.seqs <= 0 || d.max_pages <= 0 || d.pages <= 0 || !page_size_ok(d.page_size) || d.table_stride < 0 ||
                   !multiple_of_8({d.kc_page, d.kc_slot, d.kc_head, d.vc_page, d.vc_slot, d.vc_head})))
        return NQ_ERR_SHAPE;
    if (!aligned_to(16, (const char*)d.q, (const char*)d.k, (const char*)d.v, (const char*)d.q_out, (const char*)d.k_out, (const char*)d.k_cache, (const char*)d.v_cache,
                    (const char*)d.q_weight, (const char*)d.k_weight) ||
        !aligned_to(4, (const char*)d.inv_freq, (const char*)d.sequences, (const char*)d.block_table) || !aligned_to((unsigned)d.position_bits / 8, (const char*)d.positions))
        return NQ_ERR_ALIGN;
    HeadsParams P{d, log2_of(cached ? d.page_size : 8), 1, d.weight_dtype == NQ_F32, 1, 1};
    while (16 * P.group < d.D) P.group *= 2;
    const int heads = d.q_heads + d.k_heads * (cached ? 2 : 1), parts = (heads * P.group + 511) / 512;
    P.heads = (heads + parts - 1) / parts;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((unsigned)((P.heads * P.group + 31) / 32 * 32));
    // as many CTAs as fit the SMs at once, a token each at least
    const int at_once = 1024 / (int)cfg.blockDim.x > 16 ? 16 : 1024 / (int)cfg.blockDim.x;
    const int64_t most = (int64_t)sm_count() * at_once / parts > 0 ? (int64_t)sm_count() * at_once / parts : 1;
    P.tokens = (int)((d.T + most - 1) / most);
    cfg.gridDim = dim3((unsigned)((d.T + P.tokens - 1) / P.tokens), (unsigned)((heads + P.heads - 1) / P.heads));
    cfg.dynamicSmemBytes = (size_t)4 * kHeadsBatch * ((d.R / 2 + 7) / 8) * sizeof(float4);
    cfg.stream = as_stream(stream);
    const int pairs = d.interleaved ? kNeighbours : d.R % 16 == 0 ? kHalves : kHalvesAnywhere;
    static const auto pick = [](auto bf, auto in_cache, int pairs) -> const void* {
        constexpr bool kBf = decltype(bf)::value, kIn = decltype(in_cache)::value;
        return pairs == kNeighbours ? (const void*)heads_kernel<kBf, kNeighbours, kIn> : pairs == kHalves ? (const void*)heads_kernel<kBf, kHalves, kIn>
                                                                                                        : (const void*)heads_kernel<kBf, kHalvesAnywhere, kIn>;
    };
    const std::true_type yes;
    const std::false_type no;
    const void* fn = d.dtype == NQ_BF16 ? (cached ? pick(yes, yes, pairs) : pick(yes, no, pairs)) : (cached ? pick(no, yes, pairs) : pick(no, no, pairs));
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    return launch_dependent(cfg, attr, 0, fn, args);
}

}  // extern "C"
