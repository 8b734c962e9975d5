// Queries and keys behind their projections: RMS norm of each head, rotation by the token's position, and keys and values into the paged cache.
//
//     x^ = x / sqrt(mean(x^2) + eps) w        (a, b) -> (a cos - b sin, b cos + a sin) scaling,   angle = p f_i
//
// Bound by memory: 2 bytes in and 2 out per element, everything read once.  A head belongs to a group of 4, 8 or 16 lanes with
// 16 elements each, so that a norm is a few shuffles; the two elements of a pair are in one lane (chunks of 8 that are R/2 apart, or neighbours).
// A CTA takes a range of tokens, eight at a time: their angles and places in the cache are computed once, by the CTA's threads side by side while their first
// heads are on the way, and shared by all heads; from then on every group has its next head under way while it works on one.
//
// Angles.  p f leaves the precision of fp32 for far positions (131072 x 1: an angle is known to 2^-7).  It is formed in 64 bits, where the product of a position
// below 2^29 and an fp32 frequency is exact, divided by 2 pi and reduced to half a turn there; cospi and sinpi take the rest in fp32.
#include "nq_attn.cuh"

namespace nq {

struct HeadsParams {
    nq_heads_desc d;
    int shift;               // log2(page_size)
    int group;               // lanes of a head
    int w32;
    int tokens;              // of a CTA
};
constexpr int kHeadsBatch = 8;        // tokens whose angles are in shared memory

enum : int { kHalves = 0, kNeighbours = 1, kHalvesAnywhere = 2 };      // pairs: R/2 apart (whole chunks of 8), neighbours, R/2 apart

template <bool BF16>
__device__ __forceinline__ void head_weights(const void* w, int w32, int c, float (&f)[8]) {
    if (w32) {
        const float4 a = static_cast<const float4*>(w)[c >> 2], b = static_cast<const float4*>(w)[(c >> 2) + 1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        const uint4 u = static_cast<const uint4*>(w)[c >> 3];
        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = head_float<BF16>(v[e >> 1], e & 1);
    }
}
template <bool BF16>
__device__ __forceinline__ float head_weight(const void* w, int w32, int c) {
    if (w32) return static_cast<const float*>(w)[c];
    return head_float<BF16>(static_cast<const uint16_t*>(w)[c], 0);
}

template <bool BF16, int PAIRS>
__global__ void __launch_bounds__(512) heads_kernel(const __grid_constant__ HeadsParams P) {
    extern __shared__ float4 all_turns[];             // of a token: (cos, sin) of two pairs each, pair 8 g + j at [j / 2][g]
    __shared__ long long place[kHeadsBatch];          // page and slot of a token (-1: nowhere; -2: padding)
    const nq_heads_desc& d = P.d;
    const int lanes = P.group, g = threadIdx.x & (lanes - 1), first = threadIdx.x / lanes, step = blockDim.x / lanes;
    const bool cached = d.k_cache != nullptr;
    const int chunks = d.D >> 3, half = d.R >> 4, heads = d.q_heads + d.k_heads * (cached ? 2 : 1);
    // this lane's two chunks of 8 elements
    int c0 = 2 * g, c1 = 2 * g + 1;
    if (PAIRS == kHalves) {
        c0 = g < half ? g : 2 * g;
        c1 = g < half ? g + half : 2 * g + 1;
    }
    const bool live0 = c0 < chunks, live1 = c1 < chunks;
    const int columns = (d.R / 2 + 7) / 8;            // of `turns`

    auto source = [&](long long t, int h) -> const uint16_t* {
        if (h < d.q_heads) return static_cast<const uint16_t*>(d.q) + t * d.q_token + (long long)h * d.q_head;
        if (h < d.q_heads + d.k_heads) return static_cast<const uint16_t*>(d.k) + t * d.k_token + (long long)(h - d.q_heads) * d.k_head;
        return static_cast<const uint16_t*>(d.v) + t * d.v_token + (long long)(h - d.q_heads - d.k_heads) * d.v_head;
    };
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const long long from = (long long)blockIdx.x * P.tokens, to = min(from + P.tokens, (long long)d.T);
    // a group's heads: those of the token, then those of the next
    auto forward = [&](long long& t, int& h) {
        h += step;
        while (h >= heads) { h -= heads; ++t; }
    };
    long long t = from, next_t;
    int h = first, next_h;
    while (h >= heads) { h -= heads; ++t; }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint4 r0 = zero, r1 = zero;
    if (t < to) {
        const uint16_t* p = source(t, h);
        if (live0) r0 = __ldcg(reinterpret_cast<const uint4*>(p) + c0);
        if (live1) r1 = __ldcg(reinterpret_cast<const uint4*>(p) + c1);
    }
    for (long long base = from; base < to; base += kHeadsBatch) {
      const int batch = (int)min((long long)kHeadsBatch, to - base);
      auto position = [&](long long at) -> long long {
          return d.position_bits == 64 ? __ldcg(static_cast<const long long*>(d.positions) + at) : __ldcg(static_cast<const int*>(d.positions) + at);
      };
      if (base > from) __syncthreads();               // (the angles before are not needed any more)
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
          float s, c;
          sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
          float2* at = reinterpret_cast<float2*>(all_turns + (b * 4 + ((k & 7) >> 1)) * columns + (k >> 3)) + (k & 1);
          *at = make_float2(c * d.scaling, s * d.scaling);
      }
      __syncthreads();

      for (; t < base + batch; t = next_t, h = next_h) {
        uint4 n0 = zero, n1 = zero;                   // the next head's, under way
        next_t = t;
        next_h = h;
        forward(next_t, next_h);
        if (next_t < to) {
            const uint16_t* p = source(next_t, next_h);
            if (live0) n0 = __ldcg(reinterpret_cast<const uint4*>(p) + c0);
            if (live1) n1 = __ldcg(reinterpret_cast<const uint4*>(p) + c1);
        }
        const float4* turns = all_turns + (int)(t - base) * 4 * columns;
        const long long where = cached ? place[t - base] : -1;
        const long long page = where >= 0 ? where >> P.shift : -1;
        const int slot = (int)(where & (d.page_size - 1));
        const bool is_q = h < d.q_heads, is_v = h >= d.q_heads + d.k_heads;
        uint16_t* out = nullptr;
        if (is_q) out = static_cast<uint16_t*>(d.q_out) + (t * d.q_heads + h) * d.D;
        else if (!cached) out = static_cast<uint16_t*>(d.k_out) + (t * d.k_heads + (h - d.q_heads)) * d.D;
        else if (page >= 0 && !is_v) out = static_cast<uint16_t*>(d.k_cache) + page * d.kc_page + slot * d.kc_slot + (h - d.q_heads) * d.kc_head;
        else if (page >= 0) out = static_cast<uint16_t*>(d.v_cache) + page * d.vc_page + slot * d.vc_slot + (h - d.q_heads - d.k_heads) * d.vc_head;
        if (!is_v) {
            const void* w = is_q ? d.q_weight : d.k_weight;
            const uint32_t raw[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
            float x[2][8];
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e >> 3][e & 7] = head_float<BF16>(raw[e >> 1], e & 1);
            float rstd = 1.f;
            if (w) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) sum = fmaf(x[e >> 3][e & 7], x[e >> 3][e & 7], sum);
                // (lanes of a group go through here together: a group has one head; the last ones' absent heads leave whole groups out)
                const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
                for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
                rstd = 1.f / sqrtf(sum / (float)d.D + d.eps);
                float f[8];
                if (live0) {
                    head_weights<BF16>(w, P.w32, 8 * c0, f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[0][e] = x[0][e] * rstd * f[e];
                }
                if (live1) {
                    head_weights<BF16>(w, P.w32, 8 * c1, f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[1][e] = x[1][e] * rstd * f[e];
                }
            }
            if constexpr (PAIRS == kHalves) {
                if (g < half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 u = turns[j * columns + g];
                        float a = x[0][2 * j], b = x[1][2 * j];
                        x[0][2 * j] = a * u.x - b * u.y;
                        x[1][2 * j] = b * u.x + a * u.y;
                        a = x[0][2 * j + 1], b = x[1][2 * j + 1];
                        x[0][2 * j + 1] = a * u.z - b * u.w;
                        x[1][2 * j + 1] = b * u.z + a * u.w;
                    }
                }
            } else if constexpr (PAIRS == kNeighbours) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (8 * g + 2 * j + k < d.R / 2) {
                            const float2 u = reinterpret_cast<const float2*>(turns + j * columns + g)[k];
                            float& ra = x[j >> 1][4 * (j & 1) + 2 * k];
                            float& rb = x[j >> 1][4 * (j & 1) + 2 * k + 1];
                            const float a = ra, b = rb;
                            ra = a * u.x - b * u.y;
                            rb = b * u.x + a * u.y;
                        }
                    }
                }
            } else {
                // an element's partner lies anywhere in the head: read again, from L1 or L2
                const uint16_t* p = source(t, h);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int c = 16 * g + e, i = c < d.R / 2 ? c : c - d.R / 2;
                    if (c < d.R) {
                        const int other = c < d.R / 2 ? c + d.R / 2 : i;
                        float b = head_float<BF16>(__ldcg(p + other), 0);
                        if (w) b = b * rstd * head_weight<BF16>(w, P.w32, other);
                        const float2 u = reinterpret_cast<const float2*>(turns + ((i & 7) >> 1) * columns + (i >> 3))[i & 1];
                        const float a = x[e >> 3][e & 7];
                        x[e >> 3][e & 7] = c < d.R / 2 ? a * u.x - b * u.y : a * u.x + b * u.y;
                    }
                }
            }
            const bool padding = where == -2;
            r0 = padding ? zero : make_uint4(head_pack<BF16>(x[0][0], x[0][1]), head_pack<BF16>(x[0][2], x[0][3]), head_pack<BF16>(x[0][4], x[0][5]), head_pack<BF16>(x[0][6], x[0][7]));
            r1 = padding ? zero : make_uint4(head_pack<BF16>(x[1][0], x[1][1]), head_pack<BF16>(x[1][2], x[1][3]), head_pack<BF16>(x[1][4], x[1][5]), head_pack<BF16>(x[1][6], x[1][7]));
        }
        if (out && live0) reinterpret_cast<uint4*>(out)[c0] = r0;
        if (out && live1) reinterpret_cast<uint4*>(out)[c1] = r1;
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
    if (d.D > kHeadMaxCols || d.q_heads > 1 << 16 || d.k_heads > 1 << 16 || d.T > 0x7fffffff) return NQ_ERR_TOO_LARGE;
    if (cached && (d.seqs <= 0 || d.max_pages <= 0 || d.pages <= 0 || !page_size_ok(d.page_size) || d.table_stride < 0 ||
                   !multiple_of_8({d.kc_page, d.kc_slot, d.kc_head, d.vc_page, d.vc_slot, d.vc_head})))
        return NQ_ERR_SHAPE;
    if (!aligned_to(16, (const char*)d.q, (const char*)d.k, (const char*)d.v, (const char*)d.q_out, (const char*)d.k_out, (const char*)d.k_cache, (const char*)d.v_cache,
                    (const char*)d.q_weight, (const char*)d.k_weight) ||
        !aligned_to(4, (const char*)d.inv_freq, (const char*)d.sequences, (const char*)d.block_table) || !aligned_to((unsigned)d.position_bits / 8, (const char*)d.positions))
        return NQ_ERR_ALIGN;
    HeadsParams P{d, log2_of(cached ? d.page_size : 8), 1, d.weight_dtype == NQ_F32, 1};
    while (16 * P.group < d.D) P.group *= 2;
    const int heads = d.q_heads + d.k_heads * (cached ? 2 : 1);
    const int64_t lanes = (int64_t)heads * P.group;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((unsigned)(lanes >= 512 ? 512 : (lanes + 31) / 32 * 32));
    // as many CTAs as fit the SMs at once, a token each at least
    const int64_t most = (int64_t)sm_count() * (1024 / cfg.blockDim.x > 16 ? 16 : 1024 / cfg.blockDim.x);
    P.tokens = (int)((d.T + most - 1) / most);
    cfg.gridDim = dim3((unsigned)((d.T + P.tokens - 1) / P.tokens));
    cfg.dynamicSmemBytes = (size_t)4 * kHeadsBatch * ((d.R / 2 + 7) / 8) * sizeof(float4);
    cfg.stream = as_stream(stream);
    const int pairs = d.interleaved ? kNeighbours : d.R % 16 == 0 ? kHalves : kHalvesAnywhere;
    const void* fn[2][3] = {{(const void*)heads_kernel<false, kHalves>, (const void*)heads_kernel<false, kNeighbours>, (const void*)heads_kernel<false, kHalvesAnywhere>},
                            {(const void*)heads_kernel<true, kHalves>, (const void*)heads_kernel<true, kNeighbours>, (const void*)heads_kernel<true, kHalvesAnywhere>}};
    cudaLaunchAttribute attr[1];
    void* args[] = {&P};
    return launch_dependent(cfg, attr, 0, fn[d.dtype == NQ_BF16][pairs], args);
}

}  // extern "C"
