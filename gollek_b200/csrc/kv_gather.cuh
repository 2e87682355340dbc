// kv_gather.cuh -- rows of the paged cache read back, dequantised, as contiguous keys and
// values (the inverse of kv_append.cuh).
//
// out[t, h, d] = pool[page(t), h, slot(t), d] * scale(page, h, slot), rounded once to the
// output type; page(t) = table[seq(t)][pos(t) / BS], slot(t) = pos(t) % BS.  Nothing is
// reused, so the pass is bound by HBM: its bytes are the rows read and the rows written.
// 32 sequences of 512 to 8192 int8 rows (8 heads of 128) to bf16: 159 us, 0.89 of the rate of
// a plain copy.
#pragma once

#include "common.cuh"

namespace gk {

struct GatherArgs {
    void *key;
    void *value;
    const void *k;
    const void *v;
    const float *k_scales;
    const float *v_scales;
    const int *token_seq;
    const int *token_pos;
    const int *block_tables;
    long long page_stride, scale_page_stride, scale_head_stride, scale_token_stride;
    int num_tokens, num_seqs, num_kv_heads, head_dim, block_size, max_blocks, num_blocks, kv_dtype, out_dtype;
};

// Pool and scale element index of token t's row of head h; false (and a status bit, raised
// by the threads with `tell`) where the position or page is not usable.
__device__ __forceinline__ bool gather_row(const GatherArgs &a, int t, int h, bool tell, long long &e0, long long &so) {
    const int seq = a.token_seq ? a.token_seq[t] : t;
    const int pos = a.token_pos[t];
    if (pos < 0 || pos >= a.max_blocks * a.block_size || seq < 0 || seq >= a.num_seqs) {
        if (tell) raise_status(GOLLEK_STATUS_BAD_POSITION);
        return false;
    }
    const int page = a.block_tables[static_cast<long long>(seq) * a.max_blocks + pos / a.block_size];
    if (page < 0 || (a.num_blocks > 0 && page >= a.num_blocks)) {
        if (tell) raise_status(GOLLEK_STATUS_BAD_BLOCK_ID);
        return false;
    }
    const int slot = pos % a.block_size;
    e0 = static_cast<long long>(page) * a.page_stride + (static_cast<long long>(h) * a.block_size + slot) * a.head_dim;
    so = static_cast<long long>(page) * a.scale_page_stride + static_cast<long long>(h) * a.scale_head_stride +
         static_cast<long long>(slot) * a.scale_token_stride;
    return true;
}

// Any shape: one thread per element.
__global__ void __launch_bounds__(256) kv_gather_generic_kernel(const GatherArgs a) {
    const long long total = static_cast<long long>(a.num_tokens) * a.num_kv_heads * a.head_dim;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
        const long long row = i / a.head_dim;
        const int d = static_cast<int>(i - row * a.head_dim);
        const int t = static_cast<int>(row / a.num_kv_heads);
        const int h = static_cast<int>(row - static_cast<long long>(t) * a.num_kv_heads);
        long long e0, so;
        float x = 0.f, y = 0.f;
        if (gather_row(a, t, h, d == 0, e0, so)) {
            x = load_kv(a.k, a.kv_dtype, e0 + d);
            y = load_kv(a.v, a.kv_dtype, e0 + d);
            if (a.k_scales) {
                x *= a.k_scales[so];
                y *= a.v_scales[so];
            }
        }
        if (a.out_dtype == GOLLEK_DTYPE_F32) {
            reinterpret_cast<float *>(a.key)[i] = x;
            reinterpret_cast<float *>(a.value)[i] = y;
        } else if (a.out_dtype == GOLLEK_DTYPE_BF16) {
            reinterpret_cast<__nv_bfloat16 *>(a.key)[i] = __float2bfloat16_rn(x);
            reinterpret_cast<__nv_bfloat16 *>(a.value)[i] = __float2bfloat16_rn(y);
        } else {
            reinterpret_cast<__half *>(a.key)[i] = __float2half_rn(x);
            reinterpret_cast<__half *>(a.value)[i] = __float2half_rn(y);
        }
    }
}

// Eight elements of the pool as fp32.
template <int KV>
__device__ __forceinline__ void load8(const void *base, long long e, uint4 (&raw)[2]) {
    if constexpr (KV == GOLLEK_DTYPE_F32) {
        const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(base) + e);
        raw[0] = __ldcs(p);
        raw[1] = __ldcs(p + 1);
    } else if constexpr (KV == GOLLEK_DTYPE_BF16 || KV == GOLLEK_DTYPE_F16) {
        raw[0] = __ldcs(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(base) + e));
    } else if constexpr (KV == GOLLEK_DTYPE_I8) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(reinterpret_cast<const int8_t *>(base) + e));
        raw[0].x = w.x;
        raw[0].y = w.y;
    } else {
        raw[0].x = __ldcs(reinterpret_cast<const unsigned *>(reinterpret_cast<const uint8_t *>(base) + (e >> 1)));
    }
}

template <int KV>
__device__ __forceinline__ void widen8(const uint4 (&raw)[2], float scale, float (&x)[8]) {
    if constexpr (KV == GOLLEK_DTYPE_F32) {
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else if constexpr (KV == GOLLEK_DTYPE_BF16 || KV == GOLLEK_DTYPE_F16) {
        using T = std::conditional_t<KV == GOLLEK_DTYPE_BF16, __nv_bfloat16, __half>;
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else if constexpr (KV == GOLLEK_DTYPE_I8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw[0].x : raw[0].y) >> (8 * (i & 3)))) * scale;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int>((raw[0].x >> (4 * i)) & 15) - 8) * scale;
    }
}

template <typename OUT>
__device__ __forceinline__ void store8(void *base, long long e, const float (&x)[8]) {
    if constexpr (std::is_same<OUT, float>::value) {
        float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(base) + e);
        __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        __stcs(reinterpret_cast<uint4 *>(reinterpret_cast<OUT *>(base) + e),
               make_uint4(pack2<OUT>(x[0], x[1]), pack2<OUT>(x[2], x[3]), pack2<OUT>(x[4], x[5]), pack2<OUT>(x[6], x[7])));
    }
}

constexpr int kGatherThreads = 256;
constexpr int kGatherTokens = 32;  // tokens per block at most
constexpr int kGatherUnroll = 2;   // chunks (of K and of V) a thread has in flight

// Rows of whole 8-element chunks with aligned pools (host: gather_vectors).  A block takes
// `tpb` consecutive tokens: one thread per token follows sequence -> page (three dependent
// loads) into shared memory, then all threads copy the tokens' chunks, K and V of
// kGatherUnroll chunks in flight each; the lookups of one block run under the copies of the
// SM's others.
template <int KV, typename OUT>
__global__ void __launch_bounds__(kGatherThreads) kv_gather_kernel(const GatherArgs a, const int tpb) {
    constexpr bool QUANT = KV == GOLLEK_DTYPE_I8 || KV == GOLLEK_DTYPE_I4;
    __shared__ long long sm_e[kGatherTokens], sm_s[kGatherTokens];
    const long long t0 = static_cast<long long>(blockIdx.x) * tpb;
    const int nt = static_cast<int>(min(static_cast<long long>(tpb), a.num_tokens - t0));
    if (threadIdx.x < nt) {
        long long e0 = -1, so = 0;
        if (!gather_row(a, static_cast<int>(t0) + threadIdx.x, 0, true, e0, so)) e0 = -1;
        sm_e[threadIdx.x] = e0;
        sm_s[threadIdx.x] = so;
    }
    __syncthreads();
    const unsigned cpr = a.head_dim / 8, cpt = cpr * a.num_kv_heads;
    const unsigned total = nt * cpt;
    const long long hstride = static_cast<long long>(a.block_size) * a.head_dim;
    for (unsigned i0 = threadIdx.x; i0 < total; i0 += kGatherUnroll * kGatherThreads) {
        uint4 rk[kGatherUnroll][2], rv[kGatherUnroll][2];
        float ks[kGatherUnroll], vs[kGatherUnroll];
        bool live[kGatherUnroll];
#pragma unroll
        for (int u = 0; u < kGatherUnroll; ++u) {
            const unsigned i = i0 + u * kGatherThreads;
            live[u] = false;
            ks[u] = vs[u] = 1.f;
            if (i >= total) continue;
            const unsigned t = i / cpt, rem = i - t * cpt;
            const unsigned h = rem / cpr, c = rem - h * cpr;
            if (sm_e[t] < 0) continue;
            live[u] = true;
            const long long e = sm_e[t] + h * hstride + 8 * c;
            load8<KV>(a.k, e, rk[u]);
            load8<KV>(a.v, e, rv[u]);
            if constexpr (QUANT) {
                const long long so = sm_s[t] + static_cast<long long>(h) * a.scale_head_stride;
                ks[u] = __ldg(a.k_scales + so);
                vs[u] = __ldg(a.v_scales + so);
            }
        }
#pragma unroll
        for (int u = 0; u < kGatherUnroll; ++u) {
            const unsigned i = i0 + u * kGatherThreads;
            if (i >= total) continue;
            float x[8], y[8];
            if (live[u]) {
                widen8<KV>(rk[u], ks[u], x);
                widen8<KV>(rv[u], vs[u], y);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
            }
            const long long o = (t0 * cpt + i) * 8;  // [token][head][dim]: the order of the chunks
            store8<OUT>(a.key, o, x);
            store8<OUT>(a.value, o, y);
        }
    }
}

}  // namespace gk
