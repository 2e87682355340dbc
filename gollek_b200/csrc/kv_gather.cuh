// kv_gather.cuh -- rows of the paged cache read back, dequantised, as contiguous keys and
// values (the inverse of kv_append.cuh).
//
// out[t, h, d] = pool[page(t), h, slot(t), d] * scale(page, h, slot), rounded once to the
// output type; page(t) = table[seq(t)][pos(t) / BS], slot(t) = pos(t) % BS.  Nothing is
// reused, so the pass is bound by HBM: its bytes are the rows read and the rows written.
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

}  // namespace gk
