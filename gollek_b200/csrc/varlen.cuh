// varlen.cuh -- what the kernels of ragged and shared-prefix paged attention have in common
// (the argument block, sequences and row masks), and the generic kernel that computes
// either for every shape and type the ABI accepts.
//
// Row i of sequence s (query token cu[s] + i; decode: one row) attends an interval of
// positions, [lo, hi):
//   pos = len - n + i                          n: the sequence's query tokens
//   hi  = causal ? max(pos + 1, min(prefix_len, len)) : len
//   lo  = max(0, pos - window + 1 (window > 0), token_start)
//   x_j = cap(scale q.k_j) - slope |pos - j|,  cap(y) = soft_cap tanh(y / soft_cap)
//   out = sum_j e^{x_j} v_j / sum_j e^{x_j};   0 where [lo, hi) is empty
// With shared prefixes the row of sequence s also attends every position of its group's
// prefix, read through the group's own table.
#pragma once

#include "common.cuh"

namespace gk {

struct AttnArgs {
    void *out;
    const void *q;
    const void *k;
    const void *v;
    const float *k_scales;
    const float *v_scales;
    const int *block_tables;   // [num_seqs][max_blocks]
    const int *context_lens;   // [num_seqs]
    const int *cu;             // [num_seqs + 1] first query token of each sequence; null: token s
    const float *slopes;       // [num_q_heads] distance bias, or null
    const int *prefix_lens;    // varlen: [num_seqs] bidirectional prefix, or null
    const int *token_starts;   // varlen: [total_q] first visible position, or null
    const int *prefix_tables;  // shared: [num_groups][max_pblocks]
    const int *group_plens;    // shared: [num_groups]
    const int *group_starts;   // shared: [num_groups + 1]
    long long page_stride;     // elements (nibbles for int4)
    long long scale_page_stride, scale_head_stride, scale_token_stride;
    int num_seqs, total_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, num_blocks;
    int num_groups, max_pblocks;
    int causal, window, q_dtype, kv_dtype;
    float q_scale;     // scale * log2(e); scale with a soft-cap
    float soft_cap;    // <= 0: none
};

__device__ __forceinline__ float load_elem(const void *p, int dtype, long long i) {
    if (dtype == GOLLEK_DTYPE_F32) return reinterpret_cast<const float *>(p)[i];
    if (dtype == GOLLEK_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(reinterpret_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ void store_elem(void *p, int dtype, long long i, float v) {
    if (dtype == GOLLEK_DTYPE_F32)
        reinterpret_cast<float *>(p)[i] = v;
    else if (dtype == GOLLEK_DTYPE_BF16)
        reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else
        reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
}

// Tokens of a table with `blocks` columns that a length may name; outside it is clamped.
__device__ __forceinline__ int clamp_len(const AttnArgs &a, int len, int blocks) {
    return min(max(len, 0), blocks * a.block_size);
}

// Query tokens [q0, q0 + n) of sequence s; n = 0 where cu is not usable there.
__device__ __forceinline__ void seq_rows(const AttnArgs &a, int s, int &q0, int &n) {
    if (!a.cu) {
        q0 = s;
        n = 1;
        return;
    }
    q0 = a.cu[s];
    const int q1 = a.cu[s + 1];
    n = (q0 >= 0 && q1 >= q0 && q1 <= a.total_q) ? q1 - q0 : 0;
}

// Sequences of group g, clipped to the batch; empty where group_starts is not usable there.
__device__ __forceinline__ void group_rows_of(const AttnArgs &a, int g, int &s0, int &n) {
    s0 = a.group_starts[g];
    const int s1 = a.group_starts[g + 1];
    n = (s0 >= 0 && s1 >= s0 && s1 <= a.num_seqs) ? s1 - s0 : 0;
}

// Raises BAD_POSITION for sequence s's (group g's) sizes outside their tables; called once
// per sequence and group and call.
__device__ __forceinline__ void check_seq(const AttnArgs &a, int s) {
    const int len = a.context_lens[s];
    bool bad = len < 0 || len > a.max_blocks * a.block_size;
    if (a.cu) {
        const int q0 = a.cu[s], q1 = a.cu[s + 1];
        bad = bad || q0 < 0 || q1 < q0 || q1 > a.total_q;
    }
    if (bad) raise_status(GOLLEK_STATUS_BAD_POSITION);
}
__device__ __forceinline__ void check_group(const AttnArgs &a, int g) {
    const int len = a.group_plens[g], s0 = a.group_starts[g], s1 = a.group_starts[g + 1];
    if (len < 0 || len > a.max_pblocks * a.block_size || s0 < 0 || s1 < s0 || s1 > a.num_seqs)
        raise_status(GOLLEK_STATUS_BAD_POSITION);
}

// The sequence that query token t belongs to, or -1 (before the first, behind the last).
__device__ __forceinline__ int seq_of_token(const AttnArgs &a, int t, int &q0, int &n) {
    if (!a.cu) {
        q0 = t;
        n = 1;
        return t;
    }
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {  // last s with cu[s] <= t
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    seq_rows(a, lo, q0, n);
    return (t >= q0 && t - q0 < n) ? lo : -1;
}

// The group that sequence s belongs to, or -1.
__device__ __forceinline__ int group_of_seq(const AttnArgs &a, int s) {
    int lo = 0, hi = a.num_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.group_starts[mid] <= s)
            lo = mid;
        else
            hi = mid - 1;
    }
    int s0, n;
    group_rows_of(a, lo, s0, n);
    return (s >= s0 && s - s0 < n) ? lo : -1;
}

// Positions [lo, hi) that query token t, at position pos of sequence s (length len), attends; [0, 0)
// where there are none, so that a caller's token_starts never enters a sum of positions.
__device__ __forceinline__ void row_range(const AttnArgs &a, int s, int t, int pos, int len, int &lo, int &hi) {
    hi = len;
    if (a.causal) {
        hi = pos + 1;
        if (a.prefix_lens) hi = max(hi, min(a.prefix_lens[s], len));
    }
    lo = 0;
    if (a.window > 0) lo = max(lo, pos - a.window + 1);
    if (a.token_starts) lo = max(lo, a.token_starts[t]);
    if (lo >= hi) lo = hi = 0;
}

// ------------------------------------------------------------------ generic kernel

constexpr int kAgWarps = 8;
constexpr int kAgTok = 4;  // tokens a warp has in flight

// One CTA per (query token, kv head, chunk of GC q heads).  Warp w takes the tokens
// kAgTok w .. of every kAgWarps * kAgTok visible ones; lane l owns head-dim columns l,
// l + 32, ... (J of them).  Online softmax per warp, all sums in fp32, states merged
// through shared memory.  Bound by the latency of its loads (2.2 ms where the tile kernels
// take 0.18 for a bf16 decode batch): it serves the shapes and types outside those, as int4
// and fp32 caches, q of another type than the cache, other head_dims and odd pages.
template <int J, int GC>
__global__ void __launch_bounds__(kAgWarps * 32) attn_generic_kernel(const AttnArgs a) {
    const int h = blockIdx.y;
    const int G = a.num_q_heads / a.num_kv_heads;
    const int g0 = blockIdx.z * GC;
    const int ng = min(GC, G - g0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int D = a.head_dim, BS = a.block_size;

    __shared__ float sm_m[kAgWarps][GC], sm_l[kAgWarps][GC];
    __shared__ float sm_acc[kAgWarps][GC][J * 32];

    if (blockIdx.x == 0 && h == 0 && blockIdx.z == 0) {
        for (int s = threadIdx.x; s < a.num_seqs; s += blockDim.x) check_seq(a, s);
        for (int g = threadIdx.x; g < a.num_groups; g += blockDim.x) check_group(a, g);
    }
    const int t = blockIdx.x;
    int q0, n;
    const int s = seq_of_token(a, t, q0, n);
    if (s < 0) return;
    const int len = clamp_len(a, a.context_lens[s], a.max_blocks);
    const int pos = len - n + (t - q0);
    int lo, hi;
    if (a.num_groups > 0) {
        lo = 0;
        hi = len;
    } else {
        row_range(a, s, t, pos, len, lo, hi);
    }

    float qr[GC][J], m[GC], l[GC], acc[GC][J], slope[GC];
    const long long qrow = (static_cast<long long>(t) * a.num_q_heads + h * G + g0) * D;
#pragma unroll
    for (int hh = 0; hh < GC; ++hh) {
        m[hh] = -INFINITY;
        l[hh] = 0.f;
        slope[hh] = (a.slopes && hh < ng) ? a.slopes[h * G + g0 + hh] * kLog2e : 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int d = lane + 32 * j;
            acc[hh][j] = 0.f;
            qr[hh][j] = (hh < ng && d < D) ? load_elem(a.q, a.q_dtype, qrow + static_cast<long long>(hh) * D + d) * a.q_scale : 0.f;
        }
    }

    const bool quant = a.kv_dtype == GOLLEK_DTYPE_I8 || a.kv_dtype == GOLLEK_DTYPE_I4;
    const bool cap = a.soft_cap > 0.f;
    // positions [plo, phi) of one table row
    auto pass = [&](const int *bt, int plo, int phi) {
        for (int p0 = plo + warp * kAgTok; p0 < phi; p0 += kAgWarps * kAgTok) {
            float kk[kAgTok][J], vv[kAgTok][J], ks[kAgTok];
            bool live[kAgTok];
#pragma unroll
            for (int u = 0; u < kAgTok; ++u) {
                const int p = p0 + u;
                live[u] = p < phi;
                ks[u] = 1.f;
                float vs = 1.f;
                long long e0 = 0;
                if (live[u]) {
                    const int page = bt[p / BS];
                    if (page < 0 || (a.num_blocks > 0 && page >= a.num_blocks)) {
                        if (lane == 0) raise_status(GOLLEK_STATUS_BAD_BLOCK_ID);
                        live[u] = false;
                    } else {
                        const int slot = p % BS;
                        e0 = static_cast<long long>(page) * a.page_stride +
                             (static_cast<long long>(h) * BS + slot) * D;
                        if (quant) {
                            const long long so = static_cast<long long>(page) * a.scale_page_stride +
                                                 static_cast<long long>(h) * a.scale_head_stride +
                                                 static_cast<long long>(slot) * a.scale_token_stride;
                            ks[u] = a.k_scales[so];
                            vs = a.v_scales[so];
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int d = lane + 32 * j;
                    const bool on = live[u] && d < D;
                    kk[u][j] = on ? load_kv(a.k, a.kv_dtype, e0 + d) : 0.f;
                    vv[u][j] = on ? load_kv(a.v, a.kv_dtype, e0 + d) * vs : 0.f;
                }
            }
#pragma unroll
            for (int hh = 0; hh < GC; ++hh) {
                if (hh >= ng) break;
                float x[kAgTok], mn = m[hh];
#pragma unroll
                for (int u = 0; u < kAgTok; ++u) {
                    float part = 0.f;
#pragma unroll
                    for (int j = 0; j < J; ++j) part += qr[hh][j] * kk[u][j];
                    x[u] = warp_sum(part) * ks[u];
                    if (cap) x[u] = a.soft_cap * tanhf(x[u] / a.soft_cap) * kLog2e;
                    x[u] -= slope[hh] * fabsf(static_cast<float>(pos - (p0 + u)));
                    if (!live[u]) x[u] = -INFINITY;
                    mn = fmaxf(mn, x[u]);
                }
                const float ref = mn == -INFINITY ? 0.f : mn;  // nothing visible yet: every p is 0
                const float alpha = (mn == m[hh]) ? 1.f : fast_exp2(m[hh] - mn);
                m[hh] = mn;
                l[hh] *= alpha;
#pragma unroll
                for (int j = 0; j < J; ++j) acc[hh][j] *= alpha;
#pragma unroll
                for (int u = 0; u < kAgTok; ++u) {
                    const float p = fast_exp2(x[u] - ref);
                    l[hh] += p;
#pragma unroll
                    for (int j = 0; j < J; ++j) acc[hh][j] = fmaf(p, vv[u][j], acc[hh][j]);
                }
            }
        }
    };
    if (a.num_groups > 0) {
        const int g = group_of_seq(a, s);
        if (g >= 0)
            pass(a.prefix_tables + static_cast<long long>(g) * a.max_pblocks, 0,
                 clamp_len(a, a.group_plens[g], a.max_pblocks));
    }
    pass(a.block_tables + static_cast<long long>(s) * a.max_blocks, lo, hi);

#pragma unroll
    for (int hh = 0; hh < GC; ++hh) {
        if (lane == 0) {
            sm_m[warp][hh] = m[hh];
            sm_l[warp][hh] = l[hh];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) sm_acc[warp][hh][lane + 32 * j] = acc[hh][j];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < ng * D; o += kAgWarps * 32) {
        const int hh = o / D, d = o - hh * D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAgWarps; ++w) M = fmaxf(M, sm_m[w][hh]);
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int w = 0; w < kAgWarps; ++w) {
            const float f = M == -INFINITY ? 1.f : fast_exp2(sm_m[w][hh] - M);
            L += sm_l[w][hh] * f;
            A += sm_acc[w][hh][d] * f;
        }
        store_elem(a.out, a.q_dtype, qrow + o, L == 0.f ? 0.f : A / L);  // a NaN stays one
    }
}

}  // namespace gk
