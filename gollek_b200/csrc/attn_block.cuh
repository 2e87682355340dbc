// attn_block.cuh -- ragged attention of many rows for every type and shape: fp32 and int4
// caches, queries of another type than the cache, head_dims and pages the tensor-core kernels
// do not take.
//
// One CTA per 64 rows -- (query token, q head) pairs of one kv head -- and tiles of 32
// positions, both as fp32 in shared memory; a thread has 4 rows x 2 positions of the scores
// and 4 rows x DP / 16 columns of the output in registers, and a row's softmax lies within
// half a warp.  All products and sums are fp32 FMAs (fp32 callers are owed fp32), which bound
// it: 2 D FMAs per row and position, at 128 a clock and SM (a third of that rate is reached,
// for want of warps: two CTAs fill an SM's shared memory).  A cache row is read once for 64
// rows instead of once per query token: 8 fp32 prompts of 96 tokens at 400 to 1500 tokens of
// context (32 q, 8 kv heads of 128) take 0.79 ms, 3.2 in the kernel of varlen.cuh.
#pragma once

#include <climits>

#include "varlen.cuh"

namespace gk {

constexpr int kAbRows = 64;
constexpr int kAbTok = 32;
constexpr int kAbThreads = 256;

template <int DP>
constexpr size_t kAbSmem = ((kAbRows + kAbTok) * (DP + 4) + kAbTok * DP + kAbRows * (kAbTok + 4) + kAbTok) * 4 + 16;

// DP: head_dim, padded with zeros.  KV: the pool's type.  qt: query tokens of a CTA's 64 rows; a
// sequence has ceil(n / qt) CTAs per kv head, in order, and the grid may have more than that.
template <int DP, int KV>
__global__ void __launch_bounds__(kAbThreads) attn_block_kernel(const AttnArgs a, const int qt) {
    constexpr int QS = DP + 4, PS = kAbTok + 4, DC = DP / 64;  // row strides (floats); float4 of output columns a thread has
    extern __shared__ __align__(16) float ab_smem[];
    float *sq = ab_smem, *sk = sq + kAbRows * QS, *sv = sk + kAbTok * QS, *sp = sv + kAbTok * DP;
    int *there = reinterpret_cast<int *>(sp + kAbRows * PS);  // [kAbTok] position has a page
    int *span = there + kAbTok;                               // first and last position of the rows
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tx = tid & 15, ty = tid >> 4;
    const int h = blockIdx.y, G = a.num_q_heads / a.num_kv_heads, D = a.head_dim, BS = a.block_size;
    constexpr bool quant = KV == GOLLEK_DTYPE_I8 || KV == GOLLEK_DTYPE_I4;
    const bool cap = a.soft_cap > 0.f;
    if (blockIdx.x == 0 && h == 0)
        for (int s = tid; s < a.num_seqs; s += kAbThreads) check_seq(a, s);

    // this CTA's sequence: the running number of blocks, 32 sequences at a time
    int s = -1, blk = blockIdx.x;
    for (int s0 = 0; s0 < a.num_seqs && s < 0; s0 += 32) {
        int first = 0, n = 0;
        if (s0 + lane < a.num_seqs) seq_rows(a, s0 + lane, first, n);
        const int mine = (n + qt - 1) / qt;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > blk);
        if (past) {
            const int at = __ffs(past) - 1;
            s = s0 + at;
            blk -= __shfl_sync(0xffffffffu, sum - mine, at);
        } else {
            blk -= __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    if (s < 0) return;
    int q0, n;
    seq_rows(a, s, q0, n);
    if (blk < 0 || blk >= (n + qt - 1) / qt) return;  // offsets that are not usable (reported)
    const int t = q0 + blk * qt, te = min(t + qt, q0 + n), rows = (te - t) * G;
    const int len = clamp_len(a, a.context_lens[s], a.max_blocks), pos0 = len - n + (t - q0);
    const int *bt = a.block_tables + static_cast<long long>(s) * a.max_blocks;
    if (tid == 0) {
        span[0] = INT_MAX;
        span[1] = 0;
    }
    for (int i = tid; i < kAbRows * DP; i += kAbThreads) {
        const int r = i / DP, d = i % DP, tok = r / G;
        float v = 0.f;
        if (r < rows && d < D)
            v = load_elem(a.q, a.q_dtype, (static_cast<long long>(t + tok) * a.num_q_heads + h * G + (r - tok * G)) * D + d) * a.q_scale;
        sq[r * QS + d] = v;
    }
    __syncthreads();
    int lo[4], hi[4], pos[4];
    float slope[4], m[4], l[4], acc[4][4 * DC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * ty + i, tok = r / G;
        lo[i] = hi[i] = pos[i] = 0;
        slope[i] = 0.f;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4 * DC; ++c) acc[i][c] = 0.f;
        if (r >= rows) continue;
        pos[i] = pos0 + tok;
        row_range(a, s, t + tok, pos[i], len, lo[i], hi[i]);
        if (a.slopes) slope[i] = a.slopes[h * G + (r - tok * G)] * kLog2e;
        if (tx == 0 && lo[i] < hi[i]) {
            atomicMin(&span[0], lo[i]);
            atomicMax(&span[1], hi[i]);
        }
    }
    __syncthreads();
    const int last = span[1], first = min(span[0], last);  // an empty span where no row sees anything
    // lane u < 4: the page of the warp's position u, looked up a tile ahead
    int next = lane < 4 && first + 4 * warp + lane < last ? bt[(first + 4 * warp + lane) / BS] : 0;
    for (int p0 = first; p0 < last; p0 += kAbTok) {
        __syncthreads();  // the last tile is read
        const int pages = next, ahead = p0 + kAbTok + 4 * warp + lane;
        if (lane < 4 && ahead < last) next = bt[ahead / BS];
        // four positions a warp, their elements in flight together
        {
            float kk[4][DP / 32], vv[4][DP / 32];
            float ks[4], vs[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int p = p0 + 4 * warp + u;
                bool live = p < last;
                const int page = __shfl_sync(0xffffffffu, pages, u);
                long long e0 = 0;
                ks[u] = vs[u] = 1.f;
                if (live) {
                    if (page < 0 || (a.num_blocks > 0 && page >= a.num_blocks)) {
                        if (lane == 0) raise_status(GOLLEK_STATUS_BAD_BLOCK_ID);
                        live = false;
                    } else {
                        const int slot = p % BS;
                        e0 = static_cast<long long>(page) * a.page_stride + (static_cast<long long>(h) * BS + slot) * D;
                        if (quant) {
                            const long long so = static_cast<long long>(page) * a.scale_page_stride +
                                                 static_cast<long long>(h) * a.scale_head_stride +
                                                 static_cast<long long>(slot) * a.scale_token_stride;
                            ks[u] = a.k_scales[so];
                            vs[u] = a.v_scales[so];
                        }
                    }
                }
                if (lane == 0) there[4 * warp + u] = live;
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    const bool on = live && lane + 32 * j < D;
                    kk[u][j] = on ? load_kv(a.k, KV, e0 + lane + 32 * j) : 0.f;
                    vv[u][j] = on ? load_kv(a.v, KV, e0 + lane + 32 * j) : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    sk[(4 * warp + u) * QS + lane + 32 * j] = kk[u][j] * ks[u];
                    sv[(4 * warp + u) * DP + lane + 32 * j] = vv[u][j] * vs[u];
                }
        }
        __syncthreads();
        float x[4][2] = {};
        for (int d = 0; d < D; d += 4) {
            float4 k4[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) k4[j] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * j) * QS + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 q4 = *reinterpret_cast<const float4 *>(sq + (4 * ty + i) * QS + d);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[i][j] = fmaf(q4.x, k4[j].x, x[i][j]);
                    x[i][j] = fmaf(q4.y, k4[j].y, x[i][j]);
                    x[i][j] = fmaf(q4.z, k4[j].z, x[i][j]);
                    x[i][j] = fmaf(q4.w, k4[j].w, x[i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mn = m[i];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int p = p0 + tx + 16 * j;
                if (cap) x[i][j] = a.soft_cap * tanhf(x[i][j] / a.soft_cap) * kLog2e;
                x[i][j] -= slope[i] * fabsf(static_cast<float>(pos[i] - p));
                if (p < lo[i] || p >= hi[i] || !there[tx + 16 * j]) x[i][j] = -INFINITY;
                mn = fmaxf(mn, x[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            const float ref = mn == -INFINITY ? 0.f : mn;  // nothing visible yet: every p is 0
            const float alpha = mn == m[i] ? 1.f : fast_exp2(m[i] - mn);
            m[i] = mn;
            l[i] *= alpha;
#pragma unroll
            for (int c = 0; c < 4 * DC; ++c) acc[i][c] *= alpha;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float pr = fast_exp2(x[i][j] - ref);
                l[i] += pr;
                sp[(4 * ty + i) * PS + tx + 16 * j] = pr;
            }
        }
        __syncwarp();  // a row's probabilities are written and read by one half warp
#pragma unroll 2
        for (int p = 0; p < kAbTok; p += 4) {
            float4 p4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p4[i] = *reinterpret_cast<const float4 *>(sp + (4 * ty + i) * PS + p);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const float4 v4 = *reinterpret_cast<const float4 *>(sv + (p + u) * DP + 64 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = u == 0 ? p4[i].x : u == 1 ? p4[i].y : u == 2 ? p4[i].z : p4[i].w;
                        acc[i][4 * c] = fmaf(w, v4.x, acc[i][4 * c]);
                        acc[i][4 * c + 1] = fmaf(w, v4.y, acc[i][4 * c + 1]);
                        acc[i][4 * c + 2] = fmaf(w, v4.z, acc[i][4 * c + 2]);
                        acc[i][4 * c + 3] = fmaf(w, v4.w, acc[i][4 * c + 3]);
                    }
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float sum = l[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int r = 4 * ty + i, tok = r / G;
        if (r >= rows) continue;
        const long long o0 = (static_cast<long long>(t + tok) * a.num_q_heads + h * G + (r - tok * G)) * D;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a NaN stays one
#pragma unroll
        for (int c = 0; c < 4 * DC; ++c) {
            const int d = 64 * (c / 4) + 4 * tx + c % 4;
            if (d < D) store_elem(a.out, a.q_dtype, o0 + d, sum == 0.f ? 0.f : acc[i][c] * inv);
        }
    }
}

}  // namespace gk
