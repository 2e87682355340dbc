// attn_rows.cuh -- the tile kernel for blocks of few rows (decode steps): up to 16 rows of one
// kv head, head_dim 128, in tiles of 128 positions.  Plan, ring and merge are attn_tile.cuh's.
//
// With the rows as the N of both products, nothing of a 128-lane tile is spent on rows that
// are not there:
//
//   S[128 pos x 16 rows] = K . Q^T      P = 2^(x - m), rounded to the cache's type
//   O[D x 16 rows]      += V^T . P      l += sum P (fp32, unrounded)
//
// One thread owns one position of a tile (an int8 position's scales are one load each) and
// one column of the output.  P goes back through 4 KB of shared memory.  The reference m of a
// row belongs to all 128 threads of a group, so they vote, tile by tile, whether any of
// their scores passes it by kLazyMax; only then is a maximum taken.
//
// Bound by HBM for 16-bit caches, each page being read once per kv head: a decode step of 64
// sequences of 512 to 8192 tokens (32 q, 8 kv heads of 128) takes 183 us, 6.2 TB/s (237 us
// in attn_tile.cuh's kernel, whose blocks of 128 rows are empty but for 4).  For int8 caches
// by the instructions that turn bytes into bf16 (of 8,700 a tile, issued in 57% of the slots,
// before their address arithmetic went): 48 such sequences take 191 us, 2.4 TB/s (286 us
// there).  K is converted by warps of its own, V by the group whose
// tile it is, which would wait for its scores' MMA meanwhile.
#pragma once

#include "attn_tile.cuh"

namespace gk {

constexpr int kFewRows = 16;
constexpr int kFewD = 128;             // the value product's M
constexpr int kRowsThreads = 352;      // 8 row warps, the MMA issuer, 2 producers
constexpr int kRowsConverters = 128;   // more for int8 caches

template <bool Q8>
struct RowsSmem {
    static constexpr int D = kFewD;
    static constexpr uint32_t kSlot = kTileTok * D * 2;
    static constexpr uint32_t kQ = kFewRows * D * 2;
    static constexpr uint32_t kP = kFewRows * kTileTok * 2;
    static constexpr int kSlots = Q8 ? 4 : 6;
    static constexpr int kRaw = Q8 ? 4 : 0;
    static constexpr int kScales = Q8 ? 8 : 0;  // copies are at most 5 tiles ahead of a tile in use
    static constexpr int kRuns = 4;
    static constexpr uint32_t q = 0;                              // [2]
    static constexpr uint32_t pr = q + 2 * kQ;                    // [2]
    static constexpr uint32_t ring = pr + 2 * kP;
    static constexpr uint32_t raw = ring + kSlots * kSlot;
    static constexpr uint32_t scales = raw + kRaw * (kSlot / 2);
    static constexpr uint32_t rows = scales + kScales * 1024;     // [8 warps][16] x 16 bytes
    static constexpr uint32_t vmax = rows + 8 * kFewRows * 16;    // [2 groups][4 warps][16] floats
    static constexpr uint32_t sums = vmax + 2 * 4 * kFewRows * 4; // [2][4][16] floats
    static constexpr uint32_t refs = sums + 2 * 4 * kFewRows * 4; // [2][16] floats
    static constexpr uint32_t flags = refs + 2 * kFewRows * 4;    // [2][4] ints
    static constexpr uint32_t runs = flags + 32;
    static constexpr uint32_t bars = runs + kRuns * 48;
    static constexpr int kBars = 2 * kSlots + 2 * kRaw + 2 * kRuns + 2 * 8 + 1;
    static constexpr uint32_t misc = bars + kBars * 8;
    static constexpr uint32_t total = misc + 16;
};

// A row as its scores need it: positions [lo, hi), its own position, its bias.
struct __align__(16) RowInfo {
    int lo, hi, pos;
    float slope;
};

template <typename T, bool Q8>
__global__ void __launch_bounds__(kRowsThreads + (Q8 ? kRowsConverters : 0), 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const TileArgs p) {
    using L = RowsSmem<Q8>;
    constexpr int D = kFewD, N = kFewRows, NS = L::kSlots;
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    const AttnArgs &a = p.a;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    const TilePipe<L> pipe(tile_smem);
    uint8_t *const ring = tile_smem + L::ring;
    RunDesc *const runs = pipe.runs;
    uint64_t *const full = pipe.full, *const empty = pipe.empty, *const run_full = pipe.run_full, *const run_free = pipe.run_free;
    volatile int *const abort = pipe.abort;
    uint64_t *s_full = pipe.own;   // [2] scores in tensor memory (and every earlier MMA done)
    uint64_t *p_full = s_full + 2; // [2] probabilities in shared memory (V cleared, O rescaled)
    uint64_t *o_full = p_full + 2; // [2] a run's last value MMA of the group done
    uint64_t *o_free = o_full + 2; // [2] O read
    uint64_t *q_full = o_free + 2; // [2] q staged in buffer 0, 1
    uint64_t *q_free = q_full + 2; // [2] q buffer read
    uint64_t *vote = q_free + 2;   // [2] the group's warps have looked at their scores
    uint64_t *sums_full = vote + 2; // [2] the group's (m, l) of a run written
    uint64_t *drained = sums_full + 2;
    uint32_t *sm_tmem = reinterpret_cast<uint32_t *>(tile_smem + L::misc + 8);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        constexpr int conv = kRowsConverters / 32;
        pipe.init(Q8 ? conv : 2, 1, 9 + (Q8 ? conv : 0), p.wait_tries);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_free[t], 4);
            mbar_init(&q_full[t], 4);
            mbar_init(&q_free[t], 1);
            mbar_init(&vote[t], 4);
            mbar_init(&sums_full[t], 4);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
    }
    if (!Q8 && warp == 9 && lane == 0) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(sm_tmem), 64);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *sm_tmem;
    auto wait = [&](uint64_t *bar, uint32_t phase) { return pipe.wait(bar, phase); };

    if (warp == 9 || warp == 10) {
        tile_producer<L, D, Q8>(p, pipe, tm_k, tm_v, lane, warp - 9);
    } else if (warp > 10) {
        if constexpr (Q8) {
            static_assert(L::kRaw == L::kSlots, "see tile_converter");
            tile_converter<L, D, kRowsConverters, true>(pipe, tid - kRowsThreads);
        }
    } else if (warp == 8) {
        // ===================================================================== MMA issuer
        // Tiles alternate between the groups; step j has the values of tile j - 2 and the scores of
        // tile j, which is the order of the ring.
        constexpr uint32_t id_s = umma_idesc_16bit(128, N, kBf16, 0, 0);
        constexpr uint32_t id_o = umma_idesc_16bit(D, N, kBf16, 1, 0);
        const uint64_t k_desc = umma_desc_sw128(smem_u32(ring), 16, 16 * D);
        const uint64_t v_desc = umma_desc_sw128(smem_u32(ring), 1024, 16 * D);
        const bool leader = elect_one();
        int slot = 0;
        uint32_t ring_ph = 0;
        uint32_t pp = 0;         // bit t: phase of group t's next probabilities
        int ou[2] = {0, 0};      // runs that used group t's O so far
        bool ok = true;
#pragma unroll 1
        for (int run = 0;; ++run) {
            const int at = run % L::kRuns;
            ok = wait(&run_full[at], run / L::kRuns);
            if (!ok) break;
            const int n = __shfl_sync(0xffffffffu, runs[at].n, 0);
            if (leader) mbar_arrive(&run_free[at]);
            if (n == 0) break;
            const int qb = run & 1;
            ok = wait(&q_full[qb], run >> 1);
            const uint64_t qd = umma_desc_sw128(smem_u32(tile_smem + L::q + qb * L::kQ), 16, 1024);
#pragma unroll 1
            for (int j = 0; ok && j < n + 2; ++j) {
                const int t = j & 1;
                if (j >= 2) {
                    const int vs = slot;
                    const uint32_t vp = ring_ph;
                    if (++slot == NS) {
                        slot = 0;
                        ring_ph ^= 1;
                    }
                    const bool first = j < 4;
                    const int used = t ? ou[1] : ou[0];
                    ok = wait(&full[vs], vp);
                    if (first && used > 0) ok = ok && wait(&o_free[t], used - 1);
                    ok = ok && wait(&p_full[t], pp >> t);
                    if (!ok) break;
                    pp ^= 1u << t;
                    tc_fence_after();
                    const uint64_t vd = v_desc + vs * (L::kSlot >> 4);
                    const uint64_t pd = umma_desc_sw128(smem_u32(tile_smem + L::pr + t * L::kP), 16, 1024);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < kTileTok / 16; ++kk)
                            umma_f16(tmem + 32 + 16 * t, vd + kk * (32 * D >> 4), pd + (kk >> 2) * (2048 >> 4) + (kk & 3) * 2, id_o,
                                     !(first && kk == 0));
                        umma_commit(&empty[vs]);
                        if (j >= n) umma_commit(&o_full[t]);  // the group's last tile
                    }
                }
                if (j < n) {
                    const int ks = slot;
                    const uint32_t kp = ring_ph;
                    if (++slot == NS) {
                        slot = 0;
                        ring_ph ^= 1;
                    }
                    ok = wait(&full[ks], kp);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t kd = k_desc + ks * (L::kSlot >> 4);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_f16(tmem + 16 * t, kd + (kk >> 2) * (1024 >> 4) + (kk & 3) * 2,
                                     qd + (kk >> 2) * (2048 >> 4) + (kk & 3) * 2, id_s, kk > 0);
                        umma_commit(&s_full[t]);
                        umma_commit(&empty[ks]);
                        if (j == n - 1) umma_commit(&q_free[qb]);
                    }
                }
            }
            if (!ok) break;
            ++ou[0];
            if (n > 1) ++ou[1];
        }
        if (!ok && lane == 0) tile_give_up(abort);
        // every MMA issued has completed before tensor memory and shared memory go
        if (leader) {
            umma_commit(drained);
            mbar_wait(drained, 0);
        }
        __syncwarp();
    } else {
        // ===================================================================== row groups
        const int G = a.num_q_heads / a.num_kv_heads;
        const unsigned g_magic = div_magic(G);
        const int t = warp >> 2, w4 = warp & 3;
        const int row = tid & 127;  // position in a tile; column of the output
        const uint32_t lanes = static_cast<uint32_t>(32 * w4) << 16;
        const uint32_t t_s = tmem + 16 * t + lanes, t_o = tmem + 32 + 16 * t + lanes;
        RowInfo *const info = reinterpret_cast<RowInfo *>(tile_smem + L::rows) + warp * N;
        float *const vmax = reinterpret_cast<float *>(tile_smem + L::vmax) + t * 4 * N;
        float *const sums = reinterpret_cast<float *>(tile_smem + L::sums);
        float *const refs = reinterpret_cast<float *>(tile_smem + L::refs);
        int *const flags = reinterpret_cast<int *>(tile_smem + L::flags) + 4 * t;
        const uint32_t my_p = smem_u32(tile_smem + L::pr + t * L::kP) + (row >> 6) * 2048 + (row & 7) * 2;
        const int my_ch = (row & 63) >> 3;
        int c0 = 0, sn = 0;             // ring position of the run's first K; this group's tiles so far
        [[maybe_unused]] int sc0 = 0;   // scales of the run's first tile
        int ou[2] = {0, 0};             // runs that used O of group 0, 1 so far
        int fills = 0;                  // of this group's q buffer so far
        bool ok = true;

        // The q of run `next`, by the group whose buffer it is; rows that are not there are zeros.
        auto fill_q = [&](int next) {
            const int at = next % L::kRuns;
            if (!(ok = wait(&run_full[at], next / L::kRuns))) return;
            const RunDesc *d = &runs[at];
            if (d->n == 0 || (next & 1) != t) return;
            if (fills > 0 && !(ok = wait(&q_free[t], fills - 1))) return;
            ++fills;
            const T *q0 = reinterpret_cast<const T *>(a.q) + (static_cast<long long>(d->tok0) * a.num_q_heads + d->h * G) * D;
            const uint32_t dst = smem_u32(tile_smem + L::q) + t * L::kQ;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = (row >> 4) + 8 * k, ch = row & 15;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < d->nrows) {
                    const int rho = d->row0 + r, tok = fast_div(rho, G, g_magic);
                    v = __ldg(reinterpret_cast<const uint4 *>(q0 + (static_cast<long long>(tok) * a.num_q_heads + (rho - tok * G)) * D) + ch);
                }
                sts_u4(dst + (ch >> 3) * 2048 + r * 128 + (((ch & 7) ^ (r & 7)) << 4), v);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
        };

#pragma unroll 1
        for (int run = -1;; ++run) {  // -1: only fetches the first run's q
            RunDesc d{};
            if (run >= 0) {
                const int at = run % L::kRuns;
                if (!(ok = wait(&run_full[at], run / L::kRuns))) break;
                d = runs[at];
                __syncwarp();
                if (lane == 0) mbar_arrive(&run_free[at]);
                if (d.n == 0) break;
            }
            const int n = d.n;
            // lane r < 16 looks after row r; the others of 16 rows see what the block sees
            RowInfo me{d.lo, d.hi, 0, 0.f};
            const long long out0 = static_cast<long long>(d.tok0) * a.num_q_heads;
            long long out_row = out0;
            if (lane < d.nrows) {
                const int rho = d.row0 + lane, i = fast_div(rho, G, g_magic), head = d.h * G + (rho - i * G);
                out_row = static_cast<long long>(d.tok0 + i) * a.num_q_heads + head;
                if ((d.flags & 3) == kOwn) {
                    me.pos = d.pos0 + i;
                    row_range(a, d.tab, d.tok0 + i, me.pos, d.len, me.lo, me.hi);
                }
                if (a.slopes) me.slope = a.slopes[head] * kLog2e;
            }
            __syncwarp();  // the last run's rows are read
            if (lane < N) info[lane] = me;
            __syncwarp();
            const int last_lo = __reduce_max_sync(0xffffffffu, me.lo), first_hi = __reduce_min_sync(0xffffffffu, me.hi);
            float m[N], l[N];  // references (exponent domain; the group's threads agree); sums of this thread's positions
#pragma unroll
            for (int r = 0; r < N; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.f;
            }
#pragma unroll 1
            for (int j = t; j < n; j += 2) {
                const int t0 = (d.tile0 - j) * kTileTok, at = t0 + row;
                ok = wait(&s_full[t], sn);
                if (!ok) break;
                tc_fence_after();
                float x[N];
                tmem_ld<N>(t_s, x);
                // V rows that no row of the block attends are cleared (a zero probability does not
                // cancel a NaN); int8: integers are finite, their scales are left out
                const bool inside = at >= d.lo && at < d.hi;
                if (!Q8 && (d.lo > t0 || d.hi < t0 + kTileTok)) {
                    const int cv = c0 + v_at(j, n);
                    ok = wait(&full[cv % NS], cv / NS);
                    if (!ok) break;
                    const uint32_t vt = smem_u32(ring) + (cv % NS) * L::kSlot;
                    if (!inside)
#pragma unroll 4
                        for (int ch = 0; ch < D / 8; ++ch) sts_u4(vt + kv_chunk_off<D>(row, ch), make_uint4(0, 0, 0, 0));
                }
                if constexpr (Q8) {
                    // V is this group's to convert (K the converter warps'): its slot is free, since the
                    // scores' commit covers the MMAs four copies back
                    const int cv = c0 + v_at(j, n);
                    ok = wait(&empty[cv % NS], cv / NS - 1) && wait(&pipe.raw_full[cv % NS], cv / NS);
                    if (!ok) break;
                    convert_tile<D, 128>(smem_u32(tile_smem + L::raw) + cv % NS * (L::kSlot / 2), smem_u32(ring) + cv % NS * L::kSlot, row);
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&full[cv % NS]);
                        mbar_arrive(&pipe.raw_free[cv % NS]);
                    }
                }
                float f = a.q_scale;
                [[maybe_unused]] float fv = 1.f;
                if constexpr (Q8) {
                    const float *s = reinterpret_cast<const float *>(tile_smem + L::scales) + (sc0 + j) % L::kScales * 256;
                    f *= s[row];
                    fv = inside ? s[128 + row] : 0.f;
                }
                tmem_wait_ld();
                if (a.soft_cap > 0.f) {
                    f *= 1.f / a.soft_cap;
#pragma unroll
                    for (int r = 0; r < N; ++r) x[r] *= f;
                    // each score in its own way: a position's 16 rows do not depend on one another, nor on the
                    // warp's other positions; the vote only leaves out the second way where none needs it
                    float big = 0.f;
#pragma unroll
                    for (int r = 0; r < N; ++r) big = fmaxf(big, fabsf(x[r]));
                    if (__any_sync(0xffffffffu, big > 0.5f)) {
#pragma unroll
                        for (int r = 0; r < N; r += 2) {
                            const float2 q = tanh_small(make_float2(x[r], x[r + 1]));
                            x[r] = fabsf(x[r]) > 0.5f ? tanh_large(x[r]) : q.x;
                            x[r + 1] = fabsf(x[r + 1]) > 0.5f ? tanh_large(x[r + 1]) : q.y;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < N; r += 2) {
                            const float2 q = tanh_small(make_float2(x[r], x[r + 1]));
                            x[r] = q.x;
                            x[r + 1] = q.y;
                        }
                    }
                    f = a.soft_cap * kLog2e;
                }
#pragma unroll
                for (int r = 0; r < N; ++r) x[r] *= f;
                if (opaque(a.slopes != nullptr)) {
#pragma unroll
                    for (int r = 0; r < N; ++r) x[r] = fmaf(-info[r].slope, fabsf(static_cast<float>(at - info[r].pos)), x[r]);
                }
                if (opaque(last_lo > t0 || first_hi < t0 + kTileTok)) {
#pragma unroll
                    for (int r = 0; r < N; ++r) x[r] = at >= info[r].lo && at < info[r].hi ? x[r] : -INFINITY;
                }
                bool up = false;
#pragma unroll
                for (int r = 0; r < N; ++r) up |= x[r] - m[r] > kLazyMax<T>;  // false of -inf - -inf
                up = __any_sync(0xffffffffu, up);
                if (up) {
#pragma unroll
                    for (int r = 0; r < N; ++r) {
                        float v = x[r];
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
                        if (lane == r) vmax[w4 * N + r] = v;
                    }
                }
                if (lane == 0) flags[w4] = up;
                __syncwarp();
                if (lane == 0) mbar_arrive(&vote[t]);
                ok = wait(&vote[t], sn++);
                if (!ok) break;
                const int4 fl = *reinterpret_cast<const int4 *>(flags);
                if (fl.x | fl.y | fl.z | fl.w) {
                    // The references rise by an integer (where there was one), and the sums and O follow.
                    const int r0 = lane & (N - 1);  // this lane's row of the 16
                    float was = m[0];
#pragma unroll
                    for (int r = 1; r < N; ++r) was = r0 == r ? m[r] : was;
                    float top = fl.x ? vmax[r0] : -INFINITY;
                    top = fmaxf(top, fl.y ? vmax[N + r0] : -INFINITY);
                    top = fmaxf(top, fl.z ? vmax[2 * N + r0] : -INFINITY);
                    top = fmaxf(top, fl.w ? vmax[3 * N + r0] : -INFINITY);
                    const bool move = top - was > kLazyMax<T>;
                    const float by = move && was != -INFINITY ? ceilf(top - was) - kBelowMax<T> : 0.f;
                    const float now = !move ? was : was == -INFINITY ? top - kBelowMax<T> : was + by;
                    const float fall = fast_exp2(-by);
                    float alpha[N];
#pragma unroll
                    for (int r = 0; r < N; ++r) {
                        m[r] = __shfl_sync(0xffffffffu, now, r);
                        alpha[r] = __shfl_sync(0xffffffffu, fall, r);
                        l[r] *= alpha[r];
                    }
                    if (j != t) {  // the scores' commit covers the group's earlier value MMAs: O is at rest
                        float o[N];
                        tmem_ld<N>(t_o, o);
                        tmem_wait_ld();
                        uint32_t u[N];
#pragma unroll
                        for (int r = 0; r < N; ++r) u[r] = __float_as_uint(o[r] * alpha[r]);
                        tmem_st16(t_o, u);
                        tmem_wait_st();
                    }
                }
#pragma unroll
                for (int r = 0; r < N; ++r) {
                    float e = fast_exp2(x[r] - (m[r] == -INFINITY ? 0.f : m[r]));
                    l[r] += e;
                    if constexpr (Q8) e *= fv;
                    T v;
                    if constexpr (kBf16)
                        v = __float2bfloat16_rn(e);
                    else
                        v = __float2half_rn(e);
                    sts_u2(my_p + r * 128 + ((my_ch ^ (r & 7)) << 4), v);
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            fill_q(run + 1);  // the next run's q, under this run's last products
            if (!ok) break;
            if (run < 0) continue;

            // ------------------------------------------------ end of the run
            const bool two = n > 1;  // both groups hold a part of each row
            if (t == 0 || two) {
                // this thread's sums over the warp: lanes 2 r and 2 r + 1 end with row r's
#pragma unroll
                for (int o = 16, h = 8; h > 0; o >>= 1, h >>= 1) {
                    const bool hi_half = lane & o;
#pragma unroll
                    for (int i = 0; i < h; ++i) {
                        const float give = hi_half ? l[i] : l[i + h], keep = hi_half ? l[i + h] : l[i];
                        l[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
                }
                l[0] += __shfl_xor_sync(0xffffffffu, l[0], 1);
                // group 0 has read what group 1 handed over before (it freed O behind that)
                if (t == 1 && ou[1] > 0) ok = wait(&o_free[1], ou[1] - 1);
                if (!ok) break;
                if (!(lane & 1)) sums[(t * 4 + w4) * N + (lane >> 1)] = l[0];
                if (w4 == 0 && lane == 0) {
#pragma unroll
                    for (int r = 0; r < N; ++r) refs[t * N + r] = m[r];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sums_full[t]);
            }
            if (t == 0) {
                ok = wait(&o_full[0], ou[0]) && wait(&sums_full[0], ou[0]) &&
                     (!two || (wait(&sums_full[1], ou[1]) && wait(&o_full[1], ou[1])));
                if (!ok) break;
                tc_fence_after();
                // lane r: row r's (m, l) of both groups, and what their O are worth
                const int r0 = lane & (N - 1);
                float mm = refs[r0], ll = sums[r0] + sums[N + r0] + sums[2 * N + r0] + sums[3 * N + r0], fa = 1.f, fb = 0.f;
                if (two) {
                    const float ma = mm, mb = refs[N + r0];
                    const float *s1 = sums + 4 * N + r0;
                    const float lb = s1[0] + s1[N] + s1[2 * N] + s1[3 * N];
                    mm = fmaxf(ma, mb);
                    fa = ma == -INFINITY ? (ll == 0.f ? 0.f : 1.f) : fast_exp2(ma - mm);
                    fb = mb == -INFINITY ? (lb == 0.f ? 0.f : 1.f) : fast_exp2(mb - mm);
                    ll = ll * fa + lb * fb;
                }
                const bool whole = d.flags & 4, direct = whole && (d.flags & 3) == kOwn;
                const float inv = ll == 0.f ? 0.f : 1.f / ll;  // a NaN stays one
                if (direct) {
                    fa *= inv;
                    fb *= inv;
                }
                // a partial state goes to the CTA's slot, a whole unit's of a call with prefixes to its row's place
                float *st_o = p.slots + (static_cast<size_t>(blockIdx.x) * 2 + (d.flags >> 3 & 1)) * (N * (D + 2));
                const long long own = static_cast<long long>(a.total_q) * a.num_q_heads;
                if (w4 == 0 && lane < d.nrows) {
                    if (!whole) {
                        st_o[lane] = mm;
                        st_o[N + lane] = ll;
                    } else if (!direct) {
                        p.ml[own + out_row] = make_float2(mm, ll);
                    }
                }
                st_o = whole ? p.acc + (own + out0) * D : st_o + 2 * N;
                // each row's factors and place, in the room of the run's RowInfo
                __syncwarp();
                if (lane < N) info[lane] = RowInfo{ll == 0.f, whole ? static_cast<int>(out_row - out0) : lane, __float_as_int(fa), fb};
                __syncwarp();
                float oa[N], ob[N];
                tmem_ld<N>(t_o, oa);
                tmem_ld<N>(t_o + 16, ob);  // group 1's; not used where it had no tile
                tmem_wait_ld();
#pragma unroll
                for (int r = 0; r < N; ++r) {
                    const RowInfo w = info[r];
                    oa[r] *= __int_as_float(w.pos);
                    if (two) oa[r] = fmaf(ob[r], w.slope, oa[r]);
                    if (direct && w.lo) oa[r] = 0.f;  // nothing seen
                }
                if (direct) {
                    T *out = reinterpret_cast<T *>(a.out) + out0 * D + row;
#pragma unroll
                    for (int r = 0; r < N; ++r) {
                        if (r >= d.nrows) break;
                        if constexpr (kBf16)
                            out[static_cast<long long>(info[r].hi) * D] = __float2bfloat16_rn(oa[r]);
                        else
                            out[static_cast<long long>(info[r].hi) * D] = __float2half_rn(oa[r]);
                    }
                } else {
                    float *out = st_o + row;
#pragma unroll
                    for (int r = 0; r < N; ++r) {
                        if (r >= d.nrows) break;
                        out[static_cast<long long>(info[r].hi) * D] = oa[r];
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&o_free[0]);
                    if (two) mbar_arrive(&o_free[1]);
                }
            }
            ++ou[0];
            if (two) ++ou[1];
            c0 += 2 * n;
            if constexpr (Q8) sc0 = (sc0 + n) % L::kScales;
        }
        if (!ok && lane == 0) tile_give_up(abort);
    }

    // ---------------------------------------------------------------- teardown
    pdl_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, 64);
}

}  // namespace gk
