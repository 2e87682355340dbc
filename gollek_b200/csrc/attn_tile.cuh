// attn_tile.cuh -- ragged and shared-prefix paged attention on the 5th-generation tensor
// cores, for bf16 or f16 caches with head_dim 64 or 128 and queries of the same type.
//
// A block is up to 256 rows -- (query token, q head) pairs of one kv head -- over the
// positions [lo, hi) that any of them attends, in tiles of 128 positions:
//
//   S[128 rows x 128 pos] = Q . K^T        P = 2^(x - m), rounded to the cache's type
//   O[128 rows x D]      += P . V          l += sum P (fp32, unrounded)
//
// One thread owns one row, so its maximum m and sum l never leave its registers.  S and O
// live in tensor memory; P overwrites S there and feeds the value MMA as its A operand, so
// probabilities never touch shared memory.  P is rounded to 16 bits because both operands
// of that MMA have one type: a half step of P, averaged over the positions, is of the size
// of the output's own rounding.  m is a lazy maximum: it moves (and O is rescaled) only
// when a score passes it by more than 2^kLazyMax, which keeps P below 2^8.
//
// Two row groups of 128 threads keep the tensor core busy while the other computes its
// probabilities:
//   blocks of more than 128 rows: group t owns rows 128 t .., every tile serves both;
//   smaller blocks (decode, a chunk's tail): both groups own the same rows, group t the
//     tiles t, t + 2, ..., each with its own m, l and O, merged at the end of the run.
//
// Work: the plan kernel lays all tiles of all (block, kv head) units in one line, each unit
// behind kRunCost tiles' worth of start-up, and cuts it into one equal range per CTA (one
// CTA per SM).  A unit cut by a range end leaves partial (m, l, O) states, which the merge
// kernel joins in a fixed order: no atomics, the same bits every time.
//
// Bound by HBM where blocks are small (decode: each page is read once per kv head), by the
// tensor and exponent pipes for long prompts (both take about as long as the other: 128 x
// 128 x 128 MACs twice per tile against 16384 exponentials).
#pragma once

#include <climits>

#include "tcgen05.cuh"
#include "varlen.cuh"

namespace gk {

constexpr int kTileTok = 128;
constexpr int kBlkRows = 256;
constexpr int kRunCostTiles = 2;      // start-up of a run (q, pipeline fill, output), in tiles
constexpr int kMaxTileCtas = 160;
constexpr int kTileThreads = 384;     // 8 row warps, 1 MMA issuer, 1 producer, 2 idle
// Registers: launched with 168 a thread (384 x 168 = 64,512 of the SM's 65,536), of which the
// third warpgroup gives the row groups 40 each: 2 x 208 + 88 = 3 x 168.  A row thread holds a
// tile's 128 scores; at 168 it would spill 560 bytes.
constexpr int kRowRegs = 208, kAuxRegs = 88;
constexpr float kLazyMax = 8.f;

// A block: rows row0 .. row0 + nrows - 1 (row r: query token tok0 + r / G, q head h G + r % G)
// over positions [lo, hi) of table row `tab`, whose length is len.
struct TileBlk {
    int tab, tok0, row0, nrows, lo, hi, len, kind;
};
enum { kOwn = 0, kPrefix = 1, kSuffix = 2 };  // varlen; shared: the group's prefix, a sequence's own tokens

struct PlanHead {
    int nb;              // blocks
    int pad;
    long long total;     // cost line's length
    long long range;     // its share per CTA
};

// Workspace layout (byte offsets).
struct TileWs {
    size_t blks, cost, ents, slots, ml, acc, total;
    long long max_blocks;
};

__host__ __device__ inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Rows of all entities cut into blocks of 256: each entity leaves at most one short block.
inline TileWs tile_ws(long long entities, long long rows, long long out_rows, int D, bool shared) {
    TileWs w;
    w.max_blocks = rows / kBlkRows + entities;
    size_t o = 256;
    w.blks = o;
    o = up256(o + w.max_blocks * sizeof(TileBlk));
    w.cost = o;
    o = up256(o + (w.max_blocks + 1) * 8);
    w.ents = o;
    o = up256(o + (entities + 1) * 4);
    w.slots = o;
    o = up256(o + static_cast<size_t>(kMaxTileCtas) * 2 * kBlkRows * (D + 2) * 4);
    w.ml = o;
    if (shared) o = up256(o + out_rows * 4 * 4);  // (m, l) of the prefix and of the own tokens, per row
    w.acc = o;
    if (shared) o = up256(o + 2 * out_rows * D * 4);
    w.total = o;
    return w;
}

struct TileArgs {
    AttnArgs a;
    PlanHead *head;
    TileBlk *blks;
    long long *cost;  // [max_blocks + 1] start of each block's cost, per kv head
    int *ents;        // [entities + 1] first block of each entity
    float *slots;     // [CTA][2]: ml [2][256], O [256][D]
    float2 *ml;       // shared: [2][rows]
    float *acc;       // shared: [2][rows][D]
    int entities, grid, max_blocks;
    long long page_rows;
};

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;

// Exclusive scan of one value per thread; *total receives the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *warp_sums, T *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        T s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T n = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += n;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    const T before = warp ? warp_sums[warp - 1] : T(0);
    *total = warp_sums[31];
    __syncthreads();
    return before + incl - v;
}

// Entity e: the rows that share a table.  Varlen: sequence e.  Shared: group e's sequences
// over its prefix, then each sequence over its own tokens.
__device__ __forceinline__ int entity_tokens(const AttnArgs &a, int e) {
    int first, n;
    if (a.num_groups == 0)
        seq_rows(a, e, first, n);
    else if (e < a.num_groups)
        group_rows_of(a, e, first, n);
    else
        n = 1;
    return n;
}

__global__ void __launch_bounds__(kPlanThreads) tile_plan_kernel(const TileArgs p) {
    const AttnArgs &a = p.a;
    const int G = a.num_q_heads / a.num_kv_heads;
    const int tid = threadIdx.x;
    __shared__ long long sm_l[32];
    pdl_launch();

    // first block of every entity; sizes that do not fit their tables are reported once
    long long nb = 0;
    for (int e0 = 0; e0 < p.entities; e0 += kPlanThreads) {
        const int e = e0 + tid;
        long long blocks = 0;
        if (e < p.entities) {
            if (a.num_groups == 0)
                check_seq(a, e);
            else if (e < a.num_groups)
                check_group(a, e);
            else
                check_seq(a, e - a.num_groups);
            blocks = (static_cast<long long>(entity_tokens(a, e)) * G + kBlkRows - 1) / kBlkRows;
        }
        long long sum;
        const long long at = block_scan(blocks, sm_l, &sum);
        // the rows of entities that overlap (reported above) may be more than there is room for
        if (e < p.entities) p.ents[e] = static_cast<int>(min(nb + at, static_cast<long long>(p.max_blocks)));
        nb = min(nb + sum, static_cast<long long>(p.max_blocks));
    }
    if (tid == 0) p.ents[p.entities] = static_cast<int>(nb);
    __syncthreads();

    // blocks and their costs
    const bool docs = a.token_starts != nullptr;
    long long run = 0;
    for (int b0 = 0; b0 < nb; b0 += kPlanThreads) {
        const int b = b0 + tid;
        TileBlk k{};
        if (b < nb) {
            int lo = 0, hi = p.entities - 1;
            while (lo < hi) {  // last entity whose first block is <= b
                const int mid = (lo + hi + 1) >> 1;
                if (p.ents[mid] <= b)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            const int e = lo;
            int first, n;
            if (a.num_groups == 0) {
                seq_rows(a, e, first, n);
                k.kind = kOwn;
                k.tab = e;
                k.len = clamp_len(a, a.context_lens[e], a.max_blocks);
            } else if (e < a.num_groups) {
                group_rows_of(a, e, first, n);
                k.kind = kPrefix;
                k.tab = e;
                k.len = clamp_len(a, a.group_plens[e], a.max_pblocks);
            } else {
                k.kind = kSuffix;
                k.tab = e - a.num_groups;
                first = k.tab;
                n = 1;
                k.len = clamp_len(a, a.context_lens[k.tab], a.max_blocks);
            }
            k.tok0 = first;
            k.row0 = (b - p.ents[e]) * kBlkRows;
            k.nrows = static_cast<int>(min(static_cast<long long>(n) * G - k.row0, static_cast<long long>(kBlkRows)));
            k.lo = 0;
            k.hi = k.len;
            if (k.kind == kOwn) {
                const int i0 = k.row0 / G, i1 = (k.row0 + k.nrows - 1) / G;
                const int pos0 = k.len - n + i0, pos1 = k.len - n + i1;
                if (a.causal) {
                    k.hi = pos1 + 1;
                    if (a.prefix_lens) k.hi = max(k.hi, min(a.prefix_lens[e], k.len));
                }
                if (a.window > 0) k.lo = max(k.lo, pos0 - a.window + 1);
            }
        }
        if (docs) {  // one warp per block: the smallest first position of its queries
            const int lane = tid & 31;
            for (int u = 0; u < 32; ++u) {
                const int nrows = __shfl_sync(0xffffffffu, k.nrows, u);
                const int row0 = __shfl_sync(0xffffffffu, k.row0, u), tok0 = __shfl_sync(0xffffffffu, k.tok0, u);
                if (nrows <= 0) continue;
                const int i0 = row0 / G, i1 = (row0 + nrows - 1) / G;
                int least = INT_MAX;
                for (int i = i0 + lane; i <= i1; i += 32) least = min(least, a.token_starts[tok0 + i]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
                if (lane == u) k.lo = max(k.lo, least);
            }
        }
        long long c = 0;
        if (b < nb) {
            if (k.lo >= k.hi) k.lo = k.hi = 0;
            if (k.hi > k.lo) c = (k.hi + kTileTok - 1) / kTileTok - k.lo / kTileTok + kRunCostTiles;
            p.blks[b] = k;
        }
        long long sum;
        const long long at = block_scan(c, sm_l, &sum);
        if (b < nb) p.cost[b] = run + at;
        run += sum;
    }
    if (tid == 0) {
        p.cost[nb] = run;
        p.head->nb = static_cast<int>(nb);
        const long long total = run * a.num_kv_heads;
        p.head->total = total;
        p.head->range = max(1LL, (total + p.grid - 1) / p.grid);
    }
}

// ---------------------------------------------------------------------------- runs

// Consecutive tiles [ta, tb) of one (block, kv head) inside one CTA's range.
struct TileRun {
    TileBlk b;
    int h, ta, tb, n;  // n: tiles of the whole unit
};

__device__ __forceinline__ void run_tiles(long long v, long long len, int &ta, int &tb) {
    ta = static_cast<int>(max(0LL, v - kRunCostTiles));
    tb = static_cast<int>(max(0LL, v + len - kRunCostTiles));
}

// The last i in [0, nb) with cost[i] * hkv <= x (warp-collective).
__device__ __forceinline__ int find_block(const TileArgs &p, int nb, long long x) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = nb;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + lane * step;
        const bool le = at < hi && p.cost[at] * p.a.num_kv_heads <= x;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, le));  // lane 0 always holds
        hi = min(hi, lo + (k + 1) * step);
        lo = lo + k * step;
    }
    return lo;
}

// The runs of a CTA in order; every lane of a warp holds the same state.
struct RunIter {
    long long x, xe, base, m;
    int i, hkv;
    TileBlk b;

    __device__ __forceinline__ void load(const TileArgs &p) {
        const long long c0 = p.cost[i];
        base = c0 * hkv;
        m = p.cost[i + 1] - c0;
        b = p.blks[i];
    }
    // warp-collective: finds the block that holds the range's first unit
    __device__ __forceinline__ void begin(const TileArgs &p, int cta) {
        const PlanHead hd = *p.head;
        hkv = p.a.num_kv_heads;
        x = min(static_cast<long long>(cta) * hd.range, hd.total);
        xe = min(x + hd.range, hd.total);
        i = 0;
        if (x >= xe) return;
        i = find_block(p, hd.nb, x);
        load(p);
    }
    __device__ __forceinline__ bool next(const TileArgs &p, TileRun &r) {
        while (x < xe) {
            while (x >= base + m * hkv) {
                ++i;
                load(p);
            }
            const long long y = x - base;
            r.h = static_cast<int>(y / m);
            const long long v = y - r.h * m;
            const long long len = min(m - v, xe - x);
            x += len;
            run_tiles(v, len, r.ta, r.tb);
            if (r.ta < r.tb) {
                r.b = b;
                r.n = static_cast<int>(m) - kRunCostTiles;
                return true;
            }
        }
        return false;
    }
};

// ---------------------------------------------------------------------------- tile kernel

template <int D>
struct TileSmem {
    static constexpr uint32_t kSlot = kTileTok * D * 2;  // K or V of one tile
    static constexpr uint32_t kQ = 128 * D * 2;          // 128 rows
    static constexpr int kSlots = D == 128 ? 5 : 10;
    static constexpr uint32_t q = 0;
    static constexpr uint32_t ring = 2 * kQ;
    static constexpr uint32_t ml = ring + kSlots * kSlot;  // [2 runs][2][128] floats
    static constexpr uint32_t bars = ml + 2 * 2 * 128 * 4;
    static constexpr int kBars = 2 * kSlots + 2 * 6 + 2;
    static constexpr uint32_t misc = bars + kBars * 8;
    static constexpr uint32_t total = misc + 16;
};

// Bounded wait of a whole warp: each lane tests on its own, one vote at the end (the
// result is warp-uniform); gives up once another warp did.
__device__ __forceinline__ bool tile_wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    bool ok = mbar_try_wait(bar, parity);
    for (unsigned i = 0; !ok && i < kSuspendTries; ++i) {
        if (*abort) break;
        ok = mbar_try_wait_suspend(bar, parity, kSuspendNs);
        if (!ok && i + 1 == kSuspendTries) raise_status(GOLLEK_STATUS_TIMEOUT);
    }
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}

// D[tmem] (+)= A[tmem] * B, issued by one thread.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}

// One lane of the converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// Byte offset of 16-byte chunk ch (elements 8 ch ..) of token tok in a K or V tile: 8-token
// core groups of D/64 slabs [8 tokens][128 bytes], 128-byte swizzle.
template <int D>
__device__ __forceinline__ uint32_t kv_chunk_off(int tok, int ch) {
    const int r8 = tok & 7;
    return static_cast<uint32_t>((tok >> 3) * (16 * D) + (ch >> 3) * 1024 + r8 * 128 + (((ch & 7) ^ r8) << 4));
}

// Page lookups and TMA boxes of a run's tiles: lane g < 8 owns the 16 positions 16 g .. of
// each tile (one box; two of 8 rows where pages hold 8).
struct PageLoc {
    int row0, row1;  // first pool row of the box / 8, or -1
};

// Ring positions, from the run's first, of K and V of tile j of n: a value product follows
// the scores of the next tile, so V is copied behind the next K and waits less for its use.
__device__ __forceinline__ int k_at(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_at(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const TileArgs p) {
    using L = TileSmem<D>;
    constexpr int NS = L::kSlots;
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    const AttnArgs &a = p.a;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    uint8_t *smem = tile_smem;
    const uint32_t q_s = smem_u32(smem + L::q);
    uint8_t *ring = smem + L::ring;
    float *sm_ml = reinterpret_cast<float *>(smem + L::ml);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::bars);
    uint64_t *empty = full + NS;
    uint64_t *s_full = empty + NS;  // [2] scores in tensor memory (and every earlier MMA done)
    uint64_t *p_full = s_full + 2;  // [2] probabilities in tensor memory (V cleared, O rescaled)
    uint64_t *o_full = p_full + 2;  // [2] a run's last value MMA of the group done
    uint64_t *o_free = o_full + 2;  // [2] O read
    uint64_t *q_full = o_free + 2;  // [2] q staged in buffer 0, 1
    uint64_t *ml_full = q_full + 2; // group 1's (m, l) handed over
    uint64_t *p_half = ml_full + 1; // [2] probabilities of the tile's first 64 positions
    uint64_t *drained = p_half + 2;
    volatile int *abort = reinterpret_cast<volatile int *>(smem + L::misc);
    uint32_t *sm_tmem = reinterpret_cast<uint32_t *>(smem + L::misc + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.num_q_heads / a.num_kv_heads;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_half[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_free[t], 4);
            mbar_init(&q_full[t], 4);
        }
        mbar_init(ml_full, 4);
        mbar_init(drained, 1);
        fence_barrier_init();
        *abort = 0;
    }
    if (warp == 9 && lane == 0) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(sm_tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *sm_tmem;
    pdl_wait();  // the plan is complete

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAuxRegs));
        RunIter it;
        it.begin(p, blockIdx.x);
        TileRun r;
        if (warp == 9) {
            // ===================================================================== producer
            // Tiles of all runs in one line, the page lookups two tiles ahead of the copies (so a run's
            // first pages are known before the last ones of the run in front have a slot).
            struct Step {
                PageLoc loc;
                bool live, first, last;
            };
            const int R = a.block_size < 16 ? a.block_size : 16, per = 16 / R;
            const int *bt = nullptr;
            int t = 0, tb = 0, ta = 0;
            auto step = [&]() {
                Step s{{-1, -1}, false, false, false};
                if (t >= tb) {
                    if (!it.next(p, r)) return s;
                    bt = r.b.kind == kPrefix ? a.prefix_tables + static_cast<long long>(r.b.tab) * a.max_pblocks
                                             : a.block_tables + static_cast<long long>(r.b.tab) * a.max_blocks;
                    t = ta = r.ta;
                    tb = r.tb;
                }
                s.live = true;
                s.first = t == ta;
                s.last = t == tb - 1;
                // pool rows / 8 of the lane's box(es); -1: nothing to load there
                const int pos = (r.b.lo / kTileTok + t) * kTileTok + lane * 16;
                auto row8 = [&](int at) {
                    if (lane >= 8 || at >= r.b.hi || at + R <= r.b.lo) return -1;
                    const int pg = at / a.block_size;
                    int e = __ldg(bt + pg);
                    if (e < 0 || (a.num_blocks > 0 && e >= a.num_blocks)) {
                        raise_status(GOLLEK_STATUS_BAD_BLOCK_ID);
                        e = 0;
                    }
                    return static_cast<int>((e * p.page_rows + static_cast<long long>(r.h) * a.block_size +
                                             (at - pg * a.block_size)) >> 3);
                };
                s.loc.row0 = row8(pos);
                if (per == 2) s.loc.row1 = row8(pos + R);
                ++t;
                return s;
            };
            int c = 0;  // ring position
            auto copy = [&](const PageLoc &l, const CUtensorMap *map) {
                const int slot = c % NS;
                if (c >= NS && !tile_wait(&empty[slot], (c / NS - 1) & 1, abort)) return false;
                const unsigned boxes = (l.row0 >= 0) + (l.row1 >= 0);
                const uint32_t bytes = __reduce_add_sync(0xffffffffu, boxes) * R * D * 2;
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], bytes);
                __syncwarp();
                uint8_t *dst = ring + slot * L::kSlot + lane * (16 * D * 2);
                if (l.row0 >= 0) tma_load_4d(dst, map, 0, 0, 0, l.row0, &full[slot]);
                if (l.row1 >= 0) tma_load_4d(dst + R * D * 2, map, 0, 0, 0, l.row1, &full[slot]);
                ++c;
                return true;
            };
            // ring order of a run: K0, K1, V0, K2, V1, ... V(n-1) (k_at, v_at)
            bool ok = true;
            Step s0 = step(), s1 = step();
            PageLoc before{-1, -1};
            while (ok && s0.live) {
                const Step s2 = step();
                ok = copy(s0.loc, &tm_k);
                if (ok && !s0.first) ok = copy(before, &tm_v);
                if (ok && s0.last) ok = copy(s0.loc, &tm_v);
                before = s0.loc;
                s0 = s1;
                s1 = s2;
            }
            if (!ok && lane == 0) *abort = 1;
            // every copy issued lands before the shared memory is released
            if (lane == 0)
                for (int k = max(0, c - NS); k < c; ++k) mbar_wait(&full[k % NS], (k / NS) & 1);
            __syncwarp();
        } else if (warp == 8) {
            // ===================================================================== MMA issuer
            // The whole warp walks the tiles with warp-uniform values (so descriptors stay in uniform
            // registers) and one elected lane issues: a lane that computed descriptors on its own took
            // 2,300 cycles for the 16 MMAs of a step that run in about 1,000.
            constexpr uint32_t id_s = umma_idesc_16bit(128, kTileTok, kBf16, 0, 0);
            constexpr uint32_t id_o = umma_idesc_16bit(128, D, kBf16, 0, 1);
            const uint64_t q_desc = umma_desc_sw128(q_s, 16, 1024);
            const uint64_t k_desc = umma_desc_sw128(smem_u32(ring), 16, 16 * D);
            const uint64_t v_desc = umma_desc_sw128(smem_u32(ring), 1024, 16 * D);
            const bool leader = elect_one();
            int c0 = 0;                   // ring position of the run's first K
            int pp[2] = {0, 0};           // probabilities taken from group t so far
            int ou[2] = {0, 0};           // runs that used O of group t so far
            int qu[2] = {0, 0};           // fills of q buffer t consumed so far
            int qb = 1;                   // q buffer of the last small block; 1 after a large one
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t par) { return tile_wait(bar, par, abort); };
            auto commit = [&](uint64_t *bar) {
                if (leader) umma_commit(bar);
            };
            auto score = [&](int t, int buf, int c) {
                const int slot = __shfl_sync(0xffffffffu, c % NS, 0);
                const uint64_t qd = q_desc + buf * (L::kQ >> 4), kd = k_desc + slot * (L::kSlot >> 4);
                const uint32_t d = tmem + 128 * t;
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        umma_f16(d, qd + (kk >> 2) * (16384 >> 4) + (kk & 3) * 2, kd + (kk >> 2) * (1024 >> 4) + (kk & 3) * 2,
                                 id_s, kk > 0);
                    umma_commit(&s_full[t]);
                }
            };
            // O += P V of group t with V of ring position c, in two halves as P arrives; O is free
            // first (its last user's run has read it)
            auto value = [&](int t, int c, bool first) {
                const int slot = __shfl_sync(0xffffffffu, c % NS, 0);
                const uint64_t vd = v_desc + slot * (L::kSlot >> 4);
                const uint32_t d = tmem + 256 + 128 * t, pa = tmem + 128 * t;
                if (first && ou[t] > 0 && !wait(&o_free[t], (ou[t] - 1) & 1)) return false;
                if (!wait(&full[slot], (c / NS) & 1)) return false;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait(half ? &p_full[t] : &p_half[t], pp[t] & 1)) return false;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                            umma_f16_ts(d, pa + 8 * kk, vd + kk * (32 * D >> 4), id_o, !(first && kk == 0));
                    }
                }
                ++pp[t];
                return true;
            };
            while (ok && it.next(p, r)) {
                const int n = r.tb - r.ta;
                if (r.b.nrows > 128) {
                    // tile j: the values of j - 1 and the scores of j of each group in turn
#pragma unroll
                    for (int t = 0; t < 2; ++t) ok = ok && wait(&q_full[t], qu[t]++ & 1);
                    for (int j = 0; ok && j <= n; ++j) {
                        const int ck = c0 + k_at(j), cv = c0 + v_at(j - 1, n);
                        if (j < n) ok = wait(&full[ck % NS], (ck / NS) & 1);
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (!ok) break;
                            if (j > 0) {
                                ok = value(t, cv, j == 1);
                                if (!ok) break;
                                if (j == n) commit(&o_full[t]);
                            }
                            tc_fence_after();
                            if (j < n) score(t, t, ck);
                        }
                        if (!ok) break;
                        if (j > 0) commit(&empty[cv % NS]);
                        if (j < n) commit(&empty[ck % NS]);
                    }
                    ++ou[0];
                    ++ou[1];
                    qb = 1;
                } else {
                    // tile j belongs to group j & 1: its scores follow the values of j - 2
                    qb ^= 1;
                    ok = qb ? wait(&q_full[1], qu[1]++ & 1) : wait(&q_full[0], qu[0]++ & 1);
                    for (int j0 = 0; ok && j0 < n + 2; j0 += 2) {
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int j = j0 + t;
                            if (!ok) break;
                            if (j >= 2 && j - 2 < n) {
                                const int cv = c0 + v_at(j - 2, n);
                                ok = value(t, cv, j - 2 < 2);
                                if (!ok) break;
                                if (j >= n) commit(&o_full[t]);
                                commit(&empty[cv % NS]);
                            }
                            if (j < n) {
                                const int ck = c0 + k_at(j);
                                ok = wait(&full[ck % NS], (ck / NS) & 1);
                                if (!ok) break;
                                tc_fence_after();
                                score(t, qb, ck);
                                commit(&empty[ck % NS]);
                            }
                        }
                    }
                    ++ou[0];
                    if (n > 1) ++ou[1];
                }
                c0 += 2 * n;
            }
            if (!ok && lane == 0) *abort = 1;
            // every MMA issued has completed before tensor memory and shared memory go
            if (leader) {
                umma_commit(drained);
                mbar_wait(drained, 0);
            }
            __syncwarp();
        }
    } else {
        // ===================================================================== row groups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
        RunIter it;
        it.begin(p, blockIdx.x);
        TileRun r;
        const int t = warp >> 2;           // group
        const int row = tid & 127;         // row of the group = tensor-memory lane
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + 128 * t + lanes, t_o = tmem + 256 + 128 * t + lanes;
        const bool cap = a.soft_cap > 0.f, biased = a.slopes != nullptr;
        const bool scaled = cap || biased || !(a.q_scale > 0.f);  // scores enter the exponent domain early
        const float f = scaled ? 1.f : a.q_scale;
        const float cap1 = cap ? 2.f * kLog2e * a.q_scale / a.soft_cap : 0.f, cap2 = a.soft_cap * kLog2e;
        int c0 = 0, sn = 0;
        int qb = 0;                        // small blocks: q buffer (0 behind a large block, then in turn)
        int ou[2] = {0, 0};                // runs that used O of group 0, 1 so far
        int mln = 0;                       // small blocks of more than one tile so far
        auto wait = [&](uint64_t *bar, int phase) { return tile_wait(bar, phase & 1, abort); };

        // 128 rows of q from row `first` of the run's block into buffer `buf`
        auto fill = [&](const TileRun &u, int buf, int first) {
            constexpr int CH = D / 8;  // 16-byte chunks of a row
            const uint32_t dst = q_s + buf * L::kQ;
            const int live = min(u.b.nrows - first, 128);
#pragma unroll 8
            for (int k = 0; k < CH; ++k) {
                const int i = row + 128 * k, rr = i / CH, ch = i % CH;
                if (rr >= live) continue;
                const int rho = u.b.row0 + first + rr;
                const long long tok = u.b.tok0 + rho / G;
                const uint4 *src = reinterpret_cast<const uint4 *>(
                    reinterpret_cast<const T *>(a.q) + (tok * a.num_q_heads + u.h * G + rho % G) * D);
                sts_u4(dst + (ch >> 3) * 16384 + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4), __ldg(src + ch));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[buf]);
        };

        // Bias, cap and mask of the tile at position t0: S becomes the score in the exponent domain
        // (scaled), -inf outside columns [jlo, jhi).
        auto rewrite = [&](int t0, int jlo, int jhi, bool masked, float slope, int pos) {
#pragma unroll 1
            for (int k = 0; k < 128; k += 32) {
                float v[32];
                tmem_ld<32>(t_s + k, v);
                tmem_wait_ld();
                if (cap) {
                    // cap tanh(y) = cap - 2 cap / (1 + e^2y): absolute error about 2^-22 cap
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        v[i] = fmaf(-2.f * cap2, __fdividef(1.f, 1.f + fast_exp2(v[i] * cap1)), cap2);
                } else if (scaled) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] *= a.q_scale;
                }
                if (biased) {
                    const float d0 = static_cast<float>(t0 + k - pos);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = fmaf(-slope, fabsf(d0 + static_cast<float>(i)), v[i]);
                }
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = (i >= jlo - k && i < jhi - k) ? v[i] : -INFINITY;
                }
                tmem_st32(t_s + k, v);
            }
            tmem_wait_st();
        };

        bool ok = true;
        bool have = it.next(p, r);
        if (have) {
            if (r.b.nrows > 128)
                fill(r, t, 128 * t);
            else if (t == 0)
                fill(r, 0, 0);
        }
        while (have) {
            const int n = r.tb - r.ta;
            const bool big = r.b.nrows > 128;
            TileRun u = r;  // the next run
            const bool more = it.next(p, u);
            const bool ubig = more && u.b.nrows > 128;
            const int qn = big ? 0 : (qb ^ 1);
            const int ri = big ? 128 * t + row : row;  // row of the block
            const bool live = ri < r.b.nrows;
            // the row's query, its positions [lo, hi) and its bias
            long long out_row = 0;
            int lo = 0, hi = 0, pos = 0;
            float slope = 0.f;
            if (live) {
                const int rho = r.b.row0 + ri, i = rho / G, head = r.h * G + rho % G;
                out_row = static_cast<long long>(r.b.tok0 + i) * a.num_q_heads + head;
                lo = r.b.lo;
                hi = r.b.hi;
                if (r.b.kind == kOwn) {
                    int q0, nq;
                    seq_rows(a, r.b.tab, q0, nq);
                    pos = r.b.len - nq + i;
                    row_range(a, r.b.tab, q0 + i, pos, r.b.len, lo, hi);
                    if (biased) slope = a.slopes[head] * kLog2e;
                }
            }
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int tile0 = r.b.lo / kTileTok + r.ta;
            float m = -INFINITY, l = 0.f;

            for (int j = big ? 0 : t; j < n; j += big ? 1 : 2) {
                const int t0 = (tile0 + j) * kTileTok;
                const int jlo = lo - t0, jhi = hi - t0;  // visible columns [jlo, jhi)
                ok = wait(&s_full[t], sn++);
                if (!ok) break;
                tc_fence_after();
                // V rows that no row of the block attends are cleared (a zero probability does not
                // cancel a NaN): by group 0 for both groups, or by the tile's own group
                const int vlo = r.b.lo - t0, vhi = r.b.hi - t0;
                if ((vlo > 0 || vhi < kTileTok) && (t == 0 || !big)) {
                    const int cv = c0 + v_at(j, n);
                    ok = wait(&full[cv % NS], cv / NS);
                    if (!ok) break;
                    const uint32_t vt = smem_u32(ring) + (cv % NS) * L::kSlot;
                    for (int i = row; i < kTileTok * (D / 8); i += 128) {
                        const int tok = i / (D / 8);
                        if (tok < vlo || tok >= vhi) sts_u4(vt + kv_chunk_off<D>(tok, i % (D / 8)), make_uint4(0, 0, 0, 0));
                    }
                    fence_proxy_async_smem();
                }
                // Short loops: the code of a tile has to fit the instruction cache closest to the warp
                // (fully unrolled over the 128 columns it ran a third slower).
                float ref = 0.f;
                if (warp_live) {
                    // bias, cap and mask, where a tile has any: the scores are rewritten in place
                    const bool masked = __any_sync(0xffffffffu, live && (jlo > 0 || jhi < kTileTok));
                    if (scaled || masked) rewrite(t0, jlo, jhi, masked, slope, pos);
                    // pass 1: the row's largest score
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    float va[16], vb[16];
                    auto largest = [&](const float (&v)[16]) {
#pragma unroll
                        for (int i = 0; i < 16; i += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fmaxf(v[i + e], v[i + e + 4]));
                    };
                    tmem_ld<16>(t_s, va);
#pragma unroll 1
                    for (int k = 0; k < 128; k += 32) {
                        tmem_wait_ld();
                        tmem_ld<16>(t_s + k + 16, vb);
                        largest(va);
                        tmem_wait_ld();
                        tmem_ld<16>(t_s + (k + 32 & 127), va);  // the last one reads the first columns for pass 2
                        largest(vb);
                    }
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * f;
                    const bool move = live && (m == -INFINITY ? top > -INFINITY : top > m + kLazyMax);
                    if (__any_sync(0xffffffffu, move)) {
                        const float mn = move ? top : m;
                        const float alpha = (mn == m || m == -INFINITY) ? 1.f : fast_exp2(m - mn);
                        m = mn;
                        l *= alpha;
                        // the scores' commit covers the group's earlier value MMAs: O is at rest
                        if (__any_sync(0xffffffffu, alpha != 1.f)) {
                            tmem_wait_ld();
#pragma unroll 1
                            for (int k = 0; k < D / 32; ++k) {
                                float o[32];
                                tmem_ld<32>(t_o + 32 * k, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] *= alpha;
                                tmem_st32(t_o + 32 * k, o);
                            }
                        }
                    }
                    ref = m == -INFINITY ? 0.f : m;
                    // pass 2: P = 2^(x - m) over the columns read already, and its sum; the value MMA of
                    // the first 64 positions starts while the others are computed
                    float2 sum = make_float2(0.f, 0.f);
                    const float2 ff = make_float2(f, f), rr = make_float2(-ref, -ref);
                    auto probs = [&](const float (&v)[16], uint32_t (&pk)[16], int at) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float2 x = fma2(make_float2(v[2 * i], v[2 * i + 1]), ff, rr);
                            x.x = fast_exp2(x.x);
                            x.y = fast_exp2(x.y);
                            sum = add2(sum, x);
                            pk[at + i] = pack2<T>(x.x, x.y);
                        }
                    };
#pragma unroll 1
                    for (int k = 0; k < 128; k += 32) {
                        uint32_t pk[16];
                        tmem_wait_ld();
                        tmem_ld<16>(t_s + k + 16, vb);
                        probs(va, pk, 0);
                        tmem_wait_ld();
                        if (k < 96) tmem_ld<16>(t_s + k + 32, va);
                        probs(vb, pk, 8);
                        tmem_st16(t_s + (k >> 1), pk);
                        if (k == 32) {
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&p_half[t]);
                        }
                    }
                    tmem_wait_st();
                    l += sum.x + sum.y;
                } else if (lane == 0) {
                    mbar_arrive(&p_half[t]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
                // this tile's scores came behind every score of the run in front: its q buffer is free
                if (j == 0 && t == 0 && more && !big && !ubig) fill(u, qn, 0);
            }
            if (!ok) break;

            // The next run's q.  Behind a small run, both groups read one buffer: a large run's fills
            // wait for the end (`late`), a small one's took the other buffer after the first tile.
            const bool late = !big && ubig;
            if (more && big) {
                if (ubig)
                    fill(u, t, 128 * t);
                else if (t == 0)
                    fill(u, 0, 0);
            }

            // ------------------------------------------------ end of the run
            const bool whole = r.ta == 0 && r.tb == r.n;
            const bool two = !big && n > 1;  // both groups hold a part of each row
            if (two && t == 1) {
                float *ml = sm_ml + (mln & 1) * 256;  // group 0 of the run before the last has read it
                ml[row] = m;
                ml[128 + row] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(ml_full);
            }
            if (big || t == 0) {
                ok = wait(&o_full[t], ou[t]);
                float fa = 1.f, fb = 0.f;
                if (ok && two) {
                    ok = wait(&o_full[1], ou[1]) && wait(ml_full, mln);
                    if (ok) {
                        const float *ml = sm_ml + (mln & 1) * 256;
                        const float mb = ml[row], lb = ml[128 + row];
                        const float mm = fmaxf(m, mb);
                        fa = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - mm);
                        fb = mb == -INFINITY ? (lb == 0.f ? 0.f : 1.f) : fast_exp2(mb - mm);
                        l = l * fa + lb * fb;
                        m = mm;
                    }
                }
                if (!ok) break;
                tc_fence_after();
                if (warp_live) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
                    const bool direct = whole && r.b.kind == kOwn;
                    // where a partial state goes: the CTA's slot, or the row's place of a whole unit
                    float *st_o = nullptr;
                    if (!direct && live) {
                        if (whole) {
                            const long long at = (r.b.kind == kSuffix ? static_cast<long long>(a.total_q) * a.num_q_heads : 0) + out_row;
                            p.ml[at] = make_float2(m, l);
                            st_o = p.acc + at * D;
                        } else {
                            float *slot = p.slots + (static_cast<size_t>(blockIdx.x) * 2 + (r.ta == 0 ? 1 : 0)) * (kBlkRows * (D + 2));
                            slot[ri] = m;
                            slot[kBlkRows + ri] = l;
                            st_o = slot + 2 * kBlkRows + ri * D;
                        }
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int k = 0; k < D / 32; ++k) {
                        float o[32];
                        tmem_ld<32>(t_o + 32 * k, o);
                        if (two) {
                            float ob[32];
                            tmem_ld<32>(t_o + 128 + 32 * k, ob);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = fmaf(o[i], fa, ob[i] * fb);
                        } else {
                            tmem_wait_ld();
                        }
                        if (live && direct) {
                            uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + out_row * D + 32 * k);
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    w[e] = l == 0.f ? 0u : pack2<T>(o[8 * q + 2 * e] * inv, o[8 * q + 2 * e + 1] * inv);
                                dst[q] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else if (live) {
                            float4 *dst = reinterpret_cast<float4 *>(st_o + 32 * k);
#pragma unroll
                            for (int q = 0; q < 8; ++q) dst[q] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                        }
                        __syncwarp();  // the next tensor-memory load is the whole warp's
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&o_free[t]);
                    if (two) mbar_arrive(&o_free[1]);
                }
            }
            if (more && late) {
                if (t == 1) {
                    // every score MMA of this run is done
                    ok = wait(&o_full[0], ou[0]);
                    if (ok && two) ok = wait(&o_full[1], ou[1]);
                    if (!ok) break;
                }
                fill(u, t, 128 * t);
            }
            if (two) ++mln;
            ++ou[0];
            if (big || two) ++ou[1];
            c0 += 2 * n;
            qb = qn;
            r = u;
            have = more;
        }
        if (!ok && lane == 0) *abort = 1;
    }

    // ---------------------------------------------------------------- teardown
    pdl_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------- merge

// Partial states of one row, joined in the order of their positions: lane l holds columns
// l C .. l C + C - 1 (C = D / 32).
template <int C>
struct RowState {
    float m = -INFINITY, l = 0.f, o[C] = {};

    __device__ __forceinline__ void add(float m2, float l2, const float (&o2)[C]) {
        const float mm = fmaxf(m, m2);
        // a state without a maximum is empty (l = 0), or holds only NaN
        const float fa = m == -INFINITY ? 1.f : fast_exp2(m - mm);
        const float fb = m2 == -INFINITY ? 1.f : fast_exp2(m2 - mm);
        l = l * fa + l2 * fb;
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = l2 == 0.f ? o[i] * fa : fmaf(o[i], fa, o2[i] * fb);
        m = mm;
    }
};

template <int C>
__device__ __forceinline__ void load_cols(const float *src, int lane, float (&o)[C]) {
    if constexpr (C == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(src) + lane);
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
        const float2 v = __ldcg(reinterpret_cast<const float2 *>(src) + lane);
        o[0] = v.x, o[1] = v.y;
    }
}

// Adds row ri's state of the unit at [u0, u0 + m) of the cost line; false if one run held the
// whole unit (its state is then elsewhere).
template <int D>
__device__ __forceinline__ bool add_pieces(const TileArgs &p, long long range, long long u0, long long m, int ri, int lane,
                                           RowState<D / 32> &st) {
    constexpr int C = D / 32, B = 4;
    const long long n = m - kRunCostTiles, u1 = u0 + m;
    const long long b1 = (u1 - 1) / range;
    for (long long b = u0 / range; b <= b1; b += B) {
        float pm[B], pl[B], po[B][C];
#pragma unroll
        for (int k = 0; k < B; ++k) {  // B pieces' loads in flight
            pm[k] = -INFINITY;
            pl[k] = 0.f;
#pragma unroll
            for (int i = 0; i < C; ++i) po[k][i] = 0.f;
            const long long v0 = max((b + k) * range, u0) - u0, v1 = min((b + k + 1) * range, u1) - u0;
            if (b + k > b1) continue;
            int ta, tb;
            run_tiles(v0, v1 - v0, ta, tb);
            if (ta >= tb) continue;
            if (ta == 0 && tb == n) return false;
            const float *slot = p.slots + (static_cast<size_t>(b + k) * 2 + (ta == 0 ? 1 : 0)) * (kBlkRows * (D + 2));
            pm[k] = __ldcg(slot + ri);
            pl[k] = __ldcg(slot + kBlkRows + ri);
            load_cols<C>(slot + 2 * kBlkRows + ri * D, lane, po[k]);
        }
#pragma unroll
        for (int k = 0; k < B; ++k) st.add(pm[k], pl[k], po[k]);
    }
    return true;
}

template <typename T, int D>
__device__ __forceinline__ void write_row(const TileArgs &p, long long row, int lane, const RowState<D / 32> &st) {
    const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
    constexpr int C = D / 32;
    uint32_t w[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i) w[i] = st.l == 0.f ? 0u : pack2<T>(st.o[2 * i] * inv, st.o[2 * i + 1] * inv);
    T *dst = reinterpret_cast<T *>(p.a.out) + row * D + lane * C;
    if constexpr (C == 4)
        *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint32_t *>(dst) = w[0];
}

constexpr int kMergeThreads = 256;
constexpr int kMergeSplit = 8;

// Varlen.  CTA (c, y): rows y * 8 + warp, ... of the unit that starts in range c and goes on
// behind it; and zeros for the rows of blocks that attend nothing.
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) tile_merge_kernel(const TileArgs p) {
    const AttnArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.num_q_heads / a.num_kv_heads;
    pdl_wait();
    const PlanHead hd = *p.head;
    for (int b = blockIdx.y * gridDim.x + blockIdx.x; b < hd.nb; b += gridDim.x * gridDim.y) {
        if (p.cost[b + 1] != p.cost[b]) continue;
        const TileBlk k = p.blks[b];
        for (int i = warp; i < k.nrows * a.num_kv_heads; i += kMergeThreads / 32) {
            const int h = i / k.nrows, rho = k.row0 + i % k.nrows;
            write_row<T, D>(p, static_cast<long long>(k.tok0 + rho / G) * a.num_q_heads + h * G + rho % G, lane,
                            RowState<D / 32>());
        }
    }
    const long long x0 = blockIdx.x * hd.range, x1 = x0 + hd.range;
    if (x1 >= hd.total) return;
    const int i = find_block(p, hd.nb, x1 - 1);
    const long long c0 = p.cost[i], m = p.cost[i + 1] - c0;
    const int h = static_cast<int>((x1 - 1 - c0 * a.num_kv_heads) / m);
    const long long u0 = c0 * a.num_kv_heads + h * m;
    if (u0 + m <= x1 || u0 < x0) return;  // ends here, or started before
    const TileBlk k = p.blks[i];
    for (int r = blockIdx.y * (kMergeThreads / 32) + warp; r < k.nrows; r += kMergeSplit * (kMergeThreads / 32)) {
        RowState<D / 32> st;
        if (!add_pieces<D>(p, hd.range, u0, m, r, lane, st)) return;
        const int rho = k.row0 + r;
        write_row<T, D>(p, static_cast<long long>(k.tok0 + rho / G) * a.num_q_heads + h * G + rho % G, lane, st);
    }
}

// Shared prefixes.  One warp per (sequence, q head): the prefix's state, then the own tokens'.
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) tile_merge_shared_kernel(const TileArgs p) {
    const AttnArgs &a = p.a;
    const int lane = threadIdx.x & 31;
    const int G = a.num_q_heads / a.num_kv_heads;
    const long long rows = static_cast<long long>(a.num_seqs) * a.num_q_heads;
    pdl_wait();
    const PlanHead hd = *p.head;
    const long long row = static_cast<long long>(blockIdx.x) * (kMergeThreads / 32) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int s = static_cast<int>(row / a.num_q_heads), head = static_cast<int>(row % a.num_q_heads);
    const int h = head / G, g = head % G;
    RowState<D / 32> st;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        int e = a.num_groups + s;
        long long rho = g;
        if (part == 0) {
            e = group_of_seq(a, s);
            if (e < 0) continue;
            rho += static_cast<long long>(s - a.group_starts[e]) * G;
        }
        const long long i = p.ents[e] + rho / kBlkRows;
        if (i >= p.ents[e + 1]) continue;  // only where group_starts is not usable
        const long long c0 = p.cost[i], m = p.cost[i + 1] - c0;
        if (m == 0) continue;
        if (!add_pieces<D>(p, hd.range, c0 * a.num_kv_heads + h * m, m, static_cast<int>(rho % kBlkRows), lane, st)) {
            const long long at = part * rows + row;
            const float2 ml = p.ml[at];
            float o[D / 32];
            load_cols<D / 32>(p.acc + at * D, lane, o);
            st.add(ml.x, ml.y, o);
        }
    }
    write_row<T, D>(p, row, lane, st);
}

}  // namespace gk
