// attn_tile.cuh -- ragged and shared-prefix paged attention on the 5th-generation tensor
// cores, for bf16 or f16 caches with queries of the same type and int8 caches with bf16
// queries, head_dim 64 or 128: the plan, the kernel for blocks of many rows, the merge.
// attn_rows.cuh has the kernel for blocks of few.
//
// A block is up to 256 rows -- (query token, q head) pairs of one kv head -- over the
// positions [lo, hi) that any of them attends, in tiles of 128 positions, the last first:
//
//   S[128 rows x 128 pos] = Q . K^T        P = 2^(x - m), rounded to the cache's type
//   O[128 rows x D]      += P . V          l += sum P (fp32, unrounded)
//
// One thread owns one row, so its reference m and sum l never leave its registers.  S and O
// live in tensor memory; P overwrites S there and feeds the value MMA as its A operand, so
// probabilities never touch shared memory.  P is rounded to 16 bits because both operands
// of that MMA have one type: a half step of P, averaged over the positions, is of the size
// of the output's own rounding.  An int8 cache's scales multiply S (K's) and P (V's), never
// the integers, which would be one rounding more.  m is a lazy maximum: it moves, by a whole
// number, only when a score passes it by more than kLazyMax; l, O and the columns of P that
// stand already are then scaled by a power of two (exact but for f16's smallest numbers).
//
// Two row groups of 128 threads keep the tensor core busy while the other computes its
// probabilities:
//   blocks of more than 128 rows: group t owns rows 128 t .., every tile serves both;
//   smaller blocks (a chunk's tail): both groups own the same rows, group t the tiles t,
//     t + 2, ..., each with its own m, l and O, merged at the end of the run.
//
// Work: the plan kernel lays all tiles of all (block, kv head) units in one line, each unit
// behind kRunCostTiles tiles' worth of start-up, and cuts it into one equal range per CTA
// (one CTA per SM).  A unit cut by a range end leaves partial (m, l, O) states, which the
// merge kernel joins in a fixed order: no atomics, the same bits every time.  Plan and merge
// take about 6 us each, most of it a launch's latency.
//
// Bound, for long prompts, by the row groups' pass over S: 128 columns take a group about
// 1000 clocks of tensor-memory reads and as long again for the exponentials, where the two
// products take 512 each; two prompts of 2,000 tokens at 8,000 tokens of context (32 q, 8 kv
// heads of 128, distance bias) take 545 us, 0.87 PFLOP/s.  What moved it: scores read once
// (572 -> 532 us), groups that take turns at the exponentials (756 -> 522 us with one MMA
// issuer each and less code).  Code size counts: at 100 KB the roles evicted each other's
// instructions all the time, which the `unroll 1` loops and opaque() keep down to 60 KB.
#pragma once

#include <climits>

#include "tcgen05.cuh"
#include "varlen.cuh"

namespace gk {

constexpr int kTileTok = 128;
constexpr int kBlkRows = 256;
constexpr int kRunCostTiles = 2;      // start-up of a run (q, pipeline fill, output), in tiles
constexpr int kMaxTileCtas = 160;
constexpr int kTileThreads = 384;     // 8 row warps, 2 MMA issuers, 2 producers
constexpr int kTileThreadsQ8 = 512;   // int8 caches: a fourth warpgroup converts
// Scores may pass their row's reference by this much (log2 units) before it moves: P stays
// below the largest number of its type, and sums of it far below fp32's.
template <typename T>
constexpr float kLazyMax = std::is_same<T, __half>::value ? 15.f : 64.f;
// The reference is set this far below a maximum.  f16's smallest step is 2^-24: with P of 1 at the
// maximum, probabilities of 2^-25 and less would be lost, and thousands of them beside one large score
// are a share that shows.
template <typename T>
constexpr float kBelowMax = std::is_same<T, __half>::value ? 8.f : 0.f;

// A block: rows row0 .. row0 + nrows - 1 (row r: query token tok0 + r / G, q head h G + r % G)
// over positions [lo, hi) of table row `tab`, whose length is len.
// A varlen row's query i sits at position pos0 + i.
struct __align__(16) TileBlk {
    int tok0, row0, nrows, kind;
    int lo, hi, tab, len;
    int pos0, pad[3];
};
enum { kPlain = 0, kBias = 1, kCap = 2 };
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

// Rows of all entities cut into blocks of blk_rows: each entity leaves at most one short block.
inline TileWs tile_ws(long long entities, long long rows, int blk_rows, long long out_rows, int D, bool shared) {
    TileWs w;
    w.max_blocks = rows / blk_rows + entities;
    size_t o = 256;
    w.blks = o;
    o = up256(o + w.max_blocks * sizeof(TileBlk));
    w.cost = o;
    o = up256(o + (w.max_blocks + 1) * 8);
    w.ents = o;
    o = up256(o + (entities + 1) * 4);
    w.slots = o;
    o = up256(o + static_cast<size_t>(kMaxTileCtas) * 2 * blk_rows * (D + 2) * 4);
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
    float *slots;     // [CTA][2]: ml [2][blk_rows], O [blk_rows][D]
    float2 *ml;       // shared: [2][rows]
    float *acc;       // shared: [2][rows][D]
    int ent0, entities, grid, max_blocks;  // entities ent0 .. ent0 + entities - 1 of the call
    int blk_rows;     // rows a block may have
    int rows_min, rows_max;  // entities of rows_min .. rows_max rows are this line's, the rest another's
    long long page_rows;
    // Tests of the waits that give up (host: test_hooks): tests a wait may take, and the tiles
    // behind which CTA 0's producers stop (-1: none).
    unsigned wait_tries;
    int stop_at;
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

// Two lines at most, one per CTA: a call whose entities go to two kernels has one for each.
struct PlanArgs {
    TileArgs line[2];
};

__global__ void __launch_bounds__(kPlanThreads) tile_plan_kernel(const __grid_constant__ PlanArgs both) {
    const TileArgs &p = both.line[blockIdx.x];
    const AttnArgs &a = p.a;
    const int G = a.num_q_heads / a.num_kv_heads;
    const int tid = threadIdx.x;
    __shared__ long long sm_l[32];
    __shared__ int2 sm_rows[kPlanThreads];  // token_starts: first query token and tokens of a block
    __shared__ int sm_least[kPlanThreads];
    pdl_launch();

    // first block of every entity; sizes that do not fit their tables are reported once
    long long nb = 0;
    for (int e0 = 0; e0 < p.entities; e0 += kPlanThreads) {
        const int e = e0 + tid;
        long long blocks = 0;
        if (e < p.entities) {
            const int ent = p.ent0 + e;
            if (a.num_groups == 0)
                check_seq(a, ent);
            else if (ent < a.num_groups)
                check_group(a, ent);
            else
                check_seq(a, ent - a.num_groups);
            const long long rows = static_cast<long long>(entity_tokens(a, ent)) * G;
            if (rows >= p.rows_min && rows <= p.rows_max) blocks = (rows + p.blk_rows - 1) / p.blk_rows;
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
            const int e = p.ent0 + lo;
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
            k.row0 = (b - p.ents[lo]) * p.blk_rows;
            k.nrows = static_cast<int>(min(static_cast<long long>(n) * G - k.row0, static_cast<long long>(p.blk_rows)));
            k.lo = 0;
            k.hi = k.len;
            if (k.kind == kOwn) {
                const int i0 = k.row0 / G, i1 = (k.row0 + k.nrows - 1) / G;
                k.pos0 = k.len - n;
                const int pos0 = k.pos0 + i0, pos1 = k.pos0 + i1;
                if (a.causal) {
                    k.hi = pos1 + 1;
                    if (a.prefix_lens) k.hi = max(k.hi, min(a.prefix_lens[e], k.len));
                }
                if (a.window > 0) k.lo = max(k.lo, pos0 - a.window + 1);
            }
        }
        if (docs) {  // the smallest first position of each block's queries: a warp per block, all warps in turn
            sm_rows[tid] = make_int2(k.nrows > 0 ? k.tok0 + k.row0 / G : 0, k.nrows > 0 ? (k.row0 + k.nrows - 1) / G - k.row0 / G + 1 : 0);
            __syncthreads();
            const int lane = tid & 31, here = static_cast<int>(min(nb - b0, static_cast<long long>(kPlanThreads)));
#pragma unroll 4
            for (int u = tid >> 5; u < here; u += kPlanThreads / 32) {
                const int2 r = sm_rows[u];
                int least = INT_MAX;
                for (int i = lane; i < r.y; i += 32) least = min(least, a.token_starts[r.x + i]);
                least = __reduce_min_sync(0xffffffffu, least);
                if (lane == 0) sm_least[u] = least;
            }
            __syncthreads();
            if (k.nrows > 0) k.lo = max(k.lo, sm_least[tid]);
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
    long long x, xe, at, m;  // at: start of unit (block i, head h), m: its length
    int i, h, hkv;
    TileBlk b;

    __device__ __forceinline__ void load(const TileArgs &p) {
        m = p.cost[i + 1] - p.cost[i];
        b = p.blks[i];
    }
    // warp-collective: finds the unit that holds the range's first tile
    __device__ __forceinline__ void begin(const TileArgs &p, int cta) {
        const PlanHead hd = *p.head;
        hkv = p.a.num_kv_heads;
        x = min(static_cast<long long>(cta) * hd.range, hd.total);
        xe = min(x + hd.range, hd.total);
        if (x >= xe) return;
        i = find_block(p, hd.nb, x);
        load(p);
        const long long base = p.cost[i] * hkv;
        h = static_cast<int>((x - base) / m);
        at = base + h * m;
    }
    __device__ __forceinline__ bool next(const TileArgs &p, TileRun &r) {
        bool found = false;
#pragma unroll 1
        while (!found && x < xe) {
            const long long v = x - at, len = min(m - v, xe - x);
            run_tiles(v, len, r.ta, r.tb);
            found = r.ta < r.tb;
            r.b = b;
            r.h = h;
            r.n = static_cast<int>(m) - kRunCostTiles;
            x += len;
            if (x == at + m) {
                at = x;
                ++h;
#pragma unroll 1
                while (x < xe && (h == hkv || m == 0)) {  // the next block; one without tiles has no units
                    ++i;
                    h = 0;
                    load(p);
                }
            }
        }
        return found;
    }
};

// ---------------------------------------------------------------------------- tile kernel

// Q8: int8 caches.  Their tiles land as bytes in a ring of their own, four converter warps
// turn them into bf16 tiles (exact: integers below 2^8), and the scales, which enter the
// scores and the probabilities, are kept by tile: with 3 + 3 slots the copies are never
// more than 5 tiles ahead of a tile in use.
template <int D, bool Q8>
struct TileSmem {
    static constexpr uint32_t kSlot = kTileTok * D * 2;  // K or V of one tile
    static constexpr uint32_t kQ = 128 * D * 2;          // 128 rows
    static constexpr int kSlots = (Q8 ? 3 : 5) * (128 / D);
    static constexpr int kRaw = Q8 ? 3 * (128 / D) : 0;  // int8 tiles in flight
    static constexpr int kScales = Q8 ? 8 * (128 / D) : 0;  // tiles whose scales are kept
    static constexpr int kRuns = 4;                        // run descriptors in flight
    static constexpr uint32_t q = 0;
    static constexpr uint32_t ring = 2 * kQ;
    static constexpr uint32_t raw = ring + kSlots * kSlot;   // [kRaw][128][D] bytes
    static constexpr uint32_t scales = raw + kRaw * (kSlot / 2);  // [kScales][K, V][128] floats
    static constexpr uint32_t ones = scales + kScales * 1024;  // Q8: [128] floats of 1
    static constexpr uint32_t ml = ones + (Q8 ? 512 : 0);  // [2][128] floats
    static constexpr uint32_t runs = ml + 2 * 128 * 4;     // [kRuns] x 48 bytes
    static constexpr uint32_t bars = runs + kRuns * 48;
    static constexpr int kBars = 2 * kSlots + 2 * kRaw + 2 * kRuns + 2 * 7 + 8 + 1;
    static constexpr uint32_t misc = bars + kBars * 8;
    static constexpr uint32_t total = misc + 16;
};

// A run as the producer hands it to the other warps (in shared memory): n tiles of a
// block's rows (n = 0: no more runs), tile j from position 128 (tile0 - j).  The last
// positions come first: a causal row's largest scores, with a distance bias above all, lie
// near its own position, so the running maximum seldom moves after the first tile.
struct __align__(16) RunDesc {
    int tok0, row0, nrows, h;
    int lo, hi, tile0, n;
    int tab, len, pos0, flags;  // flags: kind, 4: the whole unit, 8: its first tiles
};

// Bounded wait of a whole warp: each lane tests on its own, one vote at the end (the
// result is warp-uniform); gives up once another warp did.  The warp that gives up first
// raises the status (tile_give_up) at the end of its role.  The number of tests allowed
// stands behind the abort flag.  One copy of the code for all waits: see opaque() on why size
// matters here.
__device__ __noinline__ bool tile_wait(uint32_t bar, uint32_t parity, uint32_t abort) {
    bool ok = false;
    uint32_t tries = 1;
#pragma unroll 1
    for (unsigned i = 0; !ok && i < tries; ++i) {
        uint32_t done, gone;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%3], %4, %6;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "ld.volatile.shared.v2.u32 {%1, %2}, [%5];\n\t}"
            : "=&r"(done), "=&r"(gone), "=&r"(tries)
            : "r"(bar), "r"(parity), "r"(abort), "r"(kSuspendNs)
            : "memory");
        ok = done != 0;
        if (gone) break;
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void tile_give_up(volatile int *abort) {
    if (*abort == 0) raise_status(GOLLEK_STATUS_TIMEOUT);
    *abort = 1;
}

template <typename T>
__device__ __forceinline__ void sts_u2(uint32_t addr, T v) {
    static_assert(sizeof(T) == 2, "two bytes");
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(reinterpret_cast<const unsigned short &>(v)) : "memory");
}

// 16 bytes (4 bytes) of global memory into shared memory, asynchronously.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// x / d for 0 <= x < 2^31: the magic's quotient is at most one too large.
__device__ __forceinline__ unsigned div_magic(int d) { return d == 1 ? 0u : 0xFFFFFFFFu / d + 1; }
__device__ __forceinline__ int fast_div(int x, int d, unsigned magic) {
    int q = d == 1 ? x : static_cast<int>(__umulhi(x, magic));
    return q * d > x ? q - 1 : q;
}

// A value the compiler cannot reason about.  Loops test their run-wide conditions through it:
// left to itself the compiler copies each loop once per condition, and the kernel's 100 KB of
// code then missed the instruction cache all the time.
__device__ __forceinline__ bool opaque(bool x) {
    int v = x;
    asm volatile("" : "+r"(v));
    return v != 0;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
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

// Two bytes of w (SEL: a prmt selector that puts each below a byte of 0x43) as signed
// integers in bf16.
template <unsigned SEL>
__device__ __forceinline__ uint32_t byte_pair(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x43434343u, SEL);
    uint32_t a = x & 0xFF7FFF7Fu, b = x & 0xFF80FF80u, d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// tanh(y) of two values: an odd polynomial on the FMA pipe for |y| <= 1/2, the usual case (caps are
// several times the scores), relative error 2^-25.9 (the minimax polynomial of tanh(y) / y in y^2
// under the relative error, by Remez exchange) ...
__device__ __forceinline__ float2 tanh_small(float2 y) {
    const float2 y2 = mul2(y, y);
    float2 q = fma2(y2, pair(0.01724149100482f), pair(-0.05304549261928f));
    q = fma2(q, y2, pair(0.13325878977776f));
    q = fma2(q, y2, pair(-0.33333143591881f));
    return fma2(mul2(q, y2), y, y);
}
// ... and 1 - 2 / (1 + e^2y), two exponent-pipe operations, beyond.
__device__ __forceinline__ float tanh_large(float y) {
    return fmaf(-2.f, __fdividef(1.f, 1.f + fast_exp2(y * (2.f * kLog2e))), 1.f);
}
// w = tanh(w) of a row's N scores of a tile (what the others become does not matter), in the way
// that the largest of those in `seen` needs: its bits depend on what the row attends alone.  Warp-
// collective.
template <int N>
__device__ __forceinline__ void unit_cap(float (&w)[N], unsigned seen) {
    if (opaque(__any_sync(0xffffffffu, seen != ~0u))) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = seen >> i & 1 ? w[i] : 0.f;
    }
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(w[i]));
    if (big > 0.5f) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = tanh_large(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 q = tanh_small(make_float2(w[i], w[i + 1]));
            w[i] = q.x;
            w[i + 1] = q.y;
        }
    }
    __syncwarp();
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

// What lane g of 4 copies of the 16 positions 16 g .. of a tile: two halves of 8, in one page or
// (pages of 8) in one each.  `entry`: the pages' table entries, looked up two tiles ahead;
// resolved one tile ahead.
struct PageEntry {
    int e0, e1, off0, off1;  // off < 0: nothing to load there
    int h;
};
struct PageLoc {
    int row0, row1;  // first pool row of the half / 8, or -1
};
// int8 caches: the first row itself, and where the half's scales are.
struct PageLocQ8 {
    long long row0, row1, sc0, sc1;
};

// Ring positions, from the run's first, of K and V of tile j of n: a value product follows
// the scores of the next tile, so V is copied behind the next K and waits less for its use.

__device__ __forceinline__ int v_at(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

// What the producer, the converters and the other roles of a kernel share; L names the places.
template <typename L>
struct TilePipe {
    uint8_t *smem;
    RunDesc *runs;
    uint64_t *full, *empty;        // [kSlots] tile in shared memory; read
    uint64_t *raw_full, *raw_free; // [kRaw] bytes of a tile (and, with K, its scales); converted
    uint64_t *run_full, *run_free; // [kRuns] descriptor written; read by the warps that use it
    uint64_t *own;                 // the kernel's own barriers
    volatile int *abort;

    __device__ __forceinline__ explicit TilePipe(uint8_t *base) : smem(base) {
        runs = reinterpret_cast<RunDesc *>(base + L::runs);
        full = reinterpret_cast<uint64_t *>(base + L::bars);
        empty = full + L::kSlots;
        raw_full = empty + L::kSlots;
        raw_free = raw_full + L::kRaw;
        run_full = raw_free + L::kRaw;
        run_free = run_full + L::kRuns;
        own = run_free + L::kRuns;
        abort = reinterpret_cast<volatile int *>(base + L::misc);
    }
    // by one thread; `fillers` warps arrive on full, `readers` on empty, `users` read a descriptor
    __device__ __forceinline__ void init(int fillers, int readers, int users, unsigned tries) const {
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(&full[i], fillers);
            mbar_init(&empty[i], readers);
        }
        for (int i = 0; i < L::kRaw; ++i) {
            mbar_init(&raw_full[i], 64);  // the two producers' lanes
            mbar_init(&raw_free[i], fillers);
        }
        for (int i = 0; i < L::kRuns; ++i) {
            mbar_init(&run_full[i], 1);
            mbar_init(&run_free[i], users);
        }
        abort[0] = 0;
        abort[1] = tries;  // ([2]: the tensor memory's address)
    }
    // by a whole warp; the call is left to waits that have something to wait for (it takes some
    // 350 clocks)
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t phase) const {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(phase & 1)
            : "memory");
        if (__all_sync(0xffffffffu, done)) return true;
        return tile_wait(smem_u32(bar), phase & 1, smem_u32(smem + L::misc));
    }
};

// Two warps walk the runs and copy half of each tile, part 0 the first 64 positions; it also
// hands the runs' descriptors out.  The page lookups go two tiles ahead of the copies, across
// runs.  One warp alone, at some 90 clocks a box, and a lookup that waited for its table entry
// were what bounded decode (229 -> 185 us for 64 sequences of 512 to 8192 tokens, 32 q and 8 kv heads).
template <typename L, int D, bool Q8>
__device__ __forceinline__ void tile_producer(const TileArgs &p, const TilePipe<L> &pipe, const CUtensorMap &tm_k,
                                              const CUtensorMap &tm_v, int lane, int part) {
    constexpr int NS = L::kSlots;
    const AttnArgs &a = p.a;
    uint64_t *const full = pipe.full, *const empty = pipe.empty, *const run_full = pipe.run_full, *const run_free = pipe.run_free;
    [[maybe_unused]] uint64_t *const raw_full = pipe.raw_full, *const raw_free = pipe.raw_free;
    RunDesc *const runs = pipe.runs;
    volatile int *const abort = pipe.abort;
    auto wait = [&](uint64_t *bar, uint32_t phase) { return pipe.wait(bar, phase); };
    pdl_wait();  // the plan is complete
    RunIter it;
    it.begin(p, blockIdx.x);
    TileRun r{};
    using Loc = std::conditional_t<Q8, PageLocQ8, PageLoc>;
    struct Step {
        PageEntry at;
        Loc loc;
        bool live, first, last;
    };
    const int R = a.block_size < 16 ? a.block_size : 16;
    const unsigned bs_magic = div_magic(a.block_size);
    const int *bt = nullptr;
    int t = 0, tb = 0, ta = 0, nrun = 0;
    int slot = 0, copies = 0;
    uint32_t ph = 1;
    bool ok = true, more = true;
    Step s0{{0, 0, -1, -1, 0}, {-1, -1}, false, false, false}, s1 = s0;
    Loc before{-1, -1};
    [[maybe_unused]] int sc_slot = 0;  // scales of the tile copied next
    // ring order of a run: K0, K1, V0, K2, V1, ... V(n-1) (v_at).  The first two rounds only fill
    // the look-ahead; each part of the code stands here once, to keep it short.
#pragma unroll 1
    for (int round = 0; ok && (round < 2 || s0.live); ++round) {
        Step s2{{0, 0, -1, -1, 0}, {-1, -1}, false, false, false};
        if (t >= tb && more) {
            // the next run: its descriptor for the other warps, its table
            more = it.next(p, r);
            const int at = nrun % L::kRuns;
            if (nrun >= L::kRuns) ok = wait(&run_free[at], nrun / L::kRuns - 1);
            if (part == 0 && lane == 0 && ok) {
                RunDesc &d = runs[at];
                d.tok0 = r.b.tok0;
                d.row0 = r.b.row0;
                d.nrows = r.b.nrows;
                d.h = r.h;
                d.lo = r.b.lo;
                d.hi = r.b.hi;
                d.tile0 = r.b.lo / kTileTok + r.tb - 1;
                d.n = more ? r.tb - r.ta : 0;
                d.tab = r.b.tab;
                d.len = r.b.len;
                d.pos0 = r.b.pos0;
                d.flags = r.b.kind | (r.ta == 0 && r.tb == r.n ? 4 : 0) | (r.ta == 0 ? 8 : 0);
                mbar_arrive(&run_full[at]);
            }
            __syncwarp();
            ++nrun;
            bt = r.b.kind == kPrefix ? a.prefix_tables + static_cast<long long>(r.b.tab) * a.max_pblocks
                                     : a.block_tables + static_cast<long long>(r.b.tab) * a.max_blocks;
            t = ta = r.ta;
            tb = more ? r.tb : r.ta;
            if (p.stop_at >= 0 && blockIdx.x == 0) {
                tb = min(tb, ta + p.stop_at);
                more = false;
            }
        }
        if (t < tb) {
            s2.live = true;
            s2.first = t == ta;
            s2.last = t == r.tb - 1;
            const int at = (r.b.lo / kTileTok + r.tb - 1 - (t - ta)) * kTileTok + lane * 16;
            s2.at.h = r.h;
            // (straight-line, so that nothing waits for an entry before it is resolved)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int p0 = at + 8 * k;  // a page of 16 positions or more is copied 16 at a time
                if (lane >> 2 != part || (R == 16 ? at >= r.b.hi || at + 16 <= r.b.lo : p0 >= r.b.hi || p0 + 8 <= r.b.lo))
                    continue;
                const int pg = fast_div(p0, a.block_size, bs_magic);
                (k ? s2.at.off1 : s2.at.off0) = p0 - pg * a.block_size;
                if (k == 0 || R == 8) (k ? s2.at.e1 : s2.at.e0) = __ldg(bt + pg);
            }
            __syncwarp();
            ++t;
        }
        // the next tile's entries, here by now, to rows
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            int e = k == 0 || R == 16 ? s1.at.e0 : s1.at.e1;
            const int off = k ? s1.at.off1 : s1.at.off0;
            if (off < 0) continue;
            if (e < 0 || (a.num_blocks > 0 && e >= a.num_blocks)) {
                raise_status(GOLLEK_STATUS_BAD_BLOCK_ID);
                e = 0;
            }
            const long long first = e * p.page_rows + static_cast<long long>(s1.at.h) * a.block_size + off;
            if constexpr (Q8) {
                (k ? s1.loc.row1 : s1.loc.row0) = first;
                (k ? s1.loc.sc1 : s1.loc.sc0) =
                    e * a.scale_page_stride + s1.at.h * a.scale_head_stride + off * a.scale_token_stride;
            } else if (k == 0 || R == 8) {
                (k ? s1.loc.row1 : s1.loc.row0) = static_cast<int>(first >> 3);
            }
        }
        __syncwarp();
        // K of this tile, V of the tile before it in the run, V of the run's last tile
#pragma unroll 1
        for (int w = 0; w < 3 && s0.live && ok; ++w) {
            if ((w == 1 && s0.first) || (w == 2 && !s0.last)) continue;
            const Loc l = w == 1 ? before : s0.loc;
            constexpr int kRing = Q8 ? L::kRaw : NS;
            uint64_t *const r_full = Q8 ? raw_full : full, *const r_free = Q8 ? raw_free : empty;
            if (copies >= kRing) ok = wait(&r_free[slot], ph);
            if (!ok) break;
            if constexpr (Q8) {
                // 16 bytes a lane at a time: issued by the whole warp at once, where a bulk copy takes about 90
                // clocks, and a tile has 8 or 16
                const uint8_t *src = static_cast<const uint8_t *>(w ? a.v : a.k);
                constexpr int PC = D / 16, RW = 32 / PC;  // pieces of a row, rows at a time
                const int rr = lane / PC, ch = lane % PC;
                const uint32_t dst = smem_u32(pipe.smem + L::raw) + slot * (L::kSlot / 2) + rr * D + ch * 16;
#pragma unroll
                for (int i0 = 0; i0 < 8; ++i0) {
                    const int g = 8 * part + i0;
                    const long long r0 = __shfl_sync(0xffffffffu, g & 1 ? l.row1 : l.row0, g >> 1);
                    if (r0 < 0) continue;
                    const uint8_t *from = src + (r0 + rr) * D + ch * 16;
#pragma unroll
                    for (int i = 0; i < 8; i += RW) cp_async16(dst + (g * 8 + i) * D, from + i * D);
                }
                if (w == 0) {
                    // with K: both scales of its positions, NP a lane (a page's one scale as often)
                    constexpr int NP = 2;
                    const int p0 = 64 * part + lane * NP, from = p0 >> 4, h8 = p0 >> 3 & 1;
                    const uint32_t sk = smem_u32(pipe.smem + L::scales) + sc_slot * 1024 + p0 * 4;
                    const long long row0 = __shfl_sync(0xffffffffu, l.row0, from), row1 = __shfl_sync(0xffffffffu, l.row1, from);
                    const long long c0 = __shfl_sync(0xffffffffu, l.sc0, from), c1 = __shfl_sync(0xffffffffu, l.sc1, from);
                    const long long so = (h8 ? c1 : c0) + (p0 & 7) * a.scale_token_stride;
                    if ((h8 ? row1 : row0) >= 0) {
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            cp_async4(sk + 4 * i, a.k_scales + so + i * a.scale_token_stride);
                            cp_async4(sk + 512 + 4 * i, a.v_scales + so + i * a.scale_token_stride);
                        }
                    }
                    sc_slot = sc_slot + 1 == L::kScales ? 0 : sc_slot + 1;
                }
                cp_async_mbar_arrive_noinc(&r_full[slot]);
            } else {
                const unsigned boxes = (l.row0 >= 0) + (l.row1 >= 0);
                const uint32_t bytes = __reduce_add_sync(0xffffffffu, boxes) * R * 2 * D;
                if (lane == 0) mbar_arrive_expect_tx(&r_full[slot], bytes);
                __syncwarp();
                const CUtensorMap *map = w ? &tm_v : &tm_k;
                uint8_t *dst = pipe.smem + L::ring + slot * L::kSlot + lane * (16 * D * 2);
                if (l.row0 >= 0) tma_load_4d(dst, map, 0, 0, 0, l.row0, &r_full[slot]);
                if (l.row1 >= 0) tma_load_4d(dst + 8 * D * 2, map, 0, 0, 0, l.row1, &r_full[slot]);
            }
            ++copies;
            if (++slot == kRing) {
                slot = 0;
                ph ^= 1;
            }
        }
        before = s0.loc;
        s0 = s1;
        s1 = s2;
    }
    if (!ok && lane == 0) tile_give_up(abort);
    // every copy issued lands before the shared memory is released
    if (Q8)
        cp_async_wait_all();
    else if (lane == 0)
        for (int k = max(0, copies - NS); k < copies; ++k) mbar_wait(&full[k % NS], (k / NS) & 1);
    __syncwarp();
}

// A copy's 128 x D bytes to bf16 in the operand layout, 16 bytes a thread at a time.
// 0x4300 | u is bf16 128 + u for u < 128, and 0x4300 | sign bit is 128 or 256: their
// difference is the signed byte, without the conversion pipe that the exponentials use.  Kept
// lean, since int8 decode is bound by it: addresses by constant steps and the halves swapped
// before they are widened took 206 to 191 us for 48 sequences of 512 to 8192 tokens.
template <int D, int THREADS>
__device__ __forceinline__ void convert_tile(uint32_t src, uint32_t dst, int me) {
    constexpr int C = D / 16, ROWS = THREADS / C;  // 16-byte pieces of a row; rows at a time
    static_assert(ROWS % 8 == 0, "a thread keeps its place in the 8-row groups");
    // the upper half of a row's threads stores its second chunk first: no two of eight lanes meet
    // in a bank
    const int pc = me % C, swap = pc >= C / 2;
    const uint32_t first = dst + kv_chunk_off<D>(me / C, 2 * pc + swap), second = dst + kv_chunk_off<D>(me / C, 2 * pc + !swap);
#pragma unroll 2  // more is slower: its code pushes other code out of the instruction cache
    for (int i = 0; i < kTileTok / ROWS; ++i) {
        const uint4 w = lds_u4(src + me * 16 + i * (THREADS * 16));
        const uint32_t x[4] = {swap ? w.z : w.x, swap ? w.w : w.y, swap ? w.x : w.z, swap ? w.y : w.w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            o[2 * k] = byte_pair<0x4140>(x[k]);
            o[2 * k + 1] = byte_pair<0x4342>(x[k]);
        }
        sts_u4(first + i * (2 * D * ROWS), make_uint4(o[0], o[1], o[2], o[3]));
        sts_u4(second + i * (2 * D * ROWS), make_uint4(o[4], o[5], o[6], o[7]));
    }
    fence_proxy_async_smem();
}

// Converter warps: the ring's copies in order, or (K_ONLY) the K among them.
template <typename L, int D, int THREADS, bool K_ONLY>
__device__ __forceinline__ void tile_converter(const TilePipe<L> &pipe, int me) {
    constexpr int NS = L::kSlots;
    const int lane = me & 31;
    int rs = 0, bs = 0;
    uint32_t rph = 0, bph = 1;
    bool ok = true;
#pragma unroll 1
    for (int run = 0; ok; ++run) {
        const int at = run % L::kRuns;
        if (!(ok = pipe.wait(&pipe.run_full[at], run / L::kRuns))) break;
        const int n = pipe.runs[at].n;
        __syncwarp();
        if (lane == 0) mbar_arrive(&pipe.run_free[at]);
        if (n == 0) break;
#pragma unroll 1
        for (int c = 0; c < 2 * n; ++c) {
            if (!K_ONLY || c == 0 || ((c & 1) && c != 2 * n - 1)) {
                // K_ONLY: a bf16 slot's release first.  It says that the copy kSlots in front of this one
                // has landed, so that the phase of raw_full waited for is this copy's (kRaw = kSlots).
                ok = pipe.wait(&pipe.empty[bs], bph) && pipe.wait(&pipe.raw_full[rs], rph);
                if (!ok) break;
                convert_tile<D, THREADS>(smem_u32(pipe.smem + L::raw) + rs * (L::kSlot / 2),
                                         smem_u32(pipe.smem + L::ring) + bs * L::kSlot, me);
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&pipe.full[bs]);
                    mbar_arrive(&pipe.raw_free[rs]);
                }
            }
            if (++rs == L::kRaw) {
                rs = 0;
                rph ^= 1;
            }
            if (++bs == NS) {
                bs = 0;
                bph ^= 1;
            }
        }
    }
    if (!ok && lane == 0) tile_give_up(pipe.abort);
}

// FEAT: what is done to the scores besides scale and mask (kPlain, kBias: distance bias,
// kCap: soft-cap, with or without bias); separate kernels, so that each one's code stays
// short.
template <typename T, int D, int FEAT, bool Q8>
__global__ void __launch_bounds__(Q8 ? kTileThreadsQ8 : kTileThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const TileArgs p) {
    using L = TileSmem<D, Q8>;
    constexpr int NS = L::kSlots;
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    const AttnArgs &a = p.a;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    uint8_t *ring = tile_smem + L::ring;
    float *sm_ml = reinterpret_cast<float *>(tile_smem + L::ml);
    const TilePipe<L> pipe(tile_smem);
    RunDesc *const runs = pipe.runs;
    uint64_t *const full = pipe.full, *const empty = pipe.empty, *const run_full = pipe.run_full, *const run_free = pipe.run_free;
    volatile int *const abort = pipe.abort;
    uint64_t *s_full = pipe.own;               // [2] scores in tensor memory (and every earlier MMA done)
    uint64_t *p_full = s_full + 2;             // [2] probabilities in tensor memory (V cleared, O rescaled)
    uint64_t *o_full = p_full + 2;             // [2] a run's last value MMA of the group done
    uint64_t *o_free = o_full + 2;             // [2] O read
    uint64_t *q_full = o_free + 2;             // [2] q staged in buffer 0, 1
    uint64_t *q_free = q_full + 2;             // [2] q buffer read by both issuers
    uint64_t *drained = q_free + 2;            // [2] an issuer's MMAs done
    uint64_t *turn = drained + 2;              // [2][4] group t's warp may use the exponent pipe
    uint64_t *ml_full = turn + 8;              // group 1's (m, l) handed over
    uint32_t *sm_tmem = reinterpret_cast<uint32_t *>(tile_smem + L::misc + 8);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        pipe.init(Q8 ? 4 : 2, 2, Q8 ? 14 : 10, p.wait_tries);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&o_free[t], 4);
            mbar_init(&q_full[t], 4);
            mbar_init(&q_free[t], 2);
            mbar_init(&drained[t], 1);
        }
        for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
        mbar_init(ml_full, 4);
        fence_barrier_init();
    }
    if (Q8 && tid < 128) reinterpret_cast<float *>(tile_smem + L::ones)[tid] = 1.f;
    if (!Q8 && warp == 9 && lane == 0) {
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
    const uint32_t abort_s = smem_u32(tile_smem + L::misc);
    auto wait = [&](uint64_t *bar, uint32_t phase) { return tile_wait(smem_u32(bar), phase & 1, abort_s); };

    if (warp >= 8) {
        if (warp == 9 || warp == 11) {
            // ===================================================================== producers
            tile_producer<L, D, Q8>(p, pipe, tm_k, tm_v, lane, warp == 11);
        } else if (Q8 && warp >= 12) {
            // ===================================================================== converters
            if constexpr (Q8) tile_converter<L, D, 128, false>(pipe, tid - 384);
        } else if (warp == 8 || warp == 10) {
            // ===================================================================== MMA issuers
            // Warp 8 issues group 0's MMAs, warp 10 group 1's: what one waits for does not hold the
            // other up.  The warp walks its steps with warp-uniform values (descriptors stay in uniform
            // registers) and one elected lane issues.
            const int t = warp == 10;
            constexpr uint32_t id_s = umma_idesc_16bit(128, kTileTok, kBf16, 0, 0);
            constexpr uint32_t id_o = umma_idesc_16bit(128, D, kBf16, 0, 1);
            const uint64_t q_desc = umma_desc_sw128(smem_u32(tile_smem + L::q), 16, 1024);
            const uint64_t k_desc = umma_desc_sw128(smem_u32(ring), 16, 16 * D);
            const uint64_t v_desc = umma_desc_sw128(smem_u32(ring), 1024, 16 * D);
            const uint32_t t_s = tmem + 128 * t, t_o = tmem + 256 + 128 * t;
            const bool leader = elect_one();
            int slot = 0;      // next ring slot and its phase
            uint32_t ring_ph = 0;
            uint32_t pp = 0;   // phase of the next probabilities
            int ou = 0;        // runs that used this group's O so far
            uint32_t qph = 0;  // bit b: phase of the next fill of q buffer b
            int qb = 1;        // q buffer of the last small block; 1 after a large one
            bool ok = true;
#pragma unroll 1
            for (int run = 0;; ++run) {
                const int at = run % L::kRuns;
                ok = wait(&run_full[at], run / L::kRuns);
                if (!ok) break;
                const int n = __shfl_sync(0xffffffffu, runs[at].n, 0);
                const bool large = __shfl_sync(0xffffffffu, runs[at].nrows, 0) > 128;
                if (leader) mbar_arrive(&run_free[at]);
                if (n == 0) break;
                // Large block: step j has the scores of tile j and the values of tile j - 1.  Small block:
                // the scores of tile j and the values of j - 2, both of group j & 1.  The other issuer follows
                // the ring and frees the slots too: left out, it could fall behind by more than a turn of
                // the ring (runs of one tile need it for nothing) and take one phase for another.
                const int lag = large ? 1 : 2;
                const bool used = large || t == 0 || n > 1;
                qb = large ? 1 : (qb ^ 1);
                const int qbuf = large ? t : qb;
                ok = wait(&q_full[qbuf], qph >> qbuf);
                const uint32_t other = qph >> (t ^ 1);  // large: phase of the other group's q
                qph ^= large ? 3 : 1 << qbuf;
                const uint64_t qd = q_desc + qbuf * (L::kQ >> 4);
#pragma unroll 1
                for (int j = 0; ok && j < n + lag; ++j) {
                    const bool big = opaque(large);
                    const bool own = big || (j & 1) == t;
                    // ring order: K_j, V_j-1 (large), V_j-2, K_j (small)
                    const bool has_k = j < n, has_v = j >= lag;
                    int ks = 0, vs = 0;
                    uint32_t kp = 0, vp = 0;
                    auto take = [&](int &s, uint32_t &ph) {
                        s = slot;
                        ph = ring_ph;
                        if (++slot == NS) {
                            slot = 0;
                            ring_ph ^= 1;
                        }
                    };
                    if (big && has_k) take(ks, kp);
                    if (has_v) take(vs, vp);
                    if (!big && has_k) take(ks, kp);
                    const uint64_t vd = v_desc + vs * (L::kSlot >> 4);
                    const uint64_t kd = k_desc + ks * (L::kSlot >> 4);
                    // Between the last probabilities and the next scores' issue a row group waits, so what
                    // can be done before or after is.  (A small block's K comes last: its V slot is freed
                    // without waiting for it.)
                    if (big && has_k) ok = wait(&full[ks], kp);
                    if (has_v) {
                        ok = ok && wait(&full[vs], vp);
                        if (own) {
                            const bool first = j - lag < (big ? 1 : 2);
                            if (first && ou > 0) ok = ok && wait(&o_free[t], ou - 1);
                            ok = ok && wait(&p_full[t], pp);
                            tc_fence_after();
                            if (ok && leader) {
#pragma unroll
                                for (int kk = 0; kk < kTileTok / 16; ++kk)
                                    umma_f16_ts(t_o, t_s + 8 * kk, vd + kk * (32 * D >> 4), id_o, !(first && kk == 0));
                            }
                            pp ^= 1;
                            if (!big && ok && leader) umma_commit(&empty[vs]);
                        } else if (ok && leader) {
                            mbar_arrive(&empty[vs]);
                        }
                    }
                    if (!big && has_k) ok = ok && wait(&full[ks], kp);
                    if (!ok) break;
                    if (own) {
                        if (has_k) {
                            tc_fence_after();
                            if (leader) {
#pragma unroll
                                for (int kk = 0; kk < D / 16; ++kk)
                                    umma_f16(t_s, qd + (kk >> 2) * (16384 >> 4) + (kk & 3) * 2,
                                             kd + (kk >> 2) * (1024 >> 4) + (kk & 3) * 2, id_s, kk > 0);
                                umma_commit(&s_full[t]);
                                umma_commit(&empty[ks]);
                                if (j + lag >= n) umma_commit(&q_free[qbuf]);  // the group's last scores
                            }
                            if (big && j + 1 == n) {
                                // the other group's buffer waits for both issuers
                                ok = wait(&q_full[t ^ 1], other);
                                if (ok && leader) mbar_arrive(&q_free[t ^ 1]);
                            }
                        }
                        if (has_v && leader) {
                            if (big) umma_commit(&empty[vs]);
                            if (j >= n) umma_commit(&o_full[t]);  // the group's last tile
                        }
                    } else if (has_k && leader) {
                        mbar_arrive(&empty[ks]);
                    }
                }
                if (!ok) break;
                if (used)
                    ++ou;
                else if (leader)
                    mbar_arrive(&q_free[qbuf]);
            }
            if (!ok && lane == 0) tile_give_up(abort);
            // every MMA issued has completed before tensor memory and shared memory go
            if (leader) {
                umma_commit(&drained[t]);
                mbar_wait(&drained[t], 0);
            }
            __syncwarp();
        }
    } else {
        // ===================================================================== row groups
        const int G = a.num_q_heads / a.num_kv_heads;
        const unsigned g_magic = div_magic(G);
        const int t = warp >> 2;           // group
        const int row = tid & 127;         // row of the group = tensor-memory lane
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + 128 * t + lanes, t_o = tmem + 256 + 128 * t + lanes;
        int c0 = 0, sn = 0;                // ring position of the run's first K; this group's tiles so far
        [[maybe_unused]] int sc0 = 0;      // scales of the run's first tile
        int qb = 1;                        // q buffer of the last small block; 1 after a large one
        int ou[2] = {0, 0};                // runs that used O of group 0, 1 so far
        int mln = 0;                       // small blocks of more than one tile so far
        int turns = 0;                     // tiles of large blocks so far
        int fills = 0;                     // of this group's q buffer so far
        bool ok = true;

        // The q of run `next`: group t fills buffer t, with its own rows of a large block, or with those of
        // a small one whose turn that buffer is.  A buffer is free once both issuers are through with
        // its last contents; its own group alone waits for that, every time, so that no phase is
        // mistaken for another.
        auto fill_q = [&](int next) {
            const int at = next % L::kRuns;
            if (!(ok = wait(&run_full[at], next / L::kRuns))) return;
            const RunDesc *d = &runs[at];
            if (d->n == 0) return;
            const bool large = d->nrows > 128;
            if (large || t == (qb ^ 1)) {
                if (fills > 0 && !(ok = wait(&q_free[t], fills - 1))) return;
                ++fills;
                constexpr int CH = D / 8;  // 16-byte chunks of a row
                const int first = large ? 128 * t : 0, live = min(d->nrows - first, 128), rho0 = d->row0 + first;
                const T *q0 = reinterpret_cast<const T *>(a.q) + (static_cast<long long>(d->tok0) * a.num_q_heads + d->h * G) * D;
                const uint32_t dst = smem_u32(tile_smem + L::q) + t * L::kQ;
                // a thread's chunks are one column of rows row / CH, + 128 / CH, ...; eight loads in flight
                const int ch = row % CH;
#pragma unroll 1
                for (int k0 = 0; k0 < CH; k0 += 8) {
                    const int r0 = row / CH + k0 * (128 / CH);
                    if (r0 >= live) break;
                    uint4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int rho = rho0 + min(r0 + k * (128 / CH), live - 1), tok = fast_div(rho, G, g_magic);
                        v[k] = __ldg(reinterpret_cast<const uint4 *>(
                                         q0 + (static_cast<long long>(tok) * a.num_q_heads + (rho - tok * G)) * D) + ch);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int rr = r0 + k * (128 / CH);
                        if (rr < live) sts_u4(dst + (ch >> 3) * 16384 + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4), v[k]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[t]);
            }
        };

        // rewrite: where a cap, a mask or a bias of both signs asks for more than probs does, S becomes the
        // score in the exponent domain first, -inf outside columns [jlo, jhi).
        const float cap1 = FEAT == kCap ? a.q_scale / a.soft_cap : 0.f, cap2 = a.soft_cap * kLog2e;
        auto rewrite = [&](float slope, float d0, int jlo, int jhi, const float *scales) {
#pragma unroll 1
            for (int k = 0; k < 128; k += 32) {
                float w[32];
                tmem_ld<32>(t_s + k, w);
                tmem_wait_ld();
                if constexpr (Q8) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(scales + k + i);
                        w[i] *= s4.x, w[i + 1] *= s4.y, w[i + 2] *= s4.z, w[i + 3] *= s4.w;
                    }
                }
                const int l0 = jlo - k, h0 = jhi - k;
                unsigned seen = h0 >= 32 ? ~0u : h0 <= 0 ? 0u : (1u << h0) - 1;
                if (l0 > 0) seen = l0 >= 32 ? 0u : seen & (~0u << l0);
                if constexpr (FEAT == kCap) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) w[i] *= cap1;
                    unit_cap(w, seen);
                }
                const float f = FEAT == kCap ? cap2 : a.q_scale;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    float x = w[i] * f;
                    if constexpr (FEAT != kPlain) x = fmaf(-slope, fabsf(d0 + static_cast<float>(k + i)), x);
                    w[i] = (seen >> i & 1) ? x : -INFINITY;
                }
                tmem_st32(t_s + k, w);
            }
            tmem_wait_st();
        };
        float m = -INFINITY, l = 0.f;  // the row's reference (exponent domain) and sum in this run
        // The reference rises by `by` (an integer where the row had one, so that all but m scale
        // exactly), and what stands relative to it follows: l, the sum so far, the columns of P stored
        // already and O (fresh: the group has none in this run yet; what stands there may be another
        // run's that group 0 is still reading).
        auto raise = [&](bool move, float top, float2 &acc, int stored, bool fresh) {
            const float by = !move || m == -INFINITY ? 0.f : ceilf(top) - kBelowMax<T>, alpha = fast_exp2(-by);
            m = !move ? m : m == -INFINITY ? top - kBelowMax<T> : m + by;
            if (!__any_sync(0xffffffffu, by != 0.f)) return;
            l *= alpha;
            acc.x *= alpha;
            acc.y *= alpha;
            tmem_wait_ld();
            tmem_wait_st();
#pragma unroll 1
            for (int k = fresh ? D : 0; k < D + stored; k += 8) {
                // the scores' commit covers the group's earlier value MMAs: O is at rest
                const bool is_o = k < D;
                const uint32_t at = is_o ? t_o + k : t_s + (k - D);
                float o[8];
                tmem_ld<8>(at, o);
                tmem_wait_ld();
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // (in fp32, whose range the factor needs; f16 pairs below 2^-14 are rounded once more)
                    const float2 x = unpack2<T>(__float_as_uint(o[i]));
                    w[i] = is_o ? __float_as_uint(o[i] * alpha) : pack2<T>(x.x * alpha, x.y * alpha);
                }
                tmem_st8(at, w);
            }
            tmem_wait_st();
        };
        // One pass over a tile's scores: x = S f + c + se column - m (c: bias at column 0), P = 2^x over the
        // columns read already, and its sum.  S is read once, since reading it takes about as long as
        // the exponentials.
        auto probs = [&](float f, float c, float se, const float *scales_k, const float *scales_v, bool live, bool fresh) {
            constexpr int W = Q8 ? 16 : 32;  // columns at a time, the next ones' load under way
            float2 acc = make_float2(0.f, 0.f);
            float wa[W], wb[W];
            auto part = [&](float(&w)[W], int col) {
                float2 cc = pair(c - (m == -INFINITY ? 0.f : m));
                if constexpr (FEAT == kBias) {
                    cc.x = fmaf(se, static_cast<float>(col), cc.x);
                    cc.y = cc.x + se;
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < W; i += 2) {
                    float2 ff = pair(f);
                    if constexpr (Q8) ff = mul2(ff, *reinterpret_cast<const float2 *>(scales_k + col + i));
                    const float2 x = fma2(make_float2(w[i], w[i + 1]), ff, cc);
                    if constexpr (FEAT == kBias) cc = add2(cc, pair(2.f * se));
                    w[i] = x.x;
                    w[i + 1] = x.y;
                    mx[i / 2 & 1] = fmaxf(mx[i / 2 & 1], fmaxf(x.x, x.y));
                }
                const float top = fmaxf(mx[0], mx[1]);
                const bool move = live && (m == -INFINITY ? top > -INFINITY : top > kLazyMax<T>);
                if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
                    const float was = m == -INFINITY ? 0.f : m;
                    raise(move, top, acc, col / 2, fresh);
                    const float down = was - (m == -INFINITY ? 0.f : m);
#pragma unroll
                    for (int i = 0; i < W; ++i) w[i] += down;
                }
                uint32_t pk[W / 2];
#pragma unroll
                for (int i = 0; i < W; i += 2) {
                    float2 x = make_float2(fast_exp2(w[i]), fast_exp2(w[i + 1]));
                    acc = add2(acc, x);
                    if constexpr (Q8) {
                        // times the value's scale; where nothing is seen (P = 0) that may be anything
                        const float2 s2 = *reinterpret_cast<const float2 *>(scales_v + col + i);
                        x.x = x.x == 0.f ? 0.f : x.x * s2.x;
                        x.y = x.y == 0.f ? 0.f : x.y * s2.y;
                    }
                    pk[i / 2] = pack2<T>(x.x, x.y);
                }
                if constexpr (W == 32)
                    tmem_st16(t_s + (col >> 1), pk);
                else
                    tmem_st8(t_s + (col >> 1), pk);
            };
            tmem_ld<W>(t_s, wa);
#pragma unroll 1
            for (int k = 0; k < 128; k += 2 * W) {
                tmem_wait_ld();
                tmem_ld<W>(t_s + k + W, wb);
                part(wa, k);
                tmem_wait_ld();
                tmem_ld<W>(t_s + (k + 2 * W & 127), wa);  // the last round's is not used
                part(wb, k + W);
            }
            tmem_wait_ld();
            l += acc.x + acc.y;
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
            const bool big = d.nrows > 128;
            if (run >= 0) qb = big ? 1 : qb ^ 1;
            const int ri = big ? 128 * t + row : row;  // row of the block
            const bool live = ri < d.nrows;
            // the row's query, its positions [lo, hi) and its bias
            long long out_row = 0;
            int lo = 0, hi = 0, pos = 0;
            float slope = 0.f;
            if (live) {
                const int rho = d.row0 + ri, i = fast_div(rho, G, g_magic), head = d.h * G + (rho - i * G);
                out_row = static_cast<long long>(d.tok0 + i) * a.num_q_heads + head;
                lo = d.lo;
                hi = d.hi;
                if ((d.flags & 3) == kOwn) {
                    pos = d.pos0 + i;
                    row_range(a, d.tab, d.tok0 + i, pos, d.len, lo, hi);
                    if (FEAT != kPlain && a.slopes) slope = a.slopes[head] * kLog2e;
                }
            }
            const bool warp_live = __any_sync(0xffffffffu, live);
            m = -INFINITY;
            l = 0.f;
            const int j0 = big ? 0 : t, dj = big ? 1 : 2;
#pragma unroll 1
            for (int j = j0; j < n; j += dj) {
                const int t0 = (d.tile0 - j) * kTileTok;
                const int jlo = lo - t0, jhi = hi - t0;  // visible columns [jlo, jhi)
                ok = wait(&s_full[t], sn++);
                if (!ok) break;
                tc_fence_after();
                // V rows that no row of the block attends are cleared (a zero probability does not
                // cancel a NaN), by each group that uses the tile
                const int vlo = d.lo - t0, vhi = d.hi - t0;
                if (!Q8 && __builtin_expect(vlo > 0 || vhi < kTileTok, 0)) {  // int8: integers are finite
                    const int cv = c0 + v_at(j, n);
                    ok = wait(&full[cv % NS], cv / NS);
                    if (!ok) break;
                    const uint32_t vt = smem_u32(ring) + (cv % NS) * L::kSlot;
                    for (int i = row; i < kTileTok * (D / 8); i += 128) {
                        const int tok = i / (D / 8);
                        if (tok < vlo || tok >= vhi) sts_u4(vt + kv_chunk_off<D>(tok, i % (D / 8)), make_uint4(0, 0, 0, 0));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                float f = a.q_scale, se = 0.f, base = 0.f;
                [[maybe_unused]] const float *scales = nullptr, *scales_k = nullptr;
                if constexpr (Q8)
                    scales_k = scales = reinterpret_cast<const float *>(tile_smem + L::scales) + (sc0 + j) % L::kScales * 256;
                if (opaque(warp_live)) {
                    // The bias is linear in the column where the row's visible columns lie on one side of its
                    // own position.
                    const bool behind = jhi <= pos + 1 - t0, ahead = jlo >= pos - t0;
                    const bool odd = live && (jlo > 0 || jhi < kTileTok || (FEAT == kBias && slope != 0.f && !behind && !ahead));
                    const float d0 = static_cast<float>(t0 - pos);
                    if (FEAT == kCap || __any_sync(0xffffffffu, odd)) {
                        rewrite(slope, d0, jlo, jhi, scales);
                        f = 1.f;
                        scales_k = reinterpret_cast<const float *>(tile_smem + L::ones);  // applied already
                    } else if (FEAT == kBias) {
                        se = behind ? slope : -slope;
                        base = se * d0;
                    }
                }
                // Large blocks: the two groups' warps on one SM sub-partition take turns, so that one's
                // exponentials run under the other's products.  Left alone most CTAs fell into step: both
                // computed, then both waited.
                if (opaque(big)) {
                    if (turns + t > 0) ok = wait(&turn[4 * t + (warp & 3)], turns + t - 1);
                    if (!ok) break;
                    ++turns;
                }
                if (opaque(warp_live)) probs(f, base, se, scales_k, scales + 128, live, j == j0);
                if (opaque(big) && lane == 0) mbar_arrive(&turn[4 * (t ^ 1) + (warp & 3)]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            fill_q(run + 1);  // the next run's q, under this run's last products
            if (!ok) break;
            if (run < 0) continue;

            // ------------------------------------------------ end of the run
            const bool two = !big && n > 1;  // both groups hold a part of each row
            if (two && t == 1) {
                // group 0 has read what was there before (it freed O of group 1 behind that)
                if (ou[1] > 0) ok = wait(&o_free[1], ou[1] - 1);
                if (!ok) break;
                sm_ml[row] = m;
                sm_ml[128 + row] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(ml_full);
            }
            if (big || t == 0) {
                ok = wait(&o_full[t], ou[t]);
                float fa = 1.f, fb = 0.f;
                if (ok && two) {
                    // group 1's (m, l) first: by then it is through with its part of the runs in front, so
                    // that the phase of o_full[1] waited for next is this run's
                    ok = wait(ml_full, mln) && wait(&o_full[1], ou[1]);
                    if (ok) {
                        const float mb = sm_ml[row], lb = sm_ml[128 + row];
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
                    const bool whole = d.flags & 4, direct = whole && (d.flags & 3) == kOwn;
                    // where a partial state goes: the CTA's slot, or the row's place of a whole unit
                    float *st_o = nullptr;
                    if (!direct && live) {
                        if (whole) {
                            const long long to = ((d.flags & 3) == kSuffix ? static_cast<long long>(a.total_q) * a.num_q_heads : 0) + out_row;
                            p.ml[to] = make_float2(m, l);
                            st_o = p.acc + to * D;
                        } else {
                            float *ps = p.slots + (static_cast<size_t>(blockIdx.x) * 2 + (d.flags >> 3 & 1)) * (kBlkRows * (D + 2));
                            ps[ri] = m;
                            ps[kBlkRows + ri] = l;
                            st_o = ps + 2 * kBlkRows + ri * D;
                        }
                    }
                    T *out = reinterpret_cast<T *>(a.out) + out_row * D;
                    __syncwarp();
#pragma unroll 1
                    for (int k = 0; k < D; k += 32) {
                        float o[32];
                        tmem_ld<32>(t_o + k, o);
                        if (opaque(two)) {
                            float ob[32];
                            tmem_ld<32>(t_o + 128 + k, ob);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = fmaf(o[i], fa, ob[i] * fb);
                        } else {
                            tmem_wait_ld();
                        }
                        if (opaque(live && direct)) {
                            uint4 *dst = reinterpret_cast<uint4 *>(out + k);
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    w[e] = l == 0.f ? 0u : pack2<T>(o[8 * q + 2 * e] * inv, o[8 * q + 2 * e + 1] * inv);
                                dst[q] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else if (opaque(live)) {
                            float4 *dst = reinterpret_cast<float4 *>(st_o + k);
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
            if (two) ++mln;
            ++ou[0];
            if (big || two) ++ou[1];
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
            const float *slot = p.slots + (static_cast<size_t>(b + k) * 2 + (ta == 0 ? 1 : 0)) * (p.blk_rows * (D + 2));
            pm[k] = __ldcg(slot + ri);
            pl[k] = __ldcg(slot + p.blk_rows + ri);
            load_cols<C>(slot + 2 * p.blk_rows + ri * D, lane, po[k]);
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

// Varlen.  CTA (c, y, line): rows y * 8 + warp, ... of the unit that starts in range c and goes on
// behind it; and zeros for the rows of blocks that attend nothing.
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) tile_merge_kernel(const __grid_constant__ PlanArgs both) {
    const TileArgs &p = both.line[blockIdx.z];
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
__global__ void __launch_bounds__(kMergeThreads) tile_merge_shared_kernel(const __grid_constant__ PlanArgs both) {
    const AttnArgs &a = both.line[0].a;
    const int lane = threadIdx.x & 31;
    const int G = a.num_q_heads / a.num_kv_heads;
    const long long rows = static_cast<long long>(a.num_seqs) * a.num_q_heads;
    pdl_wait();
    const long long row = static_cast<long long>(blockIdx.x) * (kMergeThreads / 32) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int s = static_cast<int>(row / a.num_q_heads), head = static_cast<int>(row % a.num_q_heads);
    const int h = head / G, g = head % G;
    RowState<D / 32> st;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const TileArgs &p = both.line[part];  // the same twice where one kernel took both
        int e = a.num_groups + s;
        long long rho = g;
        if (part == 0) {
            e = group_of_seq(a, s);
            if (e < 0) continue;
            rho += static_cast<long long>(s - a.group_starts[e]) * G;
        }
        e -= p.ent0;
        const long long i = p.ents[e] + rho / kBlkRows;
        if (i >= p.ents[e + 1]) continue;  // only where group_starts is not usable
        const long long c0 = p.cost[i], m = p.cost[i + 1] - c0;
        if (m == 0) continue;
        if (!add_pieces<D>(p, p.head->range, c0 * a.num_kv_heads + h * m, m, static_cast<int>(rho % kBlkRows), lane, st)) {
            const long long at = part * rows + row;
            const float2 ml = p.ml[at];
            float o[D / 32];
            load_cols<D / 32>(p.acc + at * D, lane, o);
            st.add(ml.x, ml.y, o);
        }
    }
    write_row<T, D>(both.line[0], row, lane, st);
}

}  // namespace gk
