// gollek_varlen.cu -- host side of ragged and shared-prefix paged attention and of the
// cache read-back: argument checks, kernel selection and their C ABI (gollek_kernels.h).
#include <algorithm>
#include <cstdlib>
#include <mutex>

#include "attn_block.cuh"
#include "attn_rows.cuh"
#include "attn_tile.cuh"
#include "host.cuh"
#include "kv_gather.cuh"
#include "varlen.cuh"

namespace gk {

cudaError_t varlen_status(bool clear, unsigned *out) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(*out));
    if (e == cudaSuccess && clear) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    }
    return e;
}

namespace {

constexpr long long kMaxTokens = 1LL << 30;  // positions a table may name (32-bit arithmetic on them)

bool float_dtype(int dt) {
    return dt == GOLLEK_DTYPE_F32 || dt == GOLLEK_DTYPE_BF16 || dt == GOLLEK_DTYPE_F16;
}
bool quantised(int dt) { return dt == GOLLEK_DTYPE_I8 || dt == GOLLEK_DTYPE_I4; }

// What every entry point here checks of a pool; *stride receives the page stride in use.
int check_pool(int kv_dtype, const float *ks, const float *vs, int num_kv_heads, int head_dim, int block_size,
               int max_blocks, int num_blocks, long long page_stride, long long *stride) {
    if (num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || max_blocks <= 0 || num_blocks < 0)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "non-positive size");
    if (kv_dtype < GOLLEK_DTYPE_F32 || kv_dtype > GOLLEK_DTYPE_I4)
        return fail(GOLLEK_ERR_UNSUPPORTED, "kv dtype %d", kv_dtype);
    if (quantised(kv_dtype) && (!ks || !vs))
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "quantised KV needs k_scales and v_scales");
    const long long minimal = static_cast<long long>(num_kv_heads) * block_size * head_dim;
    if (page_stride != 0 && page_stride < minimal)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "page_stride %lld < num_kv_heads*block_size*head_dim", page_stride);
    *stride = page_stride ? page_stride : minimal;
    if (kv_dtype == GOLLEK_DTYPE_I4 && ((head_dim & 1) || (*stride & 1)))
        return fail(GOLLEK_ERR_UNSUPPORTED, "int4 pools need an even head_dim and page stride");
    if (static_cast<long long>(max_blocks) * block_size > kMaxTokens)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "max_blocks_per_seq * block_size too large");
    return GOLLEK_OK;
}

int check_attn(const AttnArgs &a) {
    if (a.num_q_heads <= 0 || a.num_q_heads % a.num_kv_heads != 0)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "num_q_heads %d not a multiple of num_kv_heads %d", a.num_q_heads,
                    a.num_kv_heads);
    if (!float_dtype(a.q_dtype)) return fail(GOLLEK_ERR_UNSUPPORTED, "q dtype %d (F32, BF16 or F16 only)", a.q_dtype);
    if (a.head_dim > 256) return fail(GOLLEK_ERR_UNSUPPORTED, "head_dim %d above 256", a.head_dim);
    if (a.num_kv_heads > 65535 || a.num_q_heads / a.num_kv_heads > 65535)
        return fail(GOLLEK_ERR_UNSUPPORTED, "more than 65535 heads");
    return GOLLEK_OK;
}

template <int J>
const void *generic_fn(int G) {
    if (G == 1) return reinterpret_cast<const void *>(&attn_generic_kernel<J, 1>);
    if (G == 2) return reinterpret_cast<const void *>(&attn_generic_kernel<J, 2>);
    if constexpr (J < 8)
        if (G > 4) return reinterpret_cast<const void *>(&attn_generic_kernel<J, 8>);
    return reinterpret_cast<const void *>(&attn_generic_kernel<J, 4>);
}

template <int DP>
int launch_block(AttnArgs &a, cudaStream_t st) {
    const void *fn = a.kv_dtype == GOLLEK_DTYPE_F32    ? reinterpret_cast<const void *>(&attn_block_kernel<DP, GOLLEK_DTYPE_F32>)
                     : a.kv_dtype == GOLLEK_DTYPE_BF16 ? reinterpret_cast<const void *>(&attn_block_kernel<DP, GOLLEK_DTYPE_BF16>)
                     : a.kv_dtype == GOLLEK_DTYPE_F16  ? reinterpret_cast<const void *>(&attn_block_kernel<DP, GOLLEK_DTYPE_F16>)
                     : a.kv_dtype == GOLLEK_DTYPE_I8   ? reinterpret_cast<const void *>(&attn_block_kernel<DP, GOLLEK_DTYPE_I8>)
                                                       : reinterpret_cast<const void *>(&attn_block_kernel<DP, GOLLEK_DTYPE_I4>);
    GK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kAbSmem<DP>)), "cudaFuncSetAttribute");
    int qt = kAbRows / (a.num_q_heads / a.num_kv_heads);
    void *args[] = {&a, &qt};
    const long long blocks = a.total_q / qt + static_cast<long long>(a.num_seqs);
    GK_CUDA(cudaLaunchKernel(fn, dim3(static_cast<unsigned>(blocks), a.num_kv_heads), dim3(kAbThreads), args, kAbSmem<DP>, st),
            "attn_block_kernel launch");
    return GOLLEK_OK;
}

// Calls that the tensor-core kernels do not take.  Varlen calls of kBlockRows rows and more a
// sequence on average go to the blocked kernel, which reads a cache row once for 64 of them (8
// fp32 sequences of 400 to 1500 tokens, 4 rows a query token: 16 rows 297 us there and 191 in
// the other, 32 rows 301 and 363, 384 rows 788 and 3232).
constexpr int kBlockRows = 32;

int launch_generic(AttnArgs &a, cudaStream_t st) {
    const int G = a.num_q_heads / a.num_kv_heads;
    if (a.num_groups == 0 && G <= kAbRows && static_cast<long long>(a.total_q) * G >= static_cast<long long>(a.num_seqs) * kBlockRows)
        return a.head_dim <= 64 ? launch_block<64>(a, st) : a.head_dim <= 128 ? launch_block<128>(a, st) : launch_block<256>(a, st);
    const int J = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 4 : 8;
    const void *fn = J == 2 ? generic_fn<2>(G) : J == 4 ? generic_fn<4>(G) : generic_fn<8>(G);
    const int GC = G == 1 ? 1 : G == 2 ? 2 : (G <= 4 || J == 8) ? 4 : 8;
    void *args[] = {&a};
    GK_CUDA(cudaLaunchKernel(fn, dim3(a.total_q, a.num_kv_heads, (G + GC - 1) / GC), dim3(kAgWarps * 32), args, 0, st),
            "attn_generic_kernel launch");
    return GOLLEK_OK;
}

// Whether the tile kernels take the call: 16-bit pool and q of one type, or int8 pool and
// bf16 q; head_dim 64 or 128, pages of 8 or a multiple of 16 tokens in whole 8-row groups, 16-byte
// aligned tensors.
bool tile_takes(const AttnArgs &a) {
    if (a.kv_dtype == GOLLEK_DTYPE_I8) {
        if (a.q_dtype != GOLLEK_DTYPE_BF16) return false;
    } else if (a.q_dtype != a.kv_dtype || (a.kv_dtype != GOLLEK_DTYPE_BF16 && a.kv_dtype != GOLLEK_DTYPE_F16)) {
        return false;
    }
    if (a.head_dim != 64 && a.head_dim != 128) return false;
    if (a.block_size != 8 && a.block_size % 16 != 0) return false;
    if (a.page_stride % (8 * a.head_dim) != 0) return false;
    if (!aligned16(a.k) || !aligned16(a.v) || !aligned16(a.q) || !aligned16(a.out)) return false;
    const long long page_rows = a.page_stride / a.head_dim;
    return a.num_blocks == 0 || a.num_blocks * page_rows < (1LL << 31);
}

// How the entities of a call are laid out: one cost line for each kernel that takes some of
// them, each with its part of the workspace.
struct CallPlan {
    struct Line {
        int ent0, entities, blk_rows, rows_min, rows_max;
        TileWs ws;
        size_t at;  // of ws
    } line[2];
    int lines;
    size_t total;
};

// attn_rows_kernel (head_dim 128, up to 16 q heads per kv head) takes entities of 16 rows at
// most: 237 -> 183 us for 64 sequences of one token.  What a call gives it, and what the kernel
// for many rows, is chosen from the sizes alone:
// - varlen, no more query tokens than sequences: all, whatever their rows (64 decode steps at 1,024
//   tokens 71 us, with both kernels launched 79).  A longer entity is cut into blocks of 16, each of which
//   reads its pages: a chunk of 512 tokens at 4,096 among 511 idle slots takes 313 us, in both 82.
// - otherwise, once the sequences give the device enough units of work (sequences times kv heads):
//   varlen, from kSplitVarlen units, the entities of few rows, the rest going to the kernel for many
//   (decode steps at 1,024 tokens beside 2 chunks of 300 at 2,048: 128 units 87.5 us in one kernel
//   and 89.2 in two, 192: 97.2 and 97.3, 256: 107.6 and 104.4, 512: 151.6 and 125.0);
//   shared prefixes, from kSplitShared, the own tokens (sequences of 300 tokens behind 4,096: 192
//   units 42.0 and 51.2, 256: 45.6 and 54.3, 384: 62.0 and 62.4, 512: 77.2 and 70.0).
// The layout of the workspace does not depend on the choice, so that what is enough for a call
// is enough for smaller ones.
constexpr int kSplitVarlen = 256, kSplitShared = 384;

CallPlan plan_call(int num_groups, int num_seqs, int total_q, int hq, int hkv, int D) {
    const int G = hq / hkv;
    const bool shared = num_groups > 0;
    const long long rows = static_cast<long long>(total_q) * G, out_rows = static_cast<long long>(total_q) * hq;
    CallPlan c{};
    const CallPlan::Line many{0, num_groups + num_seqs, kBlkRows, 0, INT_MAX,
                              tile_ws(static_cast<long long>(num_groups) + num_seqs, shared ? 2 * rows : rows, kBlkRows, out_rows, D, shared), 0};
    c.line[0] = many;
    c.lines = 1;
    c.total = many.ws.total;
    if (D != kFewD || G > kFewRows) return c;
    const CallPlan::Line few{0, num_seqs, kFewRows, 0, INT_MAX, tile_ws(num_seqs, rows, kFewRows, 0, D, false), c.total};
    c.total += few.ws.total;
    if (!shared && total_q <= num_seqs) {
        c.line[0] = few;
    } else if (static_cast<long long>(num_seqs) * hkv >= (shared ? kSplitShared : kSplitVarlen)) {
        c.lines = 2;
        c.line[1] = few;
        if (shared) {
            c.line[0].entities = num_groups;
            c.line[1].ent0 = num_groups;
        } else {
            c.line[0].rows_min = kFewRows + 1;
            c.line[1].rows_max = kFewRows;
        }
    }
    return c;
}

// 4-D map over a pool of 16-bit rows: (64 columns, 8 rows, column slabs, 8-row blocks), so a
// box of (64, 8, slabs, box_rows / 8) lands in the layout of kv_chunk_off.
int encode_tile_map(CUtensorMap *m, const void *base, int kv_dtype, int D, long long rows, int box_rows) {
    auto enc = encode_fn();
    if (!enc) return fail(GOLLEK_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
    const cuuint32_t slabs = D / 64;
    const cuuint64_t pitch = static_cast<cuuint64_t>(D) * 2;
    cuuint64_t dims[4] = {64, 8, slabs, static_cast<cuuint64_t>(rows / 8)};
    cuuint64_t strides[3] = {pitch, 128, 8 * pitch};
    cuuint32_t box[4] = {64, 8, slabs, static_cast<cuuint32_t>(box_rows / 8)};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(m, kv_dtype == GOLLEK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                     const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GOLLEK_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return GOLLEK_OK;
}

// A launch that may begin before the kernel in front of it has ended (that kernel's results are
// read behind griddepcontrol.wait).
int launch_dependent(const void *fn, dim3 grid, int threads, size_t smem, cudaStream_t st, void **args, const char *what) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    GK_CUDA(cudaLaunchKernelExC(&cfg, fn, args), what);
    return GOLLEK_OK;
}

template <typename T, int D, bool Q8 = false>
int launch_tile_as(const PlanArgs &both, int lines, const CUtensorMap &tmk, const CUtensorMap &tmv, cudaStream_t st) {
    const AttnArgs &a = both.line[0].a;
    static_assert(TileSmem<D, Q8>::total <= 227 * 1024, "shared memory of the tile kernel");
    tile_plan_kernel<<<lines, kPlanThreads, 0, st>>>(both);
    GK_CUDA(cudaGetLastError(), "tile_plan_kernel launch");
    for (int i = 0; i < lines; ++i) {
        const TileArgs &p = both.line[i];
        uint32_t smem = TileSmem<D, Q8>::total;
        int threads = Q8 ? kTileThreadsQ8 : kTileThreads;
        const void *fn = a.soft_cap > 0.f ? reinterpret_cast<const void *>(&attn_tile_kernel<T, D, kCap, Q8>)
                         : a.slopes       ? reinterpret_cast<const void *>(&attn_tile_kernel<T, D, kBias, Q8>)
                                          : reinterpret_cast<const void *>(&attn_tile_kernel<T, D, kPlain, Q8>);
        if constexpr (D == kFewD) {
            static_assert(RowsSmem<Q8>::total <= 227 * 1024, "shared memory of the kernel for few rows");
            if (p.blk_rows == kFewRows) {
                smem = RowsSmem<Q8>::total;
                fn = reinterpret_cast<const void *>(&attn_rows_kernel<T, Q8>);
                threads = kRowsThreads + (Q8 ? kRowsConverters : 0);
            }
        }
        GK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute");
        void *args[] = {const_cast<CUtensorMap *>(&tmk), const_cast<CUtensorMap *>(&tmv), const_cast<TileArgs *>(&p)};
        int rc = launch_dependent(fn, dim3(p.grid), threads, smem, st, args, "attention kernel launch");
        if (rc) return rc;
    }
    void *margs[] = {const_cast<PlanArgs *>(&both)};
    if (a.num_groups == 0)
        return launch_dependent(reinterpret_cast<const void *>(&tile_merge_kernel<T, D>), dim3(both.line[0].grid, kMergeSplit, lines),
                                kMergeThreads, 0, st, margs, "tile_merge_kernel launch");
    const long long rows = static_cast<long long>(a.num_seqs) * a.num_q_heads;
    return launch_dependent(reinterpret_cast<const void *>(&tile_merge_shared_kernel<T, D>),
                            dim3(static_cast<unsigned>((rows + kMergeThreads / 32 - 1) / (kMergeThreads / 32))), kMergeThreads,
                            0, st, margs, "tile_merge_shared_kernel launch");
}

// Hooks of the failure-detection tests (unset in normal use), those of the split-K kernels: a short
// bound for the waits (a test suspends for up to 20 us: 64 of the others'), and the tiles of CTA 0's
// first run behind which its producers issue no copies any more.
void test_hooks(TileArgs &p) {
    const char *limit = std::getenv("GOLLEK_TEST_WAIT_LIMIT"), *skip = std::getenv("GOLLEK_TEST_SKIP_GROUP");
    p.wait_tries = limit ? std::max(1u, static_cast<unsigned>(std::strtoul(limit, nullptr, 10)) >> 6) : kSuspendTries;
    p.stop_at = skip ? std::atoi(skip) : -1;
}

// Held by a call that uses the library's scratch until its launches are in the stream: the plan, the
// attention and the merge of two host threads' calls on one stream would otherwise mix, one's
// kernels working from the other's plan.
std::mutex g_plan_mu;

int launch_tile(AttnArgs &a, void *ws, size_t ws_bytes, void *stream) {
    const CallPlan c = plan_call(a.num_groups, a.num_seqs, a.total_q, a.num_q_heads, a.num_kv_heads, a.head_dim);
    if (std::max(c.line[0].ws.max_blocks, c.line[1].ws.max_blocks) > (1LL << 22))
        return fail(GOLLEK_ERR_UNSUPPORTED, "too many query rows for one call");
    int dev = 0;
    GK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    std::unique_lock<std::mutex> whole_call(g_plan_mu, std::defer_lock);
    if (!ws) {
        whole_call.lock();
        // A graph would keep the library's scratch, which a larger call frees, and share it with other
        // graphs and calls.
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        GK_CUDA(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capturing), "cudaStreamIsCapturing");
        if (capturing != cudaStreamCaptureStatusNone)
            return fail(GOLLEK_ERR_WORKSPACE, "a call that is being captured needs a workspace of its own");
        int rc = library_workspace(dev, stream, Scratch::kPlan, c.total, &ws, &ws_bytes);
        if (rc) return rc;
    }
    if (ws_bytes < c.total)
        return fail(GOLLEK_ERR_WORKSPACE, "workspace of %zu bytes < %zu needed", ws_bytes, c.total);
    if (reinterpret_cast<uintptr_t>(ws) & 255) return fail(GOLLEK_ERR_INVALID_ARGUMENT, "workspace not 256-byte aligned");
    PlanArgs both{};
    for (int i = 0; i < 2; ++i) {
        const int from = std::min(i, c.lines - 1);  // one line stands twice
        const auto &l = c.line[from];
        const TileWs &w = l.ws;
        uint8_t *base = static_cast<uint8_t *>(ws) + l.at;
        TileArgs &p = both.line[i];
        p.a = a;
        p.head = reinterpret_cast<PlanHead *>(base);
        p.blks = reinterpret_cast<TileBlk *>(base + w.blks);
        p.cost = reinterpret_cast<long long *>(base + w.cost);
        p.ents = reinterpret_cast<int *>(base + w.ents);
        p.slots = reinterpret_cast<float *>(base + w.slots);
        // the rows' states are the call's, whatever line they come from
        p.ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(ws) + c.line[0].ws.ml);
        p.acc = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + c.line[0].ws.acc);
        p.ent0 = l.ent0;
        p.entities = l.entities;
        p.blk_rows = l.blk_rows;
        p.rows_min = l.rows_min;
        p.rows_max = l.rows_max;
        p.max_blocks = static_cast<int>(w.max_blocks);
        p.page_rows = a.page_stride / a.head_dim;
        test_hooks(p);
        p.grid = std::min(std::max(1, sm_count(dev)), kMaxTileCtas);
    }
    CUtensorMap tmk{}, tmv{};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.kv_dtype == GOLLEK_DTYPE_I8)  // copied without tensor maps
        return a.head_dim == 128 ? launch_tile_as<__nv_bfloat16, 128, true>(both, c.lines, tmk, tmv, st)
                                 : launch_tile_as<__nv_bfloat16, 64, true>(both, c.lines, tmk, tmv, st);
    const long long rows = a.num_blocks > 0 ? a.num_blocks * both.line[0].page_rows : (1LL << 31) - 8;
    const int box = std::min(a.block_size, 16);
    int rc = encode_tile_map(&tmk, a.k, a.kv_dtype, a.head_dim, rows, box);
    if (!rc) rc = encode_tile_map(&tmv, a.v, a.kv_dtype, a.head_dim, rows, box);
    if (rc) return rc;
    const bool bf16 = a.kv_dtype == GOLLEK_DTYPE_BF16;
    if (a.head_dim == 128)
        return bf16 ? launch_tile_as<__nv_bfloat16, 128>(both, c.lines, tmk, tmv, st)
                    : launch_tile_as<__half, 128>(both, c.lines, tmk, tmv, st);
    return bf16 ? launch_tile_as<__nv_bfloat16, 64>(both, c.lines, tmk, tmv, st)
                : launch_tile_as<__half, 64>(both, c.lines, tmk, tmv, st);
}

int launch_attn(AttnArgs &a, void *ws, size_t ws_bytes, void *stream) {
    if (tile_takes(a)) return launch_tile(a, ws, ws_bytes, stream);
    return launch_generic(a, static_cast<cudaStream_t>(stream));
}

size_t attn_workspace(int num_groups, int num_seqs, int total_q, int hq, int hkv, int D) {
    if (num_seqs <= 0 || total_q <= 0 || num_groups < 0 || hkv <= 0 || hq <= 0 || hq % hkv || D <= 0) return 0;
    return plan_call(num_groups, num_seqs, total_q, hq, hkv, D).total;
}

template <int KV>
const void *gather_fn(int out) {
    if (out == GOLLEK_DTYPE_F32) return reinterpret_cast<const void *>(&kv_gather_kernel<KV, float>);
    if (out == GOLLEK_DTYPE_BF16) return reinterpret_cast<const void *>(&kv_gather_kernel<KV, __nv_bfloat16>);
    return reinterpret_cast<const void *>(&kv_gather_kernel<KV, __half>);
}

// Whether every row is whole 8-element chunks at addresses that the vector loads and stores
// of kv_gather_kernel may use; its kernel, or null.
const void *gather_vectors(const GatherArgs &a) {
    if (a.head_dim % 8 || a.page_stride % 8 || !aligned16(a.key) || !aligned16(a.value)) return nullptr;
    if (static_cast<long long>(a.num_kv_heads) * a.head_dim > (1 << 20)) return nullptr;  // 32-bit chunk indexes
    const uintptr_t mask = a.kv_dtype == GOLLEK_DTYPE_I8 ? 7 : a.kv_dtype == GOLLEK_DTYPE_I4 ? 3 : 15;
    if ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & mask) return nullptr;
    switch (a.kv_dtype) {
        case GOLLEK_DTYPE_F32: return gather_fn<GOLLEK_DTYPE_F32>(a.out_dtype);
        case GOLLEK_DTYPE_BF16: return gather_fn<GOLLEK_DTYPE_BF16>(a.out_dtype);
        case GOLLEK_DTYPE_F16: return gather_fn<GOLLEK_DTYPE_F16>(a.out_dtype);
        case GOLLEK_DTYPE_I8: return gather_fn<GOLLEK_DTYPE_I8>(a.out_dtype);
        default: return gather_fn<GOLLEK_DTYPE_I4>(a.out_dtype);
    }
}

}  // namespace
}  // namespace gk

using namespace gk;

extern "C" {

int gollek_paged_attention_varlen(void *out, const void *q, const void *k_cache, const void *v_cache,
                                  const float *k_scales, const float *v_scales, const int *block_tables,
                                  const int *cu_seqlens_q, const int *context_lens, const float *alibi_slopes,
                                  const int *prefix_lens, const int *token_starts, int num_seqs, int total_queries,
                                  int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                  int max_blocks_per_seq, int num_blocks, long long page_stride, int q_dtype,
                                  int kv_dtype, long long scale_page_stride, long long scale_head_stride,
                                  long long scale_token_stride, float scale, float soft_cap, int sliding_window,
                                  int causal, void *workspace, size_t workspace_bytes, void *stream) {
    t_last_error.clear();
    AttnArgs a{};
    int rc = check_pool(kv_dtype, k_scales, v_scales, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks,
                        page_stride, &a.page_stride);
    if (rc) return rc;
    if (num_seqs < 0 || total_queries < 0 || total_queries > kMaxTokens)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "num_seqs or total_queries out of range");
    if (num_seqs == 0 || total_queries == 0) return GOLLEK_OK;
    if (!out || !q || !k_cache || !v_cache || !block_tables || !cu_seqlens_q || !context_lens)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!causal && sliding_window > 0)
        return fail(GOLLEK_ERR_UNSUPPORTED, "a sliding window without causal masking");
    a.out = out;
    a.q = q;
    a.k = k_cache;
    a.v = v_cache;
    a.k_scales = quantised(kv_dtype) ? k_scales : nullptr;
    a.v_scales = quantised(kv_dtype) ? v_scales : nullptr;
    a.block_tables = block_tables;
    a.context_lens = context_lens;
    a.cu = cu_seqlens_q;
    a.slopes = alibi_slopes;
    a.prefix_lens = prefix_lens;
    a.token_starts = token_starts;
    a.scale_page_stride = scale_page_stride;
    a.scale_head_stride = scale_head_stride;
    a.scale_token_stride = scale_token_stride;
    a.num_seqs = num_seqs;
    a.total_q = total_queries;
    a.num_q_heads = num_q_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.causal = causal != 0;
    a.window = sliding_window > 0 ? std::min<int>(sliding_window, 1 << 30) : 0;
    a.q_dtype = q_dtype;
    a.kv_dtype = kv_dtype;
    a.soft_cap = soft_cap > 0.f ? soft_cap : 0.f;
    a.q_scale = a.soft_cap > 0.f ? scale : scale * kLog2e;
    rc = check_attn(a);
    if (rc) return rc;
    return launch_attn(a, workspace, workspace_bytes, stream);
}

size_t gollek_paged_attention_varlen_workspace_size(int num_seqs, int total_queries, int num_q_heads, int num_kv_heads,
                                                    int head_dim) {
    return attn_workspace(0, num_seqs, total_queries, num_q_heads, num_kv_heads, head_dim);
}

int gollek_paged_attention_shared_prefix(void *out, const void *q, const void *k_cache, const void *v_cache,
                                         const float *k_scales, const float *v_scales, const int *prefix_tables,
                                         const int *prefix_lens, const int *group_starts, const int *block_tables,
                                         const int *context_lens, int num_groups, int max_prefix_blocks, int num_seqs,
                                         int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                         int max_blocks_per_seq, int num_blocks, long long page_stride, int q_dtype,
                                         int kv_dtype, long long scale_page_stride, long long scale_head_stride,
                                         long long scale_token_stride, float scale, float soft_cap, void *workspace,
                                         size_t workspace_bytes, void *stream) {
    t_last_error.clear();
    AttnArgs a{};
    int rc = check_pool(kv_dtype, k_scales, v_scales, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks,
                        page_stride, &a.page_stride);
    if (rc) return rc;
    if (num_seqs < 0 || num_groups <= 0 || max_prefix_blocks <= 0 ||
        static_cast<long long>(max_prefix_blocks) * block_size > kMaxTokens)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "num_seqs, num_groups or max_prefix_blocks out of range");
    if (num_seqs == 0) return GOLLEK_OK;
    if (!out || !q || !k_cache || !v_cache || !prefix_tables || !prefix_lens || !group_starts || !block_tables ||
        !context_lens)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "null tensor pointer");
    a.out = out;
    a.q = q;
    a.k = k_cache;
    a.v = v_cache;
    a.k_scales = quantised(kv_dtype) ? k_scales : nullptr;
    a.v_scales = quantised(kv_dtype) ? v_scales : nullptr;
    a.block_tables = block_tables;
    a.context_lens = context_lens;
    a.prefix_tables = prefix_tables;
    a.group_plens = prefix_lens;
    a.group_starts = group_starts;
    a.scale_page_stride = scale_page_stride;
    a.scale_head_stride = scale_head_stride;
    a.scale_token_stride = scale_token_stride;
    a.num_seqs = num_seqs;
    a.total_q = num_seqs;
    a.num_groups = num_groups;
    a.max_pblocks = max_prefix_blocks;
    a.num_q_heads = num_q_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.q_dtype = q_dtype;
    a.kv_dtype = kv_dtype;
    a.soft_cap = soft_cap > 0.f ? soft_cap : 0.f;
    a.q_scale = a.soft_cap > 0.f ? scale : scale * kLog2e;
    rc = check_attn(a);
    if (rc) return rc;
    return launch_attn(a, workspace, workspace_bytes, stream);
}

size_t gollek_paged_attention_shared_prefix_workspace_size(int num_groups, int num_seqs, int num_q_heads,
                                                           int num_kv_heads, int head_dim) {
    return num_groups <= 0 ? 0 : attn_workspace(num_groups, num_seqs, num_seqs, num_q_heads, num_kv_heads, head_dim);
}

int gollek_kv_gather(void *key, void *value, int out_dtype, const int *token_seq, const int *token_pos,
                     const int *block_tables, int num_seqs, int max_blocks_per_seq, int num_blocks,
                     const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
                     int kv_dtype, int num_tokens, int num_kv_heads, int head_dim, int block_size,
                     long long page_stride, long long scale_page_stride, long long scale_head_stride,
                     long long scale_token_stride, void *stream) {
    t_last_error.clear();
    GatherArgs a{};
    int rc = check_pool(kv_dtype, k_scales, v_scales, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks,
                        page_stride, &a.page_stride);
    if (rc) return rc;
    if (!float_dtype(out_dtype)) return fail(GOLLEK_ERR_UNSUPPORTED, "output dtype %d (F32, BF16 or F16 only)", out_dtype);
    if (num_tokens < 0 || num_seqs < 0) return fail(GOLLEK_ERR_INVALID_ARGUMENT, "negative size");
    if (num_tokens == 0) return GOLLEK_OK;
    if (!key || !value || !token_pos || !block_tables || !k_cache || !v_cache)
        return fail(GOLLEK_ERR_INVALID_ARGUMENT, "null tensor pointer");
    a.key = key;
    a.value = value;
    a.k = k_cache;
    a.v = v_cache;
    a.k_scales = quantised(kv_dtype) ? k_scales : nullptr;
    a.v_scales = quantised(kv_dtype) ? v_scales : nullptr;
    a.token_seq = token_seq;
    a.token_pos = token_pos;
    a.block_tables = block_tables;
    a.scale_page_stride = scale_page_stride;
    a.scale_head_stride = scale_head_stride;
    a.scale_token_stride = scale_token_stride;
    a.num_tokens = num_tokens;
    a.num_seqs = num_seqs;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.kv_dtype = kv_dtype;
    a.out_dtype = out_dtype;
    int dev = 0;
    GK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    const int sms = std::max(1, sm_count(dev));
    if (const void *fn = gather_vectors(a)) {
        // About 2048 chunks per block (8 a thread), fewer where that leaves fewer than four
        // blocks per SM.
        const int cpt = num_kv_heads * head_dim / 8;
        int tpb = std::min(std::max(2048 / cpt, 1), kGatherTokens);
        tpb = std::min(tpb, std::max(1, num_tokens / (4 * sms)));
        void *args[] = {&a, &tpb};
        GK_CUDA(cudaLaunchKernel(fn, dim3((num_tokens + tpb - 1) / tpb), dim3(kGatherThreads), args, 0,
                                 static_cast<cudaStream_t>(stream)),
                "kv_gather_kernel launch");
        return GOLLEK_OK;
    }
    const long long total = static_cast<long long>(num_tokens) * num_kv_heads * head_dim;
    const long long grid = std::min<long long>((total + 255) / 256, 32LL * sms);
    kv_gather_generic_kernel<<<static_cast<unsigned>(grid), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    GK_CUDA(cudaGetLastError(), "kv_gather_generic_kernel launch");
    return GOLLEK_OK;
}

}  // extern "C"
