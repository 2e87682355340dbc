"""Tensor-level wrappers over the C ABI (torch CUDA tensors in, status checked).

Every function here is a thin call into libgollek_kernels.so on the tensors' device
and the current torch stream; none has a CPU path.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from ._lib import BF16, F16, F32, I4, I8, check

_FLOAT = (torch.float32, torch.bfloat16, torch.float16)
_TORCH_DTYPE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.int8: I8}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor, stream=None):
    if stream is not None:
        return stream.cuda_stream if hasattr(stream, "cuda_stream") else stream
    return torch.cuda.current_stream(t.device).cuda_stream


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("gollek_b200 ops take CUDA tensors only (no CPU path)")


def kv_dtype_code(t: torch.Tensor, int4: bool = False) -> int:
    if int4:
        return I4
    if t.dtype not in _TORCH_DTYPE:
        raise ValueError(f"unsupported KV dtype {t.dtype}")
    return _TORCH_DTYPE[t.dtype]


def workspace_size(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    return int(_lib.load().gollek_paged_attention_workspace_size(num_seqs, num_q_heads,
                                                                 num_kv_heads, head_dim))


def new_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, device) -> torch.Tensor:
    """Caller-owned split-K scratch, zero-filled (the kernels leave it zeroed)."""
    n = workspace_size(num_seqs, num_q_heads, num_kv_heads, head_dim)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_attention(q, k_cache, v_cache, block_tables, context_lens, *, num_kv_heads,
                    block_size, scale=None, num_blocks=0, page_stride=0, k_scales=None,
                    v_scales=None, scale_strides=(0, 0, 0), soft_cap=0.0, sliding_window=0,
                    int4=False, out=None, workspace=None, stream=None):
    """Decode attention (gollek_paged_attention_v2).

    q: [S, Hq, D] fp32/bf16.  k_cache/v_cache: pool tensors (any shape) whose element
    (page p, head h, token t, dim d) sits at p*page_stride + (h*BS + t)*D + d.
    """
    _require_cuda(q, k_cache, v_cache, block_tables, context_lens, k_scales, v_scales, out)
    S, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty_like(q)
    sps, shs, sts = scale_strides
    lib = _lib.load()
    rc = lib.gollek_paged_attention_v2(
        _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scales), _ptr(v_scales),
        _ptr(block_tables), _ptr(context_lens), S, Hq, int(num_kv_heads), D, int(block_size),
        block_tables.shape[1], int(num_blocks), int(page_stride), _TORCH_DTYPE[q.dtype],
        kv_dtype_code(k_cache, int4), int(sps), int(shs), int(sts), float(scale),
        float(soft_cap), int(sliding_window), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(),
        _stream(q, stream))
    check(rc)
    return out


def paged_attention_prefill(q, k_cache, v_cache, block_tables, context_lens, *, num_kv_heads,
                            block_size, scale=None, causal=True, num_blocks=0, page_stride=0,
                            k_scales=None, v_scales=None, scale_strides=(0, 0, 0), soft_cap=0.0,
                            sliding_window=0, int4=False, out=None, workspace=None, stream=None):
    """Multi-query attention (gollek_paged_attention_prefill): q [S, Tq, Hq, D]; the Tq
    queries of sequence s sit at positions context_lens[s] - Tq .. context_lens[s] - 1."""
    _require_cuda(q, k_cache, v_cache, block_tables, context_lens, k_scales, v_scales, out)
    S, Tq, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty_like(q)
    sps, shs, sts = scale_strides
    rc = _lib.load().gollek_paged_attention_prefill(
        _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scales), _ptr(v_scales),
        _ptr(block_tables), _ptr(context_lens), S, Tq, Hq, int(num_kv_heads), D, int(block_size),
        block_tables.shape[1], int(num_blocks), int(page_stride), _TORCH_DTYPE[q.dtype],
        kv_dtype_code(k_cache, int4), int(sps), int(shs), int(sts), float(scale),
        float(soft_cap), int(sliding_window), int(bool(causal)), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(),
        _stream(q, stream))
    check(rc)
    return out


def paged_attention_launch(out, q, k_cache, v_cache, block_tables, context_lens, scale):
    """The legacy fp32 entry point (synchronous): q/out [S,H,D], K/V [NB,H,BS,D]."""
    _require_cuda(out, q, k_cache, v_cache, block_tables, context_lens)
    S, H, D = q.shape
    rc = _lib.load().paged_attention_launch(
        _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables), _ptr(context_lens),
        S, H, D, k_cache.shape[2], block_tables.shape[1], float(scale))
    check(rc)
    return out


def kv_append(key, value, token_pos, block_tables, k_cache, v_cache, *, block_size,
              num_blocks=0, token_seq=None, page_stride=0, k_scales=None, v_scales=None,
              scale_strides=(0, 0, 0), int4=False, stream=None):
    """Write [T, Hkv, D] key/value rows into their pages (gollek_kv_append)."""
    _require_cuda(key, value, token_pos, block_tables, k_cache, v_cache, token_seq, k_scales,
                  v_scales)
    T, Hkv, D = key.shape
    sps, shs, sts = scale_strides
    rc = _lib.load().gollek_kv_append(
        _ptr(key), _ptr(value), _TORCH_DTYPE[key.dtype], _ptr(token_seq), _ptr(token_pos),
        _ptr(block_tables), block_tables.shape[1], int(num_blocks), _ptr(k_cache), _ptr(v_cache),
        _ptr(k_scales), _ptr(v_scales), kv_dtype_code(k_cache, int4), T, Hkv, D, int(block_size),
        int(page_stride), int(sps), int(shs), int(sts), _stream(key, stream))
    check(rc)


def _check(name, t, shape, dtype, device, packed=True):
    """Shape (None: any size), type (None: any), device and layout of one argument; says what
    is wrong with it."""
    if t is None:
        raise ValueError(f"{name} is required")
    if t.device.type != "cuda":
        raise ValueError("gollek_b200 ops take CUDA tensors only (no CPU path)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if shape is not None and (t.dim() != len(shape) or
                              any(w is not None and w != n for w, n in zip(shape, t.shape))):
        raise ValueError(f"{name} must have shape {tuple('*' if w is None else w for w in shape)}, "
                         f"not {tuple(t.shape)}")
    if packed and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_vectors(device, rows):
    """_check of 1-D arguments, (name, tensor, length, dtype) each, None tensors skipped: the
    common case in as few Python steps as possible, since small calls wait for them."""
    for name, t, n, dtype in rows:
        if t is not None and not (t.dtype is dtype and t.shape == (n,) and t.device == device
                                  and t.is_contiguous()):
            _check(name, t, (n,), dtype, device)


def _first(name, t, dims):
    """The argument that fixes the device: a contiguous CUDA tensor of `dims` dimensions."""
    if t is None or t.device.type != "cuda" or t.dim() != dims or not t.is_contiguous():
        _check(name, t, (None,) * dims, None, None if t is None else t.device)
    return t.device


def _behind(t):
    """Elements from a tensor's first one to the end of its storage: what a base pointer with
    strides of its own (one layer of a pool) may reach."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


def _check_pool(k_cache, v_cache, k_scales, v_scales, scale_strides, num_kv_heads, head_dim,
                block_size, num_blocks, page_stride, int4, device):
    """A K/V pool: both caches of one type (int4: bytes) on `device`, reaching num_blocks
    pages (scales too) when that is given.  With page_stride the tensors are base pointers
    (one layer of a larger pool); without it they are whole and contiguous."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t is None or t.device != device or not (page_stride or t.is_contiguous()):
            _check(name, t, None, None, device, packed=not page_stride)
        if int4:
            if t.dtype not in (torch.uint8, torch.int8):
                raise ValueError(f"an int4 {name} is a tensor of bytes, not {t.dtype}")
        elif t.dtype not in _TORCH_DTYPE:
            raise ValueError(f"unsupported KV dtype {t.dtype}")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache have different types")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t is not None and (t.dtype is not torch.float32 or t.device != device):
            _check(name, t, None, torch.float32, device, packed=False)
    if num_blocks > 0 and num_kv_heads > 0 and block_size > 0 and head_dim > 0:
        page = num_kv_heads * block_size * head_dim
        need = (num_blocks - 1) * (page_stride or page) + page
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
            have = _behind(t) if page_stride else t.numel()
            if have * (2 if int4 else 1) < need:
                raise ValueError(f"{name} is smaller than {num_blocks} pages")
        if int4 or k_cache.dtype is torch.int8:
            sps, shs, sts = scale_strides
            last = (num_blocks - 1) * sps + (num_kv_heads - 1) * shs + (block_size - 1) * sts
            for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
                if t is not None and (min(sps, shs, sts) < 0 or _behind(t) <= last):
                    raise ValueError(f"{name} is smaller than {num_blocks} pages of its strides")


class _on:
    """Runs a call on the device of its tensors and on `stream` (default: that device's
    current stream); what is allocated inside belongs to that stream."""

    def __init__(self, device, stream):
        self.device, self.given = device, stream

    def __enter__(self):
        self.guard = None
        if self.given is None and torch._C._cuda_getDevice() == self.device.index:
            return torch._C._cuda_getCurrentRawStream(self.device.index)
        if self.given is not None:
            s = self.given
            if getattr(s, "device", self.device) != self.device:
                raise ValueError(f"stream is on {s.device}, not {self.device}")
            if not hasattr(s, "cuda_stream"):
                s = torch.cuda.ExternalStream(int(s), device=self.device)
            self.guard = torch.cuda.stream(s)
        else:
            self.guard = torch.cuda.device(self.device)
        self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _scratch(need, workspace, device):
    """The caller's workspace (checked), or a fresh one from torch's allocator: stream
    ordered, and private to a captured graph."""
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None, need
    _check("workspace", workspace, None, None, device)
    return workspace, workspace.numel() * workspace.element_size()


@functools.lru_cache(maxsize=1024)
def varlen_workspace_size(num_seqs, total_queries, num_q_heads, num_kv_heads, head_dim) -> int:
    return int(_lib.load().gollek_paged_attention_varlen_workspace_size(
        num_seqs, total_queries, num_q_heads, num_kv_heads, head_dim))


def paged_attention_varlen(q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, *,
                           num_kv_heads, block_size, scale=None, causal=True, num_blocks=0,
                           page_stride=0, k_scales=None, v_scales=None, scale_strides=(0, 0, 0),
                           soft_cap=0.0, sliding_window=0, alibi_slopes=None, prefix_lens=None,
                           token_starts=None, int4=False, out=None, workspace=None, stream=None):
    """Ragged attention (gollek_paged_attention_varlen): q [total, Hq, D] fp32/bf16/f16, the
    queries of sequence s in rows cu_seqlens_q[s] .. cu_seqlens_q[s+1] - 1, the last of them
    at position context_lens[s] - 1.

    alibi_slopes [Hq] subtracts slope * |distance| from the scores; prefix_lens [S] makes each
    sequence's first positions visible to all its queries; token_starts [total] is the first
    position each query may attend.  Rows of `out` in no sequence are not written.
    """
    dev = _first("q", q, 3)
    total, Hq, D = q.shape
    if q.dtype not in _FLOAT:
        raise ValueError(f"unsupported q dtype {q.dtype}")
    _check("block_tables", block_tables, (None, None), torch.int32, dev)
    S, width = block_tables.shape
    _check_vectors(dev, (("cu_seqlens_q", cu_seqlens_q, S + 1, torch.int32),
                         ("context_lens", context_lens, S, torch.int32),
                         ("alibi_slopes", alibi_slopes, Hq, torch.float32),
                         ("prefix_lens", prefix_lens, S, torch.int32),
                         ("token_starts", token_starts, total, torch.int32)))
    if cu_seqlens_q is None or context_lens is None:
        raise ValueError("cu_seqlens_q and context_lens are required")
    if out is not None:
        _check("out", out, q.shape, q.dtype, dev)
    _check_pool(k_cache, v_cache, k_scales, v_scales, scale_strides, int(num_kv_heads), D,
                int(block_size), int(num_blocks), int(page_stride), int4, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    sps, shs, sts = scale_strides
    lib = _lib.load()
    with _on(dev, stream) as st:
        if out is None:
            out = torch.empty_like(q)
        ws, nbytes = _scratch(0 if workspace is not None else varlen_workspace_size(
            S, total, Hq, int(num_kv_heads), D), workspace, dev)
        check(lib.gollek_paged_attention_varlen(
            _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scales), _ptr(v_scales),
            _ptr(block_tables), _ptr(cu_seqlens_q), _ptr(context_lens), _ptr(alibi_slopes),
            _ptr(prefix_lens), _ptr(token_starts), S, total, Hq, int(num_kv_heads), D,
            int(block_size), width, int(num_blocks), int(page_stride),
            _TORCH_DTYPE[q.dtype], kv_dtype_code(k_cache, int4), int(sps), int(shs), int(sts),
            float(scale), float(soft_cap), int(sliding_window), int(bool(causal)), _ptr(ws),
            nbytes, st))
    return out


@functools.lru_cache(maxsize=1024)
def shared_prefix_workspace_size(num_groups, num_seqs, num_q_heads, num_kv_heads, head_dim) -> int:
    return int(_lib.load().gollek_paged_attention_shared_prefix_workspace_size(
        num_groups, num_seqs, num_q_heads, num_kv_heads, head_dim))


def paged_attention_shared_prefix(q, k_cache, v_cache, prefix_tables, prefix_lens, group_starts,
                                  block_tables, context_lens, *, num_kv_heads, block_size,
                                  scale=None, num_blocks=0, page_stride=0, k_scales=None,
                                  v_scales=None, scale_strides=(0, 0, 0), soft_cap=0.0, int4=False,
                                  out=None, workspace=None, stream=None):
    """Decode attention of groups that share prefixes (gollek_paged_attention_shared_prefix):
    q [S, Hq, D] fp32/bf16/f16; sequences group_starts[g] .. group_starts[g+1] - 1 attend the
    prefix_lens[g] tokens of prefix_tables[g] and their own context_lens[s] tokens.  The tensor-core
    kernels read a prefix once for 256 of its group's rows, the generic kernel (fp32 and int4
    caches, q of another type, other head_dims) once per sequence."""
    dev = _first("q", q, 3)
    S, Hq, D = q.shape
    if q.dtype not in _FLOAT:
        raise ValueError(f"unsupported q dtype {q.dtype}")
    _check("prefix_tables", prefix_tables, (None, None), torch.int32, dev)
    groups = prefix_tables.shape[0]
    _check("block_tables", block_tables, (S, None), torch.int32, dev)
    _check_vectors(dev, (("prefix_lens", prefix_lens, groups, torch.int32),
                         ("group_starts", group_starts, groups + 1, torch.int32),
                         ("context_lens", context_lens, S, torch.int32)))
    if prefix_lens is None or group_starts is None or context_lens is None:
        raise ValueError("prefix_lens, group_starts and context_lens are required")
    if out is not None:
        _check("out", out, q.shape, q.dtype, dev)
    _check_pool(k_cache, v_cache, k_scales, v_scales, scale_strides, int(num_kv_heads), D,
                int(block_size), int(num_blocks), int(page_stride), int4, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    sps, shs, sts = scale_strides
    lib = _lib.load()
    with _on(dev, stream) as st:
        if out is None:
            out = torch.empty_like(q)
        ws, nbytes = _scratch(0 if workspace is not None else shared_prefix_workspace_size(
            groups, S, Hq, int(num_kv_heads), D), workspace, dev)
        check(lib.gollek_paged_attention_shared_prefix(
            _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scales), _ptr(v_scales),
            _ptr(prefix_tables), _ptr(prefix_lens), _ptr(group_starts), _ptr(block_tables),
            _ptr(context_lens), groups, prefix_tables.shape[1], S, Hq, int(num_kv_heads), D,
            int(block_size), block_tables.shape[1], int(num_blocks), int(page_stride),
            _TORCH_DTYPE[q.dtype], kv_dtype_code(k_cache, int4), int(sps), int(shs), int(sts),
            float(scale), float(soft_cap), _ptr(ws), nbytes, st))
    return out


def kv_gather(k_cache, v_cache, token_pos, block_tables, *, num_kv_heads, head_dim, block_size,
              num_blocks=0, token_seq=None, page_stride=0, k_scales=None, v_scales=None,
              scale_strides=(0, 0, 0), int4=False, dtype=torch.float32, key=None, value=None,
              stream=None):
    """Read rows of the cache back (gollek_kv_gather): (key, value), each [T, Hkv, head_dim] of
    `dtype` (fp32/bf16/f16), dequantised; row i is position token_pos[i] of sequence
    token_seq[i] (default: i)."""
    dev = _first("token_pos", token_pos, 1)
    T = token_pos.shape[0]
    _check_vectors(dev, (("token_pos", token_pos, T, torch.int32),
                         ("token_seq", token_seq, T, torch.int32)))
    _check("block_tables", block_tables, (None, None), torch.int32, dev)
    if dtype not in _FLOAT:
        raise ValueError(f"unsupported output dtype {dtype}")
    shape = (T, int(num_kv_heads), int(head_dim))
    if key is not None:
        _check("key", key, shape, dtype, dev)
    if value is not None:
        _check("value", value, shape, dtype, dev)
    _check_pool(k_cache, v_cache, k_scales, v_scales, scale_strides, int(num_kv_heads),
                int(head_dim), int(block_size), int(num_blocks), int(page_stride), int4, dev)
    sps, shs, sts = scale_strides
    with _on(dev, stream) as st:
        key = torch.empty(shape, dtype=dtype, device=dev) if key is None else key
        value = torch.empty(shape, dtype=dtype, device=dev) if value is None else value
        check(_lib.load().gollek_kv_gather(
            _ptr(key), _ptr(value), _TORCH_DTYPE[dtype], _ptr(token_seq), _ptr(token_pos),
            _ptr(block_tables), block_tables.shape[0], block_tables.shape[1], int(num_blocks),
            _ptr(k_cache), _ptr(v_cache), _ptr(k_scales), _ptr(v_scales),
            kv_dtype_code(k_cache, int4), T, int(num_kv_heads), int(head_dim), int(block_size),
            int(page_stride), int(sps), int(shs), int(sts), st))
    return key, value


def pool_blocks(pool, block_stride, bytes_per_block) -> int:
    """Whole blocks of `bytes_per_block` bytes, `block_stride` bytes apart, that fit in
    the tensor `pool` (the bound the migration and checksum kernels check ids against)."""
    nbytes = pool.numel() * pool.element_size()
    if nbytes < bytes_per_block or block_stride <= 0:
        return 0 if block_stride <= 0 else -1
    return (nbytes - bytes_per_block) // block_stride + 1


def kv_migrate(src_k, src_v, dst_k, dst_v, src_blocks, dst_blocks, *, src_block_stride,
               dst_block_stride, bytes_per_block, device=None, stream=None, dst_k_ptr=None,
               dst_v_ptr=None, src_num_blocks=None, dst_num_blocks=None):
    """Block-remapped copy (gollek_kv_migrate).  Strides/sizes in bytes.

    dst_k_ptr/dst_v_ptr override the destination with raw device addresses (a peer
    pointer mapped through CUDA IPC); give dst_num_blocks with them.  Pool sizes default
    to what the tensors hold, so ids outside a pool are skipped on the device and
    reported by device_status() (GOLLEK_STATUS_BAD_BLOCK_ID)."""
    dev = src_k.device.index if device is None else device
    dk = dst_k_ptr if dst_k_ptr is not None else _ptr(dst_k)
    dv = dst_v_ptr if dst_v_ptr is not None else _ptr(dst_v)
    if src_num_blocks is None:
        src_num_blocks = pool_blocks(src_k, src_block_stride, bytes_per_block)
    if dst_num_blocks is None:
        dst_num_blocks = (pool_blocks(dst_k, dst_block_stride, bytes_per_block)
                          if dst_k_ptr is None else 0)
    if src_num_blocks < 0 or dst_num_blocks < 0:
        raise ValueError("a pool tensor is smaller than one block")
    rc = _lib.load().gollek_kv_migrate(
        _ptr(src_k), _ptr(src_v), dk, dv, _ptr(src_blocks), _ptr(dst_blocks), src_blocks.numel(),
        int(src_num_blocks), int(dst_num_blocks), int(src_block_stride), int(dst_block_stride),
        int(bytes_per_block), int(dev), _stream(src_k, stream))
    check(rc)


def block_checksums(pool, blocks, *, block_stride, bytes_per_block, num_blocks=None, stream=None):
    """Per-block 64-bit checksums (gollek_kv_block_checksum) as an int64 tensor."""
    if num_blocks is None:
        num_blocks = pool_blocks(pool, block_stride, bytes_per_block)
    if num_blocks < 0:
        raise ValueError("the pool tensor is smaller than one block")
    out = torch.empty(blocks.numel(), dtype=torch.int64, device=pool.device)
    rc = _lib.load().gollek_kv_block_checksum(_ptr(pool), _ptr(blocks), blocks.numel(),
                                              int(num_blocks), int(block_stride),
                                              int(bytes_per_block), _ptr(out), _stream(pool, stream))
    check(rc)
    return out


def device_status(device: int = 0, clear: bool = True) -> int:
    import ctypes
    v = ctypes.c_uint(0)
    check(_lib.load().gollek_device_status(int(device), int(clear), ctypes.byref(v)))
    return int(v.value)


def enable_peer_access(device: int, peer: int) -> None:
    check(_lib.load().gollek_enable_peer_access(int(device), int(peer)))
