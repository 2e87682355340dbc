"""Ragged and shared-prefix paged attention and the cache read-back in 64 bits, from their
definitions (numpy, CPU), and the error bounds their kernels are held to."""
from __future__ import annotations

import numpy as np

# half a step relative to the value, by type
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Pool:
    """A paged cache: its stored form (arrays to upload) and its values in 64 bits."""

    def __init__(self, kind, k, v, scales="token"):
        """k, v: [NB, H, BS, D] float64; kind f32/bf16/f16/i8/i4; scales: per token or page."""
        self.kind, self.scales = kind, scales
        self.k, self.sk, self.fk = self._store(k)
        self.v, self.sv, self.fv = self._store(v)
        nb, h, bs, d = k.shape
        self.nb, self.h, self.bs, self.d = k.shape
        self.strides = ((h * bs, bs, 1) if scales == "token" else (h, 1, 0)) if kind in ("i8", "i4") else (0, 0, 0)

    def _store(self, x):
        import torch
        if self.kind in ("f32", "bf16", "f16"):
            t = torch.from_numpy(x).to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[self.kind])
            return t, None, t.double().numpy()
        top = 127 if self.kind == "i8" else 7
        fin = np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
        scale = (np.abs(fin).max(axis=3 if self.scales == "token" else (2, 3)) / top).astype(np.float32)
        scale = np.where(scale == 0, np.float32(1), scale)
        wide = scale[..., None] if self.scales == "token" else scale[:, :, None, None]
        q = np.clip(np.floor(fin / wide + 0.5), -top - (self.kind == "i4"), top)
        full = q * wide.astype(np.float64)
        if self.kind == "i8":
            stored = q.astype(np.int8)
        else:
            u = (q + 8).astype(np.uint8).reshape(x.shape[0], -1, 2)
            stored = np.ascontiguousarray(u[..., 0] | (u[..., 1] << 4))
        return torch.from_numpy(stored), torch.from_numpy(scale), full

    def rows(self, which, table, count):
        """[count, H, D]: the first `count` positions of one table row."""
        src = self.fk if which == "k" else self.fv
        pos = np.arange(count)
        return src[np.asarray(table)[pos // self.bs], :, pos % self.bs]

    def args(self, dev):
        up = lambda t: None if t is None else t.to(dev)
        return dict(k_cache=up(self.k), v_cache=up(self.v), k_scales=up(self.sk), v_scales=up(self.sv),
                    scale_strides=self.strides, num_kv_heads=self.h, block_size=self.bs, num_blocks=self.nb,
                    int4=self.kind == "i4")


def attend(q, k, v, seen, scale, bias=None, cap=0.0):
    """q [n, Hq, D], k/v [L, Hkv, D], seen [n, L], bias [Hq, n, L] or None -> (out, bound on
    |x| error units): softmax over the seen positions, zeros for rows without any."""
    n, hq, d = q.shape
    grp = hq // k.shape[1]
    out = np.zeros((n, hq, d))
    for h in range(hq):
        kk, vv = k[:, h // grp], v[:, h // grp]
        live = seen.any(axis=0)  # what nobody sees may hold anything
        x = np.full((n, k.shape[0]), -np.inf)
        x[:, live] = q[:, h] @ kk[live].T * scale
        if cap > 0:
            x = cap * np.tanh(x / cap)
        if bias is not None:
            x = x + bias[h]
        x = np.where(seen, x, -np.inf)
        some = seen.any(axis=1)
        if not some.any():
            continue
        x = x[some]
        p = np.exp(x - x.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[some, h] = p[:, live] @ vv[live]
    return out


def varlen(q, pool, tables, cu, ctx, scale, *, causal=True, window=0, slopes=None, prefix=None, starts=None, cap=0.0):
    """Definition of ragged attention; rows in no sequence are NaN (not written)."""
    out = np.full(q.shape, np.nan)
    for s in range(len(ctx)):
        n, c = int(cu[s + 1] - cu[s]), int(ctx[s])
        if n == 0:
            continue
        rows = slice(int(cu[s]), int(cu[s + 1]))
        pos = (c - n + np.arange(n))[:, None]
        key = np.arange(c)[None]
        hi = np.full((n, 1), c)
        if causal:
            hi = pos + 1
            if prefix is not None:
                hi = np.maximum(hi, min(int(prefix[s]), c))
        lo = np.zeros((n, 1), np.int64)
        if window > 0:
            lo = np.maximum(lo, pos - window + 1)
        if starts is not None:
            lo = np.maximum(lo, np.asarray(starts[rows])[:, None])
        seen = (key >= lo) & (key < hi)
        bias = None
        if slopes is not None:
            bias = -np.asarray(slopes, np.float64)[:, None, None] * np.abs(pos - key)[None]
        out[rows] = attend(q[rows], pool.rows("k", tables[s], c), pool.rows("v", tables[s], c), seen, scale, bias, cap)
    return out


def shared_prefix(q, pool, ptables, plens, starts, tables, ctx, scale, cap=0.0):
    out = np.zeros(q.shape)
    for s in range(len(ctx)):
        ks, vs = [], []
        for g in range(len(plens)):
            if starts[g] <= s < starts[g + 1]:
                ks.append(pool.rows("k", ptables[g], int(plens[g])))
                vs.append(pool.rows("v", ptables[g], int(plens[g])))
        ks.append(pool.rows("k", tables[s], int(ctx[s])))
        vs.append(pool.rows("v", tables[s], int(ctx[s])))
        k, v = np.concatenate(ks), np.concatenate(vs)
        out[s] = attend(q[s:s + 1], k, v, np.ones((1, len(k)), bool), scale, None, cap)[0]
    return out


def bound(want, q, pool, scale, qkind, *, p_kind=None, most_bias=0.0, cap=0.0):
    """Largest error of an output element.

    A score is a sum of D products in fp32: off by at most (D + 4) 2^-24 of
    sum |q||k| scale (the + 4: scale, cap, bias and the change of base), and the bias and the
    capped score by 2^-23 of their size; exp2 and its argument add 2^-21.  A relative error e
    of every probability moves a weighted mean of values by at most 2 e max|v|.  The tile
    kernel rounds each probability to p_kind before the value product (the normaliser keeps
    the unrounded ones): e grows by that type's half step, once.  Sums over positions and the
    merge of partial states are fp32 with at most a few hundred terms a thread: 2^-16 covers
    them.  The result is rounded once to the output type."""
    fin = lambda x: np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    qk = scale * np.abs(fin(q)).sum(-1).max() * np.abs(fin(pool.fk)).max()
    if cap > 0:
        qk = max(qk, 4 * cap)
    vmax = np.abs(fin(pool.fv)).max()
    e = (q.shape[-1] + 4) * 2.0 ** -24 * qk + 2.0 ** -23 * (most_bias + qk) + 2.0 ** -21
    e = 2 * e + 2.0 ** -16
    if p_kind:
        e += HALF_STEP[p_kind]
    return e * vmax + HALF_STEP[qkind] * np.abs(want)
