"""Sharper checks of paged attention than an element's worst case (tests/paged_ref.py): pools whose outputs count
positions, and the norm of a row's error.  Both see one page, and the first one position, that is left out or taken
twice in thousands."""
from __future__ import annotations

import numpy as np

from tests import paged_ref as R

# a value whose int8 (127 / 128) and int4 (7 / 8) scales are powers of two, so that no type rounds it
ONE = {"i8": 127 / 128, "i4": 7 / 8}


def counting_pool(kind, tables, lens, hkv, d, bs, nb, rng, dead=np.nan):
    """V rows that are one-hot: head h of position j is 1 (ONE of quantised types) in column j % d (even h) or
    j // d % d (odd h).  With q = 0 every visible position has the same weight, exactly, and an output column is the
    share of the visible positions that fall on it.  Slots of nobody hold `dead`."""
    k = rng.standard_normal((nb, hkv, bs, d))
    v = np.full((nb, hkv, bs, d), dead)
    k[:] = np.where(np.isnan(dead), np.nan, k)
    for row, c in zip(tables, lens):
        pos = np.arange(int(c))
        page, slot = np.asarray(row)[pos // bs], pos % bs
        for h in range(hkv):
            col = pos // d % d if h & 1 else pos % d
            v[page, h, slot] = 0.0
            v[page, h, slot, col] = ONE.get(kind, 1.0)
            k[page, h, slot] = rng.standard_normal((len(pos), d))
    return R.Pool(kind, k, v)


def counts_agree(got, want, qkind):
    """Elementwise: zero exactly where no position falls on the column; else one rounding of the output, with
    2^-20 for the reciprocal of the sum and the factors 2^0 of exp2."""
    tol = (R.HALF_STEP[qkind] + 2.0 ** -20) * want
    return bool((np.abs(got - want) <= tol).all())


def norms_agree(got, want, q, pool, scale, qkind, *, p_kind=None, most_bias=0.0, cap=0.0):
    """Per (row, head): |got - want|_2 <= (h_p + h_out) |want| + 2 e max|v_j|_2.

    Each probability is rounded by at most h_p relative, all columns alike, independently of the others: the error
    is sum_j p_j d_j v_j with |d_j| <= h_p.  For values that are independent and of mean zero its square is D sum
    p_j^2 d_j^2 <= h_p^2 |want|^2 up to the correlations of different v_j, about D^-1/2, which the rounding's own spread
    (a root mean square of 0.4 h_p) outweighs.  The output's rounding adds h_out |want|.  An error e of every score moves
    the weighted mean by at most 2 e of the longest value row (e: as tests/paged_ref.py derives it; |q . k| by
    Cauchy-Schwarz)."""
    fin = lambda x: np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    norm = lambda x: np.sqrt((fin(x) ** 2).sum(-1))
    qk = scale * norm(q).max() * norm(pool.fk).max()
    size = max(qk, 4 * cap) if cap > 0 else qk
    e = (q.shape[-1] + 4) * 2.0 ** -24 * size + 2.0 ** -23 * (most_bias + size) + 2.0 ** -21
    h = R.HALF_STEP[qkind] + (R.HALF_STEP[p_kind] if p_kind else 0.0) + 2.0 ** -16
    return bool((norm(got - want) <= h * norm(want) + 2 * e * norm(pool.fv).max()).all())
