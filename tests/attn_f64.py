"""Attention over paged K/V in 64 bits, one query row at a time (not collected).

`TOL` is what the kernels' results may be off, as the largest error of a row
relative to its largest value.  Queries and weights are carried as pairs of f16
(2^-22 relative), as three int8 limbs (2^-17 of the largest) or in f32, sums in f32:
a score of the tests' inputs (|score| < 32 in log2 units) is off by at most about
32 * 2^-22 + 16 * 2^-24 * 32 = 4e-5 in the worst case and 1e-6 typically (errors of
d products add like a random walk), a weight by that times ln 2, and an output row
averages the errors of its weights."""
from __future__ import annotations

import numpy as np
import torch

from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A
from lnskv.device import PagedKV

TOL = 1e-5
DTYPES = [DTYPE_F32, DTYPE_F16, DTYPE_Q8A]


def values(pk: PagedKV) -> tuple[np.ndarray, np.ndarray]:
    """K and V of every slot as f64 [slots][n_kv][d]."""
    out = []
    for t, sc in ((pk.k, pk.ks), (pk.v, pk.vs)):
        x = t.cpu().numpy().astype(np.float64).reshape(-1, pk.n_kv, pk.head_dim)
        out.append(x if sc is None else x * sc.cpu().numpy().astype(np.float64)[..., None])
    return out[0], out[1]


def row(kv, q, slots, scale: float) -> np.ndarray:
    """One query row q [n_heads][d] over the slots it attends."""
    K, V = kv
    n_kv, d = K.shape[1:]
    rep = q.shape[0] // n_kv
    if len(slots) == 0:
        return np.zeros(q.shape)
    qh = q.astype(np.float64).reshape(n_kv, rep, d)
    s = np.einsum("hrd,thd->hrt", qh, K[slots]) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    o = np.einsum("hrt,thd->hrd", p, V[slots]) / p.sum(-1, keepdims=True)
    return o.reshape(q.shape)


def slots_of(table, tokens, num_pages: int) -> np.ndarray:
    """Slots of the tokens of a table row whose page exists."""
    t = np.asarray(list(tokens), np.int64)
    if len(t) == 0:
        return t
    page = np.asarray(table)[t // 16].astype(np.int64) & 0xFFFFFFFF
    ok = page < num_pages
    return (page * 16 + t % 16)[ok]


def worst(out: torch.Tensor, ref: np.ndarray) -> float:
    """Largest row error relative to the row's largest value; rows of zeros must be zeros."""
    o = out.cpu().numpy().astype(np.float64).reshape(-1, ref.shape[-1])
    r = ref.reshape(-1, ref.shape[-1])
    assert np.isfinite(o).all()
    top = np.abs(r).max(-1)
    err = np.abs(o - r).max(-1)
    assert (err[top == 0] == 0).all()
    return float((err[top > 0] / top[top > 0]).max(initial=0.0))


def make_tables(lens, held, rng, extra: int = 2):
    """Tables [n][stride] (uint32) with a page of its own for every logical page in
    held[s]; the other entries hold NO_PAGE.  Returns (tables, number of pages)."""
    stride = max(1, max(-(-max(L, 1) // 16) for L in lens))
    n = sum(len(h) for h in held) + extra
    order = rng.permutation(n).astype(np.uint32)
    t = np.full((len(lens), stride), 0xFFFFFFFF, np.uint32)
    at = 0
    for s, h in enumerate(held):
        for p in h:
            t[s, p] = order[at]
            at += 1
    return t, n


def fill(pk: PagedKV, seed: int) -> None:
    """N(0, 1) K and V (Q8A: codes and scales of that size)."""
    g = torch.Generator(device=pk.device).manual_seed(seed)
    if pk.dtype == DTYPE_Q8A:
        for t in (pk.k, pk.v):
            t.copy_((torch.randn(t.shape, generator=g, device=pk.device) * 32).round().clamp(-127, 127).to(torch.int8))
        for t in (pk.ks, pk.vs):
            t.copy_(torch.rand(t.shape, generator=g, device=pk.device) * 0.02 + 0.02)
        return
    for t in (pk.k, pk.v):
        t.copy_(torch.randn(t.shape, generator=g, device=pk.device).to(t.dtype))


def poison(pk: PagedKV, attended: np.ndarray) -> None:
    """NaN and infinities in every slot that nothing attends (Q8A: in their scales)."""
    mask = torch.ones(pk.num_pages * 16, dtype=torch.bool, device=pk.device)
    mask[torch.from_numpy(np.unique(attended)).to(pk.device)] = False
    bad = torch.where(torch.arange(mask.numel(), device=pk.device) % 3 == 0, float("inf"), float("nan"))[mask]
    if pk.dtype == DTYPE_Q8A:
        pk.ks[mask] = bad[:, None].expand(-1, pk.n_kv)
        pk.vs[mask] = bad[:, None].expand(-1, pk.n_kv)
        return
    shape = (-1, pk.n_kv, pk.head_dim)
    for t in (pk.k, pk.v):
        t.view(shape)[mask] = bad[:, None, None].expand(shape[0], *shape[1:]).to(t.dtype)


__all__ = ["DTYPES", "TOL", "fill", "make_tables", "poison", "row", "slots_of", "values", "worst", "DTYPE_F16",
           "DTYPE_F32", "DTYPE_Q8A"]
