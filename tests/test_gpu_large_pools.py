"""Pools past 4 GiB: the append by axes, windows with sinks and shared prefixes on the
last pages of a large pool give the bits that they give on a small one."""
import numpy as np
import pytest
import torch

import attn_f64 as A
from gpu_util import dev_f32, dev_i32, say
from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A
from lnskv.device import MRopeTable, PagedKV, PrefixGroups, RopeTable

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL, KV, REP = 120, 8, 4


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 128), (DTYPE_Q8A, 256), (DTYPE_F16, 64), (DTYPE_F32, 64)])
def test_the_last_pages_of_a_large_pool(dtype, d):
    say("large pool", dtype, d)
    rng = np.random.default_rng(12)
    page = 16 * KV * d * {DTYPE_F32: 4, DTYPE_F16: 2, DTYPE_Q8A: 1}[dtype]
    pages = (4 << 30) // page + 1000  # past 2^32 bytes
    small = PagedKV(SMALL, KV, d, dtype, DEV)
    A.fill(small, 4)
    big = PagedKV(pages, KV, d, dtype, DEV)
    off = pages - SMALL
    for name in ("k", "v"):
        getattr(big, name)[off:] = getattr(small, name)
    if dtype == DTYPE_Q8A:
        big.ks[off * 16:], big.vs[off * 16:] = small.ks, small.vs
    lens = [700, 620, 333]
    H, scale = KV * REP, 1.0 / np.sqrt(d)
    order = rng.permutation(SMALL)
    tables = np.full((3, 44), 0xFFFFFFFF, np.uint32)
    tables[0], tables[1, 20:39], tables[2, :21] = order[:44], order[44:63], order[63:84]
    tables[1, :20] = tables[0, :20]
    held = tables != 0xFFFFFFFF
    t_small, t_big = dev_i32(tables, DEV), dev_i32(np.where(held, tables + off, tables).astype(np.uint32), DEV)
    kl = dev_i32(np.array(lens, np.int32), DEV)
    rope = MRopeTable(RopeTable(64, 1e6, device=DEV).inv_freqs, [12, 10, 10])
    q, k, v = (dev_f32(rng.standard_normal((3, h, d)), DEV) for h in (H, KV, KV))
    axes, seqs = dev_i32(np.array([[5, 9, 70000]] * 3, np.int32), DEV), dev_i32(np.arange(3, dtype=np.int32), DEV)
    chunks, pq = dev_i32(np.array([[0, 640, 60, 0], [2, 300, 33, 60]], np.int32), DEV), dev_f32(rng.standard_normal((93, H, d)), DEV)
    got = []
    for pk, t in ((small, t_small), (big, t_big)):
        turned = pk.mrope_append(rope, k, v, axes, seqs, dev_i32(np.array(lens, np.int32) - 1, DEV), t, q=q)
        outs = [turned]
        for window, sink in ((100, 20), (600, 4)):
            outs.append(pk.sink_decode(turned, t, kl, n_heads=H, max_kv_len=700, scale=scale, window=window, n_sink=sink))
        outs.append(pk.prefix_decode(turned, t, kl, PrefixGroups([(0, 2, 320)]), n_heads=H, max_kv_len=700, scale=scale))
        if d != 64:
            outs.append(pk.sink_prefill_attention(pq, chunks, t, n_heads=H, scale=scale, window=200, n_sink=10))
        got.append(outs)
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert torch.equal(big.k[off:], small.k) and torch.equal(big.v[off:], small.v)
    assert not big.k[:off].any() and not big.v[:off].any()
