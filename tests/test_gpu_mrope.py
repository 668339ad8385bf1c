"""The append with rotary positions of several axes on the GPU (lnskv_mrope_append),
bit for bit against numpy: angles, sines and cosines in f64, rounded once; the turn in
f32, each product and sum rounded; the page conversions of lnskv_append."""
import numpy as np
import pytest
import torch

import attn_f64 as A
from gpu_util import dev_f32, dev_i32, say
from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A
from lnskv.device import MRopeTable, PagedKV, RopeTable

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def axis_of(sections, interleaved):
    n, half = len(sections), sum(sections)
    if interleaved:
        return [i % n if i % n and i < n * sections[i % n] else 0 for i in range(half)]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def turn(x, pos, inv, axis):
    """x [tok][heads][d] f32 turned; pos [axes][tok]."""
    half = len(axis)
    ang = pos[axis].T.astype(np.float64) * inv.astype(np.float64)[None, :]
    c, s = np.cos(ang).astype(np.float32)[:, None], np.sin(ang).astype(np.float32)[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def store(dtype, pools, slot, rows):
    """rows [kv][d] f32 into the slot of (data, scales)."""
    data, scales = pools
    if dtype == DTYPE_Q8A:
        amax = np.abs(rows).max(-1)
        sc = np.where(amax == 0, np.float32(1), amax / np.float32(127)).astype(np.float32)
        y = (rows / sc[:, None]).astype(np.float32).astype(np.float64)
        data[slot] = np.clip(np.sign(y) * np.floor(np.abs(y) + 0.5), -127, 127).astype(np.int8)
        scales[slot] = sc
    else:
        data[slot] = rows.astype(data.dtype)


def run(dtype, d, kv, H, sections, interleaved, toks, far, seed, odd=False, inplace=False, with_q=True):
    """toks: (table row, position) of each token."""
    rng = np.random.default_rng(seed)
    n, rows, stride = len(toks), 3, 6
    tables = rng.permutation(rows * stride + 2)[:rows * stride].reshape(rows, stride).astype(np.uint32)
    tables[2, 3] = 0xFFFFFFFF
    tables[2, 4] = 5000
    num_pages = rows * stride + 2
    pk = PagedKV(num_pages, kv, d, dtype, DEV)
    A.fill(pk, seed)
    inv = RopeTable(2 * sum(sections), 1e6, device=DEV)
    rope = MRopeTable(inv.inv_freqs, sections, interleaved)
    mk = lambda h: rng.standard_normal((n, h, d)).astype(np.float32) * np.exp(rng.standard_normal((n, h, 1))).astype(np.float32)  # noqa: E731
    q, k, v = mk(H), mk(kv), mk(kv)
    if n > 2:
        k[1] = 0.0
    pos = rng.integers(-far, far, (len(sections), n), endpoint=True).astype(np.int32)
    axis = axis_of(sections, interleaved)

    def dev(x):
        if not odd:
            return dev_f32(x, DEV)
        buf = torch.empty(x.size + 1, device=DEV)  # 4-byte aligned only
        buf[1:].copy_(dev_f32(x, DEV).view(-1))
        return buf[1:].view(x.shape)

    want = []
    for t, sc, x in ((pk.k, pk.ks, turn(k, pos, inv.inv_freqs_host, axis)), (pk.v, pk.vs, v)):
        data = t.cpu().numpy().reshape(-1, kv, d).copy()
        scales = None if sc is None else sc.cpu().numpy().copy()
        for i, (r, p) in enumerate(toks):
            if 0 <= r < rows and 0 <= p < 16 * stride and tables[r, p // 16] < num_pages:
                store(dtype, (data, scales), int(tables[r, p // 16]) * 16 + p % 16, x[i])
        want.append((data, scales))
    dq, dk, dv = dev(q), dev(k), dev(v)
    q_out = (dq if inplace else torch.empty_like(dq)) if with_q else None
    got = pk.mrope_append(rope, dk, dv, dev_i32(pos, DEV), dev_i32(np.array([r for r, _ in toks], np.int32), DEV),
                          dev_i32(np.array([p for _, p in toks], np.int32), DEV), dev_i32(tables, DEV),
                          q=dq if with_q else None, q_out=q_out)
    torch.cuda.synchronize()
    for t, sc, (data, scales) in ((pk.k, pk.ks, want[0]), (pk.v, pk.vs, want[1])):
        assert np.array_equal(t.cpu().numpy().reshape(-1, kv, d), data)
        if sc is not None:
            assert np.array_equal(sc.cpu().numpy(), scales)
    assert torch.equal(dk, dev_f32(k, DEV)) and torch.equal(dv, dev_f32(v, DEV))
    if with_q:
        assert np.array_equal(got.cpu().numpy(), turn(q, pos, inv.inv_freqs_host, axis))
        if not inplace:
            assert torch.equal(dq, dev_f32(q, DEV))
    else:
        assert got is None


TOKS = [(0, 0), (1, 17), (2, 5), (0, 95), (2, 50), (2, 70), (1, 96), (3, 1), (-1, 4), (0, -1), (1, 31), (0, 32)]
SHAPES = [(64, [32], False), (64, [16, 8, 8], False), (64, [11, 6, 5], False), (128, [24, 20, 20], False),
          (128, [24, 20, 20], True), (128, [1], False), (256, [12, 10, 10], True), (256, [64, 32, 16, 16], False),
          (256, [33, 0, 32, 30], False), (128, [22, 21, 21], True), (64, [3, 2], True)]


@pytest.mark.parametrize("dtype", A.DTYPES)
@pytest.mark.parametrize("d,sections,interleaved", SHAPES)
def test_bits(dtype, d, sections, interleaved):
    say("mrope", dtype, d, sections, interleaved)
    run(dtype, d, 2, 8, sections, interleaved, TOKS, 20000, seed=sum(sections))


@pytest.mark.parametrize("dtype", A.DTYPES)
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("d,sections", [(128, [24, 20, 20]), (64, [11, 6, 5])])
def test_alignment_and_in_place(dtype, odd, inplace, d, sections):
    say("mrope odd", dtype, odd, inplace, d)
    run(dtype, d, 3, 6, sections, False, TOKS, 300000, seed=3, odd=odd, inplace=inplace)


@pytest.mark.parametrize("dtype", A.DTYPES)
@pytest.mark.parametrize("kv,H", [(1, 1), (1, 8), (8, 32), (5, 40)])
def test_heads_and_one_token(dtype, kv, H):
    say("mrope heads", dtype, kv, H)
    run(dtype, 128, kv, H, [24, 20, 20], False, [(1, 20)], 100, seed=4)
    run(dtype, 128, kv, H, [24, 20, 20], False, TOKS, 100, seed=5, with_q=False)


def test_many_tokens_take_the_other_launch_shape():
    """From 1024 tokens on a block takes all rows of its token."""
    for dtype in A.DTYPES:
        n, kv, d = 1111, 2, 64
        rng = np.random.default_rng(1)
        pages = -(-n // 16)
        tables = rng.permutation(pages).astype(np.uint32)[None]
        rope = MRopeTable(RopeTable(64, 1e4, device=DEV).inv_freqs, [16, 8, 8])
        q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (8, kv, kv))
        pos = rng.integers(0, 5000, (3, n)).astype(np.int32)
        seq, at, t = np.zeros(n, np.int32), np.arange(n, dtype=np.int32), dev_i32(tables, DEV)
        one, many = PagedKV(pages, kv, d, dtype, DEV), PagedKV(pages, kv, d, dtype, DEV)
        a = many.mrope_append(rope, dev_f32(k, DEV), dev_f32(v, DEV), dev_i32(pos, DEV), dev_i32(seq, DEV),
                              dev_i32(at, DEV), t, q=dev_f32(q, DEV))
        b = [one.mrope_append(rope, dev_f32(k[c], DEV), dev_f32(v[c], DEV), dev_i32(pos[:, c], DEV), dev_i32(seq[c], DEV),
                              dev_i32(at[c], DEV), t, q=dev_f32(q[c], DEV)) for c in (slice(0, 600), slice(600, n))]
        assert torch.equal(a, torch.cat(b)) and torch.equal(many.k, one.k) and torch.equal(many.v, one.v)


@pytest.mark.parametrize("dtype", A.DTYPES)
def test_equal_axes_are_the_rope_append(dtype):
    """Three axes at the token's own position give lnskv_rope_append's pages, but for that
    call's f32 angle (off by at most position * 2^-24)."""
    n, kv, d = 40, 2, 128
    rng = np.random.default_rng(2)
    table = RopeTable(128, 1e4, device=DEV)
    k, v = (dev_f32(rng.standard_normal((n, kv, d)), DEV) for _ in range(2))
    seq, at = dev_i32(np.zeros(n, np.int32), DEV), dev_i32(np.arange(n, dtype=np.int32), DEV)
    t = dev_i32(np.array([[2, 0, 1]], np.uint32), DEV)
    a, b = PagedKV(3, kv, d, dtype, DEV), PagedKV(3, kv, d, dtype, DEV)
    a.rope_append(table, k, v, seq, at, t)
    b.mrope_append(MRopeTable(table.inv_freqs, [24, 20, 20]), k, v, at.repeat(3), seq, at, t)
    ka, kb = A.values(a)[0], A.values(b)[0]
    # the angle's error turns a pair by at most 40 * 2^-24; values are below 6, a page's step is 2^-11 (f16) or a
    # code (Q8A: one step of max/127 where a value falls on the other side of a border)
    step = {DTYPE_F32: 2.0 ** -22, DTYPE_F16: 6 * 2.0 ** -11, DTYPE_Q8A: 6 / 127}[dtype]
    assert np.abs(ka - kb).max() <= 6 * 40 * 2.0 ** -24 + step
    assert np.array_equal(A.values(a)[1], A.values(b)[1])


def test_extreme_positions_stay_exact():
    """Positions at both ends of int32: the turn keeps pair norms and f64 angles."""
    rope = MRopeTable(RopeTable(64, 1e6, device=DEV).inv_freqs, [16, 16])
    pk = PagedKV(1, 1, 64, DTYPE_F32, DEV)
    rng = np.random.default_rng(3)
    k = rng.standard_normal((2, 1, 64)).astype(np.float32)
    pos = np.array([[2**31 - 1, -2**31], [-2**31, 2**31 - 1]], np.int32)
    pk.mrope_append(rope, dev_f32(k, DEV), dev_f32(k, DEV), dev_i32(pos, DEV), dev_i32(np.zeros(2, np.int32), DEV),
                    dev_i32(np.arange(2, dtype=np.int32), DEV), dev_i32(np.array([[0]], np.uint32), DEV))
    got = pk.k.cpu().numpy().reshape(16, 1, 64)[:2].astype(np.float64)
    inv = rope.inv_freqs.cpu().numpy().astype(np.float64)
    ang = pos[[0] * 16 + [1] * 16].T.astype(np.float64) * inv[None, :]
    z = (k[..., :32] + 1j * k[..., 32:]) * np.exp(1j * ang)[:, None]
    # f64 angles up to 2^31 are off by 2^-22 in the product, and as much in the reduction by pi/2
    assert np.abs(got - np.concatenate([z.real, z.imag], -1)).max() < 4 * (3 * 2.0 ** -22 + 2.0 ** -23)


def test_captured_and_replayed():
    rng = np.random.default_rng(4)
    n, kv, d = 3, 2, 128
    pk, want = PagedKV(8, kv, d, DTYPE_Q8A, DEV), PagedKV(8, kv, d, DTYPE_Q8A, DEV)
    rope = MRopeTable(RopeTable(128, 1e4, device=DEV).inv_freqs, [24, 20, 20], True)
    q, k, v = (dev_f32(rng.standard_normal((n, h, d)), DEV) for h in (8, kv, kv))
    out = torch.empty_like(q)
    t = dev_i32(np.arange(6, dtype=np.uint32).reshape(3, 2), DEV)
    seq, at = dev_i32(np.arange(3, dtype=np.int32), DEV), dev_i32(np.array([3, 17, 30], np.int32), DEV)
    pos = dev_i32(np.full((3, n), 9, np.int32), DEV)
    pk.mrope_append(rope, k, v, pos, seq, at, t, q=q, q_out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pk.mrope_append(rope, k, v, pos, seq, at, t, q=q, q_out=out)
    want.mrope_append(rope, k, v, pos, seq, at, t, q=q)
    for i in range(3):
        q.copy_(dev_f32(rng.standard_normal((n, 8, d)), DEV))
        k.copy_(dev_f32(rng.standard_normal((n, kv, d)), DEV))
        pos.add_(100 + i)
        at.sub_(1)
        eager = want.mrope_append(rope, k, v, pos, seq, at, t, q=q)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pk.k, want.k) and torch.equal(pk.ks, want.ks)
