"""Sliding-window attention with sinks on the GPU (lnskv_sink_decode,
lnskv_sink_prefill_attention) against f64: every page type, head layout and
schedule; windows and sinks that start and end inside pages; contexts shorter than
either; slots that nothing attends hold NaN and infinities, and pages that hold no
attended token are missing."""
import numpy as np
import pytest
import torch

import attn_f64 as A
from gpu_util import dev_f32, dev_i32, say
from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A, LnskvError
from lnskv.device import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def tokens(L, window, sink):
    return [t for t in range(L) if t < sink or window == 0 or t >= L - window]


def decode_case(dtype, d, kv, rep, lens, window, sink, seed, gate=False, ws=True, poison=True, max_len=None, bad=()):
    rng = np.random.default_rng(seed)
    seen = [[] if s in bad else tokens(L, window, sink) for s, L in enumerate(lens)]
    held = [sorted({t // 16 for t in x}) for x in seen]
    tables, n_pages = A.make_tables(lens, held, rng)
    pk = PagedKV(n_pages, kv, d, dtype, DEV)
    A.fill(pk, seed)
    slots = [A.slots_of(tables[s], x, n_pages) for s, x in enumerate(seen)]
    if poison:
        A.poison(pk, np.concatenate(slots + [np.zeros(0, np.int64)]))
    H = kv * rep
    q = (2 * rng.standard_normal((len(lens), H, d))).astype(np.float32)
    scale = 1.0 / np.sqrt(d)
    vals = A.values(pk)
    ref = np.stack([A.row(vals, q[s], slots[s], scale) for s in range(len(lens))])
    g = None
    if gate:
        gh = rng.random((len(lens), H, d)).astype(np.float32)
        g, ref = dev_f32(gh, DEV), ref * gh
    max_len = max(lens) if max_len is None else max_len
    out = torch.full((len(lens), H, d), float("nan"), device=DEV)
    work = None
    if ws:
        work = torch.zeros(max(16, pk.sink_workspace_size(len(lens), H, max_len, window, sink)), dtype=torch.uint8, device=DEV)
    pk.sink_decode(dev_f32(q, DEV), dev_i32(tables, DEV), dev_i32(np.array(lens, np.int32), DEV), n_heads=H,
                   max_kv_len=max_len, scale=scale, window=window, n_sink=sink, gate=g, workspace=work, out=out)
    torch.cuda.synchronize()
    return A.worst(out, ref)


GEOMS = [(64, 4, 8), (64, 2, 1), (128, 2, 4), (128, 3, 1), (128, 2, 8), (256, 2, 4), (256, 1, 2), (256, 1, 8)]


@pytest.mark.parametrize("dtype", A.DTYPES)
@pytest.mark.parametrize("d,kv,rep", GEOMS)
@pytest.mark.parametrize("window,sink", [(16, 4), (33, 17), (100, 0), (1, 1), (0, 5), (64, 16), (50, 200)])
def test_decode_against_f64(dtype, d, kv, rep, window, sink):
    say("sink decode", dtype, d, kv, rep, window, sink)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 100, 133, 209, 500]
    assert decode_case(dtype, d, kv, rep, lens, window, sink, seed=window * 7 + sink, gate=sink == 17) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 128), (DTYPE_F16, 256), (DTYPE_Q8A, 256), (DTYPE_F32, 64)])
@pytest.mark.parametrize("schedule", ["stream-k", "workgroup"])
def test_decode_schedules_and_long_windows(dtype, d, schedule, monkeypatch):
    say("sink schedules", dtype, d, schedule)
    monkeypatch.setenv("LNSKV_DECODE_SCHEDULE", schedule)
    lens = [5000, 1300, 7, 4096, 1025, 3000]
    assert decode_case(dtype, d, 2, 4, lens, 1024, 70, seed=3) < A.TOL
    assert decode_case(dtype, d, 2, 4, [9001], 2000, 4, seed=4, ws=False) < A.TOL


@pytest.mark.parametrize("dtype", A.DTYPES)
def test_decode_of_many_sequences(dtype):
    say("sink many", dtype)
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(1, 300, 150)]
    assert decode_case(dtype, 128, 2, 4, lens, 40, 4, seed=8) < A.TOL
    assert decode_case(dtype, 128, 2, 4, [4 * L for L in lens[:100]], 800, 4, seed=9) < A.TOL
    assert decode_case(dtype, 64, 2, 4, [4 * L for L in lens[:100]], 700, 33, seed=9) < A.TOL


@pytest.mark.parametrize("dtype", [DTYPE_F16, DTYPE_Q8A])
def test_decode_of_more_sequences_than_a_launch_takes(dtype):
    say("sink 4200", dtype)
    rng = np.random.default_rng(10)
    lens = [int(x) for x in rng.integers(1, 60, 4200)]
    assert decode_case(dtype, 128, 1, 1, lens, 20, 3, seed=8) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256), (DTYPE_F32, 128), (DTYPE_F16, 64)])
def test_decode_rows_that_attend_nothing(dtype, d):
    """Length 0, a length past max_kv_len, and a sequence whose pages are all missing give zero rows."""
    say("sink empty", dtype, d)
    lens = [40, 0, 200, 90, 33]
    assert decode_case(dtype, d, 2, 2, lens, 30, 4, seed=5, max_len=100, bad=(1, 2, 4)) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 128), (DTYPE_F16, 256), (DTYPE_F32, 64)])
def test_no_sinks_is_the_windowed_decode_and_no_window_the_plain_one(dtype, d):
    say("sink vs decode", dtype, d)
    rng = np.random.default_rng(2)
    lens = [1, 50, 300, 777]
    tables, n = A.make_tables(lens, [range(-(-L // 16)) for L in lens], rng)
    pk = PagedKV(n, 2, d, dtype, DEV)
    A.fill(pk, 1)
    q = dev_f32(2 * rng.standard_normal((4, 8, d)), DEV)
    t, kl = dev_i32(tables, DEV), dev_i32(np.array(lens, np.int32), DEV)
    for window in (0, 100):
        ps = dev_i32(np.array([max(0, L - window) if window else 0 for L in lens], np.int32), DEV)
        a = pk.decode(q, t, kl, n_heads=8, max_kv_len=777, scale=0.1, p_start=ps)
        b = pk.sink_decode(q, t, kl, n_heads=8, max_kv_len=777, scale=0.1, window=window, n_sink=0)
        assert A.worst(b, a.cpu().numpy().astype(np.float64)) < A.TOL


# ---------------------------------------------------------------------------


def prefill_case(dtype, d, kv, rep, chunks, window, sink, seed, poison=True):
    """chunks: (first position, length) of one sequence each."""
    rng = np.random.default_rng(seed)
    ends = [a + b for a, b in chunks]
    seen = [[t for t in range(a + b) if t < sink or window == 0 or t > a - window] for a, b in chunks]
    held = [sorted({t // 16 for t in x}) for x in seen]
    tables, n_pages = A.make_tables(ends, held, rng)
    pk = PagedKV(n_pages, kv, d, dtype, DEV)
    A.fill(pk, seed)
    if poison:
        A.poison(pk, np.concatenate([A.slots_of(tables[s], x, n_pages) for s, x in enumerate(seen)]))
    H, n_tok = kv * rep, sum(b for _, b in chunks)
    q = (2 * rng.standard_normal((n_tok, H, d))).astype(np.float32)
    scale = 1.0 / np.sqrt(d)
    vals, ref, desc, at = A.values(pk), np.zeros((n_tok, H, d)), [], 0
    for s, (a, b) in enumerate(chunks):
        desc.append([s, a, b, at])
        for i in range(b):
            p = a + i
            tok = [t for t in range(p + 1) if t < sink or window == 0 or t > p - window]
            ref[at + i] = A.row(vals, q[at + i], A.slots_of(tables[s], tok, n_pages), scale)
        at += b
    out = torch.full((n_tok, H, d), float("nan"), device=DEV)
    pk.sink_prefill_attention(dev_f32(q, DEV), dev_i32(np.array(desc, np.int32), DEV), dev_i32(tables, DEV), n_heads=H,
                              scale=scale, window=window, n_sink=sink, out=out)
    torch.cuda.synchronize()
    return A.worst(out, ref)


@pytest.mark.parametrize("dtype", [DTYPE_F16, DTYPE_Q8A])
@pytest.mark.parametrize("d,kv,rep", [(128, 2, 4), (128, 1, 8), (128, 2, 1), (128, 1, 2), (256, 1, 4), (256, 2, 1)])
@pytest.mark.parametrize("window,sink", [(16, 4), (70, 33), (1, 1), (0, 9), (200, 0), (48, 64), (30, 1000)])
def test_prefill_against_f64(dtype, d, kv, rep, window, sink):
    say("sink prefill", dtype, d, kv, rep, window, sink)
    chunks = [(0, 1), (0, 70), (5, 33), (150, 90), (31, 1), (400, 17)]
    assert prefill_case(dtype, d, kv, rep, chunks, window, sink, seed=window + sink) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256)])
def test_prefill_of_a_long_context(dtype, d):
    """More table entries than one window of 64, sinks and window far apart."""
    say("sink prefill long", dtype, d)
    assert prefill_case(dtype, d, 1, 4, [(6000, 40), (2500, 20)], 1500, 20, seed=1) < A.TOL
    assert prefill_case(dtype, d, 1, 4, [(3000, 20)], 500, 1200, seed=2) < A.TOL


def test_prefill_without_sinks_is_the_windowed_prefill():
    rng = np.random.default_rng(3)
    tables, n = A.make_tables([400], [range(25)], rng)
    pk = PagedKV(n, 2, 128, DTYPE_F16, DEV)
    A.fill(pk, 3)
    q = dev_f32(rng.standard_normal((300, 8, 128)), DEV)
    ch, t = dev_i32(np.array([[0, 100, 300, 0]], np.int32), DEV), dev_i32(tables, DEV)
    for window in (0, 90):
        a = pk.prefill_attention(q, ch, t, n_heads=8, scale=0.1, window=window)
        b = pk.sink_prefill_attention(q, ch, t, n_heads=8, scale=0.1, window=window, n_sink=0)
        if pk.sink_prefill_workspace_size(1, 300, 25, window, 0, 8) == 0:
            assert torch.equal(a, b)
        else:  # split along the keys: both are within TOL of the exact result, so within 2 TOL of each other
            assert window == 0 and A.worst(b, a.cpu().numpy()) < 2 * A.TOL


def test_prefill_skips_chunks_outside_the_inputs():
    rng = np.random.default_rng(4)
    tables, n = A.make_tables([100], [range(7)], rng)
    pk = PagedKV(n, 1, 128, DTYPE_F16, DEV)
    A.fill(pk, 3)
    q = dev_f32(rng.standard_normal((64, 4, 128)), DEV)
    ch = dev_i32(np.array([[1, 0, 10, 0], [0, 10, 8, 60], [0, 10, 8, 8], [-1, 0, 4, 20]], np.int32), DEV)
    out = torch.full((64, 4, 128), 7.0, device=DEV)
    pk.sink_prefill_attention(q, ch, dev_i32(tables, DEV), n_heads=4, scale=0.1, window=8, n_sink=2, out=out)
    torch.cuda.synchronize()
    touched = (out != 7.0).flatten(1).any(1).cpu().numpy()
    assert touched[8:16].all() and not touched[:8].any() and not touched[16:].any()


@pytest.mark.parametrize("window", [100, 800])
def test_decode_captured_and_replayed(window):
    """A captured call replayed over changed inputs, with eager work between."""
    rng = np.random.default_rng(6)
    lens = [900, 40, 333]
    tables, n = A.make_tables(lens, [range(-(-L // 16)) for L in lens], rng)
    pk = PagedKV(n, 2, 128, DTYPE_Q8A, DEV)
    A.fill(pk, 3)
    q = dev_f32(rng.standard_normal((3, 8, 128)), DEV)
    t, kl = dev_i32(tables, DEV), dev_i32(np.array(lens, np.int32), DEV)
    ws = torch.zeros(pk.sink_workspace_size(3, 8, 900, window, 4), dtype=torch.uint8, device=DEV)
    eager_ws = torch.zeros_like(ws)
    out = torch.empty((3, 8, 128), device=DEV)
    call = dict(n_heads=8, max_kv_len=900, scale=0.1, window=window, n_sink=4)
    pk.sink_decode(q, t, kl, workspace=ws, out=out, **call)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pk.sink_decode(q, t, kl, workspace=ws, out=out, **call)
    for i in range(4):
        q.copy_(dev_f32(rng.standard_normal((3, 8, 128)), DEV))
        kl.copy_(dev_i32(np.array([900 - 100 * i, 40 - i, 333 - 7 * i], np.int32), DEV))
        want = pk.sink_decode(q, t, kl, workspace=eager_ws, **call)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("window", [50, 1000])
def test_decode_on_another_stream_and_wrong_inputs(window):
    rng = np.random.default_rng(7)
    tables, n = A.make_tables([200], [range(13)], rng)
    pk = PagedKV(n, 2, 128, DTYPE_F16, DEV)
    A.fill(pk, 3)
    q = dev_f32(rng.standard_normal((1, 8, 128)), DEV)
    t, kl = dev_i32(tables, DEV), dev_i32(np.array([200], np.int32), DEV)
    call = dict(n_heads=8, max_kv_len=208, scale=0.1, window=window, n_sink=4)
    want = pk.sink_decode(q, t, kl, **call)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ws = torch.zeros(pk.sink_workspace_size(1, 8, 208, window, 4), dtype=torch.uint8, device=DEV)
        got = pk.sink_decode(q, t, kl, workspace=ws, **call)
    s.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(LnskvError):  # more tokens than one workgroup takes
        pk.sink_decode(q, t, kl, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV),
                       **dict(call, max_kv_len=9000, window=5000))
    with pytest.raises(ValueError):
        pk.sink_decode(q.transpose(1, 2), t, kl, **call)
    with pytest.raises(TypeError):
        pk.sink_decode(q.half(), t, kl, **call)


@pytest.mark.parametrize("dtype,d,rep", [(DTYPE_F16, 128, 4), (DTYPE_Q8A, 256, 4), (DTYPE_F16, 256, 1), (DTYPE_Q8A, 128, 8)])
def test_prefill_split_along_the_keys(dtype, d, rep):
    """Few queries on a long window: with a workspace, the library's buffer and a
    workspace too small to split; rows of no chunk keep what they hold."""
    say("sink prefill split", dtype, d, rep)
    rng = np.random.default_rng(5)
    chunks, window, sink = [(5000, 37), (2990, 20)], 2500, 600
    lens = [a + b for a, b in chunks]
    seen = [[t for t in range(L) if t < sink or t > a - window] for (a, _), L in zip(chunks, lens)]
    tables, n = A.make_tables(lens, [sorted({t // 16 for t in x}) for x in seen], rng)
    pk = PagedKV(n, 1, d, dtype, DEV)
    A.fill(pk, 5)
    A.poison(pk, np.concatenate([A.slots_of(tables[s], x, n) for s, x in enumerate(seen)]))
    n_tok, scale = 64, 1.0 / np.sqrt(d)
    q = (2 * rng.standard_normal((n_tok, rep, d))).astype(np.float32)
    vals, ref = A.values(pk), np.full((n_tok, rep, d), 7.0)
    desc = np.array([[0, 5000, 37, 0], [1, 2990, 20, 40]], np.int32)
    for s, a, b, at in desc:
        for i in range(b):
            tok = [t for t in range(a + i + 1) if t < sink or t > a + i - window]
            ref[at + i] = A.row(vals, q[at + i], A.slots_of(tables[s], tok, n), scale)
    size = pk.sink_prefill_workspace_size(2, n_tok, tables.shape[1], window, sink, rep)
    assert size > 0
    for ws in (torch.full((size,), 0xFF, dtype=torch.uint8, device=DEV), None, torch.zeros(64, dtype=torch.uint8, device=DEV)):
        out = torch.full((n_tok, rep, d), 7.0, device=DEV)
        pk.sink_prefill_attention(dev_f32(q, DEV), dev_i32(desc, DEV), dev_i32(tables, DEV), n_heads=rep, scale=scale,
                                  window=window, n_sink=sink, workspace=ws, out=out)
        torch.cuda.synchronize()
        assert A.worst(out, ref) < A.TOL
        assert (out[37:40] == 7.0).all() and (out[60:] == 7.0).all()
