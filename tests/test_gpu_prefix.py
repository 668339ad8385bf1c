"""Decode of sequences that share a prefix on the GPU (lnskv_prefix_decode) against
f64: every page type and head layout, groups of one to many sequences, prefixes that
end inside a page, lengths that end inside the prefix, sequences outside every group.
Only the group's first row holds the shared pages; the other rows' entries for them are
missing or garbage, and slots that nothing attends hold NaN and infinities."""
import numpy as np
import pytest
import torch

import attn_f64 as A
from gpu_util import dev_f32, dev_i32, say
from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A, BlockTables, PagePool
from lnskv.device import MRopeTable, PagedKV, PrefixGroups, RopeTable

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(params=["auto", "workgroup"], autouse=True)
def _setting(request, monkeypatch):
    """With a schedule forced, short sequences too take the prefix's kernel and their own."""
    if request.param != "auto":
        monkeypatch.setenv("LNSKV_DECODE_SCHEDULE", request.param)


def case(dtype, d, kv, rep, groups, lens, seed, gate=False, ws=True, max_len=None, missing=(), same=False):
    """groups: (first, sequences, tokens); lens: kv_len of every sequence; missing: logical
    pages without a page in every row; same: every row of a group holds the shared pages."""
    rng = np.random.default_rng(seed)
    n = len(lens)
    owner = np.arange(n)
    shared = np.zeros(n, int)
    for f, m, tok in groups:
        owner[f:f + m], shared[f:f + m] = f, tok // 16
    most = {f: max(max(lens[f:f + m]), tok) for f, m, tok in groups}
    held = []
    for s, L in enumerate(lens):
        pages = -(-max(L, most.get(s, 0)) // 16)
        held.append([p for p in range(pages) if (p >= shared[s] or owner[s] == s) and p not in missing])
    tables, n_pages = A.make_tables([max(L, most.get(s, 0)) for s, L in enumerate(lens)], held, rng)
    pk = PagedKV(n_pages, kv, d, dtype, DEV)
    A.fill(pk, seed)
    view = tables.copy()
    for s in range(n):
        view[s, :shared[s]] = tables[owner[s], :shared[s]]
    limit = max(lens) if max_len is None else max_len
    slots = [A.slots_of(view[s], range(L) if L <= limit else [], n_pages) for s, L in enumerate(lens)]
    A.poison(pk, np.concatenate(slots + [np.zeros(0, np.int64)]))
    given = view.copy() if same else tables.copy()
    if not same:
        for s in range(n):
            if owner[s] != s:
                given[s, :shared[s]] = np.where(np.arange(shared[s]) % 2, 0xFFFFFFFF, 0x7FFFFFF0).astype(np.uint32)
    H = kv * rep
    q = (2 * rng.standard_normal((n, H, d))).astype(np.float32)
    scale = 1.0 / np.sqrt(d)
    vals = A.values(pk)
    ref = np.stack([A.row(vals, q[s], slots[s], scale) for s in range(n)])
    g = None
    if gate:
        gh = rng.random((n, H, d)).astype(np.float32)
        g, ref = dev_f32(gh, DEV), ref * gh
    out = torch.full((n, H, d), float("nan"), device=DEV)
    plan = PrefixGroups(groups)
    work = None
    if ws:
        work = torch.full((max(16, pk.prefix_workspace_size(plan, n, H, limit)),), 0xFF, dtype=torch.uint8, device=DEV)
        work[:4096] = 0
    pk.prefix_decode(dev_f32(q, DEV), dev_i32(given, DEV), dev_i32(np.array(lens, np.int32), DEV), plan, n_heads=H,
                     max_kv_len=limit, scale=scale, gate=g, workspace=work, out=out)
    torch.cuda.synchronize()
    return A.worst(out, ref)


GEOMS = [(64, 4, 8), (64, 2, 1), (128, 2, 4), (128, 3, 1), (128, 1, 8), (256, 2, 4), (256, 1, 2), (256, 1, 8)]


@pytest.mark.parametrize("dtype", A.DTYPES)
@pytest.mark.parametrize("d,kv,rep", GEOMS)
@pytest.mark.parametrize("tok", [16, 37, 100, 513])
def test_against_f64(dtype, d, kv, rep, tok):
    say("prefix", dtype, d, kv, rep, tok)
    rng = np.random.default_rng(tok)
    lens = [tok + int(x) for x in rng.integers(1, 90, 9)]
    assert case(dtype, d, kv, rep, [(0, 9, tok)], lens, seed=tok, gate=tok == 37) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256), (DTYPE_F32, 64), (DTYPE_F16, 64), (DTYPE_Q8A, 128)])
def test_several_groups_and_sequences_outside_them(dtype, d):
    say("prefix groups", dtype, d)
    groups = [(1, 2, 80), (3, 1, 64), (5, 7, 15), (12, 4, 333)]
    lens = [70, 90, 81, 65, 1, 20, 16, 17, 33, 15, 40, 31, 400, 334, 350, 340, 5, 64]
    assert case(dtype, d, 2, 4, groups, lens, seed=1) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256), (DTYPE_F32, 128), (DTYPE_Q8A, 64), (DTYPE_F16, 256)])
def test_lengths_that_end_inside_the_prefix(dtype, d):
    """Also length 0, exactly the shared pages, and a length out of range (zero row)."""
    say("prefix short", dtype, d)
    lens = [200, 1, 5, 16, 17, 100, 0, 128, 129, 130, 300]
    assert case(dtype, d, 2, 4, [(0, 11, 130)], lens, seed=2, max_len=250) < A.TOL
    assert case(dtype, d, 2, 2, [(0, 4, 320)], [3, 0, 20, 9], seed=3, max_len=320) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 128), (DTYPE_F32, 64)])
def test_missing_pages_are_skipped(dtype, d):
    say("prefix missing", dtype, d)
    assert case(dtype, d, 2, 4, [(0, 3, 200)], [210, 240, 290], seed=4, missing=(0, 3, 13, 14)) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256), (DTYPE_F32, 128), (DTYPE_F16, 64)])
def test_long_prefixes(dtype, d):
    say("prefix long", dtype, d)
    lens = [2500, 2100, 4000, 2051, 2049, 700]
    assert case(dtype, d, 2, 4, [(0, 5, 2048)], lens, seed=5) < A.TOL
    assert case(dtype, d, 1, 2, [(0, 2, 6000)], [6001, 6100], seed=6, ws=False) < A.TOL


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256), (DTYPE_F32, 64)])
def test_many_sequences(dtype, d):
    say("prefix many", dtype, d)
    rng = np.random.default_rng(7)
    lens = [150 + int(x) for x in rng.integers(1, 60, 200)]
    assert case(dtype, d, 1, 4, [(0, 150, 149), (150, 50, 97)], lens, seed=7, same=True) < A.TOL


@pytest.mark.parametrize("dtype", [DTYPE_F16, DTYPE_Q8A])
def test_more_sequences_than_a_launch_takes(dtype):
    say("prefix 4200", dtype)
    rng = np.random.default_rng(8)
    lens = [33 + int(x) for x in rng.integers(0, 30, 4200)]
    groups = [(50, 2000, 32), (2050, 2100, 33)]
    assert case(dtype, 128, 1, 1, groups, lens, seed=8) < A.TOL


@pytest.mark.parametrize("dtype", [DTYPE_F16, DTYPE_Q8A])
@pytest.mark.parametrize("kv,rep,n", [(32, 2, 128), (8, 8, 160)])
def test_long_prefixes_of_many_rows(dtype, kv, rep, n):
    """Tiles of 256 rows (the last one partly empty or not), against the plain decode:
    each is within TOL of the exact result, so they are within 2 TOL of each other."""
    say("prefix wide", dtype, kv, rep, n)
    rng = np.random.default_rng(13)
    tok, H = 3200, kv * rep
    tables = np.full((n, 202), 0xFFFFFFFF, np.uint32)
    order = rng.permutation(200 + 2 * n + 1)
    tables[:, :200] = order[:200]
    tables[:, 200:] = order[200:200 + 2 * n].reshape(n, 2)
    lens = tok + rng.integers(0, 33, n)
    lens[[3, n - 1]] = [1777, 0]
    pk = PagedKV(len(order), kv, 128, dtype, DEV)
    A.fill(pk, 13)
    q, t, kl = dev_f32(rng.standard_normal((n, H, 128)), DEV), dev_i32(tables, DEV), dev_i32(lens.astype(np.int32), DEV)
    call = dict(n_heads=H, max_kv_len=3232, scale=0.1)
    want = pk.decode(q, t, kl, **call)
    got = pk.prefix_decode(q, t, kl, PrefixGroups([(0, n, tok)]), **call)
    assert A.worst(got, want.cpu().numpy().astype(np.float64)) < 2 * A.TOL


def test_two_calls_at_once():
    """Prefixes and sinks on two streams with workspaces of their own, as one after the other."""
    rng = np.random.default_rng(14)
    lens = [900, 877, 850, 1100]
    tables, n = A.make_tables([1100] * 4, [range(69)] * 4, rng)
    tables[1:, :50] = tables[0, :50]
    pk = PagedKV(n, 4, 128, DTYPE_Q8A, DEV)
    A.fill(pk, 3)
    q, t, kl = dev_f32(rng.standard_normal((4, 16, 128)), DEV), dev_i32(tables, DEV), dev_i32(np.array(lens, np.int32), DEV)
    plan, call = PrefixGroups([(0, 4, 800)]), dict(n_heads=16, max_kv_len=1100, scale=0.1)
    chunks, pq = dev_i32(np.array([[0, 860, 40, 0]], np.int32), DEV), dev_f32(rng.standard_normal((40, 16, 128)), DEV)
    sizes = [pk.prefix_workspace_size(plan, 4, 16, 1100), pk.sink_workspace_size(4, 16, 1100, 1000, 4),
             pk.sink_prefill_workspace_size(1, 40, 69, 700, 4, 16)]
    assert min(sizes) > 0

    def all_of(ws):
        return [pk.prefix_decode(q, t, kl, plan, workspace=ws[0], **call),
                pk.sink_decode(q, t, kl, window=1000, n_sink=4, workspace=ws[1], **call),
                pk.sink_prefill_attention(pq, chunks, t, n_heads=16, scale=0.1, window=700, n_sink=4, workspace=ws[2])]
    spaces = [[torch.zeros(x, dtype=torch.uint8, device=DEV) for x in sizes] for _ in range(2)]
    want = all_of(spaces[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, ws in zip(streams, spaces):
            with torch.cuda.stream(s):
                got.append(all_of(ws))
        torch.cuda.synchronize()
        for outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_no_groups_is_the_plain_decode():
    rng = np.random.default_rng(9)
    lens = [50, 300, 7]
    tables, n = A.make_tables(lens, [range(-(-L // 16)) for L in lens], rng)
    pk = PagedKV(n, 2, 128, DTYPE_F16, DEV)
    A.fill(pk, 1)
    q = dev_f32(rng.standard_normal((3, 8, 128)), DEV)
    t, kl = dev_i32(tables, DEV), dev_i32(np.array(lens, np.int32), DEV)
    a = pk.decode(q, t, kl, n_heads=8, max_kv_len=300, scale=0.1)
    for groups in ([], [(0, 3, 15)], [(1, 1, 0)]):
        b = pk.prefix_decode(q, t, kl, PrefixGroups(groups), n_heads=8, max_kv_len=300, scale=0.1)
        assert A.worst(b, a.cpu().numpy().astype(np.float64)) < A.TOL


def test_captured_and_replayed_on_two_workspaces():
    """Two graphs with workspaces of their own, replayed in turn over changed inputs."""
    rng = np.random.default_rng(10)
    lens = [700, 650, 513, 900]
    tables, n = A.make_tables([900] * 4, [range(57)] * 4, rng)
    tables[1:, :32] = tables[0, :32]
    pk = PagedKV(n, 2, 128, DTYPE_F16, DEV)
    A.fill(pk, 3)
    t, plan = dev_i32(tables, DEV), PrefixGroups([(0, 4, 512)])
    call = dict(n_heads=8, max_kv_len=900, scale=0.1)
    size = pk.prefix_workspace_size(plan, 4, 8, 900)
    graphs = []
    for i in range(2):
        q = dev_f32(rng.standard_normal((4, 8, 128)), DEV)
        kl = dev_i32(np.array(lens, np.int32), DEV)
        ws, out = torch.zeros(size, dtype=torch.uint8, device=DEV), torch.empty((4, 8, 128), device=DEV)
        pk.prefix_decode(q, t, kl, plan, workspace=ws, out=out, **call)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pk.prefix_decode(q, t, kl, plan, workspace=ws, out=out, **call)
        graphs.append((g, q, kl, ws, out))
    for i in range(4):
        for j, (g, q, kl, ws, out) in enumerate(graphs):
            q.copy_(dev_f32(rng.standard_normal((4, 8, 128)), DEV))
            kl.copy_(dev_i32(np.array([700 - i, 650 - 60 * i, 513 + j, 900 - 300 * i + 1], np.int32).clip(0, 900), DEV))
        wants = [pk.prefix_decode(q, t, kl, plan, **call).clone() for _, q, kl, _, _ in graphs]
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, out), want in zip(graphs, wants):
            assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,d", [(DTYPE_F16, 128), (DTYPE_Q8A, 256)])
def test_a_prompt_forked_into_answers(dtype, d):
    """As a serving program runs them together: a prompt with a picture appended by
    positions of three axes and attended, forked into four answers on the host tables,
    then decode steps (append by axes, groups from the tables, shared-prefix decode),
    each step against f64 over the stored pages."""
    say("prefix pipeline", dtype, d)
    kv, rep, T, n = 2, 4, 75, 4
    H, scale = kv * rep, 1.0 / np.sqrt(d)
    rng = np.random.default_rng(11)
    pool, tables = PagePool(64), BlockTables(n, 12)
    pk = PagedKV(64, kv, d, dtype, DEV)
    rope = MRopeTable(RopeTable(64, 1e6, device=DEV).inv_freqs, [12, 10, 10])
    dev_tables = dev_i32(tables.array(), DEV)
    new = lambda k: [dev_f32(rng.standard_normal((k, h, d)), DEV) for h in (H, kv, kv)]  # noqa: E731

    for p in range(T):
        tables.ensure_kv_page(pool, 0, p)
    tables.sync(dev_tables.data_ptr(), torch.cuda.current_stream().cuda_stream)
    axes = np.stack([np.minimum(np.arange(T), 20), np.arange(T) // 3, np.arange(T) % 7]).astype(np.int32)
    q, k, v = new(T)
    zeros, pos = dev_i32(np.zeros(T, np.int32), DEV), dev_i32(np.arange(T, dtype=np.int32), DEV)
    turned = pk.mrope_append(rope, k, v, dev_i32(axes, DEV), zeros, pos, dev_tables, q=q)
    out = pk.sink_prefill_attention(turned, dev_i32(np.array([[0, 0, T, 0]], np.int32), DEV), dev_tables, n_heads=H,
                                    scale=scale, window=40, n_sink=4)
    vals, row0 = A.values(pk), tables.array()[0]
    qh = turned.cpu().numpy()
    ref = np.stack([A.row(vals, qh[p], A.slots_of(row0, [t for t in range(p + 1) if t < 4 or t > p - 40], 64), scale)
                    for p in range(T)])
    assert A.worst(out, ref) < A.TOL

    for child in range(1, n):
        src, dst = tables.fork_sequence(pool, 0, child, T)
        pk.page_copy(dev_i32(np.array([src], np.int32), DEV), dev_i32(np.array([dst], np.int32), DEV))
    seqs = dev_i32(np.arange(n, dtype=np.int32), DEV)
    for step in range(8):
        p = T + step
        for s in range(n):
            tables.ensure_kv_page(pool, s, p)
        tables.sync(dev_tables.data_ptr(), torch.cuda.current_stream().cuda_stream)
        groups = tables.shared_prefix_groups()
        assert groups == [(0, n, 64)]
        q, k, v = new(n)
        at = dev_i32(np.full((3, n), 30 + step, np.int32), DEV)
        pk.mrope_append(rope, k, v, at, seqs, dev_i32(np.full(n, p, np.int32), DEV), dev_tables, q=q, q_out=q)
        kl = dev_i32(np.full(n, p + 1, np.int32), DEV)
        out = pk.prefix_decode(q, dev_tables, kl, PrefixGroups(groups), n_heads=H, max_kv_len=p + 1, scale=scale)
        vals, host = A.values(pk), tables.array()
        qh = q.cpu().numpy()
        ref = np.stack([A.row(vals, qh[s], A.slots_of(host[s], range(p + 1), 64), scale) for s in range(n)])
        assert A.worst(out, ref) < A.TOL
