"""What lnskv_mrope_append, lnskv_sink_decode, lnskv_sink_prefill_attention and
lnskv_prefix_decode refuse, before anything is launched (CPU only: the pointers are
never followed), and their workspace queries."""
import ctypes as C

import pytest
import torch

from lnskv import _lib
from lnskv._lib import Pages, Rope
from lnskv.device import MRopeTable, PagedKV, PrefixGroups

INV, UNS, WS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE
P = 4096  # a pointer that nothing may follow


def pages(dtype=_lib.DTYPE_F32, d=64, kv=4, n=64):
    return Pages(P, P, P, P, n, kv, d, dtype)


def i32(*x):
    return (C.c_int32 * max(1, len(x)))(*x)


def status(fn, *args):
    rc = getattr(_lib.lib(), fn)(*args)
    return rc, _lib.last_error()


def mrope(c=None, rope=Rope(P, 64), sections=(16, 8, 8), n_axes=3, interleaved=0, q=P, q_out=P, n_heads=8, k=P, v=P,
          axis=P, seq=P, pos=P, n_tok=4, bt=P, stride=2, rows=1):
    return status("lnskv_mrope_append", C.byref(c or pages()), C.byref(rope) if rope else None,
                  i32(*sections) if sections is not None else None, n_axes, interleaved, q, q_out, n_heads, k, v, axis,
                  seq, pos, n_tok, bt, stride, rows, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(rope=None), INV, "rope"), (dict(rope=Rope(None, 64)), INV, "inverse"), (dict(rope=Rope(P, 63)), INV, "rotary_dim"),
    (dict(rope=Rope(P, 66)), INV, "rotary_dim"), (dict(rope=Rope(P, 0)), INV, "rotary_dim"),
    (dict(sections=None), INV, "sections"), (dict(n_axes=0), INV, "n_axes"), (dict(n_axes=5, sections=(1,) * 5), INV, "n_axes"),
    (dict(sections=(16, 8, 9)), INV, "sum"), (dict(sections=(40, -16, 8)), INV, "negative"),
    (dict(sections=(2**31 - 1, 2**31 - 1, 34)), INV, "sum"),
    (dict(interleaved=2), INV, "interleaved"), (dict(interleaved=1, sections=(8, 12, 12)), INV, "dealt"),
    (dict(n_tok=-1), INV, "n_tok"), (dict(q=None), INV, "together"), (dict(q_out=None), INV, "together"),
    (dict(n_heads=6), INV, "multiple"), (dict(n_heads=0), INV, "multiple"), (dict(k=None), INV, "non-null"),
    (dict(axis=None), INV, "non-null"), (dict(bt=None), INV, "non-null"), (dict(stride=0), INV, "bt_stride"),
    (dict(rows=-1), INV, "n_rows"), (dict(q_out=P + 64), INV, "overlap"),
    (dict(c=pages(d=96)), UNS, "head_dim"), (dict(c=Pages(None, P, P, P, 64, 4, 64, 0)), INV, "NULL"),
])
def test_mrope_append_refuses(kw, rc, text):
    got, msg = mrope(**kw)
    assert got == rc and text in msg, (got, msg)


def test_mrope_append_of_no_tokens():
    assert mrope(n_tok=0)[0] == 0
    assert mrope(n_tok=0, sections=(12, 10, 10), interleaved=1)[0] == 0
    assert mrope(n_tok=0, q=None, q_out=None, n_heads=-1)[0] == 0


def sink(c=None, q=P, out=P, gate=None, bt=P, stride=4, kv_len=P, n_seq=2, n_heads=8, max_len=64, window=16, n_sink=4,
         scale=0.1, ws=P, ws_bytes=1 << 30):
    return status("lnskv_sink_decode", C.byref(c or pages()), q, out, gate, bt, stride, kv_len, n_seq, n_heads, max_len,
                  window, n_sink, scale, ws, ws_bytes, None)


def prefix(groups=((0, 2, 32),), c=None, q=P, out=P, gate=None, bt=P, stride=4, kv_len=P, n_seq=2, n_heads=8, max_len=64,
           scale=0.1, ws=P, ws_bytes=1 << 30, n_groups=None):
    flat = None if groups is None else i32(*[x for g in groups for x in g])
    n = n_groups if n_groups is not None else len(groups or ())
    return status("lnskv_prefix_decode", C.byref(c or pages()), q, out, gate, bt, stride, kv_len, flat, n, n_seq, n_heads,
                  max_len, scale, ws, ws_bytes, None)


COMMON = [
    (dict(q=None), INV, "non-null"), (dict(out=None), INV, "non-null"), (dict(bt=None), INV, "non-null"),
    (dict(kv_len=None), INV, "non-null"), (dict(stride=0), INV, "bt_stride"), (dict(n_seq=0), INV, "n_seq"),
    (dict(n_seq=65536), INV, "n_seq"), (dict(n_heads=6), INV, "multiple"), (dict(n_heads=12), UNS, "not supported"),
    (dict(n_heads=64), UNS, "not supported"), (dict(max_len=-1), INV, "max_kv_len"), (dict(scale=0.0), INV, "scale"),
    (dict(scale=float("nan")), INV, "scale"), (dict(c=pages(d=32)), UNS, "head_dim"), (dict(ws=P + 8), WS, "aligned"),
    (dict(c=Pages(P, P, None, None, 64, 4, 64, _lib.DTYPE_Q8A)), INV, "scales"),
]


@pytest.mark.parametrize("call", [sink, prefix])
@pytest.mark.parametrize("kw,rc,text", COMMON)
def test_decodes_refuse(call, kw, rc, text):
    got, msg = call(**kw)
    assert got == rc and text in msg, (got, msg)


@pytest.mark.parametrize("kw,rc,text", [(dict(window=-1), INV, "window"), (dict(n_sink=-1), INV, "n_sink"),
                                        (dict(n_sink=2**30 + 1), INV, "n_sink"),
                                        (dict(max_len=4096, window=0, ws_bytes=4096), WS, "needed")])
def test_sink_decode_refuses(kw, rc, text):
    got, msg = sink(**kw)
    assert got == rc and text in msg, (got, msg)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(groups=((0, 3, 32),)), INV, "group 0"), (dict(groups=((2, 1, 32),)), INV, "group 0"),
    (dict(groups=((-1, 1, 32),)), INV, "group 0"), (dict(groups=((0, 0, 32),)), INV, "group 0"),
    (dict(groups=((0, 1, -1),)), INV, "group 0"), (dict(groups=((1, 1, 32), (0, 1, 32))), INV, "group 1"),
    (dict(groups=((0, 2, 32), (1, 1, 32))), INV, "group 1"), (dict(groups=((1, 2**31 - 1, 32),)), INV, "group 0"),
    (dict(groups=None, n_groups=1), INV, "non-null"), (dict(n_groups=-1), INV, "n_groups"),
    (dict(groups=[(i, 1, 32) for i in range(129)], n_seq=200), INV, "n_groups"), (dict(max_len=4096, ws_bytes=4096), WS, "needed"),
])
def test_prefix_decode_refuses(kw, rc, text):
    got, msg = prefix(**kw)
    assert got == rc and text in msg, (got, msg)


def test_prefix_decode_of_large_q8a_pools():
    """2^22 pages x 8 kv heads: 2 GiB of scales, past the page pipeline's 32-bit offsets."""
    big = pages(_lib.DTYPE_Q8A, 128, kv=8, n=1 << 22)
    got, msg = prefix(c=big, n_heads=8)
    assert got == UNS and "2 GiB" in msg
    for ok in (pages(_lib.DTYPE_Q8A, 128, kv=8, n=(1 << 22) - 1), pages(_lib.DTYPE_F16, 128, kv=8, n=1 << 22),
               pages(_lib.DTYPE_Q8A, 64, kv=8, n=1 << 22)):
        got, msg = prefix(c=ok, n_heads=8, max_len=4096, ws_bytes=16)  # further checks come after
        assert got == WS and "needed" in msg


def test_sink_prefill_workspace_query():
    lib, out = _lib.lib(), C.c_size_t(7)

    def size(c, n_chunks=1, n_tok=64, stride=512, window=4096, n_sink=4, n_heads=8):
        rc = lib.lnskv_sink_prefill_workspace_size(C.byref(c), n_chunks, n_tok, stride, window, n_sink, n_heads,
                                                   C.byref(out))
        return rc, out.value
    f16 = pages(_lib.DTYPE_F16, 128)
    assert lib.lnskv_sink_prefill_workspace_size(C.byref(f16), 1, 64, 512, 4096, 4, 8, None) == INV
    for kw in (dict(window=-1), dict(n_sink=-1), dict(n_heads=6)):
        assert size(f16, **kw) == (INV, 0)
    assert size(pages(d=128)) == (UNS, 0) and size(pages(_lib.DTYPE_F16, 64)) == (UNS, 0)
    rc, few = size(f16)  # 64 queries on 4096 tokens: split, a row per query head and split
    assert rc == 0 and few >= 2 * 64 * 8 * (128 + 2) * 4
    assert size(f16, n_tok=1 << 20) == (0, 0)  # tiles enough for every compute unit
    assert size(f16, stride=2) == (0, 0)  # one pair of pages


def test_sink_prefill_refuses():
    def call(c, window=16, n_sink=4, n_heads=8, chunks=P):
        return status("lnskv_sink_prefill_attention", C.byref(c), P, P, chunks, 1, 4, P, 4, 1, window, n_sink, n_heads, 0.1,
                      None, 0, None)
    f16 = pages(_lib.DTYPE_F16, 128)
    for c, kw, rc, text in [(pages(_lib.DTYPE_F16, 64), {}, UNS, "head_dim"), (pages(d=128), {}, UNS, "f16 and Q8A"),
                            (f16, dict(window=-1), INV, "window"), (f16, dict(n_sink=-1), INV, "n_sink"),
                            (f16, dict(n_sink=2**30 + 1), INV, "n_sink"), (f16, dict(n_heads=12), UNS, "not supported"),
                            (f16, dict(chunks=P + 4), INV, "aligned"), (f16, dict(chunks=None), INV, "non-null")]:
        got, msg = call(c, **kw)
        assert got == rc and text in msg, (got, msg)


def test_workspace_queries():
    lib, out = _lib.lib(), C.c_size_t(7)
    c = pages()
    assert lib.lnskv_sink_decode_workspace_size(C.byref(c), 2, 8, 64, 16, 4, None) == INV
    assert lib.lnskv_sink_decode_workspace_size(C.byref(c), 2, 6, 64, 16, 4, C.byref(out)) == INV and out.value == 0
    assert lib.lnskv_sink_decode_workspace_size(C.byref(c), 2, 8, 40, 16, 4, C.byref(out)) == 0 and out.value == 0
    # the window, not the context, decides: partitions of the pages that are read
    sizes = []
    for max_len in (100000, 1000000):
        assert lib.lnskv_sink_decode_workspace_size(C.byref(c), 2, 8, max_len, 1000, 4, C.byref(out)) == 0
        sizes.append(out.value)
    assert sizes[0] == sizes[1] < 1 << 20
    g = i32(0, 2, 32)
    assert lib.lnskv_prefix_decode_workspace_size(C.byref(c), g, 1, 2, 8, 64, None) == INV
    assert lib.lnskv_prefix_decode_workspace_size(C.byref(c), None, 0, 2, 8, 40, C.byref(out)) == 0
    assert out.value == 0  # nothing shared, one partition
    assert lib.lnskv_prefix_decode_workspace_size(C.byref(c), g, 1, 2, 8, 64, C.byref(out)) == 0
    assert out.value == 0  # short: one launch
    assert lib.lnskv_prefix_decode_workspace_size(C.byref(c), g, 1, 2, 8, 4096, C.byref(out)) == 0
    assert out.value >= 4096 + 2 * 8 * (64 + 2) * 4  # a row per query head


def test_python_layer_checks_before_the_call():
    pk = PagedKV(4, 2, 64, _lib.DTYPE_F32, "cpu")
    q, t, kl = torch.zeros(2, 4, 64), torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    kw = dict(n_heads=4, max_kv_len=4, scale=0.1)
    for bad in (dict(q=q.double()), dict(q=q[:1]), dict(kl=kl.long()), dict(t=t[:1]), dict(t=t[0]), dict(gate=q[:, :2])):
        with pytest.raises((TypeError, ValueError)):
            pk.sink_decode(bad.get("q", q), bad.get("t", t), bad.get("kl", kl), window=4, n_sink=1,
                           gate=bad.get("gate"), **kw)
        with pytest.raises((TypeError, ValueError)):
            pk.prefix_decode(bad.get("q", q), bad.get("t", t), bad.get("kl", kl), PrefixGroups([(0, 2, 16)]),
                             gate=bad.get("gate"), **kw)
    with pytest.raises(ValueError):
        PrefixGroups([(0, 2)])
    rope = MRopeTable(torch.ones(32), [16, 16])
    k, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        pk.mrope_append(rope, k, k, i, i, i, t)  # positions of one axis for two
    with pytest.raises(ValueError):
        pk.mrope_append(rope, k, k, i.repeat(2), i, i, t, q_out=q)
    with pytest.raises(ValueError):
        pk.mrope_append(rope, k, k, i.repeat(2), i, i, t.float())
