"""Operators around the paged K/V cache, as timed cases: the decode step of sequences that share a prefix
(`prefix`), sliding-window attention whose first tokens stay visible, for single tokens (`sink`) and prompt chunks
(`sink_prompt`), and the append that turns q and K by positions of several axes on the way into the pages (`mrope`).

A case names the geometry (query heads, kv heads, head_dim, page type) and the batch; lengths come from the stream
`lens`, so that a case's work does not depend on the seed.  The seed makes the values and the order of the pages in
the pool.  Stored K and V are N(0, 1) in the page's own type (Q8A: codes with a scale per token and kv head), queries
N(0, 2^2), so that scores have the spread of a trained layer's rather than a flat softmax.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 16
ELEM = {"f32": 4, "f16": 2, "q8a": 1}
THETA = 1.0e7
MAX_BYTES = 4.5e8    # what a drawn case reads and writes
MAX_FLOPS = 3.4e10   # and computes
MAX_PLAIN = 2.2e9    # f32 K values that a drawn case's plain form gathers
DEV = "cuda"


def _geom(name, op, pages, heads, kv_heads, dim, lens=1, **more):
    return {"name": name, "op": op, "pages": pages, "heads": heads, "kv_heads": kv_heads, "dim": dim, "lens": lens, **more}


def _prefix(name, pages, heads, kv_heads, dim, seqs, groups, shared, lo, hi, lens=1, gate=False):
    return _geom(name, "prefix", pages, heads, kv_heads, dim, lens, seqs=seqs, groups=groups, shared=shared, lo=lo, hi=hi, gate=gate)


def _sink(name, pages, heads, kv_heads, dim, seqs, lo, hi, window, sink, lens=1, gate=False):
    return _geom(name, "sink", pages, heads, kv_heads, dim, lens, seqs=seqs, lo=lo, hi=hi, window=window, sink=sink, gate=gate)


def _prompt(name, pages, heads, kv_heads, dim, seqs, chunk, lo, hi, window, sink, lens=1):
    return _geom(name, "sink_prompt", pages, heads, kv_heads, dim, lens, seqs=seqs, chunk=chunk, lo=lo, hi=hi, window=window, sink=sink)


def _mrope(name, pages, heads, kv_heads, dim, seqs, chunk, rot, axes, dealt, far, lens=1):
    return _geom(name, "mrope", pages, heads, kv_heads, dim, lens, seqs=seqs, chunk=chunk, rot=rot, axes=axes, dealt=dealt, far=far)


def listed():
    return [
        # The smallest shared step: two answers sampled from one short prompt, 64-wide heads, f32 pages.
        _prefix("prefix_f32_d64_b2", "f32", 32, 4, 64, 2, 1, 256, 1, 64),
        # A batch of 32 users behind one system prompt of 2048 tokens, each some way into its own turn, f16 pages.
        _prefix("prefix_f16_b32", "f16", 32, 8, 128, 32, 1, 2048, 1, 512),
        # Three documents with 16 questions each, 256-wide gated heads on Q8A pages; the prefixes end inside a page.
        _prefix("prefix_q8a_d256_b48", "q8a", 16, 4, 256, 48, 3, 4090, 16, 300, gate=True),
        # A full server behind one long document.
        _prefix("prefix_f16_b128_16k", "f16", 32, 8, 128, 128, 1, 16384, 64, 1024),
        # One user far into a conversation: the window and the first tokens, Q8A pages.  Latency and launches only.
        _sink("sink_q8a_b1", "q8a", 32, 8, 128, 1, 32768, 32768, 1024, 4),
        # A batch of 32 at ragged contexts, some of them shorter than the window, f16 pages.
        _sink("sink_f16_b32", "f16", 32, 8, 128, 32, 512, 16384, 4096, 4),
        # 64-wide heads, f32 pages, a window and a sink that end inside pages.
        _sink("sink_f32_d64_b24", "f32", 32, 4, 64, 24, 40, 9000, 1000, 21),
        # The next prompt tokens of eight sequences, up to 512 each, f16 pages.
        _prompt("sink_prompt_f16_b8", "f16", 32, 8, 128, 8, 512, 64, 8192, 1024, 4),
        # One long prompt's next 1000 tokens, 256-wide heads on Q8A pages.
        _prompt("sink_prompt_q8a_d256_b1", "q8a", 16, 4, 256, 1, 1000, 5003, 5003, 2048, 16),
        # A decode step's append at batch 32: one token of every sequence.  Latency only.
        _mrope("mrope_step_f16_b32", "f16", 32, 8, 128, 32, 1, 128, 3, False, 20000),
        # A prompt with pictures: 4096 tokens, 64 of 256 dims turned by three axes dealt in turn, Q8A pages.
        _mrope("mrope_prompt_q8a_d256", "q8a", 16, 4, 256, 2, 2048, 64, 3, True, 4096),
        # An odd count of tokens, 44 of 64 dims turned, f32 pages.
        _mrope("mrope_prompt_f32_d64", "f32", 32, 4, 64, 7, 143, 44, 3, False, 300),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "sink", "sink", "sink_prompt", "mrope"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 4, 256), (32, 4, 64), (16, 8, 128), (32, 4, 128), (8, 8, 64), (8, 4, 128)])
    pages, lens, gate = rng.choice(["f32", "f16", "f16", "q8a", "q8a"]), rng.randint(2, 1 << 20), rng.random() < 0.25
    if op == "prefix":
        seqs = _log_int(rng, 2, 128)
        hi = _log_int(rng, 2, 1024)
        c = _prefix("", pages, heads, kv, dim, seqs, rng.randint(1, min(4, seqs)), _log_int(rng, 40, 16384), max(1, hi // 8), hi, lens, gate)
        while _too_much(c):
            c["shared"], c["hi"] = c["shared"] * 3 // 4, max(2, c["hi"] * 3 // 4)
            c["lo"] = max(1, c["hi"] // 8)
    elif op == "sink":
        hi = _log_int(rng, 64, 32768)
        c = _sink("", pages, heads, kv, dim, _log_int(rng, 1, 64), hi // 8, hi, _log_int(rng, 16, 4096), rng.randint(0, 64), lens, gate)
        while _too_much(c):
            c["window"] = c["window"] * 3 // 4
    elif op == "sink_prompt":
        if dim == 64:
            heads, kv, dim = 16, 4, 128
        hi = _log_int(rng, 64, 16384)
        c = _prompt("", rng.choice(["f16", "q8a"]), heads, kv, dim, _log_int(rng, 1, 8), _log_int(rng, 16, 1024), hi // 8, hi, _log_int(rng, 32, 4096), rng.randint(0, 64), lens)
        while _too_much(c):
            c["window"], c["chunk"] = max(32, c["window"] * 3 // 4), max(16, c["chunk"] * 3 // 4)
    else:
        axes, rot = rng.randint(1, 3), rng.choice([dim, dim, dim // 2, 44])
        c = _mrope("", pages, heads, kv, dim, _log_int(rng, 1, 16), _log_int(rng, 1, 1024), rot, axes, rng.random() < 0.5, _log_int(rng, 10, 100000), lens)
        while _too_much(c):
            c["chunk"] = c["chunk"] * 3 // 4
    del c["name"]
    return c


def _too_much(c):
    w = work(c)
    plain = 0
    if c["op"] == "prefix":
        plain = c["seqs"] * (c["shared"] + c["hi"]) * c["kv_heads"] * c["dim"]
    elif c["op"] == "sink":
        plain = c["seqs"] * (c["window"] + c["sink"]) * c["kv_heads"] * c["dim"]
    elif c["op"] == "sink_prompt":
        plain = c["seqs"] * c["chunk"] * c["heads"] * (c["window"] + c["chunk"] + c["sink"])
    return w["bytes"] > MAX_BYTES or w["flops"] > MAX_FLOPS or plain > MAX_PLAIN


# ---------------------------------------------------------------------------
# Lengths (from `lens` alone) and inputs (from the seed)


def _lengths(c):
    """prefix: tokens of each sequence past its prefix; sink: tokens of each context, the newest among them;
    sink_prompt, mrope: (tokens before the chunk, tokens of the chunk)."""
    r = random.Random(c["lens"])
    if c["op"] in ("prefix", "sink"):
        return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    if c["op"] == "sink_prompt":
        return [(r.randint(c["lo"], c["hi"]), r.randint((c["chunk"] + 1) // 2, c["chunk"])) for _ in range(c["seqs"])]
    return [(r.randint(0, 40), c["chunk"]) for _ in range(c["seqs"])]


def _groups(c):
    """(first sequence, sequences, shared tokens) of each group; the prefixes differ by some tokens."""
    n, g = c["seqs"], c["groups"]
    cut = [n * i // g for i in range(g + 1)]
    return [(cut[i], cut[i + 1] - cut[i], c["shared"] + 7 * i) for i in range(g)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29)


def _pool(c, num_pages, g):
    kv, d = c["kv_heads"], c["dim"]
    shape = (num_pages, PAGE, kv, d)
    if c["pages"] == "q8a":
        codes = [torch.randn(shape, generator=g, device=DEV).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
        scales = [0.02 + 0.02 * torch.rand((num_pages * PAGE, kv), generator=g, device=DEV) for _ in range(2)]
        return codes + scales
    t = torch.float32 if c["pages"] == "f32" else torch.float16
    return [torch.randn(shape, generator=g, device=DEV, dtype=t) for _ in range(2)] + [None, None]


def _tables(rows, stride, order):
    """Tables [len(rows)][stride] of -1 (no page); rows[s] lists the logical pages of row s that have one.  Pages come
    from `order` one after the other."""
    at = torch.full((len(rows), stride), -1, dtype=torch.int64)
    n = 0
    for s, logical in enumerate(rows):
        at[s, torch.tensor(logical, dtype=torch.int64)] = torch.arange(n, n + len(logical))
        n += len(logical)
    at = at.to(DEV)
    return torch.where(at >= 0, order[at.clamp_min(0)], at).to(torch.int32)


def _inputs(c, seed):
    g, d, kv, H, op = _gen(seed), c["dim"], c["kv_heads"], c["heads"], c["op"]
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    lens, n = _lengths(c), c["seqs"]
    x = {}
    if op == "prefix":
        groups = _groups(c)
        full = {f: P // PAGE for f, _, P in groups}          # whole shared pages, held by the group's first row
        of = [(f, P) for f, m, P in groups for _ in range(m)]
        kv_len = [P + t for (_, P), t in zip(of, lens)]
        stride = -(-max(kv_len) // PAGE)
        rows = [list(range(0 if s == f else full[f], -(-L // PAGE))) for s, ((f, _), L) in enumerate(zip(of, kv_len))]
        x["groups"], x["kv_len"], x["max_len"] = groups, kv_len, max(kv_len)
    elif op == "sink":
        kv_len = lens
        stride = -(-max(kv_len) // PAGE)
        held = lambda L: [p for p in range(-(-L // PAGE)) if p * PAGE < c["sink"] or (p + 1) * PAGE > L - c["window"]]  # noqa: E731
        rows = [held(L) for L in kv_len]
        x["kv_len"], x["max_len"] = kv_len, max(kv_len)
    else:
        stride = max(-(-(a + b) // PAGE) for a, b in lens)
        if op == "sink_prompt":
            rows = [[p for p in range(-(-(a + b) // PAGE)) if p * PAGE < c["sink"] or (p + 1) * PAGE > a + 1 - c["window"]] for a, b in lens]
        else:
            rows = [list(range(-(-(a + b) // PAGE))) for a, b in lens]
    num_pages = sum(map(len, rows)) + 3
    order = torch.randperm(num_pages, generator=g, device=DEV)
    x["tables"] = _tables(rows, stride, order)
    if op == "prefix":
        first = torch.tensor([f for f, m, _ in groups for _ in range(m)], device=DEV)
        whole = torch.tensor([P // PAGE for _, m, P in groups for _ in range(m)], device=DEV)
        x["tables"] = torch.where(torch.arange(stride, device=DEV)[None, :] < whole[:, None], x["tables"][first], x["tables"])
    x["k"], x["v"], x["ks"], x["vs"] = _pool(c, num_pages, g)
    x["num_pages"] = num_pages
    tok = n if op in ("prefix", "sink") else sum(b for _, b in lens)
    x["q"] = 2.0 * rand(tok, H, d)
    x["gate"] = torch.sigmoid(rand(tok, H, d)) if c.get("gate") else None
    if op == "mrope":
        x["k_new"], x["v_new"] = rand(tok, kv, d), rand(tok, kv, d)
        x["axis_pos"] = torch.randint(0, c["far"], (c["axes"], tok), generator=g, device=DEV, dtype=torch.int32)
        half = c["rot"] // 2
        x["inv"] = torch.pow(torch.tensor(THETA, dtype=torch.float64), -torch.arange(half, dtype=torch.float64) / half).float().to(DEV)
    return x


def _sections(c):
    half, axes = c["rot"] // 2, c["axes"]
    if c["dealt"]:  # axis a > 0 has pairs a, a + axes, ...; axis 0 the others
        rest = [len(range(a, half, axes)) for a in range(1, axes)]
    else:
        rest = [half * 3 // 8 if axes == 3 else half // 2] * (axes - 1)
    return [half - sum(rest)] + rest


def prepare(case, seed):
    c, x = case, _inputs(case, seed)
    s = {"case": c, "scale": 1.0 / math.sqrt(c["dim"]), "out": torch.empty_like(x["q"]), **x}
    op, n, lens = c["op"], c["seqs"], _lengths(c)
    if op in ("prefix", "sink"):
        s["kv_len"] = torch.tensor(x["kv_len"], dtype=torch.int32, device=DEV)
    else:
        s["tok_seq"] = torch.tensor([i for i, (_, b) in enumerate(lens) for _ in range(b)], dtype=torch.int32, device=DEV)
        s["tok_pos"] = torch.tensor([a + j for a, b in lens for j in range(b)], dtype=torch.int32, device=DEV)
    if op == "prefix":
        s["first"] = torch.tensor([f for f, m, _ in x["groups"] for _ in range(m)], device=DEV)
        s["whole"] = torch.tensor([P // PAGE for _, m, P in x["groups"] for _ in range(m)], device=DEV)
    if op == "sink_prompt":
        starts = [sum(b for _, b in lens[:i]) for i in range(n)]
        s["chunks"] = torch.tensor([[i, a, b, f] for i, ((a, b), f) in enumerate(zip(lens, starts))], dtype=torch.int32, device=DEV)
    if op == "mrope":
        s["sections"] = _sections(c)
    if own:  # what a program of this library keeps: the layer's pools, the plan and the workspace
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lns-ml_amd"))
        from lnskv import DTYPE_F16, DTYPE_F32, DTYPE_Q8A
        from lnskv.device import MRopeTable, PagedKV, PrefixGroups

        pk = PagedKV(x["num_pages"], c["kv_heads"], c["dim"], {"f32": DTYPE_F32, "f16": DTYPE_F16, "q8a": DTYPE_Q8A}[c["pages"]], DEV)
        for name in ("k", "v", "ks", "vs"):
            if x[name] is not None:
                getattr(pk, name).copy_(x[name])
                s[name] = getattr(pk, name)
        s["pk"] = pk
        if op == "prefix":
            s["plan"] = PrefixGroups(x["groups"])
            s["ws"] = torch.zeros(max(16, pk.prefix_workspace_size(s["plan"], n, c["heads"], x["max_len"])), dtype=torch.uint8, device=DEV)
        elif op == "sink":
            s["ws"] = torch.zeros(max(16, pk.sink_workspace_size(n, c["heads"], x["max_len"], c["window"], c["sink"])), dtype=torch.uint8, device=DEV)
        elif op == "mrope":
            s["rope"] = MRopeTable(x["inv"], s["sections"], interleaved=c["dealt"])
    return s


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if op == "mrope":
        if own:
            s["pk"].mrope_append(s["rope"], s["k_new"], s["v_new"], s["axis_pos"], s["tok_seq"], s["tok_pos"], s["tables"],
                                 q=s["q"], q_out=s["out"])
        else:
            _plain_mrope(s, c)
        if c["pages"] == "q8a":  # codes as the values they stand for
            shape = s["k"].shape[:3] + (1,)
            return {"q": s["out"], "k": s["k"] * s["ks"].view(shape), "v": s["v"] * s["vs"].view(shape)}
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if not own:
        return {"out": {"prefix": _plain_prefix, "sink": _plain_sink, "sink_prompt": _plain_prompt}[op](s, c)}
    kw = dict(n_heads=c["heads"], scale=s["scale"], out=s["out"])
    if op == "prefix":
        out = s["pk"].prefix_decode(s["q"], s["tables"], s["kv_len"], s["plan"], max_kv_len=s["max_len"], gate=s["gate"], workspace=s["ws"], **kw)
    elif op == "sink":
        out = s["pk"].sink_decode(s["q"], s["tables"], s["kv_len"], max_kv_len=s["max_len"], window=c["window"], n_sink=c["sink"], gate=s["gate"], workspace=s["ws"], **kw)
    else:
        out = s["pk"].sink_prefill_attention(s["q"], s["chunks"], s["tables"], window=c["window"], n_sink=c["sink"], **kw)
    return {"out": out}


# ---------------------------------------------------------------------------
# The plain forms


def _rows_of(pool, scales, slots):
    """K or V of slots [n, L] as f32 [n, kv, L, d]."""
    kv, d = pool.shape[2], pool.shape[3]
    t = pool.view(-1, kv, d)[slots].permute(0, 2, 1, 3).to(torch.float32)
    if scales is not None:
        t = t * scales[slots].permute(0, 2, 1)[..., None]
    return t.contiguous()


def _slots(tables, pos):
    """Slot of position pos [n, L] of row n; 0 where pos is outside the row or its page is missing, and where it is not."""
    page = torch.div(pos, PAGE, rounding_mode="floor")
    ok = (pos >= 0) & (page < tables.shape[1])
    phys = torch.gather(tables.long(), 1, page.clamp(0, tables.shape[1] - 1))
    ok = ok & (phys >= 0)
    return torch.where(ok, phys * PAGE + pos % PAGE, torch.zeros_like(pos)), ok


def _attend(q, K, V, seen, scale):
    """q [n, kv, m, d] over K, V [n, kv, L, d]; seen broadcasts to [n, kv, L, m].  Rows that see nothing give zeros."""
    score = torch.matmul(K, q.transpose(2, 3).contiguous()) * scale
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(2, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(2)
    o = torch.matmul(p.transpose(2, 3).contiguous(), V)
    return o / torch.where(total > 0, total, torch.ones_like(total))[..., None]


def _heads_of(s, c):
    return s["q"].view(c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"])


def _plain_prefix(s, c):
    t = s["tables"]
    page = torch.arange(t.shape[1], device=DEV)
    t = torch.where(page[None, :] < s["whole"][:, None], t[s["first"]], t)
    pos = torch.arange(s["max_len"], device=DEV)[None, :].expand(c["seqs"], -1)
    slots, ok = _slots(t, pos)
    seen = (ok & (pos < s["kv_len"].long()[:, None]))[:, None, :, None]
    out = _attend(_heads_of(s, c), _rows_of(s["k"], s["ks"], slots), _rows_of(s["v"], s["vs"], slots), seen, s["scale"]).reshape(s["q"].shape)
    return out * s["gate"] if s["gate"] is not None else out


def _sink_positions(first, count, sink):
    """The sinks' positions, then `count` from first [n] on; a position of both kinds counts once."""
    at = torch.cat([torch.arange(sink, device=DEV)[None, :].expand(first.shape[0], -1), first[:, None] + torch.arange(count, device=DEV)[None, :]], 1)
    once = torch.arange(at.shape[1], device=DEV)[None, :] < sink
    return at, once | (at >= sink)


def _plain_sink(s, c):
    L = s["kv_len"].long()
    pos, once = _sink_positions(L - c["window"], c["window"], c["sink"])
    slots, ok = _slots(s["tables"], pos)
    seen = (ok & once & (pos < L[:, None]))[:, None, :, None]
    out = _attend(_heads_of(s, c), _rows_of(s["k"], s["ks"], slots), _rows_of(s["v"], s["vs"], slots), seen, s["scale"]).reshape(s["q"].shape)
    return out * s["gate"] if s["gate"] is not None else out


def _plain_prompt(s, c):
    ch, kv, d, T = s["chunks"].long(), c["kv_heads"], c["dim"], c["chunk"]
    rep = c["heads"] // kv
    start, length, at = ch[:, 1], ch[:, 2], ch[:, 3]
    pos, once = _sink_positions(start - c["window"] + 1, c["window"] - 1 + T, c["sink"])
    slots, ok = _slots(s["tables"], pos)
    i = torch.arange(T, device=DEV)
    row = (at[:, None] + torch.minimum(i[None, :], length[:, None] - 1))  # past a chunk's end: its last token again
    q = s["q"].view(-1, kv, rep, d)[row].permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, T * rep, d)
    qpos = (start[:, None] + i[None, :]).repeat_interleave(rep, 1)[:, None, :]
    p = pos[:, :, None]
    seen = (ok & once)[:, :, None] & (p <= qpos) & ((p > qpos - c["window"]) | (p < c["sink"]))
    o = _attend(q, _rows_of(s["k"], s["ks"], slots), _rows_of(s["v"], s["vs"], slots), seen[:, None], s["scale"])
    o = o.view(c["seqs"], kv, T, rep, d).permute(0, 2, 1, 3, 4).reshape(c["seqs"] * T, c["heads"], d)
    return o[(i[None, :] < length[:, None]).reshape(-1)]


def _axis_of(c, half):
    """The axis that turns each pair."""
    i = torch.arange(half, device=DEV)
    sec = _sections(c)
    if c["dealt"]:
        return i % c["axes"]
    return torch.repeat_interleave(torch.arange(c["axes"], device=DEV), torch.tensor(sec, device=DEV), output_size=half)


def _turn(x, cos, sin, half):
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1)


def _quantise(x):
    """Q8A codes and scales of x [..., dim]: absmax / 127, f32 quotients, half away from zero."""
    amax = x.abs().amax(-1)
    scale = torch.where(amax == 0, torch.ones_like(amax), (amax.double() / 127.0).float())
    y = (x.double() / scale.double()[..., None]).float().double()
    return torch.clamp(torch.sign(y) * torch.floor(y.abs() + 0.5), -127, 127).to(torch.int8), scale


def _plain_mrope(s, c):
    half, kv, d = c["rot"] // 2, c["kv_heads"], c["dim"]
    angle = s["axis_pos"].double()[_axis_of(c, half)].t() * s["inv"].double()[None, :]  # far positions: 64 bits
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    s["out"].copy_(_turn(s["q"], cos, sin, half))
    rows = {"k": _turn(s["k_new"], cos, sin, half), "v": s["v_new"]}
    pos = s["tok_pos"].long()
    phys = s["tables"][s["tok_seq"].long(), torch.div(pos, PAGE, rounding_mode="floor")].long()
    slot = phys * PAGE + pos % PAGE
    if c["pages"] == "q8a":
        (s["k"].view(-1, kv, d)[slot], s["ks"][slot]), (s["v"].view(-1, kv, d)[slot], s["vs"][slot]) = _quantise(rows["k"]), _quantise(rows["v"])
    else:
        s["k"].view(-1, kv, d)[slot] = rows["k"].to(s["k"].dtype)
        s["v"].view(-1, kv, d)[slot] = rows["v"].to(s["v"].dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    c = case
    lens, kv, d, H = _lengths(c), c["kv_heads"], c["dim"], c["heads"]
    token = 2 * kv * (d * ELEM[c["pages"]] + (4 if c["pages"] == "q8a" else 0))
    row = H * d * 4
    if c["op"] == "mrope":
        n = sum(b for _, b in lens)
        return {"bytes": n * (2 * row + 2 * kv * d * 4 + token + 4 * (c["axes"] + 2)), "flops": n * (H + kv) * c["rot"] * 3}
    if c["op"] == "prefix":
        shared = [(m, P // PAGE * PAGE) for _, m, P in _groups(c)]
        total = [P + t for P, t in zip([P for _, m, P in _groups(c) for _ in range(m)], lens)]
        tokens = sum(total) - sum((m - 1) * P for m, P in shared)
        pairs, rows = sum(total), c["seqs"]
    elif c["op"] == "sink":
        seen = [min(L, c["window"] + min(c["sink"], max(0, L - c["window"]))) for L in lens]
        tokens = pairs = sum(seen)
        rows = c["seqs"]
    else:
        w, k = c["window"], c["sink"]
        pairs = sum(min(p + 1, w + min(k, max(0, p + 1 - w))) for a, b in lens for p in range(a, a + b))
        tokens = sum(min(a + b, w - 1 + b + min(k, max(0, a + 1 - w))) for a, b in lens)
        rows = sum(b for _, b in lens)
    return {"bytes": tokens * token + rows * row * (3 if c.get("gate") else 2) + 4 * -(-tokens // PAGE), "flops": 4 * pairs * H * d}


# ---------------------------------------------------------------------------
# The same in 64 bits, one sequence and kv head at a time


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    kv, d, H, lens = c["kv_heads"], c["dim"], c["heads"], _lengths(c)
    rep = H // kv
    if c["op"] == "mrope":
        return _exact_mrope(c, x, lens)
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device=DEV)

    def attend(rows, tok, h, see):
        """Query rows `rows` (their heads of kv head h) over slots `tok`; see [len(tok), rows] or None."""
        K, V = (p.view(-1, kv, d)[tok, h].double() * (1.0 if sc is None else sc[tok, h].double()[:, None]) for p, sc in ((x["k"], x["ks"]), (x["v"], x["vs"])))
        q = x["q"][rows, h * rep:(h + 1) * rep].double().reshape(-1, d)
        score = (K @ q.t().contiguous()) / math.sqrt(d)
        if see is not None:
            score[~see.repeat_interleave(rep, 1)] = -math.inf
        w = torch.softmax(score, 0)
        out[rows, h * rep:(h + 1) * rep] = (w.t().contiguous() @ V).view(-1, rep, d)

    tables = x["tables"].cpu().tolist()
    at = 0
    for s in range(c["seqs"]):
        if c["op"] == "prefix":
            first, P = next((f, P) for f, m, P in x["groups"] if f <= s < f + m)
            tok, see, rows = list(range(x["kv_len"][s])), None, slice(s, s + 1)
            page = [tables[first if t < P // PAGE * PAGE else s][t // PAGE] for t in tok]
        elif c["op"] == "sink":
            L = x["kv_len"][s]
            tok, see, rows = [t for t in range(L) if t < c["sink"] or t >= L - c["window"]], None, slice(s, s + 1)
            page = [tables[s][t // PAGE] for t in tok]
        else:
            a, b = lens[s]
            tok, rows = [t for t in range(a + b) if t < c["sink"] or t > a - c["window"]], slice(at, at + b)
            at += b
            page = [tables[s][t // PAGE] for t in tok]
            t, p = torch.tensor(tok, device=DEV)[:, None], torch.arange(a, a + b, device=DEV)[None, :]
            see = (t <= p) & ((t < c["sink"]) | (p - t < c["window"]))
        slot = torch.tensor([g * PAGE + t % PAGE for g, t in zip(page, tok)], device=DEV)
        for h in range(kv):
            attend(rows, slot, h, see)
    return {"out": out * x["gate"].double() if x["gate"] is not None else out}


def _exact_mrope(c, x, lens):
    half, kv, d = c["rot"] // 2, c["kv_heads"], c["dim"]
    sec = _sections(c)
    axis = [i % c["axes"] for i in range(half)] if c["dealt"] else [a for a in range(c["axes"]) for _ in range(sec[a])]
    turned = {}
    for name in ("q", "k_new"):
        v = x[name].double()
        z = torch.complex(v[..., :half], v[..., half:2 * half])
        angle = torch.stack([x["axis_pos"][a].double() * x["inv"][i].double() for i, a in enumerate(axis)], 1)
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
        turned[name] = torch.cat([z.real, z.imag, v[..., 2 * half:]], -1)
    if c["pages"] == "q8a":  # codes: roundings, not sums
        return {"q": turned["q"], "k": None, "v": None}
    pools = {"k": x["k"].double(), "v": x["v"].double()}
    tables, n = x["tables"].cpu().tolist(), 0
    for s, (a, b) in enumerate(lens):
        slot = torch.tensor([tables[s][t // PAGE] * PAGE + t % PAGE for t in range(a, a + b)], device=DEV)
        pools["k"].view(-1, kv, d)[slot] = turned["k_new"][n:n + b]
        pools["v"].view(-1, kv, d)[slot] = x["v_new"][n:n + b].double()
        n += b
    return {"q": turned["q"], **pools}
