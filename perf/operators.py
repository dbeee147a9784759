"""Operators of a serving loop over a paged key/value cache, as cases whose time and outputs can be measured.

  rope     lq8.rope_device: rotary positions with one to three axes (text; height, width; time, height, width).
  append   lq8.paged_append_device: per-head RmsNorm of q and k, their rotation, k and v into the pages of a batch.
  attend   lq8.paged_attention_device: attention of a ragged batch over its pages, single tokens and prompt chunks.
  prefix   lq8.prefix_attention_device: the same for groups of sequences that share a prefix.

Where `own` is false, `run` computes the same with elementary torch operations in 32 bits (angles and norm statistics
in 64); where it is true, through the library.  `exact` restates the definitions in 64 bits.
"""
import ctypes
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
THETA = 1e6
EPS = 1e-6
# (query heads, kv heads, head_dim): Qwen3-0.6B's, 4B's and 30B-A3B's heads, heads of their own, small heads
HEADS = [(16, 8, 128), (32, 8, 128), (32, 4, 128), (8, 8, 128), (14, 2, 64), (12, 12, 64)]
PAIRS_TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]
LARGEST_KV = 8 * 131072 * 8 * 128  # elements of K that the largest listed case holds


def listed():
    return [
        # the rotation of one new token's q and k heads, three axes: the smallest call, launch latency
        {"name": "rope_token", "op": "rope", "rows": 1, "heads": 24, "dim": 128, "rotary": 128, "axes": 3, "inter": True, "type": "f32"},
        # the patches of an image (70 x 70) through a vision tower's attention: two axes, 80-wide heads
        {"name": "rope_image", "op": "rope", "rows": 4900, "heads": 32, "dim": 80, "rotary": 80, "axes": 2, "inter": False, "type": "bf16"},
        # one decode step of a busy server: a row per sequence, f32 activations, 16-bit pages
        {"name": "append_decode", "op": "append", "seqs": 48, "chunk": 1, "length": 700, "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "axes": 1, "norm": True, "type": "f32", "cache": "bf16"},
        # ragged prompts with images in them: three axes
        {"name": "append_prompts", "op": "append", "seqs": 5, "chunk": 2047, "length": 2047, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "axes": 3, "norm": True, "type": "bf16", "cache": "bf16"},
        # a single chat token after a page of text, the model's own types
        {"name": "token_1", "op": "attend", "seqs": 1, "chunk": 1, "length": 1001, "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "type": "f32", "cache": "f32"},
        # one decode step of 64 conversations of all lengths
        {"name": "token_64", "op": "attend", "seqs": 64, "chunk": 1, "length": 8190, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "type": "bf16", "cache": "bf16"},
        # long documents: a K of more than 2^31 bytes
        {"name": "token_long", "op": "attend", "seqs": 8, "chunk": 1, "length": 131072, "heads": 32, "kv": 8, "dim": 128, "page": 256,
         "type": "f32", "cache": "bf16"},
        # prompt chunks of three requests behind what is cached already
        {"name": "chunk_bf16", "op": "attend", "seqs": 3, "chunk": 2048, "length": 6100, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "type": "bf16", "cache": "bf16"},
        # the same in the model's own types, one request
        {"name": "chunk_f32", "op": "attend", "seqs": 1, "chunk": 951, "length": 2999, "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "type": "f32", "cache": "f32"},
        # a burst of short questions, small heads
        {"name": "chunk_small", "op": "attend", "seqs": 32, "chunk": 97, "length": 97, "heads": 14, "kv": 2, "dim": 64, "page": 32,
         "type": "bf16", "cache": "bf16"},
        # 64 conversations behind one long system prompt, a token each
        {"name": "prefix_64", "op": "prefix", "seqs": 64, "groups": 1, "prefix": 8192, "chunk": 1, "length": 700, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # two prompts with a few candidates each, three rows a sequence (drafted tokens)
        {"name": "prefix_drafts", "op": "prefix", "seqs": 11, "groups": 2, "prefix": 2001, "chunk": 3, "length": 150, "heads": 16, "kv": 8,
         "dim": 128, "page": 16, "type": "f32", "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend", "prefix", "prefix"])
    if op == "rope":
        dim = 16 * rng.randint(2, 16)
        axes = rng.randint(1, 3)
        return {"op": op, "rows": _log(rng, 1, 6000), "heads": _log(rng, 1, 40), "dim": dim, "rotary": rng.choice([dim, dim, 16 * rng.randint(1, dim // 16)]),
                "axes": axes, "inter": axes == 3 and rng.random() < 0.5, "type": rng.choice(sorted(TYPES))}
    heads, kv, dim = rng.choice(HEADS)
    act, cache = rng.choice(PAIRS_TYPES)
    base = {"op": op, "heads": heads, "kv": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "type": act, "cache": cache}
    single = rng.random() < 0.5
    while True:
        seqs = _log(rng, 1, 64)
        chunk = 1 if single else _log(rng, 2, 2048)
        length = chunk + _log(rng, 1, 40000 if op == "attend" else 3000) - 1
        prefix = _log(rng, 1, 20000) if op == "prefix" else 0
        if op == "append" and seqs * chunk <= 8192 and seqs * length <= 100000:
            return dict(base, seqs=seqs, chunk=chunk, length=length, axes=rng.choice([1, 3]), norm=rng.random() < 0.6)
        kept = seqs * length * kv * dim <= LARGEST_KV // 8 and seqs * chunk * heads * (length + prefix) <= 1 << 30
        if op == "attend" and kept:
            return dict(base, seqs=seqs, chunk=chunk, length=length)
        if op == "prefix" and kept:
            return dict(base, seqs=seqs, chunk=chunk, length=length, prefix=prefix, groups=rng.randint(1, min(3, seqs)))


# ---- the batch of a case: lengths go by the case alone, so that its work does ------------------------------------

def _ragged(most, least, n):
    """n lengths between least and most, the first of them most."""
    return [most - int((most - least) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _counts(case):
    """New rows of each sequence, and its positions with them."""
    n, c = case["seqs"], case["chunk"]
    rows = _ragged(c, max(1, c // 2), n)
    lengths = [max(r, t) for r, t in zip(rows, _ragged(case["length"], max(1, case["length"] // 16), n))]
    if n > 6:  # a place of the batch that no request holds
        rows[5], lengths[5] = (rows[5], 0) if c == 1 else (0, 0)
    return rows, lengths


def _groups(case):
    """First sequence of each group (and the end), and the prefixes' lengths."""
    n, g = case["seqs"], case["groups"]
    return [n * i // g for i in range(g + 1)], _ragged(case["prefix"], max(1, case["prefix"] // 4), g)


def _sections(case):
    """Pairs of each axis: the first one has what an even share leaves over."""
    pairs, axes = case.get("rotary", case["dim"]) // 2, case["axes"]
    return [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)


def _axis_of(case):
    """The axis of each pair."""
    sec, pairs = _sections(case), case.get("rotary", case["dim"]) // 2
    if not case.get("inter"):
        return sum(([a] * s for a, s in enumerate(sec)), [])
    return [i % len(sec) if i < len(sec) * sec[i % len(sec)] else 0 for i in range(pairs)]


# ---- inputs -------------------------------------------------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what * 7919 + 23) % (1 << 62))
    return g


def _normal(seed, what, shape, dtype, std=1.0):
    x = torch.randn(shape, generator=_gen(seed, what), device="cuda", dtype=torch.float32)
    return x.mul_(std).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class _State:
    def __init__(self, case):
        self.case, self.calls, self.handles = case, None, []

    def __del__(self):
        for h in self.handles:
            try:
                h.free()
            except Exception:
                pass


def _positions(case, seed, n):
    """[axes][n] positions: a running time, and the row and column of a patch; some far into a long context."""
    axes = case["axes"]
    at = torch.arange(n, device="cuda", dtype=torch.int64)
    first = int(torch.randint(0, 200000, (1,), generator=_gen(seed, 90), device="cuda"))
    return torch.stack([first + at // (1 + 3 * (axes > 1)), at // 70, at % 70][:axes] if axes != 2 else [at // 70, at % 70]).to(torch.int32).contiguous()


def prepare(case, seed):
    s, op = _State(case), case["op"]
    t = TYPES[case["type"]]
    if op == "rope":
        s.x = _normal(seed, 1, (case["rows"], case["heads"], case["dim"]), t)
        s.y = torch.empty_like(s.x)
        s.positions = _positions(case, seed, case["rows"])
        return s
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    rows, lengths = _counts(case)
    width = max(1, -(-max(lengths) // page))
    lots = [width] * case["seqs"]
    if op == "prefix":
        first, plens = _groups(case)
        pwidth = -(-max(plens) // page)
        lots += [pwidth] * case["groups"]
    s.pages_n = sum(lots) + 3
    order = torch.randperm(s.pages_n, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    s.pages = order[:case["seqs"] * width].reshape(case["seqs"], width).contiguous()
    s.width, s.lengths, s.row_begin = width, _ints(lengths), None
    s.rows = sum(rows)
    s.row_seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), torch.tensor(rows, device="cuda"), output_size=s.rows)
    begin = [sum(rows[:i]) for i in range(len(rows) + 1)]
    s.begin = torch.tensor(begin, device="cuda")
    if case["chunk"] > 1:
        s.row_begin = _ints(begin)
    shape = (s.pages_n, kv, page, dim)
    s.k, s.v = (_normal(seed, w, shape, TYPES[case["cache"]]) for w in (3, 4))
    if op == "append":
        # the projections' output rows, q | k | v side by side
        s.qkv = _normal(seed, 5, (s.rows, heads + 2 * kv, dim), t, 2.0)
        s.q_norm, s.k_norm = (1.0 + _normal(seed, w, (dim,), torch.float32, 0.1) for w in (6, 7))
        s.q_out = torch.empty((s.rows, heads, dim), dtype=t, device="cuda")
        s.positions = _positions(case, seed, s.rows) if case["axes"] > 1 else None
    else:
        s.q = _normal(seed, 5, (s.rows, heads, dim), t, 1.5)
        s.out = torch.empty_like(s.q)
        if op == "prefix":
            s.first, s.plens, s.pwidth = _ints(first), _ints(plens), pwidth
            s.ppages = order[case["seqs"] * width:case["seqs"] * width + case["groups"] * pwidth].reshape(case["groups"], pwidth).contiguous()
    return s


# ---- through the library ------------------------------------------------------------------------------------------

class _Memory:
    """A torch tensor where the library's device calls want a buffer."""

    def __init__(self, t, at=0):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr() + at * t.element_size())


_kept = []


def _context():
    if not _kept:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-omni-inference-rs_amd"))
        import lq8

        _kept.extend([lq8, lq8.Context(0)])
    return _kept


def _mem(t, at=0):
    return None if t is None else _Memory(t, at)


def _descriptors(s):
    """What a serving loop keeps from step to step: the rotation, the descriptions of its cache, batch and buffers."""
    lq8, ctx = _context()
    c = s.case
    dt = {"f32": lq8.DTYPE_F32, "bf16": lq8.DTYPE_BF16}
    if c["op"] in ("rope", "append"):
        rope = lq8.Rope(ctx, c["dim"], THETA, rotary_dim=c.get("rotary"), sections=_sections(c), interleaved=bool(c.get("inter")))
        s.handles.append(rope)
    if c["op"] == "rope":
        return rope, lq8.RopeRows(_Memory(s.x), _Memory(s.y), c["rows"], c["heads"], c["dim"], _Memory(s.positions), dtype=dt[c["type"]])
    kv = lq8.KVPages(_Memory(s.k), _Memory(s.v), s.pages_n, c["page"], c["kv"], c["dim"], dtype=dt[c["cache"]])
    batch = lq8.PagedBatch(_Memory(s.lengths), _Memory(s.pages), c["seqs"], s.width, rows=s.rows, row_begin=_mem(s.row_begin), max_rows=c["chunk"])
    if c["op"] == "append":
        h, d, wide = c["heads"], c["dim"], (c["heads"] + 2 * c["kv"]) * c["dim"]
        norms = (_Memory(s.q_norm), _Memory(s.k_norm)) if c["norm"] else (None, None)
        rows = lq8.QkvRows(_Memory(s.qkv), _Memory(s.qkv, h * d), _Memory(s.qkv, (h + c["kv"]) * d), h, d, q_out=_Memory(s.q_out), stride=wide,
                           q_norm=norms[0], k_norm=norms[1], eps=EPS, positions=_mem(s.positions), positions_stride=s.rows, dtype=dt[c["type"]])
        return rope, kv, batch, rows
    rows = lq8.AttnRows(_Memory(s.q), _Memory(s.out), c["heads"], c["dim"], dtype=dt[c["type"]])
    if c["op"] == "attend":
        return kv, batch, rows
    return kv, batch, lq8.SharedPrefix(_Memory(s.first), _Memory(s.plens), _Memory(s.ppages), c["groups"], s.pwidth), rows


def _library(s):
    lq8, ctx = _context()
    if s.calls is None:
        s.calls = _descriptors(s)
    op = s.case["op"]
    if op == "rope":
        lq8.rope_device(ctx, *s.calls)
        return s.y
    if op == "append":
        lq8.paged_append_device(ctx, *s.calls)
        return {"q": s.q_out, "k": s.k, "v": s.v}
    if op == "attend":
        lq8.paged_attention_device(ctx, *s.calls)
        return s.out
    lq8.prefix_attention_device(ctx, *s.calls)
    return s.out


# ---- the plain form -----------------------------------------------------------------------------------------------

def _rotate(x, positions, case):
    """x [rows][heads][dim] in 32 bits, positions [axes][rows]."""
    rot = case.get("rotary", case["dim"])
    half = rot // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    axis = torch.tensor(_axis_of(case), device=x.device)
    angle = positions.double()[axis].t() * torch.exp(-2.0 * i / rot * math.log(THETA))
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _norm(x, w):
    """RmsNorm of the library: input, weight and result rounded to bf16."""
    v = x.to(torch.bfloat16).double()
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w.to(torch.bfloat16).double()
    return y.float().to(torch.bfloat16).float()


def _slots(s):
    """The position of each new row in its sequence."""
    end = s.begin[1:][s.row_seq]
    return s.lengths[s.row_seq].long() - (end - torch.arange(s.rows, device="cuda"))


def _append(s):
    c = s.case
    h, g = c["heads"], c["kv"]
    x = s.qkv.float()
    q, k, v = x[:, :h], x[:, h:h + g], x[:, h + g:]
    if c["norm"]:
        q, k = _norm(q, s.q_norm), _norm(k, s.k_norm)
    at = _slots(s)
    positions = s.positions if s.positions is not None else at.reshape(1, -1)
    q, k = _rotate(q, positions, c), _rotate(k, positions, c)
    keep = at >= 0
    at, seq = at[keep], s.row_seq[keep]
    page = s.pages[seq, at // c["page"]].long()
    s.k[page, :, at % c["page"]] = k[keep].to(s.k.dtype)
    s.v[page, :, at % c["page"]] = v[keep].to(s.v.dtype)
    return {"q": q.to(s.qkv.dtype), "k": s.k, "v": s.v}


def _dense(cache, pages):
    """[n][positions][kv][dim] in 32 bits, a sequence's pages one behind the other."""
    n, width = pages.shape
    x = cache[pages.long()]  # [n][width][kv][page][dim]
    return x.permute(0, 2, 1, 3, 4).reshape(n, x.shape[2], width * x.shape[3], x.shape[4]).float()


def _scores(q, k, scale, seen):
    return (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill_(~seen, -math.inf)


def _attend(s):
    """All sequences side by side, each padded to the most rows and positions."""
    c = s.case
    heads, kv, dim, n, R = c["heads"], c["kv"], c["dim"], c["seqs"], c["chunk"]
    group, scale = heads // kv, 1.0 / math.sqrt(dim)
    index = torch.arange(s.rows, device="cuda") - s.begin[s.row_seq]
    q = torch.zeros((n, R, heads, dim), device="cuda")
    q[s.row_seq, index] = s.q.float()
    q = q.reshape(n, R, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, R * group, dim)
    k, v = _dense(s.k, s.pages), _dense(s.v, s.pages)
    rows = s.begin[1:] - s.begin[:-1]
    last = s.lengths.long().reshape(-1, 1) - rows.reshape(-1, 1) + torch.arange(R, device="cuda")  # a row's last position
    seen = torch.arange(k.shape[2], device="cuda").reshape(1, 1, -1) <= last.unsqueeze(-1)
    seen = seen.repeat_interleave(group, 1).unsqueeze(1)
    x = _scores(q, k, scale, seen)
    if c["op"] == "prefix":
        of = torch.repeat_interleave(torch.arange(c["groups"], device="cuda"), (s.first[1:] - s.first[:-1]).long(), output_size=n)
        pk, pv = _dense(s.k, s.ppages), _dense(s.v, s.ppages)
        pseen = (torch.arange(pk.shape[2], device="cuda").reshape(1, -1) < s.plens.reshape(-1, 1))[of].reshape(n, 1, 1, -1)
        x = torch.cat([_scores(q, pk[of], scale, pseen), x], -1)
        v = torch.cat([pv[of], v], 2)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    y = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    y = torch.where(torch.isfinite(m), y, torch.zeros_like(y))  # a row that sees nothing
    y = y.reshape(n, kv, R, group, dim).permute(0, 2, 1, 3, 4).reshape(n, R, heads, dim)
    return y[s.row_seq, index].to(s.q.dtype)


def run(s):
    if own:
        return _library(s)
    if s.case["op"] == "rope":
        return _rotate(s.x.float(), s.positions, s.case).to(s.x.dtype)
    return _append(s) if s.case["op"] == "append" else _attend(s)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    a = TYPES[case["type"]].itemsize
    if case["op"] == "rope":
        x = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * x * a + 4 * case["axes"] * case["rows"], "flops": 3 * x}
    rows, lengths = _counts(case)
    c, heads, kv, dim = TYPES[case["cache"]].itemsize, case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        new = sum(r for r, t in zip(rows, lengths) if t)
        return {"bytes": sum(rows) * (2 * heads + 2 * kv) * dim * a + new * 2 * kv * dim * c, "flops": 8 * sum(rows) * (heads + kv) * dim}
    # row i of n sees positions 0 .. length - n + i
    seen = sum(r * (t - r) + r * (r + 1) // 2 for r, t in zip(rows, lengths) if t)
    held = sum(lengths)
    if case["op"] == "prefix":
        first, plens = _groups(case)
        seen += sum(sum(rows[b:e]) * p for b, e, p in zip(first, first[1:], plens))
        held += sum(plens)
    return {"bytes": 2 * held * kv * dim * c + 2 * sum(rows) * heads * dim * a, "flops": 4 * seen * heads * dim}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _turned(x, positions, case):
    x = x.double()
    rot, of = case.get("rotary", case["dim"]), _axis_of(case)
    y = x.clone()
    for i in range(rot // 2):
        angle = (positions[of[i]].double() * THETA ** (-2.0 * i / rot)).reshape(-1, 1)
        a, b = x[..., i], x[..., i + rot // 2]
        y[..., i] = a * torch.cos(angle) - b * torch.sin(angle)
        y[..., i + rot // 2] = a * torch.sin(angle) + b * torch.cos(angle)
    return y


def _softmax_rows(q, k, v, last, scale):
    """One kv head: q [rows][dim], k and v [positions][dim]; row r sees positions 0 .. last[r]."""
    x = q @ k.t() * scale
    x.masked_fill_(torch.arange(k.shape[0], device=q.device).reshape(1, -1) > last.reshape(-1, 1), -math.inf)
    return torch.softmax(x, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s.x, s.positions, case)
    rows, lengths = _counts(case)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    at = [0]
    for r in rows:
        at.append(at[-1] + r)
    if case["op"] == "append":
        slots = torch.tensor([t - r + i for r, t in zip(rows, lengths) for i in range(r)], device="cuda")
        x = s.qkv.double()

        def normed(y, w):
            y = y.to(torch.bfloat16).double()
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.to(torch.bfloat16).double()
            return y.float().to(torch.bfloat16).double()

        q, k, v = x.split([heads, kv, kv], 1)
        if case["norm"]:
            q, k = normed(q, s.q_norm), normed(k, s.k_norm)
        positions = [slots] * case["axes"] if s.positions is None else s.positions
        q, k = _turned(q, positions, case), _turned(k, positions, case)
        kc, vc = s.k.double(), s.v.double()
        ids = torch.tensor([i for i, r in enumerate(rows) for _ in range(r)], device="cuda")
        ok = slots >= 0
        where = s.pages[ids[ok], slots[ok] // page].long()
        kc[where, :, slots[ok] % page], vc[where, :, slots[ok] % page] = k[ok], v[ok]
        return {"q": q, "k": kc, "v": vc}
    out = torch.zeros((s.rows, heads, dim), dtype=torch.float64, device="cuda")
    group, scale = heads // kv, dim ** -0.5
    first, plens = _groups(case) if case["op"] == "prefix" else ([0, case["seqs"]], [0])
    for b, (r, t) in enumerate(zip(rows, lengths)):
        if r == 0:
            continue
        g = max(i for i in range(len(plens)) if first[i] <= b)
        last = plens[g] + t - r + torch.arange(r, device="cuda")
        if plens[g] + t - r < 0:  # an empty place: its row sees nothing
            continue
        for h in range(kv):
            def held(cache):
                x = cache[s.pages[b].long(), h].reshape(-1, dim)[:t]
                return (torch.cat([cache[s.ppages[g].long(), h].reshape(-1, dim)[:plens[g]], x]) if plens[g] else x).double()

            q = s.q[at[b]:at[b + 1], h * group:(h + 1) * group].double().reshape(r * group, dim)
            y = _softmax_rows(q, held(s.k), held(s.v), last.repeat_interleave(group), scale)
            out[at[b]:at[b + 1], h * group:(h + 1) * group] = y.reshape(r, group, dim)
    return out
