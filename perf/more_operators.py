"""Operators around a tree of drafted tokens, a cache that loses rows and positions with several axes, as timed cases: attention
of a tree of drafts over a cache, the pre-step whose columns have positions of their own (one axis, or time, height and width), and
the compaction of a cache to a list of its rows.

Interface: listed() and draw(rng) give cases (dicts of plain values), prepare(case, seed) what a program holds before the
call, run(state) one pass and its outputs, work(case) its unavoidable bytes and flops, exact(case, seed) the same outputs
from the definitions in 64 bits.  `own` says which side run() computes: False the plain form in elementary torch
operations, True the calls of pooled_amd.capi.

Definitions.
  tree     column c of n sees the cache rows 0 .. base - 1 and each row base + j whose bit j is set in its mask:
           out[c, h] = sum_t softmax_t(q[c, h] . k[t, h'] / sqrt(hd)) v[t, h'],  h' = h / (heads per kv head),  times sigmoid(gate) if there is one.
  rope     q and k of a column are divided by their root mean square and weighted; pair i, (x[i], x[i + n_rot / 2]), turns by the angle
           f32(position of the pair's axis) f32(theta^(-2 i / n_rot)), a product in f32: that rounding belongs to the definition, for every other row
           of the cache was turned by such an angle.  q and the gate come out, k and v go to rows base + c of the cache.
  compact  row dst + i of every cache becomes what row list[i] was; the list ascends and list[i] >= dst + i.
"""
import math
import random

import torch

own = False

SHAPES = {
    "dense": dict(nh=16, nkv=8, hd=128, rot=128, theta=1e6, gate=False),
    "moe": dict(nh=16, nkv=2, hd=256, rot=64, theta=1e7, gate=True),
    "large": dict(nh=24, nkv=4, hd=256, rot=64, theta=1e7, gate=True),
}
EPS = 1e-6
PAD = 32                                                                     # rows of a head's plane behind the last one of a context


def _tree(name, shape, nodes, base, **more):
    return dict(dict(name=name, op="tree", shape=shape, nodes=nodes, base=base, layers=1, q8=False), **more)


def _rope(name, shape, cols, base, **more):
    return dict(dict(name=name, op="rope", shape=shape, cols=cols, base=base, layers=1, axes="tree"), **more)


def _compact(name, shape, rows, dst, keep, **more):
    return dict(dict(name=name, op="compact", shape=shape, rows=rows, dst=dst, keep=keep, layers=8, q8=False), **more)


def listed():
    return [
        # a small draft early in a session, through some layers of a dense model: latency
        _tree("tree_dense_5_190_x8", "dense", 5, 190, layers=8),
        # an ordinary draft over an ordinary context
        _tree("tree_moe_24_2011_x4", "moe", 24, 2011, layers=4),
        # int8 rows, odd counts
        _tree("tree_large_q8_17_20003", "large", 17, 20003, q8=True),
        # a wide draft of small heads
        _tree("tree_dense_63_7001", "dense", 63, 7001),
        # a wide draft over a long context
        _tree("tree_large_48_65536", "large", 48, 65536),
        # the pre-step of a draft: a node's position is its depth's
        _rope("rope_tree_moe_24_x8", "moe", 24, 2011, layers=8),
        # an image in a prompt: time, height and width take the pairs in turn
        _rope("rope_image_dense_1001", "dense", 1001, 37, axes="turns"),
        # a video in a longer prompt: each axis has a range of pairs
        _rope("rope_video_large_5003", "large", 5003, 20011, axes="ranges"),
        # the accepted path of a draft moves to the end of the context, in all layers
        _compact("accept_moe_5_of_24_x10", "moe", 625, 601, 5, layers=10),
        # the same of a wider draft, int8 rows
        _compact("accept_large_q8_9_of_60_x12", "large", 1063, 1003, 9, layers=12, q8=True),
        # a context that is cut to half of its rows, its first four kept in place
        _compact("evict_dense_8000_of_16003_x6", "dense", 16003, 4, 8000, layers=6),
        # the same to a third, int8 rows
        _compact("evict_large_q8_10001_of_30011_x3", "large", 30011, 1, 10001, layers=3, q8=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the same ranges: every operator, shape and option of the listed ones."""
    op, shape = rng.choice(["tree", "tree", "rope", "compact"]), rng.choice(sorted(SHAPES))
    if op == "tree":
        nodes = _log_int(rng, 1, 64)
        base = 0 if rng.random() < 0.1 else _log_int(rng, 3, min(65000, 3000000 // nodes))
        return _tree("drawn", shape, nodes, base, layers=rng.randint(1, 6) if base < 3000 else 1, q8=rng.random() < 0.4)
    if op == "rope":
        cols = _log_int(rng, 1, 4900)
        return _rope("drawn", shape, cols, _log_int(rng, 1, 20000), layers=rng.randint(1, 6) if cols < 100 else 1, axes=rng.choice(["tree", "turns", "ranges"]))
    dst, layers = _log_int(rng, 1, 9000), rng.randint(1, 8)
    if rng.random() < 0.5:
        nodes = rng.randint(2, 64)
        return _compact("drawn", shape, dst + nodes, dst, rng.randint(1, min(nodes, 12)), layers=layers, q8=rng.random() < 0.5)
    more = _log_int(rng, 500, 12000)
    return _compact("drawn", shape, dst + more, dst, _log_int(rng, more // 8, more), layers=min(layers, 4), q8=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _ancestors(nodes, rng):
    """A draft tree as each node's list of parents up to its root, itself among them; a parent comes before its children."""
    lines = []
    for c in range(nodes):
        above = rng.randint(max(-1, c - 9), c - 1)
        lines.append((lines[above] if above >= 0 else []) + [c])
    return lines


def _words(lines):
    """The lists as rows of 32-bit mask words."""
    n = len(lines)
    bits = torch.zeros(n, -(-n // 32) * 32, dtype=torch.int64)
    for c, line in enumerate(lines):
        bits[c, line] = 1
    words = (bits.reshape(n, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _axes(case):
    """The axis of each pair and the positions [axes][columns]."""
    s, n, kind = SHAPES[case["shape"]], case["cols"], case["axes"]
    half, c = s["rot"] // 2, torch.arange(n)
    if kind == "tree":
        return torch.zeros(half, dtype=torch.int64), None
    pair = torch.arange(half)
    axis = pair % 3 if kind == "turns" else (pair * 8 >= half * 2).long() + (pair * 8 >= half * 5).long()
    width = max(1, int(math.sqrt(n / (1 if kind == "turns" else 8))))       # frames of width x width patches
    start = case["base"] // 2 + 1                                            # images and videos take fewer positions than rows
    return axis, torch.stack([c // (width * width) + start, c // width % width + start, c % width + start])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = random.Random(int(seed))
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    s, L = SHAPES[case["shape"]], case["layers"]
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]

    def caches(rows):
        """K and V of the layers, [layer][kv head][rows + PAD][hd], the padding zero; int8 with a scale per 32 values."""
        out = {}
        for name in ("k", "v"):
            if case.get("q8"):
                x = torch.randint(-127, 128, (L, nkv, rows + PAD, hd), device="cuda", dtype=torch.int8, generator=gen)
                sc = (torch.rand(L, nkv, rows + PAD, hd // 32, device="cuda", generator=gen) + 0.5) / 73.3
                sc[:, :, rows:] = 0
                out[name + "s"] = sc
            else:
                x = torch.empty(L, nkv, rows + PAD, hd, device="cuda", dtype=torch.float16)
                for l in range(L):
                    x[l] = rand(nkv, rows + PAD, hd).half()
            x[:, :, rows:] = 0
            out[name] = x
        return out

    if case["op"] == "tree":
        n = case["nodes"]
        d = caches(case["base"] + n)
        d["mask"] = _words(_ancestors(n, rng)).cuda()
        d["q"] = 1.5 * rand(L, n, nh * hd)
        d["gate"] = rand(L, n, nh * hd) if s["gate"] else None
        return d
    if case["op"] == "rope":
        n = case["cols"]
        axis, pos = _axes(case)
        if pos is None:
            pos = torch.tensor([[case["base"] + len(line) - 1 for line in _ancestors(n, rng)]])
        inv = (s["theta"] ** (-2.0 * torch.arange(s["rot"] // 2, dtype=torch.float64) / s["rot"])).float()
        d = {k: torch.zeros(L, nkv, case["base"] + n + PAD, hd, device="cuda", dtype=torch.float16) for k in ("k", "v")}
        return dict(d, q_in=rand(L, n, nh * hd * (2 if s["gate"] else 1)), k_in=rand(L, n, nkv * hd), v_in=rand(L, n, nkv * hd),
                    qw=1 + 0.1 * rand(L, hd), kw=1 + 0.1 * rand(L, hd), pos=pos.int().cuda(), axis=axis.cuda(), inv=inv.cuda())
    d = caches(case["rows"])
    at = sorted(rng.sample(range(case["dst"], case["rows"]), case["keep"]))
    return dict(d, sel=torch.tensor([len(at)] + at, dtype=torch.int32).cuda())


# ---- the plain forms: elementary operations in 32 bits ----------------------------------------------------------------

def _wide(d, name, l):
    """A layer's rows as f32."""
    x = d[name][l].float()
    return (x.reshape(*x.shape[:-1], -1, 32) * d[name + "s"][l][..., None]).reshape(x.shape) if name + "s" in d else x


def _plain_tree(case, d, l):
    s, n, base = SHAPES[case["shape"]], case["nodes"], case["base"]
    nkv, hd, G = s["nkv"], s["hd"], s["nh"] // s["nkv"]
    T = base + n
    j = torch.arange(n, device="cuda")
    seen = torch.cat([torch.ones(n, base, device="cuda", dtype=torch.bool), (d["mask"][:, j // 32] >> (j % 32) & 1).bool()], 1)
    q = d["q"][l].reshape(n, nkv, G, hd).permute(1, 0, 2, 3).reshape(nkv, n * G, hd)
    k, v = _wide(d, "k", l)[:, :T].contiguous(), _wide(d, "v", l)[:, :T].contiguous()
    x = (torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)).reshape(nkv, n, G, T)
    x = torch.where(seen[None, :, None], x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul((p / p.sum(-1, keepdim=True)).reshape(nkv, n * G, T), v)
    o = o.reshape(nkv, n, G, hd).permute(1, 0, 2, 3).reshape(n, -1)
    return (o / (1 + torch.exp(-d["gate"][l])) if s["gate"] else o).half()


def _turn(x, w, cos, sin):
    """[n][heads][hd] normed, weighted and rotated."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_rope(case, d, l):
    s, n, base = SHAPES[case["shape"]], case["cols"], case["base"]
    nkv, hd = s["nkv"], s["hd"]
    angle = (d["pos"].t()[:, d["axis"]].float() * d["inv"]).double()         # the product in f32, its cosine and sine in 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = d["q_in"][l].reshape(n, s["nh"], -1)
    q = _turn(x[..., :hd], d["qw"][l], cos, sin).reshape(n, -1)
    d["k"][l][:, base:base + n] = _turn(d["k_in"][l].reshape(n, nkv, hd), d["kw"][l], cos, sin).half().transpose(0, 1)
    d["v"][l][:, base:base + n] = d["v_in"][l].reshape(n, nkv, hd).half().transpose(0, 1)
    return [q] + ([x[..., hd:].reshape(n, -1)] if s["gate"] else [])


def _planes(d):
    return [d[name] for name in ("k", "v", "ks", "vs") if name in d]


def _plain(st):
    case, d = st["case"], st["in"]
    if case["op"] == "tree":
        return [_plain_tree(case, d, l) for l in range(case["layers"])]
    if case["op"] == "rope":
        return [[_plain_rope(case, d, l) for l in range(case["layers"])][-1], d["k"], d["v"]]
    rows, dst = d["sel"][1:].long(), case["dst"]
    for planes in _planes(d):
        for x in planes:
            x[:, dst:dst + case["keep"]] = x[:, rows]
    return _planes(d)


# ---- the library's calls --------------------------------------------------------------------------------------------

class _Buf:
    """A tensor where the binding takes one of its device buffers."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


class _Memory:
    """Device memory of a context as torch sees it; keeps the context alive as long as a view of it lives."""

    def __init__(self, pa, ptr, shape, kind):
        self.pa = pa
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, data=(ptr, False), version=2)


_streams = []


def _context(case, rows, cols):
    """A context with the case's layers on the program's stream, closed with its last reference."""
    from pooled_amd.capi import PooledAttn

    class Context(PooledAttn):
        def __del__(self):
            if getattr(self, "ctx", None):
                self.sync()
                self.close()

    s = SHAPES[case["shape"]]
    if not _streams:
        _streams.append(torch.cuda.Stream())
    pa = Context(dict(n_heads=s["nh"], n_kv_heads=s["nkv"], head_dim=s["hd"], n_rot=s["rot"], rope_theta=s["theta"], eps=EPS, gate=s["gate"], kv_q8=bool(case.get("q8"))),
                 rows, n_layers=case["layers"], max_cols=cols)
    for l in range(case["layers"]):
        pa.layer_alloc(l)
    pa.sync()
    pa._chk(pa.L.pa_set_stream(pa.ctx, _streams[0].cuda_stream))
    return pa


def _prepare_own(st):
    from pooled_amd import capi

    case, d = st["case"], st["in"]
    s, L, op = SHAPES[case["shape"]], case["layers"], case["op"]
    cols = case["nodes"] if op == "tree" else case["cols"] if op == "rope" else 1
    pa = st["pa"] = _context(case, case["rows"] if op == "compact" else case["base"] + cols, cols)
    # the caches hold the inputs' rows; the inputs' own copy goes
    views = []
    for which, name in enumerate(("k", "v", "ks", "vs")):
        if name in d:
            x = d.pop(name)
            kind = {torch.float16: "<f2", torch.int8: "|i1", torch.float32: "<f4"}[x.dtype]
            mine = [torch.as_tensor(_Memory(pa, pa.L.pa_kv_device_ptr(pa.ctx, l, which), tuple(x[l].shape), kind), device="cuda") for l in range(L)]
            for l in range(L):
                mine[l].copy_(x[l])
            views.append(mine)
    st["caches"], st["qd"] = views, s["nh"] * s["hd"]
    if op == "tree":
        st["mask"] = _Buf(d["mask"])
        st["out"] = [torch.empty(case["nodes"], st["qd"], device="cuda", dtype=torch.float16) for _ in range(L)]
        st["bufs"] = [(_Buf(d["q"][l]), _Buf(d["gate"][l]) if s["gate"] else None, _Buf(st["out"][l])) for l in range(L)]
        st["f16"] = capi.PA_OUT_F16
    elif op == "rope":
        pa.set_rope_axes(d["axis"].tolist())
        st["pos"] = _Buf(d["pos"])
        st["bufs"] = [[_Buf(d[k][l]) for k in ("q_in", "k_in", "v_in", "qw", "kw")] for l in range(L)]
        shape = (cols, st["qd"])
        st["out"] = [torch.as_tensor(_Memory(pa, ptr(), shape, "<f4"), device="cuda") for ptr in (pa.q_buffer_ptr, pa.gate_buffer_ptr)[:2 if s["gate"] else 1]]
    else:
        st["sel"] = _Buf(d["sel"])


def _own(st):
    case, pa, qd = st["case"], st["pa"], st["qd"]
    if case["op"] == "tree":
        n, base, mask, words = case["nodes"], case["base"], st["mask"], st["mask"].tensor.shape[1]
        for l, (q, gate, out) in enumerate(st["bufs"]):
            pa.attn_tree(l, q, qd, gate, qd, mask, words, base, n, out, qd, st["f16"])
        return st["out"]
    if case["op"] == "rope":
        n, base, pos = case["cols"], case["base"], st["pos"]
        for l, (q, k, v, qw, kw) in enumerate(st["bufs"]):
            pa.glue_kv_at(l, q, q.tensor.shape[1], k, k.tensor.shape[1], v, v.tensor.shape[1], qw, kw, pos, n, base, n)
        return [st["out"]] + st["caches"]
    pa.kv_compact(case["dst"], st["sel"], case["keep"])
    return st["caches"]


# ---- interface ------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    """The inputs and, for the library's side, a context whose caches hold their rows."""
    st = dict(case=case, **{"in": _inputs(case, seed)})
    if own:
        _prepare_own(st)
    else:
        for name in ("k", "v", "ks", "vs"):
            if name in st["in"]:
                st["in"][name] = list(st["in"][name])
    torch.cuda.synchronize()
    return st


def run(st):
    """One pass: the layers' attention; the q and gate that the pre-step leaves for the last layer, and the layers' caches; or the compacted caches."""
    return _own(st) if own else _plain(st)


def work(case):
    s, L = SHAPES[case["shape"]], case["layers"]
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    row = nkv * (hd + hd // 32 * 4 if case.get("q8") else 2 * hd)             # bytes of a cache row
    if case["op"] == "tree":
        n, base = case["nodes"], case["base"]
        own_rows = n * min(n, 5)                                             # a node sees its ancestors
        return dict(bytes=L * (2 * (base + n) * row + n * nh * hd * (4 + 2 + (4 if s["gate"] else 0))), flops=L * 4.0 * nh * hd * (n * base + own_rows))
    if case["op"] == "rope":
        n, gate = case["cols"], 2 if s["gate"] else 1
        q_layers = L + 1                                                     # the last layer's q and gate stay: of the others, the inputs alone
        return dict(bytes=n * (q_layers * 4 * gate * nh * hd + L * 2 * nkv * hd * (4 + 2)), flops=L * 6.0 * n * hd * (nh + nkv))
    return dict(bytes=L * 4 * case["keep"] * row, flops=0)


def exact(case, seed):
    """The definitions in 64 bits, head by head."""
    d = _inputs(case, seed)
    s, L = SHAPES[case["shape"]], case["layers"]
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    if case["op"] == "compact":
        for x in _planes(d):
            x[:, :, case["dst"]:case["dst"] + case["keep"]] = torch.index_select(x, 2, d["sel"][1:].long())
        return [[x[l].double() if x.is_floating_point() else x[l] for l in range(L)] for x in _planes(d)]
    if case["op"] == "tree":
        n, base, outs = case["nodes"], case["base"], []
        words = d["mask"].cpu().numpy().astype("uint32")
        seen = torch.ones(n, base + n, dtype=torch.bool)
        for c in range(n):
            for j in range(n):
                seen[c, base + j] = bool(int(words[c, j // 32]) >> j % 32 & 1)
        seen = seen.cuda()
        for l in range(L):
            o = torch.empty(n, nh, hd, device="cuda", dtype=torch.float64)
            for h in range(nh):
                k, v = (_row_64(d, name, l, h // (nh // nkv))[:base + n] for name in ("k", "v"))
                x = (d["q"][l].double().reshape(n, nh, hd)[:, h] @ k.t()) / math.sqrt(hd)
                o[:, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
            o = o.reshape(n, -1)
            outs.append(o * torch.sigmoid(d["gate"][l].double()) if s["gate"] else o)
        return outs
    n, base, half, outs = case["cols"], case["base"], s["rot"] // 2, []
    turn = torch.empty(n, half, device="cuda", dtype=torch.complex128)
    for i in range(half):
        angle = (d["pos"][int(d["axis"][i])].float() * d["inv"][i]).double()  # the angle is an f32 product by definition
        turn[:, i] = torch.polar(torch.ones_like(angle), angle)
    K, V = d["k"].double(), d["v"].double()
    for l in range(L):
        def head(x, w):
            x = x.double()
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / hd + EPS) * w.double()
            z = torch.complex(x[:, :half], x[:, half:2 * half]) * turn
            return torch.cat([z.real, z.imag, x[:, 2 * half:]], 1)
        x = d["q_in"][l].reshape(n, nh, -1)
        outs.append([torch.stack([head(x[:, h, :hd], d["qw"][l]) for h in range(nh)], 1).reshape(n, -1)] + ([x[..., hd:].reshape(n, -1).double()] if s["gate"] else []))
        for h in range(nkv):
            at = slice(h * hd, (h + 1) * hd)
            K[l, h, base:base + n] = head(d["k_in"][l][:, at], d["kw"][l])
            V[l, h, base:base + n] = d["v_in"][l][:, at].double()
    return [outs[-1], list(K), list(V)]


def _row_64(d, name, l, h):
    x = d[name][l, h].double()
    return x * d[name + "s"][l, h].double().repeat_interleave(32, -1) if name + "s" in d else x
