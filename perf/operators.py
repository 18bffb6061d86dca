"""The blocks of a hybrid model's layer other than attention, as timed cases: the gated delta rule (token by token and in
chunks), its pre-step, and the mixture-of-experts feed-forward over a few tokens.

Interface: listed() and draw(rng) give cases (dicts of plain values), prepare(case, seed) what a program holds before the
call, run(state) one pass and its outputs, work(case) its unavoidable bytes and flops, exact(case, seed) the same outputs
from the definitions in 64 bits.  `own` says which side run() computes: False the plain form in elementary torch
operations, True the calls of pooled_amd.capi.

The token cases run a few layers of a model, each with a state of its own, as one token's pass does; states go on from
pass to pass as they do in a program.
"""
import math

import torch

own = False

# q/k heads, v heads and their sizes: two and three v heads to a k head, as in mid-size and larger hybrid models, and a
# small shape whose k and v heads differ in size
HEADS = {
    "h32": dict(nk=16, nv=32, hk=128, hv=128),
    "h48": dict(nk=16, nv=48, hk=128, hv=128),
    "small": dict(nk=4, nv=8, hk=64, hv=96),
}
L2_EPS, NORM_EPS = 1e-6, 1e-6
CHUNK = 64
WEIGHT_BYTES = {"f32": 4.0, "q8_0": 1.0625, "q4_0": 0.5625}


def _delta(name, op, heads, cols, **more):
    return dict(dict(name=name, op=op, heads=heads, cols=cols, layers=1, commit=cols, out="f32"), **more)


def _moe(name, cols, **more):
    return dict(dict(name=name, op="moe", cols=cols, dim=2048, ffn=512, experts=256, top_k=8, kind="q4_0", shared=True, renorm=True), **more)


def listed():
    return [
        # one token through the linear-attention layers of a room worker's share of a model: latency
        _delta("delta_token_h32_x8", "decode", "h32", 1, layers=8),
        # a draft of seven tokens of which three were accepted, more v heads
        _delta("delta_verify_h48_7_3_x4", "decode", "h48", 7, commit=3, layers=4),
        # the ragged rest of a prompt
        _delta("delta_rest_h32_77", "prefill", "h32", 77),
        # small heads of unequal sizes, an odd length, f16 results
        _delta("delta_chunk_small_1001_f16", "prefill", "small", 1001, out="f16"),
        # a prompt chunk of the larger shape
        _delta("delta_chunk_h48_2048", "prefill", "h48", 2048),
        # a wide chunk of a long prompt
        _delta("delta_chunk_h32_8192", "prefill", "h32", 8192),
        # the pre-step of one token, of the same layers
        _delta("glue_token_h32_x8", "glue", "h32", 1, layers=8, width=4),
        # the pre-step of a wide prompt chunk
        _delta("glue_chunk_h48_4096", "glue", "h48", 4096, width=4),
        # one token through a feed-forward of many small experts
        _moe("moe_token_q4", 1),
        # a draft of five tokens, int8 weights
        _moe("moe_verify_q8_5", 5, kind="q8_0"),
        # a full-width pass of an engine that feeds its prompts 16 columns at a time
        _moe("moe_pass_q4_16", 16),
        # a small model's unquantised experts, odd counts and sizes, no shared expert, plain probabilities
        _moe("moe_small_f32_27", 27, dim=1056, ffn=352, experts=61, top_k=5, kind="f32", shared=False, renorm=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the same ranges: every operator, shape and option of the listed ones."""
    op = rng.choice(["decode", "prefill", "prefill", "glue", "moe", "moe"])
    heads = rng.choice(sorted(HEADS))
    if op == "decode":
        n = rng.randint(1, 16)
        return _delta("", op, heads, n, commit=rng.randint(0, n), layers=rng.randint(1, 8), out=rng.choice(["f32", "f16"])) | {"name": "drawn"}
    if op == "prefill":
        return _delta("drawn", op, heads, _log_int(rng, 17, 5000 if heads == "h48" else 8000), out=rng.choice(["f32", "f16"]))
    if op == "glue":
        n = _log_int(rng, 1, 4000)
        return _delta("drawn", op, heads, n, commit=n if n > 16 else rng.randint(0, n), layers=rng.randint(1, 8) if n <= 16 else 1, width=rng.choice([2, 3, 4]))
    experts = rng.choice([32, 61, 128, 256])
    return _moe("drawn", _log_int(rng, 1, 32), dim=32 * rng.randint(16, 64), ffn=32 * rng.randint(8, 24), experts=experts, top_k=rng.randint(1, 8),
                kind=rng.choice(["q4_0", "q4_0", "q8_0"] + (["f32"] if experts <= 61 else [])), shared=rng.random() < 0.6, renorm=rng.random() < 0.7)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    unif = lambda *shape: torch.rand(*shape, device="cuda", generator=gen)  # noqa: E731
    n = case["cols"]
    if case["op"] == "moe":
        D, F, E = case["dim"], case["ffn"], case["experts"]
        d = dict(x=rand(n, D), norm=1 + 0.1 * rand(D), router=rand(E, D) * (1.5 / D ** 0.5), shared_gate=rand(D) / D ** 0.5)
        many = E + (1 if case["shared"] else 0)            # the shared expert is kept last
        for name, rows, cols in (("gate", F, D), ("up", F, D), ("down", D, F)):
            spread = unif(many, rows, cols // 32) + 0.5
            if case["kind"] == "f32":
                d[name], d[name + "_s"] = rand(many, rows, cols) / cols ** 0.5, None
            elif case["kind"] == "q8_0":
                d[name] = torch.randint(-127, 128, (many, rows, cols), device="cuda", dtype=torch.int8, generator=gen)
                d[name + "_s"] = (spread / (73.3 * cols ** 0.5)).half()
            else:
                low, high = torch.randint(1, 16, (2, many, rows, cols // 2), device="cuda", dtype=torch.uint8, generator=gen)
                d[name], d[name + "_s"] = low | high << 4, (spread / (4.5 * cols ** 0.5)).half()
        return d
    h, L = HEADS[case["heads"]], case["layers"]
    nk, nv, hk, hv = h["nk"], h["nv"], h["hk"], h["hv"]
    ch = 2 * nk * hk + nv * hv
    a_log = torch.log(1 + 15 * unif(L, nv))                # decay rates of 1 to 16 per unit of time step
    dt = torch.exp(math.log(1e-3) + unif(L, nv) * math.log(100.0))
    if case["op"] == "glue":
        return dict(qkv=rand(L, n, ch), conv_w=rand(L, ch, case["width"]) / case["width"] ** 0.5, conv_b=0.1 * rand(L, ch), a=rand(L, n, nv), b=rand(L, n, nv),
                    a_log=a_log, dt_bias=torch.log(torch.expm1(dt)), state=rand(L, case["width"] - 1, ch))
    # behind the convolution and its activation: values above -0.28 with a positive mean, so that keys are alike
    mixed = torch.nn.functional.silu(rand(L, n, ch))
    step = torch.nn.functional.softplus(rand(L, n, nv) + torch.log(torch.expm1(dt))[:, None])
    return dict(qkv=mixed, g=-torch.exp(a_log)[:, None] * step, beta=torch.sigmoid(rand(L, n, nv)), state=0.1 * rand(L, nv, hv, hk))


# ---- the plain forms: elementary operations in 32 bits ----------------------------------------------------------------

def _heads(case, qkv):
    """[cols, channels] -> q, k of the v heads and v, each [nv, cols, size]; q and k of unit length, q scaled."""
    h = HEADS[case["heads"]]
    nk, nv, hk, hv = h["nk"], h["nv"], h["hk"], h["hv"]
    q, k, v = qkv.split([nk * hk, nk * hk, nv * hv], dim=1)
    unit = lambda t: t * torch.rsqrt((t * t).sum(-1, keepdim=True) + L2_EPS)  # noqa: E731
    wide = lambda t: unit(t.reshape(-1, nk, hk)).repeat_interleave(nv // nk, 1).transpose(0, 1).contiguous()  # noqa: E731
    return wide(q) * hk ** -0.5, wide(k), v.reshape(-1, nv, hv).transpose(0, 1).contiguous()


def _plain_steps(case, qkv, g, beta, S):
    """Token by token; the state after the committed columns."""
    q, k, v = _heads(case, qkv)
    out, kept = [], S
    decay, beta = torch.exp(g).t()[:, :, None, None], beta.t()[:, :, None]
    for t in range(case["cols"]):
        S = decay[:, t] * S
        u = beta[:, t] * (v[:, t] - (S * k[:, t, None, :]).sum(-1))
        S = S + u[:, :, None] * k[:, t, None, :]
        out.append((S * q[:, t, None, :]).sum(-1))
        if t + 1 == case["commit"]:
            kept = S
    return torch.stack(out).reshape(case["cols"], -1), kept


def _plain_chunks(case, qkv, g, beta, S):
    """In chunks: within one, the updates are the solution of a triangular system; between chunks the state is carried."""
    n, (q, k, v) = case["cols"], _heads(case, qkv)
    m = -(-n // CHUNK)
    pad = lambda t: torch.cat([t, t.new_zeros(t.shape[0], m * CHUNK - n, *t.shape[2:])], 1).reshape(t.shape[0], m, CHUNK, *t.shape[2:])  # noqa: E731
    q, k, v, beta = pad(q), pad(k), pad(v), pad(beta.t())
    G = pad(g.t().double()).cumsum(-1)                                       # far sums, near differences
    lower = torch.ones(CHUNK, CHUNK, device=g.device, dtype=torch.bool).tril()
    between = torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], -math.inf)).float()
    kt = k.transpose(-1, -2).contiguous()
    A = torch.matmul(k, kt) * between * beta[..., None]
    P = torch.matmul(q, kt) * between
    T = torch.eye(CHUNK, device=g.device).expand_as(A).clone()
    for i in range(1, CHUNK):                                                # T = (1 + strictly lower A)^-1, row by row
        T[..., i, :i] = -(A[..., i, :i, None] * T[..., :i, :i]).sum(-2)
    start, rest = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
    whole, S = torch.exp(G[..., -1]).float()[..., None, None], S.transpose(-1, -2).contiguous()
    kr, out = (k * rest).transpose(-1, -2).contiguous(), []
    for c in range(m):
        u = torch.matmul(T[:, c], beta[:, c, :, None] * (v[:, c] - start[:, c] * torch.matmul(k[:, c], S)))
        out.append(start[:, c] * torch.matmul(q[:, c], S) + torch.matmul(P[:, c], u))
        S = whole[:, c] * S + torch.matmul(kr[:, c], u)
    return torch.cat(out, 1)[:, :n].transpose(0, 1).reshape(n, -1), S.transpose(-1, -2).contiguous()


def _plain_glue(case, d, l):
    W, n = case["width"], case["cols"]
    x = torch.cat([d["state"][l], d["qkv"][l]])
    y = sum(x[j:j + n] * d["conv_w"][l, :, j] for j in range(W)) + d["conv_b"][l]
    z = d["a"][l] + d["dt_bias"][l]
    softplus = torch.maximum(z, torch.zeros_like(z)) + torch.log1p(torch.exp(-z.abs()))
    d["state"][l] = x[case["commit"]:case["commit"] + W - 1].clone()
    return y / (1 + torch.exp(-y)), -torch.exp(d["a_log"][l]) * softplus, 1 / (1 + torch.exp(-d["b"][l]))


def _wide(case, w, s):
    """Weight planes as f32."""
    if case["kind"] == "f32":
        return w
    if case["kind"] == "q8_0":
        q = w.float().reshape(*w.shape[:-1], -1, 32)
    else:
        b = w.reshape(*w.shape[:-1], -1, 16)
        q = torch.cat([b & 15, b >> 4], -1).float() - 8
    return (q * s.float()[..., None]).reshape(*w.shape[:-1], -1)


def _plain_moe(case, d):
    x, n, E, top = d["x"], case["cols"], case["experts"], case["top_k"]
    xn = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS) * d["norm"]
    logits = torch.matmul(xn, d["router"].t())
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    weight, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    weight, ids = weight[:, :top], ids[:, :top]
    if case["renorm"]:
        weight = weight / weight.sum(-1, keepdim=True)
    use, factor = ids, weight
    if case["shared"]:
        gate = 1 / (1 + torch.exp(-torch.matmul(xn, d["shared_gate"])))
        use, factor = torch.cat([ids, torch.full_like(ids[:, :1], E)], 1), torch.cat([weight, gate[:, None]], 1)
    take = lambda name: _wide(case, d[name][use], None if d[name + "_s"] is None else d[name + "_s"][use])  # noqa: E731  (the chosen experts' planes alone)
    a, b = torch.matmul(take("gate"), xn[:, None, :, None]), torch.matmul(take("up"), xn[:, None, :, None])
    y = torch.matmul(take("down"), a / (1 + torch.exp(-a)) * b)[..., 0]
    return [x + (y * factor[..., None]).sum(1), ids.int(), weight]


def _plain(st):
    case, d = st["case"], st["in"]
    if case["op"] == "moe":
        return _plain_moe(case, d)
    if case["op"] == "glue":
        return [list(_plain_glue(case, d, l)) + [d["state"][l]] for l in range(case["layers"])]
    form, outs = _plain_steps if case["op"] == "decode" else _plain_chunks, []
    for l in range(case["layers"]):
        o, d["state"][l] = form(case, d["qkv"][l], d["g"][l], d["beta"][l], d["state"][l])
        outs.append([o.half() if case["out"] == "f16" else o, d["state"][l]])
    return outs


# ---- the library's calls --------------------------------------------------------------------------------------------

class _Buf:
    """A tensor, or a part of one, where the binding takes one of its device buffers."""

    def __init__(self, tensor, offset=0):
        self.tensor, self.ptr = tensor, tensor.data_ptr() + 4 * offset


class _Memory:
    """Device memory of a handle as torch sees it; keeps the context alive as long as a view of it lives."""

    def __init__(self, pa, ptr, shape):
        self.pa = pa
        self.__cuda_array_interface__ = dict(shape=shape, typestr="<f4", data=(ptr, False), version=2)


_streams = []


def _context(most):
    """A context on the program's stream, closed with its last reference."""
    from pooled_amd.capi import PooledAttn

    class Context(PooledAttn):
        def __del__(self):
            if getattr(self, "ctx", None):
                self.sync()
                self.close()

    if not _streams:
        _streams.append(torch.cuda.Stream())
    pa = Context(dict(n_heads=1, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=NORM_EPS), max(most, 16), n_layers=1, max_cols=max(most, 16))
    pa._chk(pa.L.pa_set_stream(pa.ctx, _streams[0].cuda_stream))
    return pa


def _prepare_own(st):
    from pooled_amd import capi

    case, d, n = st["case"], st["in"], st["case"]["cols"]
    pa = st["pa"] = _context(n)
    if case["op"] == "moe":
        many, host = case["experts"], lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
        part = lambda at: {k: host(at(d[k])) for k in ("gate", "up", "down")} | {k + "_s": None if d[k + "_s"] is None else host(at(d[k + "_s"]).view(torch.int16)) for k in ("gate", "up", "down")}  # noqa: E731
        shared = dict(part(lambda t: t[many]), weight=host(d["shared_gate"])) if case["shared"] else None
        st["moe"] = pa.moe(dict(dim=case["dim"], ffn=case["ffn"], n_experts=many, top_k=case["top_k"], kind={"f32": capi.PA_W_F32, "q8_0": capi.PA_W_Q8_0, "q4_0": capi.PA_W_Q4_0}[case["kind"]],
                                norm_topk=case["renorm"]), host(d["router"]), part(lambda t: t[:many]), shared)
        st["out"] = [torch.empty_like(d["x"]), torch.empty(n, case["top_k"], device="cuda", dtype=torch.int32), torch.empty(n, case["top_k"], device="cuda")]
        st["bufs"] = [_Buf(t) for t in (d["norm"], d["x"], *st["out"])]
        return
    h, L = HEADS[case["heads"]], case["layers"]
    dn = st["dn"] = pa.delta(dict(n_k_heads=h["nk"], n_v_heads=h["nv"], head_k=h["hk"], head_v=h["hv"], conv_width=case.get("width", 0), n_layers=L, eps=L2_EPS, l2norm=True))
    which = 1 if case["op"] == "glue" else 0
    states = [torch.as_tensor(_Memory(pa, pa.delta_state_ptr(dn, l, which), tuple(d["state"][l].shape)), device="cuda") for l in range(L)]
    st["out"], st["bufs"] = [], []
    for l in range(L):
        states[l].copy_(d["state"][l])
        if case["op"] == "glue":
            st["out"].append([torch.empty_like(d["qkv"][l]), torch.empty_like(d["a"][l]), torch.empty_like(d["b"][l]), states[l]])
            st["bufs"].append([_Buf(d[k][l]) for k in ("qkv", "conv_w", "conv_b", "a", "b", "a_log", "dt_bias")] + [_Buf(t) for t in st["out"][l][:3]])
        else:
            o = torch.empty(n, h["nv"] * h["hv"], device="cuda", dtype=torch.float16 if case["out"] == "f16" else torch.float32)
            st["out"].append([o, states[l]])
            st["bufs"].append([_Buf(d["qkv"][l], at) for at in (0, h["nk"] * h["hk"], 2 * h["nk"] * h["hk"])] + [_Buf(d["g"][l]), _Buf(d["beta"][l]), _Buf(o)])
    st["dtype"] = capi.PA_OUT_F16 if case["out"] == "f16" else capi.PA_OUT_F32


def _own(st):
    case, pa, n = st["case"], st["pa"], st["case"]["cols"]
    if case["op"] == "moe":
        norm, x, y, ids, probs = st["bufs"]
        pa.moe_layer(st["moe"], norm, x, case["dim"], n, y, case["dim"], ids, probs)
        return st["out"]
    h, dn = HEADS[case["heads"]], st["dn"]
    nv, col = h["nv"], h["nv"] * h["hv"]
    ch = 2 * h["nk"] * h["hk"] + col
    for l, b in enumerate(st["bufs"]):
        if case["op"] == "glue":
            qkv, w, bias, a, bb, a_log, dt_bias, y, g, beta = b
            pa.delta_glue(dn, l, qkv, ch, w, bias, a, bb, nv, a_log, dt_bias, n, case["commit"], y, ch, g, beta, nv)
        elif case["op"] == "decode":
            q, k, v, g, beta, o = b
            pa.delta_decode(dn, l, q, ch, k, ch, v, ch, g, beta, nv, n, case["commit"], o, col, st["dtype"])
        else:
            q, k, v, g, beta, o = b
            pa.delta_prefill(dn, l, q, ch, k, ch, v, ch, g, beta, nv, n, o, col, st["dtype"])
    return st["out"]


# ---- interface ------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    """The inputs and, for the library's side, the handle with the layers' states or the experts' weights."""
    st = dict(case=case, **{"in": _inputs(case, seed)})
    if own:
        _prepare_own(st)
    torch.cuda.synchronize()
    return st


def run(st):
    """One pass: per layer its results and the state it leaves; for the experts the new residual, the choices and their weights."""
    return _own(st) if own else _plain(st)


def work(case):
    n = case["cols"]
    if case["op"] == "moe":
        D, F, E, top = case["dim"], case["ffn"], case["experts"], case["top_k"]
        # planes of the experts that n tokens choose, were the choices independent
        planes = E * (1 - (1 - top / E) ** n) + (1 if case["shared"] else 0)
        used = top + (1 if case["shared"] else 0)
        return dict(bytes=int(planes * 3 * D * F * WEIGHT_BYTES[case["kind"]] + 4 * E * D + 8 * n * D + 8 * n * top), flops=n * (6.0 * D * F * used + 2.0 * D * E))
    h, L = HEADS[case["heads"]], case["layers"]
    ch, nv = 2 * h["nk"] * h["hk"] + h["nv"] * h["hv"], h["nv"]
    if case["op"] == "glue":
        W = case["width"]
        return dict(bytes=L * 4 * (2 * n * ch + 4 * n * nv + (W + 1) * ch + (W - 1) * ch * (2 if case["commit"] else 1)), flops=L * n * ch * (2.0 * W + 4))
    state = nv * h["hk"] * h["hv"]
    out = n * nv * h["hv"] * (2 if case["out"] == "f16" else 4)
    return dict(bytes=L * (4 * n * (ch + 2 * nv) + out + 4 * state * (2 if case["commit"] else 1)), flops=L * 6.0 * n * state)


def exact(case, seed):
    """The definitions in 64 bits, token by token."""
    d = {k: t.double() if t is not None and t.dtype in (torch.float32, torch.float16) else t for k, t in _inputs(case, seed).items()}
    n = case["cols"]
    if case["op"] == "moe":
        E, rows = case["experts"], []
        for t in range(n):
            x = d["x"][t]
            xn = x / torch.sqrt((x ** 2).mean() + NORM_EPS) * d["norm"]
            p = torch.softmax(d["router"] @ xn, 0)
            ids = sorted(range(E), key=lambda e, p=p.tolist(): (-p[e], e))[:case["top_k"]]
            w = p[ids] / (p[ids].sum() if case["renorm"] else 1)
            parts = list(zip(ids, w)) + ([(E, torch.sigmoid(d["shared_gate"] @ xn))] if case["shared"] else [])
            y = x.clone()
            for e, f in parts:
                gate, up, down = (_widen_64(case["kind"], d[m][e], None if d[m + "_s"] is None else d[m + "_s"][e]) for m in ("gate", "up", "down"))
                a = gate @ xn
                y += f * (down @ (a * torch.sigmoid(a) * (up @ xn)))
            rows.append((y, torch.tensor(ids, dtype=torch.int32, device="cuda"), w))
        return [torch.stack([r[i] for r in rows]) for i in range(3)]
    h = HEADS[case["heads"]]
    nk, nv, hk, hv = h["nk"], h["nv"], h["hk"], h["hv"]
    outs = []
    for l in range(case["layers"]):
        if case["op"] == "glue":
            line = torch.cat([d["state"][l], d["qkv"][l]])
            y = torch.zeros_like(d["qkv"][l]) + d["conv_b"][l]
            for j in range(case["width"]):
                y += line[j:j + n] * d["conv_w"][l, :, j]
            outs.append([y * torch.sigmoid(y), -torch.exp(d["a_log"][l]) * torch.logaddexp(d["a"][l] + d["dt_bias"][l], torch.zeros((), device="cuda", dtype=torch.float64)),
                         torch.sigmoid(d["b"][l]), line[case["commit"]:case["commit"] + case["width"] - 1]])
            continue
        x, S, o = d["qkv"][l], d["state"][l], []
        q, k, v = x[:, :nk * hk].reshape(n, nk, hk), x[:, nk * hk:2 * nk * hk].reshape(n, nk, hk), x[:, 2 * nk * hk:].reshape(n, nv, hv, 1)
        of = torch.arange(nv, device="cuda") // (nv // nk)
        q = (q / torch.sqrt((q ** 2).sum(-1, keepdim=True) + L2_EPS) / math.sqrt(hk))[:, of, :, None]
        k = (k / torch.sqrt((k ** 2).sum(-1, keepdim=True) + L2_EPS))[:, of, :, None]
        decay, beta, kept = torch.exp(d["g"][l])[..., None, None], d["beta"][l][..., None, None], S
        for t in range(n):
            S = S * decay[t]
            S = torch.baddbmm(S, beta[t] * (v[t] - torch.bmm(S, k[t])), k[t].reshape(nv, 1, hk))
            o.append(torch.bmm(S, q[t])[..., 0])
            if t + 1 == case["commit"]:
                kept = S
        outs.append([torch.stack(o).reshape(n, -1), kept])
    return outs


def _widen_64(kind, w, s):
    if kind == "f32":
        return w
    rows = w.shape[0]
    if kind == "q8_0":
        return (w.double().reshape(rows, -1, 32) * s[..., None]).reshape(rows, -1)
    block = w.to(torch.int64).reshape(rows, -1, 1, 16)
    nibbles = torch.cat([block % 16, block // 16], 2) - 8
    return (nibbles.double().reshape(rows, -1, 32) * s[..., None]).reshape(rows, -1)
