"""The operators of hybrid state-space / mixture-of-experts decoders whose
speed is measured, in two forms: elementary torch operations, and (where
`own` is true) the graphs a user of this backend computes.

Kinds of cases
  conv    the short causal convolution of a state-space mixer: the carried
          columns joined with the step's (CONCAT), SSM_CONV, its bias, SILU,
          and the columns carried on to the next step
  scan    the selective state-space scan (SSM_SCAN) over a cache of states:
          every sequence's outputs and its state after the last token
  router  the experts of each token: the k largest of its logits (lowest
          expert first among equals) and the softmax over those k
  up      the experts' first products: SILU(W_gate x) * (W_up x) for each of
          a token's experts (two MUL_MAT_ID, SILU, MUL)
  down    the experts' last products, weighted and summed over a token's
          experts (MUL_MAT_ID, MUL, ADDs)

Products round their activations as ggml defines it for the weight's type:
to f16 for F16 weights, to Q8_0 blocks for Q8_0, to Q8_K blocks for Q4_K.
"""

import math

import torch

own = False

DEVICE = "cuda"
CHUNK = 64  # tokens of a chunk of the plain scan


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one decoded token of 32 streams
        dict(name="conv-decode-b32", kind="conv", channels=5376, width=4, tokens=1, seqs=32),
        # two prompts of an odd length
        dict(name="conv-prompt-b2-1777", kind="conv", channels=5376, width=4, tokens=1777, seqs=2),
        # one decoded token of 48 streams: a decay a head
        dict(name="scan-decode-b48", kind="scan", decay="head", state=128, dim=64, heads=80, groups=1, tokens=1,
             seqs=48),
        # two long prompts
        dict(name="scan-prompt-b2-2048", kind="scan", decay="head", state=128, dim=64, heads=80, groups=1,
             tokens=2048, seqs=2),
        # one short prompt of an odd length, several groups
        dict(name="scan-prompt-333", kind="scan", decay="head", state=64, dim=64, heads=24, groups=2, tokens=333,
             seqs=1),
        # a prompt with a decay a state element (one channel a head)
        dict(name="scan-element-1000", kind="scan", decay="element", state=16, dim=1, heads=5120, groups=1,
             tokens=1000, seqs=1),
        # the router of one decoded token: the smallest call, bound by its launch
        dict(name="router-decode-1", kind="router", experts=128, used=8, tokens=1),
        # the router of a batch of prompts
        dict(name="router-prompt-4096", kind="router", experts=128, used=8, tokens=4096),
        # eight decode streams, 4-bit weights: most of the experts read once
        dict(name="up-q4_K-decode-8", kind="up", wtype="q4_K", experts=128, used=8, embd=2048, ffn=768, tokens=8),
        # a prompt of an odd length, f16 weights
        dict(name="up-f16-prompt-1501", kind="up", wtype="f16", experts=32, used=4, embd=2048, ffn=1024, tokens=1501),
        # a prompt, 8-bit weights
        dict(name="down-q8_0-prompt-700", kind="down", wtype="q8_0", experts=64, used=8, embd=2048, ffn=768,
             tokens=700),
        # one decoded token, f16 weights
        dict(name="down-f16-decode-1", kind="down", wtype="f16", experts=32, used=4, embd=2048, ffn=1024, tokens=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["conv", "scan", "scan", "scan", "router", "up", "up", "down", "down"])
    if kind == "conv":
        channels, tokens = _log(rng, 64, 5376), _log(rng, 1, 2000)
        return dict(kind=kind, channels=channels, width=rng.choice([2, 3, 4, 4]), tokens=tokens,
                    seqs=rng.randint(1, max(1, min(32, 4000 // tokens))))
    if kind == "scan":
        tokens = rng.choice([1, _log(rng, 2, 2048)])
        seqs = rng.randint(1, max(1, min(48, 4096 // max(tokens, 64))))
        if rng.random() < 0.3:
            return dict(kind=kind, decay="element", state=16, dim=1, heads=_log(rng, 64, 4096), groups=1,
                        tokens=min(tokens, 1000), seqs=min(seqs, 2))
        groups = rng.choice([1, 1, 2, 4])
        return dict(kind=kind, decay="head", state=rng.choice([64, 128]), dim=rng.choice([32, 64, 64]),
                    heads=groups * rng.randint(1, 80 // groups), groups=groups, tokens=tokens, seqs=seqs)
    if kind == "router":
        return dict(kind=kind, experts=rng.randint(8, 256), used=rng.randint(1, 8), tokens=_log(rng, 1, 4096))
    wtype = rng.choice(["f16", "q8_0", "q4_K"])
    unit = {"f16": 8, "q8_0": 32, "q4_K": 256}[wtype]
    embd, ffn = unit * rng.randint(512 // unit, 2048 // unit), unit * rng.randint(256 // unit, 1024 // unit)
    if kind == "up":  # the products' rows need not come in whole blocks
        ffn = 16 * rng.randint(16, 64)
    else:
        embd = 16 * rng.randint(32, 128)
    experts = rng.choice([8, 16, 32, 48, 64])
    return dict(kind=kind, wtype=wtype, experts=experts, used=rng.randint(1, min(8, experts // 2)), embd=embd, ffn=ffn,
                tokens=_log(rng, 1, 1000))


# ----------------------------------------------------------------- inputs --

def _rng(seed, stream):
    r = torch.Generator(device=DEVICE)
    r.manual_seed((seed * 1000003 + stream) % (1 << 62))
    return r


def _normal(seed, stream, *shape, std=1.0):
    return torch.randn(*shape, generator=_rng(seed, stream), device=DEVICE) * std


def _uniform(seed, stream, lo, hi, *shape):
    return torch.rand(*shape, generator=_rng(seed, stream), device=DEVICE) * (hi - lo) + lo


def _pack(wtype, w):
    """w [..., rows, k] f32 -> f16 weights, or the bytes of ggml's blocks [..., rows, row bytes]"""
    if wtype == "f16":
        return w.half()
    lead = w.shape[:-1]
    if wtype == "q8_0":
        b = w.reshape(-1, 32)
        d = (b.abs().amax(1, keepdim=True) / 127).half()
        q = torch.round(b / d.float().clamp_min(1e-20)).clamp(-127, 127).to(torch.int8)
        return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], 1).reshape(*lead, -1)
    b = w.reshape(-1, 8, 32)
    lo = b.amin(2).clamp_max(0.0)
    scale = (b.amax(2) - lo) / 15
    d = (scale.amax(1, keepdim=True) / 63).half()
    dmin = ((-lo).amax(1, keepdim=True) / 63).half()
    sc = torch.round(scale / d.float()).clamp(1, 63).to(torch.int32)
    mn = torch.round(-lo / dmin.float()).clamp(0, 63).to(torch.int32)
    s32, m32 = d.float() * sc, dmin.float() * mn
    q = torch.round((b + m32[:, :, None]) / s32[:, :, None]).clamp(0, 15).to(torch.uint8)
    scales = torch.cat([(sc[:, :4] & 63) | ((sc[:, 4:] >> 4) << 6), (mn[:, :4] & 63) | ((mn[:, 4:] >> 4) << 6),
                        (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)], 1).to(torch.uint8)
    qs = (q[:, 0::2] | (q[:, 1::2] << 4)).reshape(-1, 128)
    return torch.cat([d.view(torch.uint8), dmin.view(torch.uint8), scales, qs], 1).reshape(*lead, -1)


def _routing(c, seed):
    """each token's experts, some asked for more often than others, and their weights"""
    t, e, k = c["tokens"], c["experts"], c["used"]
    logits = _normal(seed, 1, t, e) + 0.7 * _normal(seed, 2, e)
    top = torch.topk(logits, k, dim=1)
    return top.indices.to(torch.int32).contiguous(), torch.softmax(top.values, 1).contiguous()


def prepare(case, seed):
    c = case
    if c["kind"] == "conv":
        return dict(case=c, x=_normal(seed, 1, c["seqs"], c["tokens"], c["channels"]),
                    carried=_normal(seed, 2, c["seqs"], c["channels"], c["width"] - 1),
                    w=_normal(seed, 3, c["channels"], c["width"], std=0.5), b=_normal(seed, 4, c["channels"], std=0.2))
    if c["kind"] == "scan":
        s, t, h, p, g, n = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
        slots = s + 3  # the cache holds other sequences too
        ids = torch.randperm(slots, generator=_rng(seed, 9), device=DEVICE)[:s].to(torch.int32)
        step = torch.exp(_uniform(seed, 1, math.log(1e-3), math.log(1e-1), h))  # the heads' usual step sizes
        dt = torch.log(torch.expm1(step)) + _normal(seed, 2, s, t, h, std=0.5)  # softplus comes in the scan
        a = -_uniform(seed, 3, 1.0, 16.0, *((h, 1) if c["decay"] == "head" else (h, n)))
        return dict(case=c, ids=ids, dt=dt, a=a, x=_normal(seed, 4, s, t, h, p), b=_normal(seed, 5, s, t, g, n),
                    c=_normal(seed, 6, s, t, g, n), states=_normal(seed, 7, slots, h, p, n, std=0.5))
    if c["kind"] == "router":
        return dict(case=c, logits=_normal(seed, 1, c["tokens"], c["experts"], std=2.0))
    ids, weights = _routing(c, seed)
    e, d, f, t = c["experts"], c["embd"], c["ffn"], c["tokens"]
    if c["kind"] == "up":
        return dict(case=c, ids=ids, x=_normal(seed, 3, t, d), gate=_pack(c["wtype"], _normal(seed, 4, e, f, d, std=0.02)),
                    up=_pack(c["wtype"], _normal(seed, 5, e, f, d, std=0.02)))
    return dict(case=c, ids=ids, weights=weights, h=_normal(seed, 3, t, c["used"], f),
                down=_pack(c["wtype"], _normal(seed, 4, e, d, f, std=0.02)))


# ------------------------------------------------------------ plain forms --

def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(s):
    c = s["case"]
    cols = torch.cat([s["carried"], s["x"].transpose(1, 2)], 2)
    y = (cols.unfold(2, c["width"], 1) * s["w"][:, None, :]).sum(3) + s["b"][:, None]
    return {"y": _silu(y).transpose(1, 2).contiguous(), "carried": cols[:, :, c["tokens"]:].contiguous()}


def _softplus(x):
    return torch.where(x <= 20, torch.log1p(torch.exp(x)), x)


def _plain_scan_heads(s):
    """chunks of tokens as matrix products, their states joined by the decays between chunks"""
    c = s["case"]
    S, T, H, P, G, N = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
    L = min(CHUNK, T)
    nc = -(-T // L)
    pad = nc * L - T
    dt = _softplus(s["dt"])
    a = dt.double() * s["a"][:, 0].double()
    x = s["x"] * dt[..., None]

    def chunks(v):  # [S, T, ...] -> [S, nc, L, ...], what is past T zero: it neither decays nor adds
        v = torch.cat([v, v.new_zeros(S, pad, *v.shape[2:])], 1) if pad else v
        return v.reshape(S, nc, L, *v.shape[2:])

    cum = chunks(a).cumsum(2).permute(0, 1, 3, 2).contiguous()                         # [S, nc, H, L]
    x = chunks(x).permute(0, 1, 3, 2, 4).contiguous()                                  # [S, nc, H, L, P]
    b, cc = (chunks(s[k]).permute(0, 1, 3, 2, 4).contiguous() for k in ("b", "c"))     # [S, nc, G, L, N]
    rep = H // G
    bh, ch = (v[:, :, :, None].expand(S, nc, G, rep, L, N).reshape(S, nc, H, L, N) for v in (b, cc))
    seen = torch.ones(L, L, dtype=torch.bool, device=DEVICE).tril()
    decay = torch.where(seen, torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(~seen, 0.0)), 0.0).float()
    cb = torch.matmul(cc, b.transpose(-1, -2))[:, :, :, None].expand(S, nc, G, rep, L, L).reshape(S, nc, H, L, L)
    y = torch.matmul(cb * decay, x)
    left = torch.exp(cum[..., -1:] - cum).float()                                      # from a token to its chunk's end
    add = torch.matmul((x * left[..., None]).transpose(-1, -2), bh)                    # [S, nc, H, P, N]
    first = s["states"][s["ids"].long()]
    add = torch.cat([first[:, None], add], 1)
    ends = torch.cat([cum.new_zeros(S, 1, H), cum[..., -1].cumsum(1)], 1).transpose(1, 2)  # [S, H, nc + 1]
    seen = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=DEVICE).tril()
    between = torch.where(seen, torch.exp((ends[..., :, None] - ends[..., None, :]).masked_fill(~seen, 0.0)), 0.0).float()
    states = torch.matmul(between, add.permute(0, 2, 1, 3, 4).reshape(S, H, nc + 1, P * N))
    states = states.reshape(S, H, nc + 1, P, N)
    entering = states[:, :, :nc].permute(0, 2, 1, 3, 4)
    y = y + torch.matmul(ch * torch.exp(cum).float()[..., None], entering.transpose(-1, -2))
    y = y.permute(0, 1, 3, 2, 4).reshape(S, nc * L, H, P)[:, :T].contiguous()
    return {"y": y, "states": states[:, :, nc].contiguous()}


def _plain_scan_elements(s):
    """a doubling prefix scan of the recurrences h = a h + b"""
    c = s["case"]
    S, T, H, P, G, N = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
    dt = _softplus(s["dt"])

    def heads(v):
        return v[:, :, :, None].expand(S, T, G, H // G, N).reshape(S, T, H, 1, N)

    a = torch.exp(dt[..., None] * s["a"]).reshape(S, T, H, 1, N)
    h = (s["x"] * dt[..., None])[..., None] * heads(s["b"])
    h[:, 0] += a[:, 0] * s["states"][s["ids"].long()]
    at = 1
    while at < T:
        h = torch.cat([h[:, :at], h[:, at:] + a[:, at:] * h[:, :-at]], 1)
        a = torch.cat([a[:, :at], a[:, at:] * a[:, :-at]], 1)
        at *= 2
    return {"y": (h * heads(s["c"])).sum(4), "states": h[:, T - 1].contiguous()}


def _plain_router(s):
    values, ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    k = s["case"]["used"]
    e = torch.exp(values[:, :k] - values[:, :1])
    return {"ids": ids[:, :k].to(torch.int32), "weights": e / e.sum(1, keepdim=True)}


def _rounded(wtype, x):
    """x [n, k] f32 as the product of this weight type sees it"""
    if wtype == "f16":
        return x.half().float()
    # quotients of two tensors: a number among the operands is multiplied by, as a reciprocal
    if wtype == "q8_0":
        b = x.reshape(-1, 32)
        top = b.abs().amax(1, keepdim=True)
        n = torch.full_like(top, 127.0)
        q = torch.round(b * torch.where(top > 0, n / top, 0.0))
        return (q * (top / n).half().float()).reshape(x.shape)
    b = x.reshape(-1, 256)
    top = torch.gather(b, 1, b.abs().argmax(1, keepdim=True))  # with its sign
    scale = torch.where(top != 0, torch.full_like(top, -127.0) / top, 0.0)
    q = torch.round(b * scale).clamp_max(127.0)
    return (q * torch.where(top != 0, torch.ones_like(top) / scale, 0.0)).reshape(x.shape)


def _weights(wtype, raw, k):
    """the f32 weights [..., rows, k] of packed ones"""
    if wtype == "f16":
        return raw.float()
    lead = raw.shape[:-1]
    if wtype == "q8_0":
        b = raw.reshape(-1, 34)
        return (b[:, 2:].view(torch.int8).float() * b[:, :2].contiguous().view(torch.float16).float()).reshape(*lead, k)
    b = raw.reshape(-1, 144)
    d, dmin = (b[:, i:i + 2].contiguous().view(torch.float16).float() for i in (0, 2))
    s = b[:, 4:16].to(torch.int32)
    sc = torch.cat([s[:, :4] & 63, (s[:, 8:] & 15) | ((s[:, :4] >> 6) << 4)], 1).float()
    mn = torch.cat([s[:, 4:8] & 63, (s[:, 8:] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1).float()
    q = b[:, 16:].reshape(-1, 4, 1, 32)
    q = torch.cat([q & 15, q >> 4], 2).reshape(-1, 8, 32).float()
    return ((d * sc)[:, :, None] * q - (dmin * mn)[:, :, None]).reshape(*lead, k)


def _plain_products(wtype, packed, x, expert):
    """row i of x [n, k] by expert[i]'s matrix of each packed [E, rows, ...]: the experts gathered
    where there are few rows, else expert by expert"""
    n, k = x.shape
    x = _rounded(wtype, x)
    rows = packed[0].shape[1]
    if n * rows * k <= 1 << 28:
        return [torch.matmul(_weights(wtype, p[expert], k), x[:, :, None])[:, :, 0] for p in packed]
    order = torch.argsort(expert, stable=True)
    counts = torch.bincount(expert, minlength=packed[0].shape[0]).tolist()
    parts = torch.split(order, counts)
    out = [x.new_empty(n, rows) for _ in packed]
    for p, o in zip(packed, out):
        w = _weights(wtype, p, k)
        for e, at in enumerate(parts):
            if len(at):
                o[at] = torch.matmul(x[at], w[e].t())
    return out


def _plain_up(s):
    c = s["case"]
    t, k = c["tokens"], c["used"]
    x = s["x"][:, None].expand(t, k, c["embd"]).reshape(t * k, -1)
    gate, up = _plain_products(c["wtype"], [s["gate"], s["up"]], x, s["ids"].reshape(-1).long())
    return {"h": (_silu(gate) * up).reshape(t, k, -1)}


def _plain_down(s):
    c = s["case"]
    t, k = c["tokens"], c["used"]
    y, = _plain_products(c["wtype"], [s["down"]], s["h"].reshape(t * k, -1), s["ids"].reshape(-1).long())
    return {"y": (y.reshape(t, k, -1) * s["weights"][:, :, None]).sum(1)}


PLAIN = {"conv": _plain_conv, "router": _plain_router, "up": _plain_up, "down": _plain_down}


# ------------------------------------------------------- the backend's form --

class _Memory:
    """device memory for torch; a tensor made of it keeps its owner, and so the memory, alive"""

    def __init__(self, owner, ptr, shape, strides, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=typestr, data=(ptr, False), version=3,
                                             strides=tuple(strides))


class _Program:
    """one ggml graph over a state's tensors, and torch views of its results"""

    def __init__(self, n_tensors=64):
        from openasr_amd import ggml as g
        self.g = g
        self.G = g.Graph(n_tensors=n_tensors, graph_size=n_tensors)
        self.lib, self.ctx = self.G.lib, self.G.ctx
        self.backend = g.plugin().backend
        self.packed = []

    def over(self, t, *ne):
        """a graph tensor whose bytes are those of the torch tensor t"""
        types = {torch.float32: self.g.F32, torch.float16: self.g.F16, torch.int32: self.g.I32, torch.uint8: self.g.Q4_K}
        return self.G.over(types[t.dtype], *ne, memory=t)

    def weights(self, wtype, raw, k):
        """a model's expert matrices [E, rows, row]: f16 and Q4_K as they are in memory, Q8_0 through the backend's own layout"""
        e, rows = raw.shape[:2]
        if wtype != "q8_0":
            return self.over(raw, k, rows, e)
        t = self.G.new(self.g.Q8_0, k, rows, e, weight=True)
        self.packed.append((t, raw))
        return t

    def done(self, **outputs):
        """the graph allocated for these results: name -> (tensor, shape, offset in bytes)"""
        self.G.build(*dict.fromkeys(t for t, _, _ in outputs.values()))
        self.G.allocate(self.g.plugin().buft)
        for t, raw in self.packed:
            self.G.set(t, raw.reshape(-1).cpu().numpy())
        self.packed = []
        torch.cuda.current_stream().synchronize()  # the state's tensors are written before the first compute reads them
        self.views = {}
        for name, (t, shape, at) in outputs.items():
            tt = self.g.tensor(t)
            kind, size = {self.g.F32: ("<f4", 4), self.g.I32: ("<i4", 4)}[tt.type]
            if at is None:  # rows of a wider tensor
                strides = [int(tt.nb[1]), size]
            else:
                strides = [size * math.prod(shape[i + 1:]) for i in range(len(shape))]
            self.views[name] = torch.as_tensor(_Memory(self.G, tt.data + (at or 0), shape, strides, kind), device=DEVICE)
        return self

    def __call__(self):
        if self.G.compute(self.backend) != 0:
            raise RuntimeError("graph compute failed")
        return dict(self.views)


def _own_conv(s):
    c = s["case"]
    C, W, T, S = c["channels"], c["width"], c["tokens"], c["seqs"]
    p = _Program()
    L, ctx = p.lib, p.ctx
    cols = L.ggml_concat(ctx, p.over(s["carried"], W - 1, C, S), L.ggml_transpose(ctx, p.over(s["x"], C, T, S)), 0)
    y = L.ggml_ssm_conv(ctx, cols, p.over(s["w"], W, C))
    y = L.ggml_silu(ctx, L.ggml_add(ctx, y, p.over(s["b"], C)))
    row = 4 * (W - 1 + T)
    carried = L.ggml_cont(ctx, L.ggml_view_3d(ctx, cols, W - 1, C, S, row, row * C, 4 * T))
    return p.done(y=(y, [S, T, C], 0), carried=(carried, [S, C, W - 1], 0))


def _own_scan(s):
    c = s["case"]
    S, T, H, P, G, N = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
    p = _Program()
    y = p.lib.ggml_ssm_scan(p.ctx, p.over(s["states"], N, P, H, s["states"].shape[0]), p.over(s["x"], P, H, T, S),
                            p.over(s["dt"], H, T, S), p.over(s["a"], s["a"].shape[1], H), p.over(s["b"], N, G, T, S),
                            p.over(s["c"], N, G, T, S), p.over(s["ids"], S))
    return p.done(y=(y, [S, T, H, P], 0), states=(y, [S, H, P, N], 4 * S * T * H * P))


def _own_router(s):
    c = s["case"]
    E, k, T = c["experts"], c["used"], c["tokens"]
    p = _Program()
    L, ctx = p.lib, p.ctx
    logits = p.over(s["logits"], E, T)
    ids = L.ggml_top_k(ctx, logits, k)
    w = L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, logits, 1, E, T), ids)
    w = L.ggml_soft_max(ctx, L.ggml_reshape_2d(ctx, w, k, T))
    return p.done(ids=(ids, [T, k], None), weights=(w, [T, k], 0))


def _own_up(s):
    c = s["case"]
    K, F, T, k = c["embd"], c["ffn"], c["tokens"], c["used"]
    p = _Program()
    L, ctx = p.lib, p.ctx
    x, ids = p.over(s["x"], K, 1, T), p.over(s["ids"], k, T)
    gate, up = (L.ggml_mul_mat_id(ctx, p.weights(c["wtype"], s[n], K), x, ids) for n in ("gate", "up"))
    return p.done(h=(L.ggml_mul(ctx, L.ggml_silu(ctx, gate), up), [T, k, F], 0))


def _own_down(s):
    c = s["case"]
    M, F, T, k = c["embd"], c["ffn"], c["tokens"], c["used"]
    p = _Program()
    L, ctx = p.lib, p.ctx
    y = L.ggml_mul_mat_id(ctx, p.weights(c["wtype"], s["down"], F), p.over(s["h"], F, k, T), p.over(s["ids"], k, T))
    y = L.ggml_mul(ctx, y, p.over(s["weights"], 1, k, T))
    parts = [L.ggml_view_2d(ctx, y, M, T, 4 * M * k, 4 * M * i) for i in range(k)]
    out = parts[0] if k > 1 else L.ggml_cont(ctx, parts[0])
    for q in parts[1:]:
        out = L.ggml_add(ctx, out, q)
    return p.done(y=(out, [T, M], 0))


OWN = {"conv": _own_conv, "scan": _own_scan, "router": _own_router, "up": _own_up, "down": _own_down}


def run(state):
    c = state["case"]
    if own:
        if "program" not in state:
            state["program"] = OWN[c["kind"]](state)
        return state["program"]()
    if c["kind"] == "scan":
        return (_plain_scan_heads if c["decay"] == "head" else _plain_scan_elements)(state)
    return PLAIN[c["kind"]](state)


# ------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "conv":
        n = c["channels"] * c["seqs"]
        moved = n * (2 * c["tokens"] + 2 * (c["width"] - 1)) + c["channels"] * (c["width"] + 1)
        return {"bytes": 4.0 * moved, "flops": n * c["tokens"] * (2.0 * c["width"] + 5)}
    if c["kind"] == "scan":
        s, t, h, p, g, n = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
        moved = s * t * (2 * h * p + h + 2 * g * n) + 2 * s * h * p * n + h * (n if c["decay"] == "element" else 1)
        # a token's step adds x B to the state and takes C from it
        return {"bytes": 4.0 * moved, "flops": 4.0 * s * t * h * p * n}
    if c["kind"] == "router":
        return {"bytes": 4.0 * c["tokens"] * (c["experts"] + 2 * c["used"]), "flops": 1.0 * c["tokens"] * c["experts"]}
    pairs = c["tokens"] * c["used"]
    a_weight = {"f16": 2.0, "q8_0": 34 / 32, "q4_K": 144 / 256}[c["wtype"]]
    read = min(c["experts"], pairs) * c["embd"] * c["ffn"] * a_weight  # at most so many experts are asked for
    if c["kind"] == "up":
        return {"bytes": 2 * read + 4.0 * (c["tokens"] * c["embd"] + pairs * (c["ffn"] + 1)),
                "flops": 4.0 * pairs * c["embd"] * c["ffn"]}
    return {"bytes": read + 4.0 * (pairs * (c["ffn"] + 2) + c["tokens"] * c["embd"]),
            "flops": 2.0 * pairs * c["embd"] * c["ffn"]}


# ------------------------------------------------------------------ exact --

def _exact_conv(s):
    c = s["case"]
    x, carried, w, b = (s[k].double() for k in ("x", "carried", "w", "b"))
    cols = torch.cat([carried.transpose(1, 2), x], 1)
    y = b + sum(cols[:, i:i + c["tokens"]] * w[:, i] for i in range(c["width"]))
    return {"y": y * torch.sigmoid(y), "carried": cols[:, c["tokens"]:].transpose(1, 2).contiguous()}


def _exact_scan(s):
    """token by token"""
    c = s["case"]
    S, T, H, P, G, N = (c[k] for k in ("seqs", "tokens", "heads", "dim", "groups", "state"))
    h = s["states"][s["ids"].long()].double()
    a, r = s["a"].double(), H // G
    y = torch.empty(S, T, H, P, dtype=torch.float64, device=DEVICE)
    for t in range(T):
        d = s["dt"][:, t].double()
        d = torch.where(d <= 20, torch.log1p(torch.exp(d)), d)
        b, cc = (s[k][:, t].double().repeat_interleave(r, 1)[:, :, None] for k in ("b", "c"))
        h = h * torch.exp(d[:, :, None] * a)[:, :, None] + (s["x"][:, t].double() * d[:, :, None])[..., None] * b
        y[:, t] = (h * cc).sum(3)
    return {"y": y, "states": h}


def _exact_router(s):
    k = s["case"]["used"]
    order = torch.argsort(-s["logits"].double(), dim=1, stable=True)[:, :k]
    return {"ids": order.to(torch.int32), "weights": torch.softmax(torch.gather(s["logits"].double(), 1, order), 1)}


def _exact_activations(wtype, x):
    """the rounded activations as (whole numbers, scales): the blocks' rounding is the operator's definition, in f32"""
    if wtype == "f16":
        return x.half().double()
    if wtype == "q8_0":
        v = x.reshape(-1, 32)
        m = v.abs().max(1, keepdim=True).values
        q = torch.round(v * (127.0 / m.double()).float()).nan_to_num(0.0).double()
        return (q * (m.double() / 127.0).float().half().double()).reshape(x.shape)
    v = x.reshape(-1, 256)
    hi, lo = v.max(1, keepdim=True).values, v.min(1, keepdim=True).values
    m = torch.where(hi >= -lo, hi, lo)
    i = (-127.0 / m.double()).float()
    q = torch.round(v * i).clamp_max(127.0).nan_to_num(0.0).double()
    return (q * (1.0 / i.double()).float().double()).reshape(x.shape)


def _exact_matrix(wtype, raw, k):
    """one expert's weights in f64, block by block of the storage format"""
    if wtype == "f16":
        return raw.double()
    rows = raw.shape[0]
    if wtype == "q8_0":
        v = raw.reshape(rows, k // 32, 34)
        return (v[..., :2].contiguous().view(torch.float16).double() * v[..., 2:].contiguous().view(torch.int8).double()).reshape(rows, k)
    v = raw.reshape(rows, k // 256, 144)
    d, dmin = v[..., 0:2].contiguous().view(torch.float16).double(), v[..., 2:4].contiguous().view(torch.float16).double()
    u = v[..., 4:16].int()
    out = torch.empty(rows, k // 256, 8, 32, dtype=torch.float64, device=DEVICE)
    for j in range(8):
        if j < 4:
            sc, mn = u[..., j] & 63, u[..., j + 4] & 63
        else:
            sc, mn = (u[..., j + 4] & 15) | (u[..., j - 4] >> 6 << 4), (u[..., j + 4] >> 4) | (u[..., j] >> 6 << 4)
        q = v[..., 16 + 32 * (j // 2):48 + 32 * (j // 2)].int()
        q = (q >> 4 if j % 2 else q & 15).double()
        out[:, :, j] = d * sc[..., None] * q - dmin * mn[..., None]
    return out.reshape(rows, k)


def _exact_products(wtype, packed, x, expert):
    x = _exact_activations(wtype, x)
    y = torch.zeros(x.shape[0], packed.shape[1], dtype=torch.float64, device=DEVICE)
    for e in range(packed.shape[0]):
        mine = torch.nonzero(expert == e)[:, 0]
        if mine.numel():
            y[mine] = x[mine] @ _exact_matrix(wtype, packed[e], x.shape[1]).t()
    return y


def _exact_up(s):
    c = s["case"]
    expert = s["ids"].reshape(-1)
    x = s["x"].repeat_interleave(c["used"], 0)
    g, u = (_exact_products(c["wtype"], s[n], x, expert) for n in ("gate", "up"))
    return {"h": (g * torch.sigmoid(g) * u).reshape(c["tokens"], c["used"], -1)}


def _exact_down(s):
    c = s["case"]
    y = _exact_products(c["wtype"], s["down"], s["h"].reshape(-1, c["ffn"]), s["ids"].reshape(-1))
    return {"y": (y.reshape(c["tokens"], c["used"], -1) * s["weights"].double()[:, :, None]).sum(1)}


EXACT = {"conv": _exact_conv, "scan": _exact_scan, "router": _exact_router, "up": _exact_up, "down": _exact_down}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))
