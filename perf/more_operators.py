"""The token mixers of hybrid decoders whose speed is measured, in two forms:
elementary torch operations, and (where `own` is true) the graphs a user of
this backend computes.

Kinds of cases
  delta  the gated delta rule over a cache of states (GATED_DELTA_NET), its
         queries and keys brought to length one (L2_NORM): every sequence's
         outputs and its state after the last token. A head's state S [K, V]
         takes one token by
             S <- e^g S,   S <- S + beta k (v - S^T k)^T,   y = S^T q / sqrt(K)
         with g one number a head or one an element of the keys
  attn   attention whose scores are capped by a tanh, or get a bias that
         depends on distance, under causal, document, prefix and decode masks
         (FLASH_ATTN_EXT with a logit_softcap or a max_bias):
             s = q k * scale,  s <- cap tanh(s / cap),  s <- s + slope(head) mask,
             softmax, and the values' sum

Attention rounds its queries to f16 as ggml defines it for f16 keys. Masks are
f16 tensors, as ggml has them: -inf where a query does not see a position,
else 0 or, for a bias, minus the distance.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6  # of the keys' and queries' lengths


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one decoded token of one stream: the smallest call, bound by its launch
        dict(name="delta-decode-1", kind="delta", gate="head", key=128, value=128, kheads=16, vheads=32, tokens=1, seqs=1),
        # one decoded token of 48 streams: the states are read and written once
        dict(name="delta-decode-b48", kind="delta", gate="head", key=128, value=128, kheads=16, vheads=32, tokens=1,
             seqs=48),
        # a long prompt
        dict(name="delta-prompt-4096", kind="delta", gate="head", key=128, value=128, kheads=16, vheads=32, tokens=4096,
             seqs=1),
        # three prompts of an odd length, smaller heads
        dict(name="delta-prompt-b3-777", kind="delta", gate="head", key=64, value=96, kheads=12, vheads=12, tokens=777,
             seqs=3),
        # a prompt with a gate an element of the keys
        dict(name="delta-element-500", kind="delta", gate="element", key=128, value=128, kheads=16, vheads=16,
             tokens=500, seqs=1),
        # one decoded token of one stream over a short cache
        dict(name="attn-cap-decode-1", kind="attn", dim=128, heads=16, kvheads=8, queries=1, span=1024, seqs=1, cap=30.0,
             bias=0.0, mask="decode"),
        # one decoded token of eight streams of different lengths
        dict(name="attn-cap-decode-b8-4096", kind="attn", dim=128, heads=16, kvheads=8, queries=1, span=4096, seqs=8,
             cap=50.0, bias=0.0, mask="decode"),
        # a decoded token far into its streams, scores biased by distance, five query heads a key head
        dict(name="attn-bias-decode-b4-20000", kind="attn", dim=64, heads=20, kvheads=4, queries=1, span=20000, seqs=4,
             cap=0.0, bias=8.0, mask="decode"),
        # a prompt: capped scores, causal
        dict(name="attn-cap-prompt-2048", kind="attn", dim=128, heads=16, kvheads=8, queries=2048, span=2048, seqs=1,
             cap=50.0, bias=0.0, mask="causal"),
        # two prompts of an odd length, scores biased by distance
        dict(name="attn-bias-prompt-b2-1500", kind="attn", dim=64, heads=16, kvheads=16, queries=1500, span=1500, seqs=2,
             cap=0.0, bias=8.0, mask="causal"),
        # documents packed in a row, each causal in itself, wide heads
        dict(name="attn-docs-1777", kind="attn", dim=256, heads=8, kvheads=4, queries=1777, span=1777, seqs=1, cap=50.0,
             bias=0.0, mask="documents"),
        # a chunk of new tokens behind a cache whose first part all of them see, both bias and cap
        dict(name="attn-prefix-333-of-4096", kind="attn", dim=128, heads=32, kvheads=8, queries=333, span=4096, seqs=1,
             cap=30.0, bias=8.0, mask="prefix"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.45:
        tokens = rng.choice([1, _log(rng, 2, 4096), _log(rng, 2, 4096)])
        seqs = rng.randint(1, max(1, min(48, 4096 // max(tokens, 64))))
        kheads = rng.randint(1, 16)
        if rng.random() < 0.25:
            return dict(kind="delta", gate="element", key=rng.choice([64, 128]), value=16 * rng.randint(2, 8), kheads=kheads,
                        vheads=kheads, tokens=min(tokens, 500), seqs=min(seqs, 4))
        return dict(kind="delta", gate="head", key=rng.choice([64, 96, 128]), value=16 * rng.randint(2, 8), kheads=kheads,
                    vheads=kheads * rng.choice([1, 1, 2]), tokens=tokens, seqs=seqs)
    dim = rng.choice([64, 128, 128, 256])
    kvheads = rng.randint(1, 8)
    heads = kvheads * rng.choice([1, 2, 3, 4, 8])
    cap, bias = rng.choice([(30.0, 0.0), (50.0, 0.0), (0.0, 8.0), (30.0, 8.0)])
    if rng.random() < 0.4:
        span = _log(rng, 1, 20000)
        return dict(kind="attn", dim=dim, heads=heads, kvheads=kvheads, queries=1, span=span,
                    seqs=rng.randint(1, max(1, min(8, 40000 // span))), cap=cap, bias=bias, mask="decode")
    mask = rng.choice(["causal", "documents", "prefix"])
    queries = _log(rng, 2, 1800)
    span = queries if mask != "prefix" else queries + _log(rng, 1, 3000)
    return dict(kind="attn", dim=dim, heads=heads, kvheads=kvheads, queries=queries, span=span,
                seqs=rng.randint(1, max(1, min(4, 1024 // queries))), cap=cap, bias=bias, mask=mask)


# ----------------------------------------------------------------- inputs --

def _rng(seed, stream):
    r = torch.Generator(device=DEVICE)
    r.manual_seed((seed * 1000003 + stream) % (1 << 62))
    return r


def _normal(seed, stream, *shape, std=1.0):
    return torch.randn(*shape, generator=_rng(seed, stream), device=DEVICE) * std


def _uniform(seed, stream, lo, hi, *shape):
    return torch.rand(*shape, generator=_rng(seed, stream), device=DEVICE) * (hi - lo) + lo


def _first_seen(c):
    """(first, last): query i of sequence s sees the positions [first, last] (both [seqs, queries])"""
    i = torch.arange(c["queries"]).expand(c["seqs"], c["queries"])
    if c["mask"] == "causal":
        return torch.zeros_like(i), i
    if c["mask"] == "documents":  # three documents in a row, the middle one the longest
        n = c["queries"]
        cuts = [0, n // 5, n - n // 4]
        first = torch.zeros_like(i)
        for cut in cuts:
            first = torch.where(i >= cut, cut, first)
        return first, i
    if c["mask"] == "prefix":  # the new tokens come after the cache's own
        return torch.zeros_like(i), i + (c["span"] - c["queries"])
    # decode: streams of different lengths in caches of one size
    s = torch.arange(c["seqs"])[:, None]
    return torch.zeros_like(i), (c["span"] - 1 - (s * 977) % max(1, c["span"] // 2)).expand_as(i)


def _mask(c):
    """[seqs, queries, span] f16; one sequence's where all are alike"""
    first, last = _first_seen(c)
    if c["mask"] != "decode":
        first, last = first[:1], last[:1]
    first, last = first.to(DEVICE)[:, :, None], last.to(DEVICE)[:, :, None]
    j = torch.arange(c["span"], device=DEVICE)
    value = -(last - j).clamp_min(0).float() if c["bias"] > 0 else torch.zeros_like(last - j).float()
    return value.masked_fill((j < first) | (j > last), -math.inf).half().contiguous()


def prepare(case, seed):
    c = case
    if c["kind"] == "attn":
        s, d, n = c["seqs"], c["dim"], c["span"]
        # queries and keys that were brought to a like length, as before capped scores
        return dict(case=c, q=_normal(seed, 1, s, c["queries"], c["heads"], d, std=1.5),
                    k=_normal(seed, 2, s, c["kvheads"], n, d).half(), v=_normal(seed, 3, s, c["kvheads"], n, d).half(),
                    mask=_mask(c))
    s, t, hk, hv, dk, dv = (c[k] for k in ("seqs", "tokens", "kheads", "vheads", "key", "value"))
    x = _normal(seed, 1, s, t, 2 * hk * dk + hv * dv)  # a convolution's channels after their SILU: q, k, v
    # the gates' usual range: a token keeps between most and a fifth of the state
    rate = _uniform(seed, 2, 1.0, 16.0, hv, 1) * torch.exp(_uniform(seed, 3, math.log(1e-3), math.log(1e-1), hv, 1))
    per = dk if c["gate"] == "element" else 1
    g = -rate * torch.exp(0.5 * _normal(seed, 4, s, t, hv, per))
    return dict(case=c, x=x / (1 + torch.exp(-x)), g=g.contiguous(), beta=torch.sigmoid(_normal(seed, 5, s, t, hv)),
                states=_normal(seed, 6, s, hv, dv, dk, std=0.3))  # a state's rows: the values, their columns the keys


# ------------------------------------------------------------ plain forms --

def _heads(s):
    """q, k [S, T, Hk, K] and v [S, T, Hv, V] of the channels"""
    c = s["case"]
    n, m = c["kheads"] * c["key"], c["vheads"] * c["value"]
    q, k, v = torch.split(s["x"], [n, n, m], dim=2)
    lead = s["x"].shape[:2]
    return q.reshape(*lead, c["kheads"], c["key"]), k.reshape(*lead, c["kheads"], c["key"]), v.reshape(*lead, c["vheads"], c["value"])


def _unit(x):
    return x / torch.sqrt((x * x).sum(3, keepdim=True)).clamp_min(EPS)


def _plain_delta_step(s):
    """one token: the rule itself"""
    c = s["case"]
    q, k, v = (x[:, 0] for x in _heads(s))
    rep = c["vheads"] // c["kheads"]
    q, k = (_unit(x[:, None])[:, 0].repeat(1, rep, 1)[:, :, None] for x in (q, k))   # [S, H, 1, K]
    h = s["states"] * torch.exp(s["g"][:, 0, :, None])                               # [S, H, V, K]
    d = s["beta"][:, 0, :, None] * (v - (h * k).sum(3))
    h = h + d[..., None] * k
    return {"y": ((h * q).sum(3) / math.sqrt(c["key"]))[:, None], "states": h}


def _plain_delta(s):
    """chunks of tokens as matrix products; a chunk turns the state it meets into M S + N, and the
    chunks' turns are joined by a doubling prefix scan"""
    c = s["case"]
    S, T, H, K, V = (c[k] for k in ("seqs", "tokens", "vheads", "key", "value"))
    q, k, v = _heads(s)
    rep = H // c["kheads"]
    q, k = (_unit(x).repeat(1, 1, rep, 1) for x in (q, k))
    L = min(64 if c["gate"] == "head" else 16, T)
    nc = -(-T // L)
    pad = nc * L - T

    def chunks(x):  # [S, T, H, n] -> [S, H, nc, L, n], what is past T zero: it neither decays nor adds
        x = torch.cat([x, x.new_zeros(S, pad, *x.shape[2:])], 1) if pad else x
        return x.reshape(S, nc, L, H, x.shape[3]).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v, beta, cum = (chunks(x) for x in (q, k, v, s["beta"][..., None], s["g"].double()))
    cum = cum.cumsum(3)                                                              # [S, H, nc, L, 1 | K]
    seen = torch.ones(L, L, dtype=torch.bool, device=DEVICE).tril()
    if c["gate"] == "head":
        between = torch.exp((cum - cum.transpose(3, 4)).masked_fill(~seen, 0.0)).masked_fill(~seen, 0.0)
        kk = torch.matmul(k, k.transpose(3, 4)).double() * between
        qk = (torch.matmul(q, k.transpose(3, 4)) * between).float()
    else:
        rows, cols = torch.exp(cum), torch.exp(-cum)
        kc = (k * cols).transpose(3, 4)
        kk, qk = (torch.matmul(x * rows, kc).masked_fill(~seen, 0.0) for x in (k, q))
        qk = qk.float()
    a = (beta * kk).tril(-1)
    # (1 + a)^-1, a^L being zero: (1 - a) (1 + a^2) (1 + a^4) ...
    inv, power, at = torch.eye(L, dtype=torch.float64, device=DEVICE) - a, torch.matmul(a, a), 2
    while at < L:
        inv, power, at = inv + torch.matmul(inv, power), torch.matmul(power, power), 2 * at
    inv = inv.float()
    grown = torch.exp(cum).float()
    u, w = torch.matmul(inv, beta * v), torch.matmul(inv, beta * grown * k)
    left = (k * torch.exp(cum[..., -1:, :] - cum)).float().transpose(3, 4)            # what of a key is there at the chunk's end
    M = torch.diag_embed(grown[..., -1, :].expand(S, H, nc, K)) - torch.matmul(left, w)
    N = torch.matmul(left, u)
    first = s["states"].transpose(2, 3)                                              # [S, H, K, V]
    N[:, :, 0] += torch.matmul(M[:, :, 0], first)
    at = 1
    while at < nc:
        N = torch.cat([N[:, :, :at], N[:, :, at:] + torch.matmul(M[:, :, at:], N[:, :, :-at])], 2)
        M = torch.cat([M[:, :, :at], torch.matmul(M[:, :, at:], M[:, :, :-at])], 2)
        at *= 2
    entering = torch.cat([first[:, :, None], N[:, :, :-1]], 2)
    y = torch.matmul(grown * q, entering) + torch.matmul(qk, u - torch.matmul(w, entering))
    y = (y / math.sqrt(K)).permute(0, 2, 3, 1, 4).reshape(S, nc * L, H, V)[:, :T].contiguous()
    return {"y": y, "states": N[:, :, -1].transpose(2, 3).contiguous()}


def _slopes(c):
    """one a query head: powers of 2^(-bias / n) for the first n = 2^floor(log2 heads) heads, the odd powers of its root after them"""
    n = 1 << (c["heads"].bit_length() - 1)
    return [2.0 ** (-c["bias"] / n * (h + 1)) if h < n else 2.0 ** (-c["bias"] / 2 / n * (2 * (h - n) + 1))
            for h in range(c["heads"])]


def _plain_attn(s):
    c = s["case"]
    S, H, G, D, Q = c["seqs"], c["heads"], c["kvheads"], c["dim"], c["queries"]
    q = s["q"].half().float().permute(0, 2, 1, 3).reshape(S, G, H // G * Q, D)
    x = torch.matmul(q, s["k"].float().transpose(2, 3)) * (1.0 / math.sqrt(D))
    if c["cap"] > 0:
        x = c["cap"] * torch.tanh(x / c["cap"])
    x = x.reshape(S, H, Q, c["span"])
    mask = s["mask"].float()[:, None]
    x = x + (mask * torch.tensor(_slopes(c), device=DEVICE)[:, None, None] if c["bias"] > 0 else mask)
    top = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))  # a query that sees nothing: zeros
    total = p.sum(3, keepdim=True)
    y = torch.matmul(p.reshape(S, G, H // G * Q, c["span"]), s["v"].float()).reshape(S, H, Q, D)
    return {"y": torch.where(total > 0, y / total, 0.0).permute(0, 2, 1, 3).contiguous()}


# ------------------------------------------------------- the backend's form --

class _Memory:
    """device memory for torch; a tensor made of it keeps its owner, and so the memory, alive"""

    def __init__(self, owner, ptr, shape):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr="<f4", data=(ptr, False), version=3, strides=None)


class _Program:
    """one ggml graph over a state's tensors, and torch views of its results"""

    def __init__(self, n_tensors=64):
        from openasr_amd import ggml as g
        self.g = g
        self.G = g.Graph(n_tensors=n_tensors, graph_size=n_tensors)
        self.lib, self.ctx = self.G.lib, self.G.ctx
        self.backend = g.plugin().backend

    def over(self, t, *ne):
        """a graph tensor whose bytes are those of the torch tensor t"""
        return self.G.over({torch.float32: self.g.F32, torch.float16: self.g.F16}[t.dtype], *ne, memory=t)

    def done(self, **outputs):
        """the graph allocated for these results: name -> (tensor, shape, offset in bytes)"""
        self.G.build(*dict.fromkeys(t for t, _, _ in outputs.values()))
        self.G.allocate(self.g.plugin().buft)
        torch.cuda.current_stream().synchronize()  # the state's tensors are written before the first compute reads them
        self.views = {name: torch.as_tensor(_Memory(self.G, self.g.tensor(t).data + at, shape), device=DEVICE)
                      for name, (t, shape, at) in outputs.items()}
        return self

    def __call__(self):
        if self.G.compute(self.backend) != 0:
            raise RuntimeError("graph compute failed")
        return dict(self.views)


def _own_delta(s):
    c = s["case"]
    S, T, Hk, H, K, V = (c[k] for k in ("seqs", "tokens", "kheads", "vheads", "key", "value"))
    C = 2 * Hk * K + H * V
    p = _Program()
    L, ctx = p.lib, p.ctx
    x = p.over(s["x"], C, T, S)
    q, k, v = (L.ggml_view_4d(ctx, x, n, h, T, S, 4 * n, 4 * C, 4 * C * T, 4 * at)
               for n, h, at in ((K, Hk, 0), (K, Hk, Hk * K), (V, H, 2 * Hk * K)))
    y = L.ggml_gated_delta_net(ctx, L.ggml_l2_norm(ctx, q, EPS), L.ggml_l2_norm(ctx, k, EPS), v,
                               p.over(s["g"], s["g"].shape[3], H, T, S), p.over(s["beta"], 1, H, T, S),
                               p.over(s["states"], K, V, H, S))
    return p.done(y=(y, [S, T, H, V], 0), states=(y, [S, H, V, K], 4 * S * T * H * V))


def _own_attn(s):
    c = s["case"]
    S, H, G, D, Q, N = (c[k] for k in ("seqs", "heads", "kvheads", "dim", "queries", "span"))
    p = _Program()
    q = p.lib.ggml_permute(p.ctx, p.over(s["q"], D, H, Q, S), 0, 2, 1, 3)
    y = p.lib.ggml_flash_attn_ext(p.ctx, q, p.over(s["k"], D, N, G, S), p.over(s["v"], D, N, G, S),
                                  p.over(s["mask"], N, Q, 1, s["mask"].shape[0]), 1.0 / math.sqrt(D), c["bias"], c["cap"])
    return p.done(y=(y, [S, Q, H, D], 0))


def run(state):
    attn = state["case"]["kind"] == "attn"
    if own:
        if "program" not in state:
            state["program"] = (_own_attn if attn else _own_delta)(state)
        return state["program"]()
    if not attn and state["case"]["tokens"] == 1:
        return _plain_delta_step(state)
    return (_plain_attn if attn else _plain_delta)(state)


# ------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "delta":
        s, t, hk, hv, dk, dv = (c[k] for k in ("seqs", "tokens", "kheads", "vheads", "key", "value"))
        gates = hv * (dk if c["gate"] == "element" else 1)
        # a token's step decays the state, takes k from it, adds to it and takes q from it
        return {"bytes": 4.0 * (s * t * (2 * hk * dk + 2 * hv * dv + gates + hv) + 2 * s * hv * dk * dv),
                "flops": 7.0 * s * t * hv * dk * dv}
    first, last = _first_seen(c)
    pairs = float((last - first + 1).sum())  # of a query head
    keys = float((last.amax(1) + 1).sum())   # positions that some query sees
    masks = c["queries"] * (keys if c["mask"] == "decode" else c["span"])
    moved = 8.0 * c["seqs"] * c["queries"] * c["heads"] * c["dim"] + 4.0 * keys * c["kvheads"] * c["dim"] + 2.0 * masks
    return {"bytes": moved, "flops": 4.0 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------ exact --

def _exact_delta(s):
    """token by token"""
    c = s["case"]
    K, n, m = c["key"], c["kheads"] * c["key"], c["vheads"] * c["value"]
    x = s["x"].double()
    keys = [x[..., at:at + n].unflatten(2, (c["kheads"], K)) for at in (0, n)]
    q, k = (v / v.norm(dim=3, keepdim=True).clamp_min(EPS) for v in keys)
    of = torch.arange(c["vheads"], device=DEVICE) % c["kheads"]  # the key head of each
    q, k, v = q[:, :, of] / K ** 0.5, k[:, :, of], x[..., 2 * n:2 * n + m].unflatten(2, (c["vheads"], c["value"]))
    h, g, beta = s["states"].double(), s["g"].double().exp(), s["beta"].double()
    y = torch.empty(c["seqs"], c["tokens"], c["vheads"], c["value"], dtype=torch.float64, device=DEVICE)
    for t in range(c["tokens"]):
        h = h * g[:, t, :, None]
        off = v[:, t] - (h * k[:, t, :, None]).sum(3)
        h = h + (beta[:, t, :, None] * off)[..., None] * k[:, t, :, None]
        y[:, t] = (h * q[:, t, :, None]).sum(3)
    return {"y": y, "states": h}


def _exact_attn(s):
    """head by head"""
    c = s["case"]
    y = torch.zeros(c["seqs"], c["queries"], c["heads"], c["dim"], dtype=torch.float64, device=DEVICE)
    mask = s["mask"].double().expand(c["seqs"], -1, -1)
    n = 2 ** math.floor(math.log2(c["heads"]))
    for h in range(c["heads"]):
        kv = h // (c["heads"] // c["kvheads"])
        z = s["q"][:, :, h].half().double() @ s["k"][:, kv].double().mT / math.sqrt(c["dim"])
        if c["cap"]:
            z = torch.tanh(z / c["cap"]) * c["cap"]
        if c["bias"]:
            z = z + mask * (2 ** (-c["bias"] * (h + 1) / n) if h < n else 2 ** (-c["bias"] * (h - n + 0.5) / n))
        else:
            z = z + mask
        y[:, :, h] = torch.softmax(z, 2).nan_to_num(0.0) @ s["v"][:, kv].double()
    return {"y": y}


def exact(case, seed):
    return (_exact_attn if case["kind"] == "attn" else _exact_delta)(prepare(case, seed))
