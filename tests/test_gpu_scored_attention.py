"""FLASH_ATTN_EXT with capped or biased scores, masks a head, heads of 256 and
any group size, on the device against its definition in float64.

Bounds count roundings: u = 2^-24 is half a step of f32.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def slopes(heads, bias):
    if bias == 0:
        return np.ones(heads)
    n = 1 << (heads.bit_length() - 1)
    return np.array([2.0 ** (-bias / n * (h + 1)) if h < n else 2.0 ** (-bias / 2 / n * (2 * (h - n) + 1)) for h in range(heads)])


def attention64(q, k, v, mask, scale, cap, bias):
    """q [S, H, Q, D] f32 (rounded to f16 here), k, v [S | 1.., G, N, D] f16, mask [1 | S, 1 | H, Q, N] f16 or
    None -> out [S, Q, H, D] and how far f32 arithmetic may take it off"""
    S, H, Q, D = q.shape
    q = q.astype(np.float16).astype(np.float64)
    k, v = (np.repeat(np.repeat(x, S // x.shape[0], 0), H // x.shape[1], 1).astype(np.float64) for x in (k, v))
    N = k.shape[2]
    mk = np.zeros((1, 1, Q, N)) if mask is None else np.tile(mask.astype(np.float64), (1, H // mask.shape[1], 1, 1))
    mk = mk + np.zeros((S, H, 1, 1))
    seen = mk != -np.inf
    k_seen = np.where(seen.any(2)[..., None], k, 0.0)  # what no query sees may hold anything
    with np.errstate(invalid="ignore"):
        s = (q @ k_seen.transpose(0, 1, 3, 2)) * scale
        size = (np.abs(q) @ np.abs(k_seen).transpose(0, 1, 3, 2)) * abs(scale)
    b = np.where(seen, mk, 0.0) * slopes(H, bias)[:, None, None]
    z = cap * np.tanh(s / cap) if cap else s
    t = np.where(seen, z + b, -np.inf)
    top = t.max(3, keepdims=True)
    top = np.where(np.isfinite(top), top, 0.0)
    p = np.where(seen, np.exp(t - top), 0.0)
    total = p.sum(3, keepdims=True)
    w = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
    # a score's own: the product's sum (D roundings of its terms' size), the scale, the cap (its
    # polynomial or its quotient: ten roundings of the result and of the cap), the slope and the
    # bias, the sum, the maximum subtracted, all in the exponent's base
    tiles = N // 64 + 2
    E = (D + 4) * U * size + 10 * U * (np.abs(z) + cap) + 4 * U * np.abs(b) + 4 * U * (np.abs(z) + np.abs(b) + np.abs(top) + 20) + 8 * U
    E = np.where(seen, E, 0.0) + (N + 4 * tiles) * U  # the sums over positions and the tiles' factors
    vv = [np.where(seen[:, :, i, :, None], v, 0.0) for i in range(Q)]
    out, err = np.zeros((S, H, Q, D)), np.zeros((S, H, Q, D))
    for i in range(Q):
        out[:, :, i] = (w[:, :, i, None] @ vv[i])[:, :, 0]
        err[:, :, i] = ((w * E)[:, :, i, None] @ np.abs(vv[i]))[:, :, 0] + np.abs(out[:, :, i]) * (w * E).sum(3)[:, :, i, None]
        # p's low half has a smallest step, 2^-25 of numbers scaled by 2^12
        err[:, :, i] += N * 2.0 ** -36 * np.abs(vv[i]).max(2) + 4 * U * np.abs(out[:, :, i])
    return out.transpose(0, 2, 1, 3), 2 * err.transpose(0, 2, 1, 3) + 1e-37


def make_mask(kind, S, H, Q, N, bias, rng):
    i, j = np.arange(Q)[:, None] + (N - Q), np.arange(N)[None]
    dist = -np.abs(i - j).astype(np.float64) if bias else np.zeros((Q, N))
    m = np.where(j <= i, dist, -np.inf)
    if kind == "none":
        return None
    if kind == "causal":
        m = m[None, None]
    elif kind == "documents":
        cut = np.sort(rng.choice(np.arange(1, N), min(3, N - 1), replace=False)) if N > 1 else np.array([], int)
        doc = np.searchsorted(cut, np.arange(N), side="right")
        m = np.where(doc[None] == doc[np.minimum(i, N - 1)[:, 0]][:, None], m, -np.inf)[None, None]
    elif kind == "prefix":  # all see the first part, the rest is causal
        m = np.where(j < N // 3, dist, m)[None, None]
    elif kind == "window":  # the first 100 positions and the last 200, beside the causal mask
        m = np.where((j < 100) | (j > i - 200), m, -np.inf)[None, None]
    elif kind == "empty":  # rows that see nothing, in one sequence a whole block of them
        m = np.repeat(m[None, None], S, 0)
        m[:, :, rng.random(Q) < 0.3] = -np.inf
        m[0, :, : (Q + 1) // 2] = -np.inf
    elif kind == "lowest":  # masked by f16's lowest value, and in one row everything
        m = np.where(np.isinf(m), -65504.0, m)[None, None]
        m[:, :, -1] = -65504.0
    elif kind == "heads":
        m = np.repeat(np.repeat(m[None, None], S, 0), H, 1)
        m[rng.random(m.shape) < 0.5] = -np.inf
        m[..., 0] = 0
    elif kind == "some heads":  # two masks, in turn over the heads
        m = np.repeat(m[None, None], 2, 1)
        m[:, 1] = np.where(rng.random((Q, N)) < 0.7, dist, -np.inf)
    elif kind == "random":
        m = np.where(rng.random((S, 1, Q, N)) < 0.4, rng.standard_normal((S, 1, Q, N)) * 3, -np.inf)
    elif kind == "lengths":
        m = np.repeat(dist[None, None], S, 0)
        for s in range(S):
            m[s, :, :, max(1, N - 1 - (s * 37) % N):] = -np.inf
    return m.astype(np.float16)


def attention(ggml, gpu, q, k, v, mask, scale, cap, bias, prec=None, kv32=False, times=3):
    S, H, Q, D = q.shape
    G = ggml.Graph(64, 64)
    X = G.new(ggml.F32, D, H, Q, S)  # token by token, as a projection leaves them
    t = ggml.F32 if kv32 else ggml.F16
    K, V = (G.new(t, D, x.shape[2], x.shape[1], x.shape[0]) for x in (k, v))
    M = G.new(ggml.F16, mask.shape[3], mask.shape[2], mask.shape[1], mask.shape[0]) if mask is not None else None
    y = G.lib.ggml_flash_attn_ext(G.ctx, G.lib.ggml_permute(G.ctx, X, 0, 2, 1, 3), K, V, M, scale, bias, cap)
    assert y
    if prec is not None:
        G.lib.ggml_flash_attn_ext_set_prec(y, prec)
    G.build(y)
    G.allocate(gpu.buft)
    G.set(X, q.transpose(0, 2, 1, 3))
    for T, x in ((K, k), (V, v)):
        G.set(T, x.astype(np.float32) if kv32 else x.view(np.uint16))
    if M:
        G.set(M, mask.view(np.uint16))
    outs = []
    for _ in range(times):
        assert G.compute(gpu.backend) == 0
        outs.append(G.get(y).reshape(S, Q, H, D))
    G.free()
    for o in outs[1:]:
        assert np.array_equal(o, outs[0], equal_nan=True)
    return outs[0]


def check(got, want, bound, what=""):
    assert np.isfinite(got).all(), what
    off = np.abs(got.astype(np.float64) - want) - bound
    assert (off <= 0).all(), f"{what}: off by {np.abs(got - want).flat[np.argmax(off)]:.3g}, allowed {bound.flat[np.argmax(off)]:.3g}"


def operands(rng, S, H, G, Q, N, D, std=1.0, kv_seqs=None):
    q = (std * rng.standard_normal((S, H, Q, D))).astype(np.float32)
    k, v = (rng.standard_normal((kv_seqs or S, G, N, D)).astype(np.float16) for _ in range(2))
    return q, k, v


#        D    H   G  Q    N    S  mask        cap   bias
CASES = [(128, 4, 2, 1, 1, 1, "causal", 30.0, 0.0),
         (128, 4, 2, 1, 300, 3, "lengths", 50.0, 0.0),
         (64, 20, 4, 1, 1000, 2, "lengths", 0.0, 8.0),
         (256, 3, 1, 1, 130, 1, "lengths", 30.0, 8.0),
         (128, 12, 1, 1, 65, 1, "causal", 0.0, 8.0),
         (64, 2, 2, 2, 2, 1, "causal", 50.0, 0.0),
         (128, 4, 2, 65, 65, 1, "causal", 50.0, 0.0),
         (64, 6, 2, 130, 131, 2, "causal", 0.0, 8.0),
         (256, 4, 2, 70, 200, 1, "causal", 30.0, 8.0),
         (128, 6, 2, 77, 77, 1, "documents", 50.0, 0.0),
         (64, 5, 1, 200, 200, 1, "documents", 0.0, 4.0),
         (128, 16, 2, 33, 400, 1, "prefix", 30.0, 8.0),
         (64, 4, 4, 40, 100, 2, "empty", 30.0, 0.0),
         (128, 4, 1, 20, 129, 2, "empty", 0.0, 8.0),
         (64, 2, 1, 20, 90, 1, "lowest", 30.0, 0.0),
         (64, 4, 2, 30, 100, 2, "heads", 30.0, 8.0),
         (128, 6, 3, 1, 200, 2, "heads", 0.0, 0.0),
         (64, 4, 2, 70, 72, 1, "some heads", 0.0, 0.0),
         (128, 4, 2, 50, 257, 2, "random", 0.0, 8.0),
         (64, 8, 1, 9, 500, 2, "random", 50.0, 0.0),
         (64, 2, 1, 70, 100, 1, "none", 30.0, 0.0),
         (256, 2, 2, 5, 64, 1, "none", 0.0, 0.0),
         (128, 3, 1, 1, 700, 1, "none", 30.0, 0.0),
         (128, 40, 2, 7, 333, 1, "causal", 50.0, 0.0),
         (64, 64, 1, 3, 70, 1, "causal", 50.0, 0.0),
         (128, 2, 1, 300, 1500, 1, "causal", 30.0, 0.0)]


@pytest.mark.parametrize("D,H,G,Q,N,S,kind,cap,bias", CASES)
def test_scored_attention(ggml, gpu, D, H, G, Q, N, S, kind, cap, bias):
    print(f"scored attention D={D} H={H} G={G} Q={Q} N={N} S={S} {kind} cap={cap} bias={bias}", flush=True)
    rng = np.random.default_rng(D + H + Q + N)
    q, k, v = operands(rng, S, H, G, Q, N, D, std=2.0)
    mask = make_mask(kind, S, H, Q, N, bias, rng)
    scale = 1 / np.sqrt(D)
    want, bound = attention64(q, k, v, mask, scale, cap, bias)
    for prec in (None, ggml.GGML_PREC_F32):
        check(attention(ggml, gpu, q, k, v, mask, scale, cap, bias, prec), want, bound, f"prec {prec}")


#        D    H   G  Q    N     S  mask        cap   bias
LONG = [(128, 8, 8, 100, 5000, 1, "window", 30.0, 0.0),  # tiles seen lie more than 64 apart
        (64, 16, 8, 40, 9001, 1, "window", 0.0, 8.0),
        (128, 16, 8, 300, 1200, 1, "causal", 50.0, 0.0),  # several blocks of 256 rows, in pieces
        (64, 8, 8, 700, 700, 2, "causal", 0.0, 8.0),
        (256, 8, 2, 200, 1000, 1, "prefix", 50.0, 0.0),
        (128, 3, 3, 500, 2000, 1, "none", 50.0, 0.0),
        (128, 64, 1, 5, 3000, 2, "random", 30.0, 8.0),
        (64, 8, 8, 300, 300, 3, "empty", 50.0, 0.0),
        (256, 8, 8, 130, 700, 2, "heads", 30.0, 8.0)]


@pytest.mark.parametrize("D,H,G,Q,N,S,kind,cap,bias", LONG)
def test_long_spans(ggml, gpu, D, H, G, Q, N, S, kind, cap, bias):
    print(f"long span D={D} H={H} G={G} Q={Q} N={N} S={S} {kind} cap={cap} bias={bias}", flush=True)
    rng = np.random.default_rng(D + H + Q + N)
    q, k, v = operands(rng, S, H, G, Q, N, D, std=2.0)
    mask = make_mask(kind, S, H, Q, N, bias, rng)
    want, bound = attention64(q, k, v, mask, 1 / np.sqrt(D), cap, bias)
    check(attention(ggml, gpu, q, k, v, mask, 1 / np.sqrt(D), cap, bias), want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [0.0, 200.0])
def test_maxima_that_grow(ggml, gpu, D, cap):
    """each tile's scores lie far over the last one's, in half of the rows far under them"""
    rng = np.random.default_rng(D)
    Q, N, H = 150, 700, 2
    q, k, v = operands(rng, 1, H, 1, Q, N, D)
    q[..., 0] = np.where(np.arange(Q) % 2, -1.0, 1.0)[None, None]
    k[..., 0] = (np.arange(N) / 4).astype(np.float16)
    mask = make_mask("causal", 1, H, Q, N, 0.0, rng)
    want, bound = attention64(q, k, v, mask, 1.0, cap, 0.0)
    check(attention(ggml, gpu, q, k, v, mask, 1.0, cap, 0.0), want, bound)


@pytest.mark.parametrize("D,Q", [(64, 300), (128, 300), (256, 150)])
def test_values_not_finite_in_later_tiles(ggml, gpu, D, Q):
    """an infinite value reaches the rows that see it, in its dims, and no others"""
    rng = np.random.default_rng(D + Q)
    N, H = Q, 2
    q, k, v = operands(rng, 1, H, 2, Q, N, D)
    clean = v.copy()
    spots = [(0, 70, 3, np.inf), (1, 130, D - 1, -np.inf), (0, 140, 17, np.nan), (0, N - 1, 40, np.inf)]
    for g, n, d, x in spots:
        v[0, g, n, d] = x
        clean[0, g, n, d] = 0
    mask = make_mask("causal", 1, H, Q, N, 0.0, rng)
    got = attention(ggml, gpu, q, k, v, mask, 0.1, 30.0, 0.0)
    hit = np.zeros(got.shape, bool)
    for g, n, d, x in spots:
        hit[0, n:, g, d] = True
        sign = got[0, n:, g, d]
        assert np.isnan(sign).all() if np.isnan(x) else (sign == x).all(), (g, n, d)
    want, bound = attention64(q, k, clean, mask, 0.1, 30.0, 0.0)
    check(np.where(hit, 0, got), np.where(hit, 0, want), bound)


@pytest.mark.parametrize("Q,N", [(1, 200), (40, 200)])
@pytest.mark.parametrize("std", [3.0, 20.0, 300.0])
def test_scores_past_the_cap(ggml, gpu, Q, N, std):
    """scores about the cap and far past it: the tanh's other branch"""
    rng = np.random.default_rng(3)
    q, k, v = operands(rng, 1, 4, 2, Q, N, 64, std=std)
    mask = make_mask("causal", 1, 4, Q, N, 0, rng)
    want, bound = attention64(q, k, v, mask, 0.125, 5.0, 0.0)
    check(attention(ggml, gpu, q, k, v, mask, 0.125, 5.0, 0.0), want, bound)


@pytest.mark.parametrize("D,Q,N", [(64, 1, 150), (128, 30, 200), (64, 100, 130), (256, 9, 80)])
@pytest.mark.parametrize("bias", [0.0, 8.0])
def test_masked_places_hold_anything(ggml, gpu, D, Q, N, bias):
    """NaN and infinities in K and V where the mask hides them, for all queries and for some"""
    rng = np.random.default_rng(D + Q)
    q, k, v = operands(rng, 2, 4, 2, Q, N, D)
    mask = np.repeat(make_mask("causal", 2, 4, Q, N, bias, rng), 2, 0)
    hidden = rng.random(N) < 0.2          # nobody sees these
    hidden[0] = False
    mask[..., hidden] = -np.inf
    some = ~hidden & (np.arange(N) > N // 2) & (rng.random(N) < 0.2)  # the last query alone does not
    mask[:, :, -1, some] = -np.inf
    want, bound = attention64(q, k, v, mask, 0.1, 30.0, bias)
    k2, v2 = k.copy(), v.copy()
    for x in (k2, v2):
        x[:, :, hidden] = np.array([np.nan, np.inf, -np.inf, 3.0], np.float16)[rng.integers(0, 4, (2, 2, hidden.sum(), D))]
    v3 = v2.copy()
    v3[:, :, some, 5] = np.inf            # reaches its dim, and only of the queries that see it
    check(attention(ggml, gpu, q, k2, v2, mask, 0.1, 30.0, bias), want, bound)
    got = attention(ggml, gpu, q, k2, v3, mask, 0.1, 30.0, bias)
    sees = (mask[..., some] != -np.inf).any(3)[0, 0] if some.any() else np.zeros(Q, bool)
    rest = np.ones(got.shape, bool)
    rest[:, sees, :, 5] = False
    assert not np.isfinite(got[:, sees, :, 5]).any()
    check(np.where(rest, got, 0), np.where(rest, want, 0), bound)


@pytest.mark.parametrize("Q", [1, 20])
def test_layouts(ggml, gpu, Q):
    """f32 K and V, K and V shared by sequences, one mask for all of them, a mask of more rows and odd strides"""
    rng = np.random.default_rng(5)
    q, k, v = operands(rng, 4, 6, 2, Q, 101, 64, kv_seqs=2)
    mask = make_mask("causal", 4, 6, Q, 101, 8.0, rng)
    want, bound = attention64(q, k, v, mask, 0.125, 30.0, 8.0)
    check(attention(ggml, gpu, q, k, v, mask, 0.125, 30.0, 8.0), want, bound, "f16")
    check(attention(ggml, gpu, q, k, v, mask, 0.125, 30.0, 8.0, kv32=True), want, bound, "f32")
    more = np.concatenate([mask, np.full((1, 1, 3, 101), np.nan, np.float16)], 2)
    check(attention(ggml, gpu, q, k, v, more, 0.125, 30.0, 8.0), want, bound, "more rows")


def test_part_of_a_cache(ggml, gpu):
    """the first positions of a cache whose other rows are written later"""
    rng = np.random.default_rng(6)
    D, H, G, Q, N, S, rows = 128, 4, 2, 9, 70, 2, 256
    q, k, v = operands(rng, S, H, G, Q, rows, D)
    mask = make_mask("causal", S, H, Q, N, 0, rng)
    want, bound = attention64(q, k[:, :, :N], v[:, :, :N], mask, 0.1, 20.0, 0.0)
    g = ggml.Graph(64, 64)
    X, K, V = g.new(ggml.F32, D, Q, H, S), g.new(ggml.F16, D, rows, G, S), g.new(ggml.F16, D, rows, G, S)
    M = g.new(ggml.F16, N, Q, 1, 1)
    kv = [g.lib.ggml_view_4d(g.ctx, t, D, N, G, S, 2 * D, 2 * D * rows, 2 * D * rows * G, 0) for t in (K, V)]
    y = g.lib.ggml_flash_attn_ext(g.ctx, X, *kv, M, 0.1, 0.0, 20.0)
    g.build(y)
    g.allocate(gpu.buft)
    for t, a in ((X, q), (K, k.view(np.uint16)), (V, v.view(np.uint16)), (M, mask.view(np.uint16))):
        g.set(t, a)
    for _ in range(3):
        assert g.compute(gpu.backend) == 0
        check(g.get(y).reshape(S, Q, H, D), want, bound)
    g.free()


def test_supports(ggml, gpu):
    """what the device refuses, and says so"""
    G = ggml.Graph(64, 64)

    def ok(D=64, H=4, Gh=2, mask=(9, 5, 1, 1), kv=None, bias=8.0, cap=30.0):
        q = G.new(ggml.F32, D, 5, H, 1)
        k = kv or G.new(ggml.F16, D, 9, Gh, 1)
        m = G.new(ggml.F16, *mask) if mask else None
        return gpu_supports(G.lib.ggml_flash_attn_ext(G.ctx, q, k, k, m, 0.1, bias, cap))

    def gpu_supports(t):
        return G.lib.ggml_backend_supports_op(gpu.backend, t)

    assert ok() and ok(D=256) and ok(H=10, Gh=2) and ok(mask=(9, 5, 4, 1)) and ok(mask=(9, 5, 2, 1))
    assert ok(mask=None, bias=0.0)
    assert not ok(D=96) and not ok(H=130, Gh=2)
    wide = G.new(ggml.F16, 68, 9, 2, 1)  # rows of 136 bytes
    assert not ok(kv=G.lib.ggml_view_4d(G.ctx, wide, 64, 9, 2, 1, 136, 136 * 9, 136 * 18, 0))
    G.free()


@pytest.mark.parametrize("Q", [1, 20])
@pytest.mark.parametrize("D,N", [(64, 65), (128, 130), (256, 40), (64, 9000)])
@pytest.mark.parametrize("kind", ["lengths", "heads"])
@pytest.mark.parametrize("where", ["query", "first", "last", "middle"])
def test_nan_that_is_seen(ggml, gpu, Q, D, N, kind, where):
    """a NaN in a query, or in a key that a query sees, is that row's result, wherever the key lies"""
    rng = np.random.default_rng(D + N + Q)
    S, H, G = 2, 4, 2
    q, k, v = operands(rng, S, H, G, Q, N, D)
    mask = np.zeros((S, H if kind == "heads" else 1, Q, N), np.float16)
    if kind == "heads":
        mask[:, 1, :, ::3] = -np.inf
    want, bound = attention64(q, k, v, mask, 0.1, 30.0, 0.0)
    hit = np.zeros((S, Q, H), bool)
    if where == "query":
        q[1, 2, Q // 2, 7] = np.nan
        hit[1, Q // 2, 2] = True
    else:
        n = {"first": 0, "last": N - 1, "middle": N // 2}[where]
        k[1, 0, n, 3] = np.nan  # of query heads 0 and 1
        hit[1] = np.isfinite(np.broadcast_to(mask, (S, H, Q, N))[1, :, :, n]).T & (np.arange(H) < H // G)
    got = attention(ggml, gpu, q, k, v, mask, 0.1, 30.0, 0.0)
    assert np.isnan(got[hit]).all()
    check(got[~hit], want[~hit], bound[~hit])


@pytest.mark.parametrize("D,Q,N,lead,cap,bias", [(256, 30, 150, 64, 0.0, 0.0)] +
                         [(*x, *y) for x in [(64, 20, 200, 64), (128, 70, 300, 130), (256, 30, 150, 64), (64, 300, 2000, 700), (128, 1, 300, 200)]
                          for y in [(30.0, 0.0), (0.0, 8.0), (30.0, 8.0)]])
@pytest.mark.parametrize("low", [-65504.0, -3000.0])
def test_tiles_of_low_scores_first(ggml, gpu, D, Q, N, lead, cap, bias, low):
    """a padded front masked by a large finite number: what follows keeps its own precision"""
    rng = np.random.default_rng(D + Q)
    q, k, v = operands(rng, 2, 4, 2, Q, N, D)
    mask = np.repeat(make_mask("causal", 2, 4, Q, N, bias, rng), 2, 0)
    mask[0, :, :, :lead] = low
    mask[1, :, :, :lead - 30] = low
    mask[1, :, 0, :] = low  # a row of nothing else
    want, bound = attention64(q, k, v, mask, 0.1, cap, bias)
    check(attention(ggml, gpu, q, k, v, mask, 0.1, cap, bias), want, bound)


@pytest.mark.parametrize("Q,S,kv_seqs", [(0, 2, 2), (0, 2, 1), (1, 0, 1), (5, 0, 1)])
def test_no_queries(ggml, gpu, Q, S, kv_seqs):
    """a batch that has run empty: nothing is launched, and no size of it divides anything"""
    G = ggml.Graph(16, 16)
    q, k, m = G.new(ggml.F32, 64, Q, 4, S), G.new(ggml.F16, 64, 9, 2, kv_seqs), G.new(ggml.F16, 9, max(Q, 1), 1, 1)
    y = G.lib.ggml_flash_attn_ext(G.ctx, q, k, k, m, 0.1, 0.0, 30.0)
    assert G.lib.ggml_backend_supports_op(gpu.backend, y)
    G.build(y)
    G.allocate(gpu.buft)
    assert G.compute(gpu.backend) == 0 and G.get(y).size == 0
    G.free()


@pytest.mark.parametrize("Q,N", [(1, 100), (40, 200)])
@pytest.mark.parametrize("scale,cap", [(0.1, 1e-30), (0.1, 1e-9), (1e7, 50.0), (1e-20, 1e-9), (0.1, 1e30), (1e-30, 1e-10), (0.0, 30.0), (-0.1, 30.0)])
def test_caps_and_scales_at_their_ends(ggml, gpu, Q, N, scale, cap):
    """caps far under and over the scores, scales far from one, rows of queries that are zero"""
    rng = np.random.default_rng(Q)
    q, k, v = operands(rng, 1, 4, 2, Q, N, 64)
    q[:, 1:3] = 0
    mask = make_mask("causal", 1, 4, Q, N, 0, rng)
    want, bound = attention64(q, k, v, mask, scale, cap, 0.0)
    # (the cap's roundings are relative to a score while that is far under the cap)
    if cap == 1e30:
        want, bound = attention64(q, k, v, mask, scale, 0.0, 0.0)
        bound = 2 * bound
    check(attention(ggml, gpu, q, k, v, mask, scale, cap, 0.0), want, bound)


def test_caps_refused(ggml, gpu):
    G = ggml.Graph(16, 16)
    q, k = G.new(ggml.F32, 64, 5, 4, 1), G.new(ggml.F16, 64, 9, 2, 1)
    for scale, cap, ok in ((0.1, 1e-30, True), (1e5, 1e-30, False), (0.1, 1e30, True), (float("inf"), 30.0, False)):
        y = G.lib.ggml_flash_attn_ext(G.ctx, q, k, k, None, scale, 0.0, cap)
        assert G.lib.ggml_backend_supports_op(gpu.backend, y) == ok
    G.free()


def expanded(ggml, G, x, heads):
    """a cache's kv heads [D, N, heads] repeated to the query heads"""
    L, (D, N, g) = G.lib, (int(n) for n in ggml.tensor(x).ne[:3])
    x = L.ggml_repeat_4d(G.ctx, L.ggml_reshape_4d(G.ctx, x, D, N, 1, g), D, N, heads // g, g)
    return L.ggml_reshape_3d(G.ctx, x, D, N, heads)


@pytest.mark.parametrize("D,H,G", [(64, 6, 2), (128, 7, 1), (64, 32, 2), (128, 24, 2), (64, 128, 1), (256, 4, 2)])
@pytest.mark.parametrize("Q", [1, 30])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_expanded_heads_of_any_group(ggml, gpu, D, H, G, Q, cap):
    """K and V repeated to the query heads: groups that only this form has, and one that none has"""
    if H // G > 64 and cap == 0.0:
        cap = 50.0  # (read as they are repeated, so in a form of one head a group)
    rng = np.random.default_rng(H)
    N = 150
    q, k, v = operands(rng, 1, H, G, Q, N, D)
    mask = make_mask("causal", 1, H, Q, N, 0, rng)
    want, bound = attention64(q, k, v, mask, 0.1, cap, 0.0)
    g = ggml.Graph(64, 64)
    X, K, V, M = g.new(ggml.F32, D, Q, H, 1), g.new(ggml.F16, D, N, G), g.new(ggml.F16, D, N, G), g.new(ggml.F16, N, Q, 1, 1)
    y = g.lib.ggml_flash_attn_ext(g.ctx, X, expanded(ggml, g, K, H), expanded(ggml, g, V, H), M, 0.1, 0.0, cap)
    g.build(y)
    g.allocate(gpu.buft)
    for t, a in ((X, q), (K, k.view(np.uint16)), (V, v.view(np.uint16)), (M, mask.view(np.uint16))):
        g.set(t, a)
    for _ in range(3):
        assert g.compute(gpu.backend) == 0
        check(g.get(y).reshape(1, Q, H, D), want, bound)
    names = [x.split(":", 1)[0] for x, _ in gpu.profile(g.gf, 1)]
    assert "flash_attn_scored" in names and ("repeat" in names) == (H // G > 64)
    g.free()


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_output_over_the_source_of_repeated_heads(ggml, gpu, cap):
    """an allocator may give the attention's output the memory of K before it was repeated: it is not read then"""
    rng = np.random.default_rng(8)
    D, H, G, Q, N = 64, 8, 2, 32, 512
    q, k, v = operands(rng, 1, H, G, Q, N, D)
    want, bound = attention64(q, k, v, None, 0.1, cap, 0.0)
    g = ggml.Graph(64, 64)
    X, K, V = g.new(ggml.F32, D, Q, H, 1), g.new(ggml.F16, D, G, N), g.new(ggml.F16, D, G, N)
    kc, vc = (g.lib.ggml_cont(g.ctx, g.lib.ggml_permute(g.ctx, t, 0, 2, 1, 3)) for t in (K, V))
    y = g.lib.ggml_flash_attn_ext(g.ctx, X, expanded(ggml, g, kc, H), expanded(ggml, g, vc, H), None, 0.1, 0.0, cap)
    g.lib.ggml_flash_attn_ext_set_prec(y, ggml.GGML_PREC_F32)
    g.build(y)
    g.allocate(gpu.buft)
    at = [(ggml.tensor(t).data, g.lib.ggml_nbytes(t)) for t in (kc, vc, y)]
    assert any(a < at[2][0] + at[2][1] and at[2][0] < a + n for a, n in at[:2])
    for t, a in ((X, q), (K, k[0].transpose(1, 0, 2).view(np.uint16)), (V, v[0].transpose(1, 0, 2).view(np.uint16))):
        g.set(t, a)
    for _ in range(3):
        assert g.compute(gpu.backend) == 0
        check(g.get(y).reshape(1, Q, H, D), want, bound)
    assert "repeat" in [x.split(":", 1)[0] for x, _ in gpu.profile(g.gf, 1)]
    g.free()
