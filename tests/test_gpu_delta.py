"""The gated delta rule (GATED_DELTA_NET) and L2_NORM on the device against
their definitions in float64, through the C ABI as a host drives them.

Bounds count roundings: u = 2^-24 is half a step of f32.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all() or not np.isfinite(want).all(), what
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), f"{what}: {np.argmax(off)} off by {np.abs(got - want).flat[np.argmax(off)]:.3g}, " \
                             f"allowed {np.broadcast_to(bound, want.shape).flat[np.argmax(off)]:.3g}"


def unit(x):
    return x / np.maximum(np.sqrt((x * x).sum(-1, keepdims=True)), EPS)


def rule64(q, k, v, g, beta, st):
    """q, k [S, T, Hk, K], v [S, T, H, V], g [S, T, H, 1 | K], beta [S, T, H], st [S, H, V, K], token by
    token -> y, states, every token's corrections d [S, T, H, V] and the states before it [S, T, H, V, K]"""
    q, k, v, g, beta, h = (np.asarray(x, np.float64) for x in (q, k, v, g, beta, st))
    S, T, H = beta.shape
    of = np.arange(H) % k.shape[2]
    y, d, before = np.zeros_like(v), np.zeros_like(v), np.zeros((S, T, *h.shape[1:]))
    for t in range(T):
        before[:, t] = h
        h = h * np.exp(g[:, t, :, None])
        kt = k[:, t, of, None]
        d[:, t] = beta[:, t, :, None] * (v[:, t] - (h * kt).sum(3))
        h = h + d[:, t, :, :, None] * kt
        y[:, t] = (h * q[:, t, of, None]).sum(3) / np.sqrt(k.shape[3])
    return y, h, d, before


def rule_bounds(q, k, v, g, beta, st, L=64):
    """How far f32 sums may take y and the states off, for keys of length at most one, decays at most one
    and beta in [0, 1]: a token's turn of the state is then no longer than one, so errors made before do
    not grow; a chunk's own come through |(1 + A)^-1|, A its tokens' products. Each value is made with
    at most c = 2 K + 100 roundings (a product over K, the two lengths over K, a sum over a chunk of 64,
    the decay, a dozen more)."""
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    y64, end, d, before = rule64(q, k, v, g, beta, st)
    S, T, H = beta.shape
    K = k.shape[3]
    c, of = (2 * K + 100) * U, np.arange(H) % k.shape[2]
    by, e = np.zeros_like(y64), np.zeros((S, H, v.shape[3]))  # e: of a state's row, as a length
    norm = np.sqrt((np.asarray(st, np.float64) ** 2).sum(3))
    for t0 in range(0, T, L):
        n = min(L, T - t0)
        at = slice(t0, t0 + n)
        kk, qq = k[:, at, of].transpose(0, 2, 1, 3), q[:, at, of].transpose(0, 2, 1, 3)    # [S, H, n, K]
        cum = np.cumsum(np.broadcast_to(g[:, at], (S, n, H, K)), 1).transpose(0, 2, 1, 3)
        low = np.tril(np.ones((n, n)))
        with np.errstate(invalid="ignore"):
            gap = cum[:, :, :, None] - cum[:, :, None]                                      # (-inf and -inf: nothing is left)
        L_ts = np.exp(np.minimum(np.nan_to_num(gap, nan=-np.inf, neginf=-np.inf), 0.0)) * low[..., None]
        akk = (np.abs(kk)[:, :, :, None] * np.abs(kk)[:, :, None] * L_ts).sum(4)
        aqk = (np.abs(qq)[:, :, :, None] * np.abs(kk)[:, :, None] * L_ts).sum(4)
        b = beta[:, at].transpose(0, 2, 1)
        A = b[..., None] * (kk[:, :, :, None] * kk[:, :, None] * L_ts).sum(4) * np.tril(low, -1)
        T_inv = np.abs(np.linalg.inv(np.eye(n) + A))
        D = np.abs(d[:, at]).transpose(0, 2, 1, 3)                                          # [S, H, n, V]
        own = c * (b[..., None] * (np.abs(v[:, at]).transpose(0, 2, 1, 3) + norm[:, :, None]) + b[..., None] * (akk @ D) + D)
        dD = T_inv @ own
        # the states met may be off by e, which the corrections see too: e counted once more through them
        most = norm + D.sum(2)
        e_y = e[:, :, None] + aqk @ dD + c * (norm[:, :, None] + aqk @ D)
        by[:, at] = (e_y / np.sqrt(K)).transpose(0, 2, 1, 3)
        e = e + dD.sum(2) + c * most
        norm = most
    by += 4 * U * np.abs(y64) + 1e-37
    return y64, end, by, e[..., None] + 4 * U * np.abs(end) + 1e-37


def inputs(K, V, Hk, H, T, S, elem=False, seed=0, rate=0.5):
    r = np.random.default_rng(seed + 1000 * K + 10 * T + S)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v = n(S, T, Hk, K), n(S, T, Hk, K), n(S, T, H, V)
    g = -(rate * np.exp(n(S, T, H, K if elem else 1))).astype(np.float32)
    beta = (1 / (1 + np.exp(-n(S, T, H)))).astype(np.float32)
    return q, k, v, g, beta, (0.3 * n(S, H, V, K)).astype(np.float32)


def graph(ggml, gpu, q, k, v, g, beta, st, norm=True, mixed=False, after=None, names=None):
    """the graph and its tensors: operands apart, or (mixed) q, k and v as a convolution's channels"""
    S, T, Hk, K = q.shape
    H, V = v.shape[2:]
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    data = []
    if mixed:
        C = 2 * Hk * K + H * V + 4
        x = G.new(ggml.F32, C, T, S)
        data.append((x, np.concatenate([q.reshape(S, T, -1), k.reshape(S, T, -1), v.reshape(S, T, -1), np.full((S, T, 4), np.nan, np.float32)], 2)))
        q_, k_, v_ = (L.ggml_view_4d(ctx, x, n, h, T, S, 4 * n, 4 * C, 4 * C * T, 4 * at)
                      for n, h, at in ((K, Hk, 0), (K, Hk, Hk * K), (V, H, 2 * Hk * K)))
    else:
        q_, k_, v_ = G.new(ggml.F32, K, Hk, T, S), G.new(ggml.F32, K, Hk, T, S), G.new(ggml.F32, V, H, T, S)
        data += [(q_, q), (k_, k), (v_, v)]
    g_, b_, s_ = G.new(ggml.F32, g.shape[3], H, T, S), G.new(ggml.F32, 1, H, T, S), G.new(ggml.F32, K, V, H, S, weight=True)
    data += [(g_, g), (b_, beta), (s_, st)]
    qn, kn = (L.ggml_l2_norm(ctx, q_, EPS), L.ggml_l2_norm(ctx, k_, EPS)) if norm else (q_, k_)
    y = L.ggml_gated_delta_net(ctx, qn, kn, v_, g_, b_, s_)
    outs = after(G, y, s_) if after else [y]
    G.build(*outs)
    G.allocate(gpu.buft)
    for t, a in data:
        if a.size:
            G.set(t, a)
    return G, y, s_, outs


def parts(G, y, S, T, H, V, K):
    flat = G.get(y).reshape(-1)
    return flat[:S * T * H * V].reshape(S, T, H, V), flat[S * T * H * V:].reshape(S, H, V, K)


CASES = [(128, 128, 2, 4, 1, 1), (128, 128, 1, 2, 1, 33), (128, 128, 2, 4, 5, 3), (64, 96, 3, 3, 70, 2), (96, 32, 1, 2, 130, 1),
         (16, 8, 1, 1, 64, 2), (33, 7, 1, 3, 9, 2), (256, 40, 1, 1, 20, 1), (128, 64, 2, 2, 200, 1), (1, 1, 1, 1, 3, 1),
         (128, 128, 1, 1, 0, 2), (130, 20, 1, 1, 40, 1), (64, 64, 2, 2, 65, 1), (128, 16, 1, 2, 63, 2), (32, 48, 1, 1, 129, 1),
         (48, 33, 2, 4, 100, 1), (128, 112, 1, 1, 777, 1)]


@pytest.mark.parametrize("K,V,Hk,H,T,S", CASES)
@pytest.mark.parametrize("elem", [False, True], ids=["head", "element"])
def test_delta_rule(ggml, gpu, K, V, Hk, H, T, S, elem):
    print(f"delta K={K} V={V} Hk={Hk} H={H} T={T} S={S} elem={elem}", flush=True)
    x = inputs(K, V, Hk, H, T, S, elem)
    G, y, s_, _ = graph(ggml, gpu, *x)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, S, T, H, V, K)
        within(got, want, by, "y")
        within(states, end, bs, "states")
    assert np.array_equal(G.get(s_).reshape(x[5].shape), x[5])
    G.free()


@pytest.mark.parametrize("T", [1, 3, 150])
@pytest.mark.parametrize("norm", [True, False])
def test_channels_of_one_tensor(ggml, gpu, T, norm):
    """q, k and v as views of a convolution's channels, with and without their lengths taken"""
    K, V, Hk, H, S = 64, 32, 2, 4, 2
    x = list(inputs(K, V, Hk, H, T, S, seed=3))
    if not norm:
        x[0], x[1] = unit(x[0]).astype(np.float32), (unit(x[1]) * 0.9).astype(np.float32)
    G, y, _, _ = graph(ggml, gpu, *x, norm=norm, mixed=True)
    q, k = (unit(np.asarray(a, np.float64)) if norm else a for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, S, T, H, V, K)
        within(got, want, by, "y")
        within(states, end, bs, "states")
    G.free()


@pytest.mark.parametrize("T", [1, 4, 100])
@pytest.mark.parametrize("case", ["in place", "another cache", "part of a cache", "states read too", "copied twice"])
def test_states_carried_on(ggml, gpu, T, case):
    """the new states copied into the cache they came from, or elsewhere: three steps, each from the one before"""
    K, V, Hk, H, S = 128, 32, 1, 2, 3
    x = inputs(K, V, Hk, H, T, S, seed=5)
    n, ny = S * H * V * K, S * T * H * V
    other = {}

    def after(G, y, s_):
        L, ctx = G.lib, G.ctx
        states = L.ggml_view_1d(ctx, y, n, 4 * ny)
        if case == "another cache":
            other["c"] = G.new(ggml.F32, n, weight=True)
        if case == "part of a cache":
            other["whole"] = G.new(ggml.F32, 2 * n + 8, weight=True)
            other["c"] = L.ggml_view_1d(ctx, other["whole"], n, 4 * 4)
        c = L.ggml_cpy(ctx, states, other.get("c", s_))
        out = L.ggml_scale(ctx, L.ggml_view_1d(ctx, y, ny, 0), 2.0)
        if case == "states read too":
            return [out, L.ggml_scale(ctx, states, 3.0), c]
        if case == "copied twice":
            other["d"] = G.new(ggml.F32, n, weight=True)
            return [out, c, L.ggml_cpy(ctx, states, other["d"])]
        return [out, c]

    G, y, s_, outs = graph(ggml, gpu, *x, after=after)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    if case == "part of a cache":
        G.set(other["whole"], np.full(2 * n + 8, 7.0, np.float32))
    st = x[5]
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        want, end, by, bs = rule_bounds(q, k, *x[2:5], st)
        within(G.get(outs[0]).reshape(want.shape), 2 * want, 2 * by, "y")
        if case == "part of a cache":
            w = G.get(other["whole"]).reshape(-1)
            assert (w[:4] == 7).all() and (w[4 + n:] == 7).all()
            got = w[4:4 + n]
        else:
            got = G.get(other.get("c", s_))
        got = got.reshape(end.shape)
        within(got, end, bs, "states")
        if case == "states read too":
            assert np.array_equal(G.get(outs[1]).reshape(end.shape), (3 * got).astype(np.float32))
        if case == "copied twice":
            assert np.array_equal(G.get(other["d"]).reshape(end.shape), got)
        if "c" not in other:
            st = got
    G.free()


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("elem", [False, True], ids=["head", "element"])
@pytest.mark.parametrize("gate", ["forget", "keep", "deep"])
def test_gates_at_their_ends(ggml, gpu, T, elem, gate):
    """a decay of minus infinity forgets the state, one of zero keeps it, deep ones underflow"""
    K, V, Hk, H, S = 64, 32, 1, 2, 1
    x = list(inputs(K, V, Hk, H, T, S, elem, seed=7))
    r = np.random.default_rng(3)
    if gate == "forget":
        x[3][r.random(x[3].shape) < 0.2] = -np.inf
    if gate == "keep":
        x[3][:] = 0.0
        x[4][r.random(x[4].shape) < 0.3] = 0.0
        x[4][r.random(x[4].shape) < 0.3] = 1.0
    if gate == "deep":
        x[3] = (x[3] * 60).astype(np.float32)
    G, y, _, _ = graph(ggml, gpu, *x)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    assert G.compute(gpu.backend) == 0
    got, states = parts(G, y, S, T, H, V, K)
    # (a value under f32's smallest normal may come out as zero)
    within(got, want, by + 1e-36, "y")
    within(states, end, bs + 1e-36, "states")
    G.free()


@pytest.mark.parametrize("T", [2, 100])
def test_values_that_are_not_finite_stay_their_own(ggml, gpu, T):
    """an infinite value reaches its own column of one sequence, and only from its token on"""
    K, V, Hk, H, S = 64, 48, 1, 2, 2
    x = inputs(K, V, Hk, H, T, S, seed=9)
    clean = graph(ggml, gpu, *x)
    at = T // 2
    x[2][1, at, 1, 17] = np.inf
    G, y, _, _ = graph(ggml, gpu, *x)
    assert G.compute(gpu.backend) == 0 and clean[0].compute(gpu.backend) == 0
    got, states = parts(G, y, S, T, H, V, K)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    v = x[2].copy()
    v[1, at, 1, 17] = 0
    want, end, by, bs = rule_bounds(q, k, v, *x[3:])
    bad, bads = np.zeros(got.shape, bool), np.zeros(states.shape, bool)
    bad[1, at:, 1, 17] = True
    bads[1, 1, 17] = True
    within(got[~bad], want[~bad], by[~bad], "y")
    within(states[~bads], end[~bads], np.broadcast_to(bs, end.shape)[~bads], "states")
    assert not np.isfinite(got[bad]).any() and not np.isfinite(states[bads]).any()
    G.free()
    clean[0].free()


def test_keys_without_length(ggml, gpu):
    """rows of zeros, and rows under eps, through L2_NORM"""
    K, V, Hk, H, T, S = 64, 16, 1, 1, 6, 1
    x = inputs(K, V, Hk, H, T, S, seed=11)
    x[0][0, 1], x[1][0, 1] = 0, 0
    x[0][0, 3] *= 1e-9
    x[1][0, 3] *= 1e-9
    G, y, _, _ = graph(ggml, gpu, *x)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    assert G.compute(gpu.backend) == 0
    got, states = parts(G, y, S, T, H, V, K)
    within(got, want, by, "y")
    within(states, end, bs, "states")
    G.free()


@pytest.mark.parametrize("n,rows", [(128, 50), (1, 3), (65, 7), (4, 300), (1000, 9), (2048, 2)])
@pytest.mark.parametrize("strided", [False, True])
def test_l2_norm(ggml, gpu, n, rows, strided):
    r = np.random.default_rng(n)
    x = r.standard_normal((rows, n + 3 if strided else n)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e-12
    G = ggml.Graph(16, 16)
    X = G.new(ggml.F32, x.shape[1], rows)
    v = G.lib.ggml_view_2d(G.ctx, X, n, rows, 4 * x.shape[1], 8) if strided else X
    y = G.lib.ggml_l2_norm(G.ctx, v, 1e-6)
    G.build(y)
    G.allocate(gpu.buft)
    G.set(X, x)
    z = (x[:, 2:2 + n] if strided else x).astype(np.float64)
    want = z / np.maximum(np.sqrt((z * z).sum(1, keepdims=True)), 1e-6)
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        # the sum's rounding to f32, the root, the quotient, the product
        within(G.get(y).reshape(rows, n), want, 5 * U * np.abs(want) + 1e-37)
    G.free()


@pytest.mark.parametrize("T", [20, 200, 500])
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("case", ["short", "of many lengths", "long", "one key, beta two"])
def test_keys_of_other_lengths(ggml, gpu, T, K, case):
    """keys that are not of length one: a state far under v, corrections that turn it over"""
    V, H = 48, 2
    q, k, v, g, beta, st = inputs(K, V, 1, H, T, 1, seed=13)
    q, k = unit(q).astype(np.float32), unit(k)
    g[:] = -0.5
    if case == "short":
        k = k * 1e-4
    if case == "of many lengths":
        k = k * np.exp(-8 * np.random.default_rng(1).random((1, T, 1, 1)))
    if case == "long":
        k = k * 1.4
    if case == "one key, beta two":
        k = np.repeat(k[:, :1], T, 1)
        beta[:], g[:] = 2.0, -0.125
    k = k.astype(np.float32)
    want, end, d, before = rule64(q, k, v, g, beta, st)
    G, y, _, _ = graph(ggml, gpu, q, k, v, g, beta, st, norm=False)
    # |1 - beta k k^T| <= 1 here, so an error made at a token is left, s tokens on, at most e^(g s) times
    # as long: the sum of what 2 K + 100 roundings a token make of the old state, its product with k, d
    # and its own. A chunk's tokens come through |(1 + A)^-1|, rows of at most 64, or else one by one
    turns = 64 if case == "one key, beta two" else 4
    decay, e = np.exp(np.float64(g[0, 0, 0, 0])), np.zeros((1, H, V))
    by = np.zeros_like(want)
    for t in range(T):
        lk = np.sqrt((k[:, t].astype(np.float64) ** 2).sum(2))[..., None]
        made = np.sqrt((before[:, t] ** 2).sum(3)) * decay + np.abs(d[:, t]) * lk + np.abs(beta[:, t, :, None] * v[:, t]) * lk
        e = e * decay + turns * (2 * K + 100) * U * made
        by[:, t] = (e + (2 * K + 100) * U * made) / np.sqrt(K)
    for _ in range(2):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, 1, T, H, V, K)
        within(got, want, by + 1e-37, "y")
        within(states, end, e[..., None] + 1e-37, "states")
    G.free()


def test_gates_an_element_over_slabs(ggml, gpu):
    """more tokens than the rows made ready at once hold: the same bits as in two calls"""
    K, V, H, S, T, T1 = 256, 8, 32, 1, 1300, 600
    q, k, v, g, beta, st = inputs(K, V, H, H, T, S, elem=True, seed=17)
    whole, y, _, _ = graph(ggml, gpu, q, k, v, g, beta, st)
    first, y1, _, _ = graph(ggml, gpu, q[:, :T1], k[:, :T1], v[:, :T1], g[:, :T1], beta[:, :T1], st)
    assert whole.compute(gpu.backend) == 0 and first.compute(gpu.backend) == 0
    got, end = parts(whole, y, S, T, H, V, K)
    got1, end1 = parts(first, y1, S, T1, H, V, K)
    second, y2, _, _ = graph(ggml, gpu, q[:, T1:], k[:, T1:], v[:, T1:], g[:, T1:], beta[:, T1:], end1)
    assert second.compute(gpu.backend) == 0
    got2, end2 = parts(second, y2, S, T - T1, H, V, K)
    assert np.array_equal(got[:, :T1], got1) and np.array_equal(got[:, T1:], got2) and np.array_equal(end, end2)
    # and the state's first heads against the definition
    n = slice(0, 2)
    want, last, _, _ = rule64(unit(q[:, :, n].astype(np.float64)), unit(k[:, :, n].astype(np.float64)), v[:, :, n], g[:, :, n], beta[:, :, n], st[:, n])
    # (decays of 0.5 on the mean: an error is left a few tokens; 2 K + 100 roundings each of sums of terms as large as these)
    size = 32 * (2 * K + 100) * U * (np.abs(v[:, :, n]).max() + np.abs(st).max() * np.sqrt(K))
    within(got[:, :, n], want, size / np.sqrt(K), "y")
    within(end[:, n], last, size, "states")
    for x in (whole, first, second):
        x.free()


@pytest.mark.parametrize("T", [24, 64, 200])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("case", ["nothing", "leading", "trailing", "one chunk"])
def test_chunks_of_zero_keys(ggml, gpu, T, norm, case):
    """prompts that warm up, or are padded, with rows of zeros: a chunk whose keys are all zero leaves e^g S"""
    K, V, Hk, H, S = 64, 48, 1, 2, 2
    x = list(inputs(K, V, Hk, H, T, S, seed=19, rate=0.1))
    if not norm:
        x[0], x[1] = unit(x[0]).astype(np.float32), (unit(x[1]) * 0.9).astype(np.float32)
    zero = {"nothing": slice(0, T), "leading": slice(0, min(T, 70)), "trailing": slice(T // 4, T), "one chunk": slice(64, 128)}[case]
    x[1][:, zero], x[2][:, zero] = 0, 0
    if case == "nothing":
        x[0][:] = 0
    if case in ("nothing", "leading"):
        x[5][0] = 0
        x[5][1] *= 1e-4
    if case == "trailing":  # what is left of the state lies far under one
        x[3][:] = -0.15
        x[5] *= 1e-3
        x[2] *= 1e-3
    G, y, _, _ = graph(ggml, gpu, *x, norm=norm)
    q, k = (unit(np.asarray(a, np.float64)) if norm else a for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    for _ in range(2):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, S, T, H, V, K)
        within(got, want, by, "y")
        within(states, end, bs, "states")
    G.free()


def token_bounds(q, k, v, g, beta, st):
    """As rule_bounds, for a gate a head and keys and queries of length at most one: an error made at a
    token is left, later on, at most as long as the decays since then leave it (a token's turn is no longer
    than one; a chunk's tokens come through |(1 + A)^-1|, rows of at most 4 for keys like these). A token
    makes c = 2 K + 100 roundings of the old state's row, of its value and of its correction."""
    want, end, d, before = rule64(q, k, v, g, beta, st)
    K, c = k.shape[3], (2 * k.shape[3] + 100) * U
    by, e = np.zeros_like(want), np.zeros(end.shape[:3])
    for t in range(want.shape[1]):
        decay = np.exp(np.float64(g[:, t]))
        made = np.sqrt((before[:, t] ** 2).sum(3)) * decay + np.abs(d[:, t]) + beta[:, t, :, None] * np.abs(v[:, t].astype(np.float64))
        e = e * decay + 4 * c * made
        by[:, t] = (e + c * made) / np.sqrt(K)
    return want, end, by + 1e-37, e[..., None] + 1e-37


@pytest.mark.parametrize("K,V,T,S", [(64, 32, 100, 2), (128, 48, 200, 1), (128, 20, 24, 1), (96, 64, 130, 3), (256, 32, 150, 1)])
@pytest.mark.parametrize("case", ["columns", "one column", "states", "tokens", "forgotten", "falling"])
def test_values_of_many_sizes(ggml, gpu, K, V, T, S, case):
    """small columns beside large ones, and small tokens before or after large ones: each as good as alone"""
    Hk, H = 1, 2
    x = list(inputs(K, V, Hk, H, T, S, seed=23, rate=0.05))
    col = np.array([1, 1e-3, 1e-5, 1e-6], np.float32)[np.arange(V) % 4]
    if case == "columns":
        x[2] *= col
        x[5] *= col[:, None]
    if case == "one column":
        x[2][..., 5] *= 1e6
    if case == "states":
        x[5] *= 1e4 * col[:, None]
        x[2] *= col
    if case == "tokens":  # a chunk's first values are far under its last ones
        x[2] *= (10.0 ** (np.arange(T) % 64 / 63 * 5 - 5)).astype(np.float32)[:, None, None]
        x[5][:] = 0
    if case == "forgotten":  # what was large is gone, in the middle of a chunk
        x[2][:, :T // 3] *= 1e4
        x[3][:, T // 3] = -40.0
    if case == "falling":  # the state of a chunk lies far under the last one's
        x[2][:, T // 4:] *= 1e-5
        x[3][:, T // 4:T // 2] = -1.0
    G, y, _, _ = graph(ggml, gpu, *x)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    want, end, by, bs = token_bounds(q, k, *x[2:])
    for _ in range(2):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, S, T, H, V, K)
        within(got, want, by, "y")
        within(states, end, bs, "states")
    G.free()


@pytest.mark.parametrize("T", [1, 100])
@pytest.mark.parametrize("elem", [False, True], ids=["head", "element"])
def test_no_sequences(ggml, gpu, T, elem):
    """a batch that has run empty: nothing is launched, and no size of it divides anything"""
    x = inputs(64, 32, 1, 2, T, 0, elem)
    G, y, _, _ = graph(ggml, gpu, *x)
    assert G.lib.ggml_backend_supports_op(gpu.backend, y)
    assert G.compute(gpu.backend) == 0 and G.get(y).size == 0
    G.free()


@pytest.mark.parametrize("T", [1, 100])
@pytest.mark.parametrize("eps", [0.0, 1e-25, 1e-12])
def test_small_eps(ggml, gpu, T, eps):
    """rows far shorter than f32's squares reach, brought to length by an eps that lets them"""
    K, V, Hk, H, S = 64, 32, 1, 2, 2
    x = list(inputs(K, V, Hk, H, T, S, seed=29))
    x[0] *= np.float32(max(eps, 1e-22))
    x[1] *= np.float32(max(eps, 1e-22))
    G = ggml.Graph(64, 64)
    q_, k_, v_ = G.new(ggml.F32, K, Hk, T, S), G.new(ggml.F32, K, Hk, T, S), G.new(ggml.F32, V, H, T, S)
    g_, b_, s_ = G.new(ggml.F32, 1, H, T, S), G.new(ggml.F32, 1, H, T, S), G.new(ggml.F32, K, V, H, S)
    y = G.lib.ggml_gated_delta_net(G.ctx, G.lib.ggml_l2_norm(G.ctx, q_, eps), G.lib.ggml_l2_norm(G.ctx, k_, eps), v_, g_, b_, s_)
    G.build(y)
    G.allocate(gpu.buft)
    for t, a in zip((q_, k_, v_, g_, b_, s_), x):
        G.set(t, a)
    q, k = (np.asarray(a, np.float64) / np.sqrt((np.asarray(a, np.float64) ** 2).sum(-1, keepdims=True)) for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        got, states = parts(G, y, S, T, H, V, K)
        within(got, want, by, "y")
        within(states, end, bs, "states")
    G.free()


@pytest.mark.parametrize("n", [1, 64, 300])
def test_l2_norm_of_any_length(ggml, gpu, n):
    """rows whose squares leave f32, on both sides"""
    r = np.random.default_rng(n)
    x = (r.standard_normal((9, n)) * 10.0 ** np.array([-30, -24, -20, -15, 0, 15, 19, 25, 36])[:, None]).astype(np.float32)
    for eps in (0.0, 1e-28):
        G = ggml.Graph(16, 16)
        X = G.new(ggml.F32, n, 9)
        y = G.lib.ggml_l2_norm(G.ctx, X, eps)
        G.build(y)
        G.allocate(gpu.buft)
        G.set(X, x)
        z = x.astype(np.float64)
        want = z / np.maximum(np.sqrt((z * z).sum(1, keepdims=True)), eps)
        assert G.compute(gpu.backend) == 0
        within(G.get(y).reshape(9, n), want, 5 * U * np.abs(want) + 1e-37)
        G.free()


@pytest.mark.parametrize("K", [64, 128, 33, 256])
@pytest.mark.parametrize("T", [1, 100])
@pytest.mark.parametrize("elem", [False, True], ids=["head", "element"])
def test_long_rows_brought_to_length(ggml, gpu, K, T, elem):
    """rows whose squares are past f32 come to length one inside the rule as they do in L2_NORM"""
    V, Hk, H, S = 32, 1, 2, 2
    x = list(inputs(K, V, Hk, H, T, S, elem, seed=31))
    for a in x[:2]:
        a *= np.where(np.random.default_rng(1).random((S, T, Hk, 1)) < 0.3, 1e25, 1.0).astype(np.float32)
    x[0][0, 0] *= np.float32(1e30 / np.abs(x[0][0, 0]).max())
    G, y, _, _ = graph(ggml, gpu, *x)
    q, k = (unit(np.asarray(a, np.float64)) for a in x[:2])
    want, end, by, bs = rule_bounds(q, k, *x[2:])
    assert G.compute(gpu.backend) == 0
    got, states = parts(G, y, S, T, H, V, K)
    within(got, want, by, "y")
    within(states, end, bs, "states")
    G.free()
