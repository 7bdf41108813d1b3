"""The mixture-of-experts and state-space operators on the device against
their definitions in float64, through the C ABI as a host drives them.

Bounds count roundings: u = 2^-24 is half a step of f32. A sum of n terms in
any order is within n u of the sum of their magnitudes.
"""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def compute(gpu, G, times=3):
    """eagerly, captured, replayed"""
    for _ in range(times):
        assert G.compute(gpu.backend) == 0


def within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all() or not np.isfinite(want).all(), what
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), f"{what}: {np.argmax(off)} off by {np.abs(got - want).flat[np.argmax(off)]:.3g}, " \
                             f"allowed {np.asarray(bound).flat[np.argmax(off)]:.3g}"


# ---------------------------------------------------------------- conv ---

def conv64(sx, w):
    """sx [S, C, taps - 1 + T], w [C, taps] -> y [S, T, C] and the sum of the terms' magnitudes"""
    taps, T = w.shape[1], sx.shape[2] - w.shape[1] + 1
    y = np.zeros((sx.shape[0], T, sx.shape[1]))
    m = np.zeros_like(y)
    for j in range(taps):
        term = (sx[:, :, j:j + T] * w[:, j, None]).transpose(0, 2, 1)
        y += term
        m += np.abs(term)
    return y, m


CONV = [(64, 4, 1, 1), (65, 4, 1, 3), (200, 4, 7, 2), (37, 3, 130, 1), (256, 2, 64, 2), (1, 4, 33, 1), (130, 1, 5, 2),
        (300, 6, 70, 1), (16, 4, 0, 2), (1000, 4, 515, 2)]


@pytest.mark.parametrize("C,taps,T,S", CONV)
def test_ssm_conv(ggml, gpu, C, taps, T, S):
    print(f"ssm_conv C={C} taps={taps} T={T} S={S}", flush=True)
    rng = np.random.default_rng(C + T)
    sx = rng.standard_normal((S, C, taps - 1 + T)).astype(np.float32)
    w = rng.standard_normal((C, taps)).astype(np.float32)
    G = ggml.Graph(64, 64)
    X, W = G.new(ggml.F32, taps - 1 + T, C, S), G.new(ggml.F32, taps, C)
    y = G.lib.ggml_ssm_conv(G.ctx, X, W)
    G.build(y)
    G.allocate(gpu.buft)
    if sx.size:
        G.set(X, sx)
    G.set(W, w)
    compute(gpu, G)
    if T:
        want, m = conv64(sx.astype(np.float64), w.astype(np.float64))
        within(G.get(y).reshape(S, T, C), want, taps * U * m)
    G.free()


def mixer_conv(ggml, G, X, ST, W, B, C, taps, T, S, cache=None):
    """the host's sequence: carried columns, the step's, convolution, bias, SILU, the columns carried on"""
    L, ctx = G.lib, G.ctx
    cols = L.ggml_concat(ctx, ST, L.ggml_transpose(ctx, X), 0)
    y = L.ggml_ssm_conv(ctx, cols, W)
    if B is not None:
        y = L.ggml_add(ctx, y, B)
    y = L.ggml_silu(ctx, y)
    row = 4 * (taps - 1 + T)
    last = L.ggml_view_3d(ctx, cols, taps - 1, C, S, row, row * C, 4 * T)
    return y, (L.ggml_cont(ctx, last) if cache is None else L.ggml_cpy(ctx, last, cache))


@pytest.mark.parametrize("C,taps,T,S", [(64, 4, 1, 1), (96, 4, 1, 5), (72, 4, 2, 2), (200, 4, 65, 2), (513, 3, 300, 1),
                                        (40, 2, 9, 3), (640, 4, 1, 32)])
@pytest.mark.parametrize("bias,inplace", [(True, False), (False, True), (True, True)])
def test_mixer_convolution(ggml, gpu, C, taps, T, S, bias, inplace):
    """CONCAT -> SSM_CONV -> ADD -> SILU and the carried columns, written
    into a result or over the cache they came from (twice: the second step
    reads what the first wrote)"""
    print(f"mixer conv C={C} taps={taps} T={T} S={S} bias={bias} inplace={inplace}", flush=True)
    rng = np.random.default_rng(C + T)
    x = rng.standard_normal((S, T, C)).astype(np.float32)
    st = rng.standard_normal((S, C, taps - 1)).astype(np.float32)
    w, b = rng.standard_normal((C, taps)).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    G = ggml.Graph(64, 64)
    X, W, B = G.new(ggml.F32, C, T, S), G.new(ggml.F32, taps, C), G.new(ggml.F32, C)
    ST = G.new(ggml.F32, taps - 1, C, S, weight=True)
    y, last = mixer_conv(ggml, G, X, ST, W, B if bias else None, C, taps, T, S, ST if inplace else None)
    G.build(y, last)
    G.allocate(gpu.buft)
    G.set(ST, st)
    for t, v in ((X, x), (W, w)) + (((B, b),) if bias else ()):
        G.set(t, v)
    for _ in range(4):
        assert G.compute(gpu.backend) == 0
        cols = np.concatenate([st, x.transpose(0, 2, 1)], 2).astype(np.float64)
        pre, m = conv64(cols, w.astype(np.float64))
        if bias:
            pre, m = pre + b, m + np.abs(b)
        # |silu'| < 1.1; exp, the sum, the quotient: four roundings of the result
        want = pre / (1 + np.exp(-pre))
        within(G.get(y).reshape(S, T, C), want, 1.1 * (taps + 1) * U * m + 4 * U * np.abs(want) + 1e-37, "y")
        nxt = cols[:, :, T:].astype(np.float32)
        got = G.get(ST if inplace else last).reshape(S, C, taps - 1)
        assert np.array_equal(got, nxt)
        if inplace:
            st = nxt
    G.free()


@pytest.mark.parametrize("C,taps,T,S", [(64, 4, 1, 1), (100, 4, 70, 2), (61, 3, 33, 1), (128, 2, 8, 3), (40, 6, 20, 1),
                                        (256, 40, 70, 1)])
@pytest.mark.parametrize("silu", [False, True])
def test_conv_of_adjacent_channels(ggml, gpu, C, taps, T, S, silu):
    """the columns as a transposed tensor: channels adjacent in memory"""
    print(f"adjacent channels C={C} taps={taps} T={T} S={S} silu={silu}", flush=True)
    rng = np.random.default_rng(C + T)
    sx = rng.standard_normal((S, taps - 1 + T, C)).astype(np.float32)
    w = rng.standard_normal((C, taps)).astype(np.float32)
    G = ggml.Graph(64, 64)
    X, W = G.new(ggml.F32, C, taps - 1 + T, S), G.new(ggml.F32, taps, C)
    y = G.lib.ggml_ssm_conv(G.ctx, G.lib.ggml_transpose(G.ctx, X), W)
    if silu:
        y = G.lib.ggml_silu(G.ctx, y)
    G.build(y)
    G.allocate(gpu.buft)
    G.set(X, sx)
    G.set(W, w)
    compute(gpu, G)
    want, m = conv64(sx.transpose(0, 2, 1).astype(np.float64), w.astype(np.float64))
    bound = taps * U * m
    if silu:
        want = want / (1 + np.exp(-want))
        bound = 1.1 * bound + 4 * U * np.abs(want) + 1e-37
    within(G.get(y).reshape(S, T, C), want, bound)
    G.free()


@pytest.mark.parametrize("case", ["carried first", "columns read too", "bias is an output", "two carried", "x over its cache",
                                  "x is an intermediate", "y is an intermediate"])
def test_mixer_convolution_variants(ggml, gpu, case):
    """orders and readers with which the sequence may not, or may only partly,
    run as one launch: the results are the same"""
    print(f"mixer conv: {case}", flush=True)
    C, taps, T, S = 96, 4, 21, 2
    rng = np.random.default_rng(7)
    x = rng.standard_normal((S, T, C)).astype(np.float32)
    st = rng.standard_normal((S, C, taps - 1)).astype(np.float32)
    w, b = rng.standard_normal((C, taps)).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    W, B = G.new(ggml.F32, taps, C), G.new(ggml.F32, C)
    X = G.new(ggml.F32, C, T, S, weight=True)
    ST = G.new(ggml.F32, taps - 1, C, S, weight=True)
    # (an intermediate's memory is free once it is joined: the result may lie over it)
    from_x = L.ggml_scale(ctx, X, 1.0) if case == "x is an intermediate" else X
    cols = L.ggml_concat(ctx, ST, L.ggml_transpose(ctx, from_x), 0)
    conv = L.ggml_ssm_conv(ctx, cols, W)
    pre = L.ggml_add(ctx, conv, B)
    y = L.ggml_silu(ctx, pre)
    row = 4 * (taps - 1 + T)
    carried = L.ggml_cpy(ctx, L.ggml_view_3d(ctx, cols, taps - 1, C, S, row, row * C, 4 * T), ST)
    outs = {"carried first": [carried, y], "columns read too": [y, carried, L.ggml_scale(ctx, cols, 2.0)],
            "bias is an output": [pre, y, carried],
            "two carried": [y, carried, L.ggml_cont(ctx, L.ggml_view_3d(ctx, cols, taps - 1, C, S, row, row * C, 0))],
            "x is an intermediate": [y, carried], "y is an intermediate": [carried, L.ggml_scale(ctx, y, 1.0)],
            # y's copy over x, which the sequence's launch would still be reading
            "x over its cache": [carried, L.ggml_cpy(ctx, y, X)]}[case]
    G.build(*outs)
    G.allocate(gpu.buft)
    for t, v in ((X, x), (ST, st), (W, w), (B, b)):
        G.set(t, v)
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        joined = np.concatenate([st, x.transpose(0, 2, 1)], 2)
        want, m = conv64(joined.astype(np.float64), w.astype(np.float64))
        want, m = want + b, m + np.abs(b)
        if case == "bias is an output":
            within(G.get(pre).reshape(S, T, C), want, (taps + 1) * U * m, "pre")
        want = want / (1 + np.exp(-want))
        got = G.get(X if case == "x over its cache" else outs[1] if case == "y is an intermediate" else y).reshape(S, T, C)
        within(got, want, 1.1 * (taps + 1) * U * m + 4 * U * np.abs(want) + 1e-37, "y")
        if case == "columns read too":
            assert np.array_equal(G.get(outs[2]).reshape(joined.shape), 2 * joined)
        if case == "two carried":
            assert np.array_equal(G.get(outs[2]).reshape(st.shape), st)
        if case == "x over its cache":
            x = got
        st = joined[:, :, T:]
        assert np.array_equal(G.get(ST).reshape(st.shape), st)
    G.free()


# ---------------------------------------------------------------- scan ---

def scan64(s, x, dt, A, B, C, ids):
    """token by token, with a bound on f32's error: every step multiplies by a
    rounded exp(z) (z off by 3 u |z|, exp by 2 u), adds a product of three
    rounded factors and rounds; the outputs sum n terms. A chunked form rounds
    decays over several steps at once, from sums of z, and adds a chunk's
    tokens in any order: T and n more roundings of the magnitudes."""
    S, T, H, P = x.shape
    n, G = B.shape[3], B.shape[2]
    dt = dt.astype(np.float64)
    dt = np.where(dt <= 20, np.log1p(np.exp(np.minimum(dt, 20))), dt)
    h = np.zeros((S, H, P, n))
    for i, k in enumerate(ids):
        if 0 <= k < s.shape[0]:
            h[i] = s[k]
    mag, err = np.abs(h), np.zeros_like(h)
    y, yb = np.zeros((S, T, H, P)), np.zeros((S, T, H, P))
    ch = min(T, 64)
    for t in range(T):
        z = dt[:, t, :, None] * A  # [S, H, 1 | n]
        a = np.exp(z)[:, :, None]
        b, c = (np.repeat(v[:, t].astype(np.float64), H // G, 1)[:, :, None] for v in (B, C))
        add = (x[:, t].astype(np.float64) * dt[:, t, :, None])[..., None] * b
        err = a * (err + U * (6 + 6 * np.abs(z))[:, :, None] * mag) + 6 * U * np.abs(add)
        h = a * h + add
        mag = a * mag + np.abs(add)
        err = err + U * mag
        y[:, t] = (h * c).sum(3)
        yb[:, t] = ((err + (n + ch) * U * mag) * np.abs(c)).sum(3)
    return y, yb, h, err + (ch + 2) * U * mag


def scan_inputs(rng, S, T, H, P, G, n, elem, slots, fast=False):
    s = rng.standard_normal((slots, H, P, n)).astype(np.float32)
    x = rng.standard_normal((S, T, H, P)).astype(np.float32)
    step = np.exp(rng.uniform(np.log(1e-3), np.log(2.0 if fast else 1e-1), H))
    dt = (np.log(np.expm1(step)) + 0.5 * rng.standard_normal((S, T, H))).astype(np.float32)
    A = -rng.uniform(1, 16, (H, n if elem else 1)).astype(np.float32)
    B, C = (rng.standard_normal((S, T, G, n)).astype(np.float32) for _ in range(2))
    return s, x, dt, A, B, C


def run_scan(ggml, gpu, s, x, dt, A, B, C, ids, times=3):
    S, T, H, P = x.shape
    n, Gr = B.shape[3], B.shape[2]
    G = ggml.Graph(64, 64)
    arrays = [(s, (n, P, H, s.shape[0])), (x, (P, H, T, S)), (dt, (H, T, S)), (A, (A.shape[1], H)), (B, (n, Gr, T, S)),
              (C, (n, Gr, T, S)), (np.asarray(ids, np.int32), (S,))]
    t = [G.new(ggml.I32 if v.dtype == np.int32 else ggml.F32, *ne) for v, ne in arrays]
    y = G.lib.ggml_ssm_scan(G.ctx, *t)
    assert G.lib.ggml_backend_supports_op(gpu.backend, y)
    G.build(y)
    G.allocate(gpu.buft)
    for a, (v, _) in zip(t, arrays):
        if v.size:
            G.set(a, v)
    compute(gpu, G, times)
    out = G.get(y).reshape(-1)
    assert np.array_equal(G.get(t[0]).reshape(s.shape), s)  # the cache is only read
    G.free()
    return out[:x.size].reshape(x.shape), out[x.size:].reshape(S, H, P, n)


# S, T, H, P, groups, n, element decays
SCAN = [(1, 1, 2, 64, 1, 128, False), (3, 1, 6, 64, 2, 64, False), (5, 1, 3, 32, 1, 128, False), (2, 2, 4, 64, 1, 128, False),
        (1, 63, 4, 64, 1, 128, False), (2, 64, 4, 64, 2, 128, False), (1, 65, 2, 64, 1, 64, False),
        (2, 200, 3, 64, 3, 128, False), (1, 257, 4, 32, 1, 128, False), (1, 130, 2, 24, 1, 20, False),
        (1, 70, 2, 128, 1, 256, False), (1, 1100, 2, 64, 1, 128, False), (3, 600, 5, 80, 5, 100, False), (2, 90, 3, 7, 1, 5, False), (1, 333, 2, 64, 2, 64, False),
        (1, 1, 40, 1, 1, 16, True), (2, 33, 40, 1, 1, 16, True), (1, 300, 70, 1, 1, 16, True), (1, 45, 6, 4, 2, 16, True),
        (2, 20, 3, 64, 1, 128, True), (1, 700, 5, 1, 1, 8, True), (1, 0, 4, 64, 1, 128, False), (2, 0, 8, 1, 1, 16, True)]


@pytest.mark.parametrize("S,T,H,P,Gr,n,elem", SCAN)
def test_ssm_scan(ggml, gpu, S, T, H, P, Gr, n, elem):
    print(f"ssm_scan S={S} T={T} H={H} P={P} G={Gr} n={n} elem={elem}", flush=True)
    rng = np.random.default_rng(S * 1000 + T + n)
    a = scan_inputs(rng, S, T, H, P, Gr, n, elem, S + 2)
    ids = rng.permutation(S + 2)[:S]
    y, h = run_scan(ggml, gpu, *a, ids)
    wy, by, wh, bh = scan64(*a, ids)
    within(y, wy, by + 1e-37, "y")
    within(h, wh, bh + 1e-37, "states")


@pytest.mark.parametrize("T", [1, 9, 150])
@pytest.mark.parametrize("elem", [False, True])
def test_ssm_scan_slots_and_decays(ggml, gpu, T, elem):
    """slots used twice, slots outside the cache (they start from zeros),
    steps so long that a state vanishes at once, dt on both sides of 20"""
    rng = np.random.default_rng(T)
    S, H, P, n = 4, 3, 1 if elem else 64, 16 if elem else 128
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, elem, 3, fast=True)
    dt[:, ::3, 0] = 25.0
    dt[0, :, 1] = 19.9999
    dt[1, :, 2] = -60.0
    ids = [1, 1, -1, 3]
    y, h = run_scan(ggml, gpu, s, x, dt, A, B, C, ids)
    wy, by, wh, bh = scan64(s, x, dt, A, B, C, ids)
    within(y, wy, by + 1e-30, "y")
    within(h, wh, bh + 1e-30, "states")


@pytest.mark.parametrize("T", [1, 70, 330])
@pytest.mark.parametrize("what", ["x", "B", "C", "dt", "state", "long_dt"])
def test_ssm_scan_keeps_non_finite_values_where_they_are(ggml, gpu, T, what):
    """a NaN or infinity reaches what the recurrence takes it to: not the
    tokens before it, not other channels, heads or sequences. A step of dt
    1e9 forgets the state at once, without spoiling the steps after it."""
    rng = np.random.default_rng(T)
    S, H, P, n, at = 2, 3, 64, 64, T // 2
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, False, S)
    if what == "x":
        x[0, at, 1, 5] = np.nan
    elif what == "state":
        s[0, 1, 5, 3] = np.inf
    elif what == "long_dt":
        dt[0, at, 1] = 1e9
    else:
        {"B": B, "C": C, "dt": dt[..., None]}[what][0, at, 0, 0] = np.nan
    y, h = run_scan(ggml, gpu, s, x, dt, A, B, C, range(S))
    with np.errstate(all="ignore"):
        wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
    for got, want, bound in ((y, wy, by), (h, wh, bh)):
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine)
        within(got[fine], want[fine], bound[fine] + 1e-30, what)


# short states cut into segments of tokens, the last rows of a group alone;
# states in 16-byte pieces, rows left over
PIECES = [(1, 1000, 130, 1, 2, 16, True), (2, 150, 33, 3, 1, 5, True), (1, 500, 64, 1, 1, 16, False), (1, 40, 5, 7, 1, 12, False),
          (3, 97, 1, 1, 1, 1, True), (1, 31, 200, 1, 1, 16, True), (1, 32, 200, 1, 1, 16, True), (40, 64, 300, 1, 3, 16, True),
          (2, 3, 5, 20, 1, 256, False), (1, 7, 3, 33, 1, 36, False), (1, 5, 2, 64, 1, 128, True), (2, 1, 3, 50, 3, 64, True),
          (1, 1, 3, 9, 1, 192, False), (1, 40, 3, 12, 1, 24, False), (2, 2, 3, 17, 1, 131, False), (2, 11, 3, 64, 1, 128, False), (2, 12, 3, 64, 1, 128, False),
          (1, 13, 4, 40, 2, 72, False)]


@pytest.mark.parametrize("S,T,H,P,Gr,n,elem", PIECES)
def test_ssm_scan_segments_and_pieces(ggml, gpu, S, T, H, P, Gr, n, elem):
    test_ssm_scan(ggml, gpu, S, T, H, P, Gr, n, elem)


@pytest.mark.parametrize("T", [1, 70, 530])
@pytest.mark.parametrize("what", ["x", "dt", "state", "long_dt", "rising", "zeros"])
def test_ssm_scan_of_short_states_keeps_values_where_they_are(ggml, gpu, T, what):
    """a NaN or an infinity in one channel, a step that forgets everything,
    decays above one, states of zero under them"""
    rng = np.random.default_rng(T)
    S, H, P, n, at = 2, 70, 1, 16, T // 2
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, True, S)
    if what == "x":
        x[0, at, 5] = np.nan
    elif what == "dt":
        dt[1, at, 7] = np.nan
    elif what == "state":
        s[0, 5, 0, 3] = np.inf
        dt[0, :, 5] = -4
        A[5] = -1  # (an infinite state under a decay of zero would be a NaN)
    elif what == "long_dt":
        dt[0, at, 1] = 1e9
    else:
        A[3], A[4, ::2] = 2.0, 0.0
        dt[:, :, 3:5] = -3.0  # 2 log1p(e^-3) T: e^51 at most
        if what == "zeros":
            s[:] = 0
            x[:, :, 3] = 0
            dt[:, :, 3] = 3.0  # without a state: no growth to see
    y, h = run_scan(ggml, gpu, s, x, dt, A, B, C, range(S))
    with np.errstate(all="ignore"):
        wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
        by, bh = np.nan_to_num(by, nan=0.0, posinf=3e38), np.nan_to_num(bh, nan=0.0, posinf=3e38)
    if what == "zeros":  # in f64 too, 0 times a decay past its range
        wy[:, :, 3], wh[:, 3] = 0.0, 0.0
        by[:, :, 3], bh[:, 3] = 0.0, 0.0
    for got, want, bound in ((y, wy, by), (h, wh, bh)):
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine)
        within(got[fine], want[fine], bound[fine] + 1e-30, what)


@pytest.mark.parametrize("scale", [1e-20, 1e-6, 1e12])
@pytest.mark.parametrize("T", [2, 130])
def test_ssm_scan_scales(ggml, gpu, T, scale):
    """inputs far from one: every operand's own scale"""
    rng = np.random.default_rng(4)
    S, H, P, n = 1, 3, 64, 128
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, False, S)
    x[:, :, 0] *= scale
    B[:, ::3] *= scale
    C[:, 1::2] /= np.float32(scale)
    x[..., 5] *= scale
    x[:, 3::4, 1] *= scale
    a = (s, x, dt, A, B, C, range(S))
    y, h = run_scan(ggml, gpu, *a)
    wy, by, wh, bh = scan64(*a)
    within(h, wh, bh + 1e-30, "states")
    within(y, wy, by + 1e-30, "y")


@pytest.mark.parametrize("T", [1, 5, 140])
def test_ssm_scan_reads_views(ggml, gpu, T):
    """x, B and C as the column views of one projection that a mixer scans, dt a row view of a wider one"""
    rng = np.random.default_rng(3)
    S, H, P, Gr, n = 2, 4, 64, 2, 128
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, Gr, n, False, S)
    w = H * P + 2 * Gr * n
    wide = np.concatenate([v.reshape(S, T, -1) for v in (x, B, C)], 2)
    dtw = np.concatenate([np.full((S, T, 3), 7, np.float32), dt], 2)
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    X, D = G.new(ggml.F32, w, T, S), G.new(ggml.F32, 3 + H, T, S)
    sv, av, iv = G.new(ggml.F32, n, P, H, S), G.new(ggml.F32, 1, H), G.new(ggml.I32, S)
    row = 4 * w
    xv = L.ggml_view_4d(ctx, X, P, H, T, S, 4 * P, row, row * T, 0)
    bv = L.ggml_view_4d(ctx, X, n, Gr, T, S, 4 * n, row, row * T, 4 * H * P)
    cv = L.ggml_view_4d(ctx, X, n, Gr, T, S, 4 * n, row, row * T, 4 * (H * P + Gr * n))
    dv = L.ggml_view_3d(ctx, D, H, T, S, 4 * (3 + H), 4 * (3 + H) * T, 12)
    y = L.ggml_ssm_scan(ctx, sv, xv, dv, av, bv, cv, iv)
    G.build(y)
    G.allocate(gpu.buft)
    for t, v in ((X, wide), (D, dtw), (sv, s), (av, A), (iv, np.arange(S, dtype=np.int32))):
        G.set(t, v)
    compute(gpu, G)
    out = G.get(y).reshape(-1)
    wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
    within(out[:x.size].reshape(x.shape), wy, by, "y")
    within(out[x.size:].reshape(S, H, P, n), wh, bh, "states")
    G.free()


def test_ssm_scan_step_by_step_is_the_prompt(ggml, gpu):
    """a prompt's states, carried through single tokens, continue it"""
    rng = np.random.default_rng(8)
    S, T, H, P, n = 2, 70, 3, 64, 128
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, False, S)
    wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
    st = s
    for lo, hi in ((0, 66), (66, 67), (67, 68), (68, 70)):
        y, st = run_scan(ggml, gpu, st, *(v[:, lo:hi].copy() for v in (x, dt)), A, *(v[:, lo:hi].copy() for v in (B, C)),
                         range(S), times=1)
        within(y, wy[:, lo:hi], 2 * by[:, lo:hi], f"tokens {lo} to {hi}")
    within(st, wh, 2 * bh, "states")


# What of a chunk lies far under or over the rest: dt, x, B, C and the states, over tokens and over the states' elements
WIDE = [("dt", -20), ("dt", -25), ("dt", -30), ("x up", 16), ("x up", 20), ("x up", 23), ("x up", 30), ("x down", 16), ("x down", 24),
        ("x down", 40), ("x outlier", 20), ("x outlier", 23), ("n", 12), ("n", 20), ("n", 40), ("B row", 24), ("C row", 24),
        ("B column", -27), ("B column", -40), ("state", 20), ("state", 40)]


@pytest.mark.parametrize("T", [11, 64, 150])
@pytest.mark.parametrize("what,e", WIDE)
def test_ssm_scan_of_wide_ranges(ggml, gpu, T, what, e):
    """every element keeps its bits, whatever the tokens and elements beside
    it: the recurrence's bound holds element by element"""
    print(f"wide ranges T={T} {what} {e}", flush=True)
    rng = np.random.default_rng(T + abs(e))
    S, H, P, n, Gr = 2, 3, 64, 128, 1
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, Gr, n, False, S)
    half, k = T // 2, np.float32(2.0 ** e)
    if what == "dt":  # short steps first, from a state of zeros
        s[:] = 0
        dt[:, :half], dt[:, half:] = e, np.log(np.expm1(1.0))
    elif what == "x up":
        s[:] = 0
        x[:, half:] *= k
    elif what == "x down":  # a large token, decayed away before the chunk's end
        A[:] = -16
        dt[:] = np.log(np.expm1(0.1))
        for t in range(0, T, 64):
            x[:, t] *= k
    elif what == "x outlier":
        s[:] = 0
        x[:, half] *= k
    elif what == "n":  # y is the same, the states are not
        v = np.exp2(rng.uniform(-e, e, n)).astype(np.float32)
        B, C, s = B * v, C / v, s * v
    elif what == "B row":
        B[:, ::3] *= k
        B[:, 1::3] /= k
    elif what == "C row":
        C[:, ::3] *= k
        C[:, 1::3] /= k
    elif what == "B column":
        B[..., ::5] *= k
        s[..., ::5] *= k
    else:
        s[..., ::7] *= k
        s[..., 1::7] /= k
    a = (s, x, dt, A, B, C, range(S))
    y, h = run_scan(ggml, gpu, *a)
    wy, by, wh, bh = scan64(*a)
    within(h, wh, bh + 1e-30, "states")
    within(y, wy, by + 1e-30, "y")


# rows of x, y and states without 16-byte pieces, an odd number of blocks a group, several blocks a head, the
# largest states over several segments of chunks
FORMS = [(1, 700, 3, 64, 1, 256, False), (2, 300, 3, 30, 1, 30, False), (1, 200, 5, 64, 5, 130, False), (1, 1500, 7, 200, 7, 64, False),
         (1, 2200, 1, 64, 1, 128, False), (2, 129, 2, 18, 2, 253, False), (5, 12, 3, 16, 1, 16, False), (1, 128, 3, 65, 1, 129, False)]


@pytest.mark.parametrize("S,T,H,P,Gr,n,elem", FORMS)
def test_ssm_scan_forms_of_chunks(ggml, gpu, S, T, H, P, Gr, n, elem):
    test_ssm_scan(ggml, gpu, S, T, H, P, Gr, n, elem)


@pytest.mark.parametrize("n", [24, 128, 200])
def test_ssm_scan_by_token_beside_chunks(ggml, gpu, n):
    """one channel's NaN, one head's step past every number and one token's
    huge B each send their own part token by token, the rest stays as it is"""
    rng = np.random.default_rng(n)
    S, T, H, P, Gr = 2, 330, 4, 64, 2
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, Gr, n, False, S)
    x[0, 100, 0, 37] = np.nan
    dt[0, 200, 1] = 1e9
    B[1, 70, 1] *= np.float32(2.0 ** 40)
    s[1, 0, 3] *= np.float32(2.0 ** 90)
    y, h = run_scan(ggml, gpu, s, x, dt, A, B, C, range(S))
    with np.errstate(all="ignore"):
        wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
    for got, want, bound in ((y, wy, by), (h, wh, bh)):
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine)
        within(got[fine], want[fine], bound[fine] + 1e-30)


def test_ssm_scan_does_not_look_ahead(ggml, gpu):
    """a token's y has the same bits whatever comes after it in its chunk"""
    rng = np.random.default_rng(2)
    S, T, H, P, n = 1, 64, 2, 64, 128
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, 1, n, False, S)
    y, _ = run_scan(ggml, gpu, s, x, dt, A, B, C, range(S))
    x2, dt2, B2, C2 = (v.copy() for v in (x, dt, B, C))
    x2[:, 40:] *= np.float32(2.0 ** 22)
    dt2[:, 40:] += 4
    B2[:, 40:] *= np.float32(2.0 ** 10)
    C2[:, 40:] *= np.float32(2.0 ** 10)
    y2, _ = run_scan(ggml, gpu, s, x2, dt2, A, B2, C2, range(S))
    assert np.array_equal(y[:, :40], y2[:, :40])


@pytest.mark.parametrize("S,T,H,P,Gr,n,elem", [(2, 1, 3, 16, 1, 20, False), (1, 1, 3, 5, 1, 21, False), (1, 1, 2, 16, 1, 100, True),
                                               (1, 5, 2, 16, 1, 36, False), (1, 70, 2, 24, 1, 20, False), (1, 70, 3, 5, 1, 5, True),
                                               (1, 3, 2, 8, 1, 65, True)])
@pytest.mark.parametrize("what", ["dt", "growth"])
def test_ssm_scan_infinities_with_part_rows(ggml, gpu, S, T, H, P, Gr, n, elem, what):
    """a step or a decay past every number makes infinities, not NaN: states
    shorter than a row of lanes have nothing beside them that could"""
    print(f"infinities {what} S={S} T={T} H={H} P={P} n={n} elem={elem}", flush=True)
    rng = np.random.default_rng(n)
    s, x, dt, A, B, C = scan_inputs(rng, S, T, H, P, Gr, n, elem, S)
    s, x, B, C = (np.abs(v) + 0.5 for v in (s, x, B, C))
    if what == "dt":
        dt[:, 0, 1] = np.inf
    else:
        dt[:, 0, 1], A[1] = 1e3, 2.0  # e^2000
        dt[:, 1:, 1] = -30
    y, h = run_scan(ggml, gpu, s, x, dt, A, B, C, range(S))
    with np.errstate(all="ignore"):
        wy, by, wh, bh = scan64(s, x, dt, A, B, C, range(S))
    assert np.isinf(wy[:, :, 1]).all() and np.isfinite(wy[:, :, 0]).all()
    for got, want, bound in ((y, wy, by), (h, wh, bh)):
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine]) and np.isfinite(got[fine]).all()
        within(got[fine], want[fine], bound[fine] + 1e-30, what)


# -------------------------------------------------------------- experts ---

WT = {"f16": 1, "f32": 0, "q8_0": 8, "q4_K": 12}


def expert_weights(ggml, ref, rng, wt, E, M, K):
    """bytes, and the f64 values they stand for"""
    w = (0.05 * rng.standard_normal((E, M, K))).astype(np.float32)
    if wt == ggml.F32:
        return w, w.astype(np.float64)
    if wt == ggml.F16:
        h = w.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    q = ggml.quantize(wt, w.reshape(E * M, K))
    return q, ref.dequantize(wt, q, w.size).astype(np.float64).reshape(E, M, K)


def columns(ggml, ref, wt, x):
    """x as a product with this weight type sees it, in f64"""
    if wt == ggml.F32:
        return x.astype(np.float64)
    if wt == ggml.F16:
        return x.astype(np.float16).astype(np.float64)
    t = ref.Q8_0 if wt == ggml.Q8_0 else ref.Q8_K
    rows = x.reshape(-1, x.shape[-1])
    return np.stack([ref.dequantize(t, ref.quantize_act(t, r), r.size) for r in rows]).astype(np.float64).reshape(x.shape)


def experts64(w, x, ids):
    """w [E, M, K], x [T, b, K], ids [T, k] -> products [T, k, M] and the sums of the terms' magnitudes"""
    T, k = ids.shape
    y, m = np.zeros((T, k, w.shape[1])), np.zeros((T, k, w.shape[1]))
    for t in range(T):
        for s in range(k):
            e = ids[t, s]
            if 0 <= e < w.shape[0]:
                c = x[t, s % x.shape[1]]
                y[t, s], m[t, s] = w[e] @ c, np.abs(w[e]) @ np.abs(c)
    return y, m


def roundings(K):
    """of a sum of K products in f32, the factors' own (Q4_K: scale, minimum, their products) and the result's"""
    return K + 8


def routes(rng, T, E, k, how):
    if how == "spread":
        return np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    if how == "one":  # all tokens to the same experts, the others have none
        return np.tile(np.arange(E - k, E, dtype=np.int32), (T, 1))
    ids = rng.integers(0, E, (T, k)).astype(np.int32)  # an expert may come twice for a token
    if how == "outside":
        ids[rng.random((T, k)) < 0.3] = -1
        ids[0, 0] = E
    return ids


# E, k, M, K, T
EXPERTS = [(8, 2, 64, 256, 1), (4, 1, 48, 512, 3), (16, 4, 128, 256, 5), (32, 8, 200, 512, 9), (8, 2, 256, 768, 40),
           (6, 3, 176, 256, 100), (8, 4, 128, 512, 300), (64, 6, 96, 256, 130)]


@pytest.mark.parametrize("wname", ["f16", "q8_0", "q4_K", "f32"])
@pytest.mark.parametrize("E,k,M,K,T", EXPERTS)
@pytest.mark.parametrize("how,slots", [("spread", False), ("one", True), ("twice", False), ("outside", True)])
def test_mul_mat_id(ggml, gpu, ref, wname, E, k, M, K, T, how, slots):
    print(f"mul_mat_id {wname} E={E} k={k} M={M} K={K} T={T} {how} {slots}", flush=True)
    wt = WT[wname]
    rng = np.random.default_rng(E + M + T)
    raw, w = expert_weights(ggml, ref, rng, wt, E, M, K)
    x = rng.standard_normal((T, k if slots else 1, K)).astype(np.float32)
    ids = routes(rng, T, E, k, how)
    G = ggml.Graph(64, 64)
    W, X, I = G.new(wt, K, M, E, weight=True), G.new(ggml.F32, K, x.shape[1], T), G.new(ggml.I32, k, T)
    y = G.lib.ggml_mul_mat_id(G.ctx, W, X, I)
    assert G.lib.ggml_backend_supports_op(gpu.backend, y)
    G.build(y)
    G.allocate(gpu.buft)
    G.set(W, raw)
    G.set(X, x)
    G.set(I, ids)
    compute(gpu, G)
    want, mag = experts64(w, columns(ggml, ref, wt, x), ids)
    got = G.get(y).reshape(T, k, M)
    within(got, want, roundings(K) * U * mag, wname)
    assert not got[(ids < 0) | (ids >= E)].any()
    G.free()


# the borders between the forms: 32 and 256 pairs, 24 and 40 pairs an expert, K in part steps
# and part groups of scales, more experts than the wide form sorts
BORDERS = [(8, 4, 40, 96, 64), (8, 4, 40, 96, 65), (12, 4, 130, 160, 71), (12, 4, 130, 160, 72), (3, 1, 70, 1120, 300),
           (1000, 2, 16, 64, 200), (960, 2, 16, 64, 200), (1, 1, 129, 320, 257), (5, 5, 65, 224, 120),
           (8, 4, 40, 96, 8), (8, 3, 40, 96, 11), (1000, 2, 16, 64, 50), (10, 4, 40, 128, 99), (10, 4, 40, 128, 100)]


@pytest.mark.parametrize("wname", ["f16", "q8_0"])
@pytest.mark.parametrize("E,k,M,K,T", BORDERS)
@pytest.mark.parametrize("how", ["spread", "outside"])
def test_mul_mat_id_borders(ggml, gpu, ref, wname, E, k, M, K, T, how):
    test_mul_mat_id(ggml, gpu, ref, wname, E, k, M, K, T, how, how == "outside")


@pytest.mark.parametrize("wname", ["f16", "q8_0", "q4_K", "f32"])
@pytest.mark.parametrize("k,b,T", [(6, 2, 5), (6, 3, 90), (7, 1, 60), (12, 4, 21), (12, 4, 40)])
def test_mul_mat_id_slots_share_columns(ggml, gpu, ref, wname, k, b, T):
    """b columns a token, slot s takes column s % b"""
    print(f"mul_mat_id shared columns {wname} k={k} b={b} T={T}", flush=True)
    E, M, K = 14, 80, 256
    wt = WT[wname]
    rng = np.random.default_rng(k + T)
    raw, w = expert_weights(ggml, ref, rng, wt, E, M, K)
    x = rng.standard_normal((T, b, K)).astype(np.float32)
    ids = routes(rng, T, E, k, "outside")
    G = ggml.Graph(64, 64)
    W, X, I = G.new(wt, K, M, E, weight=True), G.new(ggml.F32, K, b, T), G.new(ggml.I32, k, T)
    y = G.lib.ggml_mul_mat_id(G.ctx, W, X, I)
    G.build(y)
    G.allocate(gpu.buft)
    for t, v in ((W, raw), (X, x), (I, ids)):
        G.set(t, v)
    compute(gpu, G)
    want, mag = experts64(w, columns(ggml, ref, wt, x), ids)
    within(G.get(y).reshape(T, k, M), want, roundings(K) * U * mag, wname)
    G.free()


@pytest.mark.parametrize("E,k,M,K,T", [(4, 2, 48, 768, 65), (3, 2, 200, 256, 300), (2, 1, 140, 1280, 290)])
def test_mul_mat_id_borders_of_super_blocks(ggml, gpu, ref, E, k, M, K, T):
    test_mul_mat_id(ggml, gpu, ref, "q4_K", E, k, M, K, T, "twice", True)


@pytest.mark.parametrize("M,K", [(77, 100), (33, 7), (130, 1000), (64, 1)])
@pytest.mark.parametrize("wname,T", [("f16", 2), ("f16", 90), ("f32", 90)])
def test_mul_mat_id_odd_rows(ggml, gpu, ref, wname, M, K, T):
    """rows that end inside a vector load"""
    print(f"mul_mat_id odd {wname} M={M} K={K} T={T}", flush=True)
    wt, E, k = WT[wname], 5, 2
    rng = np.random.default_rng(M)
    raw, w = expert_weights(ggml, ref, rng, wt, E, M, K)
    x = rng.standard_normal((T, 1, K)).astype(np.float32)
    ids = routes(rng, T, E, k, "spread")
    G = ggml.Graph(64, 64)
    W, X, I = G.new(wt, K, M, E, weight=True), G.new(ggml.F32, K, 1, T), G.new(ggml.I32, k, T)
    y = G.lib.ggml_mul_mat_id(G.ctx, W, X, I)
    G.build(y)
    G.allocate(gpu.buft)
    for t, v in ((W, raw), (X, x), (I, ids)):
        G.set(t, v)
    compute(gpu, G)
    want, mag = experts64(w, columns(ggml, ref, wt, x), ids)
    within(G.get(y).reshape(T, k, M), want, roundings(K) * U * mag)
    G.free()


@pytest.mark.parametrize("wname", ["f16", "q8_0", "q4_K"])
@pytest.mark.parametrize("E,k,F,K,T", [(8, 2, 96, 256, 1), (16, 4, 176, 512, 6), (8, 4, 128, 256, 200)])
@pytest.mark.parametrize("swap", [False, True])
def test_experts_up(ggml, gpu, ref, wname, E, k, F, K, T, swap):
    """SILU(gate) * up of two MUL_MAT_ID"""
    print(f"experts up {wname} E={E} k={k} F={F} K={K} T={T} swap={swap}", flush=True)
    wt = WT[wname]
    rng = np.random.default_rng(F + T)
    (rg, wg), (ru, wu) = (expert_weights(ggml, ref, rng, wt, E, F, K) for _ in range(2))
    x = rng.standard_normal((T, 1, K)).astype(np.float32)
    ids = routes(rng, T, E, k, "spread")
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    WG, WU = (G.new(wt, K, F, E, weight=True) for _ in range(2))
    X, I = G.new(ggml.F32, K, 1, T), G.new(ggml.I32, k, T)
    if swap:  # the second product built first
        up = L.ggml_mul_mat_id(ctx, WU, X, I)
        h = L.ggml_mul(ctx, up, L.ggml_silu(ctx, L.ggml_mul_mat_id(ctx, WG, X, I)))
    else:
        h = L.ggml_mul(ctx, L.ggml_silu(ctx, L.ggml_mul_mat_id(ctx, WG, X, I)), L.ggml_mul_mat_id(ctx, WU, X, I))
    G.build(h)
    G.allocate(gpu.buft)
    for t, v in ((WG, rg), (WU, ru), (X, x), (I, ids)):
        G.set(t, v)
    compute(gpu, G)
    c = columns(ggml, ref, wt, x)
    (g, gm), (u, um) = experts64(wg, c, ids), experts64(wu, c, ids)
    s = g / (1 + np.exp(-g))
    n = roundings(K) * U
    within(G.get(h).reshape(T, k, F), s * u, 1.1 * n * gm * np.abs(u) + np.abs(s) * n * um + n * n * gm * um + 6 * U * np.abs(s * u))
    G.free()


@pytest.mark.parametrize("wname", ["f16", "q8_0", "q4_K"])
@pytest.mark.parametrize("E,k,M,F,T", [(8, 2, 96, 256, 1), (8, 1, 96, 256, 3), (16, 5, 176, 512, 6), (8, 4, 128, 256, 200)])
@pytest.mark.parametrize("weighted", [True, False])
def test_experts_down(ggml, gpu, ref, wname, E, k, M, F, T, weighted):
    """the weighted sum over a token's experts of MUL_MAT_ID's columns"""
    print(f"experts down {wname} E={E} k={k} M={M} F={F} T={T} weighted={weighted}", flush=True)
    wt = WT[wname]
    rng = np.random.default_rng(M + T)
    raw, w = expert_weights(ggml, ref, rng, wt, E, M, F)
    h = rng.standard_normal((T, k, F)).astype(np.float32)
    gate = rng.random((T, k)).astype(np.float32)
    ids = routes(rng, T, E, k, "twice")
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    W, H, I, P = G.new(wt, F, M, E, weight=True), G.new(ggml.F32, F, k, T), G.new(ggml.I32, k, T), G.new(ggml.F32, 1, k, T)
    y = L.ggml_mul_mat_id(ctx, W, H, I)
    if weighted:
        y = L.ggml_mul(ctx, y, P)
    parts = [L.ggml_view_2d(ctx, y, M, T, 4 * M * k, 4 * M * i) for i in range(k)]
    out = parts[0] if k > 1 else L.ggml_cont(ctx, parts[0])
    for q in parts[1:]:
        out = L.ggml_add(ctx, out, q)
    G.build(out)
    G.allocate(gpu.buft)
    for t, v in ((W, raw), (H, h), (I, ids)) + (((P, gate),) if weighted else ()):
        G.set(t, v)
    compute(gpu, G)
    y64, mag = experts64(w, columns(ggml, ref, wt, h), ids)
    g = gate[:, :, None].astype(np.float64) if weighted else 1.0
    within(G.get(out).reshape(T, M), (y64 * g).sum(1), ((roundings(F) + k + 1) * U * mag * g).sum(1))
    G.free()


@pytest.mark.parametrize("wname", ["f16", "q8_0", "q4_K", "f32"])
@pytest.mark.parametrize("E,k,M,K,T", [(8, 2, 40, 256, 1), (8, 2, 40, 256, 9), (8, 4, 140, 512, 100)])
def test_mul_mat_id_keeps_non_finite_columns_apart(ggml, gpu, ref, wname, E, k, M, K, T):
    """a column with a NaN or an infinity spoils its own results only"""
    print(f"mul_mat_id non-finite columns {wname} E={E} k={k} M={M} K={K} T={T}", flush=True)
    wt = WT[wname]
    rng = np.random.default_rng(M + T)
    raw, w = expert_weights(ggml, ref, rng, wt, E, M, K)
    x = rng.standard_normal((T, k, K)).astype(np.float32)
    bad = np.zeros((T, k), bool)
    bad[::3, 0] = True
    x[bad, 5] = np.where(np.arange(bad.sum()) % 2, np.nan, np.inf)
    ids = routes(rng, T, E, k, "twice")
    G = ggml.Graph(64, 64)
    W, X, I = G.new(wt, K, M, E, weight=True), G.new(ggml.F32, K, k, T), G.new(ggml.I32, k, T)
    y = G.lib.ggml_mul_mat_id(G.ctx, W, X, I)
    G.build(y)
    G.allocate(gpu.buft)
    for t, v in ((W, raw), (X, x), (I, ids)):
        G.set(t, v)
    compute(gpu, G)
    got = G.get(y).reshape(T, k, M)
    clean = np.where(bad[:, :, None], np.float32(0), x)
    want, mag = experts64(w, columns(ggml, ref, wt, clean), ids)
    within(got[~bad], want[~bad], roundings(K) * U * mag[~bad], wname)
    if wname in ("f16", "f32"):
        assert not np.isfinite(got[bad]).any()
    G.free()


@pytest.mark.parametrize("k", [2, 3])
@pytest.mark.parametrize("last", ["silu", "scale"])
def test_experts_down_by_weights_made_in_place(ggml, gpu, ref, k, last):
    """the slots' weights come from an operator right before the product with
    them: they are there when the sum reads them"""
    print(f"experts down by {last} weights k={k}", flush=True)
    E, M, F, T = 8, 96, 256, 5
    rng = np.random.default_rng(k)
    raw, w = expert_weights(ggml, ref, rng, ggml.F16, E, M, F)
    h = rng.standard_normal((T, k, F)).astype(np.float32)
    gate = rng.standard_normal((T, k)).astype(np.float32)
    ids = routes(rng, T, E, k, "twice")
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    W, H, I, P = G.new(ggml.F16, F, M, E, weight=True), G.new(ggml.F32, F, k, T), G.new(ggml.I32, k, T), G.new(ggml.F32, 1, k, T)
    p = L.ggml_silu(ctx, P) if last == "silu" else L.ggml_scale(ctx, P, 0.5)
    y = L.ggml_mul(ctx, L.ggml_mul_mat_id(ctx, W, H, I), p)
    parts = [L.ggml_view_2d(ctx, y, M, T, 4 * M * k, 4 * M * i) for i in range(k)]
    out = parts[0]
    for q in parts[1:]:
        out = L.ggml_add(ctx, out, q)
    G.build(out)
    G.allocate(gpu.buft)
    y64, mag = experts64(w, columns(ggml, ref, ggml.F16, h), ids)
    for t, v in ((W, raw), (H, h), (I, ids)):
        G.set(t, v)
    for _ in range(4):  # other weights each time: none from the pass before
        gate = rng.standard_normal((T, k)).astype(np.float32)
        G.set(P, gate)
        assert G.compute(gpu.backend) == 0
        g = gate.astype(np.float64)
        g = (g / (1 + np.exp(-g)) if last == "silu" else 0.5 * g)[:, :, None]
        # the weight's own roundings: four of the SILU's
        within(G.get(out).reshape(T, M), (y64 * g).sum(1), ((roundings(F) + k + 5) * U * mag * np.abs(g)).sum(1))
    G.free()


@pytest.mark.parametrize("k,T", [(2, 5), (4, 130)])
def test_experts_of_one_row(ggml, gpu, ref, k, T):
    """SILU(gate) * up of experts with one row each, summed over the slots: a
    row of weights and one of products look alike"""
    print(f"experts of one row k={k} T={T}", flush=True)
    E, K = 6, 256
    rng = np.random.default_rng(T)
    (rg, wg), (ru, wu) = (expert_weights(ggml, ref, rng, ggml.F16, E, 1, K) for _ in range(2))
    x = rng.standard_normal((T, 1, K)).astype(np.float32)
    ids = routes(rng, T, E, k, "twice")
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    WG, WU = (G.new(ggml.F16, K, 1, E, weight=True) for _ in range(2))
    X, I = G.new(ggml.F32, K, 1, T), G.new(ggml.I32, k, T)
    g = L.ggml_silu(ctx, L.ggml_mul_mat_id(ctx, WG, X, I))
    y = L.ggml_mul(ctx, L.ggml_mul_mat_id(ctx, WU, X, I), g)
    parts = [L.ggml_view_2d(ctx, y, 1, T, 4 * k, 4 * i) for i in range(k)]
    out = parts[0]
    for q in parts[1:]:
        out = L.ggml_add(ctx, out, q)
    G.build(out)
    G.allocate(gpu.buft)
    for t, v in ((WG, rg), (WU, ru), (X, x), (I, ids)):
        G.set(t, v)
    compute(gpu, G)
    xc = columns(ggml, ref, ggml.F16, x)
    (a, am), (b, bm) = experts64(wg, xc, ids), experts64(wu, xc, ids)
    act = a / (1 + np.exp(-a))
    # the gate's error grows by SILU's slope, 1.1 at most; SILU's own and the product's roundings
    bound = roundings(K) * U * (1.1 * am * np.abs(b) + np.abs(act) * bm) + 6 * U * np.abs(act * b)
    within(G.get(out).reshape(T), (act * b).sum((1, 2)), (bound + k * U * np.abs(act * b)).sum((1, 2)))
    G.free()


@pytest.mark.parametrize("shape", [(1, 6, 5), (64, 1, 5), (1, 1, 1), (64, 6, 5)])
def test_product_with_a_broadcast_silu(ggml, gpu, shape):
    """MUL with a SILU of fewer elements than the product has"""
    print(f"broadcast silu {shape}", flush=True)
    rng = np.random.default_rng(1)
    a, b = rng.standard_normal((5, 6, 64)).astype(np.float32), rng.standard_normal(shape[::-1]).astype(np.float32)
    G = ggml.Graph(64, 64)
    A, B = G.new(ggml.F32, 64, 6, 5), G.new(ggml.F32, *shape)
    y = G.lib.ggml_mul(G.ctx, A, G.lib.ggml_silu(G.ctx, B))
    G.build(y)
    G.allocate(gpu.buft)
    G.set(A, a)
    G.set(B, b)
    compute(gpu, G)
    want = a * (b / (1 + np.exp(-b.astype(np.float64))))
    within(G.get(y).reshape(5, 6, 64), want, 6 * U * np.abs(want))
    G.free()


def test_experts_down_without_rows(ggml, gpu):
    """experts of no rows: nothing to sum, nothing done"""
    E, k, K, T = 4, 3, 32, 2
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    W, H, I, P = G.new(ggml.F16, K, 0, E), G.new(ggml.F32, K, k, T), G.new(ggml.I32, k, T), G.new(ggml.F32, 1, k, T)
    y = L.ggml_mul(ctx, L.ggml_mul_mat_id(ctx, W, H, I), P)
    parts = [L.ggml_view_2d(ctx, y, 0, T, 0, 0) for i in range(k)]
    out = parts[0]
    for q in parts[1:]:
        out = L.ggml_add(ctx, out, q)
    G.build(out)
    G.allocate(gpu.buft)
    G.set(I, np.zeros((T, k), np.int32))
    compute(gpu, G)
    G.free()


# --------------------------------------------------------------- router ---

def sorted64(a, desc):
    """numpy's stable sort of the keys, NaN the largest"""
    a = a.astype(np.float64) + 0.0
    nan = np.isnan(a)
    key = np.where(nan, 0.0, -a if desc else a)
    return np.lexsort((key, ~nan if desc else nan), axis=-1)


@pytest.mark.parametrize("n,rows", [(1, 1), (2, 3), (8, 1), (37, 5), (64, 4), (100, 130), (128, 1), (256, 9), (300, 3),
                                    (1000, 2), (2048, 2), (5000, 1), (8192, 1), (16, 0)])
@pytest.mark.parametrize("desc", [0, 1])
def test_argsort(ggml, gpu, n, rows, desc):
    print(f"argsort n={n} rows={rows} desc={desc}", flush=True)
    rng = np.random.default_rng(n)
    a = np.round(rng.standard_normal((rows, n)) * 8).astype(np.float32) / 8  # many equal values
    a[rng.random(a.shape) < 0.05] = -0.0
    if n > 20:
        a[:, 3], a[:, 5], a[:, 7], a[:, 11] = np.nan, np.inf, -np.inf, -np.nan
        a[rng.random(a.shape) < 0.05] = np.finfo(np.float32).min
    G = ggml.Graph(64, 64)
    X = G.new(ggml.F32, n, rows)
    y = G.lib.ggml_argsort(G.ctx, X, desc)
    G.build(y)
    G.allocate(gpu.buft)
    if rows:
        G.set(X, a)
    compute(gpu, G)
    if rows:
        assert np.array_equal(G.get(y).reshape(rows, n), sorted64(a, desc))
    G.free()


def test_argsort_refuses_long_rows(ggml, gpu):
    G = ggml.Graph(64, 64)
    y = G.lib.ggml_argsort(G.ctx, G.new(ggml.F32, 8193, 1), 1)
    assert not G.lib.ggml_backend_supports_op(gpu.backend, y)
    G.free()


@pytest.mark.parametrize("n,rows", [(1, 1), (8, 4), (77, 130), (1000, 3)])
def test_sum_rows(ggml, gpu, n, rows):
    rng = np.random.default_rng(n)
    a = rng.standard_normal((rows, n)).astype(np.float32)
    G = ggml.Graph(64, 64)
    X = G.new(ggml.F32, n, rows)
    y = G.lib.ggml_sum_rows(G.ctx, X)
    G.build(y)
    G.allocate(gpu.buft)
    G.set(X, a)
    compute(gpu, G)
    a = a.astype(np.float64)
    within(G.get(y).reshape(rows), a.sum(1), n * U * np.abs(a).sum(1))
    G.free()


def router(ggml, G, logits, E, k, T, gating):
    """ids and weights: softmax over the chosen logits, or the probabilities (renormalised)"""
    L, ctx = G.lib, G.ctx
    if gating == "chosen":
        ids = L.ggml_top_k(ctx, logits, k)
        w = L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, logits, 1, E, T), ids)
        return ids, L.ggml_soft_max(ctx, L.ggml_reshape_2d(ctx, w, k, T))
    probs = L.ggml_soft_max(ctx, logits)
    ids = L.ggml_top_k(ctx, probs, k)
    w = L.ggml_reshape_2d(ctx, L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, probs, 1, E, T), ids), k, T)
    return ids, w if gating == "probs" else L.ggml_div(ctx, w, L.ggml_sum_rows(ctx, w))


@pytest.mark.parametrize("E,k,T", [(8, 2, 1), (64, 6, 3), (128, 8, 1), (128, 8, 200), (100, 1, 7), (60, 4, 33),
                                   (256, 8, 65), (512, 10, 20), (16, 16, 5), (300, 32, 9)])
@pytest.mark.parametrize("gating", ["chosen", "probs", "normed"])
def test_router(ggml, gpu, E, k, T, gating):
    print(f"router E={E} k={k} T={T} {gating}", flush=True)
    rng = np.random.default_rng(E + T)
    # distances between a row's logits that no rounding of the softmax hides
    a = np.stack([rng.permutation(E) for _ in range(T)]).astype(np.float32) / 16 + rng.standard_normal((T, 1)).astype(np.float32)
    if gating == "chosen":
        a[:, : E // 2] = np.round(a[:, : E // 2])  # and equal ones
    G = ggml.Graph(64, 64)
    X = G.new(ggml.F32, E, T)
    ids, w = router(ggml, G, X, E, k, T, gating)
    ic = G.lib.ggml_cont(G.ctx, ids)
    G.build(ic, w)
    G.allocate(gpu.buft)
    G.set(X, a)
    compute(gpu, G)
    want = sorted64(a, 1)[:, :k]
    assert np.array_equal(G.get(ic).reshape(T, k), want)
    p = np.exp(a.astype(np.float64) - a.max(1, keepdims=True))
    chosen = np.take_along_axis(p, want, 1)
    p = chosen / (p.sum(1, keepdims=True) if gating == "probs" else chosen.sum(1, keepdims=True))
    within(G.get(w).reshape(T, k), p, (8 + k) * U * p)
    G.free()


@pytest.mark.parametrize("n,k", [(8, 1), (8, 8), (63, 5), (65, 32), (129, 3), (1000, 32), (1024, 7), (1025, 7), (200, 33)])
@pytest.mark.parametrize("rows", [1, 6])
def test_top_k_of_any_values(ggml, gpu, n, k, rows):
    """equal values, both zeros, NaN (the largest), infinities; a second view of fewer columns"""
    print(f"top_k n={n} k={k} rows={rows}", flush=True)
    rng = np.random.default_rng(n)
    a = (np.round(rng.standard_normal((rows, n)) * 2) / 2).astype(np.float32)
    a[rng.random(a.shape) < 0.1] = -0.0
    a[0, n // 2:], a[0, 0] = -np.inf, np.inf
    a[-1, n // 3] = np.nan
    a[rows // 2, :] = np.finfo(np.float32).min
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    X = G.new(ggml.F32, n, rows)
    ids = L.ggml_top_k(ctx, X, k)
    fewer = L.ggml_view_2d(ctx, ids, (k + 1) // 2, rows, 4 * n, 0)
    w = L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, X, 1, n, rows), ids)
    outs = [L.ggml_cont(ctx, ids), L.ggml_cont(ctx, fewer), w]
    G.build(*outs)
    G.allocate(gpu.buft)
    G.set(X, a)
    compute(gpu, G)
    want = sorted64(a, 1)[:, :k]
    assert np.array_equal(G.get(outs[0]).reshape(rows, k), want)
    assert np.array_equal(G.get(outs[1]).reshape(rows, -1), want[:, :(k + 1) // 2])
    assert np.array_equal(G.get(w).reshape(rows, k), np.take_along_axis(a, want, 1), equal_nan=True)
    G.free()


@pytest.mark.parametrize("case", ["all places read", "places are an output", "values are an output", "values read twice", "offset view"])
def test_router_variants(ggml, gpu, case):
    """readers with which the choice may not, or may only partly, run as one launch"""
    E, k, T = 64, 6, 11
    rng = np.random.default_rng(5)
    a = rng.standard_normal((T, E)).astype(np.float32)
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    X = G.new(ggml.F32, E, T)
    order = L.ggml_argsort(ctx, X, 1)
    at = 2 if case == "offset view" else 0
    ids = L.ggml_view_2d(ctx, order, k, T, 4 * E, 4 * at)
    g = L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, X, 1, E, T), ids)
    g2 = L.ggml_reshape_2d(ctx, g, k, T)
    w = L.ggml_soft_max(ctx, g2)
    outs = [w, L.ggml_cont(ctx, ids)]
    if case == "all places read":
        outs.append(L.ggml_cont(ctx, order))
    if case == "places are an output":
        outs.append(order)
    if case == "values are an output":
        outs.append(g)
    if case == "values read twice":
        outs.append(L.ggml_scale(ctx, g2, 2.0))
    G.build(*outs)
    G.allocate(gpu.buft)
    G.set(X, a)
    compute(gpu, G)
    full = sorted64(a, 1)
    want = full[:, at:at + k]
    v = np.take_along_axis(a, want, 1)
    p = np.exp(v.astype(np.float64) - v.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    within(G.get(w).reshape(T, k), p, (8 + k) * U * p)
    assert np.array_equal(G.get(outs[1]).reshape(T, k), want)
    if case in ("all places read", "places are an output"):
        assert np.array_equal(G.get(outs[2]).reshape(T, E), full)
    if case == "values are an output":
        assert np.array_equal(G.get(g).reshape(T, k), v)
    if case == "values read twice":
        assert np.array_equal(G.get(outs[2]).reshape(T, k), 2 * v)
    G.free()


@pytest.mark.parametrize("gating", ["chosen", "normed"])
def test_router_of_intermediates(ggml, gpu, gating):
    """logits whose memory is free after their last reader, weights and places used by products"""
    E, k, T, K, M = 16, 3, 37, 64, 48
    rng = np.random.default_rng(9)
    a = rng.standard_normal((T, E)).astype(np.float32)
    raw = (0.1 * rng.standard_normal((E, M, K))).astype(np.float16)
    x = rng.standard_normal((T, 1, K)).astype(np.float32)
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    A, X, W = G.new(ggml.F32, E, T), G.new(ggml.F32, K, 1, T), G.new(ggml.F16, K, M, E, weight=True)
    ids, w = router(ggml, G, L.ggml_scale(ctx, A, 1.0), E, k, T, gating)
    y = L.ggml_mul_mat_id(ctx, W, L.ggml_scale(ctx, X, 1.0), ids)
    y = L.ggml_mul(ctx, y, L.ggml_reshape_3d(ctx, w, 1, k, T))
    total = None
    for j in range(k):
        v = L.ggml_view_2d(ctx, y, M, T, 4 * M * k, 4 * M * j)
        total = v if total is None else L.ggml_add(ctx, total, v)
    out = L.ggml_scale(ctx, total, 1.0)
    G.build(out)
    G.allocate(gpu.buft)
    for t, v in ((A, a), (X, x), (W, raw.view(np.uint16))):
        G.set(t, v)
    want = sorted64(a, 1)[:, :k]
    p = np.exp(np.take_along_axis(a, want, 1).astype(np.float64))
    p /= p.sum(1, keepdims=True)
    prod, m = experts64(raw.astype(np.float64), x.astype(np.float16).astype(np.float64), want)
    # the weights (a softmax: 8 + k roundings, over all E for the shares), the product, the sum of k
    bound = (roundings(K) + 8 + E + 2 * k + 2) * U
    for _ in range(4):
        assert G.compute(gpu.backend) == 0
        got = G.get(out).reshape(T, M)
        within(got, (prod * p[..., None]).sum(1), bound * (m * p[..., None]).sum(1) + 1e-37)
    G.free()


def test_an_output_flag_is_part_of_a_captured_graph(ggml, gpu):
    """the same nodes in the same memory, one more of them an output: its
    launches are planned anew, not replayed from the graph without it"""
    E, k, T = 64, 6, 11
    rng = np.random.default_rng(6)
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    X = G.new(ggml.F32, E, T)
    order = L.ggml_argsort(ctx, X, 1)
    w = L.ggml_get_rows(ctx, L.ggml_reshape_3d(ctx, X, 1, E, T), L.ggml_view_2d(ctx, order, k, T, 4 * E, 0))
    G.build(w, order)  # (both have memory of their own)
    G.allocate(gpu.buft)
    t = ggml.tensor(order)
    flagged = t.flags
    plain = flagged & ~2  # GGML_TENSOR_FLAG_OUTPUT
    assert plain != flagged
    for flags in (plain, flagged, plain, flagged):
        t.flags = flags
        a = rng.standard_normal((T, E)).astype(np.float32)
        G.set(X, a)
        compute(gpu, G, 4)
        full = sorted64(a, 1)
        assert np.array_equal(G.get(w).reshape(T, k), np.take_along_axis(a, full[:, :k], 1))
        if flags == flagged:
            assert np.array_equal(G.get(order).reshape(T, E), full)
    G.free()


@pytest.mark.parametrize("n,rows", [(255, 7), (256, 3), (257, 3), (511, 2), (513, 2), (4096, 2), (4097, 1)])
@pytest.mark.parametrize("desc", [0, 1])
def test_argsort_lengths(ggml, gpu, n, rows, desc):
    test_argsort(ggml, gpu, n, rows, desc)


def test_graphs_that_share_a_workspace(ggml, gpu, ref):
    """a scan in segments and a wide experts' product, each in its own graph on
    one backend, computed in turn until both are captured and replayed"""
    rng = np.random.default_rng(11)
    S, T, H, P, n = 1, 700, 3, 64, 128
    a = scan_inputs(rng, S, T, H, P, 1, n, False, S)
    E, k, M, K, N = 8, 2, 96, 256, 150
    raw, w = expert_weights(ggml, ref, rng, ggml.F16, E, M, K)
    x = rng.standard_normal((N, 1, K)).astype(np.float32)
    ids = routes(rng, N, E, k, "spread")
    G1, G2 = ggml.Graph(64, 64), ggml.Graph(64, 64)
    arrays = [(a[0], (n, P, H, S)), (a[1], (P, H, T, S)), (a[2], (H, T, S)), (a[3], (1, H)), (a[4], (n, 1, T, S)),
              (a[5], (n, 1, T, S)), (np.zeros(1, np.int32), (S,))]
    t = [G1.new(ggml.I32 if v.dtype == np.int32 else ggml.F32, *ne) for v, ne in arrays]
    y1 = G1.lib.ggml_ssm_scan(G1.ctx, *t)
    G1.build(y1)
    G1.allocate(gpu.buft)
    for q, (v, _) in zip(t, arrays):
        G1.set(q, v)
    W, X, I = G2.new(ggml.F16, K, M, E, weight=True), G2.new(ggml.F32, K, 1, N), G2.new(ggml.I32, k, N)
    y2 = G2.lib.ggml_mul_mat_id(G2.ctx, W, X, I)
    G2.build(y2)
    G2.allocate(gpu.buft)
    for q, v in ((W, raw), (X, x), (I, ids)):
        G2.set(q, v)
    wy, by, wh, bh = scan64(*a, [0])
    want, m = experts64(w, columns(ggml, ref, ggml.F16, x), ids)
    for _ in range(4):
        assert G1.compute(gpu.backend) == 0 and G2.compute(gpu.backend) == 0
        out = G1.get(y1).reshape(-1)
        within(out[:a[1].size].reshape(a[1].shape), wy, by, "y")
        within(out[a[1].size:].reshape(wh.shape), wh, bh, "states")
        within(G2.get(y2).reshape(N, k, M), want, roundings(K) * U * m + 1e-37, "experts")
    G1.free()
    G2.free()


def test_compute_without_allocations(ggml, gpu, ref):
    """the same results from the static scratch as from the backend's own"""
    import ctypes

    lib = gpu.cdll
    lib.ggml_backend_mi355x_graph_compute_static.restype = ctypes.c_int
    lib.ggml_backend_mi355x_graph_compute_static.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    rng = np.random.default_rng(13)
    H, T, n, E, k, M, K = 70, 300, 16, 8, 4, 96, 256
    a = scan_inputs(rng, 1, T, H, 1, 1, n, True, 1)
    raw, _ = expert_weights(ggml, ref, rng, ggml.Q8_0, E, M, K)
    x, lg = rng.standard_normal((T, 1, K)).astype(np.float32), rng.standard_normal((T, E)).astype(np.float32)
    G = ggml.Graph(64, 64)
    arrays = [(a[0], (n, 1, H, 1)), (a[1], (1, H, T, 1)), (a[2], (H, T, 1)), (a[3], (n, H)), (a[4], (n, 1, T, 1)),
              (a[5], (n, 1, T, 1)), (np.zeros(1, np.int32), (1,)), (lg, (E, T)), (x, (K, 1, T))]
    t = [G.new(ggml.I32 if v.dtype == np.int32 else ggml.F32, *ne) for v, ne in arrays]
    W = G.new(ggml.Q8_0, K, M, E, weight=True)
    ids, w = router(ggml, G, t[7], E, k, T, "normed")
    outs = [G.lib.ggml_ssm_scan(G.ctx, *t[:7]), w, G.lib.ggml_mul_mat_id(G.ctx, W, t[8], ids)]
    G.build(*outs)
    G.allocate(gpu.buft)
    for q, (v, _) in zip(t, arrays):
        G.set(q, v)
    G.set(W, raw)
    assert lib.ggml_backend_mi355x_graph_compute_static(gpu.backend, G.gf) == 0
    got = [G.get(o).copy() for o in outs]
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        for o, g in zip(outs, got):
            assert np.isfinite(g).all() and np.array_equal(G.get(o), g)
    G.free()


@pytest.mark.parametrize("what", ["w3", "x3", "ids2", "ids3", "y3", "sort", "sum", "taps2", "conv3", "scan_ids", "nothing"])
def test_supports_only_whole_shapes(ggml, gpu, what):
    """an outer dimension that an operator would leave out is refused (nodes
    as other hosts may make them; the constructors here do not)"""
    G = ggml.Graph(64, 64)
    L, ctx = G.lib, G.ctx
    W, X, I = G.new(ggml.F16, 64, 24, 5), G.new(ggml.F32, 64, 1, 7), G.new(ggml.I32, 3, 7)
    y = L.ggml_mul_mat_id(ctx, W, X, I)
    A = G.new(ggml.F32, 40, 6)
    srt, sm = L.ggml_argsort(ctx, A, 1), L.ggml_sum_rows(ctx, A)
    TW = G.new(ggml.F32, 4, 6)
    conv = L.ggml_ssm_conv(ctx, G.new(ggml.F32, 11, 6, 2), TW)
    S = G.new(ggml.I32, 2)
    scan = L.ggml_ssm_scan(ctx, G.new(ggml.F32, 16, 8, 4, 3), G.new(ggml.F32, 8, 4, 5, 2), G.new(ggml.F32, 4, 5, 2), G.new(ggml.F32, 1, 4),
                           G.new(ggml.F32, 16, 1, 5, 2), G.new(ggml.F32, 16, 1, 5, 2), S)
    node, of, dim = {"w3": (y, W, 3), "x3": (y, X, 3), "ids2": (y, I, 2), "ids3": (y, I, 3), "y3": (y, y, 3), "sort": (srt, srt, 2),
                     "sum": (sm, sm, 3), "taps2": (conv, TW, 2), "conv3": (conv, conv, 3), "scan_ids": (scan, S, 1), "nothing": (y, W, 3)}[what]
    for n in (y, srt, sm, conv, scan):
        assert L.ggml_backend_supports_op(gpu.backend, n)
    if what != "nothing":
        ggml.tensor(of).ne[dim] = 2
        assert not L.ggml_backend_supports_op(gpu.backend, node)
    G.free()


# ------------------------------------------------------ memory of others ---

OVER = """
import numpy as np, torch
x = torch.randn(7, 40, device="cuda")  # torch's runtime first: the plugin then shares it
from openasr_amd import ggml
gpu = ggml.plugin()
G = ggml.Graph(64, 64)
y = G.lib.ggml_silu(G.ctx, G.over(ggml.F32, 40, 7, memory=x))
G.build(y)
G.allocate(gpu.buft)
for _ in range(4):
    x.normal_()
    torch.cuda.synchronize()
    assert G.compute(gpu.backend) == 0
    v = x.double().cpu().numpy()
    want = v / (1 + np.exp(-v))
    assert (np.abs(G.get(y).reshape(7, 40) - want) <= 6 * 2.0 ** -24 * np.abs(want)).all()
G.free()
x.zero_()
torch.cuda.synchronize()  # still the caller's

def refused(m, n):
    try:
        G.over(ggml.F32, n, memory=m)
    except ValueError as e:
        return "plugin's device" in str(e)
    return False

G = ggml.Graph(64, 64)
dev = torch.zeros(1 << 20, device="cuda")
assert refused(torch.zeros(64), 64) and refused(torch.zeros(64, pin_memory=True), 64)
assert refused(dev[1:65], 64)  # not 16-byte aligned
make = gpu.cdll.ggml_backend_mi355x_buffer_from_device_ptr
assert not make(gpu.dev, dev.data_ptr(), 1 << 50)
assert not make(gpu.dev, None, 64) and not make(gpu.dev, dev.data_ptr(), 0) and not make(None, dev.data_ptr(), 64)
G.free()
print("over: done", flush=True)
"""


def test_graph_over_memory_of_another_runtime():
    """inputs where torch has them, read anew by every compute; memory that is
    not the device's is refused (in a process of its own, whose torch is
    loaded before the plugin)"""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", OVER], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "over: done" in r.stdout, r.stdout + r.stderr


WRITES = """
import numpy as np, torch
x = torch.zeros(1 << 16, device="cuda")
y = torch.zeros(1 << 16, device="cuda")
from openasr_amd import ggml
gpu = ggml.plugin()
G = ggml.Graph(64, 64)
a, b = (G.over(ggml.F32, 1 << 16, memory=m) for m in (x, y))
side = torch.cuda.Stream()
rng = np.random.default_rng(1)
for n in (4, 64, 1 << 16):
    v = rng.standard_normal(1 << 16).astype(np.float32)
    with torch.cuda.stream(side):
        x.fill_(-1)
    side.synchronize()
    assert G.lib.ggml_backend_tensor_set(a, v.ctypes.data, 16, 4 * n - 16 if n == 1 << 16 else 4 * n) == 0
    m = n - 4 if n == 1 << 16 else n
    with torch.cuda.stream(side):  # written when the call returns, for any stream
        got = x.cpu().numpy()
    assert np.array_equal(got[4:4 + m], v[:m]) and (got[:4] == -1).all() and (got[4 + m:] == -1).all(), n
for _ in range(20):
    with torch.cuda.stream(side):
        x.fill_(-1)
    side.synchronize()
    assert G.lib.ggml_backend_tensor_memset(a, 0, 64, 4 << 14) == 0
    with torch.cuda.stream(side):
        got = x.cpu().numpy()
    assert (got[16:16 + (1 << 14)] == 0).all() and (got[:16] == -1).all() and (got[16 + (1 << 14):] == -1).all()
G.free()
print("writes: done", flush=True)
"""


def test_transfers_to_memory_of_another_runtime_are_finished():
    """what ggml_backend_tensor_set and memset write is there for the memory's
    owner when they return"""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", WRITES], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "writes: done" in r.stdout, r.stdout + r.stderr


# ----------------------------------------------------------- a whole layer ---

@pytest.mark.parametrize("T,S", [(1, 1), (1, 4), (70, 2)])
def test_hybrid_layer(ggml, gpu, ref, T, S):
    """a mixer (convolution, scan) and a feed-forward of routed experts in one
    graph, both caches carried on in place, two steps"""
    print(f"hybrid layer T={T} S={S}", flush=True)
    rng = np.random.default_rng(T)
    H, P, n, taps, E, k, F = 4, 64, 64, 4, 8, 2, 96
    C, D = H * P + 2 * n, H * P
    G = ggml.Graph(256, 256)
    L, ctx = G.lib, G.ctx
    f32 = {name: (rng.standard_normal(shape) * scale).astype(np.float32) for name, shape, scale in (
        ("x", (S, T, C), 1), ("dt", (S, T, H), 0.3), ("w", (C, taps), 0.5), ("b", (C,), 0.2), ("conv", (S, C, taps - 1), 1),
        ("ssm", (S, H, P, n), 0.3), ("logits", (S * T, E), 2))}
    f32["A"] = -rng.uniform(1, 4, (H, 1)).astype(np.float32)
    wr = {m: (0.05 * rng.standard_normal((E, r, c))).astype(np.float16) for m, r, c in (("gate", F, D), ("up", F, D), ("down", D, F))}
    X, DT, LG = G.new(ggml.F32, C, T, S), G.new(ggml.F32, H, T, S), G.new(ggml.F32, E, T * S)
    W, B, A = (G.new(ggml.F32, *f32[v].shape[::-1], weight=True) for v in ("w", "b", "A"))
    CS, SS = G.new(ggml.F32, taps - 1, C, S, weight=True), G.new(ggml.F32, n, P, H, S, weight=True)
    IDS = G.new(ggml.I32, S)
    EW = {m: G.new(ggml.F16, v.shape[2], v.shape[1], E, weight=True) for m, v in wr.items()}
    y, carried = mixer_conv(ggml, G, X, CS, W, B, C, taps, T, S, CS)
    row = 4 * C
    xs = L.ggml_view_4d(ctx, y, P, H, T, S, 4 * P, row, row * T, 0)
    Bs, Cs = (L.ggml_view_4d(ctx, y, n, 1, T, S, 4 * n, row, row * T, 4 * at) for at in (D, D + n))
    sc = L.ggml_ssm_scan(ctx, SS, xs, DT, A, Bs, Cs, IDS)
    ny = S * T * D
    kept = L.ggml_cpy(ctx, L.ggml_view_1d(ctx, sc, S * D * n, 4 * ny), SS)
    h = L.ggml_view_3d(ctx, sc, D, 1, T * S, 4 * D, 4 * D, 0)
    ids, wt = router(ggml, G, LG, E, k, T * S, "normed")
    up = L.ggml_mul(ctx, L.ggml_silu(ctx, L.ggml_mul_mat_id(ctx, EW["gate"], h, ids)), L.ggml_mul_mat_id(ctx, EW["up"], h, ids))
    dn = L.ggml_mul(ctx, L.ggml_mul_mat_id(ctx, EW["down"], up, ids), L.ggml_reshape_3d(ctx, wt, 1, k, T * S))
    out = L.ggml_add(ctx, *(L.ggml_view_2d(ctx, dn, D, T * S, 4 * D * k, 4 * D * i) for i in range(k)))
    G.build(out, carried, kept)
    G.allocate(gpu.buft)
    for t, v in ((X, f32["x"]), (DT, f32["dt"]), (LG, f32["logits"]), (W, f32["w"]), (B, f32["b"]), (A, f32["A"]),
                 (CS, f32["conv"]), (SS, f32["ssm"]), (IDS, np.arange(S, dtype=np.int32))):
        G.set(t, v)
    for m, v in wr.items():
        G.set(EW[m], v.view(np.uint16))
    conv, ssm = f32["conv"].astype(np.float64), f32["ssm"].astype(np.float64)
    for step in range(4):
        assert G.compute(gpu.backend) == 0
        cols = np.concatenate([conv, f32["x"].transpose(0, 2, 1)], 2)
        pre = conv64(cols, f32["w"].astype(np.float64))[0] + f32["b"]
        act = pre / (1 + np.exp(-pre))
        conv = cols[:, :, T:]
        y64, _, ssm, _ = scan64(ssm, act[:, :, :D].reshape(S, T, H, P), f32["dt"], f32["A"], act[:, :, None, D:D + n],
                                act[:, :, None, D + n:], range(S))
        hv = y64.reshape(T * S, D)
        want = np.zeros((T * S, D))
        order = sorted64(f32["logits"], 1)[:, :k]
        p = np.exp(f32["logits"].astype(np.float64) - f32["logits"].max(1, keepdims=True))
        for t in range(T * S):
            g = p[t, order[t]] / p[t, order[t]].sum()
            for s in range(k):
                e = {m: v[order[t, s]].astype(np.float64) for m, v in wr.items()}
                a = e["gate"] @ hv[t].astype(np.float16).astype(np.float64)
                u = e["up"] @ hv[t].astype(np.float16).astype(np.float64)
                want[t] += g[s] * (e["down"] @ (a / (1 + np.exp(-a)) * u).astype(np.float16).astype(np.float64))
        got = G.get(out).reshape(T * S, D)
        # f16 roundings of the columns may fall on either side: half a step of f16 of a share of the terms
        assert np.linalg.norm(got - want) <= 2.0 ** -11 * np.linalg.norm(want), f"step {step}"
        assert np.array_equal(G.get(CS).reshape(conv.shape), conv.astype(np.float32))
        within(G.get(SS).reshape(ssm.shape), ssm, 200 * U * np.abs(ssm).max(), f"step {step} states")
    G.free()
