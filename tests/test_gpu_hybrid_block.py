"""The operators of a hybrid decoder together, as its blocks use them: a
convolution's channels, their lengths (L2_NORM), the gated delta rule with its
states carried on in place, and attention with capped scores over a cache,
by the rule's outputs. Each stage against its definition in float64 of the
device's own values of the stage before.

Bounds count roundings: u = 2^-24 is half a step of f32.
"""

import threading

import numpy as np
import pytest

from test_gpu_delta import EPS, U, rule_bounds, unit, within
from test_gpu_scored_attention import attention64, make_mask

pytestmark = pytest.mark.gpu
HK, H, K, V, GROUPS = 2, 4, 64, 64, 2
CAP, SCALE, TAPS = 30.0, 1.0, 4


class Block:
    """T tokens of S streams: a graph of its own, its states in a cache of its own"""

    def __init__(self, ggml, buft, T, S, N, seed):
        self.T, self.S, self.N = T, S, N
        self.rng = np.random.default_rng(seed)
        self.G = G = ggml.Graph(64, 64)
        L, ctx = G.lib, G.ctx
        C = 2 * HK * K + H * V
        self.x = G.new(ggml.F32, T + TAPS - 1, C, S)
        self.w = G.new(ggml.F32, TAPS, C, weight=True)
        self.g, self.beta = G.new(ggml.F32, 1, H, T, S), G.new(ggml.F32, 1, H, T, S)
        self.st = G.new(ggml.F32, K, V, H, S, weight=True)
        self.k, self.v = (G.new(ggml.F16, V, N, GROUPS, S, weight=True) for _ in range(2))
        self.mask = G.new(ggml.F16, N, T)
        self.conv = L.ggml_silu(ctx, L.ggml_ssm_conv(ctx, self.x, self.w))  # [C, T, S]
        q, k, v = (L.ggml_view_4d(ctx, self.conv, n, h, T, S, 4 * n, 4 * C, 4 * C * T, 4 * at)
                   for n, h, at in ((K, HK, 0), (K, HK, HK * K), (V, H, 2 * HK * K)))
        y = L.ggml_gated_delta_net(ctx, L.ggml_l2_norm(ctx, q, EPS), L.ggml_l2_norm(ctx, k, EPS), v, self.g, self.beta, self.st)
        ny = S * T * H * V
        self.y = L.ggml_scale(ctx, L.ggml_view_4d(ctx, y, V, H, T, S, 4 * V, 4 * V * H, 4 * V * H * T, 0), 4.0)
        self.carry = L.ggml_cpy(ctx, L.ggml_view_1d(ctx, y, S * H * V * K, 4 * ny), self.st)
        self.out = L.ggml_flash_attn_ext(ctx, L.ggml_permute(ctx, self.y, 0, 2, 1, 3), self.k, self.v, self.mask, SCALE, 0.0, CAP)
        G.build(self.conv, self.y, self.carry, self.out)
        G.allocate(buft)
        n = self.rng.standard_normal
        self.wv, self.states = (0.5 * n((C, TAPS))).astype(np.float32), (0.1 * n((S, H, V, K))).astype(np.float32)
        self.kv, self.vv = (n((S, GROUPS, N, V)).astype(np.float16) for _ in range(2))
        self.mv = make_mask("causal", S, H, T, N, 0.0, self.rng)
        for t, a in ((self.w, self.wv), (self.st, self.states), (self.k, self.kv.view(np.uint16)), (self.v, self.vv.view(np.uint16)),
                     (self.mask, self.mv.view(np.uint16))):
            G.set(t, a)

    def step(self, backend):
        n, T, S = self.rng.standard_normal, self.T, self.S
        self.xv = n((S, len(self.wv), T + TAPS - 1)).astype(np.float32)
        self.gv, self.bv = -np.exp(n((S, T, H, 1))).astype(np.float32), (1 / (1 + np.exp(-n((S, T, H))))).astype(np.float32)
        for t, a in ((self.x, self.xv), (self.g, self.gv), (self.beta, self.bv)):
            self.G.set(t, a)
        assert self.G.compute(backend) == 0

    def check(self):
        T, S = self.T, self.S
        conv = self.G.get(self.conv).reshape(S, T, -1)
        x, w = self.xv.astype(np.float64), self.wv.astype(np.float64)
        z = sum(x[:, :, i:i + T] * w[:, i, None] for i in range(TAPS)).transpose(0, 2, 1)
        size = sum(np.abs(x[:, :, i:i + T] * w[:, i, None]) for i in range(TAPS)).transpose(0, 2, 1)
        want = z / (1 + np.exp(-z))
        # the sum's roundings through a slope of at most 1.1, the sigmoid's exponential of |z| and its quotient
        within(conv, want, 2 * TAPS * U * size + (16 + 4 * np.abs(z)) * U * np.abs(want) + 1e-30, "convolution")
        q, k, v = (conv[..., a:a + h * m].reshape(S, T, h, m) for a, h, m in ((0, HK, K), (HK * K, HK, K), (2 * HK * K, H, V)))
        want, end, by, bs = rule_bounds(unit(q.astype(np.float64)), unit(k.astype(np.float64)), v, self.gv, self.bv, self.states)
        y = self.G.get(self.y).reshape(S, T, H, V)
        within(y, 4 * want, 4 * by, "rule")
        self.states = self.G.get(self.st).reshape(S, H, V, K)
        within(self.states, end, bs, "states")
        want, by = attention64(y.transpose(0, 2, 1, 3), self.kv, self.vv, self.mv, SCALE, CAP, 0.0)
        within(self.G.get(self.out).reshape(S, T, H, V), want, by, "attention")


SHAPES = [(1, 1, 300), (1, 3, 70), (5, 2, 130), (100, 2, 150), (300, 1, 300)]


@pytest.mark.parametrize("T,S,N", SHAPES)
def test_block(ggml, gpu, T, S, N):
    b = Block(ggml, gpu.buft, T, S, N, T + S)
    for _ in range(5):  # launched, recorded, replayed
        b.step(gpu.backend)
        b.check()
    b.G.free()


def test_blocks_in_turn(ggml, gpu):
    """graphs of different sizes on one backend, which share its scratch memory"""
    blocks = [Block(ggml, gpu.buft, T, S, N, 7 * T + S) for T, S, N in SHAPES]
    for r in range(4):
        for b in blocks if r % 2 else blocks[::-1]:
            b.step(gpu.backend)
        for b in blocks:
            b.check()
    for b in blocks:
        b.G.free()


def test_blocks_at_once(ggml, gpu):
    """two backends of the device, each on its own stream, from two threads; launched each time (a recording
    refuses the other thread's transfers while it lasts)"""
    lib = ggml.base()
    backends = [lib.ggml_backend_dev_init(gpu.dev, None) for _ in range(2)]
    for b in backends:
        gpu.cdll.ggml_backend_mi355x_set_hip_graphs(b, False)
    failed = []

    def work(backend, seed):
        try:
            blocks = [Block(ggml, gpu.buft, T, S, N, seed + T) for T, S, N in ((1, 2, 200), (100, 2, 150))]
            for _ in range(6):
                for b in blocks:
                    b.step(backend)
                    b.check()
            for b in blocks:
                b.G.free()
        except BaseException as e:  # noqa: BLE001 -- reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(b, 100 * i)) for i, b in enumerate(backends)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for b in backends:
        lib.ggml_backend_free(b)
    assert not failed, failed


def set_far_rows(G, t, rows, step):
    """rows [n, m] to a tensor of n rows of step elements (gigabytes in all)"""
    for i, row in enumerate(np.ascontiguousarray(rows)):
        assert G.lib.ggml_backend_tensor_set(t, row.ctypes.data, i * step * rows.itemsize, row.nbytes) == 0


@pytest.mark.parametrize("Q", [1, 20])
def test_attention_offsets_past_32_bits(ggml, gpu, Q):
    """K and V rows 64 MB apart: 5 GB from the first to the last"""
    rng = np.random.default_rng(Q)
    N, D, step = 80, 64, 32 << 20
    q = rng.standard_normal((1, 2, Q, D)).astype(np.float32)
    kv = rng.standard_normal((N, D)).astype(np.float16)
    mask = make_mask("causal", 1, 2, Q, N, 0.0, rng)
    G = ggml.Graph(64, 64)
    X, M = G.new(ggml.F32, D, Q, 2, 1), G.new(ggml.F16, N, Q)
    T = G.new(ggml.F16, step, N, weight=True)
    rows = G.lib.ggml_view_4d(G.ctx, T, D, N, 1, 1, 2 * step, 2 * step * N, 2 * step * N, 0)
    y = G.lib.ggml_flash_attn_ext(G.ctx, X, rows, rows, M, SCALE / 8, 0.0, CAP)
    G.build(y)
    G.allocate(gpu.buft)
    set_far_rows(G, T, kv, step)
    G.set(X, q)
    G.set(M, mask.view(np.uint16))
    want, by = attention64(q, kv[None, None], kv[None, None], mask, SCALE / 8, CAP, 0.0)
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        within(G.get(y).reshape(want.shape), want, by)
    G.free()


@pytest.mark.parametrize("elem", [False, True], ids=["head", "element"])
def test_delta_offsets_past_32_bits(ggml, gpu, elem):
    """a token's rows 128 MB after the last one's"""
    Hv = 1
    T, D, W = 40, 64, 32 << 20
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((1, T, 1, D)).astype(np.float32) for _ in range(3))
    g = -np.exp(rng.standard_normal((1, T, 1, D if elem else 1))).astype(np.float32)
    beta, st = rng.random((1, T, 1)).astype(np.float32), rng.standard_normal((1, 1, D, D)).astype(np.float32)
    G = ggml.Graph(64, 64)
    x = G.new(ggml.F32, W, T, weight=True)
    L, ctx = G.lib, G.ctx
    ge = g.shape[3]
    view = lambda n, at: L.ggml_view_4d(ctx, x, n, 1, T, 1, 4 * n, 4 * W, 4 * W * T, 4 * at)  # noqa: E731
    s_ = G.new(ggml.F32, D, D, Hv, 1, weight=True)
    y = L.ggml_gated_delta_net(ctx, L.ggml_l2_norm(ctx, view(D, 0), EPS), L.ggml_l2_norm(ctx, view(D, D), EPS), view(D, 2 * D),
                               view(ge, 3 * D), view(1, 3 * D + ge), s_)
    G.build(y)
    G.allocate(gpu.buft)
    set_far_rows(G, x, np.concatenate([a.reshape(T, -1) for a in (q, k, v, g, beta)], 1), W)
    G.set(s_, st)
    want, end, by, bs = rule_bounds(unit(q.astype(np.float64)), unit(k.astype(np.float64)), v, g, beta, st)
    for _ in range(3):
        assert G.compute(gpu.backend) == 0
        flat = G.get(y).reshape(-1)
        within(flat[:T * D].reshape(want.shape), want, by, "y")
        within(flat[T * D:].reshape(end.shape), end, bs, "states")
    G.free()


def test_static_scratch(ggml, gpu):
    """prompts whose partials and slabs are cut to a caller's 64 MB"""
    import ctypes
    lib = gpu.cdll
    lib.ggml_backend_mi355x_graph_compute_static.restype = ctypes.c_int
    lib.ggml_backend_mi355x_graph_compute_static.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    b = Block(ggml, gpu.buft, 300, 1, 300, 3)
    b.step(gpu.backend)
    b.check()
    n = b.rng.standard_normal
    for _ in range(2):
        b.gv, b.bv = -np.exp(n((1, 300, H, 1))).astype(np.float32), (1 / (1 + np.exp(-n((1, 300, H))))).astype(np.float32)
        for t, a in ((b.x, b.xv), (b.g, b.gv), (b.beta, b.bv)):
            b.G.set(t, a)
        assert lib.ggml_backend_mi355x_graph_compute_static(gpu.backend, b.G.gf) == 0
        b.check()
    b.G.free()
    # and attention in as many pieces as fit
    rng = np.random.default_rng(9)
    q, k, v = rng.standard_normal((1, 4, 900, 128)).astype(np.float32), *(rng.standard_normal((1, 4, 900, 128)).astype(np.float16) for _ in range(2))
    mask = make_mask("causal", 1, 4, 900, 900, 0.0, rng)
    G = ggml.Graph(64, 64)
    X, M = G.new(ggml.F32, 128, 900, 4, 1), G.new(ggml.F16, 900, 900)
    kt, vt = (G.new(ggml.F16, 128, 900, 4, 1) for _ in range(2))
    y = G.lib.ggml_flash_attn_ext(G.ctx, X, kt, vt, M, 0.1, 0.0, CAP)
    G.build(y)
    G.allocate(gpu.buft)
    for t, a in ((X, q), (M, mask.view(np.uint16)), (kt, k.view(np.uint16)), (vt, v.view(np.uint16))):
        G.set(t, a)
    assert lib.ggml_backend_mi355x_graph_compute_static(gpu.backend, G.gf) == 0
    want, by = attention64(q, k, v, mask, 0.1, CAP, 0.0)
    within(G.get(y).reshape(want.shape), want, by, "attention")
    G.free()
