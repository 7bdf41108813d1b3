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
