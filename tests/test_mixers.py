"""Constructors of the gated delta rule, L2_NORM and attention with capped or
biased scores: the shapes they give and what they refuse. No device is needed."""

import pytest


@pytest.fixture()
def G(ggml):
    g = ggml.Graph(n_tensors=64, graph_size=64)
    yield g
    g.free()


DELTA = dict(q=(16, 2, 7, 3), k=(16, 2, 7, 3), v=(8, 4, 7, 3), g=(1, 4, 7, 3), beta=(1, 4, 7, 3), state=(16, 8, 4, 3))


def delta(ggml, G, types=None, **other):
    shapes = {**DELTA, **other}
    t = [G.new((types or {}).get(k, ggml.F32), *shapes[k]) if shapes[k] else None for k in DELTA]
    return G.lib.ggml_gated_delta_net(G.ctx, *t)


def test_delta_shapes(ggml, G):
    for other in (dict(), dict(g=(16, 4, 7, 3)), dict(q=(16, 4, 7, 3), k=(16, 4, 7, 3))):
        y = ggml.tensor(delta(ggml, G, **other))
        assert [int(v) for v in y.ne] == [8 * 4 * 7 * 3 + 16 * 8 * 4 * 3, 1, 1, 1] and y.type == ggml.F32
    none = ggml.tensor(delta(ggml, G, q=(16, 2, 0, 3), k=(16, 2, 0, 3), v=(8, 4, 0, 3), g=(1, 4, 0, 3), beta=(1, 4, 0, 3)))
    assert int(none.ne[0]) == 16 * 8 * 4 * 3


@pytest.mark.parametrize("other", [dict(q=(16, 1, 7, 3)), dict(k=(15, 2, 7, 3), q=(15, 2, 7, 3)), dict(k=(16, 3, 7, 3), q=(16, 3, 7, 3)),
                                   dict(v=(9, 4, 7, 3)), dict(v=(8, 4, 6, 3)), dict(g=(2, 4, 7, 3)), dict(g=(1, 2, 7, 3)),
                                   dict(beta=(8, 4, 7, 3)), dict(beta=(1, 4, 7, 1)), dict(state=(16, 8, 4, 2)), dict(state=None),
                                   dict(q=None)],
                         ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
def test_delta_refuses(ggml, G, other):
    assert not delta(ggml, G, **other)


@pytest.mark.parametrize("name", list(DELTA))
def test_delta_refuses_types(ggml, G, name):
    assert not delta(ggml, G, types={name: ggml.F16})


def test_l2_norm(ggml, G):
    a = G.new(ggml.F32, 40, 6, 2)
    assert [int(v) for v in ggml.tensor(G.lib.ggml_l2_norm(G.ctx, a, 1e-6)).ne] == [40, 6, 2, 1]
    assert not G.lib.ggml_l2_norm(G.ctx, a, -1.0)
    assert not G.lib.ggml_l2_norm(G.ctx, a, float("nan"))
    assert not G.lib.ggml_l2_norm(G.ctx, G.new(ggml.F16, 40, 6), 1e-6)
    assert not G.lib.ggml_l2_norm(G.ctx, G.lib.ggml_transpose(G.ctx, a), 1e-6)
    assert not G.lib.ggml_l2_norm(G.ctx, None, 1e-6)


def test_attention_refuses(ggml, G):
    q, k, v = G.new(ggml.F32, 64, 5, 4, 2), G.new(ggml.F16, 64, 9, 2, 2), G.new(ggml.F16, 64, 9, 2, 2)
    m = G.new(ggml.F16, 9, 5, 1, 2)
    fa = G.lib.ggml_flash_attn_ext
    assert fa(G.ctx, q, k, v, m, 0.1, 8.0, 30.0) and fa(G.ctx, q, k, v, None, 0.1, 0.0, 30.0)
    assert not fa(G.ctx, q, k, v, None, 0.1, 8.0, 0.0)  # a bias is the mask's
    for bias, cap in ((-1.0, 0.0), (0.0, -1.0), (float("inf"), 0.0), (0.0, float("inf")), (float("nan"), 0.0), (0.0, float("nan"))):
        assert not fa(G.ctx, q, k, v, m, 0.1, bias, cap)


def test_attention_refuses_what_has_no_heads(ggml, G):
    q = G.new(ggml.F32, 64, 5, 4, 2)
    fa = G.lib.ggml_flash_attn_ext
    k = G.new(ggml.F16, 64, 9, 2, 2)
    for other in ((64, 9, 0, 2), (64, 9, 2, 0)):
        e = G.new(ggml.F16, *other)
        assert not fa(G.ctx, q, e, e, None, 0.1, 0.0, 30.0)
    for other in ((9, 5, 0, 1), (9, 5, 1, 0)):
        assert not fa(G.ctx, q, k, k, G.new(ggml.F16, *other), 0.1, 0.0, 30.0)


def test_attention_refuses_caps_past_f32(ggml, G):
    q, k = G.new(ggml.F32, 64, 5, 4, 2), G.new(ggml.F16, 64, 9, 2, 2)
    fa = G.lib.ggml_flash_attn_ext
    for cap in (0.0, 1e-30, 30.0, 1e30):
        assert fa(G.ctx, q, k, k, None, 0.1, 0.0, cap)
    for cap in (1e-40, 1e-38, 3e30, 2.9e38):
        assert not fa(G.ctx, q, k, k, None, 0.1, 0.0, cap)
