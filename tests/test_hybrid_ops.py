"""Constructors of the mixture-of-experts and state-space operators
(MUL_MAT_ID, ARGSORT / top_k, SUM_ROWS, SSM_CONV, SSM_SCAN): the shapes they
give and what they refuse. No device is needed."""

import pytest


@pytest.fixture()
def G(ggml):
    g = ggml.Graph(n_tensors=64, graph_size=64)
    yield g
    g.free()


def shape(ggml, t):
    return [int(v) for v in ggml.tensor(t).ne]


def test_mul_mat_id_shapes(ggml, G):
    W = G.new(ggml.F16, 64, 24, 5)
    ids = G.new(ggml.I32, 3, 7)
    for b1 in (1, 3):
        y = G.lib.ggml_mul_mat_id(G.ctx, W, G.new(ggml.F32, 64, b1, 7), ids)
        assert shape(ggml, y) == [24, 3, 7, 1] and ggml.tensor(y).type == ggml.F32


@pytest.mark.parametrize("what", ["depth", "tokens", "slots", "ids_type", "b_type", "ids_dims", "null"])
def test_mul_mat_id_refuses(ggml, G, what):
    W = G.new(ggml.F16, 64, 24, 5)
    b = G.new(ggml.F32, 32 if what == "depth" else 64, 2 if what == "slots" else 1, 7) if what != "b_type" else \
        G.new(ggml.F16, 64, 1, 7)
    ids = G.new(ggml.F32 if what == "ids_type" else ggml.I32, 3, 8 if what == "tokens" else 7,
                2 if what == "ids_dims" else 1)
    assert not G.lib.ggml_mul_mat_id(G.ctx, W, None if what == "null" else b, ids)


def test_top_k_is_a_view_of_the_sort(ggml, G):
    a = G.new(ggml.F32, 40, 6)
    k = ggml.tensor(G.lib.ggml_top_k(G.ctx, a, 5))
    assert [int(v) for v in k.ne] == [5, 6, 1, 1] and int(k.nb[1]) == 160 and k.type == ggml.I32
    s = ggml.tensor(k.view_src)
    assert [int(v) for v in s.ne] == [40, 6, 1, 1] and s.op_params[0] == ggml.GGML_SORT_ORDER_DESC


def test_sort_refuses(ggml, G):
    a = G.new(ggml.F32, 40, 6)
    assert not G.lib.ggml_top_k(G.ctx, a, 0)
    assert not G.lib.ggml_top_k(G.ctx, a, 41)
    assert not G.lib.ggml_argsort(G.ctx, a, 2)
    assert not G.lib.ggml_argsort(G.ctx, G.new(ggml.F16, 40, 6), 0)
    assert not G.lib.ggml_argsort(G.ctx, None, 0)
    assert not G.lib.ggml_sum_rows(G.ctx, G.new(ggml.I32, 40, 6))


@pytest.mark.parametrize("cols,taps,tokens", [(11, 4, 8), (3, 4, 0), (4, 4, 1), (9, 1, 9)])
def test_ssm_conv_shapes(ggml, G, cols, taps, tokens):
    y = G.lib.ggml_ssm_conv(G.ctx, G.new(ggml.F32, cols, 6, 2), G.new(ggml.F32, taps, 6))
    assert shape(ggml, y) == [6, tokens, 2, 1]


def test_ssm_conv_refuses(ggml, G):
    sx = G.new(ggml.F32, 9, 6, 2)
    assert not G.lib.ggml_ssm_conv(G.ctx, sx, G.new(ggml.F32, 4, 7))
    assert not G.lib.ggml_ssm_conv(G.ctx, sx, G.new(ggml.F32, 11, 6))
    assert not G.lib.ggml_ssm_conv(G.ctx, sx, G.new(ggml.F16, 4, 6))
    assert not G.lib.ggml_ssm_conv(G.ctx, G.new(ggml.F32, 9, 6, 2, 2), G.new(ggml.F32, 4, 6))


SCAN = dict(s=(16, 8, 4, 5), x=(8, 4, 7, 2), dt=(4, 7, 2), A=(1, 4), B=(16, 2, 7, 2), C=(16, 2, 7, 2), ids=(2,))


def scan(ggml, G, **other):
    shapes = {**SCAN, **other}
    t = [G.new(ggml.I32 if k == "ids" else ggml.F32, *shapes[k]) for k in SCAN]
    return G.lib.ggml_ssm_scan(G.ctx, *t)


def test_ssm_scan_shapes(ggml, G):
    for A in ((1, 4), (16, 4)):
        assert shape(ggml, scan(ggml, G, A=A)) == [8 * 4 * 7 * 2 + 16 * 8 * 4 * 2, 1, 1, 1]
    none = scan(ggml, G, x=(8, 4, 0, 2), dt=(4, 0, 2), B=(16, 2, 0, 2), C=(16, 2, 0, 2))
    assert shape(ggml, none)[0] == 16 * 8 * 4 * 2


@pytest.mark.parametrize("other", [dict(x=(9, 4, 7, 2)), dict(x=(8, 3, 7, 2)), dict(dt=(4, 6, 2)), dict(dt=(4, 7, 1)),
                                   dict(A=(2, 4)), dict(A=(1, 3)), dict(B=(15, 2, 7, 2)), dict(B=(16, 3, 7, 2)),
                                   dict(C=(16, 1, 7, 2)), dict(ids=(3,)), dict(ids=(2, 2))],
                         ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
def test_ssm_scan_refuses(ggml, G, other):
    assert not scan(ggml, G, **other)


def test_over_refuses_what_it_cannot_lay_out(ggml, G):
    class Memory:
        def __init__(self, n, contiguous=True):
            self.n, self.c = n, contiguous

        def is_contiguous(self):
            return self.c

        def numel(self):
            return self.n

        def element_size(self):
            return 4

        def data_ptr(self):
            return 4096

    with pytest.raises(ValueError, match="bytes for a"):
        G.over(ggml.F32, 8, 2, memory=Memory(15))
    with pytest.raises(ValueError, match="contiguous"):
        G.over(ggml.F32, 8, 2, memory=Memory(16, False))
    with pytest.raises(ValueError, match="Q8_0"):
        G.over(ggml.Q8_0, 32, 2, memory=Memory(17))
