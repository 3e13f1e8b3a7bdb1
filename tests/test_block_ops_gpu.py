"""Layer norm, dropout, 8-bit rows and 8-bit products on the GPU against tests/block_ops.py, at the sizes where the kernels
change their form, and in compiled functions."""
import ctypes
import time

import numpy as np
import pytest

import cgt_b200 as cgt
from cgt_b200 import core, nn, runtime
from tests import block_ops as ref
from tests.gpu_util import Dev, call, code

pytestmark = pytest.mark.gpu

ROWS_COLS = [(1, 1), (3, 2), (5, 3), (2, 4), (7, 31), (33, 32), (130, 33), (1, 256), (128, 256), (9, 255), (257, 128), (64, 784), (37, 1000), (5, 1001),
             (11, 1024), (6, 1028), (300, 2048), (19, 2050), (21, 4096), (8, 4097), (4, 8192), (3, 8200), (5, 12345), (2, 20000), (3000, 4), (5001, 17)]


def _norm_inputs(R, C, dtype, seed=0):
    rs = np.random.RandomState(seed)
    x = (rs.randn(R, C) * np.exp(rs.randn(R, 1)) + 3 * rs.randn(R, 1)).astype(dtype)
    return x, (1 + 0.3 * rs.randn(C)).astype(dtype), rs.randn(C).astype(dtype), rs.randn(R, C).astype(dtype)


def _forward(x, gain, bias, eps):
    y = Dev(np.full(x.shape, 7, x.dtype))
    dx, dg, db = Dev(x), Dev(gain), Dev(bias)
    call("cgtb_layer_norm_forward", code(x.dtype), dx.ptr, x.shape[0], x.shape[1], dg.ptr, db.ptr, eps, y.ptr)
    return y.get()


def _backward(x, gain, gy, eps):
    outs = [Dev(np.full(x.shape, 7, x.dtype)), Dev(np.full(gain.shape, 7, x.dtype)), Dev(np.full(gain.shape, 7, x.dtype))]
    dx, dg, dy = Dev(x), Dev(gain), Dev(gy)
    call("cgtb_layer_norm_backward", code(x.dtype), dx.ptr, dg.ptr, dy.ptr, x.shape[0], x.shape[1], eps, *[o.ptr for o in outs])
    return [o.get() for o in outs]


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("R,C", ROWS_COLS)
def test_layer_norm(rt, R, C, dtype):
    x, gain, bias, gy = _norm_inputs(R, C, dtype)
    eps = 1e-5
    bounds = ref.norm_bounds(x, gain, bias, gy, eps)
    wants = (ref.norm(x, gain, bias, eps)[0],) + tuple(ref.norm_gradients(x, gain, gy, eps))
    for (name, got, want, bound) in zip(("y", "dx", "dgain", "dbias"), [_forward(x, gain, bias, eps)] + _backward(x, gain, gy, eps), wants, bounds):
        off = np.abs(got - want)
        assert (off <= bound).all(), (name, float((off / bound).max()))


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("C", [5, 64, 1000, 5000])
def test_layer_norm_of_rows_far_from_zero(rt, C, dtype):
    """A common offset of 1000 spreads: the variance is that of the centred values, not a difference of large sums."""
    rs = np.random.RandomState(1)
    x = (rs.randn(40, C) + 1000).astype(dtype)
    gain, bias = np.ones(C, dtype), np.zeros(C, dtype)
    assert (np.abs(_forward(x, gain, bias, 1e-5) - ref.norm(x, gain, bias, 1e-5)[0]) <= ref.norm_bounds(x, gain, bias, None, 1e-5)).all()


@pytest.mark.parametrize("C", [8, 300, 4096, 9000])
def test_layer_norm_keeps_rows_apart(rt, C):
    """Rows of equal values, of zeros, and with an infinity or a NaN: only the last two are NaN, in themselves and, as the sum
    over all rows has to be, in the gradient of the gain."""
    x, gain, bias, gy = _norm_inputs(12, C, "f4")
    x[2], x[3] = 0, 5
    want, bounds = ref.norm(x, gain, bias, 1e-5)[0], ref.norm_bounds(x, gain, bias, gy, 1e-5)
    dx = ref.norm_gradients(x, gain, gy, 1e-5)[0]
    bad = x.copy()
    bad[5, C // 2], bad[7, C - 1] = np.inf, np.nan
    fine = [r for r in range(12) if r not in (5, 7)]
    y = _forward(bad, gain, bias, 1e-5)
    gx, dgain, dbias = _backward(bad, gain, gy, 1e-5)
    assert np.isnan(y[[5, 7]]).all() and np.isnan(gx[[5, 7]]).all() and np.isnan(dgain).all() and np.isfinite(dbias).all()
    assert (np.abs(y - want) <= bounds[0])[fine].all() and (np.abs(gx - dx) <= bounds[1])[fine].all()


def test_layer_norm_without_rows(rt):
    x, gain, bias, gy = _norm_inputs(0, 40, "f4")
    assert _forward(x, gain, bias, 1e-5).shape == (0, 40)
    assert [np.abs(g).sum() for g in _backward(x, gain, gy, 1e-5)] == [0, 0, 0]


@pytest.mark.parametrize("R,C,dtype", [(128, 256, "f4"), (700, 1000, "f8"), (70, 9000, "f4")])
def test_layer_norm_is_reproducible(rt, R, C, dtype):
    x, gain, bias, gy = _norm_inputs(R, C, dtype)
    first = _backward(x, gain, gy, 1e-5)
    for _ in range(3):
        assert all(np.array_equal(a, b) for (a, b) in zip(first, _backward(x, gain, gy, 1e-5)))


def test_layer_norm_gradients_against_differences(rt):
    rs = np.random.RandomState(3)
    x, gain, bias, gy = _norm_inputs(4, 9, "f8")
    got = _backward(x, gain, gy, 1e-3)

    def loss(x, gain, bias):
        return float((_forward(x, gain, bias, 1e-3) * gy).sum())
    h = 1e-5
    for (k, g) in enumerate(got):
        for _ in range(6):
            args = [x.copy(), gain.copy(), bias.copy()]
            at = tuple(rs.randint(n) for n in args[k].shape)
            args[k][at] += h
            up = loss(*args)
            args[k][at] -= 2 * h
            # central differences: h^2 times the third derivative (some units here, 1e-10 x), and 2^-53 * |loss| / h
            assert abs((up - loss(*args)) / (2 * h) - g[at]) < 1e-7, (k, at)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("R,C", [(9, 64), (5, 100), (3, 1024), (7, 1001), (3, 8192)])
def test_layer_norm_of_arrays_that_start_anywhere(rt, R, C, dtype, offset):
    """The results do not depend on where the arrays begin: views of rows start on any element."""
    x, gain, bias, gy = _norm_inputs(R, C, dtype)
    size = x.dtype.itemsize

    def shifted(a):
        d = Dev(np.concatenate([np.zeros(offset, dtype), a.reshape(-1), np.full(4, 9, dtype)]))
        return d, ctypes.c_void_p(d.w.data + offset * size)
    arrays = [shifted(a) for a in (x, gain, bias, gy)]
    px, pg, pb, pgy = [p for (_d, p) in arrays]
    outs = [shifted(np.full_like(a, 7)) for a in (x, x, gain, gain)]
    call("cgtb_layer_norm_forward", code(dtype), px, R, C, pg, pb, 1e-5, outs[0][1])
    call("cgtb_layer_norm_backward", code(dtype), px, pg, pgy, R, C, 1e-5, *[p for (_d, p) in outs[1:]])
    bounds = ref.norm_bounds(x, gain, bias, gy, 1e-5)
    wants = (ref.norm(x, gain, bias, 1e-5)[0],) + tuple(ref.norm_gradients(x, gain, gy, 1e-5))
    for ((d, _p), want, bound) in zip(outs, wants, bounds):
        flat = d.get()
        assert (np.abs(flat[offset:offset + want.size].reshape(want.shape) - want) <= bound).all()
        assert (flat[:offset] == 0).all() and (flat[offset + want.size:] == 9).all()      # nothing outside is written


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
def _dropout(x, p, seed, step, site, shift=0):
    size = x.dtype.itemsize
    d = Dev(np.concatenate([np.zeros(shift, x.dtype), x.reshape(-1)]))
    y = Dev(np.full(x.size + shift + 8, 7, x.dtype))
    state = Dev(np.array([seed, step], "i8"))
    call("cgtb_dropout", code(x.dtype), ctypes.c_void_p(d.w.data + shift * size), x.size, p, state.ptr, site, ctypes.c_void_p(y.w.data + shift * size))
    flat = y.get()
    assert (flat[:shift] == 7).all() and (flat[shift + x.size:] == 7).all()
    return flat[shift:shift + x.size].reshape(x.shape)


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 127, 1024, 4099, 65537, 1 << 20, (1 << 21) + 3])
def test_dropout(rt, n, dtype):
    x = np.random.RandomState(n).randn(n).astype(dtype)
    for (p, seed, step, site, shift) in ((0.5, 0, 0, 0, 0), (0.1, 12345678901234567, 999, 3, 1), (0.93, -5, 2 ** 32 + 7, 1, 2), (1e-12, 1, 1, 1, 3), (0.0, 1, 1, 1, 0)):
        assert np.array_equal(_dropout(x, p, seed, step, site, shift), ref.dropout(x, p, seed, step, site)), (p, seed, step, site, shift)


def test_a_dropped_element_is_zero_whatever_it_was(rt):
    x = np.random.RandomState(0).randn(4096).astype("f4")
    keep = ref.kept(x.size, 0.5, 8, 2, 0)
    x[~keep] = np.tile(np.array([np.inf, -np.inf, np.nan], "f4"), x.size)[:int((~keep).sum())]
    y = _dropout(x, 0.5, 8, 2, 0)
    assert (y[~keep] == 0).all() and np.array_equal(y[keep], 2 * x[keep])


def test_dropout_of_its_own_memory(rt):
    x = np.random.RandomState(0).randn(5001).astype("f4")
    d, state = Dev(x), Dev(np.array([4, 5], "i8"))
    call("cgtb_dropout", code("f4"), d.ptr, x.size, 0.3, state.ptr, 2, d.ptr)
    assert np.array_equal(d.get(), ref.dropout(x, 0.3, 4, 5, 2))


# ------------------------------------------------------------------------------------------------
# 8-bit rows and products
# ------------------------------------------------------------------------------------------------
def _quantize(x):
    codes, scales = Dev(np.full((x.shape[0], -(-x.shape[1] // 16) * 16), 99, "i1")), Dev(np.full(x.shape[0], 7, "f4"))
    d = Dev(x)
    call("cgtb_quantize_rows", d.ptr, x.shape[0], x.shape[1], codes.ptr, scales.ptr)
    return codes.get(), scales.get()


def _same(got, want):
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1], equal_nan=True)


@pytest.mark.parametrize("R,C", ROWS_COLS)
def test_quantize_rows(rt, R, C):
    x = _norm_inputs(R, C, "f4")[0]
    _same(_quantize(x), ref.quantize(x))


@pytest.mark.parametrize("C", [16, 40, 700, 3001, 17000])
def test_quantize_rows_at_ties_and_at_the_ends_of_the_type(rt, C):
    rs = np.random.RandomState(C)
    x = np.zeros((16, C), "f4")
    x[0] = rs.randint(-254, 255, size=C) / 2.0
    x[0, C - 1] = 127                                            # every half is a tie
    x[1] = x[0] * np.float32(2.0 ** -140)                        # denormal
    x[2] = x[0] * np.float32(2.0 ** 120)
    x[3] = rs.randn(C) * 1e-44
    x[4] = rs.uniform(-1, 1, C) * 3.4e38
    x[6, 0] = 1e-45
    x[7, 0], x[8, C - 1], x[9, C // 2] = np.inf, np.nan, -np.inf
    x[10, 3], x[10, 4] = -0.0, -3.0
    base = rs.uniform(0.5, 1, 4).astype("f4")
    for i in range(4):                                           # next to a tie on both sides
        largest = base[i]
        half = (np.arange(C) % 127 + 0.5) * float(largest) / 127
        x[11 + i] = np.nextafter(half.astype("f4"), np.float32(4 * (i % 2))) if i < 2 else half.astype("f4")
        x[11 + i, 0] = -largest
    _same(_quantize(x), ref.quantize(x))


def test_quantize_no_rows_and_no_columns(rt):
    _same(_quantize(np.zeros((0, 33), "f4")), (np.zeros((0, 48), "i1"), np.zeros(0, "f4")))
    _same(_quantize(np.zeros((5, 0), "f4")), (np.zeros((5, 0), "i1"), np.zeros(5, "f4")))


PRODUCTS = [(1, 1, 16), (1, 1000, 784), (1, 4096, 4096), (2, 33, 48), (4, 10, 1008), (7, 129, 2000), (8, 256, 256), (9, 64, 144), (15, 100, 160),
            (16, 128, 128), (17, 127, 112), (31, 500, 1024), (33, 65, 96), (64, 1000, 512), (65, 17, 4112), (100, 256, 32), (127, 1, 208), (128, 128, 128),
            (129, 257, 400), (200, 300, 2064), (255, 1001, 1008), (256, 512, 64), (500, 96, 800), (1000, 10, 784), (1025, 515, 272), (3, 5000, 8192), (2500, 2100, 160),
            (300, 19000, 48), (4099, 2304, 1040), (100, 20001, 32), (2047, 4999, 16), (2, 1001, 1040),
            (2, 10, 256), (1, 7, 8192), (3, 17, 16), (300000, 1, 32), (130, 1030, 1008), (13, 70000, 16), (9, 1000, 2064), (17, 5, 1040),
            (200000, 2, 16), (300, 1100, 96), (513, 1001, 1008), (65, 4000, 2000), (16, 8192, 4096), (32, 4099, 144)]


def _product(a, sa, b, sb, bias):
    y = Dev(np.full((len(a), len(b)), 7, "f4"))
    da, dsa, db, dsb = Dev(a), Dev(sa), Dev(b), Dev(sb)
    dbias = Dev(bias) if bias is not None else None
    call("cgtb_int8_product", da.ptr, dsa.ptr, db.ptr, dsb.ptr, dbias.ptr if bias is not None else None, len(a), len(b), a.shape[1], y.ptr)
    return y.get()


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_int8_product(rt, M, N, K):
    rs = np.random.RandomState(M + N + K)
    a, b = rs.randint(-128, 128, (M, K)).astype("i1"), rs.randint(-128, 128, (N, K)).astype("i1")
    sa, sb = rs.rand(M).astype("f4"), (rs.rand(N) * 0.01).astype("f4")
    for bias in (None, rs.randn(N).astype("f4")):
        want, bound = ref.product(a, sa, b, sb, bias)
        off = np.abs(_product(a, sa, b, sb, bias) - want)
        assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("M,N", [(1, 3), (20, 5), (130, 3)])
def test_int8_product_fills_its_sums(rt, M, N):
    """The largest magnitudes at the longest row: 128 * 128 * 131056 is just below 2^31."""
    K = 131056
    a, b = np.full((M, K), -128, "i1"), np.full((N, K), -128, "i1")
    b[1] = 127
    one_m, one_n = np.ones(M, "f4"), np.ones(N, "f4")
    want, bound = ref.product(a[:1], one_m[:1], b, one_n, None)
    assert (np.abs(_product(a, one_m, b, one_n, None) - want) <= bound).all()


def test_int8_product_of_rows_without_a_scale(rt):
    """A row that could not be quantized (scale NaN) is NaN in the result, a row of zeros is the bias; the others are neither."""
    rs = np.random.RandomState(0)
    x = rs.randn(40, 100).astype("f4")
    x[3], x[5, 7] = 0, np.inf
    w, bias = rs.randn(50, 100).astype("f4"), rs.randn(50).astype("f4")
    (a, sa), (b, sb) = _quantize(x), _quantize(w)
    y = _product(a, sa, b, sb, bias)
    assert np.isnan(y[5]).all() and np.array_equal(y[3], bias) and np.isfinite(np.delete(y, 5, 0)).all()


def test_int8_product_without_rows_channels_or_terms(rt):
    z = np.zeros
    assert _product(z((0, 32), "i1"), z(0, "f4"), z((5, 32), "i1"), z(5, "f4"), None).shape == (0, 5)
    assert _product(z((5, 32), "i1"), z(5, "f4"), z((0, 32), "i1"), z(0, "f4"), None).shape == (5, 0)
    for M in (1, 40, 200):
        bias = np.arange(3, dtype="f4")
        assert np.array_equal(_product(z((M, 0), "i1"), z(M, "f4"), z((3, 0), "i1"), z(3, "f4"), bias), np.tile(bias, (M, 1)))


def test_refused_calls_leave_the_library_usable(rt):
    L = runtime.lib()
    d = Dev(np.zeros((4, 32), "f4"))
    c = Dev(np.zeros((4, 32), "i1"))
    s = Dev(np.zeros(4, "f4"))
    state = Dev(np.array([0, 0], "i8"))
    off = ctypes.c_void_p(c.w.data + 1)
    refused = [
        ("cgtb_layer_norm_forward", (11, d.ptr, -1, 32, d.ptr, d.ptr, 1e-5, d.ptr)),
        ("cgtb_layer_norm_forward", (11, d.ptr, 4, 32, d.ptr, d.ptr, -1e-5, d.ptr)),
        ("cgtb_layer_norm_forward", (11, d.ptr, 4, 32, d.ptr, d.ptr, float("nan"), d.ptr)),
        ("cgtb_layer_norm_forward", (7, d.ptr, 4, 32, d.ptr, d.ptr, 1e-5, d.ptr)),
        ("cgtb_layer_norm_backward", (7, d.ptr, d.ptr, d.ptr, 4, 32, 1e-5, d.ptr, d.ptr, d.ptr)),
        ("cgtb_dropout", (11, d.ptr, 32, 1.0, state.ptr, 0, d.ptr)),
        ("cgtb_dropout", (11, d.ptr, 32, -0.1, state.ptr, 0, d.ptr)),
        ("cgtb_dropout", (5, d.ptr, 32, 0.1, state.ptr, 0, d.ptr)),
        ("cgtb_dropout", (11, d.ptr, -32, 0.1, state.ptr, 0, d.ptr)),
        ("cgtb_quantize_rows", (d.ptr, -1, 32, c.ptr, s.ptr)), ("cgtb_quantize_rows", (d.ptr, 1, 16, off, s.ptr)),
        ("cgtb_int8_product", (c.ptr, s.ptr, c.ptr, s.ptr, None, 4, 4, 24, d.ptr)),
        ("cgtb_int8_product", (c.ptr, s.ptr, c.ptr, s.ptr, None, 4, 4, 131072, d.ptr)),
        ("cgtb_int8_product", (c.ptr, s.ptr, c.ptr, s.ptr, None, -4, 4, 32, d.ptr)),
        ("cgtb_int8_product", (off, s.ptr, c.ptr, s.ptr, None, 1, 1, 16, d.ptr)),
    ]
    for (name, args) in refused:
        assert getattr(L, name)(*args) != 0 and name in runtime.last_error(), (name, args)
    x = np.ones((2, 16), "f4")
    _same(_quantize(x), ref.quantize(x))


# ------------------------------------------------------------------------------------------------
# in compiled functions
# ------------------------------------------------------------------------------------------------
def _shared(a):
    return cgt.shared(a, fixed_shape_mask="all")


@pytest.mark.parametrize("precision", ["single", "double"])
def test_results_go_into_variables(rt, precision):
    """Forward and backward results kept in variables, through captured replays and for new inputs."""
    dt = "f4" if precision == "single" else "f8"
    with cgt.scoped_update_config(precision=precision):
        x, gain, bias, gy = [_shared(a) for a in _norm_inputs(50, 300, dt)]
        y = nn.layer_norm(x, gain, bias)
        news = [y] + core.pullback([y], [gy], [x, gain, bias])
        outs = [_shared(np.zeros(s, dt)) for s in ((50, 300), (50, 300), (300,), (300,))]
        f = cgt.function([], [], updates=list(zip(outs, news)))
    assert not any(getattr(i.op, "opname", "").startswith("cast") for i in f.eg.instrs if hasattr(i, "op"))     # nothing is copied
    for seed in (0, 0, 0, 0, 1, 2):
        vals = _norm_inputs(50, 300, dt, seed)
        for (v, a) in zip((x, gain, bias, gy), vals):
            v.op.set_value(a)
        f()
        bounds = ref.norm_bounds(*vals, 1e-5)
        wants = (ref.norm(*vals[:3], 1e-5)[0],) + tuple(ref.norm_gradients(vals[0], vals[1], vals[3], 1e-5))
        for (o, want, bound) in zip(outs, wants, bounds):
            assert (np.abs(o.op.get_value() - want) <= bound).all()


def test_a_gradient_that_replaces_what_it_was_computed_from(rt):
    """x := dx and gain := dgain: every result is formed from the old values."""
    vals = _norm_inputs(20, 100, "f4")
    x, gain, bias, gy = [_shared(a) for a in vals]
    y = nn.layer_norm(x, gain, bias)
    dx, dgain, dbias = core.pullback([y], [gy], [x, gain, bias])
    cgt.function([], [], updates=[(x, dx), (gain, dgain), (gy, y), (bias, dbias)])()
    bounds = ref.norm_bounds(*vals, 1e-5)
    wants = (ref.norm(*vals[:3], 1e-5)[0],) + tuple(ref.norm_gradients(vals[0], vals[1], vals[3], 1e-5))
    for (o, want, bound) in zip((gy, x, gain, bias), wants, bounds):
        assert (np.abs(o.op.get_value() - want) <= bound).all()


def test_every_step_drops_other_elements(rt):
    """The masks of a captured step follow the stream's step; two dropouts of one stream differ; forward and backward agree."""
    n = (70, 33)
    xv = np.random.RandomState(0).randn(*n).astype("f4")
    x = _shared(xv)
    stream = nn.RandomStream(77)
    a, b = nn.dropout(x, 0.4, stream), nn.dropout(x, 0.4, stream)
    dx = core.pullback([a], [x * 3.0], [x])[0]
    f = cgt.function([], [a, b, dx], updates=stream.updates())
    for step in range(6):
        got = f()
        wants = [ref.dropout(xv, 0.4, 77, step, 0), ref.dropout(xv, 0.4, 77, step, 1), ref.dropout(xv * 3, 0.4, 77, step, 0)]
        assert all(np.array_equal(g, w) for (g, w) in zip(got, wants)), step
    assert list(stream.state.op.get_value()) == [77, 6]
    g = cgt.function([], [a])            # without the update: the same elements in every call
    assert all(np.array_equal(g()[0], ref.dropout(xv, 0.4, 77, 6, 0)) for _ in range(4))


def _block(width, hidden, stream, seed):
    """Affine(rectify(Affine(layer_norm(x)))) with dropout in training, as a network's block."""
    np.random.seed(seed)
    layers = [nn.LayerNorm(width), nn.Affine(width, hidden, weight_init=nn.XavierNormal()), nn.Affine(hidden, width, weight_init=nn.XavierNormal())]

    def train(x):
        h = nn.rectify(layers[1](layers[0](x)))
        return x + nn.dropout(layers[2](nn.dropout(h, 0.2, stream)), 0.1, stream)

    def predict(x):
        return x + nn.Int8Affine(layers[2])(nn.rectify(nn.Int8Affine(layers[1])(layers[0](x))))
    return layers, train, predict


def _block_step(P, x, t, lr, seed, step):
    """The block's training step in 64 bits: loss, new parameters."""
    gain, bias, W1, b1, W2, b2 = P
    R = len(x)
    y, xh, rstd = ref.norm(x, gain, bias, 1e-5)
    z = y @ W1 + b1
    mask = z >= 0
    keep1 = ref.kept(z.size, 0.2, seed, step, 0).reshape(z.shape) / 0.8
    keep2 = ref.kept(x.size, 0.1, seed, step, 1).reshape(x.shape) / 0.9
    h = z * mask * keep1
    out = x + (h @ W2 + b2) * keep2
    g = 2 * (out - t) / R * keep2
    dh = g @ W2.T * keep1 * mask
    dy = dh @ W1.T
    grads = [(dy * xh).sum(0), dy.sum(0), y.T @ dh, dh.sum(0, keepdims=True), h.T @ g, g.sum(0, keepdims=True)]
    return ((out - t) ** 2).sum() / R, [p - lr * d for (p, d) in zip(P, grads)], out


@pytest.mark.parametrize("rows", [32, None])
def test_a_block_is_trained_and_predicts_in_8_bits(rt, rows):
    """Five steps against the formulas in 64 bits with the same masks, with a fixed and an open batch; then predictions in 8 bits
    against the trained float32 weights."""
    width, hidden, batch = 48, 120, 32
    stream = nn.RandomStream(5)
    layers, train, predict = _block(width, hidden, stream, 3)
    X, T = cgt.matrix("X", fixed_shape=(rows, width)), cgt.matrix("T", fixed_shape=(rows, width))
    loss = cgt.square(train(X) - T).sum() / float(batch)
    params = [layers[0].gain, layers[0].bias, layers[1].weight, layers[1].bias, layers[2].weight, layers[2].bias]
    f = cgt.function([X, T], [loss], updates=nn.sgd(loss, params, 0.02) + stream.updates())
    P = [p.op.get_value().astype("f8") for p in params]
    rs = np.random.RandomState(0)
    for step in range(5):
        x, t = rs.randn(batch, width).astype("f4"), rs.randn(batch, width).astype("f4")
        got = f(x, t)[0]
        want, P, _out = _block_step(P, x.astype("f8"), t.astype("f8"), 0.02, 5, step)
        # sums of up to 4000 float32 terms; a rectifier's argument next to 0 may change sides, which moves its gradient's terms by as little
        np.testing.assert_allclose(got, want, rtol=1e-5)
        for (p, w) in zip(params, P):
            np.testing.assert_allclose(p.op.get_value(), w, rtol=1e-4, atol=2e-5)
    # 8-bit rows and weights: every factor is off by at most half a code, 1 / 254 of its row's largest magnitude
    x = rs.randn(batch, width).astype("f4")
    q = cgt.function([X], [predict(X)])
    y, W1, W2 = ref.norm(x, *[p.astype("f8") for p in P[:2]], 1e-5)[0], P[2], P[4]
    z = np.maximum(y @ W1 + P[3], 0)
    exact = x + z @ W2 + P[5]

    def spread(a, W, e):   # bound on the error of a.W with a off by e
        half_a = np.abs(a).max(1, keepdims=True) / 254 + e
        half_w = np.abs(W).max(0) / 254
        return half_a * np.abs(W).sum(0) + (np.abs(a) + half_a).sum(1, keepdims=True) * half_w
    bound = spread(z, W2, spread(y, W1, 1e-6).max(1, keepdims=True) * 1.01) + 1e-4
    for _ in range(4):
        assert (np.abs(q(x)[0] - exact) <= bound).all()


def test_int8_affine_follows_numpy(rt):
    """The layer's result from the codes that numpy makes, for batches of several sizes through one function."""
    np.random.seed(1)
    layer = nn.Affine(70, 33, weight_init=nn.XavierNormal(), bias_init=nn.IIDGaussian())
    X = cgt.matrix("X", fixed_shape=(None, 70))
    f = cgt.function([X], [nn.Int8Affine(layer)(X)])
    b, sb = ref.quantize(layer.weight.op.get_value().T.copy())
    for rows in (1, 5, 5, 5, 5, 40, 200, 1):
        x = np.random.randn(rows, 70).astype("f4")
        want, bound = ref.product(*ref.quantize(x), b, sb, layer.bias.op.get_value()[0])
        assert (np.abs(f(x)[0] - want) <= bound).all()


def test_arguments_that_do_not_fit_are_errors(rt):
    x = cgt.matrix("x")
    g = _shared(np.ones(10, "f4"))
    f = cgt.function([x], [nn.layer_norm(x, g, g)])
    with pytest.raises(runtime.BackendError, match="one value for each"):
        f(np.ones((3, 11), "f4"))
    assert f(np.ones((3, 10), "f4"))[0].shape == (3, 10)
    codes, scales = nn.quantize_rows(x)
    w = _shared(np.ones((4, 32), "i1"))
    f = cgt.function([x], [nn.int8_product(codes, scales, w, _shared(np.ones(4, "f4")))])
    with pytest.raises(runtime.BackendError, match="rows of one length"):
        f(np.ones((3, 10), "f4"))
    assert f(np.ones((3, 20), "f4"))[0].shape == (3, 4)


def test_arrays_of_other_ranks(rt):
    rs = np.random.RandomState(0)
    v, t = rs.randn(24).astype("f4"), rs.randn(3, 4, 24).astype("f4")
    gain, bias = rs.randn(24).astype("f4"), rs.randn(24).astype("f4")
    a, b = cgt.vector("a"), cgt.tensor3("b")
    stream = nn.RandomStream(1)
    f = cgt.function([a, b], [nn.layer_norm(a, _shared(gain), _shared(bias)), nn.layer_norm(b, _shared(gain), _shared(bias)), nn.dropout(b, 0.5, stream)])
    ya, yb, d = f(v, t)
    for (got, x) in ((ya, v[None]), (yb, t.reshape(-1, 24))):
        assert (np.abs(got.reshape(x.shape) - ref.norm(x, gain, bias, 1e-5)[0]) <= ref.norm_bounds(x, gain, bias, None, 1e-5)).all()
    assert np.array_equal(d, ref.dropout(t, 0.5, 1, 0, 0))


def test_a_workspace_that_grew_is_not_replayed_at_its_old_place(rt):
    """A function with an open batch goes back to a shape whose captured graph used a smaller workspace: the graph is not
    launched again before it is captured anew, and all results are right."""
    with cgt.scoped_update_config(specialise_shapes=False):
        x, gain, bias = cgt.matrix("x", fixed_shape=(None, 300)), _shared(np.ones(300, "f4")), _shared(np.zeros(300, "f4"))
        y = nn.layer_norm(x, gain, bias)
        grads = core.pullback([y], [y * 2.0], [gain, bias])
        f = cgt.function([x], grads)
    wants = {}
    launches = []
    for rows in (400, 400, 400, 400, 9000, 400, 9000, 9000, 9000, 400, 400, 400, 400):
        v = np.random.RandomState(rows).randn(rows, 300).astype("f4")
        if rows not in wants:
            g = 2 * ref.norm(v, np.ones(300, "f4"), np.zeros(300, "f4"), 1e-5)[0]
            wants[rows] = [w for w in ref.norm_gradients(v, np.ones(300, "f4"), g, 1e-5)[1:]]
        for (got, want) in zip(f(v), wants[rows]):
            # sums of up to 9000 terms of either sign, each off by a few roundings
            np.testing.assert_allclose(got, want, rtol=1e-4, atol=9000 * 8 * 2.0 ** -24)
        launches.append(f.stats()["last_graph_launches"])
    assert launches[3] == 1 and launches[5] == 0 and launches[-1] == 1


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("R,C", [(9, 64), (40, 17), (5, 1001), (3, 9000)])
def test_quantize_rows_that_start_anywhere(rt, R, C, offset):
    x = _norm_inputs(R, C, "f4")[0]
    d = Dev(np.concatenate([np.zeros(offset, "f4"), x.reshape(-1), np.full(4, np.inf, "f4")]))
    Cp = -(-C // 16) * 16
    codes, scales = Dev(np.full(R * Cp + 16, 99, "i1")), Dev(np.full(R + 1, 7, "f4"))
    call("cgtb_quantize_rows", ctypes.c_void_p(d.w.data + 4 * offset), R, C, codes.ptr, scales.ptr)
    want = ref.quantize(x)
    flat = codes.get()
    assert np.array_equal(flat[:R * Cp].reshape(R, Cp), want[0]) and (flat[R * Cp:] == 99).all()
    assert np.array_equal(scales.get()[:R], want[1]) and scales.get()[R] == 7


@pytest.mark.parametrize("M,N", [(1, 33), (5, 20), (40, 50), (300, 129), (700, 257)])
def test_int8_product_writes_its_result_and_nothing_else(rt, M, N):
    """Results, scales and biases that start on any element; what lies around the result stays."""
    rs = np.random.RandomState(M)
    K = 144
    a, b = rs.randint(-128, 128, (M, K)).astype("i1"), rs.randint(-128, 128, (N, K)).astype("i1")
    sa, sb, bias = rs.rand(M).astype("f4"), rs.rand(N).astype("f4"), rs.randn(N).astype("f4")
    want, bound = ref.product(a, sa, b, sb, bias)

    def shifted(v, k):
        d = Dev(np.concatenate([np.zeros(k, "f4"), v]))
        return d, ctypes.c_void_p(d.w.data + 4 * k)
    (ka, pa), (kb, pb), (kc, pc) = shifted(sa, 1), shifted(sb, 3), shifted(bias, 2)
    da, db = Dev(a), Dev(b)
    for offset in (0, 1, 2):
        y = Dev(np.full(M * N + 8, 7, "f4"))
        call("cgtb_int8_product", da.ptr, pa, db.ptr, pb, pc, M, N, K, ctypes.c_void_p(y.w.data + 4 * offset))
        flat = y.get()
        assert (np.abs(flat[offset:offset + M * N].reshape(M, N) - want) <= bound).all()
        assert (flat[:offset] == 7).all() and (flat[offset + M * N:] == 7).all()


def test_gradients_of_a_norm_that_is_used_twice(rt):
    """One layer's gain and bias in two places: their gradients are the sums of both, in a step that is replayed."""
    rs = np.random.RandomState(2)
    R, C = 30, 77
    layer = nn.LayerNorm(C)
    layer.gain.op.set_value((1 + 0.2 * rs.randn(C)).astype("f4"))
    layer.bias.op.set_value(rs.randn(C).astype("f4"))
    x, t = cgt.matrix("x", fixed_shape=(R, C)), cgt.matrix("t", fixed_shape=(R, C))
    y = layer(cgt.tanh(layer(x)))
    loss = (y * t).sum()
    f = cgt.function([x, t], cgt.grad(loss, [layer.gain, layer.bias]))
    gain, bias = layer.gain.op.get_value().astype("f8"), layer.bias.op.get_value().astype("f8")
    for _ in range(4):
        xv, tv = rs.randn(R, C).astype("f4"), rs.randn(R, C).astype("f4")
        h1 = np.tanh(ref.norm(xv.astype("f8"), gain, bias, 1e-5)[0]).astype("f8")
        d2, g2, b2 = ref.norm_gradients(h1, gain, tv.astype("f8"), 1e-5)
        _d, g1, b1 = ref.norm_gradients(xv.astype("f8"), gain, (d2 * (1 - h1 * h1)).astype("f8"), 1e-5)
        for (got, want) in zip(f(xv, tv), (g1 + g2, b1 + b2)):
            # sums of 60 terms of order one, each through some thirty float32 roundings
            np.testing.assert_allclose(got, want.astype("f8"), atol=60 * 30 * 2.0 ** -24 * 3)


def test_one_variable_for_every_operand(rt):
    """The gradient of a leaf that is the row, the gain and the bias at once is the sum of the three."""
    v = (np.random.RandomState(0).rand(50) + 0.5).astype("f4")
    x = _shared(v)
    y = nn.layer_norm(x, x, x)
    f = cgt.function([], [y] + core.pullback([y], [x], [x]))
    want = ref.norm(v[None], v, v, 1e-5)[0][0]
    dx, dg, db = ref.norm_gradients(v[None], v, v[None], 1e-5)
    by, bx, bg, bb = ref.norm_bounds(v[None], v, v, v[None], 1e-5)
    # the two additions that join the three gradients round once each
    joined = bx[0] + bg + bb + 2 * ref.U["f4"] * (np.abs(dx[0]) + np.abs(dg) + np.abs(db))
    for _ in range(3):
        got = f()
        assert (np.abs(got[0] - want) <= by[0]).all()
        assert (np.abs(got[1] - (dx[0] + dg + db)) <= joined).all()


@pytest.mark.parametrize("which,rows", [("scales", 3), ("scales", 9), ("codes", 3), ("dx", 3), ("dgain", 3)])
def test_results_that_do_not_fit_their_variables_are_refused(rt, which, rows):
    """A result may be written straight into the variable that it updates: nothing is written when the sizes differ."""
    x, gain = _shared(np.ones((5, 16), "f4")), _shared(np.ones(16, "f4"))
    if which in ("scales", "codes"):
        result = nn.quantize_rows(x)[which == "scales"]
    else:
        result = core.pullback([nn.layer_norm(x, gain, gain * 2)], [x * 3], [x, gain])[which == "dgain"]
    shape = {"scales": (rows,), "codes": (rows, 16), "dx": (rows, 16), "dgain": (rows,)}[which]
    variable = cgt.shared(np.full(shape, 7, "i1" if which == "codes" else "f4"), fixed_shape_mask="all")
    with pytest.raises(Exception):
        cgt.function([], [], updates=[(variable, result)])()
    assert (variable.op.get_value() == 7).all()
    runtime.synchronize()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("R,C,dtype", [(1, 20484, "f4"), (3, 20482, "f4"), (67, 20500, "f4"), (130, 20496, "f4"), (5, 30001, "f4"), (3, 10242, "f8"),
                                       (65, 10244, "f8"), (7, 20481, "f8")])
def test_gradients_of_rows_that_no_block_holds(rt, R, C, dtype, offset):
    """Any number of them: what the kernels leave for the last one starts on 16 bytes."""
    x, gain, bias, gy = _norm_inputs(R, C, dtype)
    dx_, gy_ = [Dev(np.concatenate([np.zeros(offset, dtype), a.reshape(-1)])) for a in (x, gy)]
    g = Dev(gain)
    outs = [Dev(np.full(n + 4, 7, dtype)) for n in (R * C, C, C)]
    call("cgtb_layer_norm_backward", code(dtype), ctypes.c_void_p(dx_.w.data + offset * x.itemsize), g.ptr,
         ctypes.c_void_p(gy_.w.data + offset * x.itemsize), R, C, 1e-5, *[o.ptr for o in outs])
    for (o, want, bound) in zip(outs, ref.norm_gradients(x, gain, gy, 1e-5), ref.norm_bounds(x, gain, bias, gy, 1e-5)[1:]):
        flat = o.get()
        assert (np.abs(flat[:want.size].reshape(want.shape) - want) <= bound).all() and (flat[want.size:] == 7).all()


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("R,C", [(1, 4097), (300, 8193), (2, 8196), (41, 12289), (200, 16384), (3, 16385), (2, 20001), (90, 24580), (1, 32768), (3, 32769)])
def test_layer_norm_of_rows_that_blocks_share(rt, R, C, dtype):
    """Rows of two to eight blocks, at the sizes where their number changes, more rows than clusters and fewer."""
    test_layer_norm(rt, R, C, dtype)


def test_long_rows_are_the_same_in_every_call(rt):
    """Blocks that share a row add its sums in one order: no bit differs between calls, eager or replayed."""
    R, C = 40, 20001
    x, gain, bias, gy = [_shared(a) for a in _norm_inputs(R, C, "f4")]
    y = nn.layer_norm(x, gain, bias)
    f = cgt.function([], [y] + core.pullback([y], [gy], [x, gain, bias]))
    first = [a.copy() for a in f()]
    for _ in range(6):
        assert all(np.array_equal(a, b) for (a, b) in zip(f(), first))


def test_8_bit_layers_under_the_other_precision(rt):
    """Float32 variables in a function that is built and compiled in double precision: the same float32 results."""
    rs = np.random.RandomState(0)
    x, wv = rs.randn(6, 40).astype("f4"), rs.randn(9, 40).astype("f4")
    rows, w, sw = _shared(x), _shared(ref.quantize(wv)[0]), _shared(ref.quantize(wv)[1])
    with cgt.scoped_update_config(precision="double"):
        codes, scales = nn.quantize_rows(rows)
        f = cgt.function([], [nn.int8_product(codes, scales, w, sw)])
    want, bound = ref.product(*ref.quantize(x), *ref.quantize(wv), None)
    for _ in range(4):
        got = f()[0]
        assert got.dtype == np.float32 and (np.abs(got - want) <= bound).all()


IN_VAIN = [("forward", 2500, 9001, "f4"), ("forward", 2500, 5000, "f8"), ("backward", 400000, 17, "f4"), ("backward", 40000, 301, "f8"), ("backward", 10000, 2047, "f4"),
           ("backward", 3000, 3001, "f8"), ("backward", 2500, 9001, "f4"), ("backward", 2500, 9001, "f8"), ("backward", 7, 1001, "f4")]


@pytest.mark.parametrize("which,R,C,dtype", IN_VAIN)
def test_a_block_waits_in_vain_once(rt, which, R, C, dtype):
    """No copy arrives and no block is told anything: the kernels end by themselves after one limit, not one for each of a
    block's eight or more rows, the failure is reported, and the library stays usable."""
    L = runtime.lib()
    rs = np.random.RandomState(0)
    x, gy = rs.randn(R, C).astype(dtype), rs.randn(R, C).astype(dtype)
    gain, bias = rs.randn(C).astype(dtype), rs.randn(C).astype(dtype)
    dx, dgy, dg, db = Dev(x), Dev(gy), Dev(gain), Dev(bias)
    out, sums = Dev(np.full((R, C), 7, dtype)), [Dev(np.zeros(C, dtype)) for _ in range(2)]

    def run():
        if which == "forward":
            assert L.cgtb_layer_norm_forward(code(dtype), dx.ptr, R, C, dg.ptr, db.ptr, 1e-5, out.ptr) == 0
        else:
            assert L.cgtb_layer_norm_backward(code(dtype), dx.ptr, dg.ptr, dgy.ptr, R, C, 1e-5, out.ptr, *[s.ptr for s in sums]) == 0
        return L.cgtb_synchronize()
    cycles = 100_000_000                 # 0.05 s or a little more; a copy that is still awaited at the end costs three times 0.01 s
    runtime.check(L.cgtb_layer_norm_selftest_waits(cycles), "selftest")
    try:
        start = time.monotonic()
        failed = run()
        seconds = time.monotonic() - start
    finally:
        runtime.check(L.cgtb_layer_norm_selftest_waits(0), "selftest")
    assert failed and "code 9" in runtime.last_error()
    assert seconds < 0.25, seconds       # eight rows with a wait each: 0.4 s
    assert run() == 0
    got = out.get()
    some = slice(0, R, max(1, R // 50))
    if which == "forward":
        want, bound = ref.norm(x[some], gain, bias, 1e-5)[0], ref.norm_bounds(x[some], gain, bias, None, 1e-5)
    else:
        want, bound = ref.norm_gradients(x[some], gain, gy[some], 1e-5)[0], ref.norm_bounds(x[some], gain, bias, gy[some], 1e-5)[1]
    assert (np.abs(got[some] - want) <= bound).all()
    assert L.cgtb_layer_norm_selftest_waits(-1) != 0 and L.cgtb_layer_norm_selftest_waits(1 << 40) != 0


@pytest.mark.parametrize("R,C", [(6, 1000), (6, 9001)])
def test_what_is_said_of_a_wait_in_vain(rt, R, C):
    """The forward pass waits for other blocks only, the gradients of short rows for copies only: the text names both."""
    L = runtime.lib()
    x, gain, bias, gy = [Dev(a) for a in _norm_inputs(R, C + 1, "f4")]
    out, sums = Dev(np.zeros((R, C + 1), "f4")), [Dev(np.zeros(C + 1, "f4")) for _ in range(2)]
    runtime.check(L.cgtb_layer_norm_selftest_waits(100_000), "selftest")
    try:
        if C > 8192:
            assert L.cgtb_layer_norm_forward(code("f4"), x.ptr, R, C + 1, gain.ptr, bias.ptr, 1e-5, out.ptr) == 0
        else:
            assert L.cgtb_layer_norm_backward(code("f4"), x.ptr, gain.ptr, gy.ptr, R, C + 1, 1e-5, out.ptr, *[d.ptr for d in sums]) == 0
        failed = L.cgtb_synchronize()
    finally:
        runtime.check(L.cgtb_layer_norm_selftest_waits(0), "selftest")
    text = runtime.last_error()
    assert failed and "code 9" in text and "8-bit product" in text and "copy of a row or another block's sums" in text
    runtime.synchronize()


# ------------------------------------------------------------------------------------------------
# sums that are exact, so that a term that is lost or counted twice cannot hide behind the roundings of the others
# ------------------------------------------------------------------------------------------------
EXACT_COLS = [2, 3, 5, 8, 17, 33, 65, 100, 300, 1001, 1028, 2047, 4096, 4097, 8192, 8193, 8196, 9001, 12289, 16384, 16385, 20001, 24577, 28676, 32768, 32769]


def _columns(C, rs):
    """All columns of a short row; of a long one those where the parts of 2 to 8 blocks or a thread's share may begin or end, and others."""
    if C <= 1100:
        return np.arange(C)
    parts = [k * (-(-C // b // 4) * 4 if exact else -(-C // b)) for b in range(2, 9) for k in range(1, b) for exact in (False, True)]
    near = [p + d for p in parts + [0, C, 1024, 2048, 4096, 8192, 16384] for d in range(-4, 5)]
    return np.unique([c for c in near if 0 <= c < C] + list(rs.randint(0, C, 150)))


def _signs(R, C, zero):
    """Rows of +1 and -1 whose sum is 0; with an odd number of columns column `zero` of the row is 0."""
    x = np.tile(np.where(np.arange(C) % 2, -1.0, 1.0), (R, 1))
    if C % 2:
        for r in range(R):
            rest = np.arange(C) != zero[r]
            x[r, rest], x[r, zero[r]] = np.where(np.arange(C - 1) % 2, -1.0, 1.0), 0
    return x


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("C", EXACT_COLS)
def test_every_column_counts_once_in_the_statistics(rt, C, dtype):
    """One element of 1024 in a row of zeros, at every place: the result is sqrt(C - 1) there and -1 / sqrt(C - 1) elsewhere. The
    mean's sum is exact; the squares are positive terms, off by three roundings each and at most 64 additions one behind the
    other (16 or 33 of a thread, 10 of a block, 8 of a cluster); the root halves what the variance is off by: 45 roundings."""
    at = _columns(C, np.random.RandomState(C))
    x = np.zeros((len(at), C), dtype)
    x[np.arange(len(at)), at] = 1024
    want = np.full(x.shape, -1 / np.sqrt(C - 1.0))
    want[np.arange(len(at)), at] = np.sqrt(C - 1.0)
    y = _forward(x, np.ones(C, dtype), np.zeros(C, dtype), 0.0)
    assert (np.abs(y - want) <= 45 * ref.U[dtype] * np.abs(want)).all()


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("C", EXACT_COLS)
def test_every_column_counts_once_in_the_gradients_sums(rt, C, dtype):
    """Rows of +1 and -1 and a gradient that is 1024 in one place, every one in its row: all sums have one term or are whole
    numbers, so what is left are the roundings of the formula, below 40 of the mean's term and 16 of the element's own."""
    at = _columns(C, np.random.RandomState(C))
    R = len(at)
    x, own = _signs(R, C, np.where(at < C // 2, C - 1, 0)), (np.arange(R), at)
    gain = 2.0 ** (np.arange(C) % 3)
    gy = np.zeros((R, C))
    gy[own] = 1024
    rstd = np.sqrt(C / (C - C % 2))
    d = 1024 * gain[at][:, None]
    want = -rstd * d / C * (1 + x * x[own][:, None] * rstd ** 2)
    want[own] += rstd * d[:, 0]
    bound = 40 * ref.U[dtype] * rstd * d / C + np.zeros((R, C))
    bound[own] += 16 * ref.U[dtype] * rstd * d[:, 0]
    dx = _backward(x.astype(dtype), gain.astype(dtype), gy.astype(dtype), 0.0)[0]
    assert (np.abs(dx - want) <= bound).all()


@pytest.mark.parametrize("dtype", ["f4", "f8"])
@pytest.mark.parametrize("R,C", [(7, 100), (64, 256), (3000, 4), (5001, 17), (4099, 33), (2000, 64), (1025, 300), (1000, 1001), (130, 2048), (600, 4096), (201, 4097),
                                 (200, 8192), (300, 8193), (333, 12289), (90, 24580), (3, 32769), (150, 33000)])
def test_every_row_counts_once_in_the_columns_sums(rt, R, C, dtype):
    """Every row's gradient has one term, a power of two, in one column, each column's terms are different powers: the bias's gradient
    is exact, and the gain's is off by at most 20 roundings, where a row that is missing or counted twice is 1 / 4095 or more."""
    x = _signs(R, C, np.full(R, C - 1))
    xh = x[0] * np.sqrt(C / (C - C % 2))
    for first in range(0, R, 12 * C):
        rows = np.arange(first, min(R, first + 12 * C))
        gy = np.zeros((R, C))
        gy[rows, rows % C] = 2.0 ** ((rows - first) // C)
        want = gy.sum(0)
        _dx, dgain, dbias = _backward(x.astype(dtype), np.ones(C, dtype), gy.astype(dtype), 0.0)
        assert np.array_equal(dbias, want)
        assert (np.abs(dgain - want * xh) <= 20 * ref.U[dtype] * np.abs(want * xh)).all()


@pytest.mark.parametrize("C", [2, 17, 65, 300, 1001, 8192, 8193, 16384, 16385, 20480, 20481, 30001])
def test_every_column_counts_in_a_rows_scale(rt, C):
    """Rows of ones with one -254, at every place: scale 2, codes of a half that is rounded to 0."""
    at = _columns(C, np.random.RandomState(C))
    own = (np.arange(len(at)), at)
    x, codes = np.ones((len(at), C), "f4"), np.zeros((len(at), -(-C // 16) * 16), "i1")
    x[own], codes[own] = -254, -127
    _same(_quantize(x), (codes, np.full(len(at), 2, "f4")))


def test_epsilons_at_the_ends_of_the_type(rt):
    """Rows of equal values are the bias down to the smallest epsilon that is taken; smaller ones are refused."""
    L = runtime.lib()
    for (dtype, small, large) in (("f4", 1.2e-38, 3e38), ("f8", 2.3e-308, 1e308)):
        x, bias = np.full((3, 40), 5, dtype), np.arange(40).astype(dtype)
        for eps in (small, large):
            assert np.array_equal(_forward(x, np.ones(40, dtype), bias, eps), np.tile(bias, (3, 1)))
        d = Dev(x)
        for eps in (small / 10, 1e-320, large * 10):
            assert L.cgtb_layer_norm_forward(code(dtype), d.ptr, 3, 40, d.ptr, d.ptr, eps, d.ptr) != 0 and "epsilon" in runtime.last_error()
            assert L.cgtb_layer_norm_backward(code(dtype), d.ptr, d.ptr, d.ptr, 3, 40, eps, d.ptr, d.ptr, d.ptr) != 0
        assert np.array_equal(d.get(), x)
