"""Layer norm, dropout, 8-bit rows and 8-bit products without a GPU: the generator's published answers, refusals when a
graph is built, and which memory a step's results go to."""
import re
import shutil
import subprocess

import numpy as np
import pytest

import cgt_b200 as cgt
from cgt_b200 import build
from cgt_b200 import compilation, core, nn
from cgt_b200.nn_ops import dropout as dropout_ops
from cgt_b200.nn_ops import int8 as int8_ops
from cgt_b200.nn_ops import layer_norm as norm_ops
from tests import block_ops as ref
from tests.host_run import HostRun


def test_the_generator_gives_the_published_answers():
    """Known answers of Philox4x32-10 from its authors: counter and key all zeros, and all ones."""
    assert [int(w) for w in ref.philox([0], 0, 0, 0)[0]] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFFFFFFFFFF
    assert [int(w) for w in ref.philox([np.uint64(ones)], ones, 0xFFFFFFFF, ones)[0]] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_the_share_of_dropped_elements():
    n = 1 << 18
    for (p, seed, step, site) in ((0.1, 0, 0, 0), (0.5, 3, 100, 2), (0.85, -1, 7, 5)):
        # a binomial count is within five of its standard deviations, sqrt(p (1 - p) n), but for one time in a million
        assert abs((~ref.kept(n, p, seed, step, site)).sum() - p * n) < 5 * np.sqrt(p * (1 - p) * n)


def test_host_quantization_is_the_operators():
    rs = np.random.RandomState(0)
    x = rs.randn(30, 37).astype("f4")
    x[3], x[4, 5], x[5, 6], x[6] = 0, np.nan, np.inf, rs.randint(-254, 255, 37) / 2.0
    x[6, 0] = 127
    for (a, b) in zip(int8_ops._quantize(x), ref.quantize(x)):
        assert a.dtype == b.dtype and np.array_equal(a, b, equal_nan=True)


def test_refusals():
    x, v, i = cgt.matrix("x"), cgt.vector("v"), cgt.matrix("i", dtype="i8")
    stream = nn.RandomStream(0)
    for build in (lambda: nn.layer_norm(i, v, v), lambda: nn.layer_norm(x, x, v), lambda: nn.layer_norm(x, v, cgt.vector("k", dtype="i8")),
                  lambda: nn.layer_norm(cgt.scalar("s"), v, v), lambda: nn.layer_norm(x, v, v, epsilon=-1.0), lambda: nn.layer_norm(x, v, v, epsilon=float("nan")),
                  lambda: nn.layer_norm(x, v, v, epsilon=float("inf")), lambda: nn.dropout(x, 1.0, stream), lambda: nn.dropout(x, -0.1, stream),
                  lambda: nn.dropout(x, float("nan"), stream), lambda: nn.dropout(x, 0.5, 7), lambda: nn.dropout(i, 0.5, stream),
                  lambda: nn.dropout(cgt.scalar("s"), 0.5, stream), lambda: nn.quantize_rows(v), lambda: nn.quantize_rows(i),
                  lambda: nn.int8_product(x, v, x, v), lambda: nn.int8_product(cgt.matrix("c", dtype="i1"), v, cgt.matrix("d", dtype="i1"), x)):
        with pytest.raises(ValueError):
            build()
    with cgt.scoped_update_config(precision="double"):
        with pytest.raises(ValueError):
            nn.quantize_rows(cgt.matrix("x"))
        with pytest.raises(ValueError):
            nn.Int8Affine(nn.Affine(3, 4))
    with pytest.raises(ValueError):
        nn.Int8Affine(nn.Affine(131072, 1))
    assert nn.dropout(x, 0.0, stream) is x


def test_no_gradient_where_there_is_none():
    x = cgt.shared(np.ones((3, 16), "f4"), fixed_shape_mask="all")
    codes, scales = nn.quantize_rows(x)
    with pytest.raises(Exception):
        cgt.grad(scales.sum(), [x])


def test_every_dropout_of_a_stream_has_elements_of_its_own():
    x = cgt.matrix("x", fixed_shape=(4, 4))
    stream = nn.RandomStream(0)
    y = nn.dropout(x, 0.5, stream) + nn.dropout(x, 0.5, stream)
    eg = compilation.execution_graph([x], [y], [], [])[0]
    assert sorted(i.op.site for i in eg.instrs if isinstance(getattr(i, "op", None), dropout_ops.Dropout)) == [0, 1]


# ------------------------------------------------------------------------------------------------
# results that are variables: the compiled instruction list, executed on numpy arrays
# ------------------------------------------------------------------------------------------------
class _Run(HostRun):
    def _into(self, ins, reads, write):
        op = ins.op
        writes = write if isinstance(write, tuple) else (write,)
        if isinstance(op, norm_ops.LayerNorm):
            results = [ref.norm(*reads, op.epsilon)[0]]
        elif isinstance(op, norm_ops.LayerNormBackward):
            results = ref.norm_gradients(*reads, op.epsilon)
        elif isinstance(op, int8_ops.QuantizeRows):
            results = ref.quantize(reads[0])
        elif isinstance(op, dropout_ops.Dropout):
            results = [ref.dropout(reads[0], op.p, int(reads[1][0]), int(reads[1][1]), op.site)]
        else:
            return HostRun._into(self, ins, reads, write)
        for out in writes:
            assert not any(np.shares_memory(r, out) for r in reads), "%r reads the memory that it overwrites" % (op,)
        results = [np.array(r, copy=True) for r in results]
        for (out, r) in zip(writes, results):
            assert out.shape == r.shape
            out[...] = r


def _var(rs, *shape):
    return cgt.shared(rs.randn(*shape).astype("f4"), fixed_shape_mask="all")


def _copies(run):
    return sum(isinstance(op, core.ElwiseUnary) and op.opname.startswith("cast_to_") for op in run.ops())


def _case():
    rs = np.random.RandomState(0)
    x, gain, bias, gy = _var(rs, 6, 20), _var(rs, 20), _var(rs, 20), _var(rs, 6, 20)
    y = nn.layer_norm(x, gain, bias)
    old = [v.op.get_value() for v in (x, gain, bias, gy)]
    wants = [ref.norm(*old[:3], 1e-5)[0]] + list(ref.norm_gradients(old[0], old[1], old[3], 1e-5))
    return rs, (x, gain, bias, gy), [y] + core.pullback([y], [gy], [x, gain, bias]), [w.astype("f4") for w in wants]


def test_several_results_go_into_their_variables():
    rs, _inputs, news, wants = _case()
    outs = [_var(rs, *w.shape) for w in wants]
    run = _Run([], [], list(zip(outs, news)))
    assert _copies(run) == 0
    run()
    assert all(np.array_equal(run.value(o), w) for (o, w) in zip(outs, wants))


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (1, 0, 3, 2), (3, 2, 1, 0)])
def test_results_that_replace_operands(order):
    """x, gain, bias and gy get, in some order, the results that are computed from them."""
    _rs, (x, gain, bias, gy), news, wants = _case()
    targets = dict(zip(range(4), ((gy, 0), (x, 1), (gain, 2), (bias, 3))))
    pairs = [targets[k] for k in order]
    run = _Run([], [], [(v, news[i]) for (v, i) in pairs])
    run()
    assert all(np.array_equal(run.value(v), wants[i]) for (v, i) in pairs)


def test_a_variable_that_is_still_read_after_the_operation():
    """A reader of the old value that the order puts behind the operation: the operation may not write the variable."""
    rs, (x, gain, bias, gy), news, wants = _case()
    keep = _var(rs, 6, 20)
    old = keep.op.get_value()
    later = cgt.tanh(keep * news[1])       # needs dx and the old value
    out = _var(rs, 6, 20)
    run = _Run([], [later], [(keep, news[1]), (out, keep + 1.0)])
    for _ in range(2):
        got = run()[0]
        np.testing.assert_allclose(got, np.tanh(old * wants[1]), rtol=1e-6)
        np.testing.assert_allclose(run.value(out), old + 1, rtol=1e-6)
        assert np.array_equal(run.value(keep), wants[1])
        old = wants[1]


def test_one_result_for_two_variables_and_for_the_caller():
    rs, _inputs, news, wants = _case()
    a, b = _var(rs, 20), _var(rs, 20)
    run = _Run([], [news[2], news[2] * 2.0], [(a, news[2]), (b, news[2])])
    got = run()
    assert np.array_equal(run.value(a), wants[2]) and np.array_equal(run.value(b), wants[2])
    assert np.array_equal(got[0], wants[2]) and np.array_equal(got[1], 2 * wants[2])


def test_a_result_goes_into_no_variable_of_another_type():
    """scales (float32) into an int64 variable: copied, as before."""
    x = cgt.shared(np.ones((5, 16), "f4"), fixed_shape_mask="all")
    v = cgt.shared(np.zeros(5, "i8"), fixed_shape_mask="all")
    eg = compilation.execution_graph([], [], [(v, nn.quantize_rows(x)[1])], [])[0]
    assert any(getattr(getattr(i, "op", None), "opname", "").startswith("cast_to_") for i in eg.instrs)


def test_variables_that_nothing_reads():
    """A variable that is only written, from a chain, a product and a copy."""
    rs = np.random.RandomState(0)
    a, b = _var(rs, 8, 8), _var(rs, 8, 8)
    outs = [_var(rs, 8, 8) for _ in range(3)]
    run = HostRun([], [], [(outs[0], cgt.tanh(a + b)), (outs[1], a.dot(b)), (outs[2], a.reshape([8, 8]))])
    run()
    (av, bv) = (a.op.get_value(), b.op.get_value())
    np.testing.assert_allclose(run.value(outs[0]), np.tanh(av + bv), rtol=1e-5)
    np.testing.assert_allclose(run.value(outs[1]), av @ bv, rtol=1e-4, atol=1e-5)
    assert np.array_equal(run.value(outs[2]), av)


def test_dropout_in_a_step_on_the_host():
    rs = np.random.RandomState(0)
    x = _var(rs, 10, 7)
    old = x.op.get_value()
    stream = nn.RandomStream(9)
    y = nn.dropout(x, 0.3, stream)
    run = _Run([], [y], [(x, nn.dropout(y, 0.5, stream))] + stream.updates())
    for step in range(3):
        got = run()[0]
        want = ref.dropout(old, 0.3, 9, step, 0)
        assert np.array_equal(got, want)
        old = ref.dropout(want, 0.5, 9, step, 1)
        assert np.array_equal(run.value(x), old)


def test_an_extent_that_is_computed_from_an_open_one():
    x = cgt.matrix("x")
    run = _Run([x], list(nn.quantize_rows(x)))
    for shape in ((3, 20), (5, 16), (2, 1)):
        v = np.random.RandomState(0).randn(*shape).astype("f4")
        assert all(np.array_equal(a, b) for (a, b) in zip(run(v), ref.quantize(v)))


def test_a_checkpoint_holds_the_streams_state():
    x = cgt.matrix("x", fixed_shape=(4, 4))
    stream, norm = nn.RandomStream(3), nn.LayerNorm(4)
    loss = cgt.square(nn.dropout(norm(x), 0.5, stream)).sum()
    updates = nn.sgd(loss, nn.get_parameters(loss), 0.1) + stream.updates()
    held = cgt.state_variables(updates, [loss], nn.get_parameters(loss))
    assert stream.state in held and norm.gain in held and norm.bias in held and len(nn.get_parameters(loss)) == 2


def test_layers_parameters():
    layer = nn.LayerNorm(6, name="n")
    assert np.array_equal(layer.gain.op.get_value(), np.ones(6)) and np.array_equal(layer.bias.op.get_value(), np.zeros(6))
    np.random.seed(0)
    affine = nn.Affine(5, 3, weight_init=nn.XavierNormal(), bias_init=nn.IIDGaussian())
    q = nn.Int8Affine(affine)
    codes, scales = ref.quantize(affine.weight.op.get_value().T.copy())
    assert np.array_equal(q.codes.op.get_value(), codes) and np.array_equal(q.scales.op.get_value(), scales)
    assert np.array_equal(q.bias.op.get_value(), affine.bias.op.get_value()[0]) and q.codes.op.get_value().dtype == np.int8
    assert not nn.get_parameters(q(cgt.matrix("x")).sum())       # nothing to train


def test_gradients_that_do_not_exist_are_refused_beside_others():
    """Another way from the loss to the variable does not hide the one that has no gradient."""
    x = cgt.shared(np.ones((3, 32), "f4"), fixed_shape_mask="all")
    layer = nn.LayerNorm(32)
    (dx,) = core.pullback([layer(x)], [x], [x])
    affine = nn.Affine(32, 32)
    (codes, scales) = nn.quantize_rows(x)
    for loss in (cgt.square(dx).sum() + x.sum(), (nn.Int8Affine(affine)(x) + x).sum(), scales.sum() + x.sum(),
                 nn.int8_product(codes, scales, codes, scales).sum() + x.sum()):
        with pytest.raises(core.NonDifferentiable):
            cgt.grad(loss, [x])
    assert len(cgt.grad(nn.Int8Affine(affine)(x).sum() + affine(x).sum(), [affine.weight])) == 1      # x is not asked for


def test_the_longest_layer_in_8_bits():
    """131056 inputs are the longest row of codes that a product takes; one more is padded to 131072, which none does."""
    assert nn.Int8Affine(nn.Affine(131056, 1)).codes.op.get_value().shape == (1, 131056)
    for inputs in (131057, 131071):
        with pytest.raises(ValueError, match="up to 131056 inputs"):
            nn.Int8Affine(nn.Affine(inputs, 1))


def test_8_bit_results_are_float32_in_every_precision():
    """Variables of one precision in a graph that is built or compiled under the other: the kernels know float32 only."""
    x, w = cgt.shared(np.ones((3, 20), "f4"), fixed_shape_mask="all"), cgt.shared(np.ones((4, 32), "i1"), fixed_shape_mask="all")
    s = cgt.shared(np.ones(4, "f4"), fixed_shape_mask="all")
    with cgt.scoped_update_config(precision="double"):
        codes, scales = nn.quantize_rows(x)
        y = nn.int8_product(codes, scales, w, s)
        assert scales.dtype == "f4" and y.dtype == "f4"
        eg = compilation.execution_graph([], [y], [], [])[0]
    assert all(i.dtype[0] != "f" or i.dtype == "f4" for i in eg.instrs if isinstance(i, compilation.Alloc))


def _norm_kernels(C, kind, aligned):
    """The layer norm kernels that may be launched for rows of C elements of `kind`, which start on 16-byte boundaries or not."""
    size = {"float": 4, "double": 8}[kind]
    starts = aligned and C * size % 16 == 0
    names = set()

    def team(elements, most):
        return next((t for t in (1 << k for k in range(11)) if t <= most and C <= t * elements), None)
    E = 32 // size
    t = team(E, 1024)
    if t:
        E = E if starts or t == 1 or C > t * (E * 3 // 4) else E * 3 // 4
        vec = 16 // size if starts else 1
        names.add("norm_forward_kernel<%s, %d, %d, %d, false>" % (kind, vec, E // vec, t))
    elif C <= 256 * (64 // size) * 8:
        vec = 16 // size if starts else 1
        names.add("norm_forward_kernel<%s, %d, %d, 256, true>" % (kind, vec, 64 // size // vec))
    else:
        names.add("norm_forward_long_kernel<%s>" % kind)
    wide = starts and (C <= 1024 or (size == 4 and C > 4096))
    few = C <= 16 or (size == 8 and wide)
    E, vec = (32 if few else 64) // size, 16 // size if wide else 1
    t = team(E, 256 if few else 512)
    if t:
        names.update("norm_backward_kernel<%s, %d, %d, %d, %s, false>" % (kind, vec, E // vec, t, one) for one in ("false", "true"))
    elif C <= 256 * (64 // size) * 8:
        large, small = -(-C // (512 * (64 // size))), -(-C // (256 * (64 // size)))
        names.add("norm_backward_kernel<%s, 1, %d, %d, false, true>" % (kind, 64 // size, 512 if small == 2 * large else 256))
    else:
        names.update(("norm_backward_long_kernel<%s>" % kind, "norm_columns_kernel<%s>" % kind))
    names.add("norm_fold_kernel<%s, %d>" % (kind, 16 // size if 2 * C * size % 16 == 0 else 1))
    return names


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs nm")
def test_every_layer_norm_kernel_can_be_launched():
    """The library holds the kernels that some rows lead to, and no others."""
    built = subprocess.run(["nm", "-C", build.LIB], capture_output=True, text=True, check=True).stdout
    built = set(re.findall(r"\bnorm_\w+_kernel<[\w, ]+>", built))
    reached = set()
    for C in list(range(1, 2100)) + [2 ** k + d for k in range(11, 17) for d in (-1, 0, 1, 4)] + [12288, 12289, 24576, 24577, 24580]:
        for kind in ("float", "double"):
            for aligned in (False, True):
                reached |= _norm_kernels(C, kind, aligned)
    assert built == reached


def test_epsilons_that_the_type_does_not_hold():
    """They would be rounded to 0, which makes rows of equal values NaN, or to infinity."""
    x, v = cgt.matrix("x"), cgt.vector("v")
    for epsilon in (1e-60, 1e-39, 1e39):
        with pytest.raises(ValueError, match="normal number of type f4"):
            nn.layer_norm(x, v, v, epsilon=epsilon)
    for epsilon in (0.0, 1.2e-38, 3e38):
        nn.layer_norm(x, v, v, epsilon=epsilon)
    with cgt.scoped_update_config(precision="double"):
        x, v = cgt.matrix("x"), cgt.vector("v")
        nn.layer_norm(x, v, v, epsilon=1e-60)
        with pytest.raises(ValueError, match="normal number of type f8"):
            nn.layer_norm(x, v, v, epsilon=1e-310)
