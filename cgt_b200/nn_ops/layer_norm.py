"""Layer norm over an array's last axis, with its gradients. Not in the reference, whose only norm is cross_channel_lrn."""
import ctypes

import numpy as np

from .. import core


def _check(name, x, columns):
    if x.ndim < 1 or core.dtype_kind(x.dtype) != "f":
        raise ValueError("%s takes an array of floating-point numbers with at least one axis, got %s" % (name, x))
    for t in columns:
        if t.ndim != 1 or t.dtype != x.dtype:
            raise ValueError("%s takes gain and bias as vectors of type %s, got %s" % (name, x.dtype, t))


class LayerNorm(core.Op):
    """(x [..., C], gain [C], bias [C]) -> (x - m) / sqrt(v + epsilon) * gain + bias, m and v the mean and the variance of
    each row along the last axis."""
    available_impls = ("native_gpu",)

    def __init__(self, epsilon):
        self.epsilon = float(epsilon)
        if not 0 <= self.epsilon < float("inf"):
            raise ValueError("epsilon has to be a finite number that is not negative, got %s" % epsilon)

    def get_native_compile_info(self, input_types, devtype):
        return core.NativeCompileInfo(None, prebuilt="cgtb_op_layer_norm_forward", closure_triples=[("epsilon", ctypes.c_double, self.epsilon)])

    def shp_apply(self, inputs):
        return core.cgt.shape(inputs[0])

    def typ_apply(self, input_types):
        _check("layer_norm", input_types[0], input_types[1:])
        info = np.finfo(input_types[0].dtype)
        if self.epsilon and not float(info.tiny) <= self.epsilon <= float(info.max):
            raise ValueError("epsilon has to be 0 or a normal number of type %s, got %s" % (input_types[0].dtype, self.epsilon))
        return input_types[0]

    def pullback(self, inputs, output, gout):
        x, gain, _bias = inputs
        return core.unpack(core.Result(LayerNormBackward(self.epsilon), [x, gain, gout]))

    def __repr__(self):
        return "LayerNorm{%r}" % self.epsilon


class LayerNormBackward(core.Op):
    """(x, gain, gradient of the result) -> gradients of x, gain and bias, from one pass over x and the gradient."""
    available_impls = ("native_gpu",)
    results_in_variables = True

    def __init__(self, epsilon):
        self.epsilon = epsilon

    def get_native_compile_info(self, input_types, devtype):
        return core.NativeCompileInfo(None, prebuilt="cgtb_op_layer_norm_backward", closure_triples=[("epsilon", ctypes.c_double, self.epsilon)])

    def shp_apply(self, inputs):
        cgt = core.cgt
        return (cgt.shape(inputs[0]), cgt.shape(inputs[1]), cgt.shape(inputs[1]))

    def typ_apply(self, input_types):
        return core.TupleType(input_types[0], input_types[1], input_types[1])

    def pullback(self, inputs, output, gout):
        raise core.NonDifferentiable("layer_norm has first gradients only")

    def __repr__(self):
        return "LayerNormBackward{%r}" % self.epsilon


def layer_norm(x, gain, bias, epsilon=1e-5):
    """x with every row along its last axis brought to mean 0 and variance 1, then scaled and shifted by the vectors `gain`
    and `bias`, which have one value per column. A row of equal values gives `bias` (epsilon 0 makes it NaN); any other epsilon
    is a normal number of x's type, in float32 1.2e-38 or more. Gradients of gradients are refused."""
    return core.Result(LayerNorm(epsilon), [x, gain, bias])
