"""Dropout from a counter-based generator. The reference draws a random array and compares it (cgt/nn.py); here an element's
fate is a function of (seed, step, place), so no mask is stored and the backward pass forms it again."""
import ctypes

import numpy as np

from .. import core


class Dropout(core.Op):
    """(x, state int64 [2]) -> x / (1 - p) where the generator keeps an element, 0 elsewhere."""
    available_impls = ("native_gpu",)

    def __init__(self, p, site):
        self.p = float(p)
        self.site = int(site)

    def get_diff(self, n):
        return [True, False]

    def get_native_compile_info(self, input_types, devtype):
        return core.NativeCompileInfo(None, prebuilt="cgtb_op_dropout",
                                      closure_triples=[("p", ctypes.c_double, self.p), ("site", ctypes.c_int, self.site)])

    def shp_apply(self, inputs):
        return core.cgt.shape(inputs[0])

    def typ_apply(self, input_types):
        x, state = input_types
        if x.ndim < 1 or core.dtype_kind(x.dtype) != "f":
            raise ValueError("dropout takes an array of floating-point numbers with at least one axis, got %s" % x)
        assert state == core.TensorType("i8", 1)
        return x

    def pullback(self, inputs, output, gout):
        return [core.Result(self, [gout, inputs[1]]), None]

    def __repr__(self):
        return "Dropout{%r,%d}" % (self.p, self.site)


class RandomStream(object):
    """A generator's state, seed and step, as a shared variable on the GPU. Every ``dropout`` that is built with the stream
    drops elements of its own; all of them drop other elements in the next step:

        stream = nn.RandomStream(seed)
        h = nn.dropout(h, 0.5, stream)
        f = cgt.function([X, y], [loss], updates=nn.sgd(loss, params, 0.1) + stream.updates())

    Without ``stream.updates()`` every call drops the same elements. The masks depend on the seed, the step (the call's
    number, modulo 2^32), the order in which the dropouts were built and the element's place, on nothing else; ranks that train
    together need different seeds to drop different elements."""

    def __init__(self, seed):
        self.state = core.cgt.shared(np.array([seed, 0], "i8"), name="random_stream", fixed_shape_mask="all")
        self._sites = 0

    def new_site(self):
        self._sites += 1
        return self._sites - 1

    def updates(self):
        return [(self.state, self.state + core.cgt.constant(np.array([0, 1], "i8")))]


def dropout(x, p, stream):
    """x with a share p of its elements set to 0 and the others divided by 1 - p, 0 <= p < 1, in training. The elements are
    drawn from `stream`, a RandomStream; p = 0 is x itself, what a network for predictions is built with. A dropped element is
    0 and passes no gradient, whatever its value, an infinity or a NaN among them."""
    if not 0 <= p < 1:
        raise ValueError("the probability of dropping an element has to be in [0, 1), got %s" % (p,))
    if not isinstance(stream, RandomStream):
        raise ValueError("dropout takes its random numbers from a RandomStream, got %s" % type(stream))
    x = core.as_node(x)
    return core.Result(Dropout(p, stream.new_site()), [x, stream.state]) if p > 0 else x
