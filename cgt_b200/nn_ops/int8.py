"""Products in 8-bit integers for predictions: rows with a scale each, and their product with weights that have a scale per
output channel. Not in the reference."""
import ctypes

import numpy as np

from .. import core

PAD = 16               # rows of codes are a multiple of this long, so that every row starts on a 16-byte boundary
MAX_CODES = 131072     # a row, with its padding, has fewer: the sums are 32-bit integers


def _padded(columns):
    return -(-columns // PAD) * PAD


def _kinds(types):
    """(element type, rank) of each; a TensorType that is made from "f4" has the configured precision."""
    return [(t.dtype, t.ndim) for t in types]


def _float32(ndim):
    """The type of a float32 array, whatever the configured precision: the kernels write nothing else."""
    t = core.TensorType("f4", ndim)
    t.dtype = "f4"
    return t


class QuantizeRows(core.Op):
    """(x float32 [R, C]) -> codes int8 [R, C up to a multiple of 16] and scales float32 [R]."""
    available_impls = ("native_gpu",)
    results_in_variables = True

    def get_native_compile_info(self, input_types, devtype):
        return core.NativeCompileInfo(None, prebuilt="cgtb_op_quantize_rows", closure_triples=[])

    def shp_apply(self, inputs):
        cgt = core.cgt
        rows, cols = cgt.shape(inputs[0])
        return ([rows, cgt.ceil_divide(cols, PAD) * PAD], [rows])

    def typ_apply(self, input_types):
        if _kinds(input_types) != [("f4", 2)]:
            raise ValueError("quantize_rows takes a float32 matrix, got %s" % input_types[0])
        return core.TupleType(core.TensorType("i1", 2), _float32(1))

    def pullback(self, inputs, output, gout):
        raise core.NonDifferentiable("quantize_rows has no gradient")


class Int8Product(core.Op):
    """(codes [M, K], scales [M], weight codes [N, K], weight scales [N] (, bias [N])) -> float32 [M, N]."""
    available_impls = ("native_gpu",)

    def get_native_compile_info(self, input_types, devtype):
        return core.NativeCompileInfo(None, prebuilt="cgtb_op_int8_product",
                                      closure_triples=[("has_bias", ctypes.c_int, int(len(input_types) == 5))])

    def shp_apply(self, inputs):
        return [core.cgt.size(inputs[0], 0), core.cgt.size(inputs[2], 0)]

    def typ_apply(self, input_types):
        want = [("i1", 2), ("f4", 1)] * 2 + [("f4", 1)]
        if _kinds(input_types) != want[:len(input_types)]:
            raise ValueError("int8_product takes int8 matrices and float32 vectors, got %s" % (input_types,))
        return _float32(2)

    def pullback(self, inputs, output, gout):
        raise core.NonDifferentiable("int8_product has no gradient")


def quantize_rows(x):
    """(codes, scales) of a float32 matrix: x[r, c] is about codes[r, c] * scales[r], scales[r] the row's largest magnitude
    over 127, codes whole numbers from -127 to 127, rounded to nearest with ties to even. Rows of codes are padded with zeros
    to a multiple of 16. A row of zeros has scale 0; one with an infinity or a NaN has scale NaN and codes 0."""
    return tuple(core.unpack(core.Result(QuantizeRows(), [x])))


def int8_product(codes, scales, weight_codes, weight_scales, bias=None):
    """codes.dot(weight_codes.T), exact, times the scale of the row and that of the output channel, plus `bias`: float32
    [rows, channels]. Both matrices of codes as ``quantize_rows`` returns them; rows of up to 131056 codes."""
    return core.Result(Int8Product(), [codes, scales, weight_codes, weight_scales] + ([] if bias is None else [bias]))


class Int8Affine(object):
    """x.dot(W) + b of a trained ``Affine`` layer in 8-bit integers, for predictions: the weights are quantized once, with a
    scale per output channel, the rows of x in every call. The layer holds a quarter of the weights' bytes; it follows no
    later change of the ``Affine`` layer, and has no gradient."""

    def __init__(self, affine):
        weight = affine.weight.op.get_value()
        if weight.dtype != np.float32:
            raise ValueError("Int8Affine takes a float32 layer, got %s" % weight.dtype)
        if _padded(len(weight)) >= MAX_CODES:
            raise ValueError("Int8Affine takes a layer of up to %d inputs, got %d" % (MAX_CODES - PAD, len(weight)))
        codes, scales = _quantize(weight.T)
        shared = core.cgt.shared
        self.codes = shared(codes, fixed_shape_mask="all")
        self.scales = shared(scales, fixed_shape_mask="all")
        self.bias = shared(affine.bias.op.get_value().reshape(-1), fixed_shape_mask="all")

    def __call__(self, x):
        codes, scales = quantize_rows(x)
        return int8_product(codes, scales, self.codes, self.scales, self.bias)


def _quantize(x):
    """quantize_rows of a numpy matrix, on the host: same codes, same scales."""
    largest = np.abs(x).max(axis=1, keepdims=True, initial=0)
    finite = np.isfinite(largest)
    with np.errstate(all="ignore"):
        ratio = 127 * x.astype("f8") / np.where(largest > 0, largest, 1).astype("f8")
    codes = np.zeros((x.shape[0], _padded(x.shape[1])), "i1")
    codes[:, :x.shape[1]] = np.rint(np.where(finite, ratio, 0)).astype("i1")
    return codes, np.where(finite, largest / np.float32(127), np.float32(np.nan))[:, 0].astype("f4")
