"""The operators that stand around a block's affine layers, as measurable cases: layer norm with its gradients, dropout from
a counter-based generator with its gradient, rows as 8-bit integers with a scale each, and the product of such rows with
8-bit weights.

A pass of a "norm" case is the forward computation, of "norm_train" and "dropout_train" the forward and the backward one (the
gradient of the result is an input), of "quantize" one call on float32 rows, of "int8" a layer's call: float32 rows are
quantized and multiplied with weights that were quantized beforehand. All arrays stay on the GPU.
"""
import functools
import math

import numpy as np
import torch

own = False

EPSILON = 1e-5
MULTIPLIERS = (0xD2511F53, 0xCD9E8D57)   # of Philox4x32, and the increments of its two key words
INCREMENTS = (0x9E3779B9, 0xBB67AE85)
ROUNDS = 10
WORD = 0xFFFFFFFF


def listed():
    return [
        # one example through a layer of the MLP configuration, as a service answers requests: latency only
        dict(name="norm_one_row", kind="norm", rows=1, cols=256, dtype="f4"),
        # a long batch of wide rows through a trained network: bytes count
        dict(name="norm_large", kind="norm", rows=16384, cols=2048, dtype="f4"),
        # a training step's norm at the MLP configuration's batch and width
        dict(name="norm_train_b128", kind="norm_train", rows=128, cols=256, dtype="f4"),
        # the same on many wide rows (sequences times time steps)
        dict(name="norm_train_large", kind="norm_train", rows=8192, cols=4096, dtype="f4"),
        # double precision and an odd width, as gradient checks run it
        dict(name="norm_train_double", kind="norm_train", rows=1000, cols=1001, dtype="f8"),
        # dropout behind a layer of the MLP configuration
        dict(name="dropout_train_b128", kind="dropout_train", rows=128, cols=256, dtype="f4", p=0.5),
        # dropout on many wide rows
        dict(name="dropout_train_large", kind="dropout_train", rows=8192, cols=4096, dtype="f4", p=0.1),
        # a batch of digits becomes 8-bit rows
        dict(name="quantize_b128", kind="quantize", rows=128, cols=784),
        # many wide rows become 8-bit rows
        dict(name="quantize_large", kind="quantize", rows=16384, cols=2048),
        # one example through a wide layer with 8-bit weights: the weights' bytes count
        dict(name="int8_one_row", kind="int8", rows=1, cols=4096, outputs=4096, bias=True),
        # a prediction batch at sizes that fill no tile
        dict(name="int8_b500", kind="int8", rows=500, cols=1000, outputs=1001, bias=True),
        # a long batch through a wide layer: operations count
        dict(name="int8_large", kind="int8", rows=8192, cols=4096, outputs=4096, bias=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm_train", "norm_train", "dropout_train", "quantize", "int8", "int8", "int8"))
    if kind == "int8":
        cols, outputs = _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(16384, 8192 * 4096 * 4096 // (cols * outputs), (1 << 26) // outputs))
        return dict(kind=kind, rows=rows, cols=cols, outputs=outputs, bias=rng.random() < 0.5)
    cols = _log_int(rng, 1, 20000)
    rows = _log_int(rng, 1, min(1 << 20, (1 << 25) // cols))
    if kind == "quantize":
        return dict(kind=kind, rows=rows, cols=cols)
    dtype = rng.choice(("f4", "f4", "f4", "f8"))
    if dtype == "f8":
        rows = max(1, rows // 4)
    case = dict(kind=kind, rows=rows, cols=cols, dtype=dtype)
    if kind == "dropout_train":
        case["p"] = round(rng.uniform(0.02, 0.9), 3)
    return case


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _padded(cols):
    return -(-cols // 16) * 16


def _activations(g, rows, cols, dtype):
    """What a layer passes on: every row with a spread and an offset of its own, few elements far outside."""
    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    x = normal(rows, cols)
    x = torch.where(torch.rand(rows, cols, generator=g, device="cuda", dtype=dtype) < 0.002, x * 12, x)
    return x * torch.exp(0.5 * normal(rows, 1)) + 0.5 * normal(rows, 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    dtype = torch.float64 if case.get("dtype") == "f8" else torch.float32
    state = dict(case=case, x=_activations(g, rows, cols, dtype))
    if kind in ("norm_train", "dropout_train"):
        state["gy"] = torch.randn(rows, cols, generator=g, device="cuda", dtype=dtype) / cols
    if kind in ("norm", "norm_train"):
        state["gain"] = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda", dtype=dtype)
        state["bias"] = 0.2 * torch.randn(cols, generator=g, device="cuda", dtype=dtype)
    if kind == "dropout_train":   # the generator's key and the number of the training step
        state["key"] = torch.tensor([int(seed) * 0x100000001 + 7, int(seed) % 1000], device="cuda")
        state["increment"] = torch.tensor([0, 1], device="cuda")
    if kind == "int8":            # a layer's weights, quantized once: [outputs, cols], columns padded with zeros
        w = torch.randn(case["outputs"], cols, generator=g, device="cuda") / math.sqrt(cols)
        state["w_codes"], state["w_scales"] = _quantize(w)
        state["w_bias"] = 0.1 * torch.randn(case["outputs"], generator=g, device="cuda") if case["bias"] else None
    if own:   # a program keeps its variables and its compiled function; no operator runs here
        state["function"], state["results"] = _compile(state)
    return state


# ------------------------------------------------------------------------------------------------
# one pass, plain
# ------------------------------------------------------------------------------------------------
def _norm(x, gain, bias):
    centred = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPSILON)
    hat = centred * rstd
    return hat * gain + bias, hat, rstd


def _norm_gradients(hat, rstd, gain, gy):
    d = gy * gain
    dx = rstd * (d - d.mean(1, keepdim=True) - hat * (d * hat).mean(1, keepdim=True))
    return dx, (gy * hat).sum(0), gy.sum(0)


def _round(words, r):
    """One round on the four 32-bit words and the two key words, held in 64 bits."""
    (c0, c1, c2, c3, k0, k1) = words
    p0, p1 = c0 * MULTIPLIERS[0], c2 * MULTIPLIERS[1]   # the low 64 bits are the product's, whatever the sign
    return (((p1 >> 32) & WORD) ^ c1 ^ k0, p1 & WORD, ((p0 >> 32) & WORD) ^ c3 ^ k1, p0 & WORD,
            (k0 + INCREMENTS[0]) & WORD, (k1 + INCREMENTS[1]) & WORD)


def _keep(n, key, p):
    """Truth values of n elements; element i takes word i % 4 of the block with counter (i // 4, step, 0)."""
    block = torch.arange(-(-n // 4), device="cuda")
    seed, step = key[0], key[1]
    start = (block & WORD, block >> 32, (step & WORD).expand_as(block), torch.zeros_like(block), seed & WORD, (seed >> 32) & WORD)
    words = functools.reduce(_round, range(ROUNDS), start)
    return (torch.stack(words[:4], 1) >= int(round(p * 2.0 ** 32))).reshape(-1)[:n]


def _dropped(x, keep, p):
    return torch.where(keep, x * (1 / (1 - p)), torch.zeros_like(x))


def _quantize(x):
    """Codes and scales. A code is 127 x / max|x| rounded to the nearest whole number, ties to the even one: in 64 bits,
    where the quotient is never rounded across a tie."""
    largest = x.abs().amax(1, keepdim=True)
    ratio = 127 * x.double() / torch.where(largest > 0, largest, torch.ones_like(largest)).double()
    codes = torch.zeros(x.shape[0], _padded(x.shape[1]), dtype=torch.int8, device=x.device)
    codes[:, :x.shape[1]] = torch.round(ratio).to(torch.int8)
    return codes, largest[:, 0] / 127


def _product(codes, scales, w_codes, w_scales, bias):
    # sums of products of whole numbers: exact in 32 bits while they stay below 2^24, as sums of a few thousand terms of
    # both signs do
    y = (codes.float() @ w_codes.float().T) * scales[:, None] * w_scales
    return y if bias is None else y + bias


def run(state):
    if own:
        state["function"]()
        return state["results"]
    case, x = state["case"], state["x"]
    kind = case["kind"]
    if kind == "norm":
        return [_norm(x, state["gain"], state["bias"])[0]]
    if kind == "norm_train":
        y, hat, rstd = _norm(x, state["gain"], state["bias"])
        return [y] + list(_norm_gradients(hat, rstd, state["gain"], state["gy"]))
    if kind == "dropout_train":
        keep = _keep(x.numel(), state["key"], case["p"]).reshape(x.shape)
        y, dx = _dropped(x, keep, case["p"]), _dropped(state["gy"], keep, case["p"])
        state["key"] = state["key"] + state["increment"]
        return [y, dx, state["key"]]
    codes, scales = _quantize(x)
    if kind == "quantize":
        return [codes, scales]
    return [_product(codes, scales, state["w_codes"], state["w_scales"], state["w_bias"])]


# ------------------------------------------------------------------------------------------------
# one pass, by the framework
# ------------------------------------------------------------------------------------------------
class _View(object):
    """Device memory of a shared variable for torch (CUDA array interface); keeps the memory alive."""

    def __init__(self, variable):
        self.owner = variable.op._value
        self.__cuda_array_interface__ = dict(shape=tuple(self.owner.shape), typestr="<" + self.owner.dtype,
                                             data=(self.owner.data, False), version=3)


def _compile(state):
    """The compiled function of a case, and what it leaves on the GPU: the variables that a call updates."""
    import cgt_b200 as cgt
    from cgt_b200 import core, nn

    def shared(t):
        return cgt.shared(t.cpu().numpy(), fixed_shape_mask="all")

    def zeros(shape, dtype):
        return cgt.shared(np.zeros(shape, dtype), fixed_shape_mask="all")

    case = state["case"]
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    float_type, more = case.get("dtype", "f4"), []
    with cgt.scoped_update_config(precision="double" if float_type == "f8" else "single"):
        x = shared(state["x"])
        if kind in ("norm", "norm_train"):
            gain, bias = shared(state["gain"]), shared(state["bias"])
            y = nn.layer_norm(x, gain, bias, epsilon=EPSILON)
            outs = [(y, (rows, cols), float_type)]
            if kind == "norm_train":
                dx, dgain, dbias = core.pullback([y], [shared(state["gy"])], [x, gain, bias])
                outs += [(dx, (rows, cols), float_type), (dgain, (cols,), float_type), (dbias, (cols,), float_type)]
        elif kind == "dropout_train":
            stream = nn.RandomStream(0)
            stream.state.op.set_value(state["key"].cpu().numpy())
            y = nn.dropout(x, case["p"], stream)
            dx = core.pullback([y], [shared(state["gy"])], [x])[0]
            outs = [(y, (rows, cols), float_type), (dx, (rows, cols), float_type)]
            more = stream.updates()
        else:
            codes, scales = nn.quantize_rows(x)
            if kind == "quantize":
                outs = [(codes, (rows, _padded(cols)), "i1"), (scales, (rows,), "f4")]
            else:
                bias = None if state["w_bias"] is None else shared(state["w_bias"])
                y = nn.int8_product(codes, scales, shared(state["w_codes"]), shared(state["w_scales"]), bias)
                outs = [(y, (rows, case["outputs"]), "f4")]
        updates = [(zeros(shape, dtype), node) for (node, shape, dtype) in outs] + more
        f = cgt.function([], [], updates=updates)
    return f, [torch.as_tensor(_View(variable), device="cuda") for (variable, _new) in updates]


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    """Bytes: each input read once, each result written once. Flops: two for every term of a product, a handful for every
    element elsewhere."""
    kind, n, cols = case["kind"], case["rows"] * case["cols"], case["cols"]
    size = 8 if case.get("dtype") == "f8" else 4
    if kind == "norm":
        return {"bytes": size * (2.0 * n + 2 * cols), "flops": 8.0 * n}
    if kind == "norm_train":   # the backward pass reads x again: between the two lies the rest of the network
        return {"bytes": size * (5.0 * n + 5 * cols), "flops": 24.0 * n}
    if kind == "dropout_train":
        return {"bytes": size * 4.0 * n + 32, "flops": 4.0 * n}
    rows, padded = case["rows"], _padded(cols)
    if kind == "quantize":
        return {"bytes": 4.0 * n + rows * padded + 4 * rows, "flops": 4.0 * n}
    outputs = case["outputs"]
    values = n + rows * outputs + outputs * (2 if case["bias"] else 1)
    return {"bytes": 4.0 * values + outputs * padded, "flops": 2.0 * n * outputs + 4.0 * n}


def _exact_norm(state, train):
    x = state["x"].double()
    gain, bias = state["gain"].double(), state["bias"].double()
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    sigma = ((x - mean).pow(2).sum(1, keepdim=True) / n + EPSILON).sqrt()
    y = gain * (x - mean) / sigma + bias
    if not train:
        return [y]
    # by the chain rule through x - mean and sigma
    gy = state["gy"].double()
    a = gy * gain
    d_sigma = -(a * (x - mean)).sum(1, keepdim=True) / sigma.pow(2)
    d_centred = a / sigma + d_sigma * (x - mean) / (n * sigma)
    return [y, d_centred - d_centred.sum(1, keepdim=True) / n, (gy * (x - mean) / sigma).sum(0), gy.sum(0)]


def _exact_words(n, seed, step):
    """The generator's words of n elements, on the host."""
    blocks = np.arange(-(-n // 4), dtype=np.uint64)
    low = np.uint64(WORD)
    c = [blocks & low, blocks >> np.uint64(32), np.full_like(blocks, step & WORD), np.zeros_like(blocks)]
    k = [seed & WORD, (seed >> 32) & WORD]
    for _ in range(ROUNDS):
        a, b = c[0] * np.uint64(MULTIPLIERS[0]), c[2] * np.uint64(MULTIPLIERS[1])
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[i] + INCREMENTS[i]) & WORD for i in (0, 1)]
    return np.stack([w.astype(np.uint32) for w in c], axis=1).reshape(-1)[:n]


def exact(case, seed):
    state = prepare(case, seed)
    kind, x = case["kind"], state["x"]
    if kind in ("norm", "norm_train"):
        return _exact_norm(state, kind == "norm_train")
    if kind == "dropout_train":
        key = [int(v) for v in state["key"].cpu()]
        dropped = _exact_words(x.numel(), *key).reshape(tuple(x.shape)) < int(round(case["p"] * 2.0 ** 32))
        dropped = torch.from_numpy(dropped).to(x.device)
        return [(t.double() / (1.0 - case["p"])).masked_fill(dropped, 0.0) for t in (x, state["gy"])] + [None]
    x = x.double()
    unit = x.abs().max(1, keepdim=True).values / 127
    if kind == "quantize":
        return [None, unit[:, 0]]
    whole = (x / torch.where(unit > 0, unit, torch.ones_like(unit))).round()
    y = whole @ state["w_codes"][:, :case["cols"]].double().T
    y = y * unit * state["w_scales"].double()
    return [y if state["w_bias"] is None else y + state["w_bias"].double()]
