"""Performance cases of the stand-alone layer norm, dropout and their residual form, over caller-owned device arrays.

The five entry points that a program calls when it puts a network's block together from the library's building blocks:

  layer_norm                    y = (x - mean) * rstd * weight + bias for every row, with the rows' mean and rstd
  layer_norm_backward           gradients of the rows, and of weight and bias summed over the rows
  dropout                       x / (1 - rate) where the generator keeps an element, 0 elsewhere; no mask is stored
  dropout_layer_norm            h = residual + dropout(x), y = layer_norm(h)
  dropout_layer_norm_backward   gradients of x, residual, weight and bias, the mask drawn again

Arrays are torch tensors on the current device because the entry points take device addresses and a stream.
"""

import math

import numpy as np
import torch

own = False  # False: the operators in elementary torch operations; True: the library's entry points

EPSILON = 1e-5
GAMMA, M1, M2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB  # SplitMix64
TYPES = {"float32": torch.float32, "float64": torch.float64, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODES = {"float32": 0, "float64": 1, "float16": 2, "bfloat16": 3}
OPERATORS = ("layer_norm", "layer_norm_backward", "dropout", "dropout_layer_norm", "dropout_layer_norm_backward")


def _case(name, op, dtype, params, rows, cols, pad=0, rate=0.0):
    return {"name": name, "op": op, "dtype": dtype, "params": params, "rows": rows, "cols": cols, "pad": pad, "rate": rate}


def listed():
    return [
        # One point through a network of the Burgers width: evaluation of a single query.
        _case("norm, one row", "layer_norm", "float32", "float32", 1, 128),
        # Tokens of a transformer block, 16-bit activations beside float32 parameters.
        _case("norm, tokens", "layer_norm", "bfloat16", "float32", 8192, 4096),
        # A slice of a wider array whose rows start at no particular alignment, an odd number of columns.
        _case("norm, odd columns", "layer_norm", "float32", "float32", 4099, 1001, pad=6),
        # The tutorial-sized problem in the surface's default type.
        _case("norm gradient, 128 points", "layer_norm_backward", "float64", "float64", 128, 16),
        # Collocation points of the Burgers problem at its width: few columns, very many rows to reduce over.
        _case("norm gradient, points", "layer_norm_backward", "float32", "float32", 262144, 128),
        # Tokens of a wide block, everything in 16 bits.
        _case("norm gradient, wide", "layer_norm_backward", "bfloat16", "bfloat16", 8192, 8192),
        # A small hidden layer.
        _case("dropout, small", "dropout", "float32", "float32", 128, 64, rate=0.1),
        # The hidden activations of a feed-forward block, the largest array.
        _case("dropout, large", "dropout", "bfloat16", "bfloat16", 16384, 8192, rate=0.1),
        # The end of a residual branch in training.
        _case("residual norm, tokens", "dropout_layer_norm", "bfloat16", "bfloat16", 4096, 4096, rate=0.1),
        # A handful of long rows (a whole field as one row): the work of a row has to be shared.
        _case("residual norm, long rows", "dropout_layer_norm", "float32", "float32", 6, 50001, rate=0.25),
        # Its gradient at a training batch.
        _case("residual norm gradient, tokens", "dropout_layer_norm_backward", "bfloat16", "float32", 8192, 5120, rate=0.1),
        # A ragged last batch of an odd width.
        _case("residual norm gradient, ragged", "dropout_layer_norm_backward", "float16", "float16", 1003, 515, pad=13, rate=0.5),
    ]


def draw(rng):
    op = rng.choice(OPERATORS)
    dtype = rng.choice(("float32", "float32", "float64", "float16", "bfloat16", "bfloat16"))
    params = dtype if dtype in ("float32", "float64") else rng.choice((dtype, "float32"))
    most = 32768 if dtype == "float64" else 65536
    cols = int(round(math.exp(rng.uniform(math.log(8), math.log(most if rng.random() < 0.15 else 12000)))))
    if rng.random() < 0.5:  # widths are multiples of 8 as often as not
        cols = cols // 8 * 8
    rows = int(round(math.exp(rng.uniform(0.0, math.log(min(300000, (1 << 25) // cols))))))
    pad = rng.choice((0, 0, 0, 8, 64, 1, rng.randint(1, 40)))
    rate = rng.choice((0.05, 0.1, 0.2, 0.3, 0.5, 0.9)) if op.startswith("dropout") else 0.0
    case = _case("", op, dtype, params, rows, cols, pad, rate)
    del case["name"]
    return case


def _statistics_type(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def prepare(case, seed):
    rows, cols, op = case["rows"], case["cols"], case["op"]
    dtype, params = TYPES[case["dtype"]], TYPES[case["params"]]
    stat = _statistics_type(dtype)
    generator = torch.Generator(device="cuda").manual_seed(1000003 * seed + rows + 7 * cols)

    def normal(*shape):
        return torch.randn(*shape, dtype=stat, device="cuda", generator=generator)

    def array(values=None):
        """[rows][cols] inside rows of cols + pad elements."""
        whole = torch.empty(rows, cols + case["pad"], dtype=dtype, device="cuda")
        if values is not None:
            whole[:, :cols] = values
        return whole[:, :cols]

    # The rows are one of eight shards of a batch that draws from one key: the counter is the shard's first element.
    state = {"case": case, "key": (seed * 0x9E3779B9 + 0x5DEECE66D1CE4E5B) % (1 << 64), "counter": seed % 8 * rows * cols}

    # Activations: unit scale, an offset for every row, a few columns that are much larger than the others.
    def activations():
        scale = 1.0 + 7.0 * (torch.rand(cols, dtype=stat, device="cuda", generator=generator) < 0.01).to(stat)
        return normal(rows, cols) * scale + 0.5 * normal(rows, 1)

    state["x"] = array(activations())
    if op == "dropout":
        state["y"] = array()
        return state
    state["weight"] = (1.0 + 0.2 * normal(cols)).to(params)
    state["bias"] = (0.1 * normal(cols)).to(params)
    if op == "layer_norm":
        state["y"] = array()
    elif op == "dropout_layer_norm":
        state["residual"], state["h"], state["y"] = array(activations()), array(), array()
    if not op.endswith("backward"):
        state["mean"], state["rstd"] = (torch.empty(rows, dtype=stat, device="cuda") for _ in range(2))
        return state
    wide = state["x"].double()  # the row array of a backward pass: x, or the h that the forward pass left
    mean = wide.mean(1)
    state["mean"] = mean.to(stat)
    state["rstd"] = (1.0 / torch.sqrt((wide - mean[:, None]).square().mean(1) + EPSILON)).to(stat)
    state["dy"], state["dx"] = array(0.1 * normal(rows, cols)), array()
    state["dweight"], state["dbias"] = torch.empty_like(state["weight"]), torch.empty_like(state["bias"])
    if op == "dropout_layer_norm_backward":
        state["dh"], state["dresidual"] = array(0.1 * normal(rows, cols)), array()
    return state


# ---- the library's entry points --------------------------------------------------------------


def _run_own(s):
    from quabla_b200 import _lib

    lib, case = _lib.load(), s["case"]
    op, rows, cols, rate = case["op"], case["rows"], case["cols"], case["rate"]
    dtype, params = CODES[case["dtype"]], CODES[case["params"]]
    stream = torch.cuda.current_stream().cuda_stream
    x = s["x"]
    stride = x.stride(0) if rows > 1 else cols + case["pad"]
    if op == "dropout":
        _lib.check(lib.qb200_dropout(dtype, x.data_ptr(), stride, rows, cols, rate, s["key"], s["counter"], None,
                                     s["y"].data_ptr(), stride, stream))
        return s["y"]
    weight, bias, mean, rstd = s["weight"].data_ptr(), s["bias"].data_ptr(), s["mean"].data_ptr(), s["rstd"].data_ptr()
    if op == "layer_norm":
        _lib.check(lib.qb200_layer_norm(dtype, params, x.data_ptr(), stride, rows, cols, weight, bias, EPSILON,
                                        s["y"].data_ptr(), stride, mean, rstd, stream))
        return s["y"], s["mean"], s["rstd"]
    if op == "dropout_layer_norm":
        _lib.check(lib.qb200_dropout_layer_norm(dtype, params, x.data_ptr(), stride, s["residual"].data_ptr(), stride, rows,
                                                cols, rate, s["key"], s["counter"], None, weight, bias, EPSILON,
                                                s["h"].data_ptr(), stride, s["y"].data_ptr(), stride, mean, rstd, stream))
        return s["h"], s["y"], s["mean"], s["rstd"]
    if "workspace" not in s:
        import ctypes

        size = ctypes.c_size_t()
        _lib.check(lib.qb200_layer_norm_workspace(dtype, rows, cols, ctypes.byref(size)))
        s["workspace"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    workspace = s["workspace"]
    if op == "layer_norm_backward":
        _lib.check(lib.qb200_layer_norm_backward(dtype, params, s["dy"].data_ptr(), stride, x.data_ptr(), stride, rows, cols,
                                                 weight, mean, rstd, s["dx"].data_ptr(), stride, s["dweight"].data_ptr(),
                                                 s["dbias"].data_ptr(), workspace.data_ptr(), workspace.numel(), stream))
        return s["dx"], s["dweight"], s["dbias"]
    _lib.check(lib.qb200_dropout_layer_norm_backward(
        dtype, params, s["dy"].data_ptr(), stride, s["dh"].data_ptr(), stride, x.data_ptr(), stride, rows, cols, weight, mean,
        rstd, rate, s["key"], s["counter"], None, s["dx"].data_ptr(), stride, s["dresidual"].data_ptr(), stride,
        s["dweight"].data_ptr(), s["dbias"].data_ptr(), workspace.data_ptr(), workspace.numel(), stream))
    return s["dx"], s["dresidual"], s["dweight"], s["dbias"]


# ---- the operators in elementary operations --------------------------------------------------


def _signed(value):
    value %= 1 << 64
    return value - (1 << 64) if value >= 1 << 63 else value


def _shifted(z, bits):
    """Logical shift to the right of 64-bit words that torch holds as signed ones."""
    return (z >> bits) & ((1 << (64 - bits)) - 1)


def _kept(s):
    """Truth values [rows][cols]: element e takes the low (even e) or high half of word e // 2 of the key's stream."""
    case, counter = s["case"], s["counter"]
    count = case["rows"] * case["cols"]
    word = torch.arange(counter // 2 + 1, (counter + count - 1) // 2 + 2, device="cuda")
    z = word * _signed(GAMMA) + _signed(s["key"])
    z = (z ^ _shifted(z, 30)) * _signed(M1)
    z = (z ^ _shifted(z, 27)) * _signed(M2)
    z = z ^ _shifted(z, 31)
    halves = torch.stack((z & 0xFFFFFFFF, _shifted(z, 32)), dim=1).reshape(-1)
    first = counter % 2
    return (halves[first:first + count] >= math.floor(case["rate"] * 2.0**32)).view(case["rows"], case["cols"])


def _dropped(s, x):
    return torch.where(_kept(s), x * (1.0 / (1.0 - s["case"]["rate"])), 0.0)


def _normalised(s, x):
    mean = x.mean(dim=1)
    centred = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1) + EPSILON)
    return centred * rstd[:, None] * s["weight"].to(x.dtype) + s["bias"].to(x.dtype), mean, rstd


def _normalised_backward(s, x, dy):
    normal = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["weight"].to(x.dtype)
    dx = s["rstd"][:, None] * (g - g.mean(dim=1, keepdim=True) - normal * (g * normal).mean(dim=1, keepdim=True))
    return dx, (dy * normal).sum(dim=0).to(s["weight"].dtype), dy.sum(dim=0).to(s["bias"].dtype)


def run(state):
    s = state
    if own:
        return _run_own(s)
    op, dtype = s["case"]["op"], s["x"].dtype
    x = s["x"].to(_statistics_type(dtype))
    if op == "dropout":
        return _dropped(s, x).to(dtype)
    if op == "layer_norm":
        y, mean, rstd = _normalised(s, x)
        return y.to(dtype), mean, rstd
    if op == "dropout_layer_norm":
        h = s["residual"].to(x.dtype) + _dropped(s, x)
        y, mean, rstd = _normalised(s, h)
        return h.to(dtype), y.to(dtype), mean, rstd
    dx, dweight, dbias = _normalised_backward(s, x, s["dy"].to(x.dtype))
    if op == "layer_norm_backward":
        return dx.to(dtype), dweight, dbias
    dx = dx + s["dh"].to(x.dtype)
    return _dropped(s, dx).to(dtype), dx.to(dtype), dweight, dbias


# ---- the definitions in 64 bits --------------------------------------------------------------


def _exact_mask(case, key, counter):
    """The generator in NumPy's unsigned 64-bit arithmetic, one draw for each pair of elements."""
    count = case["rows"] * case["cols"]
    with np.errstate(over="ignore"):
        bits = np.arange(counter // 2, (counter + count + 1) // 2, dtype=np.uint64)
        bits += np.uint64(1)
        bits *= np.uint64(GAMMA)
        bits += np.uint64(key)
        bits ^= bits >> np.uint64(30)
        bits *= np.uint64(M1)
        bits ^= bits >> np.uint64(27)
        bits *= np.uint64(M2)
        bits ^= bits >> np.uint64(31)
    draws = bits.astype("<u8", copy=False).view("<u4")[counter % 2:][:count]
    return torch.from_numpy(draws >= np.uint32(int(case["rate"] * 4294967296.0))).cuda().view(case["rows"], case["cols"])


def exact(case, seed):
    s = prepare(case, seed)
    op, cols = case["op"], case["cols"]
    x = s["x"].double()
    if case["rate"] > 0.0:
        factor = _exact_mask(case, s["key"], s["counter"]).double() / (1.0 - case["rate"])
    if op == "dropout":
        return x * factor
    weight, bias = s["weight"].double(), s["bias"].double()
    if op in ("layer_norm", "dropout_layer_norm"):
        h = x if op == "layer_norm" else s["residual"].double() + x * factor
        mean = h.sum(1, keepdim=True) / cols
        variance = ((h - mean) ** 2).sum(1, keepdim=True) / cols
        rstd = (variance + EPSILON) ** -0.5
        outputs = ((h - mean) * rstd * weight + bias, mean.reshape(-1), rstd.reshape(-1))
        return outputs if op == "layer_norm" else (h, *outputs)
    dy, rstd = s["dy"].double(), s["rstd"].double().unsqueeze(1)
    scaled = (x - s["mean"].double().unsqueeze(1)) * rstd
    dscaled = dy * weight
    along = (dscaled * scaled).sum(1, keepdim=True) / cols
    dx = (dscaled - dscaled.sum(1, keepdim=True) / cols - along * scaled) * rstd
    sums = (torch.einsum("rc,rc->c", dy, scaled), torch.einsum("rc->c", dy))
    if op == "layer_norm_backward":
        return (dx, *sums)
    dx = dx + s["dh"].double()
    return (dx * factor, dx, *sums)


# ---- what a pass cannot do without -----------------------------------------------------------

# Arrays of rows that are read and written, parameter arrays, per-row statistics; floating operations of an element.
NEEDS = {"layer_norm": (2, 2, 2, 8), "layer_norm_backward": (3, 3, 2, 14), "dropout": (2, 0, 0, 1),
         "dropout_layer_norm": (4, 2, 2, 10), "dropout_layer_norm_backward": (5, 3, 2, 16)}


def work(case):
    arrays, parameters, statistics, flops = NEEDS[case["op"]]
    rows, cols = case["rows"], case["cols"]
    element, parameter = TYPES[case["dtype"]].itemsize, TYPES[case["params"]].itemsize
    statistic = _statistics_type(TYPES[case["dtype"]]).itemsize
    return {"bytes": arrays * rows * cols * element + parameters * cols * parameter + statistics * rows * statistic,
            "flops": flops * rows * cols}
