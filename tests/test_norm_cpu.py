"""Layer norm, dropout and their residual form without a GPU: the host mask, and every refusal (they precede device
work)."""

import ctypes as C

import numpy as np
import pytest

import quabla_b200 as qb
from quabla_b200 import _lib

ROW = 1 << 20  # an address that nothing reads: all of these calls are refused before any device work


def call(name, **changes):
    """A valid call over 4 x 8 float32 rows with `changes`; returns its status and message."""
    lib = _lib.load()
    arrays = dict(x=ROW, residual=ROW, h=ROW, y=ROW, dy=ROW, dh=ROW, dx=ROW, dresidual=ROW, weight=ROW, bias=ROW, mean=ROW,
                  rstd=ROW, dweight=ROW, dbias=ROW, workspace=ROW)
    v = dict(arrays, dtype=_lib.F32, params=_lib.F32, rows=4, cols=8, epsilon=1e-5, rate=0.1, key=1, counter=0, d_counter=None,
             workspace_bytes=1 << 20, stride=8, in_stride=8)
    v.update(changes)
    i, o = v["in_stride"], v["stride"]
    if name == "dropout":
        status = lib.qb200_dropout(v["dtype"], v["x"], i, v["rows"], v["cols"], v["rate"], v["key"], v["counter"],
                                   v["d_counter"], v["y"], o, None)
    elif name == "layer_norm":
        status = lib.qb200_layer_norm(v["dtype"], v["params"], v["x"], i, v["rows"], v["cols"], v["weight"], v["bias"],
                                      v["epsilon"], v["y"], o, v["mean"], v["rstd"], None)
    elif name == "layer_norm_backward":
        status = lib.qb200_layer_norm_backward(v["dtype"], v["params"], v["dy"], i, v["x"], i, v["rows"], v["cols"],
                                               v["weight"], v["mean"], v["rstd"], v["dx"], o, v["dweight"], v["dbias"],
                                               v["workspace"], v["workspace_bytes"], None)
    elif name == "dropout_layer_norm":
        status = lib.qb200_dropout_layer_norm(v["dtype"], v["params"], v["x"], i, v["residual"], i, v["rows"], v["cols"],
                                              v["rate"], v["key"], v["counter"], v["d_counter"], v["weight"], v["bias"],
                                              v["epsilon"], v["h"], o, v["y"], o, v["mean"], v["rstd"], None)
    else:
        status = lib.qb200_dropout_layer_norm_backward(
            v["dtype"], v["params"], v["dy"], i, v["dh"], i, v["h"], i, v["rows"], v["cols"], v["weight"], v["mean"], v["rstd"],
            v["rate"], v["key"], v["counter"], v["d_counter"], v["dx"], o, v["dresidual"], o, v["dweight"], v["dbias"],
            v["workspace"], v["workspace_bytes"], None)
    return status, lib.qb200_last_error().decode()


NORMS = ["layer_norm", "layer_norm_backward", "dropout_layer_norm", "dropout_layer_norm_backward"]
DROPS = ["dropout", "dropout_layer_norm", "dropout_layer_norm_backward"]
ALL = sorted(set(NORMS + DROPS))


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("changes", [dict(dtype=4), dict(dtype=-1), dict(rows=-1), dict(cols=0), dict(stride=7), dict(stride=-8),
                                     dict(in_stride=-1), dict(stride=1 << 60), dict(in_stride=1 << 60)])
def test_types_extents_and_strides_are_checked(name, changes):
    status, message = call(name, **changes)
    assert status == _lib.INVALID and message.startswith(name)


@pytest.mark.parametrize("name", ALL)
def test_extents_that_overflow_are_refused(name):
    assert call(name, rows=1 << 62)[0] == _lib.TOO_LARGE


@pytest.mark.parametrize("name", NORMS)
@pytest.mark.parametrize("dtype,most", [(_lib.F32, 65536), (_lib.F64, 32768), (_lib.F16, 65536), (_lib.BF16, 65536)])
def test_rows_longer_than_the_limit_are_refused(name, dtype, most):
    status, message = call(name, dtype=dtype, params=dtype, cols=most + 1, stride=most + 1)
    assert status == _lib.TOO_LARGE and str(most) in message


@pytest.mark.parametrize("name", NORMS)
@pytest.mark.parametrize("dtype,params", [(_lib.F32, _lib.F64), (_lib.F32, _lib.F16), (_lib.F64, _lib.F32),
                                          (_lib.F16, _lib.BF16), (_lib.BF16, _lib.F16), (_lib.BF16, _lib.F64), (_lib.F32, 9)])
def test_parameter_types_are_checked(name, dtype, params):
    status, message = call(name, dtype=dtype, params=params)
    assert status == _lib.INVALID and "param_dtype" in message


@pytest.mark.parametrize("name", ["layer_norm", "dropout_layer_norm"])
@pytest.mark.parametrize("epsilon", [0.0, -1e-5, float("nan"), float("inf"), 1e-60, 1e60])
def test_epsilon_is_checked(name, epsilon):
    status, message = call(name, epsilon=epsilon)
    assert status == _lib.INVALID and "epsilon" in message


@pytest.mark.parametrize("name", DROPS)
@pytest.mark.parametrize("rate", [1.0, -0.1, 1.5, float("nan"), float("inf")])
def test_rate_is_checked(name, rate):
    status, message = call(name, rate=rate)
    assert status == _lib.INVALID and "rate" in message


@pytest.mark.parametrize("name", DROPS)
def test_counters_that_pass_64_bits_are_refused(name):
    status, message = call(name, counter=2**64 - 32)
    assert status == _lib.INVALID and "counter" in message


@pytest.mark.parametrize("name,required", [
    ("dropout", ["x", "y"]), ("layer_norm", ["x", "y"]), ("dropout_layer_norm", ["x", "y"]),
    ("layer_norm_backward", ["dy", "x", "mean", "rstd", "dx"]),
    ("dropout_layer_norm_backward", ["dy", "h", "mean", "rstd", "dx"])])
def test_required_arrays(name, required):
    for array in required:
        assert call(name, **{array: None})[0] == _lib.INVALID, array


@pytest.mark.parametrize("name,arrays", [
    ("dropout", ["x", "y", "d_counter"]), ("layer_norm", ["x", "y", "weight", "bias", "mean", "rstd"]),
    ("dropout_layer_norm", ["x", "residual", "h", "y", "weight", "bias", "mean", "rstd", "d_counter"]),
    ("layer_norm_backward", ["dy", "x", "dx", "weight", "mean", "rstd", "dweight", "dbias", "workspace"]),
    ("dropout_layer_norm_backward", ["dy", "dh", "h", "dx", "dresidual", "weight", "mean", "rstd", "dweight", "dbias",
                                     "workspace", "d_counter"])])
def test_alignment_is_checked(name, arrays):
    for array in arrays:
        status, message = call(name, **{array: ROW + 2})
        assert status == _lib.INVALID and "aligned" in message, array


@pytest.mark.parametrize("name", ["layer_norm_backward", "dropout_layer_norm_backward"])
def test_workspace_is_checked(name):
    size = C.c_size_t()
    lib = _lib.load()
    _lib.check(lib.qb200_layer_norm_workspace(_lib.F32, 4, 8, C.byref(size)))
    assert call(name, workspace=None)[0] == _lib.INVALID
    status, message = call(name, workspace_bytes=size.value - 1)
    assert status == _lib.INVALID and str(size.value) in message


def test_workspace_sizes():
    lib = _lib.load()
    size = C.c_size_t()
    for dtype, most in ((_lib.F32, 65536), (_lib.F64, 32768), (_lib.BF16, 65536)):
        for cols in [1, 7, 64, 255, 256, 257, 4095, 4096, 4097, 8192, 8193, 16385, 32767, 32768, 65536]:
            if cols > most:
                continue
            for rows in (1, 2, 300, 1 << 31, 1 << 40):
                _lib.check(lib.qb200_layer_norm_workspace(dtype, rows, cols, C.byref(size)))
                assert 0 < size.value <= 19 << 20
    _lib.check(lib.qb200_layer_norm_workspace(_lib.F32, 0, 8, C.byref(size)))
    assert size.value == 0
    assert lib.qb200_layer_norm_workspace(_lib.F32, 4, 8, None) == _lib.INVALID
    assert lib.qb200_layer_norm_workspace(_lib.F32, -1, 8, C.byref(size)) == _lib.INVALID
    assert lib.qb200_layer_norm_workspace(9, 4, 8, C.byref(size)) == _lib.INVALID
    assert lib.qb200_layer_norm_workspace(_lib.F32, 4, 65537, C.byref(size)) == _lib.TOO_LARGE


@pytest.mark.parametrize("name", ["dropout", "layer_norm", "dropout_layer_norm"])
def test_no_rows_need_no_arrays(name):
    nothing = {a: None for a in ("x", "residual", "h", "y", "mean", "rstd")}
    assert call(name, rows=0, **nothing)[0] == _lib.OK


@pytest.mark.parametrize("dtype", [_lib.F16, _lib.BF16])
def test_other_entry_points_refuse_16_bit_types(dtype):
    lib = _lib.load()
    handle = C.c_void_p()
    assert lib.qb200_desc_create(dtype, C.byref(handle)) == _lib.INVALID
    assert lib.qb200_weight_gradient(dtype, ROW, ROW, 4, 4, 4, ROW, None) == _lib.INVALID
    assert lib.qb200_weight_gradient_static(dtype, ROW, ROW, 4, 4, 4, ROW, None) == _lib.INVALID


# ---- the mask on the host ---------------------------------------------------------------------


def _mix(key, j):
    mask = (1 << 64) - 1
    z = (key + (j + 1) * 0x9E3779B97F4A7C15) & mask
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
    return z ^ (z >> 31)


@pytest.mark.parametrize("counter", [0, 1, 6, 2**32 - 1, 2**40 + 3, 2**64 - 3])
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.5, 1.0 - 2.0**-53])
def test_mask_is_the_halves_of_the_stream(counter, rate):
    key = qb.random.key(0xDEADBEEFCAFEBABE)
    if counter + 21 >= 2**64:  # indices end at 2^64
        with pytest.raises(ValueError, match="counter"):
            qb.random.dropout_mask(key, (3, 7), rate, counter)
        return
    got = qb.random.dropout_mask(key, (3, 7), rate, counter)
    threshold = int(rate * 2**32)
    assert got.shape == (3, 7) and got.dtype == bool
    for i, kept in enumerate(got.reshape(-1)):
        e = counter + i
        half = _mix(key.value, e >> 1) >> (32 * (e & 1)) & 0xFFFFFFFF
        assert kept == (half >= threshold)


def test_mask_uses_the_words_of_the_other_samplers():
    key = qb.random.key(11)
    bits = qb.random.split(key, 4)  # the stream's first outputs as keys
    halves = np.array([[k.value & 0xFFFFFFFF, k.value >> 32] for k in bits]).reshape(-1)
    assert (qb.random.dropout_mask(key, (8,), 0.3) == (halves >= int(0.3 * 2**32))).all()


def test_mask_rate_shards_and_refusals():
    key = qb.random.key(5)
    whole = qb.random.dropout_mask(key, (100, 101), 0.25)
    assert abs(whole.mean() - 0.75) < 5 * np.sqrt(0.25 * 0.75 / whole.size)
    for first in (0, 33, 50):  # a shard's counter is the index of its first element
        shard = qb.random.dropout_mask(key, (50, 101), 0.25, counter=first * 101)
        assert (shard == whole[first:first + 50]).all()
    assert qb.random.dropout_mask(key, (0, 4), 0.5).shape == (0, 4)
    for rate in (1.0, -0.1, float("nan")):
        with pytest.raises(ValueError):
            qb.random.dropout_mask(key, (2,), rate)
    with pytest.raises(TypeError):
        qb.random.dropout_mask("key", (2,), 0.5)
