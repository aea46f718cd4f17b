"""Layer norm, dropout and their residual form on the device against their definitions in 64 bits (bounds: _norm_util)."""

import ctypes as C

import numpy as np
import pytest

import quabla_b200 as qb
from quabla_b200 import _lib

import _norm_util as nu

pytestmark = pytest.mark.gpu

# (rows, cols, pad, shift): one element; lanes that share a warp; rows that start on no 16-byte boundary (odd columns,
# odd strides, a shifted base); the last pack of an aligned row cut short; many rows; several warps and several CTAs for
# a row; the longest rows.
SHAPES = [(1, 1, 0, 0), (3, 7, 0, 0), (5, 16, 0, 0), (2, 33, 0, 1), (300, 64, 0, 0), (37, 257, 0, 0), (9, 100, 4, 0), (10, 250, 6, 0),
          (4, 1001, 6, 0), (2, 1001, 7, 0), (513, 48, 16, 0), (3, 4096, 0, 0), (2, 5120, 0, 3), (2, 8200, 0, 0), (1, 50001, 0, 0),
          (2, 20008, 8, 0), (20000, 3, 0, 0), (4099, 130, 0, 0)]
# 16-bit rows that start on 4-byte boundaries and no wider ones.
SHAPES += [(300, 34, 0, 0), (6, 250, 0, 0), (37, 1002, 0, 2), (2, 4098, 0, 0), (5, 18, 4, 2)]


def shapes_for(dtype):
    longest = 32768 if dtype == "float64" else 65536
    return [s for s in SHAPES if s[1] <= longest] + [(2, longest, 0, 0), (20, longest - 1, 1, 0)]


CASES = [(d, p, *s) for d, p in nu.TYPE_PAIRS for s in shapes_for(d)]


def inputs(dtype, params, rows, cols, pad, shift):
    import torch

    x = nu.Rows(rows, cols, dtype, pad, shift, nu.normal(1, rows, cols) + 0.5 * nu.normal(2, rows, 1))
    weight = nu.vector(1.0 + 0.2 * nu.normal(3, cols), params)
    bias = nu.vector(0.1 * nu.normal(4, cols), params)
    mean, rstd = (torch.full((rows,), float("nan"), dtype=nu.statistics_type(dtype), device="cuda") for _ in range(2))
    return x, weight, bias, mean, rstd


@pytest.mark.parametrize("dtype,params,rows,cols,pad,shift", CASES)
def test_layer_norm(cuda_device, dtype, params, rows, cols, pad, shift):
    x, weight, bias, mean, rstd = inputs(dtype, params, rows, cols, pad, shift)
    y = nu.Rows(rows, cols, dtype, pad, shift)
    nu.layer_norm(dtype, params, x, weight, bias, y, mean, rstd)
    nu.check_forward(dtype, x.wide(), weight, bias, y, mean, rstd)
    assert y.outside_untouched()


def saved(dtype, h):
    """What a forward pass leaves of the rows' statistics."""
    wide = h.wide()
    mean = wide.mean(1)
    rstd = ((wide - mean[:, None]).square().mean(1) + nu.EPSILON) ** -0.5
    return mean.to(nu.statistics_type(dtype)), rstd.to(nu.statistics_type(dtype))


@pytest.mark.parametrize("dtype,params,rows,cols,pad,shift", CASES)
def test_layer_norm_backward(cuda_device, dtype, params, rows, cols, pad, shift):
    import torch

    x, weight, _, _, _ = inputs(dtype, params, rows, cols, pad, shift)
    mean, rstd = saved(dtype, x)
    dy = nu.Rows(rows, cols, dtype, pad, shift, 0.1 * nu.normal(5, rows, cols))
    dx = nu.Rows(rows, cols, dtype, pad, shift)
    dweight, dbias = torch.full_like(weight, float("nan")), torch.full_like(weight, float("nan"))
    nu.layer_norm_backward(dtype, params, dy, x, weight, mean, rstd, dx, dweight, dbias)
    nu.check_backward(dtype, params, dy, x, weight, mean, rstd, dx, dweight, dbias)
    assert dx.outside_untouched()


@pytest.mark.parametrize("dtype,params,rows,cols,pad,shift", CASES)
@pytest.mark.parametrize("rate", [0.0, 0.3])
def test_dropout_layer_norm(cuda_device, dtype, params, rows, cols, pad, shift, rate):
    x, weight, bias, mean, rstd = inputs(dtype, params, rows, cols, pad, shift)
    residual = nu.Rows(rows, cols, dtype, pad, shift, nu.normal(6, rows, cols))
    h, y = nu.Rows(rows, cols, dtype, pad, shift), nu.Rows(rows, cols, dtype, pad, shift)
    key, counter = qb.random.key(99), 12345 + rows
    nu.dropout_layer_norm(dtype, params, x, residual, rate, key.value, counter, weight, bias, h, y, mean, rstd)
    kept = nu.mask(key, rows, cols, rate, counter)
    branch = nu.dropped(x.wide(), kept, rate)
    want = residual.wide() + branch
    u = nu.unit(dtype)
    # Scale and product round once each, the sum once, then h's own type.
    assert ((h.wide() - want).abs() <= nu.half_step(dtype) * (1 + 8 * u) * want.abs() + 4 * u * (branch.abs() + want.abs())
            + nu.tiny(dtype)).all()
    # The statistics are of the sum before it is rounded; its own error of 4 u is inside the bound's 64 u.
    nu.check_forward(dtype, want, weight, bias, y, mean, rstd)
    assert h.outside_untouched() and y.outside_untouched()


@pytest.mark.parametrize("dtype,params,rows,cols,pad,shift", CASES)
@pytest.mark.parametrize("rate", [0.0, 0.3])
def test_dropout_layer_norm_backward(cuda_device, dtype, params, rows, cols, pad, shift, rate):
    import torch

    h, weight, _, _, _ = inputs(dtype, params, rows, cols, pad, shift)
    mean, rstd = saved(dtype, h)
    dy = nu.Rows(rows, cols, dtype, pad, shift, 0.1 * nu.normal(5, rows, cols))
    dh = nu.Rows(rows, cols, dtype, pad, shift, 0.1 * nu.normal(7, rows, cols))
    dx, dresidual = nu.Rows(rows, cols, dtype, pad, shift), nu.Rows(rows, cols, dtype, pad, shift)
    dweight, dbias = torch.full_like(weight, float("nan")), torch.full_like(weight, float("nan"))
    key, counter = qb.random.key(98), 777 * cols
    nu.dropout_layer_norm_backward(dtype, params, dy, dh, h, weight, mean, rstd, rate, key.value, counter, dx, dresidual,
                                   dweight, dbias)
    kept = nu.mask(key, rows, cols, rate, counter)
    nu.check_backward(dtype, params, dy, h, weight, mean, rstd, dx, dweight, dbias, dh, dresidual, kept, rate)
    assert dx.outside_untouched() and dresidual.outside_untouched()


# ---- dropout ----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES + [(1, 1 << 20, 0, 0), (1, 1000003, 0, 1), (3, 70001, 5, 0)])
@pytest.mark.parametrize("counter", [0, 2**32 - 5, 2**62 + 1])
def test_dropout(cuda_device, dtype, rows, cols, pad, shift, counter):
    import torch

    x = nu.Rows(rows, cols, dtype, pad, shift, nu.normal(1, rows, cols) + 3.0)
    y = nu.Rows(rows, cols, dtype, pad, shift)
    key, rate = qb.random.key(3), 0.4
    nu.dropout(dtype, x, rate, key.value, counter, y)
    kept = nu.mask(key, rows, cols, rate, counter)
    # One product in the accumulation type, rounded to the array's.
    scale = torch.tensor(1.0 / (1.0 - rate), dtype=nu.statistics_type(dtype), device="cuda")
    want = torch.where(kept, x.view.to(scale.dtype) * scale, 0.0).to(x.view.dtype)
    assert (y.view == want).all()
    assert y.outside_untouched()


def _key_of_word(word):
    """The key whose first word is `word`: the generator's output function backwards."""
    mask = (1 << 64) - 1

    def unshift(z, by):
        out = z
        for _ in range(64 // by + 1):
            out = z ^ (out >> by)
        return out

    z = unshift(word, 31)
    z = unshift((z * pow(0x94D049BB133111EB, -1, 1 << 64)) & mask, 27)
    z = unshift((z * pow(0xBF58476D1CE4E5B9, -1, 1 << 64)) & mask, 30)
    return (z - 0x9E3779B97F4A7C15) & mask


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rate", [0.1, 0.5, 0.7, 0.9, 0.25, 1.0 - 2.0**-32, 0.5 + 2.0**-32, 2.0**-32])
@pytest.mark.parametrize("residual", [False, True])
def test_elements_at_the_threshold(cuda_device, dtype, rate, residual):
    # Words whose halves lie at the threshold and next to it, as low and as high halves, in packs that start with either.
    import torch

    threshold = int(rate * 2**32)
    halves = [h for h in range(threshold - 2, threshold + 3) if 0 <= h < 2**32]
    for half in halves:
        for word in (half, half << 32, half << 32 | 0xFFFFFFFF, half | 0xFFFFFFFF << 32):
            key = qb.random.Key(_key_of_word(word))
            assert int(qb.random._stream(key.value, 1)[0]) == word
            for counter in (0, 1):
                kept = nu.mask(key, 1, 64, rate, counter)
                x = nu.Rows(1, 64, dtype, values=torch.ones(1, 64, dtype=torch.float64))
                y, h = nu.Rows(1, 64, dtype), nu.Rows(1, 64, dtype)
                if residual:
                    nu.dropout_layer_norm(dtype, dtype, x, None, rate, key.value, counter, None, None, h, y, None, None)
                    assert ((h.view != 0) == kept).all()
                else:
                    nu.dropout(dtype, x, rate, key.value, counter, y)
                    assert ((y.view != 0) == kept).all()


def test_dropout_at_rate_zero_copies_and_rows_with_different_strides(cuda_device):
    x = nu.Rows(7, 24, "bfloat16", 8, 0, nu.normal(1, 7, 24))
    y = nu.Rows(7, 24, "bfloat16", 1, 0)
    nu.dropout("bfloat16", x, 0.0, 1, 0, y)
    assert (y.view == x.view).all() and y.outside_untouched()
    z = nu.Rows(7, 24, "bfloat16", 1, 0)
    nu.dropout("bfloat16", x, 0.5, 1, 0, z)
    kept = nu.mask(qb.random.key(1), 7, 24, 0.5)
    assert ((z.wide() == 2 * x.wide()) | ~kept).all() and (z.wide()[~kept] == 0).all()


@pytest.mark.parametrize("rate", [1e-12, 2.0**-33])
def test_a_rate_below_the_draws_resolution_scales_and_drops_nothing(cuda_device, rate):
    x, y, h = nu.Rows(3, 50, "float64", values=nu.normal(1, 3, 50)), nu.Rows(3, 50, "float64"), nu.Rows(3, 50, "float64")
    want = x.view * (1.0 / (1.0 - rate))
    assert not (want == x.view).all()
    nu.dropout("float64", x, rate, 1, 0, y)
    assert (y.view == want).all()
    nu.dropout_layer_norm("float64", "float64", x, None, rate, 1, 0, None, None, h, y, None, None)
    assert (h.view == want).all()


def test_dropped_elements_are_zero_whatever_they_hold(cuda_device):
    import torch

    x = nu.Rows(4, 64, "float32", values=nu.normal(1, 4, 64))
    kept = nu.mask(qb.random.key(1), 4, 64, 0.5)
    x.view[~kept] = float("nan")
    y = nu.Rows(4, 64, "float32")
    nu.dropout("float32", x, 0.5, 1, 0, y)
    assert torch.isfinite(y.view).all() and (y.view[~kept] == 0).all()
    # The residual form: h is finite too.
    h = nu.Rows(4, 64, "float32")
    nu.dropout_layer_norm("float32", "float32", x, None, 0.5, 1, 0, None, None, h, y, None, None)
    assert torch.isfinite(h.view).all() and torch.isfinite(y.view).all()


def test_dropout_backward_is_the_same_mask(cuda_device):
    # y . g == x . dropout(g) for the same key: dropout is its own transpose.
    x, g = (nu.Rows(65, 130, "float64", values=nu.normal(s, 65, 130)) for s in (1, 2))
    y, dx = nu.Rows(65, 130, "float64"), nu.Rows(65, 130, "float64")
    nu.dropout("float64", x, 0.2, 7, 5, y)
    nu.dropout("float64", g, 0.2, 7, 5, dx)
    assert abs((y.view * g.view).sum() - (x.view * dx.view).sum()).item() <= 1e-9


# ---- what the arguments allow -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(nu.CODES))
def test_offsets_past_32_bits(cuda_device, dtype):
    import torch

    # Rows more than 2^32 elements apart (2^31 for the types whose buffer would be larger than needed).
    stride = (1 << 32) + 8 if dtype in ("float16", "bfloat16") else (1 << 31) + 8
    cols = 40
    view = torch.empty(stride + cols, dtype=nu.torch_type(dtype), device="cuda")
    x = nu.Rows(0, cols, dtype)
    x.rows, x.stride = 2, stride
    x.view = torch.as_strided(view, (2, cols), (stride, 1))
    x.view.copy_(nu.normal(1, 2, cols))
    y, mean, rstd = nu.Rows(2, cols, dtype), *(torch.empty(2, dtype=nu.statistics_type(dtype), device="cuda") for _ in range(2))
    nu.layer_norm(dtype, dtype, x, None, None, y, mean, rstd)
    nu.check_forward(dtype, x.wide(), None, None, y, mean, rstd)
    dx, dw = nu.Rows(2, cols, dtype), torch.empty(cols, dtype=nu.torch_type(dtype), device="cuda")
    nu.layer_norm_backward(dtype, dtype, y, x, None, mean, rstd, dx, dw, None)
    nu.check_backward(dtype, dtype, y, x, None, mean, rstd, dx, dw, None)
    nu.dropout(dtype, x, 0.0, 0, 0, y)
    assert (y.view == x.view).all()


def test_more_elements_than_31_bits_count(cuda_device):
    import torch

    lib, n, key, rate = _lib.load(), (1 << 31) + 77, qb.random.key(31), 0.3
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    _lib.check(lib.qb200_dropout(_lib.F16, x.data_ptr(), n, 1, n, rate, key.value, 5, None, x.data_ptr(), n, nu.stream()))
    for first in (0, n - 1000):  # the last thousand lie on both sides of 2^31
        kept = torch.from_numpy(qb.random.dropout_mask(key, (1000,), rate, 5 + first)).cuda()
        assert ((x[first:first + 1000] != 0) == kept).all()
    del x
    rows, cols = (1 << 28) + 3, 8
    x = nu.Rows(0, cols, "float16")
    x.rows, x.view = rows, torch.empty(rows, cols, dtype=torch.float16, device="cuda").normal_()
    y, mean, rstd = torch.empty_like(x.view), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    out = nu.Rows(0, cols, "float16")
    out.rows, out.view = rows, y
    nu.layer_norm("float16", "float16", x, None, None, out, mean, rstd)
    dx = nu.Rows(0, cols, "float16")
    dx.rows, dx.view = rows, torch.empty_like(y)
    nu.layer_norm_backward("float16", "float16", out, x, None, mean, rstd, dx, None, None)
    for first in (0, (1 << 27) - 7, rows - 1000):
        part = slice(first, first + 1000)
        some = nu.Rows(1000, cols, "float16", values=x.view[part])
        got = nu.Rows(1000, cols, "float16", values=y[part])
        nu.check_forward("float16", some.wide(), None, None, got, mean[part], rstd[part])
        nu.check_backward("float16", "float16", got, some, None, mean[part], rstd[part],
                          nu.Rows(1000, cols, "float16", values=dx.view[part]), None, None)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(70, 96), (70, 97), (3, 9000)])
def test_absent_parameters_and_outputs(cuda_device, dtype, rows, cols):
    import torch

    x = nu.Rows(rows, cols, dtype, values=nu.normal(1, rows, cols))
    weight, bias = nu.vector(nu.normal(2, cols), dtype), nu.vector(nu.normal(3, cols), dtype)
    for w, b in ((None, None), (weight, None), (None, bias)):
        y = nu.Rows(rows, cols, dtype)
        nu.layer_norm(dtype, dtype, x, w, b, y, None, None)
        nu.check_forward(dtype, x.wide(), w, b, y, None, None)
    mean, rstd = saved(dtype, x)
    dy, dh = (nu.Rows(rows, cols, dtype, values=nu.normal(s, rows, cols)) for s in (4, 5))
    for want_w, want_b in ((False, False), (True, False), (False, True)):
        dx = nu.Rows(rows, cols, dtype)
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        nu.layer_norm_backward(dtype, dtype, dy, x, weight, mean, rstd, dx, dw, db)
        nu.check_backward(dtype, dtype, dy, x, weight, mean, rstd, dx, dw, db)
        nu.dropout_layer_norm_backward(dtype, dtype, dy, None, x, None, mean, rstd, 0.25, 8, 0, dx, None, dw, db)
        nu.check_backward(dtype, dtype, dy, x, None, mean, rstd, dx, dw, db, kept=nu.mask(qb.random.key(8), rows, cols, 0.25),
                          rate=0.25)
        dres = nu.Rows(rows, cols, dtype)
        nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, x, weight, mean, rstd, 0.0, 8, 0, dx, dres, dw, db)
        nu.check_backward(dtype, dtype, dy, x, weight, mean, rstd, dx, dw, db, dh, dres)
        assert nu.same_bits(dx.view, dres.view)
    # No residual, no h: inference through a block that keeps nothing.
    y = nu.Rows(rows, cols, dtype)
    nu.dropout_layer_norm(dtype, dtype, x, None, 0.0, 0, 0, weight, bias, None, y, None, None)
    nu.check_forward(dtype, x.wide(), weight, bias, y, None, None)


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols,pad", [(50, 64, 0), (50, 63, 0), (9, 1000, 24), (2, 20000, 0)])
def test_results_in_the_place_of_inputs(cuda_device, dtype, rows, cols, pad):
    import torch

    def rows_of(seed):
        return nu.Rows(rows, cols, dtype, pad, 0, nu.normal(seed, rows, cols))

    weight, bias = nu.vector(nu.normal(2, cols), dtype), nu.vector(nu.normal(3, cols), dtype)
    stats = lambda: [torch.empty(rows, dtype=nu.statistics_type(dtype), device="cuda") for _ in range(2)]  # noqa: E731
    y, (mean, rstd), x = nu.Rows(rows, cols, dtype, pad), stats(), rows_of(1)
    nu.layer_norm(dtype, dtype, x, weight, bias, y, mean, rstd)
    nu.layer_norm(dtype, dtype, x, weight, bias, x, None, None)
    assert nu.same_bits(x.view, y.view)

    x, residual, h = rows_of(1), rows_of(4), nu.Rows(rows, cols, dtype, pad)
    nu.dropout_layer_norm(dtype, dtype, x, residual, 0.3, 5, 0, weight, bias, h, y, mean, rstd)
    nu.dropout_layer_norm(dtype, dtype, x, residual, 0.3, 5, 0, weight, bias, residual, x, None, None)
    assert nu.same_bits(residual.view, h.view) and nu.same_bits(x.view, y.view)

    def backward(dy, dh, h, dx, dresidual):
        dw, db = torch.empty_like(weight), torch.empty_like(bias)
        nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, h, weight, mean, rstd, 0.3, 5, 0, dx, dresidual, dw, db)
        return dw, db

    dx, dresidual = nu.Rows(rows, cols, dtype, pad), nu.Rows(rows, cols, dtype, pad)
    dw, db = backward(rows_of(6), rows_of(7), h, dx, dresidual)
    for places in ("dy dh", "dh dy", "dy h", "h dh"):
        arrays = {"dy": rows_of(6), "dh": rows_of(7), "h": nu.Rows(rows, cols, dtype, pad, 0, h.view)}
        first, second = (arrays[p] for p in places.split())
        dw2, db2 = backward(arrays["dy"], arrays["dh"], arrays["h"], first, second)
        assert nu.same_bits(first.view, dx.view) and nu.same_bits(second.view, dresidual.view), places
        assert nu.same_bits(dw, dw2) and nu.same_bits(db, db2)

    for place in ("dy", "x"):
        arrays = {"dy": rows_of(6), "x": nu.Rows(rows, cols, dtype, pad, 0, h.view)}
        dw2 = torch.empty_like(weight)
        nu.layer_norm_backward(dtype, dtype, rows_of(6), h, weight, mean, rstd, dx, dw, None)
        nu.layer_norm_backward(dtype, dtype, arrays["dy"], arrays["x"], weight, mean, rstd, arrays[place], dw2, None)
        assert nu.same_bits(arrays[place].view, dx.view) and nu.same_bits(dw, dw2)

    x, y = rows_of(1), nu.Rows(rows, cols, dtype, pad)
    nu.dropout(dtype, x, 0.3, 5, 0, y)
    nu.dropout(dtype, x, 0.3, 5, 0, x)
    assert nu.same_bits(x.view, y.view)


@pytest.mark.parametrize("cols", [64, 65, 9000])
def test_a_row_that_is_broadcast(cuda_device, cols):
    # Stride 0: one row of gradients for all, as the gradient of a mean over rows is.
    import torch

    rows = 300
    x = nu.Rows(rows, cols, "float32", values=nu.normal(1, rows, cols))
    one = nu.normal(2, 1, cols).float()
    dy = nu.Rows(0, cols, "float32")
    dy.rows, dy.stride, dy.view = rows, 0, one.expand(rows, cols)
    mean, rstd = saved("float32", x)
    dx, dw, db = nu.Rows(rows, cols, "float32"), *(torch.empty(cols, device="cuda") for _ in range(2))
    nu.layer_norm_backward("float32", "float32", dy, x, None, mean, rstd, dx, dw, db)
    nu.check_backward("float32", "float32", dy, x, None, mean, rstd, dx, dw, db)
    y = nu.Rows(rows, cols, "float32")
    nu.layer_norm("float32", "float32", dy, None, None, y, None, None)
    assert (y.view == y.view[0]).all()


def test_no_rows(cuda_device):
    import torch

    weight = torch.ones(24, device="cuda")
    dw, db = torch.full((24,), 5.0, device="cuda"), torch.full((24,), 5.0, device="cuda")
    lib = _lib.load()
    _lib.check(lib.qb200_layer_norm_backward(0, 0, None, 24, None, 24, 0, 24, weight.data_ptr(), None, None, None, 24, dw.data_ptr(),
                                             db.data_ptr(), None, 0, nu.stream()))
    assert (dw == 0).all() and (db == 0).all()
    dw.fill_(5.0)
    _lib.check(lib.qb200_dropout_layer_norm_backward(0, 0, None, 24, None, 24, None, 24, 0, 24, None, None, None, 0.5, 0, 0, None,
                                                     None, 24, None, 24, dw.data_ptr(), None, None, 0, nu.stream()))
    assert (dw == 0).all()


def test_host_memory_is_refused(cuda_device):
    lib = _lib.load()
    host = np.zeros(64, dtype=np.float32)
    at = host.ctypes.data
    assert lib.qb200_layer_norm(0, 0, at, 8, 8, 8, None, None, 1e-5, at, 8, None, None, None) == _lib.INVALID
    assert b"device memory" in lib.qb200_last_error()
    assert lib.qb200_dropout(0, at, 8, 8, 8, 0.5, 0, 0, None, at, 8, None) == _lib.INVALID


@pytest.mark.parametrize("dtype", list(nu.CODES))
def test_rows_without_spread_and_rows_far_from_zero(cuda_device, dtype):
    # A constant row has variance 0: y is the bias, rstd 1 / sqrt(epsilon), all gradients finite.  Rows far from zero
    # keep their small spread: the variance is taken about the mean.
    import torch

    cols = 512
    x = nu.Rows(3, cols, dtype, values=torch.zeros(3, cols, dtype=torch.float64))
    x.view[0] = 2.0
    x.view[1] = (1024.0 + 8.0 * nu.normal(1, cols)).to(x.view.dtype)
    x.view[2] = (nu.normal(2, cols) * 1e-3).to(x.view.dtype)
    bias = nu.vector(nu.normal(3, cols), dtype)
    y = nu.Rows(3, cols, dtype)
    mean, rstd = (torch.empty(3, dtype=nu.statistics_type(dtype), device="cuda") for _ in range(2))
    nu.layer_norm(dtype, dtype, x, None, bias, y, mean, rstd)
    nu.check_forward(dtype, x.wide(), None, bias, y, mean, rstd)
    assert (y.view[0] == bias).all()
    dy, dx, dw = nu.Rows(3, cols, dtype, values=nu.normal(4, 3, cols)), nu.Rows(3, cols, dtype), torch.empty_like(bias)
    nu.layer_norm_backward(dtype, dtype, dy, x, None, mean, rstd, dx, dw, None)
    nu.check_backward(dtype, dtype, dy, x, None, mean, rstd, dx, dw, None)


@pytest.mark.parametrize("cols", [64, 65, 300, 9000])
def test_infinities_and_nans_stay_in_their_rows(cuda_device, cols):
    import torch

    x = nu.Rows(40, cols, "float32", values=nu.normal(1, 40, cols))
    clean, y = nu.Rows(40, cols, "float32"), nu.Rows(40, cols, "float32")
    nu.layer_norm("float32", "float32", x, None, None, clean, None, None)
    x.view[3, cols // 2], x.view[17, 0], x.view[20, cols - 1] = float("nan"), float("inf"), float("-inf")
    nu.layer_norm("float32", "float32", x, None, None, y, None, None)
    spoilt = torch.zeros(40, dtype=torch.bool, device="cuda")
    spoilt[[3, 17, 20]] = True
    assert nu.same_bits(y.view[~spoilt], clean.view[~spoilt])
    assert torch.isnan(y.view[3]).all() and not torch.isfinite(y.view[17, 0]) and not torch.isfinite(y.view[20, cols - 1])


# ---- streams, graphs, repeated calls ----------------------------------------------------------


@pytest.mark.parametrize("dtype,params,rows,cols", [("float32", "float32", 5000, 65), ("bfloat16", "float32", 3000, 1024),
                                                    ("float16", "float16", 40, 20000), ("float64", "float64", 2000, 128)])
def test_the_same_call_gives_the_same_bits(cuda_device, dtype, params, rows, cols):
    import torch

    h, weight, _, _, _ = inputs(dtype, params, rows, cols, 0, 0)
    mean, rstd = saved(dtype, h)
    dy = nu.Rows(rows, cols, dtype, values=nu.normal(5, rows, cols))
    results = []
    for _ in range(3):
        dx, dresidual = nu.Rows(rows, cols, dtype), nu.Rows(rows, cols, dtype)
        dw, db = torch.empty_like(weight), torch.empty_like(weight)
        nu.dropout_layer_norm_backward(dtype, params, dy, dy, h, weight, mean, rstd, 0.1, 3, 0, dx, dresidual, dw, db)
        results.append((dx.view, dresidual.view, dw, db))
    for other in results[1:]:
        assert all(nu.same_bits(a, b) for a, b in zip(results[0], other))


def test_two_streams_with_a_workspace_each(cuda_device):
    import torch

    sizes = [(4000, 256), (3000, 513)]
    made = []
    for i, (rows, cols) in enumerate(sizes):
        x, weight, _, _, _ = inputs("float32", "float32", rows, cols, 0, 0)
        dy = nu.Rows(rows, cols, "float32", values=nu.normal(5 + i, rows, cols))
        made.append((x, weight, *saved("float32", x), dy, nu.Rows(rows, cols, "float32"), torch.empty_like(weight),
                     torch.empty_like(weight), nu.workspace("float32", rows, cols), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for x, weight, mean, rstd, dy, dx, dw, db, space, on in made:
            nu.layer_norm_backward("float32", "float32", dy, x, weight, mean, rstd, dx, dw, db, space, on.cuda_stream)
    torch.cuda.synchronize()
    for x, weight, mean, rstd, dy, dx, dw, db, _, _ in made:
        nu.check_backward("float32", "float32", dy, x, weight, mean, rstd, dx, dw, db)


def test_a_captured_block_draws_a_new_mask_at_every_replay(cuda_device):
    import torch

    rows, cols, rate, key = 200, 320, 0.2, qb.random.key(21)
    x, weight, bias, mean, rstd = inputs("bfloat16", "float32", rows, cols, 0, 0)
    residual = nu.Rows(rows, cols, "bfloat16", values=nu.normal(6, rows, cols))
    dy = nu.Rows(rows, cols, "bfloat16", values=nu.normal(7, rows, cols))
    h, y, dx, dres = (nu.Rows(rows, cols, "bfloat16") for _ in range(4))
    dw, db, space = torch.empty_like(weight), torch.empty_like(weight), nu.workspace("bfloat16", rows, cols)
    position = torch.zeros(1, dtype=torch.int64, device="cuda")
    dropped = nu.Rows(rows, cols, "bfloat16")

    def step():
        nu.dropout_layer_norm("bfloat16", "float32", x, residual, rate, key.value, 7, weight, bias, h, y, mean, rstd, position)
        nu.dropout_layer_norm_backward("bfloat16", "float32", dy, None, h, weight, mean, rstd, rate, key.value, 7, dx, dres, dw,
                                       db, position, space)
        nu.dropout("bfloat16", x, rate, key.value, 7, dropped, position)
        position.add_(rows * cols)

    graph = torch.cuda.CUDAGraph()
    on = torch.cuda.Stream()
    with torch.cuda.stream(on):
        step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=on):
        step()
    for replay in range(1, 4):
        at = 7 + int(position.item())
        assert at == 7 + replay * rows * cols
        graph.replay()
        torch.cuda.synchronize()
        kept = nu.mask(key, rows, cols, rate, at)
        assert ((dropped.wide() != 0) == (kept & (x.wide() != 0))).all()
        want = residual.wide() + nu.dropped(x.wide(), kept, rate)
        nu.check_forward("bfloat16", want, weight, bias, y, mean, rstd)
        nu.check_backward("bfloat16", "float32", dy, h, weight, mean, rstd, dx, dw, db, None, dres, kept, rate)


# ---- gradients against differences, and a block trained from the library's parts ---------------


@pytest.mark.parametrize("rows,cols", [(3, 5), (2, 40), (4, 33)])
def test_gradients_against_differences(cuda_device, rows, cols):
    import torch

    key, rate, step = qb.random.key(4), 0.25, 1e-6
    x, residual = nu.normal(1, rows, cols), nu.normal(2, rows, cols)
    weight, bias = 1 + 0.3 * nu.normal(3, cols), nu.normal(4, cols)
    dy, dh = nu.normal(5, rows, cols), nu.normal(6, rows, cols)

    def loss(x, residual, weight, bias):
        """sum(dy * y) + sum(dh * h) through the device's forward pass."""
        h, y = nu.Rows(rows, cols, "float64"), nu.Rows(rows, cols, "float64")
        nu.dropout_layer_norm("float64", "float64", nu.Rows(rows, cols, "float64", values=x),
                              nu.Rows(rows, cols, "float64", values=residual), rate, key.value, 0, weight, bias, h, y, None, None)
        return ((dy * y.view).sum() + (dh * h.view).sum()).item()

    h, y = nu.Rows(rows, cols, "float64"), nu.Rows(rows, cols, "float64")
    mean, rstd = (torch.empty(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    nu.dropout_layer_norm("float64", "float64", nu.Rows(rows, cols, "float64", values=x),
                          nu.Rows(rows, cols, "float64", values=residual), rate, key.value, 0, weight, bias, h, y, mean, rstd)
    dx, dres = nu.Rows(rows, cols, "float64"), nu.Rows(rows, cols, "float64")
    dw, db = torch.empty_like(weight), torch.empty_like(bias)
    nu.dropout_layer_norm_backward("float64", "float64", nu.Rows(rows, cols, "float64", values=dy),
                                   nu.Rows(rows, cols, "float64", values=dh), h, weight, mean, rstd, rate, key.value, 0, dx, dres,
                                   dw, db)
    arguments = [x, residual, weight, bias]
    for n, gradient in enumerate((dx.view, dres.view, dw, db)):
        for at in np.ndindex(*gradient.shape):
            sides = []
            for sign in (1, -1):
                moved = [a.clone() for a in arguments]
                moved[n][at] += sign * step
                sides.append(loss(*moved))
            # Truncation step^2 f''' / 6 with third derivatives up to about 1e3 here, rounding 1e-15 * |loss| / step.
            assert abs((sides[0] - sides[1]) / (2 * step) - gradient[at].item()) <= 1e-7


def test_a_block_is_trained_from_the_librarys_parts(cuda_device):
    # h = residual + dropout(a W + b), y = layer_norm(h), loss = sum(dy * y): product, block, both gradients, the weight
    # gradient of the product and an Adam update, against the same step in float64 autograd.
    import torch

    from quabla_b200._plan import opt_config

    lib = _lib.load()
    rows, width, inner, rate, key = 5000, 128, 64, 0.1, qb.random.key(77)
    a, residual = nu.normal(1, rows, inner).float(), nu.normal(2, rows, width).float()
    w = (nu.normal(3, inner, width) / 8).float()
    b, gain, shift = (0.1 * nu.normal(4, width)).float(), (1 + 0.1 * nu.normal(5, width)).float(), nu.normal(6, width).float()
    dy = (nu.normal(7, rows, width) / rows).float()
    kept = nu.mask(key, rows, width, rate)
    leaves = [t.double().requires_grad_() for t in (w, b, gain, shift)]
    h64 = residual.double() + nu.dropped(a.double() @ leaves[0] + leaves[1], kept, rate)
    y64 = nu.forward_definition(h64, leaves[2], leaves[3])[0]
    (y64 * dy.double()).sum().backward()

    product = torch.empty(rows, width, device="cuda")
    _lib.check(lib.qb200_matmul_3xtf32(a.data_ptr(), w.data_ptr(), b.data_ptr(), product.data_ptr(), rows, width, inner, rows, nu.stream()))
    branch = nu.Rows(rows, width, "float32", values=product)
    h, y, dx = (nu.Rows(rows, width, "float32") for _ in range(3))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    nu.dropout_layer_norm("float32", "float32", branch, nu.Rows(rows, width, "float32", values=residual), rate, key.value, 0, gain,
                          shift, h, y, mean, rstd)
    dgain, dshift = torch.empty_like(gain), torch.empty_like(shift)
    nu.dropout_layer_norm_backward("float32", "float32", nu.Rows(rows, width, "float32", values=dy), None, h, gain, mean, rstd, rate,
                                   key.value, 0, dx, None, dgain, dshift)
    dw = torch.empty_like(w)
    cotangent = dx.view.contiguous()
    _lib.check(lib.qb200_weight_gradient(_lib.F32, a.data_ptr(), cotangent.data_ptr(), rows, inner, width, dw.data_ptr(), nu.stream()))
    # The product's 2e-6 (its own test's bound) passes through the norm; sums over 5000 rows add a few 1e-6.
    for got, leaf in ((dw, leaves[0]), (dgain, leaves[2]), (dshift, leaves[3])):
        assert ((got.double() - leaf.grad).abs().max() / leaf.grad.abs().max()).item() <= 2e-5
    assert ((y.wide() - y64).abs().max() / y64.abs().max()).item() <= 2e-5
    before = gain.clone()
    m, v = torch.zeros_like(gain), torch.zeros_like(gain)
    config = opt_config("adam", 1e-3, 0.9, 0.999, 1e-8, 0.0)
    _lib.check(lib.qb200_optimizer_apply(_lib.F32, gain.data_ptr(), dgain.data_ptr(), m.data_ptr(), v.data_ptr(), width,
                                         C.byref(config), 1, nu.stream()))
    torch.cuda.synchronize()
    moved = (gain - before).double()
    assert (moved.abs() <= 1.01e-3).all() and (torch.sign(moved) == -torch.sign(leaves[2].grad)).double().mean() > 0.99
