"""Callers and 64-bit definitions of the stand-alone layer norm and dropout, with the error bounds of the tests.

Bounds.  u is half a step of the accumulation type (2^-24, float64 2^-53), eps_t / 2 half a step of the result's type.
A sum over a row's columns passes through at most 16 additions in a thread, 5 between lanes, 16 between warps and 8
between CTAs: an error of at most 45 u times the sum of the terms' magnitudes.  With the roundings of the terms
themselves, of the quotients and of what follows, 64 u covers every first-order term below.
"""

import ctypes as C
import math

from quabla_b200 import _lib
from quabla_b200 import random as qr

EPSILON = 1e-5
CODES = {"float32": _lib.F32, "float64": _lib.F64, "float16": _lib.F16, "bfloat16": _lib.BF16}
TYPE_PAIRS = [("float32", "float32"), ("float64", "float64"), ("float16", "float16"), ("float16", "float32"),
              ("bfloat16", "bfloat16"), ("bfloat16", "float32")]


def torch_type(name):
    import torch

    return getattr(torch, name)


def statistics_type(dtype):
    import torch

    return torch.float64 if dtype == "float64" else torch.float32


def unit(dtype):
    """u of the accumulation type."""
    return 2.0**-53 if dtype == "float64" else 2.0**-24


def half_step(dtype):
    import torch

    return torch.finfo(torch_type(dtype)).eps / 2


def tiny(dtype):
    """Half a step among subnormal numbers of the type (float16 results get that small)."""
    import torch

    info = torch.finfo(torch_type(dtype))
    return info.smallest_normal * info.eps / 2


class Rows:
    """[rows][cols] of dtype inside rows of `stride` elements that start `shift` elements into a buffer.  What is not
    part of the rows holds a sentinel."""

    SENTINEL = 77.0

    def __init__(self, rows, cols, dtype, pad=0, shift=0, values=None, stride=None):
        import torch

        self.rows, self.cols = rows, cols
        self.stride = cols + pad if stride is None else stride
        size = shift + max(0, rows - 1) * self.stride + (cols if rows else 0) + 5
        self.buffer = torch.full((size,), self.SENTINEL, dtype=torch_type(dtype), device="cuda")
        self.view = torch.as_strided(self.buffer, (rows, cols), (self.stride, 1), shift)
        if values is not None:
            self.view.copy_(values)

    @property
    def ptr(self):
        return self.view.data_ptr() if self.rows else None

    def wide(self):
        return self.view.double()

    def outside_untouched(self):
        import torch

        mask = torch.ones_like(self.buffer, dtype=torch.bool)
        torch.as_strided(mask, (self.rows, self.cols), (self.stride, 1), self.view.storage_offset()).fill_(False)
        return bool((self.buffer[mask] == self.SENTINEL).all())


def normal(seed, *shape):
    import torch

    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, dtype=torch.float64, device="cuda", generator=generator)


def vector(values, dtype):
    return values.to(torch_type(dtype))


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def address(t):
    return None if t is None else t.data_ptr()


def layer_norm(dtype, params, x, weight, bias, y, mean, rstd, epsilon=EPSILON, on=None):
    _lib.check(_lib.load().qb200_layer_norm(CODES[dtype], CODES[params], x.ptr, x.stride, x.rows, x.cols, address(weight),
                                            address(bias), epsilon, y.ptr, y.stride, address(mean), address(rstd),
                                            stream() if on is None else on))


def workspace(dtype, rows, cols):
    import torch

    size = C.c_size_t()
    _lib.check(_lib.load().qb200_layer_norm_workspace(CODES[dtype], rows, cols, C.byref(size)))
    # Not zero: what an earlier use left must not matter.
    return torch.full((max(size.value, 16),), 255, dtype=torch.uint8, device="cuda")


def layer_norm_backward(dtype, params, dy, x, weight, mean, rstd, dx, dweight, dbias, space=None, on=None):
    if space is None and (dweight is not None or dbias is not None):
        space = workspace(dtype, x.rows, x.cols)
    _lib.check(_lib.load().qb200_layer_norm_backward(
        CODES[dtype], CODES[params], dy.ptr, dy.stride, x.ptr, x.stride, x.rows, x.cols, address(weight), address(mean),
        address(rstd), dx.ptr, dx.stride, address(dweight), address(dbias), address(space),
        0 if space is None else space.numel(), stream() if on is None else on))


def dropout(dtype, x, rate, key, counter, y, d_counter=None, on=None):
    _lib.check(_lib.load().qb200_dropout(CODES[dtype], x.ptr, x.stride, x.rows, x.cols, rate, key, counter,
                                         address(d_counter), y.ptr, y.stride, stream() if on is None else on))


def dropout_layer_norm(dtype, params, x, residual, rate, key, counter, weight, bias, h, y, mean, rstd, d_counter=None,
                       epsilon=EPSILON, on=None):
    _lib.check(_lib.load().qb200_dropout_layer_norm(
        CODES[dtype], CODES[params], x.ptr, x.stride, residual and residual.ptr, residual.stride if residual else 0, x.rows,
        x.cols, rate, key, counter, address(d_counter), address(weight), address(bias), epsilon, h and h.ptr,
        h.stride if h else 0, y.ptr, y.stride, address(mean), address(rstd), stream() if on is None else on))


def dropout_layer_norm_backward(dtype, params, dy, dh, h, weight, mean, rstd, rate, key, counter, dx, dresidual, dweight,
                                dbias, d_counter=None, space=None, on=None):
    if space is None and (dweight is not None or dbias is not None):
        space = workspace(dtype, h.rows, h.cols)
    _lib.check(_lib.load().qb200_dropout_layer_norm_backward(
        CODES[dtype], CODES[params], dy.ptr, dy.stride, dh and dh.ptr, dh.stride if dh else 0, h.ptr, h.stride, h.rows,
        h.cols, address(weight), address(mean), address(rstd), rate, key, counter, address(d_counter), dx.ptr, dx.stride,
        dresidual and dresidual.ptr, dresidual.stride if dresidual else 0, address(dweight), address(dbias), address(space),
        0 if space is None else space.numel(), stream() if on is None else on))


def mask(key, rows, cols, rate, counter=0):
    import torch

    return torch.from_numpy(qr.dropout_mask(key, (rows, cols), rate, counter)).cuda()


def dropped(x, kept, rate):
    import torch

    return torch.where(kept, x / (1.0 - rate), 0.0)


# ---- definitions in 64 bits, and how far a result may be from them ----------------------------


def forward_definition(h, weight, bias, epsilon=EPSILON):
    """(y, mean, rstd) and the magnitudes that the bound of y goes by, for h in float64."""
    cols = h.shape[1]
    mean = h.sum(1, keepdim=True) / cols
    variance = ((h - mean) ** 2).sum(1, keepdim=True) / cols
    rstd = (variance + epsilon) ** -0.5
    xh = (h - mean) * rstd
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    y = xh * w + b
    magnitude = abs(w) * (h.abs().mean(1, keepdim=True) * rstd + h.abs() * rstd + xh.abs()) + abs(b)
    return y, mean.reshape(-1), rstd.reshape(-1), magnitude


def check_forward(dtype, h, weight, bias, y, mean, rstd, epsilon=EPSILON):
    want_y, want_mean, want_rstd, magnitude = forward_definition(h, weight, bias, epsilon)
    u = unit(dtype)
    bound = half_step(dtype) * (1 + 64 * u) * want_y.abs() + 64 * u * magnitude + tiny(dtype)
    assert ((y.wide() - want_y).abs() <= bound).all()
    if mean is not None:
        assert ((mean.double() - want_mean).abs() <= 64 * u * h.abs().mean(1)).all()
    if rstd is not None:
        # The mean's error enters the variance squared; beside a variance near zero epsilon holds it down.
        spread = (64 * u * h.abs().mean(1)) ** 2 * want_rstd**2
        assert ((rstd.double() - want_rstd).abs() <= (64 * u + spread) * want_rstd).all()


def backward_definition(dy, h, weight, mean, rstd):
    cols = h.shape[1]
    mean, rstd = mean.double().unsqueeze(1), rstd.double().unsqueeze(1)
    xh = (h - mean) * rstd
    g = dy if weight is None else dy * weight.double()
    along_one = g.sum(1, keepdim=True) / cols
    along_normal = (g * xh).sum(1, keepdim=True) / cols
    dh = rstd * (g - along_one - xh * along_normal)
    magnitude = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    return dh, magnitude, (dy * xh), dy


def check_sum(terms, result, dtype, params):
    """A gradient that is a sum over rows.  A thread adds the rows of its group in turn (at least 18 clusters of CTAs
    share many rows), then up to 256 groups are added, the rest in double."""
    rows = terms.shape[0]
    depth = (rows if rows < 512 else math.ceil(rows / 18)) + 256 + 8
    want = terms.sum(0)
    bound = half_step(params) * 1.001 * want.abs() + depth * unit(dtype) * terms.abs().sum(0) + tiny(params)
    assert ((result.double() - want).abs() <= bound).all()


def check_backward(dtype, params, dy, h, weight, mean, rstd, dx, dweight, dbias, dh=None, dresidual=None, kept=None, rate=0.0):
    want, magnitude, along_weight, along_bias = backward_definition(dy.wide(), h.wide(), weight, mean, rstd)
    if dh is not None:
        want = want + dh.wide()
        magnitude = magnitude + dh.wide().abs()
    u = unit(dtype)
    if dresidual is not None:
        bound = half_step(dtype) * (1 + 64 * u) * want.abs() + 64 * u * magnitude + tiny(dtype)
        assert ((dresidual.wide() - want).abs() <= bound).all()
    if kept is not None:
        want, magnitude = dropped(want, kept, rate), magnitude / (1.0 - rate)
    bound = half_step(dtype) * (1 + 64 * u) * want.abs() + 64 * u * magnitude + tiny(dtype)
    assert ((dx.wide() - want).abs() <= bound).all()
    if kept is not None:
        assert (dx.wide()[~kept] == 0).all()
    if dweight is not None:
        check_sum(along_weight, dweight, dtype, params)
    if dbias is not None:
        check_sum(along_bias, dbias, dtype, params)


def same_bits(a, b):
    import torch

    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
