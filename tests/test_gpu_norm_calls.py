"""Calls of the stand-alone layer norm, dropout and their residual form that their documentation allows: beside other work
on the device, with arrays laid out differently from each other, over far offsets and very many rows.  Bounds: _norm_util."""

import pytest

import quabla_b200 as qb
from quabla_b200 import _lib

import _norm_util as nu

pytestmark = pytest.mark.gpu


def normal_rows(seed, rows, cols, dtype, scale=1.0, **layout):
    return nu.Rows(rows, cols, dtype, values=scale * nu.normal(seed, rows, cols), **layout)


def statistics(dtype, rows):
    import torch

    return [torch.full((rows,), float("nan"), dtype=nu.statistics_type(dtype), device="cuda") for _ in range(2)]


@pytest.mark.parametrize("dtype,rows,cols", [("float32", 1, 8200), ("float32", 40, 50001), ("bfloat16", 150, 65536),
                                             ("float16", 64, 20008), ("float64", 3, 32768), ("float64", 200, 4100)])
def test_rows_over_several_blocks_beside_other_work(cuda_device, dtype, rows, cols):
    # The blocks of a cluster start while other kernels come and go on the multiprocessors.
    import torch

    key, rate = qb.random.key(12), 0.2
    x, residual = normal_rows(1, rows, cols, dtype), normal_rows(2, rows, cols, dtype)
    dy, dh = normal_rows(3, rows, cols, dtype, 0.1), normal_rows(4, rows, cols, dtype, 0.1)
    weight, bias = nu.vector(1 + 0.2 * nu.normal(5, cols), dtype), nu.vector(nu.normal(6, cols), dtype)
    space, on, other = nu.workspace(dtype, rows, cols), torch.cuda.Stream(), torch.cuda.Stream()
    noise = [torch.ones(1 << n, device="cuda") for n in (14, 17, 20, 23)]

    def block():
        h, y, dx, dresidual = (nu.Rows(rows, cols, dtype) for _ in range(4))
        mean, rstd = statistics(dtype, rows)
        dweight, dbias = torch.full_like(weight, float("nan")), torch.full_like(bias, float("nan"))
        on.wait_stream(torch.cuda.current_stream())
        nu.dropout_layer_norm(dtype, dtype, x, residual, rate, key.value, 0, weight, bias, h, y, mean, rstd, on=on.cuda_stream)
        nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, h, weight, mean, rstd, rate, key.value, 0, dx, dresidual, dweight,
                                       dbias, space=space, on=on.cuda_stream)
        torch.cuda.current_stream().wait_stream(on)
        return h, y, mean, rstd, dx, dresidual, dweight, dbias

    quiet = block()
    h, y, mean, rstd, dx, dresidual, dweight, dbias = quiet
    kept = nu.mask(key, rows, cols, rate)
    nu.check_forward(dtype, residual.wide() + nu.dropped(x.wide(), kept, rate), weight, bias, y, mean, rstd)
    nu.check_backward(dtype, dtype, dy, h, weight, mean, rstd, dx, dweight, dbias, dh, dresidual, kept, rate)
    for turn in range(30):
        with torch.cuda.stream(other):
            for i in range(8):
                noise[(turn + i) % 4].mul_(1.0)
        for got, want in zip(block(), quiet):
            if isinstance(got, nu.Rows):
                got, want = got.view, want.view
            assert nu.same_bits(got, want)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("cols", [1, 40, 128, 515, 4096, 9000])
@pytest.mark.parametrize("stride", ["odd", (1 << 62) + 1, -(1 << 61) - 3, 0])
def test_one_rows_strides_are_not_looked_at(cuda_device, dtype, cols, stride):
    import torch

    key, rate = qb.random.key(6), 0.3
    weight, bias = nu.vector(nu.normal(1, cols), dtype), nu.vector(nu.normal(2, cols), dtype)

    def all_calls(stride):
        def row(seed=None):
            made = nu.Rows(1, cols, dtype, values=None if seed is None else nu.normal(seed, 1, cols))
            made.stride = stride
            return made

        x, residual, dy, dh = (row(seed) for seed in (3, 4, 5, 6))
        out = [row() for _ in range(7)]
        mean, rstd = statistics(dtype, 1)
        sums = [torch.full_like(weight, float("nan")) for _ in range(4)]
        nu.dropout(dtype, x, rate, key.value, 0, out[0])
        nu.layer_norm(dtype, dtype, x, weight, bias, out[1], mean, rstd)
        nu.layer_norm_backward(dtype, dtype, dy, x, weight, mean, rstd, out[2], sums[0], sums[1])
        nu.dropout_layer_norm(dtype, dtype, x, residual, rate, key.value, 0, weight, bias, out[3], out[4], mean, rstd)
        nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, out[3], weight, mean, rstd, rate, key.value, 0, out[5], out[6], sums[2],
                                       sums[3])
        for rows in out:
            rows.stride = cols  # the buffer's own, which torch can express
            assert rows.outside_untouched()
        return [rows.view for rows in out] + [mean, rstd] + sums

    for got, want in zip(all_calls(cols + 1 + cols % 2 if stride == "odd" else stride), all_calls(cols)):
        assert nu.same_bits(got, want)


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("stride", [1, -3, (1 << 62) + 1])
def test_strides_of_absent_arrays_are_not_looked_at(cuda_device, dtype, stride):
    # Rows that go 16 bytes at a time go so whatever stands beside a NULL, and their sums run in the same order.
    import torch

    rows, cols, rate, key, code = 200, 1000, 0.25, 17, nu.CODES[dtype]
    lib = _lib.load()
    x, dy = normal_rows(1, rows, cols, dtype), normal_rows(2, rows, cols, dtype)
    weight = nu.vector(1 + 0.2 * nu.normal(3, cols), dtype)

    def both(stride):
        y, dx = nu.Rows(rows, cols, dtype), nu.Rows(rows, cols, dtype)
        mean, rstd = statistics(dtype, rows)
        dweight, dbias = torch.full_like(weight, float("nan")), torch.full_like(weight, float("nan"))
        space = nu.workspace(dtype, rows, cols)
        _lib.check(lib.qb200_dropout_layer_norm(code, code, x.ptr, cols, None, stride, rows, cols, rate, key, 0, None,
                                                weight.data_ptr(), None, nu.EPSILON, None, stride, y.ptr, cols, mean.data_ptr(),
                                                rstd.data_ptr(), nu.stream()))
        _lib.check(lib.qb200_dropout_layer_norm_backward(code, code, dy.ptr, cols, None, stride, x.ptr, cols, rows, cols,
                                                         weight.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rate, key, 0, None,
                                                         dx.ptr, cols, None, stride, dweight.data_ptr(), dbias.data_ptr(),
                                                         space.data_ptr(), space.numel(), nu.stream()))
        return y.view, mean, rstd, dx.view, dweight, dbias

    for got, want in zip(both(stride), both(0)):
        assert nu.same_bits(got, want)
