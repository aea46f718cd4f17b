"""Calls of the stand-alone layer norm, dropout and their residual form that their documentation allows: beside other work
on the device, with arrays laid out differently from each other, over far offsets and very many rows.  Bounds: _norm_util."""

import pytest

import quabla_b200 as qb

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
