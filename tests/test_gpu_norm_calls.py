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


# ---- sums over very many rows ------------------------------------------------------------------


@pytest.mark.parametrize("dtype,params", nu.TYPE_PAIRS)
@pytest.mark.parametrize("rows,cols", [(262147, 16), (262147, 17), (100003, 64), (50021, 130), (9001, 1024), (5003, 4101), (601, 9000)])
def test_no_row_is_missing_from_the_sums(cuda_device, dtype, params, rows, cols):
    # Small whole numbers, mean 0 and rstd 1: every partial sum is a whole number below 2^24, so the sums are exact in any
    # order, and rounded once where the parameters have 16 bits.
    import torch

    generator = torch.Generator(device="cuda").manual_seed(rows + cols)

    def whole(low, high):
        return torch.randint(low, high + 1, (rows, cols), device="cuda", generator=generator)

    # A mean of a half: with terms of mean 0 a sum could hide a row behind its own rounding in 16 bits.
    dy, x = whole(-1, 2), whole(0, 2)
    dweight, dbias = (dy * x).sum(0), dy.sum(0)
    assert max((dy * x).abs().sum(0).max(), dy.abs().sum(0).max()) < 2**24
    dy, x = nu.Rows(rows, cols, dtype, values=dy), nu.Rows(rows, cols, dtype, values=x)
    mean, rstd = (torch.full((rows,), v, dtype=nu.statistics_type(dtype), device="cuda") for v in (0.0, 1.0))
    for residual in (False, True):
        dx = nu.Rows(rows, cols, dtype)
        got = [torch.full((cols,), float("nan"), dtype=nu.torch_type(params), device="cuda") for _ in range(2)]
        if residual:
            nu.dropout_layer_norm_backward(dtype, params, dy, dy, x, None, mean, rstd, 0.5, 9, 0, dx, None, *got)
        else:
            nu.layer_norm_backward(dtype, params, dy, x, None, mean, rstd, dx, *got)
        for sums, want in zip(got, (dweight, dbias)):
            assert (sums == want.to(sums.dtype)).all()


# ---- arrays that are laid out differently ------------------------------------------------------

# Several turns of the kernels' rows, but for the first two of each width: rows that share a warp, whole warps, several
# blocks.
DIFFERENT = [(3, 40), (40000, 40), (2600, 515), (900, 1024), (3, 5120), (200, 9000)]


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols", DIFFERENT)
@pytest.mark.parametrize("odd", ["x", "residual", "h", "y", "all"])
def test_forward_arrays_with_strides_and_boundaries_of_their_own(cuda_device, dtype, rows, cols, odd):
    # One array off every boundary decides how all of them are read; strides are all different.
    key, rate, counter = qb.random.key(31), 0.3, 2**32 - 5
    layout = {name: dict(pad=-cols % 8 + 8 * i, shift=0) for i, name in enumerate(("x", "residual", "h", "y"))}
    for i, name in enumerate(layout):
        if odd in (name, "all"):
            layout[name] = dict(pad=2 * i + 1 + cols % 2, shift=i + 1)
    x, residual = normal_rows(1, rows, cols, dtype, **layout["x"]), normal_rows(2, rows, cols, dtype, **layout["residual"])
    h, y = nu.Rows(rows, cols, dtype, **layout["h"]), nu.Rows(rows, cols, dtype, **layout["y"])
    weight, bias = nu.vector(1 + 0.2 * nu.normal(3, cols), dtype), nu.vector(nu.normal(4, cols), dtype)
    mean, rstd = statistics(dtype, rows)
    nu.dropout_layer_norm(dtype, dtype, x, residual, rate, key.value, counter, weight, bias, h, y, mean, rstd)
    branch = nu.dropped(x.wide(), nu.mask(key, rows, cols, rate, counter), rate)
    want, u = residual.wide() + branch, nu.unit(dtype)
    # Scale and product round once each, the sum once, then h's own type.
    assert ((h.wide() - want).abs() <= nu.half_step(dtype) * (1 + 8 * u) * want.abs() + 4 * u * (branch.abs() + want.abs())
            + nu.tiny(dtype)).all()
    nu.check_forward(dtype, want, weight, bias, y, mean, rstd)
    assert h.outside_untouched() and y.outside_untouched()
    if odd in ("x", "y"):
        y = nu.Rows(rows, cols, dtype, **layout["y"])
        nu.layer_norm(dtype, dtype, x, weight, bias, y, mean, rstd)
        nu.check_forward(dtype, x.wide(), weight, bias, y, mean, rstd)
        assert y.outside_untouched()


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols", DIFFERENT)
@pytest.mark.parametrize("odd", ["dy", "dh", "h", "dx", "dresidual", "all"])
def test_backward_arrays_with_strides_and_boundaries_of_their_own(cuda_device, dtype, rows, cols, odd):
    import torch

    key, rate, counter = qb.random.key(32), 0.3, 2**62 + 1
    layout = {name: dict(pad=-cols % 8 + 8 * i, shift=0) for i, name in enumerate(("dy", "dh", "h", "dx", "dresidual"))}
    for i, name in enumerate(layout):
        if odd in (name, "all"):
            layout[name] = dict(pad=2 * i + 1 + cols % 2, shift=i + 1)
    dy, dh = normal_rows(1, rows, cols, dtype, 0.1, **layout["dy"]), normal_rows(2, rows, cols, dtype, 0.1, **layout["dh"])
    h = normal_rows(3, rows, cols, dtype, **layout["h"])
    dx, dresidual = nu.Rows(rows, cols, dtype, **layout["dx"]), nu.Rows(rows, cols, dtype, **layout["dresidual"])
    weight = nu.vector(1 + 0.2 * nu.normal(4, cols), dtype)
    wide = h.wide()
    mean = wide.mean(1).to(nu.statistics_type(dtype))
    rstd = (((wide - wide.mean(1, keepdim=True)) ** 2).mean(1) + nu.EPSILON).rsqrt().to(mean.dtype)
    dweight, dbias = torch.full_like(weight, float("nan")), torch.full_like(weight, float("nan"))
    nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, h, weight, mean, rstd, rate, key.value, counter, dx, dresidual, dweight,
                                   dbias)
    nu.check_backward(dtype, dtype, dy, h, weight, mean, rstd, dx, dweight, dbias, dh, dresidual,
                      nu.mask(key, rows, cols, rate, counter), rate)
    assert dx.outside_untouched() and dresidual.outside_untouched()
    if odd in ("dy", "h", "dx"):
        dx = nu.Rows(rows, cols, dtype, **layout["dx"])
        nu.layer_norm_backward(dtype, dtype, dy, h, weight, mean, rstd, dx, dweight, dbias)
        nu.check_backward(dtype, dtype, dy, h, weight, mean, rstd, dx, dweight, dbias)
        assert dx.outside_untouched()


# ---- far offsets, high counters ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("cols", [40, 1000])
def test_all_arrays_past_32_bits(cuda_device, dtype, cols):
    # Every array's second row lies more than 2^32 elements (2^31 of the wider types) behind its first; the arrays stand
    # beside each other in one buffer.
    import torch

    stride = (1 << 32) + 8 if dtype in ("float16", "bfloat16") else (1 << 31) + 8
    buffer = torch.empty(stride + 10 * 1024, dtype=nu.torch_type(dtype), device="cuda")
    for first in (0, stride):
        buffer[first:first + 10 * 1024] = nu.Rows.SENTINEL

    def far(place, seed=None):
        rows = nu.Rows(0, cols, dtype)
        rows.rows, rows.stride = 2, stride
        rows.view = torch.as_strided(buffer, (2, cols), (stride, 1), place * 1024)
        if seed is not None:
            rows.view.copy_(nu.normal(seed, 2, cols))
        return rows

    key, rate, counter = qb.random.key(41), 0.2, 2**62 + 1
    x, residual, h, y, dy, dh, dx, dresidual, dropped = (far(i, i + 1 if i in (0, 1, 4, 5) else None) for i in range(9))
    mean, rstd = statistics(dtype, 2)
    sums = [torch.full((cols,), float("nan"), dtype=nu.torch_type(dtype), device="cuda") for _ in range(2)]
    kept = nu.mask(key, 2, cols, rate, counter)
    nu.dropout_layer_norm(dtype, dtype, x, residual, rate, key.value, counter, None, None, h, y, mean, rstd)
    nu.check_forward(dtype, residual.wide() + nu.dropped(x.wide(), kept, rate), None, None, y, mean, rstd)
    nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, h, None, mean, rstd, rate, key.value, counter, dx, dresidual, *sums)
    nu.check_backward(dtype, dtype, dy, h, None, mean, rstd, dx, *sums, dh, dresidual, kept, rate)
    nu.dropout(dtype, x, rate, key.value, counter, dropped)
    scale = torch.tensor(1.0 / (1.0 - rate), dtype=nu.statistics_type(dtype), device="cuda")
    assert (dropped.view == torch.where(kept, x.view.to(scale.dtype) * scale, 0.0).to(x.view.dtype)).all()
    nu.layer_norm(dtype, dtype, x, None, None, y, mean, rstd)
    nu.check_forward(dtype, x.wide(), None, None, y, mean, rstd)
    nu.layer_norm_backward(dtype, dtype, dy, x, None, mean, rstd, dx, *sums)
    nu.check_backward(dtype, dtype, dy, x, None, mean, rstd, dx, *sums)
    for first in (0, stride):
        between = buffer[first:first + 10 * 1024].view(10, 1024)
        assert (between[:, cols:] == nu.Rows.SENTINEL).all() and (between[9] == nu.Rows.SENTINEL).all()


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols,pad,shift", [(1, 1, 0, 0), (37, 33, 0, 1), (70, 96, 0, 0), (300, 34, 0, 0), (5, 4097, 3, 0), (3, 9000, 0, 0)])
@pytest.mark.parametrize("counter", [1, 2**32 - 5, 2**33 + 1, 2**62 + 1, 2**64 - 2**17])
@pytest.mark.parametrize("rate", [0.3, 0.5 + 2.0**-32])
def test_residual_masks_at_high_counters(cuda_device, dtype, rows, cols, pad, shift, counter, rate):
    import torch

    key = qb.random.key(0xFEDCBA9876543210)
    kept = nu.mask(key, rows, cols, rate, counter)
    one = nu.Rows(rows, cols, dtype, pad, shift, torch.ones(rows, cols, dtype=torch.float64, device="cuda"))
    h, y, dx, dresidual = (nu.Rows(rows, cols, dtype, pad, shift) for _ in range(4))
    mean, rstd = statistics(dtype, rows)
    nu.dropout_layer_norm(dtype, dtype, one, None, rate, key.value, counter, None, None, h, y, mean, rstd)
    assert ((h.view != 0) == kept).all()
    # With dy = 0 the gradient is dh behind the same mask.
    zero = nu.Rows(rows, cols, dtype, pad, shift, torch.zeros(rows, cols, dtype=torch.float64, device="cuda"))
    nu.dropout_layer_norm_backward(dtype, dtype, zero, one, h, None, mean, rstd, rate, key.value, counter, dx, dresidual, None, None)
    assert (dresidual.view == 1).all() and ((dx.view != 0) == kept).all()
    assert nu.same_bits(dx.view, h.view)


@pytest.mark.parametrize("dtype", list(nu.CODES))
@pytest.mark.parametrize("rows,cols", [(40, 64), (40, 65), (41, 1024), (5, 9000)])
def test_nans_stay_in_their_rows_and_columns(cuda_device, dtype, rows, cols):
    # Two 16-bit rows share a turn: what one holds must not reach the other, nor the columns of the sums that it is not in.
    import torch

    x, dy, dh = (normal_rows(seed, rows, cols, dtype) for seed in (1, 2, 3))
    mean, rstd = statistics(dtype, rows)
    y = nu.Rows(rows, cols, dtype)
    nu.layer_norm(dtype, dtype, x, None, None, y, mean, rstd)

    def backward():
        dx = nu.Rows(rows, cols, dtype)
        sums = [torch.full((cols,), 5.0, dtype=nu.torch_type(dtype), device="cuda") for _ in range(2)]
        nu.dropout_layer_norm_backward(dtype, dtype, dy, dh, x, None, mean, rstd, 0.0, 0, 0, dx, None, *sums)
        return dx.view, *sums

    clean_y, clean = y.view.clone(), backward()
    dy.view[2, cols // 3] = float("nan")
    dx, dweight, dbias = backward()
    row, column = torch.arange(rows, device="cuda") == 2, torch.arange(cols, device="cuda") == cols // 3
    assert torch.isnan(dx[2]).all() and nu.same_bits(dx[~row], clean[0][~row])
    for got, want in ((dweight, clean[1]), (dbias, clean[2])):
        assert torch.isnan(got[column]).all() and nu.same_bits(got[~column], want[~column])
    x.view[2, cols - 1] = float("nan")
    nu.layer_norm(dtype, dtype, x, None, None, y, mean, rstd)
    assert torch.isnan(y.view[2]).all() and nu.same_bits(y.view[~row], clean_y[~row])


@pytest.mark.parametrize("captured", [False, True])
def test_calls_in_order_may_share_a_workspace(cuda_device, captured):
    # The sums of one call are joined by a kernel that starts while its rows are still in work; the next call's rows must
    # not reach the workspace before it has read them.
    import torch

    sizes = [("bfloat16", 3000, 1024), ("float32", 5000, 65), ("float32", 40000, 16), ("float64", 300, 4100), ("bfloat16", 37, 20000)]
    space = torch.full((9_699_328,), 255, dtype=torch.uint8, device="cuda")
    made = []
    for i, (dtype, rows, cols) in enumerate(sizes):
        x, dy = normal_rows(2 * i, rows, cols, dtype), normal_rows(2 * i + 1, rows, cols, dtype, 0.1)
        y = nu.Rows(rows, cols, dtype)
        mean, rstd = statistics(dtype, rows)
        nu.layer_norm(dtype, dtype, x, None, None, y, mean, rstd)
        sums = [torch.full((cols,), float("nan"), dtype=nu.torch_type(dtype), device="cuda") for _ in range(2)]
        made.append((dtype, dy, x, mean, rstd, nu.Rows(rows, cols, dtype), sums))

    def calls():
        for dtype, dy, x, mean, rstd, dx, sums in made:
            nu.layer_norm_backward(dtype, dtype, dy, x, None, mean, rstd, dx, *sums, space=space)

    calls()
    torch.cuda.synchronize()
    want = []
    for dtype, dy, x, mean, rstd, dx, sums in made:
        nu.check_backward(dtype, dtype, dy, x, None, mean, rstd, dx, *sums)
        want.append([t.clone() for t in sums])
    run = calls
    if captured:
        on, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=on):
            calls()
        run = graph.replay
    for _ in range(20):
        for *_, sums in made:
            for t in sums:
                t.fill_(float("nan"))
        run()
        for (*_, sums), kept in zip(made, want):
            assert all(nu.same_bits(a, b) for a, b in zip(sums, kept))
