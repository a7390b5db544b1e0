"""The operators (GPU) where calls meet limits: waits that give up, buffers that
end with their last value, operands of different alignment, workspaces of
other calls. The plain implementations and bounds are test_operators_gpu.py's.
"""

import pytest

from test_operators_gpu import (HALF_ULP, TINY, U, _back64, _back_inputs, _linear_inputs, _linear_want, _norm64,
                                _norm_bounds, _norm_inputs, _padded, _product, _quantise_steps, _run_back, _run_linear,
                                _within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import dmx

    o = dmx.Ops(0)
    yield o
    o.check()
    o.close()


# --- waits that give up -------------------------------------------------------

# every kernel with waits: k split over a cluster and not, tiles of one CTA and
# of a pair, one round of tiles and many, one stage of k and many
@pytest.mark.parametrize("m,n,k", [(17, 130, 1100), (20, 300, 2050), (100, 512, 8192), (12, 64, 48), (300, 128, 512),
                                   (700, 2055, 1000), (20001, 40, 200), (8192, 4096, 2048), (9001, 2050, 130)])
def test_calls_behind_a_raised_flag_end_and_the_next_ones_are_right(ops, m, n, k):
    import dmx
    import torch

    x, w, xs, ws, b = _linear_inputs(m, n, k, m + k)
    want, bound = _linear_want(_product(x, w, k), xs, ws, b, 0, None, "f32")
    first = _run_linear(ops, x, w, k, "f32", xs, ws, b).clone()
    _within(first, want, bound, "before")
    for _ in range(3):
        ops.selftest_wait_timeout(20)
        for _ in range(4):
            _run_linear(ops, x, w, k, "f32", xs, ws, b)
        with pytest.raises(dmx.DmxError, match="self-test kernel: a bounded wait gave up") as e:
            ops.check()
        assert e.value.code == 4
        ops.check()  # reported once
        assert torch.equal(_run_linear(ops, x, w, k, "f32", xs, ws, b), first)
        ops.check()


def test_a_failure_is_the_contexts_and_reported_once_on_any_stream():
    import dmx
    import torch

    one, other = dmx.Ops(0), dmx.Ops(0)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    one.selftest_wait_timeout(20, a.cuda_stream)
    a.synchronize()
    other.check(a.cuda_stream)  # another context: not its failure
    with pytest.raises(dmx.DmxError, match="on any stream since the last check"):
        one.check(b.cuda_stream)
    for stream in (0, a.cuda_stream, b.cuda_stream):
        one.check(stream)
        other.check(stream)
    one.close()
    other.close()


def test_the_self_test_of_a_wait_refuses_other_limits(ops):
    import dmx

    for ms in (0, -1, 5001):
        with pytest.raises(dmx.DmxError, match="wait_ms") as e:
            ops.selftest_wait_timeout(ms)
        assert e.value.code == 1
    ops.check()


# --- rows copied ahead --------------------------------------------------------

# many rows to each group of threads, so that every stage of its ring of copies
# is read and filled again, at each depth of the ring and one or two rows at a time
@pytest.mark.parametrize("rows,cols,pad", [(5003, 1032, 0), (4001, 2048, 0), (2611, 4099, 5), (1999, 8195, 5),
                                           (1501, 10248, 0), (1207, 12288, 0), (1103, 16384, 0)])
@pytest.mark.parametrize("xt,dyt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32")])
def test_backward_of_many_long_rows(ops, rows, cols, pad, xt, dyt):
    dy, x, w, mean, rstd = _back_inputs(rows, cols, xt, dyt, rows + cols)
    _, dyv = _padded(dy, dy.dtype, pad)
    _, xv = _padded(x, x.dtype, pad)
    dx, dw, db = _run_back(ops, dyv, xv, w, mean, rstd, pad=pad)
    dx64, dw64, db64, e_dx, e_w, e_b = _back64(dy, x, w, mean, rstd)
    _within(dx, dx64, e_dx + HALF_ULP[xt] * (dx64.abs() + e_dx) + TINY[xt], "dx")
    _within(dw, dw64, e_w, "dweight")
    _within(db, db64, e_b, "dbias")


# --- buffers that end with their last value -----------------------------------

@pytest.mark.parametrize("k", [1, 3, 15, 17, 100, 509, 1031, 2050, 4097])
@pytest.mark.parametrize("m,n", [(1, 7), (2, 64), (4, 1001), (8, 130), (20, 96), (300, 33)])
def test_quantized_linear_of_buffers_that_end_with_the_last_row(ops, m, n, k):
    import torch

    x, w, xs, ws, b = _linear_inputs(m, n, k, m + n + k)
    ld = x.shape[1]

    def cut(t):  # the same rows, the last one without its padding
        flat = torch.empty((t.shape[0] - 1) * ld + k, dtype=torch.int8, device="cuda")
        rows = flat.as_strided((t.shape[0], k), (ld, 1))
        rows.copy_(t[:, :k])
        return rows

    got = _run_linear(ops, cut(x), cut(w), k, "f32", xs, ws, b)
    want, bound = _linear_want(_product(x, w, k), xs, ws, b, 0, None, "f32")
    _within(got, want, bound, "out")


# --- errors that are not the operators' ---------------------------------------

def test_an_error_the_caller_left_is_neither_reported_nor_cleared(ops):
    import ctypes

    import torch

    rt = ctypes.CDLL("libcudart.so.12")  # the one that the library and torch are linked to
    x, y, dx = torch.randn(3, 40, 48, device="cuda")
    mean, rstd, s = torch.ones(3, 40, device="cuda")
    dw = torch.empty(48, device="cuda")
    q, w = torch.zeros(2, 40, 48, dtype=torch.int8, device="cuda")
    room = torch.empty(ops.layer_norm_backward_workspace(40, 48), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    p = torch.Tensor.data_ptr
    calls = [lambda: ops.layer_norm(p(x), 0, 40, 48, p(y), 0),
             lambda: ops.layer_norm_backward(p(y), 0, p(x), 0, p(mean), p(rstd), 40, 48, p(room), room.numel(),
                                             dx=p(dx), dweight=p(dw)),
             lambda: ops.quantize_rows(p(x), 0, 40, 48, p(q), p(s)),
             lambda: ops.layer_norm_quantize(p(x), 0, 40, 48, p(q), p(s)),
             lambda: ops.quantized_linear(p(q), p(w), p(y), 0, 40, 40, 48),
             lambda: ops.quantized_linear(p(q), p(w), p(y), 0, 1, 40, 48)]
    for call in calls:
        assert rt.cudaSetDevice(100000) == 101  # cudaErrorInvalidDevice: a mistake of the caller's own
        call()
        assert rt.cudaGetLastError() == 101 and rt.cudaGetLastError() == 0
    ops.check()


# --- workspaces of other calls ------------------------------------------------

@pytest.mark.parametrize("most,fewer,cols", [(2688, (2376, 2368, 2361, 17), 512), (4095, (444, 443, 297, 148, 3), 8195),
                                             (6000, (4737, 4736, 300), 257), (3000, (1777, 1776, 740), 1500),
                                             (700, (296, 148), 17000)])
@pytest.mark.parametrize("shift", [0, 1])
def test_backward_in_the_workspace_of_a_larger_call(ops, most, fewer, cols, shift):
    # a training loop's workspace, made for its largest batch; rows on 16 bytes and off them
    import torch

    size = ops.layer_norm_backward_workspace(most, cols)
    room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    for rows in (most, *fewer):
        dy, x, w, mean, rstd = _back_inputs(rows, cols, "bf16", "bf16", rows)
        pad = (-cols) % 8 + shift
        _, dyv = _padded(dy, dy.dtype, pad)
        _, xv = _padded(x, x.dtype, pad)
        want = _run_back(ops, dyv, xv, w, mean, rstd, pad=pad)
        dx = torch.empty(rows, cols + pad, dtype=x.dtype, device="cuda")[:, :cols]
        dw, db = torch.empty(2, cols, device="cuda")
        ops.layer_norm_backward(dyv.data_ptr(), 2, xv.data_ptr(), 2, mean.data_ptr(), rstd.data_ptr(), rows, cols,
                                room.data_ptr(), size, weight=w.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(),
                                dbias=db.data_ptr(), dy_ld=cols + pad, x_ld=cols + pad, dx_ld=cols + pad)
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), want)), rows
        assert (room[size:] == 0xAB).all(), "wrote past the workspace"


# --- the GELU on its whole range ----------------------------------------------

def _gelu_of(ops, z, m, ot):
    """GELU of the f32 values z (a bias on sums of zero), through the kernel for m rows; one row of it."""
    import torch

    n, k = z.numel(), 1040
    x = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    out = _run_linear(ops, x, w, k, ot, None, None, z, 1)
    assert (out == out[:1]).all() or out.isnan().any()
    return out[0]


# rows of the three kernels, and of tiles of both widths
@pytest.mark.parametrize("m", [1, 2, 5, 20, 100, 700])
@pytest.mark.parametrize("ot", ["f32", "f16", "bf16"])
def test_gelu_and_its_tail(ops, m, ot):
    # f32: the fit is within 5.2e-8 |z|, the roundings of its sum and products and
    # ex2 (2^-22 of the exponential, at most 1/2 of which is R's) within 2.4e-7 |z|;
    # every one of them shrinks with the exponential, and below -4 the fit's clamp is
    # within 4.6 % of the value: the tail is held to 5 % of it, from -4 up to 0.3 %.
    # ex2 is 0 below f32's normal numbers.
    import torch

    z = torch.cat([torch.linspace(-14, 14, 60001), torch.linspace(-0.01, 0.01, 2001),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e5, -1e5, 3e38, -3e38])]).cuda()
    zd = z.double()
    tail = 0.5 * torch.special.erfc(zd.abs() / 2**0.5) * zd.abs()  # what max(z, 0) is less by
    want = zd.clamp(min=0) - tail
    bound = torch.minimum(3e-7 * zd.abs(), torch.where(zd.abs() > 4, 0.05, 0.003) * tail) + 2.0**-126 * zd.abs()
    bound = bound + 2.0**-24 * want.abs()
    got = _gelu_of(ops, z, m, ot)
    big = HALF_ULP[ot] * (want.abs() + bound) + TINY[ot]
    keep = want.abs() < (60000 if ot == "f16" else 1e38)  # others leave the type
    _within(got[keep], want[keep], (bound + big)[keep], "gelu")


@pytest.mark.parametrize("m", [1, 20, 700])
def test_gelu_of_what_is_not_finite(ops, m):
    import torch

    inf, nan = float("inf"), float("nan")
    got = _gelu_of(ops, torch.tensor([inf, -inf, nan, 1.0], device="cuda"), m, "f32")
    assert got[0] == inf and got[1] == 0 and got[2].isnan() and 0.841 < got[3] < 0.842


# --- one row of many weights --------------------------------------------------

# both sides of where weights are streamed, and where k or the channels are few
@pytest.mark.parametrize("n,k", [(70000, 1024), (33001, 2048), (32900, 2049), (40000, 2050), (8191, 8193), (8200, 8192),
                                 (2048, 40000), (2049, 40001), (700, 128000), (1, 131071)])
@pytest.mark.parametrize("ot", ["f32", "bf16"])
def test_quantized_linear_of_one_row_and_many_weights(ops, n, k, ot):
    x, w, xs, ws, b = _linear_inputs(1, n, k, n + k)
    xs = xs / k**0.5
    got = _run_linear(ops, x, w, k, ot, xs, ws, b)
    # columns in pieces: the product in 64 bits of all of them would be gigabytes
    for at in range(0, n, 8192):
        part = slice(at, min(at + 8192, n))
        want, bound = _linear_want(_product(x, w[part], k), xs, ws[part], b[part], 0, None, ot)
        _within(got[:, part], want, bound, "out")


# --- long rows off 16 bytes ---------------------------------------------------

# one, two and three blocks to an SM, by shifted vectors and (a weight of a third
# type) by elements; more rows than blocks, so that each takes several
@pytest.mark.parametrize("rows,cols", [(3001, 1031), (2003, 2001), (1801, 3001), (1501, 4097), (1203, 5003), (1001, 5201),
                                       (801, 8191), (701, 8195), (503, 12001), (401, 16383)])
@pytest.mark.parametrize("xt,dyt,params", [("bf16", "bf16", "bf16"), ("f32", "bf16", "f32"), ("f16", "f32", "bf16")])
def test_backward_of_many_rows_off_16_bytes(ops, rows, cols, xt, dyt, params):
    dy, x, w, mean, rstd = _back_inputs(rows, cols, xt, dyt, rows + cols, params)
    dx, dw, db = _run_back(ops, dy, x, w, mean, rstd, params=params)
    dx64, dw64, db64, e_dx, e_w, e_b = _back64(dy, x, w, mean, rstd)
    _within(dx, dx64, e_dx + HALF_ULP[xt] * (dx64.abs() + e_dx) + TINY[xt], "dx")
    _within(dw, dw64, e_w, "dweight")
    _within(db, db64, e_b, "dbias")


# --- operands of different alignment ------------------------------------------

CODE = {"f32": 0, "f16": 1, "bf16": 2}


def _placed(values, skip, pad=0, fill=7.0):
    """The rows (or vector) at `skip` elements past an allocation's start, `pad` elements apart; and what is around."""
    import torch

    rows = values if values.dim() == 2 else values[None]
    ld = rows.shape[1] + pad
    flat = torch.full((skip + rows.shape[0] * ld + 3,), fill, dtype=values.dtype, device="cuda")
    view = flat[skip:skip + rows.shape[0] * ld].view(rows.shape[0], ld)[:, :rows.shape[1]]
    view.copy_(rows)
    around = torch.ones_like(flat, dtype=torch.bool)
    around[skip:skip + rows.shape[0] * ld].view(rows.shape[0], ld)[:, :rows.shape[1]] = False
    return view if values.dim() == 2 else view[0], lambda: (flat[around] == fill).all()


# (x, y, weight, bias): where each begins and the rows' padding
@pytest.mark.parametrize("skips,pads", [((0, 1, 0, 0), (0, 0)), ((1, 0, 0, 0), (0, 0)), ((0, 0, 1, 0), (0, 0)),
                                        ((0, 0, 0, 1), (0, 0)), ((4, 4, 4, 4), (0, 4)), ((8, 4, 0, 0), (8, 12)),
                                        ((3, 5, 1, 2), (1, 2)), ((0, 0, 0, 0), (8, 1))])
@pytest.mark.parametrize("rows,cols", [(9, 64), (700, 512), (5000, 512), (6, 2048), (900, 4104), (3, 17000)])
@pytest.mark.parametrize("xt,yt,params", [("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("f16", "f16", "f16")])
def test_layer_norm_of_operands_of_different_alignment(ops, skips, pads, rows, cols, xt, yt, params):
    import torch

    x, w, b = _norm_inputs(rows, cols, xt, rows + cols, params)
    xv, _ = _placed(x, skips[0], pads[0])
    like = torch.zeros(rows, cols, device="cuda", dtype=dict(f32=torch.float32, f16=torch.float16,
                                                             bf16=torch.bfloat16)[yt])
    yv, alone = _placed(like, skips[1], pads[1])
    wv, bv = _placed(w, skips[2])[0], _placed(b, skips[3])[0]
    torch.cuda.synchronize()
    ops.layer_norm(xv.data_ptr(), CODE[xt], rows, cols, yv.data_ptr(), CODE[yt], weight=wv.data_ptr(),
                   bias=bv.data_ptr(), param_type=CODE[params], x_ld=xv.stride(0), y_ld=yv.stride(0))
    torch.cuda.synchronize()
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    e = _norm_bounds(x, h, want, w, m64, r64)[2]
    _within(yv, want, e + HALF_ULP[yt] * (want.abs() + e) + TINY[yt], "y")
    assert alone(), "wrote past the rows"


# (dy, x, dx, weight), their padding, and the workspace's start in bytes
@pytest.mark.parametrize("skips,pads,room_at", [((1, 0, 0, 0), (0, 0, 0), 0), ((0, 1, 0, 0), (0, 0, 0), 16),
                                                ((0, 0, 1, 0), (0, 0, 0), 0), ((0, 0, 0, 1), (0, 0, 0), 0),
                                                ((4, 0, 4, 4), (0, 0, 4), 48), ((8, 8, 0, 0), (8, 0, 16), 16),
                                                ((3, 1, 5, 2), (1, 2, 0), 16), ((0, 0, 0, 0), (0, 0, 0), 16)])
@pytest.mark.parametrize("rows,cols", [(40, 64), (1500, 512), (900, 2048), (320, 8200), (7, 17000)])
@pytest.mark.parametrize("xt,dyt,params", [("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("f16", "f16", "f16")])
def test_backward_of_operands_of_different_alignment(ops, skips, pads, room_at, rows, cols, xt, dyt, params):
    import torch

    dy, x, w, mean, rstd = _back_inputs(rows, cols, xt, dyt, rows + cols, params)
    dyv, xv = _placed(dy, skips[0], pads[0])[0], _placed(x, skips[1], pads[1])[0]
    dxv, alone = _placed(torch.zeros_like(x), skips[2], pads[2])
    wv = _placed(w, skips[3])[0]
    dw, db = torch.empty(2, cols, device="cuda")
    size = ops.layer_norm_backward_workspace(rows, cols)
    room = torch.full((room_at + size + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ops.layer_norm_backward(dyv.data_ptr(), CODE[dyt], xv.data_ptr(), CODE[xt], mean.data_ptr(), rstd.data_ptr(), rows,
                            cols, room.data_ptr() + room_at, size, weight=wv.data_ptr(), param_type=CODE[params],
                            dx=dxv.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(), dy_ld=dyv.stride(0),
                            x_ld=xv.stride(0), dx_ld=dxv.stride(0))
    torch.cuda.synchronize()
    dx64, dw64, db64, e_dx, e_w, e_b = _back64(dy, x, w, mean, rstd)
    _within(dxv, dx64, e_dx + HALF_ULP[xt] * (dx64.abs() + e_dx) + TINY[xt], "dx")
    _within(dw, dw64, e_w, "dweight")
    _within(db, db64, e_b, "dbias")
    assert alone(), "wrote past the rows"
    assert (room[:room_at] == 0xAB).all() and (room[room_at + size:] == 0xAB).all(), "wrote past the workspace"


# (x, q, col_scale) and the padding of x and q
@pytest.mark.parametrize("skips,pads", [((0, 1, 0), (0, 0)), ((1, 0, 0), (0, 0)), ((0, 0, 1), (0, 0)), ((4, 8, 4), (4, 8)),
                                        ((0, 16, 0), (8, 3)), ((3, 5, 2), (1, 7))])
@pytest.mark.parametrize("rows,cols", [(9, 64), (5000, 512), (300, 2048), (40, 8200), (3, 17000)])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_quantise_operands_of_different_alignment(ops, skips, pads, rows, cols, xt):
    import numpy as np
    import torch

    x, w, _ = _norm_inputs(rows, cols, xt, rows + cols, "f32")
    xv, wv = _placed(x, skips[0], pads[0])[0], _placed(w, skips[2])[0]
    qv, alone = _placed(torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), skips[1], pads[1], 7)
    scale = torch.empty(rows, device="cuda")
    torch.cuda.synchronize()
    ops.quantize_rows(xv.data_ptr(), CODE[xt], rows, cols, qv.data_ptr(), scale.data_ptr(), col_scale=wv.data_ptr(),
                      x_ld=xv.stride(0), q_ld=qv.stride(0))
    torch.cuda.synchronize()
    want_q, want_scale = _quantise_steps((x.float() * w).cpu().numpy())
    assert np.array_equal(scale.cpu().numpy(), want_scale) and np.array_equal(qv.cpu().numpy(), want_q)
    assert alone(), "wrote past the rows"
    # and with the norm before it, the same parameters as weight and bias
    mean, rstd = torch.empty(2, rows, device="cuda")
    ops.layer_norm_quantize(xv.data_ptr(), CODE[xt], rows, cols, qv.data_ptr(), scale.data_ptr(), weight=wv.data_ptr(),
                            bias=wv.data_ptr(), x_ld=xv.stride(0), q_ld=qv.stride(0), mean=mean.data_ptr(),
                            rstd=rstd.data_ptr())
    torch.cuda.synchronize()
    h, y, m64, r64 = _norm64(x, w, w, 1e-5)
    e_mean, e_rstd, e_y = _norm_bounds(x, h, y, w, m64, r64)
    _within(mean[:, None], m64, e_mean, "mean")
    _within(rstd[:, None], r64, e_rstd, "rstd")
    s = scale.double()[:, None]
    off = (qv.double() - y / s).abs()
    assert (off <= 0.5 + (e_y + 4 * U * y.abs()) / s + 1e-5).all(), off.max().item()
    assert alone(), "wrote past the rows"


# (out, residual, scales and bias) and the padding of out and residual
@pytest.mark.parametrize("skips,pads", [((0, 1, 0), (0, 0)), ((1, 0, 0), (0, 0)), ((0, 0, 1), (0, 0)), ((4, 8, 3), (4, 8)),
                                        ((8, 4, 0), (8, 4)), ((3, 5, 2), (1, 7))])
@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (6, 136, 512), (20, 256, 2048), (100, 520, 2048), (300, 512, 256),
                                   (3000, 1032, 512)])
@pytest.mark.parametrize("ot", ["f32", "f16"])
def test_linear_operands_of_different_alignment(ops, skips, pads, m, n, k, ot):
    import torch

    x, w, xs, ws, b = _linear_inputs(m, n, k, m + n + k)
    xs = xs / k**0.5
    dtype = dict(f32=torch.float32, f16=torch.float16)[ot]
    r = torch.randn(m, n, device="cuda").to(dtype)
    ov, alone = _placed(torch.zeros_like(r), skips[0], pads[0])
    rv = _placed(r, skips[1], pads[1])[0]
    xsv, wsv, bv = (_placed(t, skips[2])[0] for t in (xs, ws, b))
    torch.cuda.synchronize()
    ops.quantized_linear(x.data_ptr(), w.data_ptr(), ov.data_ptr(), CODE[ot], m, n, k, x_scale=xsv.data_ptr(),
                         w_scale=wsv.data_ptr(), bias=bv.data_ptr(), residual=rv.data_ptr(), x_ld=x.stride(0),
                         w_ld=w.stride(0), residual_ld=rv.stride(0), out_ld=ov.stride(0))
    torch.cuda.synchronize()
    want, bound = _linear_want(_product(x, w, k), xs, ws, b, 0, r, ot)
    _within(ov, want, bound, "out")
    assert alone(), "wrote past the rows"
