"""The operators on device buffers (GPU) against plain 64-bit implementations.

Tolerances are bounds of the roundings, with u = 2^-24 the unit of f32:

* a sum of n terms taken as chains of at most c additions is off by at most
  c u sum |terms|; the kernels' chains are at most _chain(n) long;
* a result held in 16 bits is off by half a unit of its last place more.

The quantiser's steps are each one f32 rounding, so its integers and scales
are compared bit for bit with the same steps in numpy.
"""

import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF_ULP = {"f32": U, "f16": 2.0**-11, "bf16": 2.0**-8}  # of 24, 11 and 8 significant bits
TINY = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-133}  # half a unit of the subnormals, at most


@pytest.fixture(scope="module")
def ops():
    import dmx

    o = dmx.Ops(0)
    yield o
    o.check()
    o.close()


def _t(name):
    import dmx
    import torch

    return {"f32": (torch.float32, dmx.TYPE_F32), "f16": (torch.float16, dmx.TYPE_F16),
            "bf16": (torch.bfloat16, dmx.TYPE_BF16)}[name]


def _chain(n):
    # additions that follow one another: a thread's own, then those across threads
    return max(64, n // 256) + 16


def _padded(values, dtype, pad, fill=float("nan")):
    """`values` in rows of a wider buffer whose other elements are `fill`."""
    import torch

    rows, cols = values.shape
    buf = torch.full((rows, cols + pad), fill, dtype=dtype, device="cuda")
    buf[:, :cols] = values.to(dtype)
    return buf, buf[:, :cols]


def _within(got, want, bound, what):
    import torch

    off = (got.double() - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert torch.isfinite(got).all(), what
    assert worst <= 0, f"{what}: {worst} over the bound, largest error {off.max().item()}"


# --- layer norm ---------------------------------------------------------------

NORM_SHAPES = [(1, 1, 0), (1, 7, 0), (3, 8, 8), (2, 31, 1), (5, 32, 0), (9, 255, 0), (4, 256, 8),
               (33, 512, 0), (7, 513, 0), (3, 513, 7), (6, 1000, 0), (300, 1024, 0), (5, 1025, 7),
               (2, 2047, 0), (3, 2048, 16), (2, 4104, 0), (3, 8195, 5), (2, 16384, 0), (2, 16385, 0),
               (1, 16392, 8), (2, 40001, 7), (2689, 24, 0), (1500, 129, 3)]
NORM_TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f16", "f16"), ("f16", "f32"),
              ("bf16", "bf16"), ("bf16", "f32"), ("f16", "bf16")]


def _norm64(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    h = (x - mean) * rstd
    y = h * (1 if weight is None else weight.double()) + (0 if bias is None else bias.double())
    return h, y, mean, rstd


def _norm_bounds(x, h, y, weight, mean, rstd):
    n = x.shape[1]
    c = _chain(n)
    e_mean = (c + 2) * U * x.double().abs().mean(1, keepdim=True)
    # the variance: its own sum, and twice the relative error of each difference
    rel_rstd = 0.5 * ((c + 6) * U + 2 * e_mean * rstd + (e_mean * rstd) ** 2) + 4 * U
    w = 1.0 if weight is None else weight.double().abs()
    e_y = w * rstd * e_mean + w * h.abs() * (rel_rstd + 3 * U) + 2 * U * (y.abs() + w * h.abs())
    return e_mean, rel_rstd * rstd, e_y


def _norm_inputs(rows, cols, xt, seed, params, offset=0.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * 1.5 + offset
    w = b = None
    if params:
        w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(_t(params)[0])
        b = (0.2 * torch.randn(cols, generator=g, device="cuda")).to(_t(params)[0])
    return x.to(_t(xt)[0]), w, b


def _run_norm(ops, xbuf, x, w, b, yt, ypad, eps=1e-5, stats=True, params="f32", stream=0):
    import torch

    rows, cols = x.shape
    ybuf = torch.full((rows, cols + ypad), 7.0, dtype=_t(yt)[0], device="cuda")
    mean = torch.full((rows,), 9.0, device="cuda")
    rstd = torch.full((rows,), 9.0, device="cuda")
    torch.cuda.synchronize()
    xtype = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
    ops.layer_norm(x.data_ptr(), xtype, rows, cols, ybuf.data_ptr(), _t(yt)[1],
                   weight=0 if w is None else w.data_ptr(), bias=0 if b is None else b.data_ptr(),
                   param_type=_t(params)[1], eps=eps, x_ld=x.stride(0), y_ld=cols + ypad,
                   mean=mean.data_ptr() if stats else 0, rstd=rstd.data_ptr() if stats else 0,
                   stream=stream)
    torch.cuda.synchronize()
    assert (ybuf[:, cols:] == 7.0).all(), "wrote past the rows"
    return ybuf[:, :cols], mean, rstd


@pytest.mark.parametrize("rows,cols,pad", NORM_SHAPES)
@pytest.mark.parametrize("xt,yt", NORM_TYPES)
def test_layer_norm_matches_64_bits(ops, rows, cols, pad, xt, yt):
    x, w, b = _norm_inputs(rows, cols, xt, rows * 7 + cols, "f32")
    xbuf, xv = _padded(x, x.dtype, pad)
    y, mean, rstd = _run_norm(ops, xbuf, xv, w, b, yt, pad)
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    e_mean, e_rstd, e_y = _norm_bounds(x, h, want, w, m64, r64)
    _within(mean[:, None], m64, e_mean, "mean")
    _within(rstd[:, None], r64, e_rstd, "rstd")
    _within(y, want, e_y + HALF_ULP[yt] * (want.abs() + e_y) + TINY[yt], "y")


@pytest.mark.parametrize("params", [None, "f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [40, 513, 4104, 16400])
def test_layer_norm_parameters_of_each_type_or_none(ops, params, cols):
    x, w, b = _norm_inputs(5, cols, "f32", cols, params)
    y, _, _ = _run_norm(ops, None, x, w, b, "f32", 0, stats=False, params=params or "f32")
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    _within(y, want, _norm_bounds(x, h, want, w, m64, r64)[2], "y")


@pytest.mark.parametrize("cols", [40, 512, 2050, 16400])
def test_layer_norm_of_rows_far_from_zero(ops, cols):
    # a mean thousands of times the spread: a variance from sums of squares would be noise
    x, w, b = _norm_inputs(6, cols, "f32", 5, "f32", offset=4096.0)
    y, mean, rstd = _run_norm(ops, None, x, w, b, "f32", 0)
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    e_mean, e_rstd, e_y = _norm_bounds(x, h, want, w, m64, r64)
    _within(rstd[:, None], r64, e_rstd, "rstd")
    _within(y, want, e_y, "y")


@pytest.mark.parametrize("cols", [1, 64, 515, 9000, 17000])
def test_layer_norm_of_constant_rows_is_the_bias(ops, cols):
    import torch

    x = torch.full((3, cols), 2.5, device="cuda")
    b = torch.arange(cols, device="cuda", dtype=torch.float32)
    y, mean, rstd = _run_norm(ops, None, x, None, b, "f32", 0)
    assert (y == b).all() and (mean == 2.5).all()
    assert torch.allclose(rstd, torch.full_like(rstd, 1 / math.sqrt(1e-5)), rtol=8 * U * 2)


@pytest.mark.parametrize("cols", [70, 512, 3000, 16500])
def test_layer_norm_of_a_row_with_nan_or_infinity_leaves_the_others_alone(ops, cols):
    import torch

    x, w, b = _norm_inputs(5, cols, "f32", 8, "f32")
    clean, _, _ = _run_norm(ops, None, x, w, b, "f32", 0)
    bad = x.clone()
    bad[1, cols // 2], bad[3, cols - 1] = float("nan"), float("inf")
    y, _, _ = _run_norm(ops, None, bad, w, b, "f32", 0)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
    assert torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


@pytest.mark.parametrize("cols", [9, 512, 1030, 8195, 17001])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_layer_norm_in_place_and_at_any_element(ops, cols, shift):
    # y == x, and buffers that start off a vector's boundary
    import torch

    x, w, b = _norm_inputs(4, cols, "f16", 3, "f16")
    flat = torch.zeros(4 * (cols + 5) + 8, dtype=torch.float16, device="cuda")
    view = flat[shift:shift + 4 * (cols + 5)].view(4, cols + 5)[:, :cols]
    view.copy_(x)
    ops.layer_norm(view.data_ptr(), 1, 4, cols, view.data_ptr(), 1, weight=w.data_ptr(),
                   bias=b.data_ptr(), param_type=1, x_ld=cols + 5, y_ld=cols + 5)
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    e = _norm_bounds(x, h, want, w, m64, r64)[2]
    _within(view, want, e + HALF_ULP["f16"] * (want.abs() + e) + TINY["f16"], "y")


def test_rows_further_apart_than_32_bits_reach(ops):
    import torch

    ld, cols = 2**30 + 8, 520
    flat = torch.empty(2 * ld + cols, dtype=torch.float16, device="cuda")
    view = flat.as_strided((3, cols), (ld, 1))
    x, w, b = _norm_inputs(3, cols, "f16", 11, "f32")
    view.copy_(x)
    y, mean, rstd = _run_norm(ops, None, view, w, b, "f32", 0)
    h, want, m64, r64 = _norm64(x, w, b, 1e-5)
    _within(y, want, _norm_bounds(x, h, want, w, m64, r64)[2], "y")
    # backward: dx written at those distances too
    dy = torch.randn(3, cols, device="cuda")
    ops.layer_norm_backward(dy.data_ptr(), 0, view.data_ptr(), 1, mean.data_ptr(), rstd.data_ptr(), 3,
                            cols, dx=view.data_ptr(), x_ld=ld, dx_ld=ld)
    got = view.clone()
    alone = torch.empty_like(x)
    ops.layer_norm_backward(dy.data_ptr(), 0, x.data_ptr(), 1, mean.data_ptr(), rstd.data_ptr(), 3, cols,
                            dx=alone.data_ptr())
    assert torch.equal(got, alone)
    # and the integers of a quantised row
    del flat, view
    q = torch.empty(2 * (2**31 - 64) + 64 + cols, dtype=torch.int8, device="cuda").as_strided(
        (3, cols), (2**31 - 64, 1))
    scale, near, near_scale = torch.empty(3, device="cuda"), torch.empty(3, cols, dtype=torch.int8,
                                                                        device="cuda"), torch.empty(3, device="cuda")
    ops.quantize_rows(x.data_ptr(), 1, 3, cols, q.data_ptr(), scale.data_ptr(), q_ld=q.stride(0))
    ops.quantize_rows(x.data_ptr(), 1, 3, cols, near.data_ptr(), near_scale.data_ptr())
    assert torch.equal(q.clone(), near) and torch.equal(scale, near_scale)
    w8 = torch.randint(-127, 128, (24, 528), device="cuda").to(torch.int8)
    far_out, out = torch.empty(3, 24, device="cuda"), torch.empty(3, 24, device="cuda")
    near16 = torch.zeros(3, 528, dtype=torch.int8, device="cuda")
    near16[:, :cols] = near
    ops.quantized_linear(q.data_ptr(), w8.data_ptr(), far_out.data_ptr(), 0, 3, 24, cols, x_ld=q.stride(0),
                         w_ld=528)
    ops.quantized_linear(near16.data_ptr(), w8.data_ptr(), out.data_ptr(), 0, 3, 24, cols, x_ld=528,
                         w_ld=528)
    assert torch.equal(far_out, out)


# --- backward -----------------------------------------------------------------

BACK_SHAPES = [(1, 1, 0), (1, 33, 0), (2, 8, 8), (3, 100, 1), (1, 513, 0), (40, 512, 0), (700, 512, 0),
               (31, 1000, 0), (5, 1024, 8), (129, 1031, 0), (64, 2048, 0), (9, 4097, 7), (150, 8195, 5),
               (3, 16384, 0), (3, 16385, 0), (20, 33001, 7), (5000, 48, 0), (2100, 257, 3)]


def _back64(dy, x, w, mean, rstd):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    h = (x - mean) * rstd
    g = dy * (1 if w is None else w.double())
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    c = _chain(x.shape[1])
    e1 = (c + 4) * U * g.abs().mean(1, keepdim=True)
    e2 = (c + 8) * U * (g * h).abs().mean(1, keepdim=True)
    m2 = (g * h).mean(1, keepdim=True).abs()
    e_dx = rstd * (e1 + h.abs() * e2) + 8 * U * rstd * (g.abs() + g.mean(1, keepdim=True).abs() + h.abs() * m2)
    # a chain of rows in a block, then one over blocks and their warps
    n = min(x.shape[0], 800) + 40
    e_w = (n + 4) * U * (dy * h).abs().sum(0)
    e_b = n * U * dy.abs().sum(0)
    return dx, (dy * h).sum(0), dy.sum(0), e_dx, e_w, e_b


def _run_back(ops, dy, x, w, mean, rstd, params="f32", want=("dx", "dweight", "dbias"), pad=0, stream=0):
    import torch

    rows, cols = x.shape
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    dxbuf = torch.full((rows, cols + pad), 7.0, dtype=x.dtype, device="cuda")
    dw = torch.full((cols,), 7.0, device="cuda")
    db = torch.full((cols,), 7.0, device="cuda")
    size = ops.layer_norm_backward_workspace(rows, cols)
    room = torch.full((size + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ops.layer_norm_backward(dy.data_ptr(), code[dy.dtype], x.data_ptr(), code[x.dtype], mean.data_ptr(),
                            rstd.data_ptr(), rows, cols, room.data_ptr(), size,
                            weight=0 if w is None else w.data_ptr(), param_type=_t(params)[1],
                            dx=dxbuf.data_ptr() if "dx" in want else 0,
                            dweight=dw.data_ptr() if "dweight" in want else 0,
                            dbias=db.data_ptr() if "dbias" in want else 0, dy_ld=dy.stride(0),
                            x_ld=x.stride(0), dx_ld=cols + pad, stream=stream)
    torch.cuda.synchronize()
    assert (room[size:] == 0xAB).all(), "wrote past the workspace"
    assert (dxbuf[:, cols:] == 7.0).all(), "wrote past the rows"
    return dxbuf[:, :cols], dw, db


def _back_inputs(rows, cols, xt, dyt, seed, params="f32"):
    import torch

    x, w, b = _norm_inputs(rows, cols, xt, seed, params)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(_t(dyt)[0])
    _, _, mean, rstd = _norm64(x, None, None, 1e-5)
    return dy, x, w, mean[:, 0].float(), rstd[:, 0].float()


@pytest.mark.parametrize("rows,cols,pad", BACK_SHAPES)
@pytest.mark.parametrize("xt,dyt", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                    ("bf16", "f32"), ("f16", "bf16")])
def test_layer_norm_backward_matches_64_bits(ops, rows, cols, pad, xt, dyt):
    dy, x, w, mean, rstd = _back_inputs(rows, cols, xt, dyt, rows + cols)
    _, dyv = _padded(dy, dy.dtype, pad)
    _, xv = _padded(x, x.dtype, pad)
    dx, dw, db = _run_back(ops, dyv, xv, w, mean, rstd, pad=pad)
    dx64, dw64, db64, e_dx, e_w, e_b = _back64(dy, x, w, mean, rstd)
    _within(dx, dx64, e_dx + HALF_ULP[xt] * (dx64.abs() + e_dx) + TINY[xt], "dx")
    _within(dw, dw64, e_w, "dweight")
    _within(db, db64, e_b, "dbias")


@pytest.mark.parametrize("want", [("dx",), ("dweight",), ("dbias",), ("dx", "dbias"), ("dweight", "dbias"), ()])
@pytest.mark.parametrize("rows,cols", [(5, 300), (70, 512), (70, 1500), (12, 17000)])
def test_layer_norm_backward_gives_what_is_asked_for(ops, want, rows, cols):
    import torch

    dy, x, w, mean, rstd = _back_inputs(rows, cols, "f32", "f32", 3)
    full = dict(zip(("dx", "dweight", "dbias"), _run_back(ops, dy, x, w, mean, rstd)))
    part = dict(zip(("dx", "dweight", "dbias"), _run_back(ops, dy, x, w, mean, rstd, want=want)))
    for name in full:
        if name in want:
            assert torch.equal(part[name], full[name]), name
        else:
            assert (part[name] == 7.0).all(), name


@pytest.mark.parametrize("params", [None, "f16", "bf16"])
@pytest.mark.parametrize("cols", [64, 1023, 4096, 17000])
def test_layer_norm_backward_parameters_of_each_type_or_none(ops, params, cols):
    dy, x, w, mean, rstd = _back_inputs(21, cols, "f32", "f32", 4, params)
    dx, dw, db = _run_back(ops, dy, x, w, mean, rstd, params=params or "f32")
    dx64, dw64, db64, e_dx, e_w, e_b = _back64(dy, x, w, mean, rstd)
    _within(dx, dx64, e_dx + U * dx64.abs(), "dx")
    _within(dw, dw64, e_w, "dweight")


def test_layer_norm_backward_of_no_rows_is_zero(ops):
    import torch

    dw, db = torch.full((2, 300), 7.0, device="cuda")
    ops.layer_norm_backward(0, 0, 0, 0, 0, 0, 0, 300, dweight=dw.data_ptr(), dbias=db.data_ptr())
    assert (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("rows,cols", [(3000, 512), (500, 3100), (40, 20000)])
def test_layer_norm_backward_is_the_same_each_time(ops, rows, cols):
    import torch

    dy, x, w, mean, rstd = _back_inputs(rows, cols, "f32", "f32", 5)
    first = [t.clone() for t in _run_back(ops, dy, x, w, mean, rstd)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _run_back(ops, dy, x, w, mean, rstd)))


@pytest.mark.parametrize("rows,cols", [(5, 24), (3, 1500)])
def test_layer_norm_gradients_match_differences(ops, rows, cols):
    # L = sum(dy * norm(x; w, b)) in 64 bits; central differences along random directions
    import torch

    dy, x, w, mean, rstd = _back_inputs(rows, cols, "f32", "f32", 6)
    dx, dw, db = (t.double() for t in _run_back(ops, dy, x, w, mean, rstd))
    b = torch.zeros_like(w)
    g = torch.Generator(device="cuda").manual_seed(7)

    def loss(x, w, b):
        return (dy.double() * _norm64(x, w, b, 1e-5)[1]).sum().item()

    step = 1e-4  # differences are off by about step^2 of the third derivative
    x, w, b = x.double(), w.double(), b.double()
    for _ in range(4):
        v = torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.float64)
        vw = torch.randn(cols, generator=g, device="cuda", dtype=torch.float64)
        scale = dy.double().norm().item()
        assert abs((loss(x + step * v, w, b) - loss(x - step * v, w, b)) / (2 * step)
                   - (dx * v).sum().item()) <= 1e-5 * scale * math.sqrt(rows * cols) / 10
        assert abs((loss(x, w + step * vw, b) - loss(x, w - step * vw, b)) / (2 * step)
                   - (dw * vw).sum().item()) <= 1e-5 * scale
        assert abs((loss(x, w, b + step * vw) - loss(x, w, b - step * vw)) / (2 * step)
                   - (db * vw).sum().item()) <= 1e-5 * scale


@pytest.mark.parametrize("which", ["dy", "x"])
@pytest.mark.parametrize("cols", [500, 2048, 3001, 17000])
def test_layer_norm_backward_in_place(ops, which, cols):
    import torch

    dy, x, w, mean, rstd = _back_inputs(30, cols, "bf16", "bf16", 9, "bf16")
    dx, dw, db = _run_back(ops, dy, x, w, mean, rstd, params="bf16")
    target = dy.clone() if which == "dy" else x.clone()
    a = {"dy": dy, "x": x, which: target}
    dw2, db2 = torch.empty_like(dw), torch.empty_like(db)
    size = ops.layer_norm_backward_workspace(30, cols)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    ops.layer_norm_backward(a["dy"].data_ptr(), 2, a["x"].data_ptr(), 2, mean.data_ptr(), rstd.data_ptr(),
                            30, cols, room.data_ptr(), size, weight=w.data_ptr(), param_type=2,
                            dx=target.data_ptr(), dweight=dw2.data_ptr(), dbias=db2.data_ptr())
    assert torch.equal(target, dx) and torch.equal(dw, dw2) and torch.equal(db, db2)


# --- quantiser ----------------------------------------------------------------

def _quantise_steps(v):
    """The quantiser's f32 steps in numpy: (q, scale)."""
    v = np.asarray(v, dtype=np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(v).max(axis=1)  # numpy's max keeps a NaN
        scale = (top / np.float32(127)).astype(np.float32)
        usable = (scale > 0) & np.isfinite(scale)
        q = np.rint((v / np.where(usable, scale, np.float32(1))[:, None]).astype(np.float32))
        q = np.where(usable[:, None], np.clip(q, -127, 127), 0)
    return q.astype(np.int8), scale


def _run_quantise(ops, xv, col_scale, qpad, xtype):
    import torch

    rows, cols = xv.shape
    qbuf = torch.full((rows, cols + qpad), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((rows,), 9.0, device="cuda")
    ops.quantize_rows(xv.data_ptr(), xtype, rows, cols, qbuf.data_ptr(), scale.data_ptr(),
                      col_scale=0 if col_scale is None else col_scale.data_ptr(), x_ld=xv.stride(0),
                      q_ld=cols + qpad)
    torch.cuda.synchronize()
    assert (qbuf[:, cols:] == 77).all(), "wrote past the rows"
    return qbuf[:, :cols].cpu().numpy(), scale.cpu().numpy()


@pytest.mark.parametrize("rows,cols,pad", NORM_SHAPES)
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mult", [False, True])
def test_quantise_is_its_steps_bit_for_bit(ops, rows, cols, pad, xt, mult):
    import torch

    x, w, _ = _norm_inputs(rows, cols, xt, rows + 3 * cols, "f32")
    _, xv = _padded(x, x.dtype, pad)
    q, scale = _run_quantise(ops, xv, w if mult else None, (-cols) % 16, _t(xt)[1])
    v = x.float() * w if mult else x.float()
    want_q, want_scale = _quantise_steps(v.cpu().numpy())
    assert np.array_equal(scale, want_scale) and np.array_equal(q, want_q)
    assert np.abs(q).max() == 127


@pytest.mark.parametrize("cols", [16, 100, 512, 1500, 4096, 17000])
def test_quantise_ties_zeros_extremes_and_what_is_not_finite(ops, cols):
    import torch

    rng = np.random.default_rng(cols)
    x = np.zeros((16, cols), dtype=np.float32)
    half = rng.integers(-126, 126, cols) + np.float32(0.5)  # exact ties at scale 1
    x[0], x[0, 0] = half, 127
    x[1] = 0
    x[2, cols // 2] = -0.0
    x[3] = rng.integers(-200, 200, cols) * np.float32(2.0**-149)  # subnormal scale
    x[4] = np.float32(2.0**-149)  # scale 0 after the division
    x[5] = rng.standard_normal(cols).astype(np.float32) * np.float32(1e38)
    x[6], x[6, cols - 1] = 1.0, np.float32(3.4e38)
    x[7], x[7, 3] = rng.standard_normal(cols), np.nan
    x[8], x[8, cols - 2] = rng.standard_normal(cols), np.inf
    x[9], x[9, 0], x[9, cols - 1] = rng.standard_normal(cols), -np.inf, np.nan
    x[10, cols - 1] = -3
    x[11] = half * np.float32(2.0**-126)  # ties at the least normal scale
    x[11, 0] = np.float32(127 * 2.0**-126)
    x[12] = half * np.float32(2.0**-140)
    x[13] = rng.standard_normal(cols) * 1e-38
    x[14] = np.float32(1e-20)
    x[15] = half * np.float32(0.1)  # near ties
    q, scale = _run_quantise(ops, torch.from_numpy(x).cuda(), None, 0, 0)
    want_q, want_scale = _quantise_steps(x)
    assert np.array_equal(scale, want_scale, equal_nan=True)
    assert np.array_equal(q, want_q)
    assert np.isnan(scale[[7, 9]]).all() and np.isinf(scale[8]) and not q[[1, 4, 7, 8, 9]].any()


@pytest.mark.parametrize("exponent", [-99, -60, 0, 40, 119])
def test_quantise_next_to_every_tie_of_many_scales(ops, exponent):
    # the floats around (k + 1/2) scale, for scales of every kind of significand
    import torch

    rng = np.random.default_rng(100 + exponent)
    rows = 3000
    top = np.ldexp(rng.integers(2**23, 2**24, rows).astype(np.float64), exponent - 23).astype(np.float32)
    ones = np.uint32(0x7FFFFF) | np.uint32((exponent + 127) << 23)  # a scale whose significand is all ones
    top[:500] = (np.frombuffer(ones.tobytes(), np.float32)[0] * 127.0).astype(np.float32)
    top[500:900] = np.ldexp(rng.integers(128, 256, 400).astype(np.float64), exponent - 7).astype(np.float32)
    scale = (top / np.float32(127)).astype(np.float32)
    k = np.arange(-126, 126) + 0.5
    near = (k[None, :] * scale[:, None].astype(np.float64)).astype(np.float32)
    x = np.concatenate([top[:, None], near, np.nextafter(near, np.float32(np.inf)),
                        np.nextafter(near, np.float32(-np.inf))], axis=1)
    x = np.clip(x, -top[:, None], top[:, None])
    q, got = _run_quantise(ops, torch.from_numpy(x).cuda(), None, 0, 0)
    want_q, want_scale = _quantise_steps(x)
    assert np.array_equal(got, want_scale) and np.array_equal(q, want_q)


@pytest.mark.parametrize("rows,cols,pad", NORM_SHAPES)
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
def test_norm_and_quantise_in_one_pass(ops, rows, cols, pad, xt):
    import torch

    x, w, b = _norm_inputs(rows, cols, xt, rows + 5 * cols, "f32")
    _, xv = _padded(x, x.dtype, pad)
    qpad = (-cols) % 16
    qbuf = torch.full((rows, cols + qpad), 77, dtype=torch.int8, device="cuda")
    scale, mean, rstd = torch.full((3, rows), 9.0, device="cuda")
    ops.layer_norm_quantize(xv.data_ptr(), _t(xt)[1], rows, cols, qbuf.data_ptr(), scale.data_ptr(),
                            weight=w.data_ptr(), bias=b.data_ptr(), x_ld=xv.stride(0), q_ld=cols + qpad,
                            mean=mean.data_ptr(), rstd=rstd.data_ptr())
    torch.cuda.synchronize()
    assert (qbuf[:, cols:] == 77).all(), "wrote past the rows"
    h, y, m64, r64 = _norm64(x, w, b, 1e-5)
    e_mean, e_rstd, e_y = _norm_bounds(x, h, y, w, m64, r64)
    _within(mean[:, None], m64, e_mean, "mean")
    _within(rstd[:, None], r64, e_rstd, "rstd")
    top, e_top = y.abs().amax(1), e_y.amax(1)
    _within(scale, top / 127, (e_top + 2 * U * top) / 127, "scale")
    # each integer is the nearest one to the value, but for the value's own error
    s = scale.double()[:, None]
    off = (qbuf[:, :cols].double() - y / s).abs()
    assert (off <= 0.5 + (e_y + 4 * U * y.abs()) / s + 1e-5).all(), off.max().item()


def test_norm_and_quantise_marks_rows_that_are_not_finite(ops):
    import torch

    for cols in (64, 1500, 17000):
        x, w, b = _norm_inputs(4, cols, "f32", 2, "f32")
        x[1, 5], x[2, cols - 1] = float("nan"), float("inf")
        q = torch.full((4, cols), 77, dtype=torch.int8, device="cuda")
        scale = torch.empty(4, device="cuda")
        ops.layer_norm_quantize(x.data_ptr(), 0, 4, cols, q.data_ptr(), scale.data_ptr(),
                                weight=w.data_ptr(), bias=b.data_ptr())
        assert torch.isnan(scale[1:3]).all() and torch.isfinite(scale[[0, 3]]).all()
        assert (q[1:3] == 0).all() and (q[[0, 3]].abs().amax(1) == 127).all()


# --- 8-bit linear -------------------------------------------------------------

def _linear_inputs(m, n, k, seed, extreme=False):
    """int8 operands in rows of whole 16 bytes whose padding holds other values."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = (k + 15) // 16 * 16

    def ints(rows):
        v = torch.randint(-128, 128, (rows, ld), generator=g, device="cuda").to(torch.int8)
        if extreme:
            v[:, :k] = -128
        return v

    xs = torch.rand(m, generator=g, device="cuda") * 0.02 + 1e-3
    ws = torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4
    b = torch.randn(n, generator=g, device="cuda")
    return ints(m), ints(n), xs, ws, b


def _product(x, w, k):
    # exact: every partial sum is an integer below 2^53
    return x[:, :k].double() @ w[:, :k].double().t()


def _gelu64(z):
    import torch

    return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))


def _linear_want(acc, xs, ws, b, act, res, ot):
    import torch

    z = acc
    e = torch.zeros_like(z)
    if xs is not None:
        z = z * xs.double()[:, None]
    if ws is not None:
        z = z * ws.double()
    e = 4 * U * z.abs()
    if b is not None:
        z = z + b.double()
        e = e + 2 * U * z.abs()
    if act:
        # |gelu'| < 1.13; the erf itself is good to 1.5e-7, and two roundings
        e = 1.13 * e + z.abs() * (0.5 * 1.5e-7 + 6 * U)
        z = _gelu64(z)
    if res is not None:
        z = z + res.double()
        e = e + U * z.abs()
    return z, e + HALF_ULP[ot] * (z.abs() + e) + TINY[ot]


def _run_linear(ops, x, w, k, ot, xs, ws, b, act=0, res=None, pad=0, in_place=False, stream=0):
    import torch

    m, n = x.shape[0], w.shape[0]
    buf = torch.full((m, n + pad), 7.0, dtype=_t(ot)[0], device="cuda")
    if in_place:
        buf[:, :n] = res
    r = buf if in_place else res
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    torch.cuda.synchronize()
    ops.quantized_linear(x.data_ptr(), w.data_ptr(), buf.data_ptr(), _t(ot)[1], m, n, k, x_scale=p(xs),
                         w_scale=p(ws), bias=p(b), activation=act, residual=p(r), x_ld=x.stride(0),
                         w_ld=w.stride(0), residual_ld=0 if r is None else r.stride(0), out_ld=n + pad,
                         stream=stream)
    torch.cuda.synchronize()
    assert (buf[:, n:] == 7.0).all(), "wrote past the rows"
    return buf[:, :n]


LINEAR_SHAPES = [(1, 1, 1), (1, 3, 15), (1, 64, 16), (1, 512, 512), (1, 1000, 4097), (1, 4096, 2050),
                 (2, 65, 33), (3, 128, 128), (4, 257, 1000), (5, 40, 8192), (7, 129, 129), (8, 2048, 512),
                 (9, 63, 31), (9, 700, 2050), (15, 100, 100), (16, 256, 256), (17, 300, 64), (31, 511, 640),
                 (32, 32, 32), (33, 1030, 127), (48, 96, 1536), (63, 200, 300), (64, 512, 512), (65, 64, 65),
                 (100, 1000, 4000), (127, 127, 127), (128, 128, 128), (129, 257, 385), (192, 2048, 96),
                 (255, 33, 2049), (256, 512, 48), (257, 65, 512), (300, 2050, 700), (500, 48, 100),
                 (672, 1536, 512), (1000, 1, 77), (1345, 513, 511), (2688, 512, 2048), (4000, 17, 130),
                 (5000, 1031, 24), (20001, 136, 200), (19001, 2055, 150)]


@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
@pytest.mark.parametrize("ot", ["f32", "f16", "bf16"])
def test_quantized_linear_matches_64_bits(ops, m, n, k, ot):
    x, w, xs, ws, b = _linear_inputs(m, n, k, m + n + k)
    xs, ws = xs / math.sqrt(k), ws
    got = _run_linear(ops, x, w, k, ot, xs, ws, b)
    want, bound = _linear_want(_product(x, w, k), xs, ws, b, 0, None, ot)
    _within(got, want, bound, "out")


@pytest.mark.parametrize("m,n,k", [(1, 520, 700), (5, 130, 512), (12, 100, 96), (40, 257, 300), (90, 640, 2048),
                                   (200, 384, 130), (700, 1025, 512), (19008, 2056, 96)])
@pytest.mark.parametrize("ot", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("res,pad", [(False, 5), (True, 0), (True, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_quantized_linear_activation_residual_and_pitch(ops, m, n, k, ot, act, res, pad, in_place):
    import torch

    if in_place and not res:
        pytest.skip("nothing to add to in place")
    x, w, xs, ws, b = _linear_inputs(m, n, k, 3 * m + n + k)
    xs = xs / math.sqrt(k)
    r = torch.randn(m, n, device="cuda").to(_t(ot)[0]) if res else None
    got = _run_linear(ops, x, w, k, ot, xs, ws, b, act, r, pad, in_place)
    want, bound = _linear_want(_product(x, w, k), xs, ws, b, act, r, ot)
    _within(got, want, bound, "out")


@pytest.mark.parametrize("m", [1, 6, 20, 300])
@pytest.mark.parametrize("given", ["", "x", "w", "b", "xw", "wb", "xb"])
def test_quantized_linear_scales_and_bias_may_be_left_out(ops, m, given):
    x, w, xs, ws, b = _linear_inputs(m, 150, 70, 77)
    xs = xs if "x" in given else None
    ws = ws if "w" in given else None
    b = b if "b" in given else None
    got = _run_linear(ops, x, w, 70, "f32", xs, ws, b)
    want, bound = _linear_want(_product(x, w, 70), xs, ws, b, 0, None, "f32")
    _within(got, want, bound, "out")
    if not given:
        assert (got.double() == want).all()  # integers below 2^24: nothing is rounded


@pytest.mark.parametrize("m", [1, 8, 24, 140])
def test_quantized_linear_longest_sum_of_the_largest_values(ops, m):
    k = 131071
    x, w, xs, ws, b = _linear_inputs(m, 20, k, 5, extreme=True)
    got = _run_linear(ops, x, w, k, "f32", None, None, None)
    want, bound = _linear_want(_product(x, w, k), None, None, None, 0, None, "f32")
    assert want.max().item() == 16384.0 * k
    _within(got, want, bound, "out")


@pytest.mark.parametrize("m", [3, 30, 200])
def test_quantized_linear_carries_a_scale_that_is_not_finite(ops, m):
    import torch

    x, w, xs, ws, b = _linear_inputs(m, 90, 64, 5)
    clean = _run_linear(ops, x, w, 64, "f32", xs, ws, b)
    x[1] = 0
    xs[1] = float("inf")
    x[2] = 0
    xs[2] = float("nan")
    got = _run_linear(ops, x, w, 64, "f32", xs, ws, b)
    assert torch.isnan(got[1:3]).all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3:], clean[3:])


def test_quantized_linear_over_many_output_elements(ops):
    # more than 2^31 bytes and elements past 32 bits of offset
    import torch

    m, n, k = 140001, 16392, 32
    x, w, xs, ws, b = _linear_inputs(m, n, k, 6)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    ops.quantized_linear(x.data_ptr(), w.data_ptr(), out.data_ptr(), 2, m, n, k, x_scale=xs.data_ptr(),
                         w_scale=ws.data_ptr(), bias=b.data_ptr(), x_ld=32, w_ld=32)
    rows = torch.tensor([0, 1, 70000, 131001, 131072, 139999, 140000], device="cuda")
    want, bound = _linear_want(_product(x[rows], w, k), xs[rows], ws, b, 0, None, "bf16")
    _within(out[rows], want, bound, "out")


@pytest.mark.parametrize("m", [1, 8, 50, 128, 300])
def test_quantized_linear_is_the_same_each_time(ops, m):
    import torch

    x, w, xs, ws, b = _linear_inputs(m, 333, 4096, 8)
    first = _run_linear(ops, x, w, 4096, "f32", xs, ws, b).clone()
    for _ in range(5):
        assert torch.equal(first, _run_linear(ops, x, w, 4096, "f32", xs, ws, b))


def test_quantized_linear_input_gradient_by_the_same_operators(ops):
    # dy w_scale quantised per row, times the transposed integers: the gradient of x within dy's 8 bits
    import torch

    m, n, k = 70, 320, 200
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-127, 128, (n, 208), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") * 0.01
    dy = torch.randn(m, n, generator=g, device="cuda")
    wt = torch.zeros(k, n, dtype=torch.int8, device="cuda")
    wt.copy_(w[:, :k].t())
    q, s = torch.empty(m, n, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    ops.quantize_rows(dy.data_ptr(), 0, m, n, q.data_ptr(), s.data_ptr(), col_scale=ws.data_ptr())
    dx = torch.empty(m, k, device="cuda")
    ops.quantized_linear(q.data_ptr(), wt.data_ptr(), dx.data_ptr(), 0, m, k, n, x_scale=s.data_ptr())
    want = (dy.double() * ws.double()) @ w[:, :k].double()
    # each of n values is off by at most half a step
    bound = 0.5001 * s.double()[:, None] * w[:, :k].double().abs().sum(0) + 8 * U * want.abs()
    _within(dx, want, bound, "dx")


# --- streams, graphs, contexts ------------------------------------------------

def test_operators_run_on_the_stream_they_are_given(ops):
    import torch

    m, k, n = 400, 512, 256
    x, w, b = _norm_inputs(m, k, "f32", 1, "f32")
    w8 = torch.randint(-127, 128, (n, k), device="cuda").to(torch.int8)
    q, s = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    out = torch.zeros(m, n, device="cuda")

    def chain(x, out, stream):
        ops.layer_norm_quantize(x.data_ptr(), 0, m, k, q.data_ptr(), s.data_ptr(), weight=w.data_ptr(),
                                bias=b.data_ptr(), stream=stream)
        ops.quantized_linear(q.data_ptr(), w8.data_ptr(), out.data_ptr(), 0, m, n, k,
                             x_scale=s.data_ptr(), stream=stream)

    chain(x, out, 0)
    ops.check()
    want = out.clone()
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the input is written after this
        late.copy_(x)
        out.zero_()
        chain(late, out, side.cuda_stream)
    ops.check(side.cuda_stream)
    assert torch.equal(out, want)


def test_operators_can_be_captured_into_a_graph(ops):
    import torch

    m, k, n = 150, 640, 384
    x, w, b = _norm_inputs(m, k, "f32", 2, "f32")
    held = torch.zeros_like(x)
    w8 = torch.randint(-127, 128, (n, k), device="cuda").to(torch.int8)
    q, s = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    out, dx = torch.zeros(m, n, device="cuda"), torch.zeros_like(x)
    mean, rstd = torch.zeros(2, m, device="cuda")
    dw = torch.zeros(k, device="cuda")
    size = ops.layer_norm_backward_workspace(m, k)
    room = torch.zeros(size, dtype=torch.uint8, device="cuda")

    def step(stream):
        ops.layer_norm_quantize(held.data_ptr(), 0, m, k, q.data_ptr(), s.data_ptr(), weight=w.data_ptr(),
                                bias=b.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), stream=stream)
        ops.quantized_linear(q.data_ptr(), w8.data_ptr(), out.data_ptr(), 0, m, n, k, x_scale=s.data_ptr(),
                             activation=1, stream=stream)
        ops.layer_norm_backward(held.data_ptr(), 0, held.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), m,
                                k, room.data_ptr(), size, dx=dx.data_ptr(), dweight=dw.data_ptr(),
                                stream=stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for scale in (1.0, -3.0):
        held.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, dx, dw)]
        step(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, (out, dx, dw)))
    ops.check()


def test_no_rows_is_no_work(ops):
    import torch

    out = torch.full((4, 8), 7.0, device="cuda")
    ops.layer_norm(0, 0, 0, 8, out.data_ptr(), 0)
    ops.quantize_rows(0, 0, 0, 8, 0, 0)
    ops.layer_norm_quantize(0, 0, 0, 8, 0, 0)
    ops.quantized_linear(0, 0, out.data_ptr(), 0, 0, 8, 8)
    ops.check()
    assert (out == 7.0).all()


# --- refusals -----------------------------------------------------------------

def test_refusals(ops):
    import dmx
    import torch

    x = torch.zeros(4, 32, device="cuda")
    p = x.data_ptr()
    s = torch.zeros(64, device="cuda").data_ptr()
    q = torch.zeros(4, 32, dtype=torch.int8, device="cuda").data_ptr()
    w = torch.zeros(8, 32, dtype=torch.int8, device="cuda").data_ptr()
    o = torch.zeros(4, 32, device="cuda").data_ptr()
    nan, inf = float("nan"), float("inf")
    calls = [
        (lambda: ops.layer_norm(0, 0, 4, 32, o, 0), "x is null"),
        (lambda: ops.layer_norm(p, 0, 4, 32, 0, 0), "y is null"),
        (lambda: ops.layer_norm(p, 3, 4, 32, o, 0), "x_type"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, -1), "y_type"),
        (lambda: ops.layer_norm(p, 0, -1, 32, o, 0), "rows"),
        (lambda: ops.layer_norm(p, 0, 4, -2, o, 0, x_ld=8, y_ld=8), "cols"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, x_ld=31), "x_ld"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, y_ld=-5), "y_ld"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, y_ld=2**40), "y_ld"),
        (lambda: ops.layer_norm(p + 2, 0, 4, 16, o, 0, x_ld=32), "x is not aligned"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o + 1, 1), "y is not aligned"),
        (lambda: ops.layer_norm(p, 0, 4, 32, p, 1), "in place"),
        (lambda: ops.layer_norm(p, 0, 4, 16, p, 0, x_ld=32, y_ld=16), "in place"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, weight=s, param_type=9), "param_type"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, bias=s + 2, param_type=0), "bias"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, eps=-1e-5), "eps"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, eps=nan), "eps"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, eps=inf), "eps"),
        (lambda: ops.layer_norm(p, 0, 4, 32, o, 0, mean=s + 1), "mean"),
        (lambda: ops.layer_norm_backward(0, 0, p, 0, s, s, 4, 32, dx=o), "dy is null"),
        (lambda: ops.layer_norm_backward(p, 0, p, 0, 0, s, 4, 32, dx=o), "mean is null"),
        (lambda: ops.layer_norm_backward(p, 0, p, 0, s, 0, 4, 32, dx=o), "rstd is null"),
        (lambda: ops.layer_norm_backward(p, 0, p, 0, s, s, 4, 32, dweight=s), "workspace"),
        (lambda: ops.layer_norm_backward(p, 0, p, 0, s, s, 4, 32, o, 8, dbias=s), "workspace is smaller"),
        (lambda: ops.layer_norm_backward(p, 0, p, 0, s, s, 4, 32, o + 4, 1 << 20, dbias=s), "workspace"),
        (lambda: ops.layer_norm_backward(p, 1, o, 0, s, s, 4, 32, dx=p), "in place"),
        (lambda: ops.layer_norm_backward(p, 0, o, 0, s, s, 4, 32, dx=q, dx_ld=3), "dx_ld"),
        (lambda: ops.quantize_rows(p, 0, 4, 32, 0, s), "q is null"),
        (lambda: ops.quantize_rows(p, 0, 4, 32, q, 0), "scale is null"),
        (lambda: ops.quantize_rows(p, 0, 4, 32, p, s), "q must not be x"),
        (lambda: ops.quantize_rows(p, 0, 4, 32, q, s, q_ld=16), "q_ld"),
        (lambda: ops.layer_norm_quantize(p, 0, 4, 32, q, s, eps=-1.0), "eps"),
        (lambda: ops.layer_norm_quantize(p, 7, 4, 32, q, s), "x_type"),
        (lambda: ops.quantized_linear(0, w, o, 0, 4, 8, 32), "x is null"),
        (lambda: ops.quantized_linear(q, 0, o, 0, 4, 8, 32), "w is null"),
        (lambda: ops.quantized_linear(q, w, 0, 0, 4, 8, 32), "out is null"),
        (lambda: ops.quantized_linear(q + 8, w, o, 0, 4, 8, 16, x_ld=32), "x is not aligned"),
        (lambda: ops.quantized_linear(q, w + 4, o, 0, 4, 8, 16, w_ld=32), "w is not aligned"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 20), "multiples of 16"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, w_ld=40), "multiples of 16"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, x_ld=16), "x_ld"),
        (lambda: ops.quantized_linear(q, w, o, 5, 4, 8, 32), "out_type"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, activation=2), "activation"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 131072), "in_features"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 0, 32, out_ld=8), "out_features"),
        (lambda: ops.quantized_linear(q, w, o, 0, -4, 8, 32), "rows"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, out_ld=7), "out_ld"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, residual=o, residual_ld=16), "in place"),
        (lambda: ops.quantized_linear(q, w, o, 0, 4, 8, 32, residual=p + 2), "residual"),
        (lambda: ops.quantized_linear(q, w, q, 1, 4, 8, 32), "out must not be x or w"),
        (lambda: dmx.Ops(1000), "no such device"),
    ]
    for call, why in calls:
        with pytest.raises(dmx.DmxError, match=why) as e:
            call()
        assert e.value.code == 1, why
    ops.check()  # nothing was launched, the context is as before
    assert ops.layer_norm_backward_workspace(-1, 8) == 0 and ops.layer_norm_backward_workspace(4, 0) == 0
    with pytest.raises(dmx.DmxError, match="ops is null"):
        dmx._check(dmx.lib().dmx_ops_check(None, None))
    assert ctypes.c_void_p(ops._h.value).value
