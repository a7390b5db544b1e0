"""The cases by which the layer norm and the 8-bit linear layer are measured.

Three operators, as the feed-forward and projection layers of a transformer
use them (tokens are rows, features are columns):

* ``norm``: the layer norm, y = (x - mean) / sqrt(var + eps) * weight + bias,
  with the row means and reciprocal deviations a training step keeps;
* ``norm_back``: its backward pass, with the gradients of x, weight and bias;
* ``linear``: act(x w^T + bias) + residual on 8-bit integers, with one scale
  per token and one per output channel. ``source`` says what the call begins
  with: ``int8`` (tokens already quantised), ``float`` (tokens it quantises
  first) or ``norm`` (tokens it normalises and quantises first).

Where ``own`` is false, ``run`` is the plain form: elementary torch operations
in 32 bits. Where it is true, ``run`` calls the library's entry points.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one 7.8 s segment's spectral tokens (8 x 336 of 512 features), 32 bits throughout
        {"name": "norm segment", "op": "norm", "rows": 2688, "cols": 512, "x": "f32", "y": "f32",
         "params": "f32", "pad": 0},
        # the 42 segments of a 240 s track in one forward, 16-bit output for the linear that follows
        {"name": "norm track", "op": "norm", "rows": 112896, "cols": 512, "x": "f32", "y": "bf16",
         "params": "f32", "pad": 0},
        # a wide model's tokens at an odd width, half precision throughout
        {"name": "norm odd", "op": "norm", "rows": 1023, "cols": 5001, "x": "f16", "y": "f16",
         "params": "f16", "pad": 0},
        # training on one segment
        {"name": "back segment", "op": "norm_back", "rows": 2688, "cols": 512, "x": "f32", "y": "f32",
         "params": "f32", "pad": 0},
        # training on a whole track's tokens, the gradient arriving in 16 bits
        {"name": "back track", "op": "norm_back", "rows": 112896, "cols": 512, "x": "f32", "y": "bf16",
         "params": "f32", "pad": 0},
        # a wide model's training step, odd in both lengths, rows padded to 16 bytes
        {"name": "back wide", "op": "norm_back", "rows": 4095, "cols": 8195, "x": "bf16", "y": "bf16",
         "params": "bf16", "pad": 5},
        # one token of a streaming decode: norm, quantise and project
        {"name": "linear token", "op": "linear", "source": "norm", "rows": 1, "k": 4096, "n": 4096,
         "x": "bf16", "y": "bf16", "act": "none", "residual": False},
        # a few tokens of an odd count on odd widths, quantised already
        {"name": "linear few", "op": "linear", "source": "int8", "rows": 37, "k": 2050, "n": 5003,
         "x": "bf16", "y": "f32", "act": "none", "residual": False},
        # the first feed-forward layer of one segment, norm included
        {"name": "linear segment", "op": "linear", "source": "norm", "rows": 2688, "k": 512, "n": 2048,
         "x": "f32", "y": "bf16", "act": "gelu", "residual": False},
        # the first feed-forward layer of a whole track
        {"name": "linear track up", "op": "linear", "source": "int8", "rows": 112896, "k": 512,
         "n": 2048, "x": "bf16", "y": "bf16", "act": "gelu", "residual": False},
        # the second one, from its 16-bit activations to the 32-bit residual stream
        {"name": "linear track down", "op": "linear", "source": "float", "rows": 112896, "k": 2048,
         "n": 512, "x": "bf16", "y": "f32", "act": "none", "residual": True},
        # the square product of a large model's prompt
        {"name": "linear large", "op": "linear", "source": "int8", "rows": 8192, "k": 8192, "n": 8192,
         "x": "bf16", "y": "bf16", "act": "none", "residual": False},
    ]


def _length(rng, low, high):
    """A length spread over the logarithm of [low, high], odd ones as often as even ones."""
    while True:
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))
        v = min(max(v, low), high)
        if rng.random() < 0.3:  # widths of whole vectors and tiles are common
            v = max(low, v - v % (16 if v < 512 else 128) or v)
        if v != 3072:
            return v


def draw(rng):
    op = rng.choice(("norm", "norm_back", "linear", "linear"))
    if op == "linear":
        while True:
            rows, k, n = _length(rng, 1, 112896), _length(rng, 32, 8192), _length(rng, 32, 8192)
            if rows * k * n <= 8192**3 and rows * max(k, n) <= 112896 * 2048:
                break
        source = rng.choice(("int8", "float", "norm"))
        # after a norm in other roundings a value near a tie may take the next integer: 16-bit outputs there
        y = rng.choice(("f16", "bf16") if source == "norm" else ("f16", "bf16", "f32"))
        return {"op": op, "source": source, "rows": rows, "k": k, "n": n,
                "x": rng.choice(("f32", "f16", "bf16")), "y": y, "act": rng.choice(("none", "gelu")),
                "residual": rng.random() < 0.3}
    while True:
        rows, cols = _length(rng, 1, 112896), _length(rng, 32, 16384)
        if rows * cols <= 112896 * 512:
            break
    x, y = rng.choice((("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"),
                       ("bf16", "f32")))
    return {"op": op, "rows": rows, "cols": cols, "x": x, "y": y, "params": rng.choice((x, "f32")),
            "pad": rng.choice((0, 0, 8 - cols % 8, 3))}


# --- inputs -----------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(g, rows, cols, dtype, pad=0):
    """Activations as a residual stream holds them: features of different spread and offset, some far larger."""
    spread = 0.5 + torch.rand(cols, generator=g, device="cuda")
    spread *= 1 + 7 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
    x = torch.randn(rows, cols + pad, generator=g, device="cuda")[:, :cols]
    x.mul_(spread).add_(0.3 * torch.randn(cols, generator=g, device="cuda"))
    if dtype is torch.float32:
        return x
    held = torch.empty(rows, cols + pad, dtype=dtype, device="cuda")[:, :cols]
    held.copy_(x)
    return held


def _pitch(n):
    """The row pitch of 8-bit rows: whole 16-byte units."""
    return (n + 15) // 16 * 16


def _weights(g, n, k):
    """An output-channel quantised weight matrix: int8 rows, one scale each."""
    w = torch.randn(n, k, generator=g, device="cuda") * (0.5 + torch.rand(n, 1, generator=g, device="cuda"))
    w /= math.sqrt(k)
    scale = w.abs().amax(dim=1) / 127
    q = torch.zeros(n, _pitch(k), dtype=torch.int8, device="cuda")[:, :k]
    q.copy_((w / scale[:, None]).round().clamp_(-127, 127))
    return q, scale


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        y = TYPES[case["y"]]
        s["w"], s["w_scale"] = _weights(g, n, k)
        s["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda")
        s["out"] = torch.empty(rows, n, dtype=y, device="cuda")
        s["res"] = torch.randn(rows, n, generator=g, device="cuda").to(y) if case["residual"] else None
        s["q"] = torch.zeros(rows, _pitch(k), dtype=torch.int8, device="cuda")[:, :k]
        s["q_scale"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        x = _tokens(g, rows, k, TYPES[case["x"]])
        if case["source"] == "int8":
            f = x.float()
            s["q_scale"].copy_(f.abs().amax(dim=1) / 127)
            s["q"].copy_((f / s["q_scale"][:, None]).round_())
        else:
            s["in"] = x
        if case["source"] == "norm":
            s["gamma"] = 1 + 0.2 * torch.randn(k, generator=g, device="cuda")
            s["beta"] = 0.1 * torch.randn(k, generator=g, device="cuda")
        return s
    rows, cols, pad = case["rows"], case["cols"], case["pad"]
    x, y, params = TYPES[case["x"]], TYPES[case["y"]], TYPES[case["params"]]
    s["in"] = _tokens(g, rows, cols, x, pad)
    s["gamma"] = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(params)
    s["beta"] = (0.1 * torch.randn(cols, generator=g, device="cuda")).to(params)
    s["mean"] = torch.empty(rows, device="cuda")
    s["rstd"] = torch.empty(rows, device="cuda")
    if case["op"] == "norm":
        s["out"] = torch.empty(rows, cols + pad, dtype=y, device="cuda")[:, :cols]
        return s
    f = s["in"].float()
    s["mean"].copy_(f.mean(dim=1))
    s["rstd"].copy_(1 / torch.sqrt(f.var(dim=1, unbiased=False) + EPS))
    s["dy"] = torch.empty(rows, cols + pad, dtype=y, device="cuda")[:, :cols]
    s["dy"].copy_(0.02 * torch.randn(rows, cols, generator=g, device="cuda"))
    s["dx"] = torch.empty(rows, cols + pad, dtype=x, device="cuda")[:, :cols]
    s["dgamma"] = torch.empty(cols, device="cuda")
    s["dbeta"] = torch.empty(cols, device="cuda")
    s["room"] = {}
    return s


# --- the plain forms --------------------------------------------------------


def _plain_norm(x, gamma, beta):
    x = x.float()
    mean = x.mean(dim=1)
    c = x - mean[:, None]
    rstd = 1 / torch.sqrt((c * c).mean(dim=1) + EPS)
    return c * rstd[:, None] * gamma.float() + beta.float(), mean, rstd


def _plain_quantise(x):
    top = x.abs().amax(dim=1)
    scale = top / torch.full_like(top, 127)  # a true quotient: by a plain number it would be a product
    return torch.nan_to_num(x / scale[:, None]).round(), scale


def _plain_linear(s):
    if s["source"] == "int8":
        q, q_scale = s["q"].float(), s["q_scale"]
    elif s["source"] == "float":
        q, q_scale = _plain_quantise(s["in"].float())
    else:
        q, q_scale = _plain_quantise(_plain_norm(s["in"], s["gamma"], s["beta"])[0])
    z = (q @ s["w"].float().t()) * q_scale[:, None] * s["w_scale"] + s["bias"]
    if s["act"] == "gelu":
        z = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if s["res"] is not None:
        z = z + s["res"].float()
    return z.to(s["out"].dtype)


def _plain(s):
    if s["op"] == "linear":
        return _plain_linear(s)
    if s["op"] == "norm":
        y, mean, rstd = _plain_norm(s["in"], s["gamma"], s["beta"])
        return {"y": y.to(s["out"].dtype), "mean": mean, "rstd": rstd}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (s["in"].float() - s["mean"][:, None]) * rstd
    g = dy * s["gamma"].float()
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))
    return {"dx": dx.to(s["in"].dtype), "dgamma": (dy * h).sum(dim=0), "dbeta": dy.sum(dim=0)}


# --- the library's operators ------------------------------------------------

_held = {}


def _library():
    """The binding and one operator context, as a program keeps them."""
    if "ops" not in _held:
        package = os.path.join(os.getcwd(), "demucs-wgpu_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import dmx

        _held["ops"] = dmx.Ops(torch.cuda.current_device())
        _held["types"] = {torch.float32: dmx.TYPE_F32, torch.float16: dmx.TYPE_F16,
                          torch.bfloat16: dmx.TYPE_BF16}
        _held["acts"] = {"none": dmx.ACT_NONE, "gelu": dmx.ACT_GELU}
    return _held["ops"], _held["types"], _held["acts"]


def _own(s):
    ops, types, acts = _library()
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "linear":
        q, q_scale, w, out, res = s["q"], s["q_scale"], s["w"], s["out"], s["res"]
        rows, k = q.shape
        if s["source"] == "float":
            x = s["in"]
            ops.quantize_rows(x.data_ptr(), types[x.dtype], rows, k, q.data_ptr(), q_scale.data_ptr(),
                              x_ld=x.stride(0), q_ld=q.stride(0), stream=stream)
        elif s["source"] == "norm":
            x = s["in"]
            ops.layer_norm_quantize(x.data_ptr(), types[x.dtype], rows, k, q.data_ptr(),
                                    q_scale.data_ptr(), weight=s["gamma"].data_ptr(),
                                    bias=s["beta"].data_ptr(), param_type=types[s["gamma"].dtype],
                                    eps=EPS, x_ld=x.stride(0), q_ld=q.stride(0), stream=stream)
        ops.quantized_linear(q.data_ptr(), w.data_ptr(), out.data_ptr(), types[out.dtype], rows,
                             w.shape[0], k, x_scale=q_scale.data_ptr(),
                             w_scale=s["w_scale"].data_ptr(), bias=s["bias"].data_ptr(),
                             activation=acts[s["act"]], residual=0 if res is None else res.data_ptr(),
                             x_ld=q.stride(0), w_ld=w.stride(0), stream=stream)
        return out
    x, gamma = s["in"], s["gamma"]
    rows, cols = x.shape
    if s["op"] == "norm":
        y = s["out"]
        ops.layer_norm(x.data_ptr(), types[x.dtype], rows, cols, y.data_ptr(), types[y.dtype],
                       weight=gamma.data_ptr(), bias=s["beta"].data_ptr(),
                       param_type=types[gamma.dtype], eps=EPS, x_ld=x.stride(0), y_ld=y.stride(0),
                       mean=s["mean"].data_ptr(), rstd=s["rstd"].data_ptr(), stream=stream)
        return {"y": y, "mean": s["mean"], "rstd": s["rstd"]}
    dy, dx = s["dy"], s["dx"]
    if "room" not in s["room"]:  # a training loop keeps its workspace
        size = ops.layer_norm_backward_workspace(rows, cols)
        s["room"]["room"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    room = s["room"]["room"]
    ops.layer_norm_backward(dy.data_ptr(), types[dy.dtype], x.data_ptr(), types[x.dtype],
                            s["mean"].data_ptr(), s["rstd"].data_ptr(), rows, cols,
                            room.data_ptr(), room.numel(), weight=gamma.data_ptr(),
                            param_type=types[gamma.dtype], dx=dx.data_ptr(),
                            dweight=s["dgamma"].data_ptr(), dbias=s["dbeta"].data_ptr(),
                            dy_ld=dy.stride(0), x_ld=x.stride(0), dx_ld=dx.stride(0), stream=stream)
    return {"dx": dx, "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def run(state):
    return _own(state) if own else _plain(state)


# --- what a pass costs, and what it gives in 64 bits --------------------------


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    rows = case["rows"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        moved = rows * k + 4 * rows if case["source"] == "int8" else rows * k * size[case["x"]]
        moved += 8 * k if case["source"] == "norm" else 0
        moved += n * k + 8 * n + rows * n * size[case["y"]] * (2 if case["residual"] else 1)
        return {"bytes": moved, "flops": 2 * rows * k * n}
    cols, x, y, params = case["cols"], size[case["x"]], size[case["y"]], size[case["params"]]
    if case["op"] == "norm":
        return {"bytes": rows * cols * (x + y) + 2 * cols * params + 8 * rows, "flops": 8 * rows * cols}
    return {"bytes": rows * cols * (2 * x + y) + cols * (params + 8) + 8 * rows, "flops": 14 * rows * cols}


def _exact_norm(x, gamma, beta):
    x = x.double()
    var, mean = torch.var_mean(x, dim=1, correction=0)
    rstd = (var + EPS).pow(-0.5)
    return torch.addcmul(beta.double(), (x - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1)), gamma.double()), mean, rstd


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        y, mean, rstd = _exact_norm(s["in"], s["gamma"], s["beta"])
        return {"y": y, "mean": mean, "rstd": rstd}
    if case["op"] == "norm_back":
        # from the chain rule through the mean and the deviation that the step was given
        n, dy = case["cols"], s["dy"].double()
        rstd = s["rstd"].double().unsqueeze(1)
        c = s["in"].double().sub_(s["mean"].double().unsqueeze(1))
        dgamma, dbeta = torch.einsum("rc,rc->c", dy, c * rstd), dy.sum(0)
        dh = dy.mul_(s["gamma"].double())
        dvar = (dh * c).sum(1, keepdim=True) * rstd.pow(3) / -2
        dx = dh * rstd - dh.sum(1, keepdim=True) * rstd / n + dvar * c * (2 / n)
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if case["source"] == "int8":
        q, q_scale = s["q"].double(), s["q_scale"].double()
    else:
        x = s["in"].double() if case["source"] == "float" else _exact_norm(s["in"], s["gamma"], s["beta"])[0]
        q_scale = torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127
        q = torch.where(q_scale.unsqueeze(1) > 0, x / q_scale.unsqueeze(1), 0).round_()
    z = torch.mm(q, s["w"].double().t())
    z.mul_(q_scale.unsqueeze(1)).mul_(s["w_scale"].double()).add_(s["bias"].double())
    if case["act"] == "gelu":
        z.mul_(torch.special.ndtr(z))
    return z if s["res"] is None else z.add_(s["res"].double())
