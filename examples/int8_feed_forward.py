"""A transformer layer's feed-forward block on 8-bit integers, and the tuning
of its layer norm.

The block is the one of the separator's cross-transformer,

    y = x + gamma * (gelu(norm(x) w1^T + b1) w2^T + b2),

with both weight matrices quantised per output channel and the activations per
token, as they come: four kernels, of which the two products run on the
tensor cores' integer path. The integers stay as they are; the norm's weight
and bias (1024 numbers) can still be trained. Here they adapt the block to
tokens whose features have drifted, each by a gain of its own, so that it gives
again what the block in 32 bits gave on the tokens before. Gradients pass
straight through the roundings: through a product as the same operators on the
transposed integers, through the norm as ``layer_norm_backward``.

    python examples/int8_feed_forward.py [checkpoint] [--steps 60]

Without a checkpoint the weights are the seeded random ones of the tests.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "demucs-wgpu_b200"))
import dmx  # noqa: E402
import synth  # noqa: E402

TYPES = {torch.float32: dmx.TYPE_F32, torch.float16: dmx.TYPE_F16, torch.bfloat16: dmx.TYPE_BF16}
LAYER = "crosstransformer.layers.0."
EPS = 1e-5


def _stream():
    return torch.cuda.current_stream().cuda_stream


class Int8Linear:
    """A linear layer's weights as int8 rows with a scale each, laid out once."""

    def __init__(self, ops, weight, bias, gain=None):
        self.ops, (self.n, self.k) = ops, weight.shape
        assert self.n % 16 == 0 and self.k % 16 == 0  # rows start on 16 bytes, transposed ones too
        self.w = torch.empty(self.n, self.k, dtype=torch.int8, device="cuda")
        self.scale = torch.empty(self.n, device="cuda")
        ops.quantize_rows(weight.data_ptr(), dmx.TYPE_F32, self.n, self.k, self.w.data_ptr(),
                          self.scale.data_ptr(), stream=_stream())
        self.bias = bias.clone()
        if gain is not None:  # a per-channel gain after the layer is part of its scales
            self.scale *= gain
            self.bias *= gain
        self.wt = None

    def __call__(self, q, q_scale, dtype, gelu=False, residual=None):
        out = torch.empty(q.shape[0], self.n, dtype=dtype, device="cuda")
        self.ops.quantized_linear(
            q.data_ptr(), self.w.data_ptr(), out.data_ptr(), TYPES[dtype], q.shape[0], self.n, self.k,
            x_scale=q_scale.data_ptr(), w_scale=self.scale.data_ptr(), bias=self.bias.data_ptr(),
            activation=dmx.ACT_GELU if gelu else dmx.ACT_NONE,
            residual=0 if residual is None else residual.data_ptr(), stream=_stream())
        return out

    def backward(self, dy):
        """The gradient of the layer's input, dy rounded to 8 bits per token too."""
        if self.wt is None:
            self.wt = self.w.t().contiguous()
        q, s = quantize(self.ops, dy, col_scale=self.scale)
        dx = torch.empty(dy.shape[0], self.k, device="cuda")
        self.ops.quantized_linear(q.data_ptr(), self.wt.data_ptr(), dx.data_ptr(), dmx.TYPE_F32,
                                  dy.shape[0], self.k, self.n, x_scale=s.data_ptr(), stream=_stream())
        return dx


def quantize(ops, x, col_scale=None):
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    scale = torch.empty(x.shape[0], device="cuda")
    ops.quantize_rows(x.data_ptr(), TYPES[x.dtype], *x.shape, q.data_ptr(), scale.data_ptr(),
                      col_scale=0 if col_scale is None else col_scale.data_ptr(), stream=_stream())
    return q, scale


class Int8FeedForward:
    """``weights`` holds the layer's tensors by the checkpoint's names."""

    def __init__(self, ops, weights):
        t = {k: torch.from_numpy(v).cuda() for k, v in weights.items() if k.startswith(LAYER)}
        self.ops = ops
        self.norm_weight = t[LAYER + "norm2.weight"].clone()
        self.norm_bias = t[LAYER + "norm2.bias"].clone()
        self.up = Int8Linear(ops, t[LAYER + "linear1.weight"], t[LAYER + "linear1.bias"])
        self.down = Int8Linear(ops, t[LAYER + "linear2.weight"], t[LAYER + "linear2.bias"],
                               gain=t[LAYER + "gamma_2.scale"])

    def _norm(self, x, mean=None, rstd=None):
        q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        scale = torch.empty(x.shape[0], device="cuda")
        self.ops.layer_norm_quantize(
            x.data_ptr(), dmx.TYPE_F32, *x.shape, q.data_ptr(), scale.data_ptr(),
            weight=self.norm_weight.data_ptr(), bias=self.norm_bias.data_ptr(), eps=EPS,
            mean=0 if mean is None else mean.data_ptr(), rstd=0 if rstd is None else rstd.data_ptr(),
            stream=_stream())
        return q, scale

    def __call__(self, x):
        hidden = self.up(*self._norm(x), torch.bfloat16, gelu=True)
        return self.down(*quantize(self.ops, hidden), torch.float32, residual=x)

    def norm_gradients(self, x, target):
        """The mean squared error against ``target`` and its gradients of the norm's weight and bias."""
        rows, cols = x.shape
        mean, rstd = torch.empty(2, rows, device="cuda")
        z = self.up(*self._norm(x, mean, rstd), torch.float32)
        hidden = torch.nn.functional.gelu(z)
        off = self.down(*quantize(self.ops, hidden), torch.float32, residual=x) - target
        dhidden = self.down.backward(off * (2 / off.numel()))
        density = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        dz = dhidden * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * density)
        dy = self.up.backward(dz)
        dweight, dbias = torch.empty(2, cols, device="cuda")
        size = self.ops.layer_norm_backward_workspace(rows, cols)
        room = torch.empty(size, dtype=torch.uint8, device="cuda")
        self.ops.layer_norm_backward(
            dy.data_ptr(), dmx.TYPE_F32, x.data_ptr(), dmx.TYPE_F32, mean.data_ptr(), rstd.data_ptr(),
            rows, cols, room.data_ptr(), size, dweight=dweight.data_ptr(), dbias=dbias.data_ptr(),
            stream=_stream())
        return (off * off).mean().item(), dweight, dbias


def feed_forward_f32(weights, x):
    """The block in 32 bits."""
    t = {k[len(LAYER):]: torch.from_numpy(v).cuda() for k, v in weights.items() if k.startswith(LAYER)}
    f = torch.nn.functional
    h = f.layer_norm(x, x.shape[1:], t["norm2.weight"], t["norm2.bias"], EPS)
    h = f.gelu(f.linear(h, t["linear1.weight"], t["linear1.bias"]))
    return x + t["gamma_2.scale"] * f.linear(h, t["linear2.weight"], t["linear2.bias"])


def load_layer(path):
    """The layer's tensors of a checkpoint file, decoded by the library."""
    with open(path, "rb") as f:
        blob = f.read()
    names = ["norm2.weight", "norm2.bias", "linear1.weight", "linear1.bias", "linear2.weight",
             "linear2.bias", "gamma_2.scale"]
    return {LAYER + n: dmx.read_tensor(blob, LAYER + n) for n in names}


def tokens(rows, seed):
    """Tokens as a residual stream holds them: features of different spread, a few far larger."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = 0.5 + torch.rand(512, generator=g, device="cuda")
    spread[torch.randperm(512, generator=g, device="cuda")[:6]] *= 12
    return torch.randn(rows, 512, generator=g, device="cuda") * spread


def drifted(weights, x, seed=9):
    """The tokens with a gain per feature, and what the block should make of them:
    the branch that the 32-bit block adds to the tokens as they were."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    seen = x * torch.exp(0.3 * torch.randn(x.shape[1], generator=g, device="cuda"))
    return seen, seen + (feed_forward_f32(weights, x) - x)


def tune(block, x, target, steps, rate=1e-2):
    """Adam on the norm's weight and bias; returns every step's error."""
    params = [block.norm_weight, block.norm_bias]
    state = [(torch.zeros_like(p), torch.zeros_like(p)) for p in params]
    errors = []
    for step in range(1, steps + 1):
        error, *grads = block.norm_gradients(x, target)
        errors.append(error)
        for p, (m, v), g in zip(params, state, grads):
            m.mul_(0.9).add_(g, alpha=0.1)
            v.mul_(0.99).addcmul_(g, g, value=0.01)
            p.sub_(rate * (m / (1 - 0.9**step)) / ((v / (1 - 0.99**step)).sqrt() + 1e-12))
    return errors


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("checkpoint", nargs="?")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--rows", type=int, default=2688, help="tokens: one segment's by default")
    args = ap.parse_args()
    weights = load_layer(args.checkpoint) if args.checkpoint else synth.random_weights(0)
    if not args.checkpoint:  # random init has gamma 1e-4, which would hide the block
        weights[LAYER + "gamma_2.scale"][:] = 1.0
    ops = dmx.Ops(0)
    block = Int8FeedForward(ops, weights)

    def report(name, x, target):
        size, error = (target - x).square().mean().item(), (block(x) - target).square().mean().item()
        print(f"{name}: the branch's signal is {10 * math.log10(size / error):.1f} dB over the error")

    x, fresh = tokens(args.rows, 1), tokens(args.rows, 2)
    report("8-bit block", x, feed_forward_f32(weights, x))
    report("on drifted tokens", *drifted(weights, fresh))
    tune(block, *drifted(weights, x), args.steps)
    report(f"norm tuned over {args.steps} steps, on other drifted tokens", *drifted(weights, fresh))
    ops.check(_stream())
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(10):
        block(x)
    begin.record()
    for _ in range(50):
        block(x)
    end.record()
    end.synchronize()
    print(f"one pass: {begin.elapsed_time(end) / 50 * 1e3:.1f} us")


if __name__ == "__main__":
    main()
