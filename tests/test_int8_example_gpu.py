"""The feed-forward example (examples/int8_feed_forward.py): its operators
together, as a program uses them."""

import os
import sys

import pytest

import synth

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module")
def setup():
    import dmx
    import int8_feed_forward as example

    weights = synth.random_weights(3)
    weights[example.LAYER + "gamma_2.scale"][:] = 1.0
    ops = dmx.Ops(0)
    yield example, weights, ops
    ops.check()
    ops.close()


def test_block_is_the_plain_one_on_the_same_integers(setup):
    # the block in 64 bits from the integers it holds; what is left are ties of
    # the activations' roundings and the hidden layer's 16 bits (2^-9 each)
    import torch

    example, weights, ops = setup
    block = example.Int8FeedForward(ops, weights)
    x = example.tokens(300, 5)
    y = block(x)
    h = torch.nn.functional.layer_norm(x.double(), (512,), block.norm_weight.double(),
                                       block.norm_bias.double(), example.EPS)

    def linear(layer, h):
        s = h.abs().amax(1, keepdim=True) / 127
        return (h / s).round() * s @ (layer.w.double() * layer.scale.double()[:, None]).t() + layer.bias.double()

    want = linear(block.down, torch.nn.functional.gelu(linear(block.up, h)))
    off = (y.double() - x.double() - want).norm() / want.norm()
    # a hidden value's 2^-9 may move it by one of its 127 steps, seldom more:
    # about 1/127 of the largest value, 1/3 / 127 of a row's norm at the worst
    assert off < 1 / 127


def test_norm_gradients_are_those_of_the_straight_through_block(setup):
    # against autograd through the same formula with the roundings' values kept
    import torch

    example, weights, ops = setup
    block = example.Int8FeedForward(ops, weights)
    x = example.tokens(256, 6)
    target = example.feed_forward_f32(weights, x)
    _, dweight, dbias = block.norm_gradients(x, target)
    w = block.norm_weight.double().requires_grad_()
    b = block.norm_bias.double().requires_grad_()

    def linear(layer, h):
        s = h.detach().abs().amax(1, keepdim=True) / 127
        h = h + ((h / s).round() * s - h).detach()
        return h @ (layer.w.double() * layer.scale.double()[:, None]).t() + layer.bias.double()

    h = torch.nn.functional.layer_norm(x.double(), (512,), w, b, example.EPS)
    y = x.double() + linear(block.down, torch.nn.functional.gelu(linear(block.up, h)))
    ((y - target.double()) ** 2).mean().backward()
    # each of the two gradients on the way is rounded to 8 bits per token: an
    # error of at most half a step, 0.5 / 127 of a row's largest value, random
    # over the 256 tokens that are summed
    for got, want in ((dweight, w.grad), (dbias, b.grad)):
        assert (got.double() - want).norm() / want.norm() < 0.05


def test_tuning_the_norm_follows_a_drift_of_the_features(setup):
    # gains of exp(0.3 n) per feature leave an error of some 0.3^2 of the signal;
    # the norm's weight can undo most of it, on tokens it has not seen too
    example, weights, ops = setup
    block = example.Int8FeedForward(ops, weights)
    x, target = example.drifted(weights, example.tokens(2688, 7))
    fresh, fresh_target = example.drifted(weights, example.tokens(2688, 1007))
    before = (block(fresh) - fresh_target).square().mean().item()
    errors = example.tune(block, x, target, 60)
    after = (block(fresh) - fresh_target).square().mean().item()
    assert errors[-1] < errors[0] / 4 and after < before / 4


def test_layer_is_read_from_a_checkpoint(setup, tmp_path):
    import numpy as np

    example, weights, ops = setup
    path = tmp_path / "model.safetensors"
    path.write_bytes(synth.write_safetensors(weights))
    got = example.load_layer(path)
    assert all(np.array_equal(v, weights[k]) for k, v in got.items()) and len(got) == 7
