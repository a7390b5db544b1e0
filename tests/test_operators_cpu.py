"""The operators' refusals that need no device, and their workspace sizes."""

import pytest

import dmx


def test_calls_without_a_context_are_refused():
    L = dmx.lib()
    calls = (
        lambda: L.dmx_layer_norm(None, 16, 0, 8, None, None, 0, 1, 8, 1e-5, 32, 0, 8, None, None, None),
        lambda: L.dmx_layer_norm_backward(None, 16, 0, 8, 32, 0, 8, None, 0, 64, 64, 1, 8, 96, 8, None,
                                          None, None, 0, None),
        lambda: L.dmx_quantize_rows(None, 16, 0, 8, None, 1, 8, 32, 8, 64, None),
        lambda: L.dmx_layer_norm_quantize(None, 16, 0, 8, None, None, 0, 1, 8, 1e-5, 32, 8, 64, None,
                                          None, None),
        lambda: L.dmx_quantized_linear(None, 16, 16, None, 32, 16, None, None, 1, 1, 16, 0, None, 1, 64,
                                       0, 1, None),
        lambda: L.dmx_ops_check(None, None),
    )
    for call in calls:
        with pytest.raises(dmx.DmxError, match="ops is null") as e:
            dmx._check(call())
        assert e.value.code == 1
    L.dmx_ops_destroy(None)


def test_a_context_needs_a_device():
    with pytest.raises(dmx.DmxError) as e:
        dmx.Ops(10_000)
    assert e.value.code in (1, 3)  # no such device, or no device at all


def test_backward_workspace_holds_its_partial_sums():
    L = dmx.lib()
    size = L.dmx_layer_norm_backward_workspace
    assert size(0, 512) == 0 and size(-1, 512) == 0 and size(4, 0) == 0 and size(4, 2**40) == 0
    last = 0
    for rows in (1, 31, 32, 33, 500, 10_000, 10**6, 2**31 - 1):
        got = size(rows, 512)
        assert got >= 2 * 512 * 4 and got % (2 * 512 * 4) == 0 and got >= last
        last = got
    assert last <= 4096 * 2 * 512 * 4  # bounded, whatever the rows
