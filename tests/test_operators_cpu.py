"""The operators' refusals that need no device, and their workspace sizes."""

import pytest

import dmx


def test_calls_without_a_context_are_refused():
    L = dmx.lib()
    calls = (
        lambda: L.dmx_layer_norm(None, bytes(128), None),
        lambda: L.dmx_layer_norm_backward(None, bytes(192), None),
        lambda: L.dmx_quantize_rows(None, bytes(128), None),
        lambda: L.dmx_layer_norm_quantize(None, bytes(128), None),
        lambda: L.dmx_quantized_linear(None, bytes(192), None),
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


def test_packed_arguments_have_the_layout_of_the_structs(tmp_path):
    # the binding's packed fields, byte for byte, against what a C++ compiler lays out
    import os
    import struct
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = {
        "dmx_layer_norm_args": (dmx._LAYER_NORM_ARGS, "x x_type x_ld weight bias param_type rows cols eps "
                                "y y_type y_ld mean rstd"),
        "dmx_layer_norm_backward_args": (
            dmx._LAYER_NORM_BACKWARD_ARGS, "dy dy_type dy_ld x x_type x_ld weight param_type mean rstd rows "
            "cols dx dx_ld dweight dbias workspace workspace_bytes"),
        "dmx_quantize_rows_args": (dmx._QUANTIZE_ROWS_ARGS, "x x_type x_ld col_scale rows cols q q_ld scale"),
        "dmx_layer_norm_quantize_args": (
            dmx._LAYER_NORM_QUANTIZE_ARGS, "x x_type x_ld weight bias param_type rows cols eps q q_ld scale "
            "mean rstd"),
        "dmx_quantized_linear_args": (
            dmx._QUANTIZED_LINEAR_ARGS, "x x_ld x_scale w w_ld w_scale bias rows out_features in_features "
            "activation residual residual_ld out out_type out_ld"),
    }
    lines = []
    for name, (_, names) in fields.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f in names.split()]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.cpp"
    src.write_text('#include <cstddef>\n#include <cstdio>\n#include "dmx.h"\nint main() {\n'
                   + "\n".join(lines) + "\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, *offsets = line.split()
        pack, names = fields[name]
        count = len(names.split())
        zeros = pack(*[0] * count)
        assert len(zeros) <= int(size) <= len(zeros) + 7  # trailing padding at most
        for i, offset in enumerate(offsets):
            one = pack(*[1 if j == i else 0 for j in range(count)])
            first = next(b for b in range(len(one)) if one[b])
            # an integer 1 is its lowest byte; the float 1 has its first set byte at offset + 2
            assert first == int(offset) + (2 if names.split()[i] == "eps" else 0), (name, names.split()[i])


def test_backward_workspace_of_more_rows_serves_fewer():
    size = dmx.lib().dmx_layer_norm_backward_workspace
    for cols in (1, 64, 200, 512, 1000, 1031, 2048, 8195, 16384, 16385, 40000):
        last = 0
        for rows in range(1, 12000 if cols <= 512 else 5000):
            got = size(rows, cols)
            assert got >= last, (rows, cols)
            last = got
        assert size(10**6, cols) >= last and size(2**31 - 1, cols) == size(2**31 - 2, cols)
