"""CPU tests of the operators on parameter rows: struct layouts, sizes and the refusals that need
no GPU."""
import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from parameter_server_amd import _abi, operators, PsxError


def test_struct_layouts_match_header(tmp_path):
    structs = {"psx_matrix": _abi.psx_matrix, "psx_adapter": _abi.psx_adapter, "psx_requests": _abi.psx_requests,
               "psx_scores": _abi.psx_scores}
    src = tmp_path / "probe.c"
    lines = [f'printf("%zu ", sizeof({n}));' + "".join(f'printf("%zu ", offsetof({n}, {f[0]}));' for f in c._fields_)
             for n, c in structs.items()]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "psx.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I", os.path.dirname(_abi.HEADER_PATH), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for c in structs.values():
        want += [ctypes.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]
    assert got == want


def test_checkpoint_bytes(built_lib):
    n = ctypes.c_size_t()
    for rows, cols, want in [(0, 0, 0), (1, 1, 33), (3, 32, 99), (3, 33, 198), (1 << 20, 1 << 14, (1 << 20) * 512 * 33)]:
        assert built_lib.psx_checkpoint_bytes(rows, cols, ctypes.byref(n)) == 0 and n.value == want
    for rows, cols in [(-1, 3), (3, -1), (1 << 40, 1 << 30)]:
        assert built_lib.psx_checkpoint_bytes(rows, cols, ctypes.byref(n)) == 1
    assert built_lib.psx_checkpoint_bytes(1, 1, None) == 1


def test_null_handles_are_rejected(built_lib):
    L, out = built_lib, ctypes.c_void_p()
    m, s, r = _abi.psx_matrix(), _abi.psx_scores(), _abi.psx_requests()
    assert L.psx_adapters_create(None, 0, 0, None, 0, ctypes.byref(out)) == 1
    assert L.psx_adapters_destroy(None) == 1
    assert L.psx_adapters_info(None, None, None) == 1
    assert L.psx_adapters_sizes(None, 1, None, None) == 1
    assert L.psx_adapters_forward(None, r, m, None, m, None, None) == 1
    assert L.psx_adapters_backward(None, r, m, None, m, None, None, None, None, None, 1.0, None, None) == 1
    assert L.psx_checkpoint_store(None, m, None, None) == 1
    assert L.psx_checkpoint_load(None, None, m, None) == 1
    assert L.psx_position_bias_create(None, 0, 0, 8, 16, 1, ctypes.byref(out)) == 1
    assert L.psx_position_bias_destroy(None) == 1
    assert L.psx_position_bias_forward(None, s, 0, None) == 1
    assert L.psx_position_bias_work(None, 1, 1, 1, None) == 1
    assert L.psx_position_bias_backward(None, s, 0, 1.0, None, None, None) == 1


class _Server:
    device = 0


@pytest.mark.parametrize("t", [torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.float64)])
def test_host_tensors_are_refused(t):
    with pytest.raises(PsxError) as e:
        operators._matrix(_Server(), t, "x")
    assert e.value.status == 1 and "device" in str(e.value)


def test_act_types():
    for dt, want in ((torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)):
        assert operators._act(dt, "x") == want
    with pytest.raises(PsxError):
        operators._act(torch.int32, "x")
