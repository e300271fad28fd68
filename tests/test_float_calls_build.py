"""The module of argument structures builds and reads tensors whatever torch's headers offer."""
import importlib
import os
import subprocess
import sys
import sysconfig

import pytest
import torch

from conftest import PKG, ROOT

SOURCE = os.path.join(ROOT, PKG, "csrc", "float_calls.c")
OLD = """#define DLPACK_MAJOR_VERSION 1
#define DLPACK_MINOR_VERSION 1
typedef struct { int major, minor; } DLPackVersion;
"""
USE = """
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("float_calls", sys.argv[1])
m = importlib.util.module_from_spec(spec)
spec.loader.exec_module(m)
m.setup(torch.Tensor, torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.empty, lambda: 0, 0, getattr(torch.Tensor, "__dlpack_c_exchange_api__", None))
for call, args in ((m.sample, (torch.zeros(2, 5), torch.zeros(2), None, 1.0, 0, 1.0, 0.0)), (m.sample, ([1.0],) + (None,) * 6)):
    try:
        call(*args)
    except ValueError as e:
        print(e)
"""


@pytest.mark.parametrize("header", [None, OLD, "torch"])
def test_it_builds_with_any_headers(tmp_path, header):
    include = tmp_path / "include"
    (include / "ATen").mkdir(parents=True)
    if header == OLD:
        (include / "ATen" / "dlpack.h").write_text(OLD)
    more = os.path.join(os.path.dirname(torch.__file__), "include") if header == "torch" else str(include)
    out = str(tmp_path / "float_calls.so")
    res = subprocess.run(["gcc", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I", sysconfig.get_paths()["include"],
                          "-I", more, "-o", out, SOURCE], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    got = subprocess.run([sys.executable, "-c", USE, out], capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    assert got.stdout.splitlines() == ["sample: logits is no tensor on a GPU", "sample: logits is no tensor"]


@pytest.mark.gpu
def test_structures_are_the_same_without_the_exchange_interface(float_libpath, tmp_path):
    """the module once more, built without the header: bytes of every call's structure"""
    K = importlib.import_module(PKG + ".float_kernel")
    out = str(tmp_path / "float_calls.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I", sysconfig.get_paths()["include"], "-o", out, SOURCE], check=True)
    spec = importlib.util.spec_from_file_location("float_calls", out)
    other = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(other)
    import ctypes
    other.setup(torch.Tensor, torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.empty, torch.cuda.current_device,
                ctypes.cast(K._paged_scratch, ctypes.c_void_p).value, getattr(torch.Tensor, "__dlpack_c_exchange_api__", None))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        pool = torch.zeros(9, 16, 2 * 64 + 8, dtype=dt, device="cuda")
        k, v = pool[..., :64].unflatten(2, (2, 32)), pool[..., 64:128].unflatten(2, (2, 32))
        table, rows, lengths = i32(0, 1, 2, 3, 4, 5).view(2, 3), i32(0, 2, 3), i32(20, 7)
        q, gate = torch.zeros(3, 4, 32, dtype=dt, device="cuda"), torch.zeros(3, 6, 32, dtype=dt, device="cuda")[:, :4]
        o, new = torch.empty_like(q), q[:, :2]
        cs, u = torch.zeros(40, 8, 2, device="cuda"), torch.zeros(3, device="cuda")
        logits, drawn = torch.zeros(3, 48, dtype=dt, device="cuda")[:, :40], torch.zeros(3, dtype=torch.int64, device="cuda")
        first = [m.paged_attention(q, k, v, table, rows, lengths, o, 0.5, 7, 2, gate, 0.7) for m in (K._calls, other)]
        # the scratch of either call is its own: the eight bytes of its address stand behind eight others
        a, b = (x[0][:64] + x[0][72:] for x in first)
        assert a == b and first[0][1].shape == first[1][1].shape
        for name, args in (("write_pages", (new, new, k, v, table, rows, lengths, q, o, cs, True)), ("copy_pages", ([pool, pool[:, :8]], [0, 1], [2, 3], 5)),
                           ("sample", (logits, u, drawn, u, 3, 0.5, u))):
            x, y = getattr(K._calls, name)(*args), getattr(other, name)(*args)
            assert x == y if name != "sample" else (x[0] == y[0] and x[1] is y[1])
