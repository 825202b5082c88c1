"""The autograd module as it is linked, without a GPU."""
import subprocess
import sys

import pytest

from need_b200 import build

REFUSED = """
import torch
from need_b200 import need_kernels as nk
x, d = torch.zeros(2, 3, 8), torch.ones(8)
for call in (lambda: nk.gated_scan_train(x, x, x), lambda: nk.ssd_scan_train(x, x, x, x, x, d, 0.001, 0.2),
             lambda: nk.ssd_conv_silu_train(x, torch.ones(8, 1, 3)), lambda: nk.rms_norm_train(x, d)):
    try:
        call()
    except RuntimeError as e:
        print(e)
"""


@pytest.fixture(scope="module")
def ext():
    build.build()
    return build.EXT


def test_the_module_runs_on_the_shared_cpp_library(ext):
    """Its own copy (a compiler that finds the archive only) would not share torch's locale."""
    with open(ext, "rb") as f:
        assert b"\0libstdc++.so.6\0" in f.read()
    cmd = build._ext_command()
    assert "-nostdlib++" in cmd and "-l:libstdc++.so.6" in cmd


def test_error_texts_format_numbers(ext):
    """In a process of its own: with a second C++ library in it, this ended it."""
    p = subprocess.run([sys.executable, "-c", REFUSED], capture_output=True, text=True, cwd=build.ROOT)
    assert p.returncode == 0, p.stderr[-500:]
    lines = p.stdout.splitlines()
    assert len(lines) == 4 and all("[2, 3, 8] on cpu" in s for s in lines), lines
