"""The serving operators at the ends of their ranges: widths, magnitudes and
positions where a step of the computation leaves the range that its result
stays in.

The forms, tolerances and helpers are those of test_gpu_serving.py; what a
test adds to a tolerance is derived beside it."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))

ALONE = """
import sys
sys.path.insert(0, {here!r})
import torch
from conftest import load_m3
from test_gpu_serving import check_norm, run_norm, strided
m3 = load_m3()
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(2, {width}, generator=g, device="cuda").bfloat16()
w = torch.randn({width}, generator=g, device="cuda").bfloat16()
if {shifted}:
    x = strided(x, 0, 1)
check_norm(x, w, {group}, *run_norm(m3, x, w, {group}))
print("fine")
"""


@pytest.mark.parametrize("width, group, shifted", [
    (12272, 12272, True), (12273, 12273, False), (12287, 12287, False), (12288, 12, False), (12288, 12288, True),
])
def test_norm_widths_near_the_default_shared_memory(m3, gpu, width, group, shifted):
    """Rows of about 48 KB in F32, as the first norm of a process: no wider row has been there before."""
    text = ALONE.format(here=HERE, width=width, group=group, shifted=shifted)
    child = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=300)
    assert child.returncode == 0 and child.stdout.strip() == "fine", child.stderr[-2000:]
