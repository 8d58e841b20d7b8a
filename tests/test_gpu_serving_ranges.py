"""The serving operators at the ends of their ranges: widths, magnitudes and
positions where a step of the computation leaves the range that its result
stays in.

The forms, tolerances and helpers are those of test_gpu_serving.py; what a
test adds to a tolerance is derived beside it."""

from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest

from test_gpu_serving import cache_rows, device_view

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


@pytest.mark.parametrize("heads, dim", [(8, 128), (3, 60)])
def test_cache_positions_past_32_bits(m3, gpu, heads, dim):
    """A start and a negative first offset whose difference passes 2^32: no such row has a slot."""
    import torch

    rows, page = 40, 16
    c = m3.Cache(8, page, heads, dim)
    table = torch.arange(8, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([-2 ** 31, rows], dtype=torch.int32, device="cuda")
    starts = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    batch = m3.CacheBatch(page_table=table.data_ptr(), page_table_stride=8, offsets=offsets.data_ptr(),
                          starts=starts.data_ptr(), sequences=1, rows=rows)
    data = torch.full((2, rows, heads, dim), 4.0, device="cuda")
    for call in (c.write, c.read):
        call(batch, cache_rows(m3, data[0]), cache_rows(m3, data[1]))
        with pytest.raises(m3.M3Failure) as failure:
            c.synchronize()
        assert failure.value.status == m3.OUT_OF_RANGE
        assert "row 0 was skipped: its position is outside the page table" in failure.value.message
    for pointer, shape, kind in zip(c.pointers(), 2 * ((8 * page, heads, dim), (8 * page, heads)), 2 * ("|u1", "<f4")):
        assert not bool(device_view(pointer, shape, kind).any())
    assert bool((data == 4.0).all())
    # a negative offset by itself is no fault: the rows go on where the sequence is
    starts.fill_(0)
    offsets.copy_(torch.tensor([-20, 30], dtype=torch.int32))
    c.write(batch, cache_rows(m3, data[0]), cache_rows(m3, data[1]))
    c.synchronize()
    written = device_view(c.pointers()[1], (8 * page, heads), "<f4").any(-1).cpu().numpy()
    assert np.array_equal(np.nonzero(written)[0], np.arange(20, 50))
