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

from test_gpu_serving import (TINY, U, cache_rows, device_view, e4m3_table, host, nearest_e4m3, run_norm, run_verify,
                              torch_dtype)

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


def check_norm_ranges(h, w, group, codes, scales, epsilon):
    """test_gpu_serving.check_norm, with the groups that hold a y past the F32 range (or of an infinite h) NaN, and
    y = 0 in the rows whose squares pass it."""
    rows, width = h.shape
    slack = ((width / 32 + 32) / 2 + 8) * U
    h, w, epsilon = host(h), host(w), float(np.float32(epsilon))
    with np.errstate(invalid="ignore", over="ignore"):
        squares = np.sum(h * h, -1, keepdims=True)
        inverse = np.where(squares < 2.0 ** 128, 1 / np.sqrt(squares / width + epsilon), 0.0)
        y = (h * inverse * w).reshape(rows, -1, group)
    bad = ~(np.abs(y) < 2.0 ** 128 * (1 - 2.0 ** -25)).all(-1)
    got_scale, got = host(scales), e4m3_table()[codes.cpu().numpy()].reshape(y.shape)
    assert np.all(np.isnan(got_scale[bad])) and np.all(np.isnan(got[bad]))
    y, got, got_scale = y[~bad], got[~bad], got_scale[~bad]
    scale = np.maximum(np.abs(y).max(-1) / 448.0, TINY)
    assert np.all(np.abs(got_scale - scale) <= slack * scale)
    q = y / scale[..., None]
    low, high = np.minimum(q * (1 - 2 * slack), q * (1 + 2 * slack)), np.maximum(q * (1 - 2 * slack), q * (1 + 2 * slack))
    assert np.all((nearest_e4m3(low) <= got) & (got <= nearest_e4m3(high)))
    return bad


# the register kernel by rows, lanes and words, in vectors and single elements, and the kernel for any width
FORMS = [(512, 512), (512, 64), (528, 48), (515, 515), (515, 5), (515, 103), (20001, 20001), (20001, 59)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width, group", FORMS)
def test_norm_y_past_the_range(m3, gpu, dtype, width, group):
    """Large weights: a y past the F32 range makes its group NaN, one at its end does not, while h * w stays small."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(width + group)
    x = (0.01 * torch.randn(5, width, generator=g, device="cuda")).to(torch_dtype(dtype))
    w = torch.ones(width, device="cuda")
    w[2 * group - 1 if 2 * group < width else width - 1] = 1e38
    x[:, 2 * group - 1 if 2 * group < width else width - 1] = torch.tensor([0.001, 0.02, 0.06, -0.08, 0.0])
    bad = check_norm_ranges(x, w, group, *run_norm(m3, x, w, group), 1e-6)
    assert bad.sum() == 2 and bad[2:4].any(-1).all()


def test_norm_scale_past_the_range(m3, gpu):
    """One element that carries its row: y / 448 itself is past the F32 range."""
    import torch

    width = 600000
    x = torch.zeros(2, width, device="cuda")
    x[0, 77] = 0.01
    x[1] = 0.01
    w = torch.full((width,), 3e38, device="cuda")
    bad = check_norm_ranges(x, w, width, *run_norm(m3, x, w, width, epsilon=1e-12), 1e-12)
    assert bad.tolist() == [[True], [False]]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width, group", FORMS)
def test_norm_squares_past_the_range(m3, gpu, dtype, width, group):
    """y = 0 in a row whose squares pass the F32 range, whatever its weights."""
    import torch

    x = torch.randn(4, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(width))
    x[0] = 2e38
    x[1, 3] = -3e38
    x = x.to(torch_dtype(dtype))
    x[3, 0] = float("inf")
    w = torch.full((width,), 4.0, device="cuda")
    codes, scales = run_norm(m3, x, w, group)
    bad = check_norm_ranges(x, w, group, codes, scales, 1e-6)
    assert bad.sum() == 1 and bad[3, 0]
    assert not bool((codes[:2] & 0x7f).any()) and np.all(host(scales[:2]) == TINY)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width, group", FORMS)
@pytest.mark.parametrize("h, weight, epsilon", [(1e16, 1e25, 1e-6), (1e-30, 1e-12, 1e-30), (1e-25, 1e-22, 1e-36)])
@pytest.mark.parametrize("residual", [None, "sum", "in place", "no sum"])
def test_norm_products_past_the_range(m3, gpu, dtype, width, group, h, weight, epsilon, residual):
    """h * w leaves the F32 range at either end, y does not; in some groups of some rows."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(width + group)
    t = torch_dtype(dtype)
    x = torch.randn(6, width, generator=g, device="cuda")
    x[::2] *= h
    x = x.to(t)
    w = torch.randn(width, generator=g, device="cuda")
    w[width // 3:] *= weight
    r = total = None
    stored = x
    if residual:
        r = (0.5 * x.float().roll(1, 1)).to(t)
        stored = (x.float() + r.float()).to(t)
        total = {"sum": torch.zeros_like(x), "in place": x.clone(), "no sum": None}[residual]
    given = total if residual == "in place" else x
    codes, scales = run_norm(m3, given, w, group, r, total, epsilon=epsilon)
    assert not check_norm_ranges(stored, w, group, codes, scales, epsilon).any()
    if total is not None:
        assert torch.equal(total, stored)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, width, group", [
    # one to eight pieces a thread of each kind, rows that share a CTA
    (2050, 1040, 1040), (2050, 4104, 4104), (5, 16384, 16384), (5, 16384, 512), (5, 16384, 8192), (5, 16376, 16376),
    (9, 516, 4), (5, 6001, 6001), (7, 256, 32), (7, 240, 24), (30, 40, 40), (30, 7, 7),
])
def test_norm_products_past_the_range_in_every_depth(m3, gpu, dtype, rows, width, group):
    """As above, with rows and groups that stay in range between those that do not, and the sum in place."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows + width)
    t = torch_dtype(dtype)
    small, weight = (2.0 ** -14, 1e-38) if dtype == "f16" else (1e-25, 1e-22)
    x = torch.randn(rows, width, generator=g, device="cuda")
    x[1::3] *= small
    x, r = x.to(t), (0.5 * x.roll(1, 1)).to(t)
    w = torch.randn(width, generator=g, device="cuda")
    w[width // 2:] *= weight
    stored = (x.float() + r.float()).to(t)
    total = x.clone()
    codes, scales = run_norm(m3, total, w, group, r, total, epsilon=1e-36)
    assert not check_norm_ranges(stored, w, group, codes, scales, 1e-36).any()
    assert torch.equal(total, stored)


def test_norm_zero_rows_with_a_small_epsilon(m3, gpu):
    import torch

    for width, group in FORMS:
        x = torch.zeros(3, width, device="cuda")
        x[1] = 1.0
        w = torch.ones(width, device="cuda")
        for epsilon in (1e-20, 1e-12):
            codes, scales = run_norm(m3, x, w, group, epsilon=epsilon)
            check_norm_ranges(x, w, group, codes, scales, epsilon)
            assert not bool((codes[::2] & 0x7f).any()) and np.all(host(scales[::2]) == TINY)


def test_norm_millions_of_elements_a_row(m3, gpu):
    """A row's squares are summed in chains of at most 256, whose sums join in 64 bits: chains and lanes are off by
    (256 + 32) / 2 steps at most, the root takes half of that, the rest is 8 steps as elsewhere."""
    import torch

    width = 4194305
    x = torch.full((1, width), 0.7, device="cuda")
    x[0, 5] = 3.0
    w = torch.ones(width, device="cuda")
    codes, scales = run_norm(m3, x, w, width)
    h = host(x)
    y = h / np.sqrt(np.mean(h * h) + 1e-6)
    slack = ((256 + 32) / 2 + 8) * U
    scale = np.abs(y).max() / 448
    assert abs(host(scales)[0, 0] - scale) <= slack * scale
    got = e4m3_table()[codes.cpu().numpy()]
    assert np.array_equal(got, nearest_e4m3(y / scale))


@pytest.mark.parametrize("dtype, drawn", [("f32", True), ("bf16", True), ("bf16", False)])
def test_verify_what_lies_behind_a_length(m3, gpu, dtype, drawn):
    """Tokens, uniforms and rows behind a sequence's drafts have no effect, whatever they hold."""
    import torch

    batch, drafts, vocabulary = 40, 37, 500
    g = torch.Generator(device="cuda").manual_seed(21)
    target = torch.softmax(2 * torch.randn(batch, drafts + 1, vocabulary, generator=g, device="cuda"), -1)
    target = target.to(torch_dtype(dtype))
    draft = target[:, :drafts].clone() if drawn else None
    drafted = target[:, :drafts].float().argmax(-1).int()
    uniforms = torch.rand(batch, drafts + 1, generator=g, device="cuda")
    uniforms[:, :drafts] *= 0.1
    lengths = (torch.arange(batch, device="cuda") % (drafts + 1)).int()
    clean = run_verify(m3, target, draft, drafted, lengths, uniforms)
    behind = torch.arange(drafts + 1, device="cuda")[None] >= lengths[:, None]
    target[behind & (torch.arange(drafts + 1, device="cuda")[None] > lengths[:, None])] = float("nan")
    drafted[behind[:, :drafts]] = -5
    uniforms[:, :drafts][behind[:, :drafts]] = 9.0
    if drawn:
        draft[behind[:, :drafts]] = float("nan")
    again = run_verify(m3, target, draft, drafted, lengths, uniforms)
    assert np.array_equal(clean[0], again[0]) and np.array_equal(clean[1], again[1])
    assert np.all(clean[1] >= 0)
    # draws from the draft model (here the target) are all accepted, given drafts as often as the target has them
    assert not drawn or clean[1].max() > 32


def test_cache_overlaps_are_refused(m3, gpu):
    """Rows that a read would write over the batch's arrays, and anything in the cache's own memory."""
    import torch

    c = m3.Cache(4, 16, 2, 64)
    ints = torch.zeros(64, dtype=torch.int32, device="cuda")
    data = torch.full((8, 2, 64), 3.0, device="cuda")
    other = torch.full((8, 2, 64), 3.0, device="cuda")
    ints[17] = 4                                    # offsets 0, 4

    def batch(**change):
        fields = dict(page_table=ints.data_ptr(), page_table_stride=2, offsets=ints.data_ptr() + 64,
                      starts=ints.data_ptr() + 128, sequences=1, rows=4)
        fields.update(change)
        return m3.CacheBatch(**fields)

    def at(pointer, token_stride=128, head_stride=64):
        return m3.CacheRows(data=pointer, dtype=m3.F32, token_stride=token_stride, head_stride=head_stride)

    fine, second = cache_rows(m3, data), cache_rows(m3, other)
    inside = data.data_ptr()
    end = inside + 4 * 128 * 4                      # of the four rows
    memory = c.pointers()
    refusals = []
    for k, name in ((0, "keys"), (1, "values")):
        pair = [second, second]
        pair[k] = fine
        for array, change in (("page table", dict(page_table=inside)), ("offsets", dict(offsets=end - 4)),
                              ("starts", dict(starts=inside + 1000)), ("page table", dict(page_table=inside - 4))):
            refusals.append((c.read, batch(**change), pair, f"cache {name} overlaps cache {array}"))
        for call in (c.write, c.read):
            pair = [second, second]
            pair[k] = at(memory[3 * k] + 256)       # the keys' codes, the values' scales
            refusals.append((call, batch(), pair, f"cache {name} overlaps the cache's memory"))
    for call in (c.write, c.read):
        for array, change in (("page table", dict(page_table=memory[0])), ("offsets", dict(offsets=memory[1])),
                              ("starts", dict(starts=memory[3]))):
            refusals.append((call, batch(**change), [fine, second], f"cache {array} overlaps the cache's memory"))
        # from below the cache into it, by the last vector
        low = at(memory[0] - 4 * (3 * 128 + 64 + 64) + 4)
        refusals.append((call, batch(), [low, second], "cache keys overlaps the cache's memory"))
        low = at(memory[0] - 4 * (3 * 64 + 512 + 64) + 4, 64, 512)
        refusals.append((call, batch(), [second, low], "cache values overlaps the cache's memory"))
    for call, b, pair, text in refusals:
        with pytest.raises(m3.M3Failure) as failure:
            call(b, *pair)
        assert failure.value.status == m3.INVALID_ARGUMENT and failure.value.message == text
    c.synchronize()
    assert bool((data == 3.0).all()) and not any(ints[18:].tolist())
    # arrays next to the rows, and between the tokens of rows that lie heads first
    c.write(batch(page_table=ints.data_ptr(), starts=None), fine, second)
    wide = torch.full((2, 8, 64), 3.0, device="cuda")
    heads_first = at(wide.data_ptr(), 64, 512)
    around = torch.full((4 * 128 + 16,), 0.0, device="cuda")
    c.write(batch(page_table=around.data_ptr() + 4 * 512), at(around.data_ptr()), second)
    c.read(batch(page_table=around.data_ptr() + 4 * 512), at(around.data_ptr()), heads_first)
    # what a write reads may be shared: zeros are a table, offsets of nothing, and numbers
    zeros = torch.zeros(8, 2, 64, device="cuda")
    c.write(batch(page_table=zeros.data_ptr(), offsets=zeros.data_ptr()), cache_rows(m3, zeros), second)
    c.synchronize()
    assert bool((wide[:, :4] != 3.0).sum() == 0) and bool((wide[:, 4:] == 3.0).all())
