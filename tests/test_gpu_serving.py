"""The serving operators on the GPU (RMS norm into E4M3, the paged E4M3 cache,
draft verification) against plain numpy forms in 64 bits.

Tolerances, with u = 2^-24 (half an F32 step):
  norm      the sum of squares is summed by at least 32 lanes, so its relative
            error is at most (width / 32 + 32) u; the inverse root takes half
            of that; the mean, the addition, the root, the two products and
            the scale's quotient round once each, all within 8 u.  A scale is
            off by `slack` = ((width / 32 + 32) / 2 + 8) u, a quotient by twice
            that, and a code is the one of a value within twice the slack.
  cache     scales and codes follow from the input by single F32 operations, so
            they are exact; so are values read back.
  verify    whole numbers: exact.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -126
NAMES = {"f32": 0, "f16": 1, "bf16": 2}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def e4m3_table():
    """The 256 values of the E4M3 codes."""
    code = np.arange(256)
    sign, exponent, significand = np.where(code & 0x80, -1.0, 1.0), (code >> 3) & 15, code & 7
    value = np.where(exponent == 0, significand * 2.0 ** -9, (8 + significand) * 2.0 ** (exponent - 10.0))
    value[(code & 0x7f) == 0x7f] = np.nan
    return sign * value


def nearest_e4m3(v):
    """The E4M3 value nearest to each v, ties to the even significand, at most 448."""
    v = np.clip(np.asarray(v, np.float64), -448.0, 448.0)
    exponent = np.clip(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -30))), -6, 8)
    exponent = np.where(2.0 ** (exponent + 1) <= np.abs(v), exponent + 1, exponent)
    step = 2.0 ** (np.clip(exponent, -6, 8) - 3)
    return np.clip(np.rint(v / step) * step, -448.0, 448.0)


def test_nearest_e4m3_is_the_tables():
    table = e4m3_table()[:0x7f]
    assert np.array_equal(nearest_e4m3(table), table)
    middle = (table[1:] + table[:-1]) / 2
    even = np.where(np.arange(126) % 2 == 0, table[:-1], table[1:])
    assert np.array_equal(nearest_e4m3(middle), even)
    assert np.array_equal(nearest_e4m3(middle * (1 + 1e-12)), table[1:])


def host(t):
    """A tensor's values in 64 bits."""
    return t.double().cpu().numpy()


def strided(t, pad, offset=0):
    """The same rows with `pad` elements between them, `offset` elements into an allocation."""
    import torch

    rows, width = t.shape
    base = torch.full((rows * (width + pad) + offset,), 7.0, dtype=t.dtype, device="cuda")
    view = base[offset:].view(rows, width + pad)[:, :width]
    view.copy_(t)
    return view


# --------------------------------------------------------------------- norm

def run_norm(m3, x, w, group, r=None, total=None, epsilon=1e-6, stream=0):
    import torch

    rows, width = x.shape
    codes = torch.full((rows * width + 64,), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows * (width // group) + 64,), -3.0, device="cuda")
    stride = lambda t: 0 if t is None else t.stride(0) if rows > 1 else width  # noqa: E731
    dtype = {torch.float32: m3.F32, torch.float16: m3.F16, torch.bfloat16: m3.BF16}
    args = m3.RmsNormE4m3Args(
        input=x.data_ptr(), residual=None if r is None else r.data_ptr(), sum=None if total is None else total.data_ptr(),
        dtype=dtype[x.dtype], input_stride=stride(x), residual_stride=stride(r), sum_stride=stride(total),
        scale=w.data_ptr(), scale_dtype=dtype[w.dtype], rows=rows, width=width, group=group, epsilon=epsilon,
        codes=codes.data_ptr(), code_scales=scales.data_ptr())
    m3.rms_norm_e4m3(args, stream=stream)
    torch.cuda.synchronize()
    # nothing behind the outputs
    assert bool((codes[rows * width:] == 0x55).all()) and bool((scales[rows * (width // group):] == -3.0).all())
    return codes[:rows * width].view(rows, width), scales[:rows * (width // group)].view(rows, -1)


def check_norm(h, w, group, codes, scales, epsilon=1e-6):
    """Codes and scales against the formula, in 64 bits, from the norm's (rounded) input."""
    rows, width = h.shape
    slack = ((width / 32 + 32) / 2 + 8) * U
    h, w = host(h), host(w)
    y = h * w / np.sqrt(np.mean(h * h, -1, keepdims=True) + epsilon)
    y = y.reshape(rows, -1, group)
    scale = np.maximum(np.abs(y).max(-1) / 448.0, TINY)
    got_scale = host(scales)
    assert np.all(np.abs(got_scale - scale) <= slack * scale)
    q = y / scale[..., None]
    got = e4m3_table()[codes.cpu().numpy()].reshape(q.shape)
    low, high = np.minimum(q * (1 - 2 * slack), q * (1 + 2 * slack)), np.maximum(q * (1 - 2 * slack), q * (1 + 2 * slack))
    assert np.all((nearest_e4m3(low) <= got) & (got <= nearest_e4m3(high)))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, width, group", [
    (1, 1, 1), (3, 7, 7), (2, 8, 8), (5, 31, 31), (4, 64, 32), (3, 96, 24), (2, 100, 4), (1, 2048, 2048),
    (300, 2048, 128), (33, 2051, 2051), (17, 2051, 7), (9, 4096, 32), (2, 4104, 8), (7, 5120, 160), (3, 8192, 8192),
    (2, 16384, 256), (2, 20000, 20000), (2, 40000, 400), (1, 40001, 40001), (1200, 256, 64), (700, 520, 520),
    # pieces of 16 and of eight elements, one to eight a thread
    (40, 528, 528), (40, 528, 16), (40, 528, 48), (3000, 1040, 1040), (2100, 8208, 8208), (5, 16384, 512),
    (2100, 4104, 4104), (3, 16376, 16376), (2500, 520, 520), (2049, 264, 264),
])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(m3, gpu, dtype, rows, width, group, residual):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows * 7919 + width)
    t = torch_dtype(dtype)
    x = torch.randn(rows, width, generator=g, device="cuda")
    x = (x * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))).to(t)
    w = torch.randn(width, generator=g, device="cuda").to(t)
    r = total = None
    h = x
    if residual:
        r = torch.randn(rows, width, generator=g, device="cuda").to(t)
        total = torch.zeros_like(x)
        h = (x.float() + r.float()).to(t)
    codes, scales = run_norm(m3, x, w, group, r, total)
    check_norm(h, w, group, codes, scales)
    if residual:
        assert torch.equal(total, h)
        again, scales2 = run_norm(m3, x, w, group, r, None)     # the sum not wanted
        assert torch.equal(again, codes) and torch.equal(scales2, scales)


@pytest.mark.parametrize("width, group", [(2048, 128), (2051, 2051), (4096, 4096), (24, 24)])
@pytest.mark.parametrize("pad, offset", [(0, 1), (8, 0), (5, 0), (64, 8), (3, 2)])
@pytest.mark.parametrize("dtype, weight", [("bf16", "f32"), ("f32", "bf16"), ("f16", "f16")])
def test_norm_strides_alignment_and_weights(m3, gpu, width, group, pad, offset, dtype, weight):
    import torch

    t = torch_dtype(dtype)
    g = torch.Generator(device="cuda").manual_seed(width + pad)
    x, r = (strided(torch.randn(21, width, generator=g, device="cuda").to(t), pad, offset) for _ in range(2))
    total = strided(torch.zeros(21, width, device="cuda", dtype=t), pad, offset)
    w = torch.randn(width + 1, generator=g, device="cuda").to(torch_dtype(weight))[offset % 2:][:width]
    h = (x.float() + r.float()).to(t)
    dense = run_norm(m3, x.contiguous(), w.clone(), group, r.contiguous(), None)
    codes, scales = run_norm(m3, x, w, group, r, total)
    check_norm(h, w, group, codes, scales)
    assert torch.equal(total, h)
    if pad:
        rest = total.as_strided((20, pad), (width + pad, 1), total.storage_offset() + width)
        assert bool((rest == 7.0).all())
    # how a tensor lies may choose another kernel, whose sums run in another order
    check_norm(h, w, group, *dense)


@pytest.mark.parametrize("width", [64, 2048, 2051, 8192])
@pytest.mark.parametrize("into", ["input", "residual"])
def test_norm_sum_in_place(m3, gpu, width, into):
    import torch

    g = torch.Generator(device="cuda").manual_seed(width)
    x, r = (torch.randn(1000, width, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(width, generator=g, device="cuda").bfloat16()
    total = torch.zeros_like(x)
    codes, scales = run_norm(m3, x, w, width, r, total)
    target = x if into == "input" else r
    codes2, scales2 = run_norm(m3, x, w, width, r, target)
    assert torch.equal(target, total) and torch.equal(codes, codes2) and torch.equal(scales, scales2)


@pytest.mark.parametrize("width, group", [(512, 512), (512, 64), (515, 515), (515, 5)])
def test_norm_special_rows(m3, gpu, width, group):
    import torch

    x = torch.randn(8, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, width - 1] = float("inf")
    x[4] *= 1e-30
    x[5] = 0.0
    x[5, 7] = -1e-20
    x[6] = -x[6].abs() * 1e15
    w = torch.ones(width, device="cuda")
    codes, scales = run_norm(m3, x, w, group)
    for row in (0, 4, 5, 6):
        check_norm(x[row:row + 1], w, group, codes[row:row + 1], scales[row:row + 1])
    value = e4m3_table()[codes.cpu().numpy()]
    assert np.all(value[1] == 0) and np.all(host(scales[1]) == TINY)
    # a NaN makes the whole row's norm NaN; an infinity makes its own element NaN and all others zero
    assert np.all(np.isnan(value[2])) and np.all(np.isnan(host(scales[2])))
    bad = (width - 1) // group
    nan = np.isnan(value[3]).reshape(-1, group)
    assert np.all(nan[bad]) and not np.any(np.delete(nan, bad, 0))
    assert np.isnan(host(scales[3])[bad]) and np.all(np.delete(host(scales[3]), bad) == TINY)
    assert np.all(codes.cpu().numpy()[2] == 0x7f)


def test_norm_small_scales(m3, gpu):
    """Scales at and near the lower bound, where v / scale needs the full division."""
    import torch

    width = 256
    x = torch.randn(64, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    w = torch.ones(width, device="cuda")
    for power in (-80, -95, -110, -118, -125, -140, -149):
        w.fill_(2.0 ** power)
        codes, scales = run_norm(m3, x, w, width)
        h = host(x)
        y32 = (h / np.sqrt(np.mean(h * h, -1, keepdims=True) + 1e-6)) * 2.0 ** power
        # an element may be a subnormal F32 number: half a step more
        scale = np.maximum(np.abs(y32).max(-1, keepdims=True) / 448.0, TINY)
        slack = ((width / 32 + 32) / 2 + 8) * U
        assert np.all(np.abs(host(scales) - scale) <= slack * scale + 2.0 ** -150 * 2)
        q, extra = y32 / scale, 2.0 ** -149 / scale
        got = e4m3_table()[codes.cpu().numpy()]
        reach = 2 * slack * np.abs(q) + extra + np.abs(q) * 2.0 ** -149 / scale
        assert np.all((nearest_e4m3(q - reach) <= got) & (got <= nearest_e4m3(q + reach)))


@pytest.mark.parametrize("width, group", [(60008, 60008), (60001, 60001), (60000, 30000), (52000, 8)])
def test_norm_rows_past_shared_memory(m3, gpu, width, group):
    import torch

    g = torch.Generator(device="cuda").manual_seed(width)
    x, r = (torch.randn(5, width, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(width, generator=g, device="cuda")
    h = (x.float() + r.float()).bfloat16()
    check_norm(h, w, group, *run_norm(m3, x, w, group, r, None))
    codes, scales = run_norm(m3, x, w, group, r, x)         # in place: read back as the sum
    assert torch.equal(x, h)
    check_norm(h, w, group, codes, scales)


@pytest.mark.parametrize("shift", [0, 1, 4, 8])
@pytest.mark.parametrize("width, group", [(256, 256), (256, 32), (2048, 256)])
def test_norm_codes_at_any_address(m3, gpu, width, group, shift):
    import torch

    x = torch.randn(9, width, device="cuda").bfloat16()
    w = torch.randn(width, device="cuda").bfloat16()
    codes = torch.full((9 * width + 32,), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(9 * (width // group) + 1, device="cuda")[1:]
    m3.rms_norm_e4m3(m3.RmsNormE4m3Args(
        input=x.data_ptr(), dtype=m3.BF16, scale=w.data_ptr(), scale_dtype=m3.BF16, rows=9, width=width, group=group,
        codes=codes.data_ptr() + shift, code_scales=scales.data_ptr()))
    torch.cuda.synchronize()
    check_norm(x, w, group, codes[shift:shift + 9 * width].view(9, width), scales.view(9, -1))
    assert bool((codes[:shift] == 0x55).all()) and bool((codes[shift + 9 * width:] == 0x55).all())


def test_norm_past_32_bit_offsets(m3, gpu):
    """More than 2^32 elements: the last rows."""
    import torch

    rows, width = 262200, 16384
    assert rows * width > 1 << 32
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, width, device="cuda").bfloat16()
    w = torch.randn(width, device="cuda").bfloat16()
    codes = torch.empty(rows, width, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, width // 128, device="cuda")
    m3.rms_norm_e4m3(m3.RmsNormE4m3Args(
        input=x.data_ptr(), dtype=m3.BF16, scale=w.data_ptr(), scale_dtype=m3.BF16, rows=rows, width=width, group=128,
        codes=codes.data_ptr(), code_scales=scales.data_ptr()))
    torch.cuda.synchronize()
    check_norm(x[-3:], w, 128, codes[-3:], scales[-3:])
    assert not bool((codes[-6:-3] & 0x7f).any()) and bool((scales[-6:-3] == TINY).all())


def test_norm_zero_rows_and_repeat(m3, gpu):
    import torch

    m3.rms_norm_e4m3(m3.RmsNormE4m3Args(rows=0, width=64, dtype=m3.F32, scale_dtype=m3.F32))
    x = torch.randn(2000, 1536, device="cuda").bfloat16()
    w = torch.randn(1536, device="cuda").bfloat16()
    first = run_norm(m3, x, w, 128)
    for _ in range(3):
        again = run_norm(m3, x, w, 128)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# -------------------------------------------------------------------- cache

class Paged:
    """A cache with random pages, a batch over it, and what it holds on the host."""

    def __init__(self, m3, rng, sequences, heads, dim, page, longest, starts=True, empty=True):
        import torch

        self.m3, self.heads, self.dim, self.page = m3, heads, dim, page
        self.lengths = rng.integers(0 if empty else 1, longest + 1, sequences)
        if sequences > 2 and empty:
            self.lengths[1] = 0
        self.starts = rng.integers(0, 3 * page + 2, sequences) if starts else np.zeros(sequences, np.int64)
        self.offsets = np.concatenate([[0], np.cumsum(self.lengths)])
        need = -(-(self.starts + self.lengths) // page)
        self.pages = int(need.sum()) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((sequences, max(1, int(need.max()))), -1, np.int64)
        for s, at in enumerate(np.cumsum(need) - need):
            self.table[s, :need[s]] = order[at:at + need[s]]
        self.cache = m3.Cache(self.pages, page, heads, dim)
        pointers = self.cache.pointers()
        shape = (self.pages * page, heads)
        self.codes = [device_view(pointers[k], shape + (dim,), "|u1") for k in (0, 2)]
        self.scales = [device_view(pointers[k], shape, "<f4") for k in (1, 3)]
        for c, s in zip(self.codes, self.scales):
            assert not bool(c.any()) and not bool(s.any())
            c.copy_(torch.from_numpy(rng.integers(0, 127, c.shape).astype(np.uint8)))
            s.copy_(torch.from_numpy(rng.uniform(0.01, 2, s.shape).astype(np.float32)))
        self.keep = []
        torch.cuda.synchronize()

    def tokens(self):
        return int(self.offsets[-1])

    def batch(self, rows=None, starts=True, **change):
        import torch

        arrays = dict(page_table=self.table, offsets=self.offsets, starts=self.starts)
        arrays.update({k: v for k, v in change.items() if k in arrays})
        held = {k: torch.from_numpy(np.ascontiguousarray(v).astype(np.int32)).cuda() for k, v in arrays.items()}
        self.keep.append(held)
        return self.m3.CacheBatch(
            page_table=held["page_table"].data_ptr(), page_table_stride=arrays["page_table"].shape[1],
            offsets=held["offsets"].data_ptr(), starts=held["starts"].data_ptr() if starts else None,
            sequences=len(arrays["offsets"]) - 1, rows=self.tokens() if rows is None else rows)

    def slots(self):
        out = np.empty(self.tokens(), np.int64)
        for s in range(len(self.lengths)):
            p = self.starts[s] + np.arange(self.lengths[s])
            out[self.offsets[s]:self.offsets[s + 1]] = self.table[s][p // self.page] * self.page + p % self.page
        return out


def device_view(pointer, shape, kind):
    import torch

    class Memory:
        __cuda_array_interface__ = {"data": (pointer, False), "shape": tuple(shape), "typestr": kind, "version": 2}

    return torch.as_tensor(Memory(), device="cuda")


def cache_rows(m3, t):
    """[rows, heads, dim] as it lies."""
    import torch

    assert t.stride(2) == 1 or t.shape[2] == 1
    dtype = {torch.float32: m3.F32, torch.float16: m3.F16, torch.bfloat16: m3.BF16}[t.dtype]
    return m3.CacheRows(data=t.data_ptr(), dtype=dtype, token_stride=t.stride(0), head_stride=t.stride(1))


def quantised(v):
    """Scales and code values by the formula's F32 operations."""
    v = v.astype(np.float32)
    scale = np.maximum(np.abs(v).max(-1) / np.float32(448), np.float32(TINY))
    return scale, nearest_e4m3(v / scale[..., None])


def laid_out(t, layout):
    """[rows, heads, dim] values in several memory layouts."""
    import torch

    rows, heads, dim = t.shape
    if layout == "fused":      # the columns of a wider projection
        wide = torch.full((rows, 3 * heads, dim), 5.0, dtype=t.dtype, device="cuda")
        view = wide[:, heads:2 * heads]
    elif layout == "heads first":
        wide = torch.full((heads, rows + 3, dim), 5.0, dtype=t.dtype, device="cuda")
        view = wide[:, :rows].transpose(0, 1)
    elif layout == "sixteen":  # aligned to 16 bytes, not to 32
        shift = 16 // t.element_size()
        wide = torch.full((rows * heads * dim + shift,), 5.0, dtype=t.dtype, device="cuda")
        view = wide[shift:].view(rows, heads, dim)
    elif layout == "odd":      # nothing aligned to a vector
        wide = torch.full((rows * (heads * (dim + 1) + 3) + 1,), 5.0, dtype=t.dtype, device="cuda")
        view = wide[1:].as_strided((rows, heads, dim), (heads * (dim + 1) + 3, dim + 1, 1), 1)
    else:
        view = torch.empty_like(t)
    view.copy_(t)
    return view


SHAPES = [
    (1, 1, 1, 1, 5), (2, 3, 8, 3, 40), (7, 5, 80, 48, 90), (3, 8, 128, 16, 70), (33, 2, 64, 16, 9), (70, 1, 128, 64, 4),
    (1, 4, 256, 16, 100), (2, 2, 257, 7, 20), (2, 1, 320, 16, 33), (5, 3, 60, 1, 12), (3, 16, 192, 100, 30),
    (1, 8, 128, 16, 1), (1, 1, 8, 16, 1000), (2, 3, 1032, 4, 9), (300, 2, 16, 8, 3), (3, 2, 576, 16, 30),
    (2, 1, 768, 16, 20), (2, 1, 776, 16, 20), (2, 3, 72, 16, 30), (1, 2, 24, 8, 20), (4, 4, 128, 16, 25),
    (3, 8, 128, 15, 25), (3, 8, 128, 17, 25), (3, 8, 128, 18, 25), (2, 2, 96, 16, 25), (2, 2, 112, 16, 25),
    (2, 2, 48, 16, 25), (1500, 1, 8, 16, 2), (2, 20, 256, 32, 40),
]


@pytest.mark.parametrize("dtypes", [("bf16", "bf16"), ("f16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("sequences, heads, dim, page, longest", SHAPES)
def test_cache_write_and_read(m3, gpu, dtypes, sequences, heads, dim, page, longest):
    import torch

    rng = np.random.default_rng(sequences * 1000 + dim)
    c = Paged(m3, rng, sequences, heads, dim, page, longest, empty=sequences > 1)
    tokens, slots = c.tokens(), c.slots()
    before = [(a.cpu().numpy().copy(), b.cpu().numpy().copy()) for a, b in zip(c.codes, c.scales)]
    layouts = [("dense", "fused"), ("heads first", "odd"), ("fused", "fused"), ("sixteen", "dense")][
        (sequences + dim + page) % 4]
    rows = []
    for name, layout in zip(dtypes, layouts):
        v = rng.normal(size=(tokens, heads, dim)) * np.exp(2 * rng.normal(size=(tokens, heads, 1)))
        rows.append(laid_out(torch.from_numpy(v).to(torch_dtype(name)).cuda(), layout))
    c.cache.write(c.batch(), cache_rows(m3, rows[0]), cache_rows(m3, rows[1]))
    c.cache.synchronize()
    others = np.setdiff1d(np.arange(c.pages * page), slots)
    for k in range(2):
        scale, value = quantised(host(rows[k]))
        got_codes, got_scales = c.codes[k].cpu().numpy(), c.scales[k].cpu().numpy()
        assert np.array_equal(got_scales[slots], scale)
        assert np.array_equal(e4m3_table()[got_codes[slots]], value)
        assert np.array_equal(got_codes[others], before[k][0][others])
        assert np.array_equal(got_scales[others], before[k][1][others])
    # and back, into the other layouts and types
    outs = [laid_out(torch.full((tokens + 2, heads, dim), 9.0, dtype=torch_dtype(n), device="cuda"), l)
            for n, l in zip(dtypes[::-1], layouts[::-1])]
    c.cache.read(c.batch(rows=tokens + 2), cache_rows(m3, outs[0]), cache_rows(m3, outs[1]))
    c.cache.synchronize()
    for k in range(2):
        value = e4m3_table()[c.codes[k].cpu().numpy()[slots]].astype(np.float32)
        want = torch.from_numpy(value * c.scales[k].cpu().numpy()[slots][..., None]).to(outs[k].dtype)
        assert torch.equal(outs[k][:tokens].cpu(), want)
        assert bool((outs[k][tokens:] == 9.0).all())      # behind the last sequence


@pytest.mark.parametrize("heads, dim, page", [(8, 128, 16), (3, 60, 7), (2, 264, 16)])
def test_cache_special_vectors(m3, gpu, heads, dim, page):
    import torch

    rng = np.random.default_rng(5)
    c = Paged(m3, rng, 1, heads, dim, page, 40, empty=False)
    tokens, slots = c.tokens(), c.slots()
    v = rng.normal(size=(tokens, heads, dim)).astype(np.float32)
    v[0, 0] = 0.0
    v[0, 1, dim - 1] = np.nan
    v[min(1, tokens - 1), 0, 3] = np.inf
    v[tokens - 1, heads - 1] *= np.float32(1e-37)
    v[tokens - 1, 0] *= np.float32(1e-42)
    v[tokens // 2, 1] *= np.float32(1e37)
    rows = torch.from_numpy(v).cuda()
    c.cache.write(c.batch(), cache_rows(m3, rows), cache_rows(m3, rows))
    out = torch.zeros(2, tokens, heads, dim, device="cuda")
    c.cache.read(c.batch(), cache_rows(m3, out[0]), cache_rows(m3, out[1]))
    c.cache.synchronize()
    bad = ~np.isfinite(v).all(-1)
    scales, codes = c.scales[0].cpu().numpy()[slots], c.codes[0].cpu().numpy()[slots]
    assert np.all(np.isnan(scales[bad])) and np.all(codes[bad] & 0x7f == 0x7f)
    assert np.all(np.isnan(out[0].cpu().numpy()[bad]))
    scale, value = quantised(v[~bad])
    assert np.array_equal(scales[~bad], scale)
    assert np.array_equal(e4m3_table()[codes[~bad]], value)
    # back: code * scale rounds once
    assert np.array_equal(out[1].cpu().numpy()[~bad], value.astype(np.float32) * scale[..., None])


def test_cache_bf16_ties(m3, gpu):
    """Quotients that are E4M3 ties: every pair of bf16 significands."""
    import torch

    m = (np.arange(128, 256) / 128.0).astype(np.float32)
    v = np.zeros((128, 1, 136), np.float32)
    v[:, 0, 0] = 2 * m                       # the largest of each vector
    v[:, 0, 1:129] = m / 2 * np.where(np.arange(128) % 2, -1, 1)
    for dim in (136, 129):
        c = m3.Cache(16, 8, 1, dim)
        rows = torch.from_numpy(v[:, :, :dim].copy()).bfloat16().cuda()
        table = torch.arange(16, dtype=torch.int32, device="cuda")
        offsets = torch.tensor([0, 128], dtype=torch.int32, device="cuda")
        batch = m3.CacheBatch(page_table=table.data_ptr(), page_table_stride=16, offsets=offsets.data_ptr(),
                              starts=None, sequences=1, rows=128)
        c.write(batch, cache_rows(m3, rows), cache_rows(m3, rows))
        c.synchronize()
        scale, value = quantised(host(rows))
        got = device_view(c.pointers()[0], (128, 1, dim), "|u1").cpu().numpy()
        assert np.array_equal(e4m3_table()[got], value)
        assert np.array_equal(device_view(c.pointers()[3], (128, 1), "<f4").cpu().numpy(), scale)


@pytest.mark.parametrize("heads, dim, page", [(8, 128, 16), (3, 60, 7)])
def test_cache_skips_bad_rows(m3, gpu, heads, dim, page):
    import torch

    rng = np.random.default_rng(9)
    c = Paged(m3, rng, 4, heads, dim, page, 50, empty=False)
    tokens, slots = c.tokens(), c.slots()
    rows = torch.randn(tokens, heads, dim, device="cuda")
    out = torch.full((2, tokens, heads, dim), 4.0, device="cuda")
    arguments = cache_rows(m3, rows), cache_rows(m3, rows)
    outs = cache_rows(m3, out[0]), cache_rows(m3, out[1])

    def row_of(sequence):
        return int(c.offsets[sequence])

    table = c.table.copy()
    first = int(c.starts[2]) // page
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        table[2, first] = bad
        good = np.ones(tokens, bool)
        at = c.starts[2] + np.arange(c.lengths[2])
        good[c.offsets[2]:c.offsets[3]] = at // page != first
        for codes in c.codes:
            codes.fill_(0x11)
        for call, where in ((c.cache.write, arguments), (c.cache.read, outs)):
            out.fill_(4.0)
            call(c.batch(page_table=table), *where)
            with pytest.raises(m3.M3Failure) as failure:
                c.cache.synchronize()
            assert failure.value.status == m3.OUT_OF_RANGE
            assert f"row {row_of(2)} was skipped: its page is outside the cache" in failure.value.message
            c.cache.synchronize()             # reported once
        scale, value = quantised(host(rows))
        got = c.codes[0].cpu().numpy()
        assert np.array_equal(e4m3_table()[got[slots[good]]], value[good])
        assert np.all(got[slots[~good]] == 0x11)
        assert bool((out[:, torch.from_numpy(~good)] == 4.0).all())
        assert not bool((out[:, torch.from_numpy(good)] == 4.0).all(-1).any())
    # positions before the first token and behind the table
    starts = c.starts.copy()
    starts[3] = c.table.shape[1] * page
    c.cache.write(c.batch(starts=True, **{"page_table": c.table}), *arguments)
    c.cache.synchronize()
    for start in (c.table.shape[1] * page, 2 ** 31 - 1, -1, -2 ** 31):
        starts[3] = start
        held = torch.from_numpy(starts.astype(np.int32)).cuda()
        batch = c.batch()
        batch.starts = held.data_ptr()
        before = c.codes[0].clone()
        c.cache.write(batch, *arguments)
        with pytest.raises(m3.M3Failure) as failure:
            c.cache.synchronize()
        assert f"row {row_of(3)} was skipped: its position is outside the page table" in failure.value.message
        if start >= 0:
            assert torch.equal(before, c.codes[0])


def test_cache_rows_outside_the_sequences(m3, gpu):
    """Rows before the first offset, behind the last and behind `rows`; offsets that do not increase."""
    import torch

    rng = np.random.default_rng(11)
    c = Paged(m3, rng, 3, 2, 64, 8, 30, empty=False)
    tokens = c.tokens()
    rows = torch.randn(tokens + 20, 2, 64, device="cuda").bfloat16()
    for offsets, live in ((c.offsets + 5, range(5, tokens + 5)), (c.offsets, range(tokens))):
        out = torch.full((2, tokens + 20, 2, 64), 4.0, device="cuda")
        c.cache.write(c.batch(rows=tokens + 20, offsets=offsets), cache_rows(m3, rows), cache_rows(m3, rows))
        c.cache.read(c.batch(rows=tokens + 20, offsets=offsets), cache_rows(m3, out[0]), cache_rows(m3, out[1]))
        c.cache.synchronize()
        touched = (out != 4.0).any(-1).any(-1).cpu().numpy()
        assert np.array_equal(np.nonzero(touched[0])[0], np.array(live))
        assert np.array_equal(touched[0], touched[1])
    out = torch.full((2, tokens, 2, 64), 4.0, device="cuda")
    c.cache.read(c.batch(rows=7), cache_rows(m3, out[0]), cache_rows(m3, out[1]))
    c.cache.synchronize()
    assert not bool((out[:, :7] == 4.0).all(-1).any()) and bool((out[:, 7:] == 4.0).all())
    # no rows, no sequences
    empty = m3.CacheRows(dtype=m3.F32)
    c.cache.write(c.batch(rows=0), empty, empty)
    c.cache.read(m3.CacheBatch(rows=5, sequences=0), cache_rows(m3, out[0]), cache_rows(m3, out[1]))
    # offsets out of order name no slot outside the cache, whatever rows they give
    c.cache.write(c.batch(offsets=c.offsets[::-1].copy()), cache_rows(m3, rows), cache_rows(m3, rows))
    try:
        c.cache.synchronize()
    except m3.M3Failure as failure:
        assert failure.status == m3.OUT_OF_RANGE


def test_cache_large_batches(m3, gpu):
    """Enough rows that a CTA walks over many, the last of them few; mostly empty sequences."""
    import torch

    for heads, dim, page, tokens in ((8, 128, 64, 20011), (1, 8, 16, 100003), (5, 80, 48, 9001)):
        sequences = 1000
        rng = np.random.default_rng(dim)
        c = m3.Cache(tokens // page + sequences + 1, page, heads, dim)
        cuts = np.sort(rng.integers(0, tokens, sequences - 1))
        cuts[100:400] = cuts[100]
        cuts = np.sort(cuts)
        offsets = np.concatenate([[0], cuts, [tokens]])
        need = -(-np.diff(offsets) // page)
        order = rng.permutation(tokens // page + sequences + 1)
        table = np.full((sequences, int(need.max())), -1)
        slots = np.empty(tokens, np.int64)
        for s, at in enumerate(np.cumsum(need) - need):
            table[s, :need[s]] = order[at:at + need[s]]
            p = np.arange(offsets[s + 1] - offsets[s])
            slots[offsets[s]:offsets[s + 1]] = table[s][p // page] * page + p % page
        held = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (table, offsets)]
        batch = m3.CacheBatch(page_table=held[0].data_ptr(), page_table_stride=table.shape[1],
                              offsets=held[1].data_ptr(), starts=None, sequences=sequences, rows=tokens)
        rows = torch.randn(2, tokens, heads, dim, device="cuda").bfloat16()
        out = torch.zeros_like(rows)
        c.write(batch, cache_rows(m3, rows[0]), cache_rows(m3, rows[1]))
        c.read(batch, cache_rows(m3, out[0]), cache_rows(m3, out[1]))
        c.synchronize()
        for k in range(2):
            v = rows[k].float()
            scale = (v.abs().amax(-1) / 448).clamp_min(TINY)
            # one place in a thousand is checked for its bits, all for their range
            places = rng.integers(0, tokens, 64)
            want_scale, value = quantised(host(rows[k][torch.from_numpy(places)]))
            got = device_view(c.pointers()[2 * k], (c.shape[0] * page, heads, dim), "|u1")
            at = torch.from_numpy(slots[places]).cuda()
            assert np.array_equal(e4m3_table()[got[at].cpu().numpy()], value)
            want = torch.from_numpy(value.astype(np.float32) * want_scale[..., None]).bfloat16()
            assert torch.equal(out[k][torch.from_numpy(places)].cpu(), want)
            # half a step of the largest binade, 16, and the value's own rounding to bf16
            assert bool(((out[k].float() - v).abs() <= scale[..., None] * (16 + 448 * 2 ** -8 + 1e-3)).all())


def test_cache_shared_prefix_and_one_slot_twice(m3, gpu):
    """A page read by several sequences; a slot written twice disturbs no other."""
    import torch

    c = m3.Cache(8, 16, 2, 128)
    rows = torch.randn(32, 2, 128, device="cuda")
    offsets = torch.tensor([0, 16, 32], dtype=torch.int32, device="cuda")
    table = torch.tensor([[3], [3]], dtype=torch.int32, device="cuda")
    batch = m3.CacheBatch(page_table=table.data_ptr(), page_table_stride=1, offsets=offsets.data_ptr(), starts=None,
                          sequences=2, rows=32)
    half = m3.CacheBatch(page_table=table.data_ptr(), page_table_stride=1, offsets=offsets.data_ptr(), starts=None,
                         sequences=1, rows=32)
    c.write(half, cache_rows(m3, rows), cache_rows(m3, rows))
    out = torch.zeros(2, 32, 2, 128, device="cuda")
    c.read(batch, cache_rows(m3, out[0]), cache_rows(m3, out[1]))
    c.synchronize()
    assert torch.equal(out[0, :16], out[0, 16:]) and torch.equal(out[0], out[1])
    c.write(batch, cache_rows(m3, rows), cache_rows(m3, rows))
    c.synchronize()
    codes = device_view(c.pointers()[0], (8, 16, 2, 128), "|u1")
    assert not bool(codes[[0, 1, 2, 4, 5, 6, 7]].any())


def test_cache_refusals_with_a_cache(m3, gpu):
    import torch

    c = m3.Cache(4, 16, 2, 64)
    data = torch.zeros(4, 2, 64, device="cuda")
    ints = torch.zeros(16, dtype=torch.int32, device="cuda")
    fine = cache_rows(m3, data)

    def batch(**change):
        fields = dict(page_table=ints.data_ptr(), page_table_stride=1, offsets=ints.data_ptr(), starts=None,
                      sequences=1, rows=4)
        fields.update(change)
        return m3.CacheBatch(**fields)

    def rows(**change):
        fields = dict(data=data.data_ptr(), dtype=m3.F32, token_stride=128, head_stride=64)
        fields.update(change)
        return m3.CacheRows(**fields)

    for b, k, v, status, text in (
            (batch(rows=1 << 31), fine, fine, m3.OUT_OF_RANGE, "too many rows"),
            (batch(sequences=1 << 31), fine, fine, m3.OUT_OF_RANGE, "too many rows"),
            (batch(page_table_stride=1 << 31), fine, fine, m3.OUT_OF_RANGE, "too many rows"),
            (batch(page_table=None), fine, fine, m3.INVALID_ARGUMENT, "cache page table is absent"),
            (batch(offsets=None), fine, fine, m3.INVALID_ARGUMENT, "cache offsets is absent"),
            (batch(starts=ints.data_ptr() + 2), fine, fine, m3.INVALID_ARGUMENT, "cache starts is absent or not aligned"),
            (batch(), rows(data=None), fine, m3.INVALID_ARGUMENT, "cache keys is required"),
            (batch(), fine, rows(data=None), m3.INVALID_ARGUMENT, "cache values is required"),
            (batch(), rows(dtype=m3.I32), fine, m3.INVALID_ARGUMENT, "cache keys must be F32, F16 or BF16"),
            (batch(), rows(data=data.data_ptr() + 2), fine, m3.INVALID_ARGUMENT, "cache keys is not aligned"),
            (batch(), rows(head_stride=63), fine, m3.INVALID_ARGUMENT, "cache keys stride is less"),
            (batch(), rows(token_stride=63), fine, m3.INVALID_ARGUMENT, "cache keys stride is less"),
            (batch(), rows(token_stride=1 << 60), fine, m3.OVERFLOW, "overflows")):
        for call in (c.write, c.read):
            with pytest.raises(m3.M3Failure) as failure:
                call(b, k, v)
            assert failure.value.status == status and text in failure.value.message
    with pytest.raises(m3.M3Failure):
        m3.Cache(4, 16, 2, 64, device=99)
    c.synchronize()


def test_cache_past_32_bit_offsets(m3, gpu):
    """Slots whose byte offsets pass 2^32 (a cache of 9 GB)."""
    import torch

    pages, page, heads, dim = 4200, 64, 16, 1024
    c = m3.Cache(pages, page, heads, dim)
    assert pages * page * heads * dim > 1 << 32
    rows = torch.randn(130, heads, dim, device="cuda").bfloat16()
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 130], dtype=torch.int32, device="cuda")
    batch = m3.CacheBatch(page_table=table.data_ptr(), page_table_stride=3, offsets=offsets.data_ptr(), starts=None,
                          sequences=1, rows=130)
    c.write(batch, cache_rows(m3, rows), cache_rows(m3, rows))
    out = torch.zeros(2, 130, heads, dim, device="cuda")
    c.read(batch, cache_rows(m3, out[0]), cache_rows(m3, out[1]))
    c.synchronize()
    scale, value = quantised(host(rows))
    assert np.array_equal(out[1].cpu().numpy(), value.astype(np.float32) * scale[..., None])
    codes = device_view(c.pointers()[2], (pages * page, heads, dim), "|u1")
    assert np.array_equal(e4m3_table()[codes[(pages - 2) * page:][:2].cpu().numpy()], value[128:])


# ------------------------------------------------------------------- verify

def verify_host(target, draft, drafted, lengths, uniforms):
    """The rule, sequence by sequence, in 64 bits."""
    batch, places, vocabulary = target.shape
    drafts = places - 1
    tokens, accepted = np.full((batch, places), -1, np.int64), np.full(batch, -1, np.int64)
    fine = lambda a: bool(np.all((a >= 0) & np.isfinite(a)))  # noqa: E731
    unit = lambda u: 0 <= u < 1  # noqa: E731
    for b in range(batch):
        length = drafts if lengths is None else lengths[b]
        if not 0 <= length <= drafts or not unit(uniforms[b, drafts]):
            continue
        m, bad = 0, False
        while m < length:
            d = drafted[b, m]
            if not 0 <= d < vocabulary or not unit(uniforms[b, m]):
                bad = True
                break
            t, q = target[b, m, d], 1.0 if draft is None else draft[b, m, d]
            if not fine(t) or not fine(q):
                bad = True
                break
            if not uniforms[b, m] * q < t:
                break
            m += 1
        if bad:
            continue
        w = target[b, m]
        if not fine(w):
            continue
        if m < length:
            if draft is None:
                w = w.copy()
                w[drafted[b, m]] = 0
            else:
                if not fine(draft[b, m]):
                    continue
                w = np.maximum(w - draft[b, m], 0)
            if not w.any():
                w = target[b, m]
        if not w.any():
            continue
        sums = np.cumsum(w)
        j = np.searchsorted(sums, uniforms[b, drafts] * sums[-1], side="right")
        tokens[b, :m], tokens[b, m], accepted[b] = drafted[b, :m], j, m
    return tokens, accepted


def run_verify(m3, target, draft, drafted, lengths, uniforms, stream=0):
    """Tensors in; target and draft may have row strides."""
    import torch

    batch, places, vocabulary = target.shape
    dtype = {torch.float32: m3.F32, torch.float16: m3.F16, torch.bfloat16: m3.BF16}[target.dtype]
    tokens = torch.full((batch + 1, places), -7, dtype=torch.int32, device="cuda")
    accepted = torch.full((batch + 1,), -7, dtype=torch.int32, device="cuda")
    m3.verify_draft(m3.VerifyDraftArgs(
        target=target.data_ptr(), draft=None if draft is None else draft.data_ptr(), dtype=dtype,
        target_stride=target.stride(1), draft_stride=0 if draft is None or places == 1 else draft.stride(1),
        draft_tokens=drafted.data_ptr(), lengths=None if lengths is None else lengths.data_ptr(),
        uniforms=uniforms.data_ptr(), batch=batch, drafts=places - 1, vocabulary=vocabulary, tokens=tokens.data_ptr(),
        accepted=accepted.data_ptr()), stream=stream)
    torch.cuda.synchronize()
    assert bool((tokens[batch] == -7).all()) and int(accepted[batch]) == -7
    return tokens[:batch].cpu().numpy(), accepted[:batch].cpu().numpy()


def check_verify(m3, target, draft, drafted, lengths, uniforms):
    got = run_verify(m3, target, draft, drafted, lengths, uniforms)
    want = verify_host(host(target), None if draft is None else host(draft), drafted.cpu().numpy(),
                       None if lengths is None else lengths.cpu().numpy(), host(uniforms))
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])
    return got


def padded_rows(t, pad):
    import torch

    wide = torch.full(t.shape[:2] + (t.shape[2] + pad,), float("nan"), dtype=t.dtype, device="cuda")
    wide[..., :t.shape[2]] = t
    return wide[..., :t.shape[2]]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("batch, drafts, vocabulary, pad", [
    (1, 1, 1, 0), (1, 4, 2, 0), (3, 2, 7, 3), (5, 33, 100, 0), (2, 70, 64, 0), (40, 5, 1000, 24), (1, 4, 32000, 0),
    (9, 3, 50257, 0), (2, 1, 50257, 7), (300, 2, 257, 0), (24, 7, 4096, 0), (1, 0, 5000, 0), (3, 8, 131072, 0),
    (2, 2, 262151, 1), (150, 3, 8192, 0),
])
def test_verify(m3, gpu, dtype, drawn, batch, drafts, vocabulary, pad):
    import torch

    g = torch.Generator(device="cuda").manual_seed(batch * 31 + vocabulary)
    t = torch_dtype(dtype)
    logits = 2 * torch.randn(batch, drafts + 1, vocabulary, generator=g, device="cuda")
    target = padded_rows(torch.softmax(logits, -1).to(t), pad)
    logits = logits[:, :drafts] + 0.5 * torch.randn(batch, drafts, vocabulary, generator=g, device="cuda")
    draft = padded_rows(torch.softmax(logits, -1).to(t), pad) if drawn else None
    noise = torch.rand(batch, drafts, vocabulary, generator=g, device="cuda").clamp_min(1e-20)
    drafted = (logits - torch.log(-torch.log(noise))).argmax(-1).int() if drafts else torch.zeros(
        batch, 0, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(batch, drafts + 1, generator=g, device="cuda")
    check_verify(m3, target, draft, drafted, None, uniforms)
    # padded places among the lengths
    lengths = torch.randint(-1, drafts + 2, (batch,), generator=g, device="cuda", dtype=torch.int32)
    _, accepted = check_verify(m3, target, draft, drafted, lengths, uniforms)
    length = lengths.cpu().numpy()
    assert np.array_equal(accepted < 0, (length < 0) | (length > drafts))


def test_verify_borders(m3, gpu):
    """Dyadic probabilities: running sums, products and comparisons that are exact, with equality."""
    import torch

    vocabulary = 4096
    target = torch.zeros(4, 2, vocabulary, device="cuda")
    draft = torch.zeros(4, 1, vocabulary, device="cuda")
    target[:, 0, 5] = 0.25
    target[:, 0, 9] = 0.75
    draft[:, 0, 5] = 0.5
    draft[:, 0, 4000] = 0.5
    target[:, 1, ::4] = 1.0 / 1024
    drafted = torch.full((4, 1), 5, dtype=torch.int32, device="cuda")
    # u q < p: 0.5 * 0.5 is not less than 0.25, the next number below is
    first = torch.tensor([0.5, float(np.nextafter(np.float32(0.5), np.float32(0))), 0.499, 0.75])
    last = torch.tensor([0.0, 0.0, 0.25, 0.999])
    uniforms = torch.stack([first, last], -1).cuda().contiguous()
    tokens, accepted = check_verify(m3, target, draft, drafted, None, uniforms)
    assert accepted.tolist() == [0, 1, 1, 0]
    # a draw at exactly a running sum belongs to the next token: 256 of 1024 are passed
    assert tokens[1].tolist() == [5, 0] and tokens[2].tolist() == [5, 4 * 256] and tokens[0].tolist() == [9, -1]


@pytest.mark.parametrize("vocabulary", [3, 1024, 5000, 131072])
def test_verify_every_border(m3, gpu, vocabulary):
    """One sequence per border of a running sum of equal weights, on it and just below it."""
    import torch

    count = 64
    at = np.unique(np.linspace(1, vocabulary - 1, count).astype(int))
    weight = 2.0 ** -18
    target = torch.full((1, 1, vocabulary), weight, device="cuda").expand(2 * len(at), 1, vocabulary).contiguous()
    total = vocabulary * weight
    on = (at * weight / total).astype(np.float32)
    uniforms = torch.from_numpy(np.concatenate([on, np.nextafter(on, np.float32(0))]))[:, None].cuda().contiguous()
    drafted = torch.zeros(2 * len(at), 0, dtype=torch.int32, device="cuda")
    check_verify(m3, target, None, drafted, None, uniforms)


def test_verify_residual_of_nothing(m3, gpu):
    """target <= draft everywhere and a rejection: the target itself is drawn from."""
    import torch

    target = torch.zeros(3, 2, 600, device="cuda")
    target[:, 0, 100] = 0.25
    target[:, 0, 400] = 0.25
    draft = target[:, :1].clone() * 2
    drafted = torch.full((3, 1), 100, dtype=torch.int32, device="cuda")
    target[:, 1, 7] = 1.0
    uniforms = torch.tensor([[0.9, 0.2], [0.9, 0.7], [0.1, 0.5]], device="cuda")
    tokens, accepted = check_verify(m3, target, draft, drafted, None, uniforms)
    assert tokens.tolist() == [[100, -1], [400, -1], [100, 7]] and accepted.tolist() == [0, 0, 1]
    # given drafts: a target that is certain of the rejected token
    target[:, 0] = 0
    target[:, 0, 100] = 0.5
    tokens, _ = check_verify(m3, target, None, drafted, None, uniforms)
    assert tokens.tolist() == [[100, -1], [100, -1], [100, 7]]


def test_verify_bad_sequences_stay_alone(m3, gpu):
    import torch

    batch, drafts, vocabulary = 24, 3, 2000
    g = torch.Generator(device="cuda").manual_seed(4)
    target = torch.softmax(torch.randn(batch, drafts + 1, vocabulary, generator=g, device="cuda"), -1)
    draft = target[:, :drafts].clone()                      # everything is accepted
    drafted = torch.randint(0, vocabulary, (batch, drafts), generator=g, device="cuda", dtype=torch.int32)
    uniforms = torch.rand(batch, drafts + 1, generator=g, device="cuda")
    drafted[1, 0] = -1
    drafted[2, 2] = vocabulary
    drafted[3, 1] = 2 ** 31 - 1
    uniforms[4, 1] = 1.0
    uniforms[5, 3] = -0.25
    uniforms[6, 0] = float("nan")
    target[7, 3, 1999] = float("nan")
    target[8, 3, 0] = -0.1
    target[9, 3, 1000] = float("inf")
    target[10, 3] = 0.0
    target[11, 1, drafted[11, 1].item()] = float("nan")
    draft[12, 0, drafted[12, 0].item()] = -1.0
    target[13, 1, drafted[13, 1].item()] = 0.0              # a rejection at 1 ...
    draft[13, 1, 77] = float("inf")                         # ... whose draft row is bad
    # what is not needed is not looked at: behind a rejection, and rows never drawn from
    target[14, 0, drafted[14, 0].item()] = 0.0
    drafted[14, 1:] = -5
    target[14, 3] = float("nan")
    uniforms[14, 1:3] = 9.0
    target[15, 1, (drafted[15, 1].item() + 1) % vocabulary] = float("nan")
    target[16, 3, 5] = -0.0                                 # a zero
    tokens, accepted = check_verify(m3, target, draft, drafted, None, uniforms)
    assert np.all(accepted[1:14] == -1) and np.all(tokens[1:14] == -1)
    assert accepted[14] == 0 and np.all(np.delete(accepted, range(1, 15)) == drafts)
    # a length that leaves the bad draft out
    lengths = torch.full((batch,), drafts, dtype=torch.int32, device="cuda")
    lengths[2] = 2
    _, accepted = check_verify(m3, target, draft, drafted, lengths, uniforms)
    assert accepted[2] == 2
    m3.verify_draft(m3.VerifyDraftArgs(batch=0, vocabulary=5))


def test_verify_past_32_bit_offsets(m3, gpu):
    """Rows of probabilities past 2^32 elements."""
    import torch

    batch, vocabulary = 16500, 131080
    target = torch.zeros(batch, 2, vocabulary, dtype=torch.float16, device="cuda")
    assert target.numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(6)
    target[-4:] = torch.softmax(torch.randn(4, 2, vocabulary, generator=g, device="cuda"), -1).half()
    target[:-4, :, 77] = 1.0
    drafted = torch.full((batch, 1), 77, dtype=torch.int32, device="cuda")
    uniforms = torch.rand(batch, 2, generator=g, device="cuda")
    uniforms[-2:, 0] = 0.0
    tokens, accepted = run_verify(m3, target, None, drafted, None, uniforms)
    want = verify_host(host(target[-4:]), None, drafted[-4:].cpu().numpy(), None, host(uniforms[-4:]))
    assert np.array_equal(tokens[-4:], want[0]) and np.array_equal(accepted[-4:], want[1])
    assert np.all(tokens[:-4] == 77) and np.all(accepted[:-4] == 1)


def test_verify_distribution(m3, gpu):
    """The first token's frequencies are the target's, whatever the draft model."""
    import torch

    batch, vocabulary = 200000, 8
    target = torch.tensor([0.3, 0.02, 0.18, 0.0, 0.1, 0.25, 0.05, 0.1], device="cuda")
    draft = torch.tensor([0.05, 0.3, 0.1, 0.2, 0.1, 0.05, 0.15, 0.05], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    drafted = torch.multinomial(draft, batch, replacement=True, generator=g).int()[:, None].contiguous()
    uniforms = torch.rand(batch, 2, generator=g, device="cuda")
    tokens, _ = run_verify(m3, target.expand(batch, 2, vocabulary).contiguous(),
                           draft.expand(batch, 1, vocabulary).contiguous(), drafted, None, uniforms)
    share = np.bincount(tokens[:, 0], minlength=vocabulary) / batch
    want = host(target)
    # six standard deviations of a share
    assert np.all(np.abs(share - want) <= 6 * np.sqrt(want * (1 - want) / batch))


# ----------------------------------------------------- streams and captures

def step_state(m3, seed, rows=64, width=1024, heads=8, dim=128, vocabulary=5000):
    """The buffers of one served step: 4 sequences of 16 tokens, 3 drafts each."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"x": normal(rows, width).bfloat16(), "r": normal(rows, width).bfloat16(), "w": normal(width).bfloat16(),
         "sum": torch.zeros(rows, width, device="cuda").bfloat16(),
         "codes": torch.zeros(rows, width, dtype=torch.uint8, device="cuda"),
         "scales": torch.zeros(rows, width // 128, device="cuda"),
         "weights": (normal(width, 2 * heads * dim) / 32),
         "kv": torch.zeros(rows, 2 * heads, dim, device="cuda"),
         "back": torch.zeros(2, rows, heads, dim, device="cuda").bfloat16(),
         "head": normal(2 * heads * dim, vocabulary) / 16,
         "target": torch.zeros(4, 4, vocabulary, device="cuda"),
         "drafted": torch.randint(0, vocabulary, (4, 3), generator=g, device="cuda", dtype=torch.int32),
         "uniforms": torch.rand(4, 4, generator=g, device="cuda"),
         "tokens": torch.zeros(4, 4, dtype=torch.int32, device="cuda"),
         "accepted": torch.zeros(4, dtype=torch.int32, device="cuda"),
         "offsets": torch.arange(0, 65, 16, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor([0, 5, 16, 40], dtype=torch.int32, device="cuda"),
         "table": torch.randperm(20, generator=g, device="cuda").int()[:16].view(4, 4).contiguous()}
    s["cache"] = m3.Cache(20, 16, heads, dim)
    s["norm"] = m3.RmsNormE4m3Args(
        input=s["x"].data_ptr(), residual=s["r"].data_ptr(), sum=s["sum"].data_ptr(), dtype=m3.BF16,
        scale=s["w"].data_ptr(), scale_dtype=m3.BF16, rows=rows, width=width, group=128, codes=s["codes"].data_ptr(),
        code_scales=s["scales"].data_ptr())
    s["batch"] = m3.CacheBatch(page_table=s["table"].data_ptr(), page_table_stride=4, offsets=s["offsets"].data_ptr(),
                               starts=s["starts"].data_ptr(), sequences=4, rows=rows)
    s["keys"], s["values"] = cache_rows(m3, s["kv"][:, :heads]), cache_rows(m3, s["kv"][:, heads:])
    s["outs"] = [cache_rows(m3, s["back"][0]), cache_rows(m3, s["back"][1])]
    s["verify"] = m3.VerifyDraftArgs(
        target=s["target"].data_ptr(), dtype=m3.F32, draft_tokens=s["drafted"].data_ptr(),
        uniforms=s["uniforms"].data_ptr(), batch=4, drafts=3, vocabulary=vocabulary, tokens=s["tokens"].data_ptr(),
        accepted=s["accepted"].data_ptr())
    return s


def step(m3, s, stream):
    """Norm, a product, the cache written and read back, a product, the drafts verified."""
    import torch

    m3.rms_norm_e4m3(s["norm"], stream=stream)
    y = s["codes"].view(torch.float8_e4m3fn).float().view(64, -1, 128) * s["scales"][..., None]
    s["kv"].copy_((y.view(64, -1) @ s["weights"]).view(s["kv"].shape))
    s["cache"].write(s["batch"], s["keys"], s["values"], stream=stream)
    s["cache"].read(s["batch"], *s["outs"], stream=stream)
    h = s["back"].float().transpose(0, 1).reshape(4, 16, -1)[:, -4:]
    s["target"].copy_(torch.softmax(h @ s["head"], -1))
    m3.verify_draft(s["verify"], stream=stream)


def check_step(m3, s):
    """Each operator of the run against its own plain form, on what it was given."""
    import torch

    torch.cuda.synchronize()
    s["cache"].synchronize()
    h = (s["x"].float() + s["r"].float()).bfloat16()
    assert torch.equal(h, s["sum"])
    check_norm(h, s["w"], 128, s["codes"], s["scales"])
    scale, value = quantised(host(s["kv"]))
    back = torch.from_numpy(value.astype(np.float32) * scale[..., None]).bfloat16()
    assert torch.equal(s["back"].transpose(0, 1).reshape(64, 16, 128).cpu(), back)
    want = verify_host(host(s["target"]), None, s["drafted"].cpu().numpy(), None, host(s["uniforms"]))
    assert np.array_equal(s["tokens"].cpu().numpy(), want[0]) and np.array_equal(s["accepted"].cpu().numpy(), want[1])


def test_step_together(m3, gpu):
    s = step_state(m3, 1)
    step(m3, s, 0)
    check_step(m3, s)


def test_step_on_two_streams_at_once(m3, gpu):
    import torch

    states = [step_state(m3, seed) for seed in (2, 3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                step(m3, s, stream.cuda_stream)
    for s in states:
        check_step(m3, s)


def test_step_captured_and_replayed(m3, gpu):
    """Two graphs captured before either is replayed, replayed in turn with new inputs."""
    import torch

    states = [step_state(m3, seed) for seed in (4, 5)]
    graphs = []
    for s in states:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(m3, s, side.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(m3, s, torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for turn in range(3):
        for s in states:
            s["x"].normal_()
            s["uniforms"].uniform_(0, 0.999)
            s["starts"].copy_(torch.tensor([3, 17, 48, turn], dtype=torch.int32))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        for s in states:
            check_step(m3, s)


# ------------------------------------------------------------- graph sessions

def raw(t):
    """A tensor as the session writes it: F32, or the 16-bit words."""
    import torch

    return t.cpu().numpy() if t.dtype in (torch.float32, torch.int32) else t.view(torch.int16).cpu().numpy()


def norm_session(m3, x, w, group, r=None, keep_sum=False, **options):
    import torch

    dtype = {torch.float32: m3.F32, torch.float16: m3.F16, torch.bfloat16: m3.BF16}
    shape = (2, x.shape[0] // 2, x.shape[1])
    g = m3.Graph()
    vx = g.value(m3.INPUT, dtype[x.dtype], shape)
    vr = vh = None
    h = vx
    if r is not None:
        vr = g.value(m3.INPUT, dtype[x.dtype], shape)
        h = vh = g.inferred("ADD", [vx, vr], m3.OUTPUT if keep_sum else m3.TEMPORARY, dtype[x.dtype])
        g.node("ADD", [vx, vr], [vh])
    vw = g.value(m3.INPUT, dtype[w.dtype], (x.shape[1],))
    codes = g.inferred("RMS_NORM_E4M3", [h, vw], m3.OUTPUT, m3.E4M3, epsilon=1e-6)
    scales = g.value(m3.OUTPUT, m3.F32, shape[:2] + (x.shape[1] // group,))
    g.node("RMS_NORM_E4M3", [h, vw], [codes, scales], epsilon=1e-6)
    s = m3.Session(g, **options)
    s.write(vx, raw(x))
    s.write(vw, raw(w))
    if vr is not None:
        s.write(vr, raw(r))
    return s, codes, scales, vh


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, width, group", [(2, 64, 64), (64, 2048, 128), (10, 515, 515), (6, 4104, 24)])
@pytest.mark.parametrize("residual", [None, "kept", "dropped"])
def test_norm_in_a_session(m3, gpu, dtype, rows, width, group, residual):
    import torch

    g = torch.Generator(device="cuda").manual_seed(width)
    t = torch_dtype(dtype)
    x = torch.randn(rows, width, generator=g, device="cuda").to(t)
    r = torch.randn(rows, width, generator=g, device="cuda").to(t) if residual else None
    w = torch.randn(width, generator=g, device="cuda").to(t)
    codes, scales = run_norm(m3, x, w, group, r, None)
    for options in (dict(), dict(fuse=False), dict(cuda_graphs=False)):
        s, vc, vs, vh = norm_session(m3, x, w, group, r, residual == "kept", **options)
        for _ in range(2):
            s.run()
        s.run_async()
        s.run_async()
        s.synchronize()
        assert np.array_equal(s.read(vc).reshape(rows, width), codes.cpu().numpy())
        assert np.array_equal(s.read(vs).reshape(rows, -1), scales.cpu().numpy())
        if residual == "kept":
            h = (x.float() + r.float()).to(t)
            assert np.array_equal(s.read(vh).reshape(rows, width).view(raw(h).dtype), raw(h))
        s.close()


def test_norm_split_over_rows(m3, gpu):
    """Two shards of one graph on this GPU give the whole graph's results."""
    import torch

    x = torch.randn(8, 2, 256, device="cuda").bfloat16()
    w = torch.randn(256, device="cuda")
    whole = run_norm(m3, x.view(16, 256), w, 64)
    codes, scales = np.zeros((8, 2, 256), np.uint8), np.zeros((8, 2, 4), np.float32)
    for rank in (0, 1):
        g = m3.Graph()
        vx, vw = g.value(m3.INPUT, m3.BF16, (8, 2, 256)), g.value(m3.INPUT, m3.F32, (256,))
        vc = g.inferred("RMS_NORM_E4M3", [vx, vw], m3.OUTPUT, m3.E4M3, epsilon=1e-6)
        vs = g.value(m3.OUTPUT, m3.F32, (8, 2, 4))
        g.node("RMS_NORM_E4M3", [vx, vw], [vc, vs], epsilon=1e-6)
        s = m3.Session(g, shard=m3.ShardOptions(rank, 2, 0))
        hx = np.ascontiguousarray(raw(x))
        s.shard_write(vx, hx.ctypes.data, hx.nbytes)
        s.write(vw, raw(w))
        s.run()
        s.shard_read(vc, codes.ctypes.data, codes.nbytes)
        s.shard_read(vs, scales.ctypes.data, scales.nbytes)
    assert np.array_equal(codes.reshape(16, 256), whole[0].cpu().numpy())
    assert np.array_equal(scales.reshape(16, 4), whole[1].cpu().numpy())


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_verify_behind_softmax_in_a_session(m3, gpu, drawn, ragged):
    """SOFTMAX of the logits, then VERIFY_DRAFT, in one graph; a NaN logit fails the run before it."""
    import torch

    batch, drafts, vocabulary = 6, 3, 1000
    rng = np.random.default_rng(3)
    logits = rng.normal(size=(batch, drafts + 1, vocabulary)).astype(np.float32) * 2
    tokens = rng.integers(0, vocabulary, (batch, drafts)).astype(np.int32)
    tokens[2:] = logits[2:, :drafts].argmax(-1)
    uniforms = rng.uniform(0, 0.05, (batch, drafts + 1)).astype(np.float32)
    lengths = np.array([3, 0, 3, 1, 2, -1], np.int32)
    g = m3.Graph()
    vl = g.value(m3.INPUT, m3.F32, logits.shape)
    p = g.inferred("SOFTMAX", [vl], m3.OUTPUT, m3.F32)
    g.node("SOFTMAX", [vl], [p])
    vt, vu = g.value(m3.INPUT, m3.I32, tokens.shape), g.value(m3.INPUT, m3.F32, uniforms.shape)
    vq = g.value(m3.INPUT, m3.F32, (batch, drafts, vocabulary)) if drawn else None
    vn = g.value(m3.INPUT, m3.I32, (batch,)) if ragged else None
    ins = [p, vt, vu, vq, vn]
    out = g.inferred("VERIFY_DRAFT", ins, m3.OUTPUT, m3.I32, 0)
    accepted = g.inferred("VERIFY_DRAFT", ins, m3.OUTPUT, m3.I32, 1)
    g.node("VERIFY_DRAFT", ins, [out, accepted])
    s = m3.Session(g)
    assert s.plan_report()[1] == "row[SOFTMAX]; row[VERIFY_DRAFT]"
    q = np.full((batch, drafts, vocabulary), 1.0 / vocabulary, np.float32)
    for value, data in ((vl, logits), (vt, tokens), (vu, uniforms), (vq, q), (vn, lengths)):
        if value is not None:
            s.write(value, data)
    s.run()
    target = s.read(p).astype(np.float64)
    want = verify_host(target, q.astype(np.float64) if drawn else None, tokens, lengths if ragged else None,
                       uniforms.astype(np.float64))
    assert np.array_equal(s.read(out), want[0]) and np.array_equal(s.read(accepted), want[1])
    assert want[1].max() > 0
    # a failing run leaves the outputs as they were
    bad = logits.copy()
    bad[1, 1, 5] = np.nan
    s.write(vl, bad)
    s.write(vu, uniforms / 2)
    status, message = s.run_status()
    assert status == m3.OUT_OF_RANGE and "softmax" in message
    assert np.array_equal(s.read(out), want[0]) and np.array_equal(s.read(accepted), want[1])
    s.write(vl, logits)
    s.run()
    want = verify_host(target, q.astype(np.float64) if drawn else None, tokens, lengths if ragged else None,
                       uniforms.astype(np.float64) / 2)
    assert np.array_equal(s.read(out), want[0]) and np.array_equal(s.read(accepted), want[1])


def test_serving_operators_beside_others_in_a_wave(m3, gpu):
    """Independent launches without a data check run at the same time."""
    import torch

    g = m3.Graph()
    x, w = g.value(m3.INPUT, m3.BF16, (512, 1024)), g.value(m3.INPUT, m3.F32, (1024,))
    codes = g.inferred("RMS_NORM_E4M3", [x, w], m3.OUTPUT, m3.E4M3, epsilon=1e-6)
    scales = g.inferred("RMS_NORM_E4M3", [x, w], m3.OUTPUT, m3.F32, 1, epsilon=1e-6)
    g.node("RMS_NORM_E4M3", [x, w], [codes, scales], epsilon=1e-6)
    target, tokens = g.value(m3.INPUT, m3.F32, (8, 3, 4000)), g.value(m3.INPUT, m3.I32, (8, 2))
    uniforms = g.value(m3.INPUT, m3.F32, (8, 3))
    out = g.inferred("VERIFY_DRAFT", [target, tokens, uniforms], m3.OUTPUT, m3.I32, 0)
    accepted = g.inferred("VERIFY_DRAFT", [target, tokens, uniforms], m3.OUTPUT, m3.I32, 1)
    g.node("VERIFY_DRAFT", [target, tokens, uniforms], [out, accepted])
    a = g.value(m3.INPUT, m3.F32, (4096, 512))
    doubled = g.inferred("ADD", [a, a], m3.OUTPUT, m3.F32)
    g.node("ADD", [a, a], [doubled])
    rng = np.random.default_rng(12)
    s = m3.Session(g)
    hx = torch.from_numpy(rng.normal(size=(512, 1024))).bfloat16()
    hw = rng.normal(size=1024).astype(np.float32)
    ht = rng.dirichlet(np.ones(4000) * 0.05, (8, 3)).astype(np.float32)
    hk, hu = ht[:, :2].argmax(-1).astype(np.int32), rng.uniform(0, 0.2, (8, 3)).astype(np.float32)
    ha = rng.normal(size=(4096, 512)).astype(np.float32)
    for value, data in ((x, raw(hx)), (w, hw), (target, ht), (tokens, hk), (uniforms, hu), (a, ha)):
        s.write(value, data)
    for _ in range(5):
        s.run_async()
    s.synchronize()
    check_norm(hx, torch.from_numpy(hw), 1024, torch.from_numpy(s.read(codes)), torch.from_numpy(s.read(scales)))
    want = verify_host(ht.astype(np.float64), None, hk, None, hu.astype(np.float64))
    assert np.array_equal(s.read(out), want[0]) and np.array_equal(s.read(accepted), want[1])
    assert np.array_equal(s.read(doubled), ha + ha)


def test_empty_batches_in_a_session(m3, gpu):
    """No rows, no sequences: the runs still count as started, and later ones work."""
    g = m3.Graph()
    x, w = g.value(m3.INPUT, m3.F32, (0, 64)), g.value(m3.INPUT, m3.F32, (64,))
    codes = g.inferred("RMS_NORM_E4M3", [x, w], m3.OUTPUT, m3.E4M3, epsilon=1e-6)
    scales = g.inferred("RMS_NORM_E4M3", [x, w], m3.OUTPUT, m3.F32, 1, epsilon=1e-6)
    g.node("RMS_NORM_E4M3", [x, w], [codes, scales], epsilon=1e-6)
    target, tokens = g.value(m3.INPUT, m3.F32, (0, 4, 100)), g.value(m3.INPUT, m3.I32, (0, 3))
    uniforms = g.value(m3.INPUT, m3.F32, (0, 4))
    out = g.inferred("VERIFY_DRAFT", [target, tokens, uniforms], m3.OUTPUT, m3.I32, 0)
    accepted = g.inferred("VERIFY_DRAFT", [target, tokens, uniforms], m3.OUTPUT, m3.I32, 1)
    g.node("VERIFY_DRAFT", [target, tokens, uniforms], [out, accepted])
    s = m3.Session(g)
    s.run()
    s.run()
    assert s.read(codes).shape == (0, 64) and s.read(accepted).shape == (0,)


def test_plugin_refuses_session_operators(m3, gpu):
    import ctypes

    lib, err, context = m3.load(), m3.M3Error(), ctypes.c_void_p()
    accessor = m3.STORAGE_DATA(lambda storage: storage)
    options = m3.BackendOptions(0, accessor, False)
    m3.check(lib.m3_cuda_backend_context_create(ctypes.byref(options), ctypes.byref(context), ctypes.byref(err)), err)
    for kind in ("RMS_NORM_E4M3", "VERIFY_DRAFT"):
        commands = (m3.Command * 1)()
        commands[0].kind = m3.OPS[kind]
        assert lib.m3_cuda_backend_execute(context, commands, 1, None, ctypes.byref(err)) == m3.UNSUPPORTED
    lib.m3_cuda_backend_destroy_context(context)
