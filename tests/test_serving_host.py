"""Refusals of the serving operators: every check of their arguments comes
before any device work, so the calls are made here without a GPU.  The
addresses are made up; a call that passed the checks would end in "no CUDA
device" on such a host, and is not made on one with a device."""

from __future__ import annotations

import ctypes

import pytest

A = 0x10000000          # a made-up, well aligned device address
STEP = 0x10000000


def refused(m3, call, status, text):
    with pytest.raises(m3.M3Failure) as failure:
        call()
    assert failure.value.status == status, failure.value
    assert text in failure.value.message


def norm_args(m3, **change):
    fields = dict(input=A, residual=A + STEP, sum=A + 2 * STEP, dtype=m3.BF16, scale=A + 3 * STEP,
                  scale_dtype=m3.F32, rows=16, width=64, group=32, codes=A + 4 * STEP, code_scales=A + 5 * STEP)
    fields.update(change)
    return m3.RmsNormE4m3Args(**fields)


@pytest.mark.parametrize("change, status, text", [
    (dict(dtype=3), 1, "norm input must be F32, F16 or BF16"),
    (dict(dtype=64), 1, "norm input must be F32, F16 or BF16"),
    (dict(scale_dtype=-1), 1, "norm scale must be F32, F16 or BF16"),
    (dict(width=0), 1, "width, group or epsilon"),
    (dict(width=1 << 31), 1, "width, group or epsilon"),
    (dict(group=48), 1, "width, group or epsilon"),
    (dict(group=128), 1, "width, group or epsilon"),
    (dict(epsilon=0.0), 1, "width, group or epsilon"),
    (dict(epsilon=-1e-6), 1, "width, group or epsilon"),
    (dict(epsilon=float("nan")), 1, "width, group or epsilon"),
    (dict(epsilon=float("inf")), 1, "width, group or epsilon"),
    (dict(residual=None), 1, "norm sum needs a residual"),
    (dict(input=None), 1, "norm input is required"),
    (dict(scale=None), 1, "norm scale is required"),
    (dict(codes=None), 1, "norm codes is required"),
    (dict(code_scales=None), 1, "norm code scales is required"),
    (dict(input=A + 1), 1, "norm input is not aligned"),
    (dict(residual=A + STEP + 1), 1, "norm residual is not aligned"),
    (dict(scale=A + 3 * STEP + 2), 1, "norm scale is not aligned"),
    (dict(code_scales=A + 5 * STEP + 2), 1, "norm code scales is not aligned"),
    (dict(input_stride=63), 1, "norm input stride is less than its row"),
    (dict(sum_stride=1), 1, "norm sum stride is less than its row"),
    (dict(rows=1 << 62), 3, "overflows"),
    (dict(input_stride=1 << 62), 3, "overflows"),
    # outputs over inputs and each other
    (dict(sum=A + 2), 1, "norm sum overlaps norm input"),
    (dict(sum=A, sum_stride=128), 1, "norm sum overlaps norm input"),
    (dict(sum=A + STEP + 128), 1, "norm sum overlaps norm residual"),
    (dict(sum=A + 3 * STEP), 1, "norm sum overlaps norm scale"),
    (dict(codes=A), 1, "norm codes overlaps norm input"),
    (dict(codes=A + STEP + 16 * 128 - 1), 1, "norm codes overlaps norm residual"),
    (dict(codes=A + 2 * STEP), 1, "norm codes overlaps norm sum"),
    (dict(code_scales=A + 4 * STEP), 1, "norm code scales overlaps norm codes"),
    (dict(code_scales=A + 3 * STEP), 1, "norm code scales overlaps norm scale"),
])
def test_norm_refusals(m3, change, status, text):
    refused(m3, lambda: m3.rms_norm_e4m3(norm_args(m3, **change)), status, text)


def test_norm_null_arguments(m3):
    err = m3.M3Error()
    assert m3.load().m3_cuda_rms_norm_e4m3(0, None, None, ctypes.byref(err)) == m3.INVALID_ARGUMENT
    assert m3.load().m3_cuda_rms_norm_e4m3(0, None, None, None) == m3.INVALID_ARGUMENT


def test_initialisers(m3):
    norm, verify = m3.RmsNormE4m3Args(rows=5), m3.VerifyDraftArgs(batch=5)
    m3.load().m3_cuda_rms_norm_e4m3_args_init(norm)
    m3.load().m3_cuda_verify_draft_args_init(verify)
    assert norm.rows == 0 and abs(norm.epsilon - 1e-6) < 1e-12 and not norm.input
    assert verify.batch == 0 and not verify.target
    cache = m3.CacheOptions(5, 5, 5, 5, 5)
    m3.load().m3_cuda_cache_options_init(cache)
    assert (cache.device, cache.pages, cache.page_tokens, cache.heads, cache.head_dim) == (-1, 0, 16, 0, 0)
    for init in ("rms_norm_e4m3_args", "verify_draft_args", "cache_options"):
        getattr(m3.load(), f"m3_cuda_{init}_init")(None)


def verify_args(m3, **change):
    fields = dict(target=A, draft=A + STEP, dtype=m3.F32, draft_tokens=A + 2 * STEP, lengths=A + 3 * STEP,
                  uniforms=A + 4 * STEP, batch=3, drafts=4, vocabulary=100, tokens=A + 5 * STEP,
                  accepted=A + 6 * STEP)
    fields.update(change)
    return m3.VerifyDraftArgs(**fields)


@pytest.mark.parametrize("change, status, text", [
    (dict(dtype=3), 1, "verified probabilities must be F32, F16 or BF16"),
    (dict(vocabulary=0), 1, "out of range"),
    (dict(vocabulary=1 << 31), 1, "out of range"),
    (dict(batch=1 << 31), 1, "out of range"),
    (dict(drafts=(1 << 31) - 1), 1, "out of range"),
    (dict(target=None), 1, "target probabilities is required"),
    (dict(draft_tokens=None), 1, "drafted tokens is required"),
    (dict(uniforms=None), 1, "verification uniforms is required"),
    (dict(tokens=None), 1, "verified tokens is required"),
    (dict(accepted=None), 1, "accepted counts is required"),
    (dict(target=A + 2), 1, "target probabilities is not aligned"),
    (dict(uniforms=A + 4 * STEP + 1), 1, "verification uniforms is not aligned"),
    (dict(target_stride=99), 1, "target probabilities stride is less than its row"),
    (dict(draft_stride=99), 1, "draft probabilities stride is less than its row"),
    (dict(target_stride=1 << 60), 3, "overflows"),
    (dict(tokens=A + 2 * STEP), 1, "verified tokens overlaps drafted tokens"),
    (dict(tokens=A), 1, "verified tokens overlaps target probabilities"),
    (dict(accepted=A + 3 * STEP), 1, "accepted counts overlaps draft lengths"),
    (dict(accepted=A + 5 * STEP + 4 * 14), 1, "accepted counts overlaps verified tokens"),
])
def test_verify_refusals(m3, change, status, text):
    refused(m3, lambda: m3.verify_draft(verify_args(m3, **change)), status, text)


@pytest.mark.parametrize("options, status, text", [
    ((0, 16, 8, 128), 1, "out of range"),
    ((1 << 31, 16, 8, 128), 1, "out of range"),
    ((10, 0, 8, 128), 1, "out of range"),
    ((10, 16, 0, 128), 1, "out of range"),
    ((10, 16, 8, 0), 1, "out of range"),
    ((10, (1 << 20) + 1, 8, 128), 1, "out of range"),
    ((10, 16, 1 << 11, 1 << 10), 1, "out of range"),
    (((1 << 31) - 1, 1 << 20, 1 << 10, 1 << 10), 3, "cache size overflows"),
])
def test_cache_creation_refusals(m3, options, status, text):
    refused(m3, lambda: m3.Cache(*options), status, text)


def test_cache_null(m3):
    lib, err = m3.load(), m3.M3Error()
    batch, rows, empty = m3.CacheBatch(), m3.CacheRows(), ctypes.c_void_p()
    assert lib.m3_cuda_cache_create(None, m3.CacheOptions(), err) == m3.INVALID_ARGUMENT
    assert lib.m3_cuda_cache_create(ctypes.byref(empty), None, err) == m3.INVALID_ARGUMENT
    for call in (lib.m3_cuda_cache_write, lib.m3_cuda_cache_read):
        assert call(None, None, batch, rows, rows, err) == m3.INVALID_ARGUMENT
        assert b"required" in err.message
    assert lib.m3_cuda_cache_synchronize(None, None, err) == m3.INVALID_ARGUMENT
    assert lib.m3_cuda_cache_device_pointers(None, None, None, None, None, err) == m3.INVALID_ARGUMENT
    lib.m3_cuda_cache_free(None)


# ------------------------------------------------------------ graph operators

def norm_graph(m3, shape=(6, 4, 128), groups=1, dtype=None, residual=False, role=None):
    g = m3.Graph()
    dtype = m3.BF16 if dtype is None else dtype
    x = g.value(m3.INPUT, dtype, shape)
    if residual:
        r = g.value(m3.INPUT, dtype, shape)
        h = g.inferred("ADD", [x, r], m3.TEMPORARY if role is None else role, dtype)
        g.node("ADD", [x, r], [h])
    else:
        h = x
    w = g.value(m3.INPUT, m3.F32, shape[-1:])
    codes = g.inferred("RMS_NORM_E4M3", [h, w], m3.OUTPUT, m3.E4M3, epsilon=1e-6)
    scales = g.value(m3.OUTPUT, m3.F32, shape[:-1] + (groups,))
    return g, (h, w), (codes, scales)


def test_norm_node_plans(m3):
    for residual, text in ((False, "row[RMS_NORM_E4M3]"), (True, "row[ADD+RMS_NORM_E4M3]")):
        g, ins, outs = norm_graph(m3, residual=residual, groups=4)
        g.node("RMS_NORM_E4M3", ins, outs, epsilon=1e-6)
        info, report, described = m3.graph_plan(g)
        assert described == text and report.launch_count == 1 and report.shadow_bytes == 0
        if residual:
            _, report, described = m3.graph_plan(g, fuse=False)
            assert described == "ew[ADD] stores=1; row[RMS_NORM_E4M3]" and report.launch_count == 2
    # one byte per code: 6 * 4 * 128 codes next to the inputs, the sum and the scales
    assert info.allocated_bytes == 6 * 4 * 128 * (2 + 2 + 2 + 1) + 128 * 4 + 6 * 4 * 4 * 4


def test_norm_node_inference(m3):
    g, ins, _ = norm_graph(m3)
    assert g.values[-2][:2] == (m3.E4M3, (6, 4, 128))
    scales = g.inferred("RMS_NORM_E4M3", ins, m3.OUTPUT, m3.F32, 1, epsilon=1e-6)
    assert g.values[scales][:2] == (m3.F32, (6, 4, 1))
    refused(m3, lambda: g.inferred("RMS_NORM_E4M3", ins, m3.OUTPUT, m3.F32, 2), m3.OUT_OF_RANGE, "no requested")
    refused(m3, lambda: g.inferred("RMS_NORM", ins, m3.OUTPUT, m3.F32, 1), m3.OUT_OF_RANGE, "no requested")


@pytest.mark.parametrize("change, text", [
    (dict(epsilon=0.0), "epsilon is invalid"),
    (dict(groups=3), "groups dividing"),
    (dict(groups=0), "groups dividing"),
    (dict(scales=(24, 4)), "groups dividing"),
    (dict(codes_dtype="F32"), "codes must be E4M3"),
    (dict(scales_dtype="BF16"), "codes must be E4M3"),
    (dict(weight=(64,)), "channel shape"),
    (dict(dtype="I32"), "floating-point"),
])
def test_norm_node_refusals(m3, change, text):
    g = m3.Graph()
    x = g.value(m3.INPUT, getattr(m3, change.get("dtype", "F16")), (6, 4, 128))
    w = g.value(m3.INPUT, m3.F32, change.get("weight", (128,)))
    codes = g.value(m3.OUTPUT, getattr(m3, change.get("codes_dtype", "E4M3")), (6, 4, 128))
    scales = g.value(m3.OUTPUT, getattr(m3, change.get("scales_dtype", "F32")),
                     change.get("scales", (6, 4, change.get("groups", 1))))
    g.node("RMS_NORM_E4M3", [x, w], [codes, scales], epsilon=change.get("epsilon", 1e-6))
    refused(m3, lambda: m3.graph_plan(g), m3.INVALID_ARGUMENT, text)


def test_no_other_operator_takes_e4m3(m3):
    for kind, status in (("COPY", m3.UNSUPPORTED), ("CAST", m3.UNSUPPORTED), ("SOFTMAX", m3.INVALID_ARGUMENT),
                         ("TANH", m3.INVALID_ARGUMENT), ("ABS_MAX", m3.INVALID_ARGUMENT),
                         ("ROW_SUM", m3.INVALID_ARGUMENT), ("CLAMP_UNIT", m3.INVALID_ARGUMENT)):
        g = m3.Graph()
        x = g.value(m3.INPUT, m3.E4M3, (4, 8))
        out = g.value(m3.OUTPUT, m3.E4M3 if kind == "COPY" else m3.F32, (4, 8))
        g.node(kind, [x], [out])
        with pytest.raises(m3.M3Failure) as failure:
            m3.graph_plan(g)
        assert failure.value.status == status, (kind, failure.value)
    for dtype in (4, 63, 65, -1):
        with pytest.raises(m3.M3Failure):
            m3.Graph().value(m3.INPUT, dtype, (4,))


def verify_graph(m3, batch=3, drafts=4, vocabulary=50, drawn=True, lengths=True, **change):
    g = m3.Graph()
    dtype = getattr(m3, change.get("dtype", "F32"))
    ins = [g.value(m3.INPUT, dtype, change.get("target", (batch, drafts + 1, vocabulary))),
           g.value(m3.INPUT, getattr(m3, change.get("tokens_dtype", "I32")), change.get("tokens", (batch, drafts))),
           g.value(m3.INPUT, getattr(m3, change.get("uniforms_dtype", "F32")),
                   change.get("uniforms", (batch, drafts + 1))),
           g.value(m3.INPUT, getattr(m3, change.get("draft_dtype", change.get("dtype", "F32"))),
                   change.get("draft", (batch, drafts, vocabulary))) if drawn else None,
           g.value(m3.INPUT, getattr(m3, change.get("lengths_dtype", "I32")), change.get("lengths_shape", (batch,)))
           if lengths else None]
    outs = [g.value(m3.OUTPUT, m3.I32, change.get("out", (batch, drafts + 1))),
            g.value(m3.OUTPUT, m3.I32, change.get("accepted", (batch,)))]
    g.node("VERIFY_DRAFT", ins, outs)
    return g, ins, outs


def test_verify_node_plans(m3):
    for drawn in (False, True):
        for lengths in (False, True):
            g, ins, _ = verify_graph(m3, drawn=drawn, lengths=lengths)
            _, report, described = m3.graph_plan(g)
            assert described == "row[VERIFY_DRAFT]" and report.shadow_bytes == 0
    tokens = g.inferred("VERIFY_DRAFT", ins, m3.OUTPUT, m3.I32, 0)
    accepted = g.inferred("VERIFY_DRAFT", ins, m3.OUTPUT, m3.I32, 1)
    assert g.values[tokens][:2] == (m3.I32, (3, 5)) and g.values[accepted][:2] == (m3.I32, (3,))


@pytest.mark.parametrize("change, text", [
    (dict(dtype="I32"), "dtype"), (dict(tokens_dtype="F32"), "dtype"), (dict(uniforms_dtype="BF16"), "dtype"),
    (dict(draft_dtype="F16"), "dtype"), (dict(lengths_dtype="F32"), "dtype"),
    (dict(target=(3, 250)), "shape"), (dict(target=(3, 5, 0)), "shape"), (dict(tokens=(3, 5)), "shape"),
    (dict(tokens=(12,)), "shape"), (dict(uniforms=(3, 4)), "shape"), (dict(draft=(3, 5, 50)), "shape"),
    (dict(draft=(3, 4, 51)), "shape"), (dict(lengths_shape=(3, 1)), "shape"), (dict(out=(3, 4)), "shape"),
    (dict(accepted=(3, 1)), "shape"),
])
def test_verify_node_refusals(m3, change, text):
    g, _, _ = verify_graph(m3, **change)
    refused(m3, lambda: m3.graph_plan(g), m3.INVALID_ARGUMENT, f"verification {text} is invalid")


def test_serving_nodes_are_the_sessions_own(m3):
    lib = m3.load()
    for kind in ("RMS_NORM_E4M3", "VERIFY_DRAFT"):
        assert not lib.m3_cuda_backend_supports_kind(m3.OPS[kind])
    assert lib.m3_cuda_backend_supports_kind(m3.OPS["RMS_NORM"])


def test_serving_nodes_split(m3):
    g, ins, outs = norm_graph(m3, shape=(8, 4, 128), groups=4)
    g.node("RMS_NORM_E4M3", ins, outs, epsilon=1e-6)
    for rank in (0, 1):
        slab, axis = m3.shard_plan(g, rank, 2, -1, outs[1])
        assert axis == 0 and slab.split and slab.begin == 4 * rank and slab.extent == 4
    refused(m3, lambda: m3.shard_plan(g, 0, 2, 2, outs[0]), m3.UNSUPPORTED, "axis 2")
    g, _, outs = verify_graph(m3)
    refused(m3, lambda: m3.shard_plan(g, 0, 2, 0, outs[0]), m3.UNSUPPORTED, "VERIFY_DRAFT (node 0) cannot be sharded")
