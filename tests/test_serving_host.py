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
