"""Which launches of a plan run at the same time (m3_cuda_graph_waves): those
that share no memory, in plans that cannot fail.  Host only."""

from __future__ import annotations

import ctypes

import pytest


def norm(m3, g, kind, shape=(64, 256), x=None):
    x = g.value(m3.INPUT, m3.BF16, shape) if x is None else x
    w = g.value(m3.INPUT, m3.F32, shape[-1:])
    if kind == "RMS_NORM_E4M3":
        outs = [g.inferred(kind, [x, w], m3.OUTPUT, m3.E4M3, epsilon=1e-6),
                g.inferred(kind, [x, w], m3.OUTPUT, m3.F32, 1, epsilon=1e-6)]
    else:
        outs = [g.inferred(kind, [x, w], m3.OUTPUT, m3.BF16, epsilon=1e-6)]
    g.node(kind, [x, w], outs, epsilon=1e-6)
    return x, outs


def add(m3, g, a=None):
    a = g.value(m3.INPUT, m3.F32, (4096, 512)) if a is None else a
    out = g.inferred("ADD", [a, a], m3.OUTPUT, m3.F32)
    g.node("ADD", [a, a], [out])
    return a, out


def verify(m3, g):
    ins = [g.value(m3.INPUT, m3.F32, (8, 3, 4000)), g.value(m3.INPUT, m3.I32, (8, 2)), g.value(m3.INPUT, m3.F32, (8, 3))]
    outs = [g.inferred("VERIFY_DRAFT", ins, m3.OUTPUT, m3.I32, k) for k in (0, 1)]
    g.node("VERIFY_DRAFT", ins, outs)


@pytest.mark.parametrize("kind", ["RMS_NORM_E4M3", "RMS_NORM", "LAYER_NORM"])
def test_independent_norms_join_one_wave(m3, kind):
    g = m3.Graph()
    g.value(m3.INPUT, m3.F32, (7,))         # a value that no node uses
    norm(m3, g, kind)
    norm(m3, g, kind)
    verify(m3, g)
    assert m3.graph_waves(g) == [0, 0, 0]
    # nor does what uses the first value wait for a norm
    g = m3.Graph()
    a, _ = add(m3, g)
    norm(m3, g, kind)
    verify(m3, g)
    assert m3.graph_waves(g) == [0, 0, 0]


def test_launches_that_share_memory_stay_apart(m3):
    g = m3.Graph()
    x, _ = norm(m3, g, "RMS_NORM")
    norm(m3, g, "RMS_NORM_E4M3", x=x)       # the same input
    add(m3, g)
    assert m3.graph_waves(g) == [0, 1, 1]
    # the sum of an ADD outside the norm's launch
    g = m3.Graph()
    x, r = g.value(m3.INPUT, m3.BF16, (64, 256)), g.value(m3.INPUT, m3.BF16, (64, 256))
    h = g.inferred("ADD", [x, r], m3.OUTPUT, m3.BF16)
    g.node("ADD", [x, r], [h])
    norm(m3, g, "RMS_NORM_E4M3", x=h)
    assert m3.graph_waves(g) == [0] and m3.graph_waves(g, fuse=False) == [0, 1]


def test_a_wave_has_four_launches_at_most(m3):
    g = m3.Graph()
    for _ in range(6):
        norm(m3, g, "RMS_NORM_E4M3")
    assert m3.graph_waves(g) == [0, 0, 0, 0, 1, 1]


def test_a_plan_that_can_fail_has_no_waves(m3):
    g = m3.Graph()
    norm(m3, g, "RMS_NORM_E4M3")
    x = g.value(m3.INPUT, m3.F32, (4, 8))
    p = g.inferred("SOFTMAX", [x], m3.OUTPUT, m3.F32)
    g.node("SOFTMAX", [x], [p])
    verify(m3, g)
    assert m3.graph_waves(g) == [0, 1, 2]


def test_waves_of_nothing_and_refusals(m3):
    g = m3.Graph()
    g.value(m3.INPUT, m3.F32, (7,))
    assert m3.graph_waves(g) == []
    lib, err = m3.load(), m3.M3Error()
    assert lib.m3_cuda_graph_waves(None, None, None, 0, None, err) == m3.INVALID_ARGUMENT
    assert lib.m3_cuda_graph_waves(g.handle, None, None, 1, None, err) == m3.INVALID_ARGUMENT
    norm(m3, g, "RMS_NORM")
    norm(m3, g, "RMS_NORM")
    one, count = (ctypes.c_uint32 * 2)(9, 9), ctypes.c_size_t()
    assert lib.m3_cuda_graph_waves(g.handle, None, one, 1, count, err) == m3.OK
    assert list(one) == [0, 9] and count.value == 2


@pytest.mark.gpu
def test_norms_of_one_wave_run_right(m3, gpu):
    import numpy as np
    import torch

    from test_gpu_serving import check_norm, raw

    g = m3.Graph()
    unused = g.value(m3.INPUT, m3.F32, (7,))
    shapes = [(512, 1024), (300, 515), (64, 2048)]
    graph = [norm(m3, g, "RMS_NORM_E4M3", shape) for shape in shapes]
    weights = [x + 1 for x, _ in graph]
    assert m3.graph_waves(g) == [0, 0, 0]
    s = m3.Session(g)
    s.write(unused, np.zeros(7, np.float32))
    rng = np.random.default_rng(5)
    data = [torch.from_numpy(rng.normal(size=shape)).bfloat16() for shape in shapes]
    scale = [rng.normal(size=shape[1]).astype(np.float32) for shape in shapes]
    for (x, _), w, hx, hw in zip(graph, weights, data, scale):
        s.write(x, raw(hx))
        s.write(w, hw)
    for _ in range(3):
        s.run_async()
    s.synchronize()
    for (_, (codes, scales)), hx, hw in zip(graph, data, scale):
        check_norm(hx, torch.from_numpy(hw), hx.shape[1], torch.from_numpy(s.read(codes)),
                   torch.from_numpy(s.read(scales)))
    s.close()
