"""Counters of captured launches belong to their graph (the host side here, two graphs at once on the GPU)."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from varlen_oracle import assert_attention, make_batch


@pytest.fixture
def captures(monkeypatch):
    """A stand-in for the stream's capture state: set ``captures.id``."""
    from types import SimpleNamespace

    from mxflashattn_b200 import backend

    state = SimpleNamespace(id=0)
    monkeypatch.setattr(backend, "_COUNTERS", {})
    monkeypatch.setattr(backend, "_CAPTURE_COUNTERS", {}, raising=False)
    monkeypatch.setattr(backend, "_capture_id", lambda device, stream: state.id, raising=False)
    # (the query of the code before captures had counters of their own)
    monkeypatch.setattr(backend, "_capturing", lambda: state.id != 0)
    return state


def test_a_capture_shares_its_counters_with_nobody(captures):
    import torch

    from mxflashattn_b200 import backend

    cpu, stream = torch.device("cpu"), 7
    captures.id = 1
    first = backend.split_counters(cpu, stream, 100)
    assert backend.split_counters(cpu, stream, 100).data_ptr() == first.data_ptr()  # one zeroing node per graph
    captures.id = 2
    second = backend.split_counters(cpu, stream, 100)
    captures.id = 0
    eager = backend.split_counters(cpu, stream, 100)
    assert len({first.data_ptr(), second.data_ptr(), eager.data_ptr()}) == 3
    assert not first.any() and not second.any() and not eager.any()
    captures.id = 3
    assert backend.split_counters(cpu, stream, 100).data_ptr() not in (first.data_ptr(), eager.data_ptr())
    captures.id = 0
    assert backend.split_counters(cpu, stream, 100).data_ptr() == eager.data_ptr()


def test_a_capture_that_needs_more_counters_gets_them(captures):
    import torch

    from mxflashattn_b200 import backend

    cpu = torch.device("cpu")
    for capture in (1, 0):
        captures.id = capture
        small = backend.split_counters(cpu, 9, 16)
        large = backend.split_counters(cpu, 9, 4 * (small.numel() + 1))
        assert large.numel() > small.numel() and not large.any()
        assert backend.split_counters(cpu, 9, 16).data_ptr() == large.data_ptr()


def test_a_stream_that_does_not_exist_is_no_capture():
    import ctypes

    from mxflashattn_b200 import _lib

    assert _lib.load().mxfa_stream_capture_id(None, None) == _lib.MXFA_ERR_INVALID
    out = ctypes.c_ulonglong(5)
    _lib.load().mxfa_stream_capture_id(None, ctypes.byref(out))
    assert out.value == 0


def _split_step(dev, seed):
    """A decode step whose sequences are split over CTAs."""
    b = make_batch(seed, [1, 1], [3000, 900], hq=8, hkv=2, quant=True)
    return b, b.device(dev), 1


def _split_pieces(dev, seed):
    """Pieces whose tiles are split over items."""
    b = make_batch(seed, [9, 40], [4000, 2500], hq=8, hkv=2)
    return b, b.device(dev), 40


def _run(t, max_q, out):
    import mxflashattn_b200 as fa

    fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], max_q, causal=True,
                                      k_scales=t["ks"], v_scales=t["vs"], out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("makers", [(_split_step, _split_pieces), (_split_pieces, _split_step),
                                    (_split_step, _split_step), (_split_pieces, _split_pieces)])
def test_two_graphs_replayed_in_any_order_and_at_once(makers, cuda_device):
    """Both captured on torch's capture stream without a run on it before; the second replayed first."""
    import torch

    from mxflashattn_b200 import _lib, backend

    _lib.read_error_flags()
    batches = [m(cuda_device, 1500 + i) for i, m in enumerate(makers)]
    assert backend.kvcache_plan(2, 1, 8, 2, 128, 3008)[0] > 1
    outs = [torch.empty_like(t["q"]) for _, t, _ in batches]
    graphs = []
    for (_, t, max_q), out in zip(batches, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _run(t, max_q, out)
            _run(t, max_q, out)
        graphs.append(graph)
    for i in (1, 0, 1):
        outs[i].fill_(float("nan"))
        graphs[i].replay()
        torch.cuda.synchronize()
        b = batches[i][0]
        assert_attention(host(outs[i]), None, b, b.d ** -0.5, True, f"graph {i}")
    want = [o.clone() for o in outs]
    eager = torch.empty_like(outs[0])
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        _run(batches[0][1], batches[0][2], eager)  # an eager launch beside them
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal(eager, want[0])
    assert _lib.read_error_flags() == 0


@pytest.mark.gpu
def test_a_captured_step_of_plan_tiles_and_unpacking_follows_the_lengths(cuda_device):
    """Plan, unpacking and split tiles recorded once; a replay reads the lengths that hold then."""
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import backend

    b = make_batch(1510, [300, 260], [2000, 900], hq=8, hkv=2, quant=True)
    assert backend.unpack_pays(560, 2, 4, 2, 128, 2000)
    t = b.device(cuda_device)
    out = torch.empty_like(t["q"])

    def step():
        plan = fa.kvcache_chunk_plan(t["cu"], t["lens"], 560, 300, q_heads=8, kv_heads=2, causal=True)
        fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 300, 2000, causal=True,
                                          k_scales=t["ks"], v_scales=t["vs"], plan=plan, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for total in ([2000, 900], [700, 260], [1990, 1]):
        t["lens"].copy_(torch.tensor(total, dtype=torch.int32))
        b.total = total
        graph.replay()
        assert_attention(host(out), None, b, b.d ** -0.5, True, f"replay {total}")
    assert np.isfinite(host(out)).all()
