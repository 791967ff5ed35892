"""The cached scratch memory of the compiled binding, beside CUDA graphs that hold its
addresses: it never moves under a graph, no graph owns it, and two graphs captured on
one stream may run at the same time."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import nibblegemm_b200 as ng
from tests import test_paged as tp

pytestmark = pytest.mark.gpu

GEMV, GEMM, ATTENTION = 0, 1, 2


def fresh_stream():
    """A stream that no call has used (torch.cuda.Stream() hands out 32 of them in turn)."""
    handle = ctypes.c_void_p()
    assert int(torch.cuda.cudart().cudaStreamCreate(ctypes.addressof(handle))) == 0
    return torch.cuda.ExternalStream(handle.value)


def scratch(stream, kind, need=0):
    return ng.extension().binding.workspace(torch.cuda.current_device(), stream.cuda_stream, kind, need)


def pool_of(pointer):
    """Which of the allocator's pools an address lies in; (0, 0) is the one that no graph owns."""
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= pointer < s["address"] + s["total_size"]:
            return tuple(s["segment_pool_id"])
    return None


def attention_inputs(dim, new, kv, hq=8, hk=2, dtype=torch.float16, seed=0):
    rng = np.random.default_rng(seed)
    torch.manual_seed(seed)
    k, v, table = tp.build_pages(rng, kv, 16, hk, dim, dtype, False)
    q = torch.randn(sum(new), hq, dim, device="cuda").to(dtype)
    return q, k, v, table, tp.ints(kv), tp.ints(np.concatenate([[0], np.cumsum(new)]))


def test_attention_scratch_does_not_move():
    s = fresh_stream()
    with torch.cuda.stream(s):
        ng.tree_attention(*attention_inputs(64, [3], [500]))
        first = scratch(s, ATTENTION).data_ptr()
        ng.tree_attention(*attention_inputs(128, [3], [500]))
        assert scratch(s, ATTENTION).data_ptr() == first
    tp.assert_clean()


@pytest.mark.parametrize("kind", [GEMV, GEMM])
def test_an_outgrown_buffer_stays_allocated(kind):
    """A graph captured before the buffer grew still writes to the old one."""
    s = fresh_stream()
    with torch.cuda.stream(s):
        w = scratch(s, kind, 1)
        old, size = w.data_ptr(), w.numel()
        del w
        assert scratch(s, kind, size + 1).data_ptr() != old
        others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
        assert all(not old <= x.data_ptr() < old + size for x in others)
        assert not scratch(s, kind).any()


def test_first_call_in_a_capture():
    """The capture owns no buffer that later calls use, and those are zero before its first replay."""
    torch.manual_seed(0)
    K, N = 512, 1024
    qw = ng.quantize(torch.randn(K, N)).to("cuda")
    x, many = (torch.randn(m, K, device="cuda").half() for m in (1, 128))
    inputs = attention_inputs(64, [3], [500])
    calls = (lambda: ng.gemv(x, qw)), (lambda: ng.gemm(many, qw)), (lambda: ng.tree_attention(*inputs))
    want = [f() for f in calls]
    torch.cuda.synchronize()
    s, graph = fresh_stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = [f() for f in calls]
    with torch.cuda.stream(s):
        for kind in (GEMV, GEMM, ATTENTION):
            assert pool_of(scratch(s, kind, 1).data_ptr()) == (0, 0)
        for kind in (GEMV, GEMM):
            assert not scratch(s, kind).any()
        again = [f() for f in calls]  # before any replay
        for y, w in zip(again, want):
            assert torch.equal(y, w)
        graph.replay()
    torch.cuda.synchronize()
    for y, w in zip(got, want):
        assert torch.equal(y, w)
    tp.assert_clean()


def test_a_captured_call_beside_later_calls():
    """A graph of a small head size, then calls of a large one on its stream: replays write nothing
    that is not theirs."""
    small, large = attention_inputs(64, [3, 40], [5000, 300]), attention_inputs(128, [3, 40], [5000, 300])
    want = ng.tree_attention(*small)
    torch.cuda.synchronize()
    s, graph, out = fresh_stream(), torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.stream(s):
        ng.tree_attention(*small)
        with torch.cuda.graph(graph, stream=s):
            ng.tree_attention(*small, out=out)
        ng.tree_attention(*large)
        others = [torch.full((n << 20,), 5, dtype=torch.uint8, device="cuda") for n in (1, 4, 20, 40, 45, 80)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all((x == 5).all() for x in others)
    tp.assert_clean()


@pytest.mark.parametrize("dim", [64, 128])
def test_graphs_of_one_stream_replayed_at_the_same_time(dim):
    """torch.cuda.graph captures on one stream unless it is told otherwise.  (Several parts an item,
    so that the scratch memory is used.)"""
    inputs = [attention_inputs(dim, new, kv, seed=i) for i, (new, kv) in enumerate((([3, 40], [9000, 3000]), ([16], [14000])))]
    want = [ng.tree_attention(*x) for x in inputs]
    torch.cuda.synchronize()
    outs, graphs = [torch.empty_like(w) for w in want], [torch.cuda.CUDAGraph() for _ in want]
    for x, out, graph in zip(inputs, outs, graphs):
        with torch.cuda.graph(graph):
            for _ in range(20):
                ng.tree_attention(*x, out=out)
    streams = [torch.cuda.Stream() for _ in want]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
    tp.assert_clean()


def test_the_route_without_the_binding():
    """Its buffers are kept in Python, under the same rules."""
    torch.manual_seed(0)
    K, N = 512, 1024
    ext, qw = ng.extension(), ng.quantize(torch.randn(K, N)).to("cuda")
    x, many = (torch.randn(m, K, device="cuda").half() for m in (1, 128))
    plain = type(ext)()
    plain.binding = None
    calls = (lambda e: e.gemv_w4a16(x, qw.qweight, qw.scales, 128)), (lambda e: e.gemm_w4a16(many, qw.qweight, qw.scales, 128))
    want = [f(ext) for f in calls]
    torch.cuda.synchronize()
    s, graph = fresh_stream(), torch.cuda.CUDAGraph()
    key = (torch.cuda.current_device(), s.cuda_stream)
    with torch.cuda.graph(graph, stream=s):
        got = [f(plain) for f in calls]
    assert key not in plain._ws and key not in plain._gws
    with torch.cuda.stream(s):
        for y, w in zip([f(plain) for f in calls], want):
            assert torch.equal(y, w)
        graph.replay()
    torch.cuda.synchronize()
    for y, w in zip(got, want):
        assert torch.equal(y, w)
    with torch.cuda.stream(s):
        old = plain._ws[key].data_ptr()
        size = plain._ws[key].numel()
        grown = plain._cached(plain._ws, size + 1, 1, x.device, s.cuda_stream)
        assert grown.data_ptr() != old and plain._ws[key] is grown
        others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
        assert all(y.data_ptr() != old for y in others)
    tp.assert_clean()
