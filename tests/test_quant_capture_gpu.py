"""Decode attention over quantised pools, captured into CUDA graphs by other means than torch.cuda.graph: scratch comes from torch's
allocator, which knows nothing of such a capture and would give it to others once the call has returned."""
import ctypes
import gc

import pytest
import torch

import quant_helpers as qh
from test_quant_paged_gpu import ib, problem  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


class Graph:
    """What calls() launches on `stream`, captured through the infinirt calls."""

    def __init__(self, stream, calls):
        from infinicore_b200.libinfiniop import LIBINFINIOP as L
        from infinicore_b200.libinfiniop import InfiniDeviceEnum, check_error

        self.L, self.check, self.stream = L, check_error, stream
        check_error(L.infinirtSetDevice(InfiniDeviceEnum.NVIDIA, 0))
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        check_error(L.infinirtStreamBeginCapture(stream.cuda_stream, 2))
        with torch.cuda.stream(stream):
            calls()
        check_error(L.infinirtStreamEndCapture(stream.cuda_stream, ctypes.byref(graph)))
        check_error(L.infinirtGraphInstantiate(ctypes.byref(self.exec), graph, None, None, 0))
        check_error(L.infinirtGraphDestroy(graph))  # the instance holds what it needs

    def replay(self, stream=None):
        self.check(self.L.infinirtGraphLuanch(self.exec, (stream or self.stream).cuda_stream))

    def destroy(self):
        self.check(self.L.infinirtGraphExecDestroy(self.exec))


def call(ib, p, out):  # noqa: F811
    ib.quant_paged_attention(p[0], *p[1], p[2], p[3], None, 0.09, out=out)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_replayed_graph_touches_no_memory_that_torch_gives_to_others(ib, bits):  # noqa: F811
    g = torch.Generator().manual_seed(71)
    p = problem(g, bits, [9000, 700, 16], heads=16)
    out = torch.zeros_like(p[0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(ib, p, out)
    torch.cuda.synchronize()
    graph = Graph(stream, lambda: call(ib, p, out))
    # everything that the allocator has free on that stream
    with torch.cuda.stream(stream):
        others = [torch.full((n << 10,), 0x5A, dtype=torch.uint8, device="cuda") for n in (64, 256, 700, 1 << 10, 3 << 10, 8 << 10) for _ in range(16)]
        out.zero_()
        for _ in range(3):
            graph.replay()
    torch.cuda.synchronize()
    assert all(bool((t == 0x5A).all()) for t in others)
    qh.close(out, p[4], p[5])
    with torch.cuda.stream(stream):
        for t in others:
            t.fill_(0xFF)
        graph.replay()
    torch.cuda.synchronize()
    qh.close(out, p[4], p[5])
    graph.destroy()


def test_two_graphs_of_one_stream_at_once_and_both_kinds_of_capture(ib):  # noqa: F811
    g = torch.Generator().manual_seed(72)
    a, b = problem(g, 4, [9000, 700]), problem(g, 8, [5, 8000, 300], heads=16)
    s1, s2, s3 = (torch.cuda.Stream() for _ in range(3))
    outs = [torch.zeros_like(x[0]) for x in (a, b, a)]
    torch.cuda.synchronize()
    for x, o in ((a, outs[0]), (b, outs[1])):
        with torch.cuda.stream(s1):
            call(ib, x, o)
    torch.cuda.synchronize()
    graphs = [Graph(s1, lambda x=x, o=o: (call(ib, x, o), call(ib, x, o))) for x, o in ((a, outs[0]), (b, outs[1]))]
    third = torch.cuda.CUDAGraph()
    with torch.cuda.graph(third, stream=s1):
        call(ib, a, outs[2])
    for _ in range(20):
        graphs[0].replay(s1)
        graphs[1].replay(s2)
        with torch.cuda.stream(s3):
            third.replay()
    torch.cuda.synchronize()
    for x, o in ((a, outs[0]), (b, outs[1]), (a, outs[2])):
        qh.close(o, x[4], x[5])
    for graph in graphs:
        graph.destroy()


def test_scratch_of_destroyed_graphs_goes_back(ib):  # noqa: F811
    """Many graphs, captured and destroyed one after the other, hold no more memory than a few do."""
    g = torch.Generator().manual_seed(73)
    p = problem(g, 4, [9000, 700], heads=16)
    out = torch.zeros_like(p[0])
    stream = torch.cuda.Stream()

    def one():
        graph = Graph(stream, lambda: call(ib, p, out))
        graph.replay()
        torch.cuda.synchronize()
        graph.destroy()
        with torch.cuda.stream(stream):
            call(ib, p, out)
        torch.cuda.synchronize()

    for _ in range(5):
        one()
    gc.collect()
    before = torch.cuda.memory_allocated()
    for _ in range(40):
        one()
    assert torch.cuda.memory_allocated() <= before + (64 << 20)  # the buffers of a few graphs that are not taken back yet
    qh.close(out, p[4], p[5])
