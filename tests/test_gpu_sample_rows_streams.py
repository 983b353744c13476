"""Sampling on streams beside one another: calls are in flight together, in front of one
synchronisation at the end."""
import ctypes as C

import pytest
import torch

from tensoros_b200 import _ffi

pytestmark = pytest.mark.gpu


def outputs(n):
    return (torch.full((n,), -77, dtype=torch.int32, device="cuda"), torch.full((n,), -7.0, device="cuda"),
            torch.full((n,), -77, dtype=torch.int32, device="cuda"))


class Batch:
    def __init__(self, rows, n, seed, k, p, m):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.x = torch.randn(rows, n, generator=g, device="cuda")
        self.u = torch.rand(rows, generator=g, device="cuda")
        self.t = torch.linspace(0.0, 1.5, rows, device="cuda")
        self.k = torch.full((rows,), k, dtype=torch.int32, device="cuda")
        self.p, self.m = torch.full((rows,), p, device="cuda"), torch.full((rows,), m, device="cuda")

    def call(self, gpu, out, stream):
        r = _ffi.Rows(self.x.data_ptr(), self.x.stride(0), 0)
        s = _ffi.SampleParams(*(t.data_ptr() for t in (self.t, self.k, self.p, self.m)))
        return gpu.tos_sample_rows_dev(C.byref(r), self.x.shape[0], self.x.shape[1], C.byref(s), self.u.data_ptr(),
                                       *(t.data_ptr() for t in out), stream)


@pytest.mark.parametrize("captured", [False, True])
def test_calls_in_flight_together(gpu, captured):
    """Different batches, cluster sizes and filters on four streams, ten calls each,
    launched or replayed without a wait in between: each gives what it gives alone."""
    batches = [Batch(5, 60000, 1, 0, 0.97, 0.0), Batch(40, 32000, 2, 50, 0.9, 0.0), Batch(90, 9000, 3, 3000, 1.0, 0.01),
               Batch(3, 1 << 18, 4, 100000, 0.5, 0.0)]
    want, got = [], [[outputs(b.x.shape[0]) for _ in range(10)] for b in batches]
    for b in batches:
        o = outputs(b.x.shape[0])
        assert b.call(gpu, o, torch.cuda.current_stream().cuda_stream or 1) == 0
        torch.cuda.synchronize()
        want.append(o)
        assert bool((o[0] >= 0).all())
    streams = [torch.cuda.Stream() for _ in batches]
    graphs = []
    if captured:
        for b, outs in zip(batches, got):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                for o in outs:
                    assert b.call(gpu, o, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    if captured:
        for _ in range(3):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
    else:
        for i in range(10):
            for b, st, outs in zip(batches, streams, got):
                assert b.call(gpu, outs[i], st.cuda_stream) == 0
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(w, o))
