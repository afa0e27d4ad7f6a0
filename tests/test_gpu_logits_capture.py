"""Inputs on the host are refused while a call is recorded into a graph, which then replays as if they had not come."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from numba_cuda_amd import logits


def test_host_inputs_are_refused_and_the_recording_goes_on():
    torch = pytest.importorskip("torch")
    x = torch.zeros(3, 5001, device="cuda")
    y = torch.empty_like(x)
    tokens = torch.tensor([1, 2, 2, 4999, 7], device="cuda", dtype=torch.int32)
    offsets = torch.tensor([0, 3, 3, 5], device="cuda")

    def call(stream, **kw):
        logits.adjust(x, y, stream=stream, **{**dict(tokens=tokens, offsets=offsets, repetition=2.0, presence=0.5), **kw})

    call(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        stream = cuda.external_stream(torch.cuda.current_stream().cuda_stream)
        for kw in (dict(tokens=[1, 2, 3, 4, 5]), dict(offsets=np.array([0, 1, 2, 3])), dict(presence=[1.0, 2.0, 3.0]),
                   dict(mask=np.zeros(157, np.uint32))):
            with pytest.raises(ValueError, match="captured into a graph needs %s in device memory" % next(iter(kw))):
                call(stream, **kw)
        call(stream)
    for n in range(4):
        x.copy_(torch.randn(3, 5001, device="cuda") * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        recorded = y.clone()
        y.zero_()
        call(0)
        torch.cuda.synchronize()
        assert torch.equal(y, recorded)
