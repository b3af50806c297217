"""A handle that the garbage collector finds while a graph is being captured does not end the capture, and is destroyed later."""
import gc

import pytest
import torch

from aidotnet.tensors_b200 import native as N

pytestmark = pytest.mark.gpu


def test_collected_during_a_capture():
    def cycle():
        h = N.Handle(device=0, qkv_dtype=N.BF16, head_dim=64, num_q_heads=1)
        h.itself = h

    x = torch.zeros(4, device="cuda")
    side = torch.cuda.Stream()
    gc.collect()
    cycle()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cycles = gc.collect()
        x += 1
    assert cycles > 0 or N._left
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 4
    N.Handle(device=0, qkv_dtype=N.BF16, head_dim=64, num_q_heads=1).close()
    assert not N._left
