"""A backward pass captured beside an eager graph of its leaves, where the operators copy a leaf first: a parameter of 16 bits,
which is widened, an input that is not aligned, which is moved."""
import pytest
import torch

import artemis_amd
from artemis_amd import _lib


def test_a_leaf_is_found_behind_copies():
    has = _lib.load_ops_host().has_leaf
    w = torch.ones(8, dtype=torch.bfloat16, requires_grad=True)
    assert has(w) and has(w.float()) and has(w.clone()) and has(w.float().clone().double())
    assert not has(w.detach()) and not has(w.detach().float())
    assert not has(w * 2) and not has(w.float() + w)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["widened weight", "widened table", "moved input"])
def test_refused_behind_a_copy(case):
    g = torch.Generator().manual_seed(37)
    x = torch.randn(1, 1, 8, 8, 96, generator=g).cuda()
    if case == "moved input":
        flat = torch.randn(x.numel() + 1, generator=g).cuda()
        leaf = flat[1:].view(x.shape).requires_grad_(True)
        assert leaf.data_ptr() % 16 == 4
    else:
        shape = (96,) if case == "widened weight" else (225, 1)
        leaf = torch.randn(shape, generator=g).bfloat16().cuda().requires_grad_(True)

    def call():
        if case == "widened weight":
            return artemis_amd.layer_norm(x, leaf)
        return artemis_amd.window_attention(*((leaf, None) if case == "moved input" else (x, leaf)), (1, 8, 8), 1)

    def step():
        out = call()
        return (out, *torch.autograd.grad(out, leaf, torch.ones_like(out)))

    want = [t.detach().clone() for t in step()]
    alive = call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="being captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        again = step()
        torch.cuda.synchronize()
        assert torch.equal(again[1], want[1])
        del again
