"""Transforms that the operators have no rules for: an error, never another result."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import artemis_amd

DEV = "cuda:0"


def norm(x):
    return artemis_amd.layer_norm(x, torch.ones(96, device=DEV))


def attention(x):
    return artemis_amd.window_attention(x.reshape(1, 1, 4, 4, 96), None, (1, 4, 4), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [norm, attention])
def test_batching(call):
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(call)(torch.randn(3, 16, 96, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("call", [norm, attention])
def test_derivatives_as_functions(call):
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda x: call(x).sum())(torch.randn(16, 96, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("call", [norm, attention])
def test_forward_mode(call):
    x = torch.randn(16, 96, device=DEV)
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        call(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
def test_an_optimizer_step_in_a_batch():
    t = [torch.zeros(2, 8, device=DEV) for _ in range(4)]

    def step(*one):
        artemis_amd.adamw_step(*([o] for o in one), 1)
        return one[0]

    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(step)(*t)
    assert all((a == 0).all() for a in t)
