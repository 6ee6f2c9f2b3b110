"""artemis_amd.layer_norm over more columns than one launch has workgroups for, in the sums of the parameters' gradients."""
import pytest
import torch

import artemis_amd

DEV = "cuda:0"
U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 2])
def test_gradients_of_more_than_2_25_columns(rows):
    cols = (1 << 25) + 21
    g = torch.Generator(DEV).manual_seed(3)
    x = torch.randn(rows, cols, device=DEV, generator=g)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    w, b = (torch.full((cols,), v, device=DEV, requires_grad=True) for v in (1.0, 0.0))
    y = artemis_amd.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(db, dy.sum(0))                        # (two terms: one rounding, in any order)
    # y is xh; each product is rounded (or not), and the sum
    terms = dy.double() * y.detach().double()
    assert bool(((dw.double() - terms.sum(0)).abs() <= 3 * U * terms.abs().sum(0)).all())
    if rows:
        assert bool((y.double().mean(1).abs() < 1e-3).all()) and bool(((y.double().var(1) - 1).abs() < 1e-3).all())
