"""Layer normalisation at the far ends of the lengths and row counts it takes, and of the means its rows have."""
import pytest
import torch

from snws import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
U = 2.0 ** -24


@gpu
@pytest.mark.parametrize("rows", [0, 17])
def test_parameter_gradients_of_the_longest_rows(rows):
    """More columns than one launch has threads for: every one of them is written.  x = 0 and eps = 1 make z = 0 and dx the
    centred gradient; dbias is a sum of integers up to 17, exact."""
    C = (1 << 26) + 40
    x = torch.zeros(rows, C, device=DEV, requires_grad=True)
    w, b = (torch.zeros(C, device=DEV, requires_grad=True) for _ in range(2))
    y = ops.layer_norm(x, w, b, 1.0)
    column = (torch.arange(C, device=DEV) % 5 == 0).float()
    dw, db = torch.autograd.grad(y, (w, b), column.expand(rows, C))
    assert dw.shape == db.shape == (C,)
    assert not bool(dw.any())
    assert torch.equal(db, rows * column)
