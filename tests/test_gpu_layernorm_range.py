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


LENGTHS = [2, 3, 30, 100, 512, 1283, 2049, 9216, 16384, 20000, 300001]


@gpu
@pytest.mark.parametrize("C", LENGTHS)
def test_constant_rows_far_from_zero(C):
    """They give the bias.  The first mean is a float32 sum in a tree of at most 73 roundings, so off by less than 146 half
    steps u with the division's; the corrected one by that share of the distance that is left; rstd is 1 / sqrt(eps)."""
    gen = torch.Generator(device=DEV).manual_seed(C)
    w, b = (torch.randn(C, generator=gen, device=DEV) for _ in range(2))
    for value in (1000.1, -77.7, 30000.3, 0.1):
        x = torch.full((3, C), value, device=DEV)
        slack = 316.3 * abs(value) * (146 * U) ** 2
        y = ops.layer_norm(x, w, b, 1e-5)
        assert bool(((y - b).abs() <= slack * w.abs() + 2 * U * b.abs()).all()), (value, float((y - b).abs().max()))


@gpu
@pytest.mark.parametrize("C", LENGTHS)
def test_rows_far_from_zero(C):
    """The mean's size is not in the bound: an element's distance to it is exact (they lie within a factor of two), its
    correction off by at most 73 roundings of the mean distance, which is at most the spread; rstd by as many.  256 u of z
    and of one covers them and the single roundings behind."""
    gen = torch.Generator(device=DEV).manual_seed(C)
    x = 1e4 * (1 + torch.rand(20, 1, generator=gen, device=DEV)) + torch.randn(20, C, generator=gen, device=DEV)
    w, b = (torch.randn(C, generator=gen, device=DEV) for _ in range(2))
    y = ops.layer_norm(x, w, b, 1e-5)
    xd = x.double()
    z = (xd - xd.mean(1, keepdim=True)) / (xd.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    want = z * w + b
    assert bool(((y - want).abs() <= 256 * U * (z.abs() + 1) * w.abs() + 4 * U * (want.abs() + b.abs())).all()), \
        float((y - want).abs().max())


@gpu
@pytest.mark.parametrize("rows,C,dtype", [(3000, 16640, torch.float32), (2000, 262160, torch.float32), (700, 40001, torch.bfloat16)])
def test_parameter_gradients_of_many_long_rows(rows, C, dtype):
    """Positive terms, so that nothing hides an error: a float32 sum of a thread's rows would be off by up to 50 roundings.
    dbias: a partial sum and the total are rounded once each.  dweight: x lies in [1, 2] with a spread of 0.29, so the mean's
    rounding is 4 half steps of z and the distance to it exact; rstd, the product and the term itself make 6 of z's own."""
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = (1 + torch.rand(rows, C, generator=gen, device=DEV)).to(dtype)
    dy = (0.5 + torch.rand(rows, C, generator=gen, device=DEV)).to(dtype)
    w, b = (torch.ones(C, device=DEV, requires_grad=True) for _ in range(2))
    dw, db = torch.autograd.grad(ops.layer_norm(x, w, b, 1e-5), (w, b), dy)
    want_w, want_b, size = (torch.zeros(C, dtype=torch.float64, device=DEV) for _ in range(3))
    for r in range(0, rows, 100):
        xs, ds = x[r:r + 100].double(), dy[r:r + 100].double()
        z = (xs - xs.mean(1, keepdim=True)) / (xs.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        want_w += (ds * z).sum(0)
        want_b += ds.sum(0)
        size += (ds * (z.abs() + 1)).sum(0)
    assert bool(((db.double() - want_b).abs() <= 2.02 * U * want_b).all()), float(((db.double() - want_b) / want_b).abs().max() / U)
    assert bool(((dw.double() - want_w).abs() <= 8 * U * size).all()), float(((dw.double() - want_w).abs() / size).max() / U)


@gpu
@pytest.mark.parametrize("C", [100, 32768, 40001, 1 << 21, (1 << 22) + 3])
def test_constant_bfloat16_rows_far_from_zero(C):
    """Up to 2^15 such elements add exactly; more of them need the correction as float32 rows do.  The result is rounded once."""
    gen = torch.Generator(device=DEV).manual_seed(C)
    w, b = (torch.randn(C, generator=gen, device=DEV) for _ in range(2))
    for value in (1004.0, -77.5, 30080.0, 25559040.0, 0.1):
        x = torch.full((2, C), value, device=DEV).bfloat16()
        slack = 316.3 * abs(float(x[0, 0])) * (146 * U) ** 2
        y = ops.layer_norm(x, w, b, 1e-5).float()
        assert bool(((y - b).abs() <= 1.01 * (slack * w.abs() + 2.0 ** -8 * b.abs())).all()), (value, float((y - b).abs().max()))


@gpu
def test_rows_beyond_32_bits_are_refused():
    """A length handed to the library is 32 bits wide: 2^32 + 8 must not arrive there as 8.  (Expanded rows: nothing of that size
    is laid out.)"""
    x = torch.zeros(1, 1, device=DEV)
    with pytest.raises(ValueError, match="too long"):
        ops.layer_norm(x.expand(1, (1 << 32) + 8))
    with pytest.raises(ValueError, match="too long"):
        ops.layer_norm(x.expand(1, 1 << 31))
