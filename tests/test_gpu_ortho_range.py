"""Orthogonalisation at the far ends of what it takes: matrices of more than 2^30 numbers, sizes beyond 32 bits, coefficients
that change."""
import math

import pytest
import torch

from snws import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu


def test_sizes_beyond_32_bits_are_refused():
    """A size handed to the library is 32 bits wide: 2^32 + 9 must not arrive there as 9."""
    big = (1 << 32) + 9
    for rows, cols in (([big], [3]), ([3], [big]), ([4, 3], [9, 1 << 31])):
        with pytest.raises(ValueError, match="too many"):
            ops._ortho_bytes(rows, cols, 5)
    with pytest.raises(ValueError, match="larger"):
        ops._ortho_bytes([3], [(1 << 31) - 1], 5)


def test_coefficients_that_change_are_read_again():
    b = torch.tensor(-4.0)
    given = (3.0, b, 2.0)
    assert list(ops._ortho_coefficients(given, 1)) == [3.0, -4.0, 2.0]
    b.fill_(-5.0)
    assert list(ops._ortho_coefficients(given, 1)) == [3.0, -5.0, 2.0]


@gpu
def test_long_matrices_are_refused():
    big = torch.zeros((1 << 32) + 9, 1, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="too many"):
        ops.orthogonalize(big)


@gpu
@pytest.mark.parametrize("rows,cols", [(1025, 1 << 20), (300000, 4096)])
def test_more_numbers_than_a_tile_s_offsets_hold(rows, cols):
    """One step with (0, 1, 0): X X^T X against float64.  A sum of n products has a relative error of at most
    e(n) = (8 + sqrt(n)) 2^-23 of the norms of its two rows (operands of 22 bits, float32 sums), so X X^T is off by at most
    e(n) |X|_F^2 = e(n) in norm, which reaches the result times |X|_2; the second product adds e(m) |A|_F |X|_F, the
    result's own rounding 2^-24 of it.  Two rows that are taken for each other make an element of X X^T that should be
    about 1 / (m sqrt(n)) as large as 1 / m."""
    m, n = min(rows, cols), max(rows, cols)
    gen = torch.Generator(device=DEV).manual_seed(rows)
    g = torch.randn(rows, cols, generator=gen, device=DEV)
    got = ops.orthogonalize(g, steps=1, coefficients=(0.0, 1.0, 0.0))
    assert got.shape == g.shape
    wide = g if rows <= cols else g.t()
    part = 1 << 15
    gram = torch.zeros(m, m, dtype=torch.float64, device=DEV)
    for c in range(0, n, part):
        x = wide[:, c:c + part].double().contiguous()
        gram += x @ x.t().contiguous()
    norm = float(gram.trace()) ** 0.5
    gram /= norm * norm
    power = gram                          # |A|_2 <= |A^8|_F^(1/8)
    for _ in range(3):
        power = power @ power
    largest = float(power.norm()) ** (1 / 16)
    err = size = 0.0
    for c in range(0, n, part):
        want = gram @ (wide[:, c:c + part].double().contiguous() / norm)
        have = (got if rows <= cols else got.t())[:, c:c + part].double()
        err += float((have - want).square().sum())
        size += float(want.square().sum())

    def e(k):
        return (8 + math.sqrt(k)) * 2.0 ** -23
    bound = e(n) * largest + e(m) * float(gram.norm()) + 2.0 ** -24 * math.sqrt(size)
    assert math.sqrt(err) <= bound, (math.sqrt(err), bound, math.sqrt(size))
