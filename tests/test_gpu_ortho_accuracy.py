"""How accurate orthogonalisation and the Muon update are: their error against float64 beside that of the plain form, single
steps with float32 products, on the same matrices."""
import math

import pytest
import torch

from snws import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
# A product here rounds each operand to 22 bits and leaves out lo * lo: in the mean (root of the mean square) 2^-23 / sqrt(3) of
# a term twice and 2^-22 / 3, together 1.05 * 2^-23.  A float32 product rounds each partial sum, 2^-24 / sqrt(3) if there is
# one and more if there are many.  So this one's error is up to 1.05 * 2 * sqrt(3) = 3.7 times that one's, and less for longer
# sums.  A lost cross product makes it 40 times and more, a group of five steps 20 to 120 times on the spectra that fall off.
FACTOR = 4.0
HALF = 2.0 ** -24


def with_spectrum(rows, cols, s, gen):
    m, n = min(rows, cols), max(rows, cols)
    u = torch.linalg.qr(torch.randn(m, m, dtype=torch.float64, generator=gen))[0]
    v = torch.linalg.qr(torch.randn(n, m, dtype=torch.float64, generator=gen))[0]
    x = ((u * s) @ v.t()).float().to(DEV)
    return x if rows <= cols else x.t().contiguous()


def spectra(m):
    t = torch.arange(m, dtype=torch.float64) / m
    return {"exp2": torch.exp(-2 * t), "exp5": torch.exp(-5 * t), "exp12": torch.exp(-12 * t), "power": 1 / (1 + m * t),
            "one": torch.where(t == 0, 1.0, 0.02), "two": torch.where(t < 0.5, 1.0, 0.05)}


def step(x, a, b, c):
    gram = x @ x.t().contiguous()
    return a * x + (b * gram + c * (gram @ gram)) @ x


def forms(g):
    """(float64, float32) of the definition."""
    out = []
    for dtype in (torch.float64, torch.float32):
        x = g.to(dtype) / g.double().norm().to(dtype)
        flip = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if flip else x
        for _ in range(5):
            x = step(x, *ops.QUINTIC)
        out.append(x.t() if flip else x)
    return out


def compare(matrices, results, what):
    """Over the matrices of a kind together, so that no lucky rounding of one decides."""
    mine = plain = size = 0.0
    for g, got in zip(matrices, results):
        want, other = forms(g)
        mine += float((got.double() - want).square().sum())
        plain += float((other.double() - want).square().sum())
        size += float(want.square().sum())
    assert math.sqrt(mine) <= FACTOR * math.sqrt(plain) + HALF * math.sqrt(size), (what, math.sqrt(mine / size), math.sqrt(plain / size))


SIZES = [(3, 9), (8, 72), (16, 36), (324, 36), (64, 64), (64, 126), (60, 500), (64, 576), (72, 400), (300, 100), (127, 600),
         (128, 300), (257, 1030), (320, 700), (1100, 512), (1024, 2300)]


@gpu
@pytest.mark.parametrize("rows,cols", SIZES)
def test_error_beside_the_plain_form_s(rows, cols):
    gen = torch.Generator().manual_seed(rows * 1009 + cols)
    kinds = {k: [with_spectrum(rows, cols, s, gen) for _ in range(4 if rows * cols < 1 << 18 else 2)]
             for k, s in spectra(min(rows, cols)).items()}
    kinds["even"] = [torch.randn(rows, cols, generator=gen).to(DEV) for _ in range(4)]
    for kind, mats in kinds.items():
        compare(mats, [ops.orthogonalize(g) for g in mats], kind)
    together = [mats[0] for mats in kinds.values()]
    compare(together, ops.orthogonalize(together), "together")


@gpu
@pytest.mark.parametrize("kind", ["exp5", "one", "two"])
def test_update_s_error_beside_the_plain_form_s(kind):
    """From zero parameters and momenta and without decay an update is the orthogonalised gradient: small filters and long
    ones, in one list."""
    gen = torch.Generator().manual_seed(5)
    for shapes in ([(4, 126), (8, 36), (16, 144), (32, 288), (64, 576)], [(8, 72), (64, 576), (128, 576), (256, 1152)]):
        sets = [[with_spectrum(r, c, spectra(min(r, c))[kind], gen) for r, c in shapes] for _ in range(4)]
        outs = []
        for grads in sets:
            params, bufs = ([torch.zeros_like(g) for g in grads] for _ in range(2))
            ops.muon_update(params, grads, bufs, lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False, adjust_lr="original")
            outs.append([-p for p in params])
        for i, shape in enumerate(shapes):
            compare([s[i] for s in sets], [o[i] for o in outs], shape)
