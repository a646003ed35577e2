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
# sums.  A lost cross product makes it 5 to 1000 times, a group of five steps 20 to 120 times on spectra that fall off
# (test_what_the_factor_tells_apart).
FACTOR = 4.0
HALF = 2.0 ** -24


def with_spectrum(rows, cols, s, gen, device=DEV):
    m, n = min(rows, cols), max(rows, cols)
    u = torch.linalg.qr(torch.randn(m, m, dtype=torch.float64, generator=gen).to(device))[0]
    v = torch.linalg.qr(torch.randn(n, m, dtype=torch.float64, generator=gen).to(device))[0]
    x = ((u * s.to(device)) @ v.t().contiguous()).float()
    return x if rows <= cols else x.t().contiguous()


def spectra(m):
    t = torch.arange(m, dtype=torch.float64) / m
    return {"exp2": torch.exp(-2 * t), "exp5": torch.exp(-5 * t), "exp12": torch.exp(-12 * t), "power": 1 / (1 + m * t),
            "one": torch.where(t == 0, 1.0, 0.02), "two": torch.where(t < 0.5, 1.0, 0.05)}


def step(x, a, b, c):
    gram = x @ x.t().contiguous()
    return a * x + (b * gram + c * (gram @ gram)) @ x


def forms(g, steps=5, coeff=ops.QUINTIC):
    """(float64, float32) of the definition."""
    out = []
    for dtype in (torch.float64, torch.float32):
        x = g.to(dtype) / g.double().norm().to(dtype)
        flip = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if flip else x
        for _ in range(steps):
            x = step(x, *coeff)
        out.append(x.t() if flip else x)
    return out


def errors(matrices, results, **kw):
    """Error, the plain form's, and size, over the matrices of a kind together: no lucky rounding of one decides."""
    mine = plain = size = 0.0
    for g, got in zip(matrices, results):
        want, other = forms(g, **kw)
        mine += float((got.double() - want).square().sum())
        plain += float((other.double() - want).square().sum())
        size += float(want.square().sum())
    return math.sqrt(mine), math.sqrt(plain), math.sqrt(size)


def compare(matrices, results, what, slack=0.0, **kw):
    mine, plain, size = errors(matrices, results, **kw)
    assert mine <= FACTOR * plain + HALF * size + slack, (what, mine / size, plain / size)


def halves(x, bound):
    """x as the numbers that two halves hold: a power of two that takes `bound` to at most 60000."""
    s = 2.0 ** math.floor(math.log2(60000 / bound))
    x = (x.double() * s).float()
    hi = x.half().float()
    return hi, (x - hi).half().float(), s


def product(p, q, lost):
    """p q^T of halves; `lost` leaves the product of p's low half out."""
    r = p[0] @ q[0].t() + p[0] @ q[1].t()
    return (r if lost else r + p[1] @ q[0].t()).double() / (p[2] * q[2])


def emulated(g, group=1, lost=()):
    """The method in float32 on the CPU, `lost`: among "gram", "square", "apply"."""
    a, b, c = ops.QUINTIC
    X = halves(g.double() / g.double().norm(), 1.0)
    eye, r = torch.eye(g.shape[0], dtype=torch.float64), 1.0
    for k in range(0, 5, group):
        A, Q, most = halves(product(X, X, "gram" in lost), r * r), None, 1.0
        for j in range(min(group, 5 - k)):
            l = torch.linspace(0, r * r, 10001, dtype=torch.float64)
            p = (a + b * l + c * l * l).abs()
            P = halves(a * eye + b * (A[0].double() + A[1]) / A[2] + c * product(A, A, "square" in lost), float(p.max()) * 1.01)
            most *= float(p.max()) * 1.01
            Q = P if Q is None else halves(product(P, Q, False), most)
            PA, r = halves(product(P, A, False), float((l * p).max()) * 1.01), float((l.sqrt() * p).max()) * 1.001
            A = halves(product(P, PA, False), r * r)
        out = product(Q, [t.t() for t in X[:2]] + [X[2]], "apply" in lost)
        X = halves(out, r)
    return out.float()


def test_what_the_factor_tells_apart():
    """The method as it is passes; without one cross product, or with all steps in one group, it does not."""
    gen = torch.Generator().manual_seed(3)
    for kind, s in spectra(48).items():
        mats = [with_spectrum(48, 300, s, gen, "cpu") for _ in range(3)]
        mine, plain, size = errors(mats, [emulated(g) for g in mats])
        assert mine <= FACTOR * plain + HALF * size, (kind, mine / size, plain / size)
        for lost in ("gram", "square", "apply"):
            mine, plain, size = errors(mats, [emulated(g, lost=(lost,)) for g in mats])
            assert mine > 1.5 * (FACTOR * plain + HALF * size), (kind, lost, mine / size, plain / size)
        if kind in ("exp5", "exp12"):
            mine, plain, size = errors(mats, [emulated(g, group=5) for g in mats])
            assert mine > 1.5 * (FACTOR * plain + HALF * size), (kind, mine / size, plain / size)


SIZES = [(3, 9), (8, 72), (16, 36), (324, 36), (64, 64), (64, 126), (60, 500), (64, 576), (72, 400), (300, 100), (127, 600),
         (128, 300), (257, 1030), (320, 700), (1100, 512), (1024, 2300), (64, 9216), (9216, 512)]


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


@gpu
@pytest.mark.parametrize("coeff", [(1.5, 0.0, -0.5), (1.5, -0.5, 0.0), (0.0, 0.0, 1.0), (0.0, 1.0, 0.0), (-1.2, 0.4, 0.0)])
@pytest.mark.parametrize("rows,cols", [(60, 300), (60, 700), (100, 300), (300, 1000), (1409, 3000), (2790, 2800)])
def test_coefficients_that_vanish_beside_the_plain_form(rows, cols, coeff):
    """In one launch, in few rows, and on each tile of the m x m products: 64 x 64, 96 x 64 (1409 rows, in threes) and 128 x 128
    (2790 rows).  Each of the steps adds the absolute rounding of what is stored, at most 2^-39 per number.  And where a is not
    zero, a X is part of the sum that makes P X, and outweighs the rest of it for these matrices: each of the 3 m / 32
    instructions rounds a sum of its size, by a step of 2^-23 at most, the operands, the stored number and the result by
    another four; the plain form adds a X once.  (The next steps do not enlarge a relative error: all singular values are
    below 0.2, where |s p'(s)| <= |p(s)|.)"""
    gen = torch.Generator().manual_seed(rows)
    g = torch.randn(rows, cols, generator=gen).to(DEV)
    got = ops.orthogonalize(g, steps=3, coefficients=coeff)
    slack = 3 * 1.5 ** 2 * 2.0 ** -39 * math.sqrt(rows * cols)
    if coeff[0]:
        size = float(forms(g, 3, coeff)[0].norm())
        slack += 3 * (3 * math.ceil(rows / 32) + 4) * 2.0 ** -23 * size
    compare([g], [got], coeff, slack=slack, steps=3, coeff=coeff)


@gpu
def test_a_list_in_two_runs():
    """Long matrices whose steps go in threes beside small ones: each as accurate as alone, eager and from a captured call that
    is replayed with other values between eager calls."""
    gen = torch.Generator().manual_seed(8)
    mats = [torch.randn(s, generator=gen).to(DEV) for s in ((64, 126), (1024, 4608), (90, 70), (1, 9), (4000, 700))]
    out = ops.orthogonalize(mats)
    for g, o in zip(mats, out):
        compare([g], [o], tuple(g.shape))
    assert all(torch.equal(p, q) for p, q in zip(out, ops.orthogonalize(mats)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = ops.orthogonalize(mats)
    for it in range(3):
        for g in mats:
            g.copy_(torch.randn(g.shape, generator=gen).to(DEV))
        want = ops.orthogonalize(mats)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, want)), it
