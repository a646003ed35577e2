"""Orthogonalisation by Newton-Schulz products and the Muon update (snws.ops.orthogonalize, snws.ops.muon_update) against
their definitions in float64: shapes, strides, types, special values, refusals, streams and captured graphs."""
import ctypes
import math

import pytest
import torch

from snws import _lib as L
from snws import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
A0 = ops.QUINTIC[0]


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refuses_cpu_tensors_and_bad_arguments():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.orthogonalize(torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.orthogonalize([torch.zeros(2, 3)])
    with pytest.raises(ValueError, match="matrices"):
        ops.orthogonalize(torch.zeros(3))
    with pytest.raises(ValueError, match="step"):
        ops.orthogonalize([], steps=0)
    with pytest.raises(ValueError, match="three"):
        ops.orthogonalize([], steps=2, coefficients=[(1.0, 2.0, 3.0)])
    with pytest.raises(ValueError, match="three"):
        ops.orthogonalize([], coefficients=(1.0, 2.0))
    assert ops.orthogonalize([]) == []
    p = torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.muon_update([p], [p.clone()], [p.clone()], lr=0.1)
    with pytest.raises(ValueError, match="1 parameters, 0 gradients"):
        ops.muon_update([p], [], [p], lr=0.1)
    with pytest.raises(ValueError, match="adjust_lr"):
        ops.muon_update([], [], [], lr=0.1, adjust_lr="other")
    assert ops.muon_lr_factor(None, 8, 2) == 2.0 and ops.muon_lr_factor("original", 2, 8) == 1.0
    assert ops.muon_lr_factor("match_rms_adamw", 4, 100) == 2.0


def test_entry_points_refuse_bad_arguments():
    P = 4096        # never dereferenced: every refusal comes before a launch
    coeff = (ctypes.c_float * 3)(*ops.QUINTIC)
    n = L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(4), (ctypes.c_int * 1)(9), 1, 1)
    assert n > 0
    assert L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(0), (ctypes.c_int * 1)(9), 1, 1) == -1
    assert L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(4), (ctypes.c_int * 1)((1 << 20) + 1), 1, 1) == -1
    assert L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(40000), (ctypes.c_int * 1)(40000), 1, 1) == -1
    assert L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(4), (ctypes.c_int * 1)(9), L.ORTHO_MAX + 1, 1) == -1

    assert L.lib().snws_ortho_workspace_bytes((ctypes.c_int * 1)(4), (ctypes.c_int * 1)(9), 1, 33) == -1

    def item(**kw):
        d = dict(x=P, out=P, ldx=9, ldo=9, rows=4, cols=9)
        d.update(kw)
        return (L.OrthoItem * 1)(L.OrthoItem(**d))
    good = [item(), 1, L.SNWS_F32, coeff, 1, 1e-7, P, n, None]
    nan = (ctypes.c_float * 3)(float("nan"), 0, 0)
    for at, value, text in ((0, None, "matrices"), (1, 0, "matrices"), (1, L.ORTHO_MAX + 1, "matrices"), (2, L.SNWS_F64, "dtype"),
                            (3, None, "steps"), (4, 0, "steps"), (4, 33, "steps"), (5, -1.0, "eps"), (5, math.inf, "eps"),
                            (6, None, "workspace"), (6, P + 8, "workspace"), (7, n - 1, "workspace"), (0, item(x=None), "NULL"),
                            (0, item(out=None), "NULL"), (0, item(ldx=8), "strides"), (0, item(ldo=8), "strides"),
                            (0, item(rows=0), "at least one"), (0, item(cols=1 << 21), "larger"), (3, nan, "grow"),
                            (3, (ctypes.c_float * 3)(2000.0, 0, 0), "grow")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=text):
            L.call("snws_orthogonalize", *args)

    def mitem(**kw):
        d = dict(param=P, grad=P, momentum=P, rows=4, cols=9, lr=0.1)
        d.update(kw)
        return (L.MuonItem * 1)(L.MuonItem(**d))
    good = [mitem(), 1, 0.95, 1, 1.0, 0.0, coeff, 1, 1e-7, P, n, None]
    for at, value, text in ((0, None, "matrices"), (1, 0, "matrices"), (2, 1.5, "momentum"), (2, -0.1, "momentum"),
                            (2, math.nan, "momentum"), (6, None, "steps"), (8, math.nan, "eps"), (9, None, "workspace"),
                            (10, 0, "workspace"), (0, mitem(param=None), "NULL"), (0, mitem(grad=None), "NULL"),
                            (0, mitem(momentum=None), "NULL"), (0, mitem(rows=-1), "at least one")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=text):
            L.call("snws_muon_update", *args)


def test_calls_hold_the_largest_first():
    parts = ops._by_size([i % 7 for i in range(70)])
    assert [len(p) for p in parts] == [32, 32, 6] and sorted(sum(parts, [])) == list(range(70))
    assert parts[0][0] % 7 == 6 and parts[-1][-1] % 7 == 0


# ------------------------------------------------------------------------------------------------ values (GPU)
def definition(g, steps=5, coeff=ops.QUINTIC, eps=1e-7):
    """float64: the result and a bound on the error of float32-accurate products.  A step's products have a relative error
    (in norm) of at most eps_k = (8 + sqrt(K)) 2^-23: both operands rounded to 22 bits, the dropped product of the low
    halves, float32 sums over K terms; later steps multiply an error by at most the polynomial's slope at zero.  A stored
    number is x times at least 2^14, and the low half's own smallest step is 2^-24: an absolute error of at most 2^-39 per
    number, 2^-39 sqrt(m n) in norm, which counts only where |G| is far below eps (|X| <= 1.2 by the coefficients used)."""
    x = g.detach().double()
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x.contiguous()
    rows = [coeff] * steps if not hasattr(coeff[0], "__len__") else coeff
    x = x / x.norm().clamp(min=eps)
    bound = 0.0
    for a, b, c in rows:
        bound = bound * max(abs(a), 1.0) + (8 + math.sqrt(x.shape[1])) * 2.0 ** -23 * max(abs(a), 1.0) * float(x.norm())
        bound += 2.0 ** -39 * math.sqrt(x.numel()) * max(abs(a), 1.0)
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.t() if flip else x), bound


def check(got, g, **kw):
    ref, bound = definition(g, **kw)
    assert got.dtype == g.dtype and got.shape == g.shape and got.is_contiguous()
    half = torch.finfo(g.dtype).eps / 2
    err = float((got.double() - ref).norm())
    assert err <= bound + half * float(ref.norm()) * 1.01, (err, bound, float(ref.norm()))


def matrix(rows, cols, seed=0, rank=None, pad=0, dtype=torch.float32, scale=1e-3):
    gen = torch.Generator(device=DEV).manual_seed(seed + rows * 1009 + cols)
    k = rank or max(1, min(rows, cols) // 4)
    w = torch.randn(rows, k, generator=gen, device=DEV) @ torch.randn(k, cols + pad, generator=gen, device=DEV)
    w = w if rank else w + torch.randn(rows, cols + pad, generator=gen, device=DEV)
    return (w * scale).to(dtype)[:, :cols]


SHAPES = [(1, 1), (1, 7), (5, 1), (2, 3), (7, 7), (31, 33), (32, 32), (33, 31), (64, 126), (64, 64), (65, 64), (126, 64), (100, 1000),
          (129, 127), (128, 300), (200, 500), (513, 90), (64, 9216), (257, 1030), (320, 2880), (640, 640), (1030, 515)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize_shapes(rows, cols, dtype):
    g = matrix(rows, cols, dtype=dtype, pad=(rows * 7 + cols) % 3)
    before = g.clone()
    got = ops.orthogonalize(g)
    check(got, g)
    assert torch.equal(g, before)
    assert torch.equal(ops.orthogonalize(g), got)


@gpu
@pytest.mark.parametrize("rows,cols", [(2048, 2100), (1024, 9216), (3000, 400)])
def test_orthogonalize_large(rows, cols):
    g = matrix(rows, cols)
    check(ops.orthogonalize(g), g)


@gpu
@pytest.mark.parametrize("rank", [1, 3, 17])
def test_orthogonalize_low_rank(rank):
    """Directions that the matrix lacks must not come up: the result's norm is that of `rank` singular values near one."""
    g = matrix(96, 200, rank=rank)
    got = ops.orthogonalize(g)
    check(got, g)
    assert float(got.norm()) <= 1.25 * math.sqrt(rank) + 0.05


@gpu
def test_orthogonalize_lists_batches_and_views():
    mats = [matrix(r, c, seed=i) for i, (r, c) in enumerate([(3, 5), (64, 126), (200, 40), (1, 1), (130, 1200), (16, 16)])]
    mats.insert(2, torch.zeros(0, 4, device=DEV))
    outs = ops.orthogonalize(mats)
    for g, o in zip(mats, outs):
        assert o.shape == g.shape
        if g.numel():
            check(o, g)
    many = [matrix(5 + i, 9 + (i * 7) % 30, seed=i) for i in range(L.ORTHO_MAX + 5)]
    for g, o in zip(many, ops.orthogonalize(tuple(many))):
        check(o, g)
    batch = torch.stack([matrix(12, 20, seed=s) for s in range(6)]).view(2, 3, 12, 20)
    got = ops.orthogonalize(batch)
    assert got.shape == batch.shape
    for i in range(2):
        for j in range(3):
            check(got[i, j], batch[i, j])
    assert ops.orthogonalize(batch[:0]).shape == (0, 3, 12, 20)
    wide = matrix(40, 90)
    check(ops.orthogonalize(wide.t()), wide.t())
    check(ops.orthogonalize(wide[::2, 3:50]), wide[::2, 3:50])
    check(ops.orthogonalize(wide[:, ::3]), wide[:, ::3])
    with pytest.raises(ValueError, match="one type"):
        ops.orthogonalize([wide, wide.bfloat16()])
    with pytest.raises(TypeError):
        ops.orthogonalize(wide.double())


@gpu
def test_orthogonalize_steps_and_coefficients():
    g = matrix(48, 100)
    for steps in (1, 2, 7):
        check(ops.orthogonalize(g, steps=steps), g, steps=steps)
    cubic = (1.5, -0.5, 0.0)
    check(ops.orthogonalize(g, steps=12, coefficients=cubic), g, steps=12, coeff=cubic)
    per_step = [(3.4445, -4.775, 2.0315), (2.8, -3.2, 1.3), (1.875, -1.25, 0.375)]
    check(ops.orthogonalize(g, steps=3, coefficients=per_step), g, steps=3, coeff=per_step)
    with pytest.raises(ValueError, match="grow"):
        ops.orthogonalize(g, coefficients=(50.0, 0.0, 0.0))


@gpu
def test_orthogonalize_special_values():
    zero = torch.zeros(20, 50, device=DEV)
    bad = matrix(40, 70)
    bad[3, 5] = float("nan")
    inf = matrix(40, 70, seed=1)
    inf[39, 0] = float("-inf")
    fine = matrix(40, 70, seed=2)
    oz, ob, oi, of = ops.orthogonalize([zero, bad, inf, fine])
    assert float(oz.abs().max()) == 0.0
    assert bool(torch.isnan(ob).all()) and bool(torch.isnan(oi).all())
    assert torch.equal(of, ops.orthogonalize(fine))
    for scale in (1e-30, 1e-10, 1e15, 1e35):          # squares leave float32's range
        g = matrix(30, 64, scale=1.0) * scale
        check(ops.orthogonalize(g, eps=0.0), g, eps=0.0)
    g = matrix(30, 64, scale=1e-12)
    check(ops.orthogonalize(g, eps=1e-3), g, eps=1e-3)
    one = torch.zeros(33, 77, device=DEV)
    one[32, 76] = -5.0
    check(ops.orthogonalize(one), one)


def muon_definition(p, g, m, lr, wd, mu, nesterov, adjust, scale=1.0, **kw):
    p, g, m = p.double(), g.double() * scale, m.double()
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    rows = p.shape[0]
    o, bound = definition(u.reshape(rows, -1), **kw)
    f = ops.muon_lr_factor(adjust, rows, p[0].numel())
    return p * (1 - lr * wd) - lr * f * o.reshape(p.shape), m, lr * f * bound


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
def test_muon_update(nesterov, adjust):
    shapes = [(10, 3, 3, 3), (64, 14, 3, 3), (1, 9), (9, 1), (130, 60, 1, 1), (33, 200), (4, 0)]
    gen = torch.Generator(device=DEV).manual_seed(4)
    params = [torch.randn(s, generator=gen, device=DEV) for s in shapes]
    grads = [torch.randn(s, generator=gen, device=DEV) * 1e-2 for s in shapes]
    bufs = [torch.randn(s, generator=gen, device=DEV) * 1e-2 for s in shapes]
    grads[5] = grads[5].t().contiguous().t()             # a gradient of other strides
    kw = dict(lr=0.05, weight_decay=0.2, momentum=0.9, nesterov=nesterov, adjust_lr=adjust, grad_scale=0.5)
    want = [muon_definition(p, g, m, 0.05, 0.2, 0.9, nesterov, adjust, 0.5) if p.numel() else None
            for p, g, m in zip(params, grads, bufs)]
    epoch = ops.WEIGHT_EPOCH
    ops.muon_update(params, grads, bufs, **kw)
    assert ops.WEIGHT_EPOCH == epoch + 1
    u = 2.0 ** -24
    for p, m, w in zip(params, bufs, want):
        if w is None:
            continue
        # the momentum: three roundings; they reach the update as a relative error of the matrix, times the slope a^5
        assert float((m.double() - w[1]).norm()) <= 4 * u * float(w[1].norm()) + 4 * u * 1e-2 * math.sqrt(m.numel())
        f = ops.muon_lr_factor(adjust, p.shape[0], p[0].numel())
        slack = w[2] + 0.05 * f * 8 * u * A0 ** 5 + 4 * u * float(w[0].norm() + 1)
        assert float((p.double() - w[0]).norm()) <= slack, p.shape
    p, g, m = params[0], grads[0], bufs[0]
    with pytest.raises(ValueError, match="twice"):
        ops.muon_update([p, p], [g, g], [m, m.clone()], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        ops.muon_update([p], [g], [p], lr=0.1)
    with pytest.raises(ValueError, match="shape"):
        ops.muon_update([p], [g[:5]], [m], lr=0.1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.muon_update([params[5].t()], [grads[5].t()], [bufs[5].t()], lr=0.1)
    with pytest.raises(TypeError):
        ops.muon_update([p], [g.bfloat16()], [m], lr=0.1)
    with pytest.raises(ValueError, match="axes"):
        ops.muon_update([p.view(-1)], [g.view(-1)], [m.view(-1)], lr=0.1)


@gpu
def test_ortho_on_other_streams_and_in_graphs():
    """Two captured graphs and eager calls in between, on streams of their own, keep apart (each call has a workspace)."""
    sets = [[matrix(64, 126, seed=s), matrix(150, 700, seed=s), matrix(40, 9, seed=s)] for s in (1, 2)]
    side = torch.cuda.Stream()
    for mats in sets:
        want = ops.orthogonalize(mats)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = ops.orthogonalize(mats)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs, outs = [], []
    for mats in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(ops.orthogonalize(mats))
        graphs.append(g)
    base = [[m.clone() for m in mats] for mats in sets]
    for it in range(4):
        for mats, b in zip(sets, base):
            for m, v in zip(mats, b):
                m.copy_(v + 1e-3 * it * v.flip(0))
        want = [ops.orthogonalize(mats) for mats in sets]
        graphs[0].replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            graphs[1].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w)), it


@gpu
@pytest.mark.parametrize("coeff", [(1.5, 0.0, -0.5), (1.5, -0.5, 0.0), (0.0, 0.0, 1.0), (0.0, 1.0, 0.0), (-1.2, 0.4, 0.0)])
@pytest.mark.parametrize("rows,cols", [(40, 90), (60, 500), (100, 300), (150, 700), (150, 160)])
def test_coefficients_that_vanish(rows, cols, coeff):
    """Zero coefficients in each way a call is run: one launch, chains of 64 and 128 rows, a launch for every product.
    The bound: a step's three products in a row (A, A^2, B X) have an error of (8 + sqrt(n)) 2^-23 each, relative to
    |a| + |b| r^2 + |c| r^4 times |X|, r the largest singular value; an error that is there grows by at most the largest
    slope |a + 3 b s^2 + 5 c s^4| over [0, r] (an odd function of the singular values); stored numbers: see definition()."""
    g = matrix(rows, cols)
    a, b, c = coeff
    x = g.double().cpu()
    x = x / x.norm()
    bound = 0.0
    for _ in range(5):
        r = float(torch.linalg.matrix_norm(x, 2))
        s = torch.linspace(0.0, r * 1.01, 1001, dtype=torch.float64)
        slope = float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max())
        size = abs(a) + abs(b) * r ** 2 + abs(c) * r ** 4
        bound = bound * slope + 3 * (8 + math.sqrt(cols)) * 2.0 ** -23 * size * float(x.norm())
        bound += 2.0 ** -39 * math.sqrt(x.numel()) * max(size, 1.0)
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    got = ops.orthogonalize(g, coefficients=coeff).double().cpu()
    assert float((got - x).norm()) <= bound + 2.0 ** -24 * 1.01 * float(x.norm()), (float((got - x).norm()), bound)


@gpu
def test_orthogonalize_tiny_matrices_without_eps():
    """Norms whose inverse leaves float32, in both ways a matrix is read."""
    for rows, cols in ((30, 64), (64, 30), (70, 200), (200, 70)):
        for scale in (1e-36, 2e-39):
            g = matrix(rows, cols, scale=1.0) * scale
            check(ops.orthogonalize(g, eps=0.0), g, eps=0.0)


@gpu
def test_muon_update_refuses_before_it_writes():
    p, m = torch.ones(4, 9, device=DEV), torch.zeros(4, 9, device=DEV)
    both = torch.zeros(2, 4, 9, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        ops.muon_update([p], [both[0]], [both[0]], lr=0.1)
    with pytest.raises(ValueError, match="overlaps"):
        ops.muon_update([both[0]], [both.view(-1)[18:54].view(4, 9)], [m], lr=0.1)
    assert not bool(both.any())
    # 33 matrices are two calls, the larger ones first; the last one is too long: nothing may have happened by then
    shapes = [(3, 1 << 20)] * 32 + [(2, (1 << 20) + 1)]
    grads = [torch.ones(shapes[0], device=DEV)] * 32 + [torch.ones(shapes[-1], device=DEV)]
    many, bufs = ([torch.zeros(t, device=DEV) for t in shapes] for _ in range(2))
    with pytest.raises(ValueError, match="larger"):
        ops.muon_update(many, grads, bufs, lr=0.1)
    assert not any(bool(t.any()) for t in many + bufs)
    del many, bufs, grads
    # one gradient for two parameters is fine
    q, mq = p.clone(), m.clone()
    ops.muon_update([p, q], [both[1] + 1] * 2, [m, mq], lr=0.1)
    assert torch.equal(p, q) and not bool((p == 1).any())


@gpu
@pytest.mark.parametrize("sizes", [[(1500, 1530)], [(1409, 3000)], [(2100, 1441)], [(2200, 2210)], [(2790, 2800)], [(1030, 2070), (1024, 1024), (1000, 2500), (70, 90)]])
def test_orthogonalize_sizes_by_tile(sizes):
    """Sizes whose m x m products take tiles of 96 x 64 and 128 x 128."""
    mats = [matrix(r, c) for r, c in sizes]
    for got, g in zip(ops.orthogonalize(mats), mats):
        check(got, g)
    assert all(torch.equal(p, q) for p, q in zip(ops.orthogonalize(mats), ops.orthogonalize(mats)))


@gpu
def test_muon_update_in_a_graph():
    """A captured update, replayed between eager ones of other parameters, follows the eager sequence bit for bit."""
    shapes = [(64, 14, 3, 3), (10, 12), (200, 300), (33, 5)]
    gen = torch.Generator(device=DEV).manual_seed(9)
    new = lambda s: [torch.randn(t, generator=gen, device=DEV) for t in s]  # noqa: E731
    params, grads, bufs = new(shapes), new(shapes), [torch.zeros(s, device=DEV) for s in shapes]
    eager = [[t.clone() for t in ts] for ts in (params, grads, bufs)]
    other = [new(shapes[:2]), new(shapes[:2]), new(shapes[:2])]
    ops.muon_update(*other, lr=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.muon_update(params, grads, bufs, lr=0.05)
    for it in range(4):
        for g, e in zip(grads, eager[1]):
            g.copy_(torch.randn(g.shape, generator=gen, device=DEV))
            e.copy_(g)
        graph.replay()
        ops.muon_update(*other, lr=0.1)
        ops.muon_update(*eager, lr=0.05)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params + bufs, eager[0] + eager[2])), it


@gpu
def test_orthogonalize_empty_batches():
    for shape in ((0, 4, 5), (3, 0, 5), (2, 3, 4, 0), (0, 2, 3, 4), (0, 7), (7, 0)):
        out = ops.orthogonalize(torch.zeros(shape, device=DEV))
        assert out.shape == shape and out.numel() == 0
    a, b = ops.orthogonalize([torch.zeros(0, 3, device=DEV), matrix(5, 9)])
    assert a.shape == (0, 3)
    check(b, matrix(5, 9))


@gpu
@pytest.mark.parametrize("rows,cols", [(64, 40000), (60000, 50), (3, 200000), (100, 30000), (33, 49153)])
def test_orthogonalize_long(rows, cols):
    g = matrix(rows, cols)
    check(ops.orthogonalize(g), g)
