"""Layer normalisation (snws.ops.layer_norm, modeling.layernorm.LayerNorm2d) against its definition in float64: values,
all three gradients, odd lengths, strides, refusals, streams and captured graphs."""
import math

import pytest
import torch

from snws import _lib as L
from snws import ops
from modeling.layernorm import LayerNorm2d

DEV = "cuda:0"
gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refuses_cpu_tensors_and_wrong_shapes():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.layer_norm(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        LayerNorm2d(4)(torch.zeros(1, 4, 2, 2))
    with pytest.raises(ValueError, match="4D"):
        LayerNorm2d(4)(torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="channels"):
        LayerNorm2d(4)(torch.zeros(1, 5, 2, 2))


def test_entry_points_refuse_bad_arguments():
    P = 4096      # never dereferenced: every refusal comes before a launch
    good = [P, 8, None, None, P, 8, L.SNWS_F32, 4, 8, 1e-5, None, None, None]
    for at, value, text in ((6, L.SNWS_F64, "dtype"), (7, -1, "sizes"), (8, 0, "sizes"), (1, 7, "sizes"), (5, 7, "sizes"),
                            (9, -1.0, "eps"), (9, float("nan"), "eps"), (0, None, "NULL"), (4, None, "NULL"),
                            (10, P, "mean and rstd")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=text):
            L.call("snws_ln_fwd", *args)
    good = [P, 8, P, 8, P, P, None, L.SNWS_F32, 4, 8, P, 8, P, P, P, 1 << 20, None]
    for at, value, text in ((7, 9, "dtype"), (8, -1, "sizes"), (9, 0, "sizes"), (1, 7, "sizes"), (3, 7, "sizes"),
                            (11, 7, "sizes"), (0, None, "NULL"), (2, None, "NULL"), (4, None, "NULL"), (5, None, "NULL"),
                            (14, None, "workspace"), (15, 1, "workspace")):
        args = list(good)
        args[8] = 4000 if text == "workspace" else args[8]        # (few rows need none)
        args[at] = value
        with pytest.raises(ValueError, match=text):
            L.call("snws_ln_bwd", *args)
    assert L.call("snws_ln_fwd", None, 8, None, None, None, 8, L.SNWS_F32, 0, 8, 1e-5, None, None, None) == 0
    assert L.lib().snws_ln_bwd_workspace_floats(L.SNWS_F32, 0, 8) == 0
    assert L.lib().snws_ln_bwd_workspace_floats(L.SNWS_F32, 256, 8) == 0
    assert L.lib().snws_ln_bwd_workspace_floats(L.SNWS_F32, 257, 8) > 0 and L.lib().snws_ln_bwd_workspace_floats(L.SNWS_BF16, 4, 3) > 0


def test_entry_points_refuse_rows_beyond_their_counters():
    P, C = 4096, (1 << 28) + 1
    with pytest.raises(ValueError, match="sizes"):
        L.call("snws_ln_fwd", P, C, None, None, P, C, L.SNWS_F32, 4, C, 1e-5, None, None, None)
    with pytest.raises(ValueError, match="sizes"):
        L.call("snws_ln_bwd", P, C, P, C, P, P, None, L.SNWS_F32, 4, C, P, C, P, P, P, 1 << 40, None)
    assert L.lib().snws_ln_bwd_workspace_floats(L.SNWS_F32, 4, C) == 0


def test_rows_of_strided_views():
    x = torch.zeros(3, 4, 10)
    assert ops._as_rows(x)[1:] == (10, 12)
    v, ld, rows = ops._as_rows(x[..., 2:9])
    assert v.data_ptr() == x.data_ptr() + 8 and (ld, rows) == (10, 12)
    v, ld, rows = ops._as_rows(x[:, 1:3])                    # rows of two strides: copied
    assert v.is_contiguous() and (ld, rows) == (10, 6)
    v, ld, rows = ops._as_rows(torch.zeros(1, 1).expand(5, 6))
    assert v.is_contiguous() and (ld, rows) == (6, 5)
    v, ld, rows = ops._as_rows(torch.zeros(1, 6).expand(5, 6))
    assert v.is_contiguous() and (ld, rows) == (6, 5)
    m = torch.zeros(2, 7, 5, 3).contiguous(memory_format=torch.channels_last)
    v, ld, rows = ops._as_rows(m.permute(0, 2, 3, 1))
    assert v.data_ptr() == m.data_ptr() and (ld, rows) == (7, 30)


# ------------------------------------------------------------------------------------------------ values (GPU)
def definition(x, w, b, dy, eps):
    """float64 on the CPU: (y, dx, dw, db, z, rstd, g)."""
    x, dy = x.double().cpu(), dy.double().cpu()
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double().cpu()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    z = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
    return z * w + b, dx, (dy * z).sum(0), dy.sum(0), z, rstd, g


def check(x, w, b, dy, eps, y, dx, dw, db):
    """Element by element.  Rounding a sum of n terms in a tree over at most 64 terms per lane and 9 joins costs at most
    73 half steps u of the sum of the absolute values; z adds the error of the mean, relative to the spread, and of rstd.
    The factor 256 u covers that with the few single roundings behind it; a half step of the type for what is stored."""
    u = 2.0 ** -24
    half = torch.finfo(x.dtype).eps / 2
    ry, rdx, rdw, rdb, z, rstd, g = definition(x, w, b, dy, eps)
    # error of z: (mean's own error + x's subtraction) * rstd, and rstd's relative error
    xa = x.double().cpu().abs()
    dz = 256 * u * ((xa.mean(-1, keepdim=True) + xa) * rstd + z.abs())
    aw = 1.0 if w is None else w.double().cpu().abs()
    ok = (y.double().cpu() - ry).abs() <= half * ry.abs() * 1.01 + dz * aw + 4 * u * (ry.abs() + (0 if b is None else b.double().cpu().abs()))
    assert bool(ok.all()), float((y.double().cpu() - ry).abs().max())
    if dx is not None:
        m1, m2 = g.abs().mean(-1, keepdim=True), (g * z).abs().mean(-1, keepdim=True)
        slack = rstd * (256 * u * (g.abs() + m1 + z.abs() * m2) + dz * m2 + z.abs() * (g.abs() * dz).mean(-1, keepdim=True))
        err = (dx.double().cpu() - rdx).abs()
        assert bool((err <= half * rdx.abs() * 1.01 + slack).all()), float((err - slack).max())
    rows = x.shape[0]
    k = 64 + min(rows, 16 + rows // 256)          # sequential adds of one lane's rows, then the joins
    ady = dy.double().cpu().abs()
    if dw is not None:
        err = (dw.double().cpu() - rdw).abs()
        assert bool((err <= 2 * k * u * (ady * z.abs()).sum(0) + (ady * dz).sum(0) + u * rdw.abs()).all()), float(err.max())
    if db is not None:
        err = (db.double().cpu() - rdb).abs()
        assert bool((err <= k * u * ady.sum(0) + u * rdb.abs()).all()), float(err.max())


def make(rows, C, dtype, pad=0, seed=0, off=1.0):
    g = torch.Generator().manual_seed(seed + 31 * rows + C)
    wide = torch.randn(rows, C + pad, generator=g) * 1.7 + off * torch.randn(rows, 1, generator=g)
    x = wide.to(dtype).to(DEV)[:, :C]
    dy = torch.randn(rows, C, generator=g).to(dtype).to(DEV)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(DEV)
    b = (0.3 * torch.randn(C, generator=g)).to(DEV)
    return x, w, b, dy


SHAPES = [(1, 1, 0), (5, 2, 0), (300, 3, 0), (2000, 7, 2), (9, 8, 0), (1, 512, 0), (160, 512, 0), (33, 77, 19), (1001, 64, 0),
          (770, 320, 0), (514, 100, 1), (37, 161, 0), (40, 640, 8), (21, 1024, 0), (19, 1283, 5), (6, 2049, 0), (5, 4096, 0),
          (4, 5000, 3), (3, 9216, 0), (3, 16384, 0), (2, 16390, 0), (2, 33000, 1), (5000, 24, 0)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,C,pad", SHAPES)
def test_layer_norm_values_and_gradients(rows, C, pad, dtype):
    x, w, b, dy = make(rows, C, dtype, pad)
    xg, wg, bg = x.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = ops.layer_norm(xg, wg, bg, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32 and y.is_contiguous()
    check(x, w, b, dy, 1e-5, y.detach(), dx, dw, db)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, 1e-5), y.detach())
    y2 = ops.layer_norm(xg, wg, bg, 1e-5)
    for p, q in zip((dx, dw, db), torch.autograd.grad(y2, (xg, wg, bg), dy)):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_layer_norm_many_rows(dtype):
    """Rows enough that every lane group walks over many of them."""
    x, w, b, dy = make(70001, 72, dtype)
    xg, wg, bg = x.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = ops.layer_norm(xg, wg, bg)
    check(x, w, b, dy, 1e-5, y.detach(), *torch.autograd.grad(y, (xg, wg, bg), dy))


@gpu
def test_layer_norm_without_parameters_and_partial_gradients():
    x, w, b, dy = make(50, 130, torch.float32)
    y = ops.layer_norm(x.requires_grad_(True))
    dx, = torch.autograd.grad(y, x, dy)
    check(x.detach(), None, None, dy, 1e-5, y.detach(), dx, None, None)
    wg = w.clone().requires_grad_(True)
    y = ops.layer_norm(x.detach(), wg, None)
    dw, = torch.autograd.grad(y, wg, dy)
    check(x.detach(), w, None, dy, 1e-5, y.detach(), None, dw, None)
    bg = b.clone().requires_grad_(True)
    y = ops.layer_norm(x.detach(), None, bg)
    db, = torch.autograd.grad(y, bg, dy)
    check(x.detach(), None, b, dy, 1e-5, y.detach(), None, None, db)
    empty = torch.zeros(0, 130, device=DEV, requires_grad=True)
    wg, bg = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = ops.layer_norm(empty, wg, bg)
    assert y.shape == (0, 130)
    dx, dw, db = torch.autograd.grad(y, (empty, wg, bg), torch.zeros(0, 130, device=DEV))
    assert dx.shape == (0, 130) and float(dw.abs().max()) == 0.0 and float(db.abs().max()) == 0.0


@gpu
def test_layer_norm_special_rows():
    """Constant rows give the bias and finite gradients; a row with NaN or infinity stays its own affair; a mean of 1e4
    times the spread costs only the mean's own rounding."""
    x, w, b, dy = make(64, 200, torch.float32)
    x = x.clone()
    x[3] = 5.0
    x[7] = 0.0
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[7], b) and float((y[3] - b).abs().max()) <= 1e-3      # sqrt(1e5) * rounding of the mean, 2^-22
    clean = ops.layer_norm(x, w, b)
    x[10, 5] = float("nan")
    x[20, 199] = float("inf")
    y = ops.layer_norm(x, w, b)
    keep = torch.ones(64, dtype=torch.bool, device=DEV)
    keep[[10, 20]] = False
    assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[10]).all()) and bool(torch.isnan(y[20, 199]))
    far, w, b, dy = make(64, 200, torch.float32, off=1e4)
    xg = far.requires_grad_(True)
    y = ops.layer_norm(xg, w, b)
    dx, = torch.autograd.grad(y, xg, dy)
    check(far.detach(), w, b, dy, 1e-5, y.detach(), dx, None, None)


@gpu
def test_layer_norm_gradient_against_differences():
    """Directional derivative of sum(dy * y) along random directions: central differences of the float64 definition at
    step 1e-4 (their own error: h^2 times the third derivative, below 1e-6 here) against the kernels' gradients."""
    x, w, b, dy = make(40, 52, torch.float32, seed=5)
    xg, wg, bg = (t.clone().requires_grad_(True) for t in (x, w, b))
    grads = torch.autograd.grad(ops.layer_norm(xg, wg, bg), (xg, wg, bg), dy)

    def f(p):
        return float((definition(*p, dy, 1e-5)[0] * dy.double().cpu()).sum())
    base = [t.double().cpu() for t in (x, w, b)]
    for i in range(3):
        d = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        h = 1e-4
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        want = (f(up) - f(down)) / (2 * h)
        got = float((grads[i].double().cpu() * d).sum())
        # 256 half steps of the sum of absolute products (see check), and the differences' own error
        assert abs(got - want) <= 256 * 2.0 ** -24 * float((grads[i].double().cpu() * d).abs().sum()) + 1e-5 * (1 + abs(want))


@gpu
def test_layer_norm_views_expanded_gradient_and_types():
    x, w, b, dy = make(24, 40, torch.float32)
    x3 = x.view(2, 3, 4, 40).permute(1, 0, 2, 3)              # leading axes out of order: copied
    y = ops.layer_norm(x3, w, b)
    want = definition(x, w, b, dy, 1e-5)[0].view(2, 3, 4, 40).permute(1, 0, 2, 3)
    assert float((y.double().cpu() - want).abs().max()) < 1e-5
    xg = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(ops.layer_norm(xg, w, b).sum(), xg)        # the gradient arrives as an expanded scalar
    check(x, w, b, torch.ones_like(x), 1e-5, ops.layer_norm(x, w, b), dx, None, None)
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x, w[:-1])
    with pytest.raises(RuntimeError, match="bias"):
        ops.layer_norm(x, w, b.cpu())
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros((), device=DEV))
    half = w.to(torch.bfloat16).requires_grad_(True)
    dw, = torch.autograd.grad(ops.layer_norm(x, half, b), half, dy)
    assert dw.dtype == torch.bfloat16
    xg = x.clone().requires_grad_(True)
    g1, = torch.autograd.grad(ops.layer_norm(xg, w, b).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g1.sum(), xg)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_layer_norm_2d_module(dtype):
    """The module on NCHW and channels-last maps and on a channel slice, against the definition; its gradients land in
    the flat optimizer's slots."""
    from snws.optim import FlatAdamW
    torch.manual_seed(3)
    m = LayerNorm2d(24, eps=1e-3).to(DEV)
    with torch.no_grad():
        m.weight.add_(0.2 * torch.randn(24, device=DEV))
        m.bias.add_(0.2 * torch.randn(24, device=DEV))
    wide = torch.randn(2, 40, 5, 7, device=DEV).to(dtype).contiguous(memory_format=torch.channels_last)
    opt = FlatAdamW(m.parameters(), lr=1e-2)
    for x in (wide[:, 8:32], wide[:, 8:32].contiguous()):
        dy = torch.randn(2, 24, 5, 7, device=DEV).to(dtype)
        opt.zero_grad()
        xg = x.detach().requires_grad_(True)
        y = m(xg)
        y.backward(dy)
        assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
        rows = lambda t: t.detach().permute(0, 2, 3, 1).reshape(-1, 24)  # noqa: E731
        check(rows(x), m.weight.detach(), m.bias.detach(), rows(dy), 1e-3, rows(y), rows(xg.grad), m.weight.grad, m.bias.grad)
        assert m.weight.grad.data_ptr() == opt.flat_g.data_ptr()
    assert LayerNorm2d(4, affine=False).weight is None


@gpu
def test_layer_norm_on_other_streams_and_in_a_graph():
    x, w, b, dy = make(300, 320, torch.bfloat16)
    xg, wg, bg = (t.detach().clone().requires_grad_(True) for t in (x, w, b))

    def step():
        y = ops.layer_norm(xg, wg, bg)
        return (y,) + torch.autograd.grad(y, (xg, wg, bg), dy)
    want = [t.detach().clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    x0 = xg.detach().clone()
    for i in range(4):
        with torch.no_grad():
            xg.copy_(x0 * (1 + 0.25 * i))
        want = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), i
        junk = torch.randn(1 << 20, device=DEV).sum()          # the program's own work between the replays
        torch.cuda.synchronize()
        assert math.isfinite(float(junk))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,C", [(1, 33), (2, 9216), (255, 8), (256, 100), (257, 100), (256, 31), (300, 1040), (30, 2048)])
def test_layer_norm_every_choice_of_gradients(rows, C, dtype):
    """Each of the seven sets of wanted gradients, on both sides of the row count up to which one launch does it all."""
    x, w, b, dy = make(rows, C, dtype, pad=3)
    for want in range(1, 8):
        leaves = [t.detach().clone().requires_grad_(bool(want >> i & 1)) for i, t in enumerate((x, w, b))]
        y = ops.layer_norm(*leaves)
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy))
        check(x, w, b, dy, 1e-5, y.detach(), *[next(grads) if t.requires_grad else None for t in leaves])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,C", [(1, 60000), (16, 33001), (17, 33001), (2, 65539)])
def test_layer_norm_rows_beyond_registers(rows, C, dtype):
    """Rows partly read again, at most 64 elements to a thread and half; with and without partial sums of the parameters."""
    x, w, b, dy = make(rows, C, dtype, pad=5)
    for want in (7, 1, 2, 6):
        leaves = [t.detach().clone().requires_grad_(bool(want >> i & 1)) for i, t in enumerate((x, w, b))]
        leaves[0] = x.detach().requires_grad_(bool(want & 1))
        y = ops.layer_norm(*leaves)
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy))
        check(x, w, b, dy, 1e-5, y.detach(), *[next(grads) if t.requires_grad else None for t in leaves])
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b), y.detach())
