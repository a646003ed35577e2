"""Cases for the layer normalisation, orthogonalisation and Muon update operators of this package.

run() computes a case in its plain form - elementary torch operations in float32, rounded once at the end - or, with the
module's flag `own` set, by the calls a program makes of snws.ops.  exact() evaluates the definitions in float64."""
import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "semantic-segmentation_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

EPS_NORM = 1e-5
EPS_ORTHO = 1e-7
QUINTIC = (3.4445, -4.775, 2.0315)
STEPS = 5
LR, WEIGHT_DECAY, MOMENTUM = 0.02, 0.01, 0.95
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # object-region vectors of one image (10 classes x 512 features) normalised in evaluation: pure latency
        {"name": "norm_eval_regions", "op": "norm", "train": False, "dtype": "f32", "rows": 10, "width": 512, "pad": 0},
        # the finest encoder map of one 512 x 512 tile in full-disk inference
        {"name": "norm_eval_tile", "op": "norm", "train": False, "dtype": "bf16", "rows": 262144, "width": 64, "pad": 0},
        # long rows: flattened 3 x 3 patches of a 1024-channel map, an odd number of them
        {"name": "norm_eval_patches", "op": "norm", "train": False, "dtype": "f32", "rows": 997, "width": 9216, "pad": 0},
        # the region vectors of a batch of 16, forward and backward
        {"name": "norm_train_regions", "op": "norm", "train": True, "dtype": "f32", "rows": 160, "width": 512, "pad": 0},
        # the bottleneck map of a batch of 16 (32 x 32, 1024 channels)
        {"name": "norm_train_bottleneck", "op": "norm", "train": True, "dtype": "bf16", "rows": 16384, "width": 1024, "pad": 0},
        # a decoder map of a batch of 16 (256 x 256, 320 channels): the largest activation
        {"name": "norm_train_decoder", "op": "norm", "train": True, "dtype": "bf16", "rows": 1048576, "width": 320, "pad": 0},
        # an odd channel slice of a wider float32 concat buffer
        {"name": "norm_train_slice", "op": "norm", "train": True, "dtype": "f32", "rows": 50001, "width": 77, "pad": 19},
        # the first convolution's gradient, 64 x (14 * 9), alone
        {"name": "ortho_first_conv", "op": "ortho", "dtype": "f32", "rows": 64, "cols": 126, "pad": 0},
        # the widest filter of the model, 1024 x (1024 * 9)
        {"name": "ortho_widest", "op": "ortho", "dtype": "f32", "rows": 1024, "cols": 9216, "pad": 0},
        # a tall bfloat16 matrix of odd sizes inside a wider buffer
        {"name": "ortho_tall_odd", "op": "ortho", "dtype": "bf16", "rows": 1000, "cols": 333, "pad": 7},
        # every filter of the small test model, one optimizer step
        {"name": "muon_unet3p_4", "op": "muon", "filters": 4, "nesterov": True},
        # every filter of the benchmark model, one optimizer step
        {"name": "muon_unet3p_64", "op": "muon", "filters": 64, "nesterov": True},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "ortho", "muon"])
    if op == "norm":
        train = rng.random() < 0.6
        width = _log_uniform(rng, 3 if rng.random() < 0.1 else 16, 12000)
        if rng.random() < 0.6:
            width = (width + 7) // 8 * 8
        rows = _log_uniform(rng, 1, min(1 << 20, (1 << 26) // width))
        return {"op": op, "train": train, "dtype": rng.choice(["f32", "bf16"]), "rows": rows, "width": width,
                "pad": rng.choice([0, 0, 8, rng.randint(1, 63)])}
    if op == "ortho":
        small = _log_uniform(rng, 1 if rng.random() < 0.2 else 16, 1024)
        large = small * _log_uniform(rng, 1, 9) + rng.randint(0, 8)
        rows, cols = (small, large) if rng.random() < 0.7 else (large, small)
        return {"op": op, "dtype": rng.choice(["f32", "f32", "bf16"]), "rows": rows, "cols": cols,
                "pad": rng.choice([0, 0, rng.randint(1, 40)])}
    return {"op": op, "filters": rng.randint(2, 60), "nesterov": rng.random() < 0.7}


def _filters(f):
    """The 3 x 3 convolution filters of the full-scale-skip model with f filters at its finest scale."""
    enc = [14, f, 2 * f, 4 * f, 8 * f, 16 * f]
    shapes = []
    for a, b in zip(enc[:-1], enc[1:]):
        shapes += [(b, a, 3, 3), (b, b, 3, 3)]
    shapes += [(f, c, 3, 3) for c in (f, 2 * f, 4 * f, 8 * f, 16 * f, 5 * f)]
    return shapes + [(5 * f, 5 * f, 3, 3)]


def _gradient(rows, cols, gen):
    """A few strong directions over a dense remainder, at the scale of a filter's gradient."""
    k = min(rows, cols) // 4 + 1
    u = torch.randn(rows, k, generator=gen, device="cuda")
    v = torch.randn(k, cols, generator=gen, device="cuda")
    strength = 2.0 / torch.arange(1, k + 1, device="cuda", dtype=torch.float32).sqrt()
    return ((u * strength) @ v / math.sqrt(k) + torch.randn(rows, cols, generator=gen, device="cuda")) * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "norm":
        rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        wide = torch.randn(rows, width + case["pad"], generator=gen, device="cuda")
        wide += 0.7 * torch.randn(rows, 1, generator=gen, device="cuda") + torch.randn(width + case["pad"], generator=gen, device="cuda")
        x = wide.mul_(1.7).to(dtype)[:, :width]
        state = {"case": case, "x": x, "weight": 1 + 0.3 * torch.randn(width, generator=gen, device="cuda"),
                 "bias": 0.3 * torch.randn(width, generator=gen, device="cuda")}
        if case["train"]:
            state["dy"] = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
            for k in ("x", "weight", "bias"):
                state[k] = state[k].detach().requires_grad_(True)
        return state
    if case["op"] == "ortho":
        g = _gradient(case["rows"], case["cols"] + case["pad"], gen).to(DTYPES[case["dtype"]])
        return {"case": case, "g": g[:, :case["cols"]]}
    shapes = _filters(case["filters"])
    grads = [_gradient(s[0], s[1] * 9, gen).view(s) for s in shapes]
    return {"case": case, "grads": grads,
            "params": [torch.randn(s, generator=gen, device="cuda") / math.sqrt(s[1] * 9) for s in shapes],
            "bufs": [0.5 * g.roll(1, 0) + 1e-3 * torch.randn(s, generator=gen, device="cuda") for g, s in zip(grads, shapes)]}


# ---------------------------------------------------------------------------------------------- plain forms (float32)
def _norm_plain(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS_NORM)
    xhat = xc * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _ortho_plain(g):
    """Five steps of X <- a X + (b A + c A^2) X with A = X X^T, from X = G over its Frobenius norm, on the wide side."""
    a, b, c = QUINTIC
    x = g.float()
    flip = x.shape[0] > x.shape[1]
    if flip:
        x = x.t()
    x = x / (x * x).sum().sqrt().clamp(min=EPS_ORTHO)
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if flip else x


def _muon_plain(s):
    for p, g, m in zip(s["params"], s["grads"], s["bufs"]):      # filters of different shapes: one after the other
        m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
        u = g * (1 - MOMENTUM) + m * MOMENTUM if s["case"]["nesterov"] else m
        o = _ortho_plain(u.reshape(u.shape[0], -1)).reshape(u.shape)
        scale = math.sqrt(max(1.0, u.shape[0] / (u.numel() / u.shape[0])))
        p.mul_(1 - LR * WEIGHT_DECAY).sub_(o, alpha=LR * scale)
    return {"params": s["params"], "bufs": s["bufs"]}


# ---------------------------------------------------------------------------------------------- the package's operators
def _run_own(s):
    from snws import ops
    case = s["case"]
    if case["op"] == "norm":
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS_NORM)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "ortho":
        return {"o": ops.orthogonalize(s["g"], steps=STEPS, coefficients=QUINTIC, eps=EPS_ORTHO)}
    ops.muon_update(s["params"], s["grads"], s["bufs"], lr=LR, weight_decay=WEIGHT_DECAY, momentum=MOMENTUM,
                    nesterov=case["nesterov"], steps=STEPS, coefficients=QUINTIC, eps=EPS_ORTHO, adjust_lr="original")
    return {"params": s["params"], "bufs": s["bufs"]}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _norm_plain(state)
    if op == "ortho":
        return {"o": _ortho_plain(state["g"]).to(state["g"].dtype)}
    return _muon_plain(state)


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], 4 if case["dtype"] == "f32" else 2
        small = 8 * case["width"]
        if case["train"]:       # x and dy in, y and dx out, the weight and bias in, their gradients out
            return {"bytes": 4 * n * size + 2 * small, "flops": 20 * n}
        return {"bytes": 2 * n * size + small, "flops": 8 * n}
    if case["op"] == "ortho":
        pairs, size, copies = [(case["rows"], case["cols"])], 4 if case["dtype"] == "f32" else 2, 2
    else:                       # parameter and momentum in and out, the gradient in
        pairs, size, copies = [(s[0], s[1] * 9) for s in _filters(case["filters"])], 4, 5
    flops = nbytes = 0
    for r, c in pairs:
        m, n = min(r, c), max(r, c)
        flops += STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)    # the two symmetric products: half each
        nbytes += copies * size * m * n
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------- definitions in float64
def _polar_exact(u):
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return _polar_exact(x.t()).t()
    x = x / torch.clamp(torch.linalg.vector_norm(x), min=EPS_ORTHO)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    a, b, c = QUINTIC
    for _ in range(STEPS):
        gram = torch.mm(x, x.t().contiguous())
        x = torch.mm(a * eye + torch.mm(gram, b * eye + c * gram), x)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ortho":
        return {"o": _polar_exact(s["g"])}
    if case["op"] == "muon":
        params, bufs = [], []
        for p, g, m in zip(s["params"], s["grads"], s["bufs"]):
            p, g, m = p.double(), g.double(), m.double()
            buf = m + (g - m) * (1 - MOMENTUM)
            u = g + (buf - g) * MOMENTUM if case["nesterov"] else buf
            r, c = p.shape[0], p[0].numel()
            step = LR * max(1.0, r / c) ** 0.5 * _polar_exact(u.reshape(r, c)).reshape(p.shape)
            params.append(p - LR * WEIGHT_DECAY * p - step)
            bufs.append(buf)
        return {"params": params, "bufs": bufs}
    with torch.no_grad():
        x, w, b = (s[k].detach().double() for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        sigma = (var + EPS_NORM) ** 0.5
        z = (x - mean) / sigma
        out = {"y": z * w + b}
        if case["train"]:
            dy = s["dy"].double()
            gw = dy * w
            # the projection of gw off the constant and off z, over sigma
            n = x.shape[1]
            out["dx"] = (gw - gw.sum(1, keepdim=True) / n - z * ((gw * z).sum(1, keepdim=True) / n)) / sigma
            out["dweight"] = (dy * z).sum(0)
            out["dbias"] = dy.sum(0)
    return out
