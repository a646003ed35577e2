"""snws.optim.FlatMuon and Trainer(optimizer="muon"): every update against its definition in float64, the state's format,
checkpoints, and a block of a standardized convolution and a layer normalisation trained with it."""
import math
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import patterns
from modeling.layernorm import LayerNorm2d
from modeling import weightstd
from oracle import snws_oracle as O
from snws import checkpoint, harness, ops
from snws.optim import FlatAdamW, FlatMuon
from test_gpu_ortho import A0, muon_definition

DEV = "cuda:0"
gpu = pytest.mark.gpu
U = 2.0 ** -24


def test_refusals_without_a_gpu():
    p = torch.nn.Parameter(torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="FlatMuon.*no CPU fallback"):
        FlatMuon([p])
    with pytest.raises(ValueError, match="FlatMuon: no parameters"):
        FlatMuon([])
    with pytest.raises(ValueError, match="step"):
        FlatMuon([p], ns_steps=0)
    with pytest.raises(ValueError, match="three"):
        FlatMuon([p], ns_coefficients=(1.0, 2.0))
    with pytest.raises(ValueError, match="adjust_lr"):
        FlatMuon([p], adjust_lr_fn="other")


def check_matrix(p, m, want, lr, adjust):
    """The update's error: the products' (want[2]), the momentum's three roundings, which reach it as a relative error of
    the matrix times the polynomials' slope at zero, and the update's own roundings."""
    f = ops.muon_lr_factor(adjust, p.shape[0], p[0].numel())
    slack = want[2] + lr * f * 8 * U * A0 ** 5 + 4 * U * float(want[0].norm() + 1)
    assert float((p.detach().double() - want[0]).norm()) <= slack, tuple(p.shape)
    assert float((m.double() - want[1]).norm()) <= 8 * U * float(want[1].norm()) + 1e-30, tuple(p.shape)


SHAPES = [(7, 3, 3, 3), (7,), (1, 5, 1, 1), (10, 7, 1, 1), (6, 4), (2,), (9, 1), (5, 4), (64, 14, 3, 3)]
MATRICES = [0, 3, 7, 8]          # 4 is given to AdamW by name, 7 receives no gradient; rows and columns of one are vectors


@gpu
@pytest.mark.parametrize("nesterov,adjust", [(True, None), (False, "match_rms_adamw")])
def test_flat_muon_matches_definitions(nesterov, adjust):
    """Four steps: matrices against the definition from the state before each step, the others against AdamW in float64.
    AdamW's bound per step: two roundings of the parameter, and an update of at most 4 lr elementwise (|g| <= 2 sqrt(v) over
    four steps) with about 20 roundings; the betas are exact in float32."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    start = [torch.randn(s, generator=gen, device=DEV) for s in SHAPES]
    pa = [torch.nn.Parameter(t.clone()) for t in start]
    pb = [torch.nn.Parameter(t.double()) for t in start]
    betas, wd = (0.875, 0.96875), 0.125
    opt = FlatMuon(pa, lr=0.02, weight_decay=wd, momentum=0.9, nesterov=nesterov, adjust_lr_fn=adjust,
                   adamw_params=iter([pa[4]]), adamw_lr=0.01, betas=betas)
    assert [id(p) for p in opt.param_groups[0]["params"]] == [id(pa[i]) for i in MATRICES]
    plain = [i for i in range(len(SHAPES)) if i not in MATRICES]
    ref = torch.optim.AdamW([pb[i] for i in plain], lr=0.01, weight_decay=wd, betas=betas)
    moments = [torch.zeros(s, device=DEV) for s in SHAPES]
    total = 0.0
    for it in range(4):
        for g in opt.param_groups + ref.param_groups:
            g["lr"] = (0.02 if "momentum" in g else 0.01) * (1 - it / 8)
        lr = 0.02 * (1 - it / 8)
        opt.zero_grad()
        coef = [torch.randn(s, generator=gen, device=DEV) for s in SHAPES]
        sum(((p * c).sum() for i, (p, c) in enumerate(zip(pa, coef)) if i != 7)).backward()
        assert all(torch.equal(p.grad, c) for i, (p, c) in enumerate(zip(pa, coef)) if i != 7)
        before = [p.detach().clone() for p in pa]
        opt.step(grad_scale=0.5)
        for i in plain:
            pb[i].grad = coef[i].double() * 0.5
        ref.step()
        total += lr
        for i in MATRICES:
            if i == 7:
                assert torch.equal(pa[i], start[i])
                continue
            want = muon_definition(before[i], coef[i], moments[i], lr, wd, 0.9, nesterov, adjust, 0.5)
            got = opt._slots[i][2]
            check_matrix(pa[i], got, want, lr, adjust)
            moments[i] = got.clone()
        for i in plain:
            err = (pa[i].detach().double() - pb[i].detach()).abs().max()
            assert float(err) <= (it + 1) * 3 * U * float(pb[i].detach().abs().max() + 1) + 4 * total * 20 * U, (it, i)


def train(opt, params, seed, steps=2):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for _ in range(steps):
        opt.zero_grad()
        sum((p * torch.randn(p.shape, generator=gen, device=DEV)).sum() for p in params).backward()
        opt.step()


@gpu
def test_flat_muon_state():
    """The state's format, its way into another optimizer and on, and what is refused (with nothing changed)."""
    def make(shapes=SHAPES, **kw):
        gen = torch.Generator(device=DEV).manual_seed(3)
        params = [torch.nn.Parameter(torch.randn(s, generator=gen, device=DEV)) for s in shapes]
        return params, FlatMuon(params, lr=0.02, adamw_params=[params[4]], **kw)
    pa, oa = make()
    assert oa.state_dict()["state"] == {}
    train(oa, pa[:7] + pa[8:], 5)
    sd = oa.state_dict()
    matrices, rest = sd["param_groups"]
    assert matrices["params"] == [0, 1, 2, 3] and rest["params"] == [4, 5, 6, 7, 8]
    assert set(matrices) == set(torch.optim.Muon([torch.nn.Parameter(torch.zeros(2, 2))]).state_dict()["param_groups"][0])
    assert set(sd["state"]) == set(range(9)) - {2}
    assert set(sd["state"][1]) == {"momentum_buffer"} and sd["state"][1]["momentum_buffer"].shape == SHAPES[3]
    assert set(sd["state"][4]) == {"step", "exp_avg", "exp_avg_sq"} and float(sd["state"][4]["step"]) == 2.0
    assert oa.exp_avg_sq.numel() == 8 + 8 + 24 + 4 + 12          # (7,) (1,5,1,1) (6,4) (2,) (9,1): none for the matrices
    pb, ob = make(momentum=0.5, betas=(0.5, 0.5))
    with torch.no_grad():
        for p, q in zip(pa, pb):
            q.copy_(p)
    ob.load_state_dict(sd)
    assert ob.param_groups[0]["momentum"] == 0.95 and ob.param_groups[1]["betas"] == (0.9, 0.999)
    train(oa, pa, 6)
    train(ob, pb, 6)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))
    kept = oa.exp_avg.clone()
    single = FlatAdamW([torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in SHAPES])
    bad = oa.state_dict()
    bad["state"][1]["momentum_buffer"] = torch.zeros(3, 3)
    for wrong in (single.state_dict(), bad):
        with pytest.raises(ValueError, match="FlatMuon.load_state_dict"):
            oa.load_state_dict(wrong)
    assert torch.equal(oa.exp_avg, kept) and oa.param_groups[0]["lr"] == 0.02
    only = [torch.nn.Parameter(torch.ones(4, 5, device=DEV))]
    opt = FlatMuon(only)
    train(opt, only, 1)
    assert opt.exp_avg_sq.numel() == 0 and not torch.equal(only[0], torch.ones(4, 5, device=DEV))
    vector = [torch.nn.Parameter(torch.ones(5, device=DEV))]
    train(FlatMuon(vector), vector, 1)
    assert bool(torch.isfinite(vector[0]).all()) and not torch.equal(vector[0], torch.ones(5, device=DEV))


@gpu
def test_trainer_muon(tmp_path):
    """Trainer(optimizer="muon") on UNet3p: every filter's update against the definition from its own gradient, the
    classification conv and the vectors with AdamW, and a checkpoint that a fresh Trainer takes up."""
    from modeling.UNet3p_SNws import UNet3p_SNws
    img, lab = patterns.synth_batch(2, 14, 64, 101)
    img, lab = img.to(DEV), lab.to(DEV)
    model = UNet3p_SNws(14, 4, 10, 1, 1)
    patterns.det_init(model)
    model = model.to(DEV)
    tr = harness.Trainer(model, optimizer="muon", total_iters=50)
    opt = tr.opt
    assert isinstance(opt, FlatMuon) and tr.buckets.slices is not None
    names = {id(p): n for n, p in model.named_parameters()}
    head = getattr(model, "cls_head", None) or model.output_seg_map
    assert id(head.weight) in [id(p) for p in opt.param_groups[1]["params"]]
    assert all(p.dim() == 4 and p.shape[0] > 1 for p in opt.param_groups[0]["params"])
    for it in range(2):
        lr = harness.poly_lr(0.002, it, 50)
        before, moments = opt.flat_p.clone(), opt.exp_avg.clone()
        assert math.isfinite(float(tr.step(img, lab)))
        seen = 0
        for i, (p, o) in enumerate(zip(opt.params, opt.offsets)):
            part = slice(o, o + p.numel())
            if not opt._touched[i]:
                assert torch.equal(opt.flat_p[part], before[part]), names[id(p)]
            elif opt.is_matrix[i]:
                seen += 1
                g, m, b = (t[part].view(p.shape) for t in (opt.flat_g, moments, before))
                want = muon_definition(b, g, m, lr, 5e-4, 0.95, True, "match_rms_adamw")
                check_matrix(p, opt._slots[i][2], want, lr, "match_rms_adamw")
            else:          # AdamW moves no element by more than lr sqrt(t) / (1 - b1) beyond its decay, and by lr at first
                most = lr * (1.01 if it == 0 else 10 * 2 ** 0.5)
                assert float((opt.flat_p[part] - before[part] * (1 - lr * 5e-4)).abs().max()) <= most, names[id(p)]
        assert seen == sum(t and p.dim() == 4 and p.shape[0] > 1 and p is not head.weight for p, t in zip(opt.params, opt._touched))
        assert seen > 0
    path = str(tmp_path / "checkpoint.pth.tar")
    checkpoint.save_checkpoint(path, model, opt, epoch=1, best_pred=0.5)
    fresh = UNet3p_SNws(14, 4, 10, 1, 1).to(DEV)
    tr2 = harness.Trainer(fresh, optimizer="muon", total_iters=50)
    assert checkpoint.load_checkpoint(path, fresh, tr2.opt) == (1, 0.5)
    for key in ("flat_p", "exp_avg", "exp_avg_sq", "steps"):
        a, b = getattr(opt, key), getattr(tr2.opt, key)
        assert torch.equal(a, b) if torch.is_tensor(a) else [min(s, 1) for s in a] == [min(s, 1) for s in b], key
    assert tr2.opt.param_groups[0]["lr"] == harness.poly_lr(0.002, 1, 50)
    tr2.close()
    tr.close()


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = weightstd.Conv2dws(6, 12, 3, 1, 1)
        self.norm = LayerNorm2d(12)
        self.head = weightstd.Conv2dws(12, 3, 1, 1, 0)

    def forward(self, x):
        return self.head(torch.nn.functional.gelu(self.norm(self.conv(x))))


def block64(x, conv, cb, gain, shift, head, hb):
    y = O.conv2dws_fwd(x, conv, cb, 1, 1, 1, 1)
    y = torch.nn.functional.layer_norm(y.permute(0, 2, 3, 1), (12,), gain, shift, 1e-5).permute(0, 3, 1, 2)
    return O.conv2dws_fwd(torch.nn.functional.gelu(y), head, hb, 1, 0, 1, 1)


@gpu
def test_block_trained_with_flat_muon():
    """Convolution, layer normalisation and update as one training loop: the gradients in the optimizer's slots against the
    same block in float64 and against its differences, then the update from them.  Seven stages forward and backward, each
    with a relative error of at most (8 + sqrt(198)) 2^-23 (198 positions are the longest sum), times 4 for what a
    normalisation adds to its input's error: 7.5e-5 of a gradient's norm.  The differences (step 1e-5, in float64) are
    within 1e-6 of the derivative."""
    torch.manual_seed(11)
    block = Block().to(DEV)
    opt = FlatMuon(block.parameters(), lr=0.02, adjust_lr_fn="match_rms_adamw", adamw_params=block.head.parameters())
    assert [tuple(p.shape) for p in opt.param_groups[0]["params"]] == [(12, 6, 3, 3)]
    x = torch.randn(2, 6, 9, 11, device=DEV)
    xs = x.contiguous(memory_format=torch.channels_last)
    for _ in range(3):
        ref = [p.detach().double().cpu().requires_grad_(True) for p in block.parameters()]
        dy = torch.randn(2, 3, 9, 11, device=DEV)
        opt.zero_grad()
        (block(xs) * dy).sum().backward()

        def loss(ps):
            return (block64(x.double().cpu(), *ps) * dy.double().cpu()).sum()
        loss(ref).backward()
        for p, r, s in zip(block.parameters(), ref, opt._slots):
            assert p.grad.data_ptr() == s[1].data_ptr()
            assert float((p.grad.double().cpu() - r.grad).norm()) <= 7.5e-5 * float(r.grad.norm()), tuple(p.shape)
        with torch.no_grad():
            for k, p in enumerate(block.parameters()):
                way = p.grad.double().cpu() / float(p.grad.norm())
                up, down = ([r + h * way if i == k else r for i, r in enumerate(ref)] for h in (1e-5, -1e-5))
                slope = float(loss(up) - loss(down)) / 2e-5
                assert abs(slope - float(p.grad.double().norm())) <= (7.5e-5 + 1e-6) * abs(slope), k
        before, moment = block.conv.weight.detach().clone(), opt._slots[0][2].clone()
        want = muon_definition(before, block.conv.weight.grad, moment, 0.02, 0.1, 0.95, True, "match_rms_adamw")
        opt.step()
        check_matrix(block.conv.weight, opt._slots[0][2], want, 0.02, "match_rms_adamw")
    opt.release()


def _rank(rank, port, q):
    import faulthandler
    faulthandler.dump_traceback_later(90, exit=True)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    from modeling.UNet3p_SNws import UNet3p_SNws
    img, lab = patterns.synth_batch(2, 14, 64, 101)
    model = UNet3p_SNws(14, 4, 10, 1, 1)
    patterns.det_init(model)
    tr = harness.Trainer(model.to(DEV), optimizer="muon", total_iters=50, bucket_mb=0.05)
    opt = tr.opt
    for it in range(2):
        before, moments = opt.flat_p.clone(), opt.exp_avg.clone()
        tr.step(img[rank:rank + 1].to(DEV), lab[rank:rank + 1].to(DEV))
        for i in (i for i, m in enumerate(opt.is_matrix) if m and opt._touched[i]):
            p, part = opt.params[i], slice(opt.offsets[i], opt.offsets[i] + opt.params[i].numel())
            g, m, b = (t[part].view(p.shape) for t in (opt.flat_g, moments, before))
            check_matrix(p, opt._slots[i][2], muon_definition(b, g, m, harness.poly_lr(0.002, it, 50), 5e-4, 0.95, True,
                                                              "match_rms_adamw"), 0.002, "match_rms_adamw")
    q.put((rank, opt.flat_p.cpu().numpy(), opt.flat_g.cpu().numpy(), len(tr.buckets.buckets)))
    dist.barrier()
    dist.destroy_process_group()


@gpu
def test_two_ranks_train_with_muon():
    """Two ranks, an image each, gradients summed in buckets of the flat buffer: every update follows from the summed
    gradient, and the replicas stay the same bit for bit."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted((q.get(timeout=100) for _ in procs), key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert res[0][3] >= 2
    assert (res[0][1] == res[1][1]).all() and (res[0][2] == res[1][2]).all()
