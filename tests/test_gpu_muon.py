"""Newton-Schulz orthogonalisation (ops.orthogonalize) and the Muon optimiser (trainer.optim.FusedMuon)
against float64 on the CPU.

Tolerance of the iteration.  One step maps an error D of the iterate (Frobenius norm) to at most a D, a
= 3.4445 the largest slope of the quintic on [0, 1.2], and commits its own: the sums of products in f32
round like a random walk, so a few half steps u = 2^-24 of the iterate's norm; four are allowed.  Over the
steps that is 4 u sum_k a^(steps - k) |X_k|, computed from the exact iterates, plus the rounding of the
result to its type (half a step of each value).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NS = (3.4445, -4.7750, 2.0315)
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ns64(g, steps=5, co=NS, eps=1e-7):
    """(result, tolerance in the Frobenius norm) of one matrix in float64."""
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    x = x / (x.square().sum().sqrt() + eps)
    a, b, c = co
    tol = 0.0
    for k in range(steps):
        tol = abs(a) * (tol + 4 * U * float(x.norm()))
        m = x @ x.T
        x = a * x + (b * m + c * m @ m) @ x
    tol += 4 * U * float(x.norm())
    return (x.T if tall else x), tol


def check_ns(got, g, dt, what, **kw):
    want, tol = ns64(g, **kw)
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    half = torch.finfo(DT[dt]).eps / 2
    tol += half * float(want.norm()) + (2.0 ** -25 * math.sqrt(want.numel()) if dt == "f16" else 0)
    err = float((got - want).norm())
    assert err <= tol, f"{what}: off by {err:.3e}, bound {tol:.3e}, norm {float(want.norm()):.3e}"


def grad_like(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    lead = shape[:-2]
    v = torch.randn(*shape, generator=g) + torch.randn(*lead, m, 1, generator=g) * torch.randn(*lead, 1, n, generator=g)
    return (v * torch.exp(0.5 * torch.randn(*lead, m, 1, generator=g)) * 1e-3).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (1, 5488), (2, 3), (16, 343), (32, 432), (64, 1728), (1728, 64), (63, 65), (64, 64),
          (65, 64), (65, 66), (70, 129), (33, 1000), (129, 128), (128, 640), (200, 200), (333, 500), (500, 333),
          (257, 1031), (512, 1024), (20, 9001), (8500, 33), (60, 20000)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dt):
    from cgan3d_amd import ops
    g = grad_like(*shape, seed=shape[0] + 3 * shape[1], dtype=DT[dt])
    check_ns(ops.orthogonalize(g.cuda()), g, dt, f"{shape} {dt}")


@pytest.mark.parametrize("shape", [(1100, 2304), (2301, 1030)])
def test_orthogonalize_large(shape):
    """The largest tiles, and a transposed result through them."""
    from cgan3d_amd import ops
    g = grad_like(*shape, seed=9)
    check_ns(ops.orthogonalize(g.cuda()), g, "f32", f"{shape}")


def test_orthogonalize_strided():
    """Rows of a wider tensor, through the C entry point's row strides: what lies between stays."""
    import ctypes
    from cgan3d_amd import _lib as L
    lib = L.lib()
    for rows, cols in ((40, 70), (90, 130), (300, 45), (200, 120)):
        g = grad_like(rows, cols, seed=3)
        src = torch.full((rows, cols + 5), 7.0).cuda()
        src[:, 2:2 + cols] = g.cuda()
        out = torch.full((rows, cols + 9), 7.0).cuda()
        m = (L.OrthoMat * 1)(L.OrthoMat(src[:, 2:].data_ptr(), out[:, 3:].data_ptr(), cols + 5, cols + 9, rows, cols))
        need = lib.cgan3d_orthogonalize_ws_bytes(m, 1, L.DT_F32)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        co = (ctypes.c_float * 3)(*NS)
        L.check(lib.cgan3d_orthogonalize(m, 1, L.DT_F32, 5, co, 1e-7, ws.data_ptr(), need, L.stream()))
        check_ns(out[:, 3:3 + cols], g, "f32", f"{rows}x{cols}")
        out[:, 3:3 + cols] = 7.0
        assert (out == 7.0).all()


@pytest.mark.parametrize("shape", [(3, 20, 30), (2, 2, 40, 16), (5, 64, 200), (2, 130, 70), (4, 96, 256), (0, 8, 8),
                                   (3, 0, 5)])
def test_orthogonalize_batches(shape):
    from cgan3d_amd import ops
    g = grad_like(*shape, seed=5)
    for m in range(math.prod(shape[:-2]) if g.numel() else 0):  # unlike sizes: each matrix has its own norm
        g.view(-1, *shape[-2:])[m] *= 10.0 ** (m - 2)
    got = ops.orthogonalize(g.cuda())
    assert got.shape == g.shape
    if g.numel():
        for m, (a, e) in enumerate(zip(got.view(-1, *shape[-2:]), g.view(-1, *shape[-2:]))):
            check_ns(a, e, "f32", f"matrix {m} of {shape}")


def test_orthogonalize_long_lists():
    """More matrices than one launch describes."""
    from cgan3d_amd import ops
    for b, m, n in ((70, 9, 12), (40, 100, 72)):
        g = grad_like(b, m, n, seed=8)
        got = ops.orthogonalize(g.cuda())
        for i in range(b):
            check_ns(got[i], g[i], "f32", f"matrix {i} of {b}")


@pytest.mark.parametrize("shape", [(40, 50), (100, 300)])
def test_orthogonalize_hard_matrices(shape):
    """Rank one, a zero matrix, a tiny and a huge one, one with a zero row, an orthogonal one."""
    from cgan3d_amd import ops
    m, n = shape
    g = torch.Generator().manual_seed(2)
    base = torch.randn(m, n, generator=g)
    zero_row = base.clone()
    zero_row[3] = 0
    cases = {"rank one": torch.randn(m, 1, generator=g) * torch.randn(1, n, generator=g), "zero": torch.zeros(m, n),
             "tiny": base * 1e-25, "huge": base * 1e25, "zero row": zero_row, "orthogonal": torch.linalg.qr(base.T)[0].T}
    for name, v in cases.items():
        v = v.contiguous()
        got = ops.orthogonalize(v.cuda(), eps=1e-30 if name == "tiny" else 1e-7)
        check_ns(got, v, "f32", name, eps=1e-30 if name == "tiny" else 1e-7)
    assert not ops.orthogonalize(torch.zeros(m, n).cuda()).any()
    assert not ops.orthogonalize(zero_row.cuda())[3].any()


@pytest.mark.parametrize("shape", [(24, 40), (90, 120)])
def test_orthogonalize_settings(shape):
    from cgan3d_amd import ops
    g = grad_like(*shape, seed=4)
    for steps in (0, 1, 2, 3, 7):
        check_ns(ops.orthogonalize(g.cuda(), steps=steps), g, "f32", f"{steps} steps", steps=steps)
    co = (1.5, -0.5, 0.0)
    check_ns(ops.orthogonalize(g.cuda(), steps=12, coefficients=co), g, "f32", "cubic", steps=12, co=co)
    inplace = g.cuda()
    assert ops.orthogonalize(inplace, out=inplace) is inplace
    check_ns(inplace, g, "f32", "in place")
    view = torch.zeros(shape[1], shape[0] + 3).cuda()
    view[:, :shape[0]] = g.T.cuda()
    check_ns(ops.orthogonalize(view[:, :shape[0]].T), g, "f32", "transposed view")


@pytest.mark.parametrize("shape", [(24, 40), (130, 80), (3, 90)])
def test_orthogonalize_coefficients_out_of_range(shape):
    """Coefficients whose iterates leave the range that the planes hold run on f32 products.  Bound, in Frobenius norms:
    a product of K terms is off by K u |A| |B|, a sum by u of its terms, and a step passes an error on by
    |a| + 3 |b| n^2 + 5 |c| n^4 at most, n = |X|."""
    from cgan3d_amd import ops
    g = grad_like(*shape, seed=6)
    s, l = min(shape), max(shape)
    for co in ((2.0, -65.0, 60.0), (70.0, 0.0, -61.0)):
        a, b, c = (abs(v) for v in co)
        for steps in (1, 2):
            x = (g.double() if shape[0] <= shape[1] else g.double().T)
            x = x / (x.square().sum().sqrt() + 1e-7)
            tol = 4 * U * float(x.norm())
            for _ in range(steps):
                n = float(x.norm())
                dm = (l + 2) * U * n ** 2
                db = b * dm + c * (2 * n ** 2 * dm + (s + 2) * U * n ** 4) + 2 * U * (b * n ** 2 + c * n ** 4)
                step = db * n + (s + 2) * U * (b * n ** 2 + c * n ** 4) * n + 3 * U * (a * n + b * n ** 3 + c * n ** 5)
                tol = (a + 3 * b * n ** 2 + 5 * c * n ** 4) * tol + 1.01 * step
                m = x @ x.T
                x = co[0] * x + (co[1] * m + co[2] * m @ m) @ x
            want = x if shape[0] <= shape[1] else x.T
            err = float((ops.orthogonalize(g.cuda(), steps=steps, coefficients=co).double().cpu() - want).norm())
            assert err <= tol, f"{co}, {steps} steps: off by {err:.3e}, bound {tol:.3e}, norm {float(want.norm()):.3e}"
            assert tol < 0.02 * float(want.norm()), "the bound says something"


@pytest.mark.parametrize("shape", [(20, 30), (80, 130)])
def test_orthogonalize_nonfinite(shape):
    """A NaN or an infinity makes its own matrix NaN, and no other."""
    from cgan3d_amd import ops
    g = grad_like(3, *shape, seed=6)
    clean = ops.orthogonalize(g.cuda())
    for bad in (float("nan"), float("inf")):
        h = g.clone()
        h[1, 2, 3] = bad
        got = ops.orthogonalize(h.cuda())
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
        assert got[1].isnan().any()


def test_orthogonalize_graph_and_repeat():
    from cgan3d_amd import ops
    for shape in ((2, 48, 500), (3, 160, 96)):
        g, h = grad_like(*shape, seed=1).cuda(), grad_like(*shape, seed=2).cuda()
        wants = [ops.orthogonalize(v) for v in (g, h)]
        assert torch.equal(ops.orthogonalize(g), wants[0])
        static, out = g.clone(), torch.empty_like(g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.orthogonalize(static, out=out)
        for v, want in ((g, wants[0]), (h, wants[1]), (g, wants[0])):
            static.copy_(v)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


# --- the optimiser ------------------------------------------------------------------------------
class Ref:
    """FusedMuon in float64, parameter by parameter."""

    def __init__(self, params, lr=0.02, momentum=0.95, weight_decay=0.0, nesterov=True, vector_lr=3e-4,
                 vector_betas=(0.9, 0.999), vector_eps=1e-8, adjust_lr="original", weight_clip=None, eps=1e-7):
        self.p = [p.detach().double().cpu().clone() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.tol = [torch.zeros(()).double() for _ in self.p]
        self.kw, self.t = dict(locals()), 0

    def step(self, grads):
        k = self.kw
        self.t += 1
        for i, g in enumerate(grads):
            g = g.detach().double().cpu()
            if g.dim() >= 2:
                self.m[i] += (1 - k["momentum"]) * (g - self.m[i])
                u = g + k["momentum"] * (self.m[i] - g) if k["nesterov"] else self.m[i]
                r = g.shape[0]
                c = g.numel() // r
                o, tol = ns64(u.reshape(r, c), eps=k["eps"])
                scale = math.sqrt(max(1, r / c)) if k["adjust_lr"] == "original" else 0.2 * math.sqrt(max(r, c))
                self.p[i] = self.p[i] * (1 - k["lr"] * k["weight_decay"]) - k["lr"] * scale * o.reshape(g.shape)
                # the update's own error (its input is off by a few u, which the iteration carries as its own)
                self.tol[i] = self.tol[i] + k["lr"] * scale * 2 * tol + 4 * U * self.p[i].norm()
            else:
                b1, b2 = k["vector_betas"]
                self.m[i] += (1 - b1) * (g - self.m[i])
                self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
                d = (self.v[i] / (1 - b2 ** self.t)).sqrt() + k["vector_eps"]
                self.p[i] = self.p[i] - k["vector_lr"] / (1 - b1 ** self.t) * self.m[i] / d
                # powf's and the quotients' few u, on an update of at most ~lr per value
                self.tol[i] = self.tol[i] + k["vector_lr"] * 1e-4 * math.sqrt(g.numel()) + 4 * U * self.p[i].norm()
            if k["weight_clip"]:
                self.p[i] = self.p[i].clamp(-k["weight_clip"], k["weight_clip"])

    def check(self, params, what):
        for i, p in enumerate(params):
            err, tol = float((p.detach().double().cpu() - self.p[i]).norm()), float(self.tol[i])
            assert err <= tol, f"{what} parameter {i} {tuple(p.shape)}: off by {err:.3e}, bound {tol:.3e}"


def _net():
    """Parameters of a small generator (2 blocks) and a few extra matrices, in an arena."""
    from cgan3d_amd.model.generator import ResnetGenerator
    torch.manual_seed(3)
    mod = torch.nn.Module()
    mod.gen = ResnetGenerator(2, 2, 8)
    mod.extra = torch.nn.ParameterList([torch.nn.Parameter(0.1 * torch.randn(s))
                                        for s in ((150, 90), (90, 150), (7,), (3, 1), (1, 1), (), (130, 2, 3, 4))])
    return mod.cuda()


@pytest.mark.parametrize("kw", [dict(), dict(lr=0.1, weight_decay=0.1, nesterov=False, adjust_lr="match_rms_adamw"),
                                dict(momentum=0.0, weight_clip=0.05, vector_betas=(0.0, 0.9), vector_lr=1e-2)])
def test_muon_steps(kw):
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.trainer.optim import FusedMuon
    mod = _net()
    arena = Arena(mod, torch.device("cuda"))
    opt = FusedMuon(arena, **kw)
    ref = Ref(arena.params, **kw)
    for t in range(3):
        for i, p in enumerate(arena.params):
            g = grad_like(p.shape[0], p.numel() // p.shape[0], seed=100 * t + i) if p.dim() >= 2 else \
                1e-3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * t + i))
            p.grad.copy_(g.reshape(p.shape))
        opt.step()
        ref.step([p.grad for p in arena.params])
        ref.check(arena.params, f"step {t} {kw}")
        assert float(opt.hyper[4]) == t + 1
    for i, p in enumerate(arena.params):
        st = opt.state[p]
        m = st["momentum_buffer" if p.dim() >= 2 else "exp_avg"]
        assert torch.allclose(m.double().cpu(), ref.m[i], rtol=1e-5, atol=1e-9)


def test_muon_many_segments():
    """More matrices (of both kinds) and vectors than one launch takes, and one whose slabs outnumber a block's."""
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.trainer.optim import FusedMuon
    gen = torch.Generator().manual_seed(7)
    mod = torch.nn.Module()
    shapes = [(5, 9001), (8200, 6)]
    for i in range(33):
        shapes += [(1 + i, 3 + 2 * i), (4 + i,)]  # a vector between two matrices is a segment of its own
        if i % 2:
            shapes += [(65 + i, 70 + 3 * i)]
    mod.ps = torch.nn.ParameterList([torch.nn.Parameter(0.1 * torch.randn(s, generator=gen)) for s in shapes])
    arena = Arena(mod.cuda(), torch.device("cuda"))
    opt, ref = FusedMuon(arena, weight_decay=0.1), Ref(arena.params, weight_decay=0.1)
    for t in range(2):
        for i, p in enumerate(arena.params):
            p.grad.copy_(grad_like(*p.shape, seed=200 * t + i) if p.dim() == 2 else
                         1e-3 * torch.randn(p.shape, generator=gen))
        opt.step()
        ref.step([p.grad for p in arena.params])
        ref.check(arena.params, f"step {t}")
        assert float(opt.hyper[4]) == t + 1


def test_muon_state_dict_and_scheduler():
    """A resumed optimiser goes on with the same bits; a scheduler drives both groups' rates."""
    from torch.optim.lr_scheduler import MultiStepLR
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.trainer.optim import FusedMuon
    mods = [_net(), _net()]
    opts = [FusedMuon(Arena(m, torch.device("cuda")), lr=0.05) for m in mods]
    scheds = [MultiStepLR(o, milestones=[1], gamma=0.1) for o in opts]

    def grads(o, t):
        o.arena.grad.copy_(1e-3 * torch.randn(o.arena.numel, generator=torch.Generator().manual_seed(t)))
    for t in range(2):
        grads(opts[0], t)
        opts[0].step()
        scheds[0].step()
    assert [round(g["lr"], 9) for g in opts[0].param_groups] == [0.005, 3e-5]
    opts[1].arena.flat.copy_(opts[0].arena.flat)
    opts[1].load_state_dict(opts[0].state_dict())
    for t in (2, 3):
        for o in opts:
            grads(o, t)
            o.step()
    a, b = (o.arena for o in opts)
    assert torch.equal(a.flat, b.flat) and torch.equal(a.exp_avg, b.exp_avg) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)
    assert torch.equal(opts[0].hyper, opts[1].hyper) and float(opts[0].hyper[0]) == pytest.approx(0.005)


def test_muon_plan_and_graph():
    """A recorded and a captured step follow new gradients and a changed rate, bit for bit as eager steps."""
    from cgan3d_amd import ops
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.trainer.optim import FusedMuon
    opts = [FusedMuon(Arena(_net(), torch.device("cuda"))) for _ in range(3)]
    for o in opts:  # every kernel once before the capture
        o.arena.grad.fill_(1e-3)
        o.step()
    ops.plan_begin()
    opts[1].launch()
    plan = ops.plan_end()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[2].launch()
    for t in range(3):
        g = 1e-3 * torch.randn(opts[0].arena.numel, generator=torch.Generator().manual_seed(t))
        for o in opts:
            o.arena.grad.copy_(g)
            for gr in o.param_groups:
                gr["lr"] *= 0.5
            o.sync_hyper()
        opts[0].launch()
        plan.run()
        graph.replay()
        torch.cuda.synchronize()
        for o in opts[1:]:
            assert torch.equal(o.arena.flat, opts[0].arena.flat), t
            assert torch.equal(o.arena.exp_avg, opts[0].arena.exp_avg), t
            assert float(o.hyper[4]) == t + 2


def test_segments_leave_the_rest():
    """Values of the arena outside every segment stay as they were."""
    from cgan3d_amd import ops
    n = 20000
    g = torch.Generator().manual_seed(1)
    flat, grad = torch.randn(n, generator=g).cuda(), 10 * torch.randn(n, generator=g).cuda()
    m, v = torch.randn(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    segs = ops.MuonSegments(n, [(101, 30, 50, 1.0), (3000, 100, 90, 1.0), (13000, 0, 5, 1.0)], [(5, 7), (12500, 1)])
    hyper = torch.tensor([10.0, 0.9, 0.0, 1.0, 0.0, 0.0, 1e-2, 0.9, 0.99, 1e-8]).cuda()
    old = [t.clone() for t in (flat, m, v)]
    ops.muon_step(flat, grad, m, v, segs, hyper)
    inside = torch.zeros(n, dtype=torch.bool)
    for lo, k in ((101, 1500), (3000, 9000), (5, 7), (12500, 1)):
        inside[lo:lo + k] = True
    for t, o in zip((flat, m), old):
        assert torch.equal((t != o).cpu(), inside)
    vec = torch.zeros(n, dtype=torch.bool)
    vec[5:12], vec[12500] = True, True
    assert torch.equal((v != old[2]).cpu(), vec)


def test_linear_layers_trained_with_muon():
    """A run of the operators together: two linear blocks with a residual, gradients, two Muon steps, against
    float64."""
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.model.linear import LinearBlock
    from cgan3d_amd.trainer.optim import FusedMuon
    torch.manual_seed(0)
    a, b = LinearBlock(48, 96, torch.nn.GELU), LinearBlock(96, 48, torch.nn.Identity)
    net = torch.nn.ModuleList([a, b])
    ref = [p.detach().double().clone().requires_grad_(True) for p in net.parameters()]
    arena = Arena(net.cuda(), torch.device("cuda"))
    opt = FusedMuon(arena, lr=0.02, weight_decay=0.01)
    oracle = Ref(arena.params, lr=0.02, weight_decay=0.01)
    g = torch.Generator().manual_seed(5)
    x, t = torch.randn(2, 5, 6, 7, 48, generator=g), torch.randn(2, 5, 6, 7, 48, generator=g)
    for step in range(2):
        opt.zero_grad()
        y = b(a(x.cuda()), residual=x.cuda())
        loss = (y - t.cuda()).square().mean()
        loss.backward()
        w1, b1, w2, b2 = ref
        xd = x.double()
        lr = ((torch.nn.functional.gelu(xd @ w1.T + b1) @ w2.T + b2 + xd) - t.double()).square().mean()
        grads = torch.autograd.grad(lr, ref)
        for p, e in zip(arena.params, grads):
            # f32 sums of up to 420 terms, twice, on weights that are off by f32's own steps
            assert float((p.grad.double().cpu() - e).norm()) <= 1e-5 * float(e.norm()), step
        opt.step()
        oracle.step([p.grad for p in arena.params])  # from the device's gradients: the step alone is compared
        oracle.check(arena.params, f"step {step}")
        ref = [p.detach().double().cpu().clone().requires_grad_(True) for p in arena.params]


@pytest.mark.parametrize("precision", ["f32", "bf16"])
def test_trainer_with_muon(tmp_path, precision, monkeypatch):
    """The drop-in Trainer with partial(FusedMuon, ...): steps from a replayed plan and eager ones, a checkpoint
    resumes."""
    from functools import partial
    import test_gpu_trainer as tt
    from cgan3d_amd.model.discriminator import PatchGANDiscriminator
    from cgan3d_amd.model.generator import ResnetGenerator
    from cgan3d_amd.model.loss import HULoss
    from cgan3d_amd.trainer.optim import FusedMuon
    from cgan3d_amd.trainer.Trainer import Trainer

    def make(plans, ckpt=None):
        torch.manual_seed(0)
        monkeypatch.setenv("CGAN3D_TRAINER_PLANS", "1" if plans else "0")
        d = dict(channels_in=1, init_channels_out=8, discriminator_depth=3, negative_slope=0.2)
        return Trainer(10, 1, 100, 1, 1, 100, 1000, partial(ResnetGenerator, 1, 2, 8),
                       partial(PatchGANDiscriminator, **d, norm_layer=torch.nn.Identity),
                       partial(FusedMuon, lr=0.01), partial(torch.optim.Adam, lr=1e-4, betas=(0.0, 0.9)),
                       HULoss(-0.2, 0.6), tt._LoggerInterface(), torch.device("cuda"), checkpoint_dir=ckpt,
                       checkpoint_every=None, precision=precision)
    runs = [make(True, tmp_path), make(False)]
    before = runs[0].optimizer_G.arena.flat.clone()
    for it in range(4):
        batch = tt._patches(np.random.default_rng(it))
        for tr in runs:
            torch.cuda.manual_seed(it)
            log = tr.train_step(batch, it)
            assert all(np.isfinite(float(v)) for v in log.values())
    flats = [tr.optimizer_G.arena.flat for tr in runs]
    assert any(p is not None for p in runs[0]._plans.values())
    assert not torch.equal(flats[0], before) and runs[0].optimizer_G._host_step == 4
    runs[0].save_checkpoint(4)
    again = make(True, tmp_path)
    assert torch.equal(again.optimizer_G.arena.flat, flats[0]) and again.optimizer_G._host_step == 4
    assert torch.equal(again.optimizer_G.arena.exp_avg, runs[0].optimizer_G.arena.exp_avg)
    again.train_step(tt._patches(np.random.default_rng(9)), 4)


def test_engine_plan_with_muon_is_bit_identical():
    """The bf16 step at 64^3 (whose gradients are summed in a fixed order) with the generator under Muon: a
    replayed plan and eager steps leave the same bits, and the update is the one of the gradient the
    device consumed."""
    from cgan3d_amd.data.synthetic import synth_patches
    from cgan3d_amd.engine import Arena, StepEngine
    from cgan3d_amd.trainer.optim import FusedMuon
    from test_gpu_step import _models
    S, b = 64, 2
    engs = []
    for _ in range(2):
        g, d = _models(dict(n_resnet_blocks=2, n_updownsample_blocks=2, init_channels_out=16))
        opt = FusedMuon(Arena(g, torch.device("cuda")), lr=0.01)
        engs.append(StepEngine(g, d, g.config, d.config, b, b, (S, S, S), precision="bf16", g_optim=opt))
    engs[1].record()
    oracle = Ref(engs[0].g_arena.params, lr=0.01)
    for j in range(3):
        opt, _ = synth_patches(b, S, 300 + j)
        sub, seg = synth_patches(b, S, 400 + j)
        bt = (torch.from_numpy(opt).cuda(), torch.from_numpy(sub).cuda(), torch.from_numpy(seg).cuda(),
              torch.full((b,), 0.25 + 0.1 * j, device="cuda"))
        for e in engs:
            e.load_inputs(*bt)
        engs[0].step()
        engs[1].run_plan()
        torch.cuda.synchronize()
        a1, a2 = (e.g_arena for e in engs)
        for t1, t2 in ((a1.grad, a2.grad), (a1.flat, a2.flat), (a1.exp_avg, a2.exp_avg), (a1.exp_avg_sq, a2.exp_avg_sq)):
            assert torch.equal(t1, t2), f"step {j}"
        oracle.step(list(a1.gviews.values()))
        oracle.check(a1.params, f"step {j}")
