"""Refusals and host logic of the linear block, the orthogonalisation and the Muon optimiser (no GPU): the
wrappers' checks in dry-run mode, and the C entry points' own, which launch nothing when they refuse."""
import ctypes as C

import pytest
import torch
from torch import nn


@pytest.fixture
def dry():
    from cgan3d_amd import ops
    ops.DRY_RUN = True
    yield ops
    ops.DRY_RUN = False


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_linear_refuses_bad_operands(dry):
    from cgan3d_amd import _lib as L
    x, w, y = t(6, 8), t(5, 8), t(6, 5)
    dry.linear(x, w, y, bias=t(5), residual=t(6, 5), act=L.ACT_GELU, preact=t(6, 5))
    bad = [
        (TypeError, dict(x=t(6, 8, dtype=torch.float64))), (TypeError, dict(w=t(5, 8, dtype=torch.bfloat16))),
        (TypeError, dict(y=t(6, 5, dtype=torch.float16))), (ValueError, dict(w=t(5, 7))), (ValueError, dict(y=t(5, 6))),
        (ValueError, dict(y=t(5, 6).T)), (ValueError, dict(x=t(6, 16)[:, ::2])), (ValueError, dict(x=t(1, 8).expand(6, 8))),
        (ValueError, dict(x=t(2, 3, 8))), (ValueError, dict(bias=t(6))), (TypeError, dict(bias=t(5).half())),
        (ValueError, dict(residual=t(1, 5))), (ValueError, dict(preact=t(6, 4))), (TypeError, dict(preact=t(6, 5).half())),
        (ValueError, dict(act=L.ACT_NEG_DTANH)), (ValueError, dict(act=17)),
        (ValueError, dict(ws=t(8))), (ValueError, dict(x=t(6, 8).to("meta"), w=t(5, 8).to("meta"))),
    ]
    for err, change in bad:
        kw = dict(x=x, w=w, y=y) | change
        with pytest.raises(err):
            dry.linear(kw.pop("x"), kw.pop("w"), kw.pop("y"), **kw)


def test_linear_backward_refuses_bad_operands(dry):
    from cgan3d_amd import _lib as L
    dy, x, w = t(6, 5), t(6, 8), t(5, 8)
    dry.linear_backward(dy, x, w, dx=t(6, 8), dw=t(5, 8), dbias=t(5), act=L.ACT_RELU, preact=t(6, 5))
    dry.linear_backward(dy, x, w, dw=t(5, 8))
    for err, kw in ((ValueError, dict(act=L.ACT_RELU)), (ValueError, dict(dx=t(6, 7))), (ValueError, dict(dw=t(8, 5))),
                    (ValueError, dict(dw=t(5, 9)[:, :8])), (TypeError, dict(dx=t(6, 8).bfloat16())),
                    (ValueError, dict(dbias=t(8))), (ValueError, dict(act=L.ACT_GELU, preact=t(5, 5)))):
        with pytest.raises(err):
            dry.linear_backward(dy, x, w, **kw)
    with pytest.raises(ValueError):
        dry.linear_backward(t(1, 5).expand(6, 5), x, w, dx=t(6, 8))


def test_cpu_tensors_are_refused():
    from cgan3d_amd import ops
    from cgan3d_amd.model.linear import fused_linear
    with pytest.raises(ValueError, match="GPU"):
        fused_linear(t(3, 4), t(5, 4))
    with pytest.raises(ValueError, match="GPU"):
        ops.orthogonalize(t(3, 4))


def test_c_entries_refuse_without_launching():
    """Overlapping outputs, short workspaces, null pointers and bad sizes come back as CGAN3D_EINVAL."""
    from cgan3d_amd import _lib as L
    lib = L.load()
    buf = (C.c_char * 4096)()
    base = (C.addressof(buf) + 255) // 256 * 256

    def args(**kw):
        a = L.LinearArgs()
        d = dict(rows=4, k=4, n=4, dtype=0, act=0, x=base, ldx=4, w=base + 256, ldw=4, y=base + 512, ldy=4,
                 dy=base + 768, lddy=4) | kw
        for k, v in d.items():
            setattr(a, k, v)
        return a
    for kw in (dict(rows=-1), dict(k=-2), dict(n=-1), dict(dtype=3), dict(dtype=-1), dict(act=4), dict(act=7), dict(x=None),
               dict(w=None), dict(y=None), dict(ldx=3), dict(ldw=2), dict(ldy=3), dict(residual=base + 1024, ldr=3),
               dict(y=base), dict(y=base + 256 + 32), dict(preact=base + 512), dict(rows=1 << 41),
               dict(residual=base + 516, ldr=4), dict(bias=base + 520)):
        assert lib.cgan3d_linear_fwd(C.byref(args(**kw)), None, 0, None) == 22, kw
        assert b"cgan3d_linear_fwd" in lib.cgan3d_get_last_error()
    assert lib.cgan3d_linear_fwd(None, None, 0, None) == 22
    for kw in (dict(dy=None), dict(lddy=3), dict(act=1), dict(dx=base, lddx=4), dict(dx=base + 1024, lddx=3),
               dict(dw=base + 768), dict(dx=base + 1024, lddx=4, dw=base + 1024), dict(dbias=base + 256 + 8)):
        assert lib.cgan3d_linear_bwd(C.byref(args(**kw)), base + 2048, 1024, None) == 22, kw
    big = args(rows=1, k=1 << 20, n=4, ldx=1 << 20, ldw=1 << 20)
    need = lib.cgan3d_linear_fwd_ws_bytes(C.byref(big))
    assert need >= 0 and lib.cgan3d_linear_fwd_ws_bytes(C.byref(args(rows=-1))) == -1
    if need:
        assert lib.cgan3d_linear_fwd(C.byref(big), base, need - 1, None) == 22
        assert lib.cgan3d_linear_fwd(C.byref(big), base + 1, need, None) == 22
    co = (C.c_float * 3)(3.0, -4.0, 2.0)
    nan = (C.c_float * 3)(float("nan"), 0.0, 0.0)

    def ortho(m, n=1, dt=0, steps=5, c=co, eps=1e-7, ws=base, b=1 << 30):
        arr = (L.OrthoMat * 1)(L.OrthoMat(*m))
        return lib.cgan3d_orthogonalize(arr, n, dt, steps, c, eps, ws, b, None)
    ok = (base, base + 512, 4, 4, 4, 4)
    for m, kw in (((None, base, 4, 4, 4, 4), {}), ((base, None, 4, 4, 4, 4), {}), ((base, base, 3, 4, 4, 4), {}),
                  ((base, base, 4, 3, 4, 4), {}), ((base, base, 4, 4, -1, 4), {}), (ok, dict(dt=5)), (ok, dict(steps=-1)),
                  (ok, dict(steps=65)), (ok, dict(c=nan)), (ok, dict(c=None)), (ok, dict(eps=-1.0)),
                  (ok, dict(eps=float("nan"))), (ok, dict(b=16)), (ok, dict(ws=None)), (ok, dict(ws=base + 4)),
                  (ok, dict(n=-1))):
        assert ortho(m, **kw) == 22, (m, kw)
    seg = (L.MuonSeg * 1)(L.MuonSeg(-4, 4, 4, 1.0))
    assert lib.cgan3d_muon_ws_bytes(seg, 1) == -1
    seg = (L.MuonSeg * 1)(L.MuonSeg(0, 4, 4, 1.0))
    p = base
    assert lib.cgan3d_muon_step(p, p, p, p, seg, 1, p, 5, co, 1e-7, base, 16, None) == 22
    assert lib.cgan3d_muon_step(None, p, p, p, seg, 1, p, 5, co, 1e-7, base, 1 << 30, None) == 22


def test_orthogonalize_refuses(dry):
    with pytest.raises(ValueError):
        dry.orthogonalize(t(4))
    with pytest.raises(TypeError):
        dry.orthogonalize(t(4, 4, dtype=torch.float64))
    with pytest.raises(ValueError):
        dry.orthogonalize(t(4, 4), coefficients=(1.0, 2.0))
    with pytest.raises(ValueError):
        dry.orthogonalize(t(4, 4), out=t(4, 5))
    with pytest.raises(ValueError):
        dry.orthogonalize(t(4, 4), out=t(4, 4, dtype=torch.float16))
    buf = t(40)
    with pytest.raises(ValueError, match="overlaps"):
        dry.orthogonalize(buf[:16].view(4, 4), out=buf[8:24].view(4, 4))
    with pytest.raises(NotImplementedError):
        dry.orthogonalize(t(4, 4).requires_grad_(True))
    assert dry.orthogonalize(t(2, 0, 4)).shape == (2, 0, 4)
    assert dry.orthogonalize(t(0, 3, 4)).shape == (0, 3, 4)


def test_fused_linear_refuses(dry):
    from cgan3d_amd.model.linear import LinearBlock, fused_linear
    with pytest.raises(ValueError):
        fused_linear(t(3, 4), t(5, 6))
    with pytest.raises(ValueError):
        fused_linear(t(3, 4), t(5, 4), residual=t(1, 5))  # no broadcasting
    with pytest.raises(ValueError):
        fused_linear(t(3, 4), t(5, 4, 1))
    with pytest.raises(TypeError):
        fused_linear(t(3, 4), t(5, 4), t(5).half())
    for act in (nn.Sigmoid, nn.ELU):
        with pytest.raises(NotImplementedError):
            LinearBlock(4, 5, act)
    with pytest.raises(NotImplementedError):
        LinearBlock(4, 5, nn.GELU, approximate="tanh")
    blk = LinearBlock(4, 5, nn.LeakyReLU, negative_slope=0.2)
    assert set(blk.state_dict()) == {"linear.weight", "linear.bias"}
    x = t(2, 3, 4).requires_grad_(True)
    y = blk(x, residual=t(2, 3, 5))
    assert y.shape == (2, 3, 5)
    g, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    assert g.shape == x.shape
    with pytest.raises(NotImplementedError):  # first order only
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_muon_optimizer_layout(dry):
    """Every weight of the generator is a matrix segment of [first axis, the rest], neighbouring vectors are
    joined, nothing is left out."""
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.model.generator import ResnetGenerator
    from cgan3d_amd.trainer.optim import FusedMuon
    arena = Arena(ResnetGenerator(4, 2, 16), torch.device("cpu"))
    opt = FusedMuon(arena, lr=0.1, vector_lr=0.2)
    segs = [opt.segs.c[i] for i in range(opt.segs.n)]
    assert sum((s.rows or 1) * s.cols for s in segs) == arena.numel
    mats = {(s.rows, s.cols) for s in segs if s.rows}
    assert mats == {(16, 343), (32, 432), (64, 864), (64, 1728), (1, 5488)}
    assert len([s for s in segs if s.rows]) == 14 and len([s for s in segs if not s.rows]) == 14
    opt.step()
    opt.param_groups[1]["lr"] = 0.5
    opt.sync_hyper()
    assert opt.hyper.tolist() == pytest.approx([0.1, 0.95, 0.0, 1.0, 0.0, 0.0, 0.5, 0.9, 0.999, 1e-8])
    assert opt.state_dict()["param_groups"][0]["momentum"] == 0.95
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(vector_betas=(0.9, 1.0)), dict(adjust_lr="none"),
               dict(ns_coefficients=(1.0,)), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            FusedMuon(arena, **kw)


def test_muon_segments_refuse():
    from cgan3d_amd import ops
    for mats, vecs in (([(0, 4, 4, 1.0), (15, 2, 2, 1.0)], []), ([(0, 4, 4, 1.0)], [(10, 3)]), ([(90, 4, 4, 1.0)], []),
                       ([(-1, 2, 2, 1.0)], []), ([], [(0, 101)])):
        with pytest.raises(ValueError):
            ops.MuonSegments(100, mats, vecs)


def test_optimizer_from_partial(dry):
    from functools import partial
    from cgan3d_amd.engine import Arena
    from cgan3d_amd.trainer.optim import FusedAdam, FusedMuon, optimizer_from_partial

    def arena():
        return Arena(nn.Linear(4, 5), torch.device("cpu"))
    assert isinstance(optimizer_from_partial(partial(torch.optim.Adam, lr=0.1), arena()), FusedAdam)
    m = optimizer_from_partial(partial(FusedMuon, lr=0.3), arena(), weight_clip=0.01)
    assert isinstance(m, FusedMuon) and float(m.hyper[0]) == pytest.approx(0.3)
    assert float(m.hyper[5]) == pytest.approx(0.01)
    assert isinstance(optimizer_from_partial(FusedMuon, arena()), FusedMuon)
    for bad in (partial(torch.optim.SGD, lr=0.1), partial(FusedMuon, 3)):
        with pytest.raises((NotImplementedError, TypeError)):
            optimizer_from_partial(bad, arena())


@pytest.mark.parametrize("clip", [False, True])
def test_engine_step_with_muon_dry_run(dry, clip):
    """The engine's step with both networks under Muon: every launch passes its checks, and the generator is
    updated at once (the split update is Adam's)."""
    from cgan3d_amd.engine import Arena, StepEngine
    from cgan3d_amd.model.discriminator import PatchGANDiscriminator
    from cgan3d_amd.model.generator import ResnetGenerator
    from cgan3d_amd.trainer.optim import FusedMuon
    g = ResnetGenerator(1, 2, 8)
    d = PatchGANDiscriminator(1, 8, 3, negative_slope=0.2, **({} if clip else dict(norm_layer=nn.Identity)))
    dev = torch.device("cpu")
    go, do = FusedMuon(Arena(g, dev)), FusedMuon(Arena(d, dev), weight_clip=0.01 if clip else None)
    eng = StepEngine(g, d, g.config, d.config, 1, 1, (32, 32, 32), device=dev, g_optim=go, d_optim=do,
                     weight_clip=0.01 if clip else None)
    eng.step()
    assert eng.g_split == 0 and go._host_step == 1 and do._host_step == 1


def test_sizes_beyond_the_limits_are_refused():
    from cgan3d_amd import _lib as L
    lib, big = L.load(), (1 << 30) + 8
    for kw in (dict(k=big, n=4, ldx=big, ldw=big), dict(k=4, n=big, ldx=4, ldw=4, ldy=big, lddy=big),
               dict(k=4, n=4, rows=(1 << 40) + 1, ldx=4, ldw=4, ldy=4, lddy=4)):
        a = L.LinearArgs(**(dict(rows=2, ldy=4, lddy=4, x=64, w=64, y=64, dy=64, dx=64, lddx=big) | kw))
        assert lib.cgan3d_linear_fwd_ws_bytes(C.byref(a)) == -1 and lib.cgan3d_linear_bwd_ws_bytes(C.byref(a)) == -1
        assert b"too large" in lib.cgan3d_get_last_error()
    m = (L.OrthoMat * 1)(L.OrthoMat(64, 64, big, big, 2, big))
    assert lib.cgan3d_orthogonalize_ws_bytes(m, 1, L.DT_F32) == -1
    s = (L.MuonSeg * 1)(L.MuonSeg(0, 2, big, 1.0))
    assert lib.cgan3d_muon_ws_bytes(s, 1) == -1
