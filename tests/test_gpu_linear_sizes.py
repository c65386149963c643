"""The linear block at sizes with one very long side, and the large tiles of its products.  Tolerances as in
test_gpu_linear.py; where every product and sum is a whole number that f32 and the type hold, results are equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def whole(gen, *shape, top=2):
    return torch.randint(-top, top + 1, shape, generator=gen, device="cuda", dtype=torch.int8)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,k,n", [(1, 4_096_000, 8), (7, 4_096_001, 8), (40, 4_096_003, 5), (8, 8, 4_096_000),
                                      (40, 7, 4_096_001), (1, 3, 4_096_003)])
def test_a_long_side_and_its_gradients(rows, k, n, dt):
    """A flattened 160^3 volume as inputs or outputs.  Every 4099th value of a long sum is not zero: whole numbers below
    2^8 at each step, so that every order of summation gives them exactly."""
    from cgan3d_amd.model.linear import fused_linear
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x, w, dy = whole(g, rows, k), whole(g, n, k), whole(g, rows, n, top=1)
    if k > 100:
        x *= (torch.arange(k, device="cuda") % 131071 == 5).to(torch.int8)  # 31 products of at most 4
    if n > 100:
        dy *= (torch.arange(n, device="cuda") % 131071 == 7).to(torch.int8)
    t = DT[dt]
    xs, ws = x.to(t).requires_grad_(True), w.to(t).requires_grad_(True)
    b = torch.zeros(n, dtype=t, device="cuda", requires_grad=True)
    y = fused_linear(xs, ws, b)
    y.backward(dy.to(t))
    x, w, dy = x.float(), w.float(), dy.float()
    assert torch.equal(y.detach().float(), x @ w.T), "y"
    assert torch.equal(xs.grad.float(), dy @ w), "dx"
    assert torch.equal(ws.grad.float(), dy.T @ x), "dw"
    assert torch.equal(b.grad.float(), dy.sum(0)), "db"


def test_grids_beyond_one_axis():
    """More blocks than a grid of one axis holds: one row, three rows, and the column sums alone."""
    from cgan3d_amd import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    for rows, k, n, t in ((1, 4, (1 << 26) + 5, torch.bfloat16), (3, 1, (1 << 27) + 19, torch.float32)):
        x, w = whole(g, rows, k).to(t), whole(g, n, k).to(t)
        y = torch.full((rows, n), 7.0, dtype=t, device="cuda")
        ops.linear(x, w, y)
        for i in range(rows):
            want = torch.zeros(n, dtype=torch.float32, device="cuda")
            for q in range(k):
                want += x[i, q].float() * w[:, q].float()
            assert torch.equal(y[i].float(), want), (rows, n)
        del y, w, want
    n = (1 << 27) + 19
    dy, db = whole(g, 2, n).float(), torch.full((n,), 7.0, device="cuda")
    ops.linear_backward(dy, torch.empty(2, 0, device="cuda"), torch.empty(n, 0, device="cuda"), dbias=db)
    assert torch.equal(db, dy[0] + dy[1])


@pytest.mark.parametrize("dt", list(DT))
def test_empty_sums_of_many_values(dt):
    """k, n or rows of zero beside sides of any route: the epilogue of zeros, and gradients of zeros."""
    from cgan3d_amd import _lib as L
    from cgan3d_amd import ops
    t = DT[dt]
    for rows, n in ((100, 70), (700, 33), (5000, 300)):
        b, r = torch.randn(n, device="cuda").to(t), torch.randn(rows, n, device="cuda").to(t)
        y = torch.full((rows, n), 7.0, dtype=t, device="cuda")
        pre = torch.full((rows, n), 7.0, dtype=ops.linear_preact_dtype(t), device="cuda")
        ops.linear(torch.empty(rows, 0, dtype=t, device="cuda"), torch.empty(n, 0, dtype=t, device="cuda"), y, bias=b,
                   residual=r, act=L.ACT_RELU, preact=pre)
        want = b.double().clamp_min(0) + r.double()
        low = torch.finfo(t).smallest_normal if dt == "f16" else 0
        assert ((y.double() - want).abs() <= torch.finfo(t).eps / 2 * 1.01 * want.abs() + low).all()
        assert ((pre.double() - b.double()).abs() <= 2.0 ** -11 * b.double().abs() + 2.0 ** -25).all()
        dx = torch.full((rows, n), 7.0, dtype=t, device="cuda")
        ops.linear_backward(torch.empty(rows, 0, dtype=t, device="cuda"), r, torch.empty(0, n, dtype=t, device="cuda"), dx=dx)
        assert not dx.any()
        dw, db = torch.full((n, rows), 7.0, dtype=t, device="cuda"), torch.full((n,), 7.0, dtype=t, device="cuda")
        ops.linear_backward(torch.empty(0, n, dtype=t, device="cuda"), torch.empty(0, rows, dtype=t, device="cuda"),
                            torch.empty(n, rows, dtype=t, device="cuda"), dw=dw, dbias=db)
        assert not dw.any() and not db.any()


@pytest.fixture
def guarded(monkeypatch):
    """Every workspace is exactly as large as was asked for, with a pattern behind it."""
    from cgan3d_amd import ops
    held = []

    def workspace(ws, need, what, device):
        assert need >= 0
        buf = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device=device)
        held.append((what, need, buf))
        return buf[:need]
    monkeypatch.setattr(ops, "_workspace", workspace)

    def check(what):
        torch.cuda.synchronize()
        for name, need, buf in held:
            assert (buf[need:] == 0xA5).all(), f"{name} wrote behind its {need} bytes: {what}"
        held.clear()
    return check


@pytest.mark.parametrize("dt", list(DT))
def test_workspaces_are_large_enough(guarded, dt):
    from cgan3d_amd import _lib as L
    from cgan3d_amd.model.linear import fused_linear
    t = DT[dt]
    for rows, k, n in ((3, 64, 48), (20, 33, 50), (500, 64, 64), (129, 129, 257), (777, 1001, 515), (64, 16384, 64), (1200, 3000, 1200),
                       (4001, 203, 4003), (520, 1000, 5000), (70, 300, 9001), (100, 0, 70), (70000, 100, 70)):
        for act in (L.ACT_NONE, L.ACT_SILU):
            leaves = [torch.randn(*s, device="cuda").to(t).requires_grad_(True) for s in ((rows, k), (n, k), (n,))]
            y = fused_linear(*leaves, act=act)
            dy = torch.randn(rows, n, device="cuda").to(t)
            torch.autograd.grad(y, leaves, dy, retain_graph=True)
            for leaf in leaves:
                torch.autograd.grad(y, leaf, dy, retain_graph=True)
            guarded(f"{rows}x{k}->{n} {act}")


def test_workspaces_of_the_iteration_are_large_enough(guarded):
    from cgan3d_amd import ops
    for shape in ((1, 1, 7), (3, 16, 343), (40, 64, 300), (1, 64, 70000), (14, 100, 72), (3, 1001, 333), (1, 600, 5000), (1, 2049, 2100)):
        g = torch.randn(*shape, device="cuda")
        for kw in ({}, dict(steps=0), dict(steps=1, coefficients=(70.0, 0.0, -61.0))):
            ops.orthogonalize(g, **kw)
            guarded(f"{shape} {kw}")
    mats, vecs, n = [], [], 0
    for r, c in [(16, 343), (64, 1728), (1, 5488), (100, 130), (2100, 300)] * 9:
        mats.append((n, r, c, 1.0))
        vecs.append((n + r * c, 5))
        n += r * c + 5
    segs = ops.MuonSegments(n, mats, vecs)
    p, g, m, v = (torch.randn(n, device="cuda").abs() for _ in range(4))
    hyper = torch.tensor([0.5, 0.75, 0.0, 1.0, 0.0, 0.0, 0.1, 0.9, 0.999, 1e-8], device="cuda")
    for kw in ({}, dict(steps=2, coefficients=(70.0, 0.0, -61.0))):
        ops.muon_step(p, g, m, v, segs, hyper, **kw)
        guarded(f"muon {kw}")
    assert float(hyper[4]) == 2.0
