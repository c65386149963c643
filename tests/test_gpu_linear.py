"""The linear block (ops.linear / ops.linear_backward, model.linear) against float64 on the CPU.

Tolerances, element by element.  u = 2^-24 (half a step of f32), e = half a step of the tensors' type
(finfo.eps / 2).  A sum of K products in f32, in any order, is off by at most (K + 4) u S with S the sum of
the products' magnitudes and the bias's (the slack of 4: the bias's addition, the joining of split sums).
An activation passes an error on with at most its slope (below 1.13 for all of them) and adds a few u of
its own; the residual's addition adds u |y|; the store adds e |y|, for f16 at least half its smallest step.
Backward: dz = dy act'(z) is rounded to the type (e |dz|), and act'(z) is off by max |act''(z)| |z err|: for
bf16 z is kept as an f16 (2^-11 |z|, and |z act''(z)| < 1 for every activation here), otherwise it is off by
the forward sum's error (|act''| < 1.2); the short forms for 16-bit tensors are good to 2^-19.  ReLU and LeakyReLU, whose derivative jumps, get inputs on
a grid on which z is exact and never nearer to 0 than 1/64.
"""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY16 = 2.0 ** -25  # half of f16's smallest step
ACTS = ("none", "relu", "lrelu", "tanh", "gelu", "silu")
SLOPE = 0.2
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

SHAPES = [  # rows, k, n
    (1, 1, 1), (1, 64, 64), (1, 257, 130), (2, 8, 3), (3, 4096, 40), (5, 33, 1), (8, 512, 1000), (17, 64, 64),
    (64, 32, 64), (65, 31, 63), (100, 1, 7), (128, 300, 128), (129, 129, 257), (256, 1024, 256), (333, 515, 77),
    (1000, 16, 32), (4096, 64, 48), (5000, 3, 5), (2049, 40, 8), (512, 640, 384), (300, 2048, 520),
    # a few rows with many columns; f32 products that are split into planes (both gradients, one of them)
    (1, 4096, 4096), (2, 100, 5000), (4, 65, 4099), (3, 4096, 520), (9, 5000, 70), (16, 2048, 1000),
    (5, 31, 8200), (2, 1024, 8192), (12, 72, 9000), (1500, 1000, 1203), (2048, 512, 1024), (8000, 1000, 100),
]


def act64(z, name):
    return {"none": lambda t: t * 1, "relu": F.relu, "lrelu": lambda t: F.leaky_relu(t, SLOPE), "tanh": torch.tanh,
            "gelu": F.gelu, "silu": F.silu}[name](z)


def code(name):
    from cgan3d_amd import _lib
    return getattr(_lib, "ACT_" + name.upper())


def make(rows, k, n, dt, act, seed, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    if act in ("relu", "lrelu"):  # z: multiples of 1/32, odd multiples of 1/64 with the bias
        x = torch.randint(-4, 5, (rows, k), generator=g) / 4.0
        w = torch.randint(-4, 5, (n, k), generator=g) / 8.0
        b = torch.randint(-8, 8, (n,), generator=g) / 32.0 + 1 / 64.0
        if not bias:
            x[:] = x.abs().clamp_min(0.25)
            w[:] = w.abs().clamp_min(0.125)  # z > 0 without a bias
    else:
        x = torch.randn(rows, k, generator=g)
        w = torch.randn(n, k, generator=g) / math.sqrt(k)
        b = 0.3 * torch.randn(n, generator=g)
    r = torch.randn(rows, n, generator=g)
    dy = torch.randn(rows, n, generator=g)
    t = DT[dt]
    return x.to(t), w.to(t), (b.to(t) if bias else None), (r.to(t) if residual else None), dy.to(t)


def half_step(dt):
    return torch.finfo(DT[dt]).eps / 2


def check(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = (got - want).abs() - tol
    assert want.numel() == 0 or float(bad.max()) <= 0, \
        f"{what}: off by {float((got - want).abs().max()):.3e}, over its bound by {float(bad.max()):.3e}"


def reference(x, w, b, r, dy, dt, act):
    x, w, dy = x.double(), w.double(), dy.double()
    k = x.shape[1]
    z = x @ w.T + (b.double() if b is not None else 0)
    s = x.abs() @ w.abs().T + (b.double().abs() if b is not None else 0)
    zerr = (k + 4) * U * s
    q = z.clone().requires_grad_(True)
    a = act64(q, act)
    y = a.detach() + (r.double() if r is not None else 0)
    e, low = half_step(dt), TINY16 if dt == "f16" else 0.0
    out = {"y": (y, 1.13 * zerr + 8 * U * (a.detach().abs() + y.abs()) + e * y.abs() * 1.01 + low)}
    dz, = torch.autograd.grad(a, q, dy)
    if act in ("none", "relu", "lrelu"):
        gerr = 4 * U * dz.abs()
    elif dt == "bf16":
        gerr = dy.abs() * (2.0 ** -11 + 1.2 * zerr + 2.0 ** -19)
    else:
        gerr = dy.abs() * (1.2 * zerr + (16 * U if dt == "f32" else 2.0 ** -19))
    raw = gerr
    if act != "none":
        gerr = gerr * 1.01 + e * dz.abs() * 1.01 + low
    rows, n = dy.shape
    for name, v, mag, er, m in (("dx", dz @ w, dz.abs() @ w.abs(), gerr @ w.abs(), n),
                                ("dw", dz.T @ x, dz.abs().T @ x.abs(), gerr.T @ x.abs(), rows),
                                ("db", dz.sum(0), dz.abs().sum(0), raw.sum(0), rows)):
        out[name] = (v, 1.01 * er + (m + 4) * U * mag + e * v.abs() * 1.01 + low)
    return out


def on_gpu(*ts):
    return [t.cuda() if t is not None else None for t in ts]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear_and_gradients(i, dt):
    """Every size with an activation of its own, all gradients."""
    from cgan3d_amd.model.linear import fused_linear
    rows, k, n = SHAPES[i]
    act = ACTS[(i + list(DT).index(dt)) % len(ACTS)]
    bias, residual = i % 3 != 1, i % 2 == 0
    x, w, b, r, dy = make(rows, k, n, dt, act, 100 + i, bias, residual)
    want = reference(x, w, b, r, dy, dt, act)
    leaves = [t.requires_grad_(True) if t is not None else None for t in on_gpu(x, w, b, r)]
    y = fused_linear(*leaves[:3], residual=leaves[3], act=code(act), slope=SLOPE)
    assert y.dtype == DT[dt]
    what = f"{rows}x{k}x{n} {dt} {act}"
    check(y, *want["y"], f"{what} y")
    y.backward(dy.cuda())
    check(leaves[0].grad, *want["dx"], f"{what} dx")
    check(leaves[1].grad, *want["dw"], f"{what} dw")
    if bias:
        check(leaves[2].grad, *want["db"], f"{what} db")
    if residual:
        assert torch.equal(leaves[3].grad.cpu(), dy)
    with torch.no_grad():  # the call that keeps nothing for a backward pass
        again = fused_linear(*leaves[:3], residual=leaves[3], act=code(act), slope=SLOPE)
    assert torch.equal(again, y.detach())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dt):
    from cgan3d_amd.model.linear import fused_linear
    x, w, b, r, dy = make(70, 48, 36, dt, act, 7)
    want = reference(x, w, b, r, dy, dt, act)
    leaves = [t.requires_grad_(True) for t in on_gpu(x, w, b, r)]
    y = fused_linear(*leaves[:3], residual=leaves[3], act=code(act), slope=SLOPE)
    check(y, *want["y"], f"{act} {dt} y")
    y.backward(dy.cuda())
    for t, nm in zip(leaves, ("dx", "dw", "db")):
        check(t.grad, *want[nm], f"{act} {dt} {nm}")


def test_gradient_against_differences():
    """f32, smooth activation: directional derivatives of <y, dy> by central differences in float64 of the
    reference formula."""
    from cgan3d_amd.model.linear import fused_linear
    x, w, b, r, dy = make(40, 30, 50, "f32", "gelu", 11)
    leaves = [t.requires_grad_(True) for t in on_gpu(x, w, b, r)]
    fused_linear(*leaves[:3], residual=leaves[3], act=code("gelu")).backward(dy.cuda())
    g = torch.Generator().manual_seed(3)
    args = [t.double() for t in (x, w, b, r)]

    def f(a):
        return float(((F.gelu(a[0] @ a[1].T + a[2]) + a[3]) * dy.double()).sum())
    for i in range(4):
        d = torch.randn(args[i].shape, generator=g).double()
        h = 1e-4
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + h * d, args[i] - h * d
        num = (f(hi) - f(lo)) / (2 * h)
        got = float((leaves[i].grad.double().cpu() * d).sum())
        # h^2 / 6 of the third derivative, and f32 gradients: both far below 1e-5 of the sum's scale
        scale = float((leaves[i].grad.double().cpu().abs() * d.abs()).sum())
        assert abs(num - got) <= 1e-5 * scale, (i, num, got, scale)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lead", [(), (0,), (3,), (2, 3, 4, 5)])
def test_leading_axes_and_empty(lead, dt):
    from cgan3d_amd.model.linear import fused_linear
    k, n = 24, 20
    rows = math.prod(lead)
    x, w, b, r, dy = make(rows, k, n, dt, "silu", 5)
    want = reference(x, w, b, r, dy, dt, "silu")
    leaves = [t.requires_grad_(True) for t in (x.view(*lead, k).cuda(), w.cuda(), b.cuda(), r.view(*lead, n).cuda())]
    y = fused_linear(*leaves[:3], residual=leaves[3], act=code("silu"))
    assert y.shape == (*lead, n)
    check(y.reshape(rows, n), *want["y"], "y")
    y.backward(dy.view(*lead, n).cuda())
    check(leaves[0].grad.reshape(rows, k), *want["dx"], "dx")
    check(leaves[1].grad, *want["dw"], "dw")
    check(leaves[2].grad, *want["db"], "db")


@pytest.mark.parametrize("dt", list(DT))
def test_no_inputs_or_outputs(dt):
    """k = 0: y = act(bias) + residual; n = 0: nothing, and zero gradients."""
    from cgan3d_amd import ops
    t = DT[dt]
    b, r = torch.randn(9).to(t).cuda(), torch.randn(5, 9).to(t).cuda()
    y = torch.empty(5, 9, dtype=t, device="cuda")
    ops.linear(torch.empty(5, 0, dtype=t, device="cuda"), torch.empty(9, 0, dtype=t, device="cuda"), y, bias=b,
               residual=r, act=code("relu"))
    want = F.relu(b.double()) + r.double()
    check(y, want.cpu(), (half_step(dt) * 1.01 * want.abs() + TINY16).cpu(), "k = 0")
    dx, x = torch.full((5, 7), 3.0, dtype=t, device="cuda"), torch.ones(5, 7, dtype=t, device="cuda")
    w0, dy0 = torch.empty(0, 7, dtype=t, device="cuda"), torch.empty(5, 0, dtype=t, device="cuda")
    ops.linear(x, w0, dy0)
    ops.linear_backward(dy0, x, w0, dx=dx)
    assert not dx.any()
    # no rows: the weight's and the bias's gradients are zero
    dw, db = torch.full((4, 7), 3.0, dtype=t, device="cuda"), torch.full((4,), 3.0, dtype=t, device="cuda")
    ops.linear_backward(torch.empty(0, 4, dtype=t, device="cuda"), torch.empty(0, 7, dtype=t, device="cuda"),
                        torch.ones(4, 7, dtype=t, device="cuda"), dw=dw, dbias=db)
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,k,n", [(1, 70, 33), (6, 128, 200), (70, 64, 64), (300, 260, 130), (513, 256, 512)])
def test_strided_rows_leave_the_rest(rows, k, n, dt):
    """Rows of wider tensors, at every alignment: what lies between and behind them stays as it was."""
    from cgan3d_amd import ops
    t = DT[dt]
    x, w, b, r, dy = make(rows, k, n, dt, "tanh", 21)
    want = reference(x, w, b, r, dy, dt, "tanh")
    for off in (0, 1, 3, 8):
        def wide(m, cols, src=None):
            buf = torch.full((m + 2, cols + 24), 7.0, dtype=t, device="cuda")
            view = buf[1:m + 1, off:off + cols]
            if src is not None:
                view.copy_(src)
            return buf, view

        def rest(buf, m, cols):
            buf = buf.clone()
            buf[1:m + 1, off:off + cols] = 7.0
            return bool((buf == 7.0).all())
        xb, xv = wide(rows, k, x)
        wb, wv = wide(n, k, w)
        rb, rv = wide(rows, n, r)
        gb, gv = wide(rows, n, dy)
        yb, yv = wide(rows, n)
        db, dv = wide(rows, k)
        pre = torch.empty(rows, n, dtype=ops.linear_preact_dtype(t), device="cuda")
        ops.linear(xv, wv, yv, bias=b.cuda(), residual=rv, act=code("tanh"), preact=pre)
        check(yv, *want["y"], f"y at {off}")
        assert rest(yb, rows, n)
        dw = torch.empty(n, k, dtype=t, device="cuda")
        dbias = torch.empty(n, dtype=t, device="cuda")
        ops.linear_backward(gv, xv, wv, dx=dv, dw=dw, dbias=dbias, act=code("tanh"), preact=pre)
        check(dv, *want["dx"], f"dx at {off}")
        check(dw, *want["dw"], f"dw at {off}")
        check(dbias, *want["db"], f"db at {off}")
        assert rest(db, rows, k)
        ops.linear(xv, wv, rv, bias=b.cuda(), residual=rv, act=code("tanh"))  # in place over the residual
        check(rv, *want["y"], f"in place at {off}")
        assert rest(rb, rows, n) and rest(xb, rows, k) and rest(wb, n, k) and rest(gb, rows, n)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,k,n", [(1, 64, 40), (70, 60, 33), (70, 100, 65), (300, 512, 256), (1500, 1000, 1203)])
def test_infinities_and_nans_stay_in_their_rows(rows, k, n, dt):
    from cgan3d_amd.model.linear import fused_linear
    x, w, b, r, _ = make(rows, k, n, dt, "none", 31)
    w = w.abs() + 0.01
    clean = fused_linear(*on_gpu(x, w, b), residual=r.cuda())
    x2 = x.clone()
    x2[0, k // 2] = float("inf")
    if rows > 5:
        x2[5, 3] = float("nan")
    y = fused_linear(*on_gpu(x2, w, b), residual=r.cuda())
    assert (y[0] == float("inf")).all()
    keep = [i for i in range(rows) if i not in ((0, 5) if rows > 5 else (0,))]
    if rows > 5:
        assert y[5].isnan().all()
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_large_values_keep_their_size(dt):
    """Values near the top and the bottom of the type's range go through the product as they are."""
    from cgan3d_amd.model.linear import fused_linear
    g = torch.Generator().manual_seed(4)
    for m, k, n in ((260, 384, 300), (1500, 1000, 1203)):
        for scale in (1e-36, 1e-30, 1e30):
            x = (torch.randn(m, k, generator=g) * scale).to(DT[dt])
            w = torch.randn(n, k, generator=g).to(DT[dt])
            y = fused_linear(x.cuda(), w.cuda())
            want = x.double() @ w.double().T
            tol = (k + 4) * U * (x.double().abs() @ w.double().abs().T) + half_step(dt) * 1.01 * want.abs()
            check(y, want, tol, f"{m}x{k}x{n}, scale {scale}")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_graph_plan_and_streams(dt):
    """The same call eager, on another stream, captured and replayed with new values, and recorded in a
    launch plan."""
    from cgan3d_amd import ops
    t = DT[dt]
    for rows, k, n in ((1, 512, 96), (96, 4096, 64), (640, 256, 512)):
        x, w, b, r, _ = make(rows, k, n, dt, "gelu", 41)
        x2 = make(rows, k, n, dt, "gelu", 42)[0]
        xs, w, b, r = on_gpu(x, w, b, r)
        y = torch.empty(rows, n, dtype=t, device="cuda")
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")

        def call():
            ops.linear(xs, w, y, bias=b, residual=r, act=code("gelu"), ws=ws)
        wants = []
        for v in (x, x2):
            xs.copy_(v)
            call()
            wants.append(y.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        y.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, wants[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        ops.plan_begin()
        call()
        plan = ops.plan_end()
        for go in (graph.replay, plan.run):
            for v, want in ((x, wants[0]), (x2, wants[1]), (x, wants[0])):
                xs.copy_(v)
                y.zero_()
                go()
                torch.cuda.synchronize()
                assert torch.equal(y, want), (rows, go)


def test_captured_training_step():
    """Forward and backward in one graph, replayed on other inputs, against the eager calls (whose autograd
    graphs are gone by then)."""
    from cgan3d_amd.model.linear import fused_linear
    x, w, b, r, dy = on_gpu(*make(200, 96, 160, "f32", "silu", 51))
    x2 = make(200, 96, 160, "f32", "silu", 52)[0].cuda()

    def step(xi):
        leaves = [t.detach().requires_grad_(True) for t in (xi, w, b, r)]
        y = fused_linear(*leaves[:3], residual=leaves[3], act=code("silu"))
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    wants = [[t.clone() for t in step(v)] for v in (x, x2)]
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for v, want in ((x, wants[0]), (x2, wants[1]), (x, wants[0])):
        static.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(got, want):
            assert torch.equal(a, e)


def test_expanded_gradient_and_views():
    """dy of a sum (an expanded scalar), a transposed x, a weight that is a slice."""
    from cgan3d_amd.model.linear import fused_linear
    g = torch.Generator().manual_seed(9)
    x = torch.randn(30, 50, generator=g).cuda().T.requires_grad_(True)  # [50, 30], columns contiguous
    w = torch.randn(20, 64, generator=g).cuda()[:, 5:35].requires_grad_(True)
    y = fused_linear(x, w)
    y.sum().backward()
    ones = torch.ones(50, 20).double()
    for got, want, mag, m in ((x.grad, ones @ w.double().cpu(), ones @ w.double().cpu().abs(), 20),
                              (w.grad, ones.T @ x.double().cpu(), ones.T @ x.double().cpu().abs(), 50)):
        check(got, want.detach(), ((m + 4) * U * mag + 2 * U * want.abs()).detach(), "grad")


def test_repeated_runs_are_equal():
    """Fixed orders of summation: the same call gives the same bits."""
    from cgan3d_amd.model.linear import fused_linear
    for rows, k, n in ((5000, 48, 40), (64, 4096, 64)):
        x, w, b, r, dy = on_gpu(*make(rows, k, n, "f32", "gelu", 61))
        first = None
        for _ in range(4):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
            y = fused_linear(*leaves[:3], residual=leaves[3], act=code("gelu"))
            got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            first = first or got
            assert all(torch.equal(a, e) for a, e in zip(got, first))


@pytest.mark.parametrize("rows,k,n", [(6, 24, 16), (700, 96, 64), (1500, 1000, 1203)])
def test_some_gradients(rows, k, n):
    """Only what is asked for is computed, and it is what the full call gives."""
    from cgan3d_amd import ops
    x, w, b, _, dy = on_gpu(*make(rows, k, n, "f32", "gelu", 71))
    y, pre = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    ops.linear(x, w, y, bias=b, act=code("gelu"), preact=pre)
    full = dict(dx=torch.empty_like(x), dw=torch.empty_like(w), dbias=torch.empty_like(b))
    ops.linear_backward(dy, x, w, **full, act=code("gelu"), preact=pre)
    for names in (("dx",), ("dw",), ("dbias",), ("dx", "dbias"), ("dw", "dbias"), ("dx", "dw"), ()):
        part = {nm: torch.full_like(full[nm], 3.0) for nm in names}
        ops.linear_backward(dy, x, w, **part, act=code("gelu"), preact=pre)
        for nm in names:
            # the same sums in the same order, unless a product takes another form without its sibling
            scale = float(full[nm].abs().max())
            assert float((part[nm] - full[nm]).abs().max()) <= 1e-5 * scale, (names, nm)


def test_two_streams_at_once():
    """Calls on two streams with workspaces of their own do not disturb each other."""
    from cgan3d_amd.model.linear import fused_linear
    args = [on_gpu(*make(640, 1024, 520, "bf16", "silu", 80 + i)) for i in range(2)]
    wants = [fused_linear(*a[:3], residual=a[3], act=code("silu")) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fused_linear(*args[i][:3], residual=args[i][3], act=code("silu")))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, wants[i]) for y in got[i])


def test_f32_products_close_to_overflow():
    """Products and sums just below f32's largest value stay finite, however the operands are held inside."""
    from cgan3d_amd.model.linear import fused_linear
    g = torch.Generator().manual_seed(91)
    m, k, n = 1500, 1000, 1203
    top = torch.finfo(torch.float32).max
    x = torch.zeros(m, k)
    # values whose nearest bf16 lies above them: rounding them up and multiplying would overflow
    x[:, 17] = 1.0 + (0.55 + 0.15 * torch.rand(m, generator=g)) * 2.0 ** -7
    w = torch.randn(n, k, generator=g)
    w[:, 17] = top / float(x[:, 17].max()) * (1 - 1e-6)
    y = fused_linear(x.cuda(), w.cuda())
    want = x.double() @ w.double().T
    assert want.abs().max() < top
    check(y, want, (k + 4) * U * want.abs(), "largest values")


@pytest.mark.parametrize("rows,k,n", [(70, 24, 40), (300, 136, 200)])
def test_saved_tensor_hooks_and_repeated_backward(rows, k, n):
    """Operands that come back from the host at other addresses, a kept graph run twice, and a transposed weight."""
    from cgan3d_amd.model.linear import fused_linear
    x, w, b, r, dy = on_gpu(*make(rows, k, n, "f32", "silu", 95))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    wants = torch.autograd.grad(fused_linear(*leaves, act=code("silu")), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = fused_linear(*leaves, act=code("silu"))
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, leaves, dy), wants))
    y = fused_linear(*leaves, act=code("silu"))
    for keep in (True, True, False):
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, leaves, dy, retain_graph=keep), wants))
    wt = w.detach().t().contiguous().requires_grad_(True)
    got = torch.autograd.grad(fused_linear(x, wt.t(), b, r, act=code("silu")), (x, wt), dy)
    assert torch.equal(got[0], wants[0]) and torch.equal(got[1], wants[1].t())
