"""Every tile of the linear block's products on planes, with odd sizes, with and without a split of the summed axis.  Which
kernels a call launches is read from a recorded plan, so that a retuned rule cannot drop a tile from the tests without a
word.  Tolerances: test_gpu_linear.py."""
import re

import pytest
import torch

from test_gpu_linear import DT, SLOPE, U, check, code, half_step, make, reference

pytestmark = pytest.mark.gpu

LAUNCH = re.compile(r"plane_kernelI\w+?Li(\d)ELb([01])ELb([01])ELi(\d+)ELi(\d+)E")
WS = 1 << 30


def launches(call):
    """Runs ``call`` from a recorded plan; its products as "tile" or "tile split", or "f32" for the f32 instructions'."""
    from cgan3d_amd import ops
    ops.plan_time_filter("plane_kernel|plane_join_kernel|mat_kernel")
    ops.plan_begin()
    try:
        call()
    finally:
        plan = ops.plan_end()
        ops.plan_time_filter(None)
    plan.run()
    torch.cuda.synchronize()
    out = []
    for _, _, _, name in plan.timeline():
        m = LAUNCH.search(name)
        if m:
            out.append(f"{m[4]}x{m[5]}")
        elif "plane_join" in name:
            out[-1] += " split"
        else:
            out.append("f32")
    return out


@pytest.fixture(scope="module")
def ws():
    return torch.empty(WS, dtype=torch.uint8, device="cuda")


FWD = [("16", 4001, 203, 4003, "256x256"), ("16", 2049, 300, 2051, "128x128"), ("16", 6001, 3001, 203, "128x128 split"),
       ("16", 300, 301, 260, "64x64"), ("16", 200, 3000, 200, "64x64 split"), ("f32", 4001, 203, 4003, "128x256"),
       ("f32", 1200, 3000, 1200, "128x256 split"), ("f32", 900, 1400, 2600, "128x128"), ("f32", 1100, 1101, 1103, "128x128 split"),
       ("f32", 1000, 1500, 1000, "64x64"), ("f32", 1500, 1000, 1203, "f32"), ("f32", 2049, 300, 2051, "f32")]
DX = [("16", 4003, 4001, 203, "256x256"), ("16", 5000, 2050, 5001, "256x256"), ("16", 4001, 1999, 2051, "128x128"),
      ("16", 520, 1000, 5000, "128x128 split"), ("16", 300, 301, 260, "64x64"), ("f32", 4003, 4001, 203, "128x256"),
      ("f32", 700, 2001, 1500, "128x256 split"), ("f32", 1200, 3000, 1200, "128x128"), ("f32", 4001, 203, 4003, "128x128 split"),
      ("f32", 901, 903, 900, "64x64"), ("f32", 2049, 300, 2051, "f32")]
DW = [("16", 5000, 2050, 5001, "256x256"), ("16", 4001, 1999, 2051, "256x256 split"), ("16", 520, 1000, 5000, "128x128"),
      ("16", 8191, 65, 4099, "128x128 split"), ("16", 2049, 300, 2051, "64x64"), ("f32", 300, 4100, 1500, "128x256"),
      ("f32", 3001, 2500, 1300, "128x256 split"), ("f32", 700, 2001, 1500, "128x128"), ("f32", 4001, 203, 4003, "128x128 split"),
      ("f32", 901, 903, 900, "64x64"), ("f32", 2049, 300, 2051, "f32")]


def types(cases):
    return [(dt, *c[1:]) for c in cases for dt in (("bf16", "f16") if c[0] == "16" else ("f32",))]


def cpu(pair):
    return [t.cpu() for t in pair]


@pytest.mark.parametrize("dt,rows,k,n,tile", types(FWD))
def test_forward_tiles(dt, rows, k, n, tile, ws):
    """With bias, activation, residual and the kept pre-activation."""
    from cgan3d_amd import ops
    x, w, b, r, dy = (t.cuda() for t in make(rows, k, n, dt, "silu", rows + n))
    y = torch.full((rows, n), 7.0, dtype=DT[dt], device="cuda")
    pre = torch.empty(rows, n, dtype=ops.linear_preact_dtype(DT[dt]), device="cuda")
    got = launches(lambda: ops.linear(x, w, y, bias=b, residual=r, act=code("silu"), preact=pre, ws=ws))
    assert got == [tile], f"{rows}x{k}->{n} {dt}: {got}"
    want = reference(x, w, b, r, dy, dt, "silu")
    check(y, *cpu(want["y"]), f"{rows}x{k}->{n} {dt} y")
    z = x.double() @ w.double().T + b.double()
    tol = (k + 4) * U * (x.double().abs() @ w.double().abs().T + b.double().abs())
    check(pre, z.cpu(), (tol + (2.0 ** -11 * z.abs() + 2.0 ** -25 if dt == "bf16" else 0)).cpu(), "preact")


@pytest.mark.parametrize("which,dt,rows,k,n,tile", [("dx", *c) for c in types(DX)] + [("dw", *c) for c in types(DW)])
def test_gradient_tiles(which, dt, rows, k, n, tile, ws):
    from cgan3d_amd import ops
    act = "silu" if (rows + n) % 2 else "none"
    x, w, b, _, dy = (t.cuda() if t is not None else None for t in make(rows, k, n, dt, act, rows + k, residual=False))
    y = torch.empty(rows, n, dtype=DT[dt], device="cuda")
    pre = torch.empty(rows, n, dtype=ops.linear_preact_dtype(DT[dt]), device="cuda")
    ops.linear(x, w, y, bias=b, act=code(act), preact=pre, ws=ws)
    out = torch.full((rows, k) if which == "dx" else (n, k), 7.0, dtype=DT[dt], device="cuda")
    got = launches(lambda: ops.linear_backward(dy, x, w, **{which: out}, act=code(act), preact=pre, ws=ws))
    assert got == [tile], f"{rows}x{k}->{n} {dt} {which}: {got}"
    check(out, *cpu(reference(x, w, b, None, dy, dt, act)[which]), f"{rows}x{k}->{n} {dt} {which}")


@pytest.mark.parametrize("rows,k,n,tiles", [(4003, 1001, 1030, ["128x128", "128x256 split"]), (901, 903, 900, ["64x64", "64x64"])])
def test_both_f32_gradients_share_their_planes(rows, k, n, tiles, ws):
    from cgan3d_amd import ops
    x, w, b, _, dy = (t.cuda() if t is not None else None for t in make(rows, k, n, "f32", "gelu", 3, residual=False))
    y, pre = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    ops.linear(x, w, y, bias=b, act=code("gelu"), preact=pre, ws=ws)
    out = dict(dx=torch.empty_like(x), dw=torch.empty_like(w), dbias=torch.empty_like(b))
    got = launches(lambda: ops.linear_backward(dy, x, w, **out, act=code("gelu"), preact=pre, ws=ws))
    assert got == tiles, got
    want = reference(x, w, b, None, dy, "f32", "gelu")
    for a, e in (("dx", "dx"), ("dw", "dw"), ("dbias", "db")):
        check(out[a], *cpu(want[e]), a)


PLANES = [(4001, 203, 4003, "128x256"), (1200, 3000, 1200, "128x256 split")]


@pytest.mark.parametrize("rows,k,n,tile", PLANES)
def test_f32_infinities_and_nans_on_planes(rows, k, n, tile, ws):
    """Sums that are not finite are computed again from the values, by the staged epilogue and by the join."""
    from cgan3d_amd import ops
    x, w, b, r, _ = make(rows, k, n, "f32", "none", 31)
    x, w, b, r = x.cuda(), (w.abs() + 0.01).cuda(), b.cuda(), r.cuda()
    clean, y = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    assert launches(lambda: ops.linear(x, w, clean, bias=b, residual=r, ws=ws)) == [tile]
    x[0, k // 2], x[5, 3], x[rows - 1, k - 1] = float("inf"), float("nan"), -float("inf")
    ops.linear(x, w, y, bias=b, residual=r, ws=ws)
    assert (y[0] == float("inf")).all() and y[5].isnan().all() and (y[-1] == -float("inf")).all()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[[0, 5, rows - 1]] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("rows,k,n,tile", PLANES)
def test_f32_sums_close_to_overflow_on_planes(rows, k, n, tile, ws):
    from cgan3d_amd import ops
    g = torch.Generator().manual_seed(91)
    top = torch.finfo(torch.float32).max
    x = torch.zeros(rows, k)
    # values whose nearest bf16 lies above them: rounding them up and multiplying would overflow
    x[:, 17] = 1.0 + (0.55 + 0.15 * torch.rand(rows, generator=g)) * 2.0 ** -7
    w = torch.randn(n, k, generator=g)
    w[:, 17] = top / float(x[:, 17].max()) * (1 - 1e-6)
    x, w, y = x.cuda(), w.cuda(), torch.empty(rows, n, device="cuda")
    assert launches(lambda: ops.linear(x, w, y, ws=ws)) == [tile]
    want = x.double() @ w.double().T
    assert want.abs().max() < top
    check(y, want.cpu(), ((k + 4) * U * want.abs()).cpu(), "largest values")


@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e30])
@pytest.mark.parametrize("rows,k,n,tile", PLANES)
def test_f32_small_and_large_values_on_planes(rows, k, n, tile, scale, ws):
    """Three bf16 planes hold an f32 down to 2^-133 (bf16's smallest step): a value below 2^-110 loses what lies under that,
    at most 2^-134 of it a plane."""
    from cgan3d_amd import ops
    g = torch.Generator().manual_seed(4)
    x, w = (torch.randn(rows, k, generator=g) * scale).cuda(), torch.randn(n, k, generator=g).cuda()
    y = torch.empty(rows, n, device="cuda")
    assert launches(lambda: ops.linear(x, w, y, ws=ws)) == [tile]
    want, mag = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    lost = 2 * 2.0 ** -134 * w.double().abs().sum(1) if scale < 1e-33 else torch.zeros(n, device="cuda").double()
    check(y, want.cpu(), ((k + 4) * U * mag + half_step("f32") * 1.01 * want.abs() + lost).cpu(), f"scale {scale}")


@pytest.mark.parametrize("dt,act", [("f32", "gelu"), ("bf16", "gelu"), ("f16", "silu"), ("bf16", "none")])
@pytest.mark.parametrize("rows,k,n", [(3, 64, 48), (700, 40, 64), (65, 33, 50), (1000, 16, 32)])
def test_some_gradients_of_few_channels(rows, k, n, dt, act):
    """dx, dw and dbias alone and in pairs are what the full call gives, in one pass over the rows and as products."""
    from cgan3d_amd import ops
    x, w, b, _, dy = (t.cuda() if t is not None else None for t in make(rows, k, n, dt, act, 71, residual=False))
    y = torch.empty(rows, n, dtype=DT[dt], device="cuda")
    pre = torch.empty(rows, n, dtype=ops.linear_preact_dtype(DT[dt]), device="cuda")
    ops.linear(x, w, y, bias=b, act=code(act), slope=SLOPE, preact=pre)
    want = {"dbias" if nm == "db" else nm: cpu(v) for nm, v in reference(x, w, b, None, dy, dt, act).items()}
    new = dict(dx=torch.empty_like(x), dw=torch.empty_like(w), dbias=torch.empty_like(b))
    for names in (("dx", "dw", "dbias"), ("dx",), ("dw",), ("dbias",), ("dx", "dbias"), ("dw", "dbias"), ("dx", "dw")):
        part = {nm: torch.full_like(new[nm], 3.0) for nm in names}
        ops.linear_backward(dy, x, w, **part, act=code(act), slope=SLOPE, preact=pre)
        for nm in names:
            check(part[nm], *want[nm], f"{names} {nm}")
