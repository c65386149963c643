"""Newton-Schulz and Muon at the ends of the range: matrices far below eps, far above one, and the largest tiles.
Tolerances of test_gpu_muon.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NS = (3.4445, -4.7750, 2.0315)
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ns64(g, steps=5, co=NS, eps=1e-7):
    """(result, tolerance in the Frobenius norm) of one matrix in float64: see test_gpu_muon.py."""
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.mT.contiguous()
    x = x / (torch.linalg.vector_norm(x) + eps)
    a, b, c = co
    tol = 0.0
    for _ in range(steps):
        tol = abs(a) * (tol + 4 * U * float(x.norm()))
        m = x @ x.mT
        x = a * x + (b * m + c * m @ m) @ x
    tol += 4 * U * float(x.norm())
    return (x.mT if tall else x), tol


def check_ns(got, g, dt, what, **kw):
    want, tol = ns64(g, **kw)
    got = got.double().to(want.device)
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    tol += torch.finfo(DT[dt]).eps / 2 * float(want.norm()) + (2.0 ** -25 * math.sqrt(want.numel()) if dt == "f16" else 0)
    err = float((got - want).norm())
    assert err <= tol, f"{what}: off by {err:.3e}, bound {tol:.3e}, norm {float(want.norm()):.3e}"


@pytest.mark.parametrize("shape", [(40, 600), (600, 40), (100, 600)])
def test_zeros_beside_the_smallest_values(shape):
    """A stretch of zeros along the long side of a matrix of f32's smallest values, without an eps: zeros stay zeros."""
    from cgan3d_amd import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(5)) * 1e-37
    long = g if shape[1] > shape[0] else g.T
    long[:, 256:512] = 0
    got = ops.orthogonalize(g.cuda(), eps=0.0)
    check_ns(got, g, "f32", f"{shape}", eps=0.0)
    assert not (got if shape[1] > shape[0] else got.T)[:, 256:512].any()


SLABS_AND_PLANES = [(40, 600), (50, 30), (64, 20000), (100, 300), (333, 97)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-5, 1e-8, 1e-11, 1e-13, 1e-16, 1e-24, 1e-36])
@pytest.mark.parametrize("shape", SLABS_AND_PLANES)
def test_matrices_far_below_eps(shape, size, dt):
    """|G| << eps: the iterates start near |G| / eps and grow by 3.4445 a step; every one of them keeps f32's accuracy
    relative to itself."""
    from cgan3d_amd import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(7))
    g = (g * (size / float(g.norm()))).to(DT[dt])
    check_ns(ops.orthogonalize(g.cuda()), g, dt, f"{shape} of {size}")


@pytest.mark.parametrize("shape", SLABS_AND_PLANES)
def test_far_below_eps_with_other_steps(shape):
    """One step, few, many; coefficients of another growth; and a list whose matrices differ by their sizes alone."""
    from cgan3d_amd import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(8)) * 1e-14
    for steps in (1, 2, 3, 9):
        check_ns(ops.orthogonalize(g.cuda(), steps=steps), g, "f32", f"{steps} steps", steps=steps)
    co = (1.5, -0.5, 0.0)
    for steps in (2, 20):
        check_ns(ops.orthogonalize(g.cuda(), steps=steps, coefficients=co), g, "f32", f"cubic, {steps}", steps=steps, co=co)
    many = torch.stack([g * s for s in (1.0, 1e14, 1e5, 0.0, 1e-9, 1e9)])
    got = ops.orthogonalize(many.cuda())
    for i in range(len(many)):
        check_ns(got[i], many[i], "f32", f"matrix {i}")
    assert torch.equal(got[1], ops.orthogonalize(many[1].cuda()))


@pytest.mark.parametrize("steps", [0, 5])
@pytest.mark.parametrize("shape", SLABS_AND_PLANES)
def test_finite_matrices_whose_norm_is_beyond_f32(shape, steps):
    from cgan3d_amd import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(9))
    g = g * (3e38 / float(g.abs().max()))
    assert torch.isfinite(g).all() and float(g.double().norm()) > torch.finfo(torch.float32).max
    check_ns(ops.orthogonalize(g.cuda(), steps=steps), g, "f32", f"{shape}", steps=steps)


@pytest.mark.parametrize("shape", SLABS_AND_PLANES)
def test_muon_step_far_below_eps(shape):
    """The parameter's change under a gradient of 1e-13 from a parameter of zeros."""
    from cgan3d_amd import ops
    n = shape[0] * shape[1]
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(10)) * (1e-13 / math.sqrt(n))
    segs = ops.MuonSegments(n, [(0, *shape, 1.0)], [])
    p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    hyper = torch.tensor([0.5, 0.75, 0.0, 0.0, 0.0, 0.0, 0.0, 0.9, 0.999, 1e-8], device="cuda")
    ops.muon_step(p, g.reshape(-1).cuda(), m, v, segs, hyper)
    assert torch.equal(m.cpu(), 0.25 * g.reshape(-1))  # exact: powers of two
    check_ns(p.view(shape) * -2.0, 0.25 * g, "f32", f"{shape}")


TILES = [  # matrices; tiles of the Gram product, the polynomial and the step
    ((1, 2049, 2100), ["128x128", "128x128", "128x256"]), ((1, 2100, 2049), ["128x128", "128x128", "128x256"]),
    ((2, 2048, 8192), ["256x256 split", "256x256 split", "128x256"]), ((1, 4101, 4097), ["256x256 split", "256x256 split", "128x256"]),
    ((2, 2049, 4099), ["128x128 split", "128x128", "128x256"]), ((1, 5500, 5601), ["256x256", "256x256", "128x256"]),
    ((1, 3005, 3001), ["256x256 split", "256x256 split", "128x128"]), ((1, 600, 5000), ["64x64 split", "64x64", "128x128"]),
]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape,tiles", TILES)
def test_the_tiles_of_large_matrices(shape, tiles, dt):
    """Symmetric and step tiles of every size, wide and tall (a tall result is turned on its way out)."""
    from test_gpu_linear_tiles import launches
    from cgan3d_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(11)
    g = torch.randn(*shape, generator=gen, device="cuda") * torch.exp(0.5 * torch.randn(*shape[:2], 1, generator=gen, device="cuda"))
    g = (g * 1e-3).to(DT[dt])
    out, ws = torch.empty_like(g), torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    got = launches(lambda: ops.orthogonalize(g, steps=2, out=out, ws=ws))
    assert got == tiles + tiles, f"{shape}: {got}"
    five = ops.orthogonalize(g, ws=ws)
    for i in range(shape[0]):
        check_ns(out[i], g[i], dt, f"{shape} matrix {i}", steps=2)
        check_ns(five[i], g[i], dt, f"{shape} matrix {i}, five steps")


@pytest.mark.parametrize("shapes", [[(2049, 2100), (2100, 2049)], [(600, 5000), (3001, 3005), (70, 90)]])
def test_muon_step_of_large_matrices(shapes):
    """The parameters' update through the large tiles' last step."""
    from cgan3d_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(12)
    mats, n = [], 0
    for r, c in shapes:
        mats.append((n, r, c, 1.0))
        n += r * c
    segs = ops.MuonSegments(n, mats, [])
    g, p = 1e-3 * torch.randn(n, generator=gen, device="cuda"), torch.randn(n, generator=gen, device="cuda")
    before, m, v = p.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    hyper = torch.tensor([0.5, 0.75, 0.125, 0.0, 0.0, 0.0, 0.0, 0.9, 0.999, 1e-8], device="cuda")
    ops.muon_step(p, g, m, v, segs, hyper)
    for at, r, c, _ in mats:
        u = 0.25 * g[at:at + r * c].view(r, c)
        x, tol = ns64(u)
        want = before[at:at + r * c].view(r, c).double() * (1 - 0.5 * 0.125) - 0.5 * x
        err = float((p[at:at + r * c].view(r, c).double() - want).norm())
        assert err <= 0.5 * tol + 4 * U * float(want.norm()), f"{(r, c)}: off by {err:.3e}"


@pytest.mark.parametrize("shape", [(2, 40, 600), (2, 100, 300)])
def test_replayed_calls_follow_the_size_of_their_input(shape):
    """A captured call keeps no exponent of the matrices it was captured on."""
    from cgan3d_amd import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(13)).cuda()
    inputs = [g, g * 1e-14, g * 1e-3, g * 1e-9, g]
    wants = [ops.orthogonalize(v) for v in inputs]
    static, out = g.clone(), torch.empty_like(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.orthogonalize(static, out=out)
    for v, want in zip(inputs, wants):
        static.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
