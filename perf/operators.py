"""Measured cases of the matrix operators: the linear block (matrix product with bias, activation and
residual in its epilogue) and its gradient, the orthogonalisation of an update by Newton-Schulz products, and
the Muon optimiser's step that uses it.

``own`` False: plain torch forms in 32 bits, rounded once at the end.  ``own`` True: the package's entry points
``cgan3d_amd.model.linear.fused_linear``, ``cgan3d_amd.ops.orthogonalize`` and
``cgan3d_amd.trainer.optim.FusedMuon``.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("none", "relu", "lrelu", "tanh", "gelu", "silu")
SLOPE = 0.2  # LeakyReLU slope of the critic
NS = (3.4445, -4.7750, 2.0315)  # quintic coefficients of the iteration
STEPS, EPS = 5, 1e-7
# Muon on the matrices, Adam on the vectors
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
V_LR, V_B1, V_B2, V_EPS = 3e-4, 0.9, 0.95, 1e-8

# the generator's parameters (4 ResNet blocks, 2 levels, 16 channels) as (rows, columns) of the
# flattened weights, and the number of values of its vectors (BatchNorm scales and shifts, last bias)
GENERATOR = "16x343,32x432,64x864," + "64x1728," * 8 + "64x864,32x432,1x5488"


def listed():
    return [
        # one token / one latent through a square projection: latency and the weight's bytes
        dict(name="linear token bf16", op="linear", rows=1, k=4096, n=4096, dtype="bf16", act="gelu", bias=True,
             residual=True),
        # the ResNet backbone's grid of one 64^3 batch of four, 64 -> 64 channels per voxel
        dict(name="linear voxels f32", op="linear", rows=16384, k=64, n=64, dtype="f32", act="lrelu", bias=True,
             residual=True),
        # nothing is a multiple of a tile or of 16 bytes
        dict(name="linear ragged f16", op="linear", rows=777, k=1001, n=515, dtype="f16", act="tanh", bias=True,
             residual=False),
        # a long batch of rows through an expanding layer
        dict(name="linear prompt bf16", op="linear", rows=4096, k=4096, n=8192, dtype="bf16", act="silu", bias=True,
             residual=True),
        # training: per-voxel channel mixing at full resolution, bound by memory
        dict(name="train voxels f32", op="train", rows=262144, k=16, n=32, dtype="f32", act="silu", bias=True,
             residual=True),
        # training in the framework's default precision
        dict(name="train f32", op="train", rows=2048, k=1024, n=4096, dtype="f32", act="tanh", bias=True,
             residual=False),
        # training, the largest layer
        dict(name="train bf16", op="train", rows=8192, k=2048, n=8192, dtype="bf16", act="gelu", bias=True,
             residual=True),
        # one ResNet-block convolution's momentum
        dict(name="ortho conv f32", op="ortho", batch=1, rows=64, cols=1728, dtype="f32"),
        # a tall matrix with odd sides
        dict(name="ortho ragged f32", op="ortho", batch=3, rows=1001, cols=333, dtype="f32"),
        # a wide layer of a larger model
        dict(name="ortho wide bf16", op="ortho", batch=2, rows=2048, cols=8192, dtype="bf16"),
        # one update of the whole generator
        dict(name="muon generator", op="muon", matrices=GENERATOR, vectors=1345),
        # one update of a stack of linear layers
        dict(name="muon linears", op="muon", matrices=",".join(["1024x4096", "4096x1024"] * 3), vectors=15360),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "train", "train", "ortho", "ortho", "muon"))
    if op in ("linear", "train"):
        while True:
            c = dict(op=op, rows=_log(rng, 1, 262144), k=_log(rng, 8, 8192), n=_log(rng, 8, 8192),
                     dtype=rng.choice(("f32", "bf16", "f16")), act=rng.choice(ACTS), bias=rng.random() < 0.8,
                     residual=rng.random() < 0.5)
            if op == "train" and c["dtype"] == "f32" and c["act"] in ("relu", "lrelu"):
                c["act"] = "gelu"  # a step's sign next to zero is not 32 bits' to tell
            if rng.random() < 0.5:  # whole tiles
                c["k"], c["n"] = -(-c["k"] // 64) * 64, -(-c["n"] // 64) * 64
            w = work(c)
            if w["flops"] <= (8e11 if c["dtype"] != "f32" else 2e11) and w["bytes"] <= 6e8:
                return c
    if op == "ortho":
        while True:
            c = dict(op=op, batch=rng.choice((1, 1, 2, 3, 5, 8)), rows=_log(rng, 1, 4096), cols=_log(rng, 1, 8192),
                     dtype=rng.choice(("f32", "bf16", "f16")))
            if rng.random() < 0.5:
                c["rows"], c["cols"] = -(-c["rows"] // 32) * 32, -(-c["cols"] // 32) * 32
            if work(c)["flops"] <= 1.1e12:
                return c
    if rng.random() < 0.5:  # generators of other widths and depths
        c0, blocks = rng.choice((4, 6, 8, 12, 16, 20, 24)), rng.randint(1, 6)
        shapes = [(c0, 343), (2 * c0, 27 * c0), (4 * c0, 54 * c0)] + [(4 * c0, 108 * c0)] * (2 * blocks)
        shapes += [(4 * c0, 54 * c0), (2 * c0, 27 * c0), (1, 343 * c0)]
        vectors = 2 * (3 * c0 + 4 * c0 + 8 * c0 * blocks + 3 * c0) + 1
    else:  # linear layers of one odd or even width
        d, e = _log(rng, 24, 1500), _log(rng, 24, 2600)
        shapes = [(e, d), (d, e)] * rng.randint(1, 3)
        vectors = sum(s[0] for s in shapes)
    return dict(op="muon", matrices=",".join("%dx%d" % s for s in shapes), vectors=vectors)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["matrices"].split(",")]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _gradient_like(gen, *shape):
    """A gradient's values: rows and columns of unlike size over a part that they share."""
    *lead, m, n = shape
    return (_randn(gen, *shape) + _randn(gen, *lead, m, 1) * _randn(gen, *lead, 1, n)) * \
        torch.exp(0.5 * _randn(gen, *lead, m, 1)) * torch.exp(0.5 * _randn(gen, *lead, 1, n)) * 1e-3


def prepare(case, seed):
    if own:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "contrast-gan-3d_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] in ("linear", "train"):
        dt, m, k, n = DTYPES[case["dtype"]], case["rows"], case["k"], case["n"]
        s["x"] = _randn(gen, m, k).to(dt)
        s["w"] = (_randn(gen, n, k) / math.sqrt(k)).to(dt)
        s["b"] = (0.1 * _randn(gen, n)).to(dt) if case["bias"] else None
        s["r"] = _randn(gen, m, n).to(dt) if case["residual"] else None
        if case["op"] == "train":
            s["dy"] = _randn(gen, m, n).to(dt)
            s["leaves"] = [t.requires_grad_(True) for t in (s["x"], s["w"], s["b"], s["r"]) if t is not None]
    elif case["op"] == "ortho":
        s["g"] = _gradient_like(gen, case["batch"], case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    else:
        shapes = _shapes(case)
        parts = [0.05 * _randn(gen, *v) for v in shapes] + [_randn(gen, case["vectors"])]
        grads = [_gradient_like(gen, *v) for v in shapes] + [1e-3 * _randn(gen, case["vectors"])]
        s["moments"] = [torch.cat([1e-3 * _randn(gen, p.numel()) for p in parts]),
                        torch.cat([1e-6 * _randn(gen, p.numel()).square() for p in parts])]
        if own:
            from cgan3d_amd.engine import Arena
            from cgan3d_amd.trainer.optim import FusedMuon
            arena = Arena(torch.nn.ParameterList(parts), torch.device("cuda"))
            arena.grad.copy_(torch.cat([g.reshape(-1) for g in grads]))
            s["optimizer"] = FusedMuon(arena, lr=LR, momentum=MOMENTUM, weight_decay=DECAY, vector_lr=V_LR,
                                       vector_betas=(V_B1, V_B2), vector_eps=V_EPS)
            arena.exp_avg.copy_(s["moments"][0])
            arena.exp_avg_sq.copy_(s["moments"][1])
        else:
            s["p"] = torch.cat([p.reshape(-1) for p in parts])
            s["g"] = torch.cat([g.reshape(-1) for g in grads])
            s["t"] = torch.zeros((), device="cuda")
    return s


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "lrelu":
        return torch.where(z > 0, z, SLOPE * z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "lrelu":
        return torch.where(z > 0, 1.0, SLOPE)
    if name == "tanh":
        return 1 - torch.tanh(z).square()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (0.5 * math.sqrt(2 / math.pi))
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def _orthogonal(g):
    """Five quintic Newton-Schulz products in 32 bits, over the short side."""
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().float() + EPS)
    a, b, c = NS
    for _ in range(STEPS):
        y = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * y + c * torch.matmul(y, y), x)
    return x.mT.contiguous() if tall else x


def run(s):
    if s["op"] == "linear":
        if own:
            from cgan3d_amd import _lib
            from cgan3d_amd.model.linear import fused_linear
            with torch.no_grad():
                return fused_linear(s["x"], s["w"], s["b"], residual=s["r"],
                                    act=getattr(_lib, "ACT_" + s["act"].upper()), slope=SLOPE)
        z = torch.matmul(s["x"].float(), s["w"].float().T)
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, s["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return y.to(s["x"].dtype)
    if s["op"] == "train":
        if own:
            from cgan3d_amd import _lib
            from cgan3d_amd.model.linear import fused_linear
            y = fused_linear(s["x"], s["w"], s["b"], residual=s["r"], act=getattr(_lib, "ACT_" + s["act"].upper()),
                             slope=SLOPE)
            return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]
        with torch.no_grad():
            x, w, dy, dt = s["x"].float(), s["w"].float(), s["dy"].float(), s["x"].dtype
            z = torch.matmul(x, w.T)
            if s["b"] is not None:
                z = z + s["b"].float()
            y = _act(z, s["act"])
            if s["r"] is not None:
                y = y + s["r"].float()
            dz = dy if s["act"] == "none" else dy * _act_grad(z, s["act"])
            out = [y.to(dt), torch.matmul(dz, w).to(dt), torch.matmul(dz.T, x).to(dt)]
            if s["b"] is not None:
                out.append(dz.sum(0).to(dt))
            if s["r"] is not None:
                out.append(s["dy"])
            return out
    if s["op"] == "ortho":
        if own:
            from cgan3d_amd import ops
            return ops.orthogonalize(s["g"], steps=STEPS, coefficients=NS, eps=EPS)
        return _orthogonal(s["g"]).to(s["g"].dtype)
    if own:
        opt = s["optimizer"]
        opt.step()
        nv = s["vectors"]
        return [opt.arena.flat, opt.arena.exp_avg, opt.arena.exp_avg_sq[-nv:]]
    p, g, (m, v) = s["p"], s["g"], s["moments"]
    s["t"] += 1
    nv, at = s["vectors"], 0
    shapes = _shapes(s)
    mats = p.numel() - nv
    m[:mats] += (1 - MOMENTUM) * (g[:mats] - m[:mats])
    u = g[:mats] + MOMENTUM * (m[:mats] - g[:mats])
    p[:mats] *= 1 - LR * DECAY
    while shapes:  # runs of one shape at once
        k = next((i for i, t in enumerate(shapes) if t != shapes[0]), len(shapes))
        r, c = shapes[0]
        o = _orthogonal(u[at:at + k * r * c].view(k, r, c))
        p[at:at + k * r * c] -= LR * math.sqrt(max(1.0, r / c)) * o.reshape(-1)
        at, shapes = at + k * r * c, shapes[k:]
    m[mats:] += (1 - V_B1) * (g[mats:] - m[mats:])
    v[mats:] = V_B2 * v[mats:] + (1 - V_B2) * g[mats:].square()
    d = (v[mats:] / (1 - V_B2 ** s["t"])).sqrt() + V_EPS
    p[mats:] -= V_LR / (1 - V_B1 ** s["t"]) * (m[mats:] / d)
    return [p, m, v[mats:]]


def _ortho_flops(r, c):
    m, n = min(r, c), max(r, c)
    return STEPS * (3.0 * m * m * n + 1.0 * m * m * m)  # X X^T and A A are symmetric: half of each


def work(case):
    if case["op"] in ("linear", "train"):
        m, k, n, e = case["rows"], case["k"], case["n"], BYTES[case["dtype"]]
        io = m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0) + m * n
        if case["op"] == "linear":
            return {"bytes": io * e, "flops": 2.0 * m * n * k}
        back = m * n + m * k + n * k + (n if case["bias"] else 0)  # dy in, the gradients out (the residual's is dy)
        return {"bytes": (io + back) * e, "flops": 6.0 * m * n * k}
    if case["op"] == "ortho":
        r, c = case["rows"], case["cols"]
        return {"bytes": 2.0 * case["batch"] * r * c * BYTES[case["dtype"]], "flops": case["batch"] * _ortho_flops(r, c)}
    shapes = _shapes(case)
    values = sum(r * c for r, c in shapes)
    return {"bytes": 4.0 * (5 * values + 7 * case["vectors"]), "flops": sum(_ortho_flops(r, c) for r, c in shapes)}


def _exact_polar(g):
    """The iteration's definition on the singular values, in 64 bits: the odd quintic applied to each of them,
    computed as a matrix polynomial of the long side's Gram matrix from the right."""
    a, b, c = NS
    x = g.double()
    flip = x.shape[-1] > x.shape[-2]
    if flip:
        x = x.mT.contiguous()  # tall: the Gram matrix of the columns is the short one
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.matmul(x.mT.contiguous(), x)
        x = torch.matmul(x, a * eye + torch.matmul(b * eye + c * gram, gram))
    return x.mT.contiguous() if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("linear", "train"):
            x, w = s["x"].double(), s["w"].double()
            z = torch.matmul(x, w.mT)
            if s["b"] is not None:
                z += s["b"].double()
            q = z.detach().requires_grad_(True)
            with torch.enable_grad():
                f = torch.nn.functional
                y = {"none": lambda t: t * 1, "relu": f.relu, "lrelu": lambda t: f.leaky_relu(t, SLOPE),
                     "tanh": torch.tanh, "gelu": f.gelu, "silu": f.silu}[case["act"]](q)
            out = y.detach() if s["r"] is None else y.detach() + s["r"].double()
            if case["op"] == "linear":
                return out
            dz, = torch.autograd.grad(y, q, s["dy"].double())
            got = [out, torch.matmul(dz, w), torch.matmul(dz.mT.contiguous(), x)]
            if s["b"] is not None:
                got.append(dz.sum(0))
            if s["r"] is not None:
                got.append(s["dy"].double())
            return got
        if case["op"] == "ortho":
            return _exact_polar(s["g"])
        p, g, m, v = (t.double() for t in (s["p"], s["g"], *s["moments"]))
        mats, at = p.numel() - case["vectors"], 0
        m2 = m.clone()
        m2[:mats] = MOMENTUM * m[:mats] + (1 - MOMENTUM) * g[:mats]
        u = (1 - MOMENTUM) * g + MOMENTUM * m2
        new = []
        for r, c in _shapes(case):
            o = _exact_polar(u[at:at + r * c].view(r, c))
            new.append((1 - LR * DECAY) * p[at:at + r * c] - LR * max(1.0, r / c) ** 0.5 * o.reshape(-1))
            at += r * c
        m2[mats:] = V_B1 * m[mats:] + (1 - V_B1) * g[mats:]
        v2 = V_B2 * v[mats:] + (1 - V_B2) * g[mats:] ** 2
        new.append(p[mats:] - V_LR * (m2[mats:] / (1 - V_B1)) / ((v2 / (1 - V_B2)).sqrt() + V_EPS))
        return [torch.cat(new), m2, v2]
