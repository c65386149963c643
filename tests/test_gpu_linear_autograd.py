"""The linear block under hooks on saved tensors, autocast and the engine's own machinery, on the GPU: against the same
call without them, to the last bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def operands(rows, k, n, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((rows, k), (n, k), (n,), (rows, n), (rows, n))]


@pytest.mark.parametrize("rows,k,n", [(700, 96, 64), (64, 8, 5), (300, 200, 120)])
@pytest.mark.parametrize("act", ["NONE", "GELU"])
def test_activations_that_leave_and_come_back_dense(rows, k, n, act):
    """A row-strided activation goes to the host, its block is freed, and the dense copy may lie at its address."""
    from cgan3d_amd import _lib as L
    from cgan3d_amd.model.linear import fused_linear
    code = getattr(L, "ACT_" + act)
    x, w, b, r, dy = operands(rows, k, n, 1)
    w.requires_grad_(True)

    def run(hooks):
        wide = torch.zeros(rows, 2 * k, device="cuda")
        wide[:, :k] = x
        wide.requires_grad_(True)
        view = (wide * 1)[:, :k]  # its block belongs to the graph alone
        assert view.stride(0) == 2 * k
        with hooks:
            y = fused_linear(view, w, b, r, code)
        del view
        junk = [torch.full((rows, k), float("nan"), device="cuda") for _ in range(3)]
        del junk
        gx, gw = torch.autograd.grad(y, (wide, w), dy)
        return gx[:, :k].clone(), gw
    want = run(torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    away = torch.autograd.graph.saved_tensors_hooks(lambda t: t if t.data_ptr() == w.data_ptr() else t.cpu(), lambda t: t.cuda())
    for _ in range(3):
        got = run(away)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(dtype):
    from cgan3d_amd.model.linear import LinearBlock
    blk = LinearBlock(72, 40, torch.nn.SiLU).cuda()
    x, _, _, r, dy = operands(130, 72, 40, 2)
    x.requires_grad_(True)
    with torch.autocast("cuda", dtype=dtype):
        y = blk(x, residual=r)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, (x, *blk.parameters()), dy.to(dtype))
    half = LinearBlock(72, 40, torch.nn.SiLU).cuda().to(dtype)
    half.load_state_dict({k: v.to(dtype) for k, v in blk.state_dict().items()})
    xh = x.detach().to(dtype).requires_grad_(True)
    yh = half(xh, residual=r.to(dtype))
    assert torch.equal(y, yh)
    want = torch.autograd.grad(yh, (xh, *half.parameters()), dy.to(dtype))
    assert all(a.dtype == torch.float32 and torch.equal(a, c.float()) for a, c in zip(got, want))


def test_checkpointed_block():
    """Recomputed in the backward pass: the operands are other tensors of the same values."""
    from torch.utils.checkpoint import checkpoint
    from cgan3d_amd.model.linear import LinearBlock
    blk = torch.nn.Sequential(LinearBlock(48, 96, torch.nn.GELU), LinearBlock(96, 48, torch.nn.Tanh)).cuda()
    x, _, _, _, dy = operands(200, 48, 48, 3)
    x.requires_grad_(True)
    leaves = (x, *blk.parameters())
    want = torch.autograd.grad(blk(x), leaves, dy)
    for reentrant in (False, True):
        y = checkpoint(blk, x, use_reentrant=reentrant)
        if reentrant:  # takes backward() alone
            for t in leaves:
                t.grad = None
            y.backward(dy)
            got = [t.grad for t in leaves]
        else:
            got = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
