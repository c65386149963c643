"""What torch's machinery around autograd does to the linear block and the orthogonalisation (no GPU: the wrappers in
dry-run mode, the C entry points' arguments recorded instead of launched)."""
import pytest
import torch


@pytest.fixture
def dry():
    from cgan3d_amd import ops
    ops.DRY_RUN = True
    yield ops
    ops.DRY_RUN = False


@pytest.fixture
def calls(dry, monkeypatch):
    """The arguments of every linear call, in order."""
    from cgan3d_amd import _lib as L
    seen = []

    def record(entry, a, device, ws, who):
        seen.append((entry, L.LinearArgs.from_buffer_copy(a)))
    monkeypatch.setattr(dry, "_linear_call", record)
    return seen


@pytest.mark.parametrize("operand", ["x", "w", "x dtype"])
def test_saved_tensors_that_come_back_dense_at_their_old_address(calls, operand):
    """A hook that gives an operand back in the block that the freed one lay in, but with other strides (or another
    type): the backward call has to go by the tensor it gets."""
    from cgan3d_amd.model.linear import fused_linear
    x = torch.randn(6, 16)[:, :8].requires_grad_(True)
    w = torch.randn(5, 24)[:, :8].requires_grad_(True)
    at = {"x": x, "w": w, "x dtype": x}[operand]

    def unpack(t):
        if t.data_ptr() != at.data_ptr():
            return t
        if operand == "x dtype":
            return t.detach().view(torch.bfloat16)[:, :8]
        dense = torch.as_strided(t.detach(), t.shape, (t.shape[1], 1))
        assert dense.data_ptr() == t.data_ptr()
        return dense
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = fused_linear(x, w)
    if operand == "x dtype":
        with pytest.raises(TypeError):
            torch.autograd.grad(y, (x, w), torch.ones(6, 5))
        return
    torch.autograd.grad(y, (x, w), torch.ones(6, 5))
    (_, fwd), (entry, bwd) = calls
    assert entry == "cgan3d_linear_bwd" and (fwd.ldx, fwd.ldw) == (16, 24)
    assert (bwd.ldx, bwd.ldw) == ((8, 24) if operand == "x" else (16, 8))
    assert (bwd.x, bwd.w) == (x.data_ptr(), w.data_ptr())


def test_saved_tensors_that_stay_take_the_forward_arguments(calls):
    from cgan3d_amd.model.linear import fused_linear
    x = torch.randn(6, 16)[:, :8].requires_grad_(True)
    w = torch.randn(5, 8).requires_grad_(True)
    torch.autograd.grad(fused_linear(x, w), (x, w), torch.ones(6, 5))
    bwd = calls[1][1]
    assert (bwd.ldx, bwd.ldw, bwd.x, bwd.w) == (16, 8, x.data_ptr(), w.data_ptr())
