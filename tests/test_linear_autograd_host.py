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


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_derivatives_are_refused(dry, which, leaf):
    """A dual tensor's tangent is not dropped without a word, whether or not something requires grad."""
    import torch.autograd.forward_ad as fw
    from cgan3d_amd.model.linear import fused_linear
    ts = [torch.randn(6, 8), torch.randn(5, 8), torch.randn(5), torch.randn(6, 5)]
    if leaf:
        ts[which].requires_grad_(True)
    with fw.dual_level():
        fused_linear(*ts)  # no tangents: as ever
        ts[which] = fw.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fused_linear(*ts)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            fused_linear(*ts)


def test_orthogonalize_refuses_forward_mode(dry):
    import torch.autograd.forward_ad as fw
    g = torch.randn(4, 4)
    with fw.dual_level():
        dry.orthogonalize(g)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            dry.orthogonalize(fw.make_dual(g, torch.ones(4, 4)))


def test_backward_refuses_a_tangent(dry):
    import torch.autograd.forward_ad as fw
    from cgan3d_amd.model.linear import fused_linear
    x = torch.randn(6, 8).requires_grad_(True)
    with fw.dual_level():
        y = fused_linear(x, torch.randn(5, 8))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, fw.make_dual(torch.ones(6, 5), torch.ones(6, 5)))


def _uses(ops):
    from cgan3d_amd.model.linear import fused_linear
    w = torch.randn(5, 8)
    return [lambda x: fused_linear(x, w), lambda x: fused_linear(x.requires_grad_(True), w),
            lambda x: ops.orthogonalize(x)]


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("use", range(3))
def test_tracing_is_refused(dry, use, mode):
    """The program would be an empty buffer."""
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(_uses(dry)[use], tracing_mode=mode)(torch.randn(6, 8))


@pytest.mark.parametrize("use", [0, 2])
def test_jit_trace_and_fake_tensors_are_refused(dry, use):
    from torch._subclasses.fake_tensor import FakeTensorMode
    f = _uses(dry)[use]
    with pytest.raises(NotImplementedError, match="jit.trace"):
        torch.jit.trace(f, (torch.randn(6, 8),))
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError, match="fake"):
        f(torch.randn(6, 8))


def test_counting_modes_and_compiled_callers_run(dry):
    """A mode that only watches is no tracer, and a compiled caller breaks its graph at the call."""
    from torch.utils.flop_counter import FlopCounterMode
    f = _uses(dry)[0]
    with FlopCounterMode(display=False):
        assert f(torch.randn(6, 8)).shape == (6, 5)
    assert torch.compile(lambda x: f(x * 2) + 1, backend="eager")(torch.randn(6, 8)).shape == (6, 5)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_autocast_casts_the_operands(calls, dt):
    """As torch's linear: half-precision activations beside f32 parameters run in autocast's type, and the parameters'
    gradients come back in their own."""
    from cgan3d_amd.model.linear import LinearBlock
    torch.set_autocast_enabled("cuda", True)
    torch.set_autocast_dtype("cuda", dt)
    try:
        blk = LinearBlock(8, 5, torch.nn.GELU)
        for x in (torch.randn(6, 8).to(dt), torch.randn(6, 8)):
            x.requires_grad_(True)
            y = blk(x, residual=torch.randn(6, 5))
            assert y.dtype == dt
            gx, gw = torch.autograd.grad(y, (x, blk.linear.weight), torch.ones_like(y))
            assert gx.dtype == x.dtype and gw.dtype == torch.float32
        with torch.no_grad():
            assert blk(x).dtype == dt
        with pytest.raises(TypeError):
            blk(torch.randn(6, 8).double())
    finally:
        torch.set_autocast_enabled("cuda", False)
        torch.set_autocast_dtype("cuda", torch.float16)
    from cgan3d_amd import _lib as L
    assert [a.dtype for _, a in calls] == [L.DTYPES[dt]] * 5


@pytest.mark.parametrize("shape", [(1, 5), (5, 1), (1, 1, 5), (5,)])
def test_bias_of_any_shape_gets_its_gradient(dry, shape):
    """n contiguous values in any shape are a bias; the gradient has that shape."""
    from cgan3d_amd.model.linear import fused_linear
    b = torch.randn(shape).requires_grad_(True)
    y = fused_linear(torch.randn(6, 8), torch.randn(5, 8), b)
    assert torch.autograd.grad(y, b, torch.ones(6, 5))[0].shape == b.shape


def test_saved_tensors_that_come_back_transposed(calls):
    """Any strides are the hook's right: what the kernels cannot read is copied."""
    from cgan3d_amd import _lib as L
    from cgan3d_amd.model.linear import fused_linear
    x, w = torch.randn(6, 8).requires_grad_(True), torch.randn(5, 8).requires_grad_(True)
    back = []

    def unpack(t):
        back.append(t.detach().t().contiguous().t())
        return back[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = fused_linear(x, w, act=L.ACT_GELU)
    torch.autograd.grad(y, (x, w), torch.ones(6, 5))
    bwd = calls[1][1]
    assert (bwd.ldx, bwd.ldw) == (8, 8) and len(back) == 3
    assert not {bwd.x, bwd.w, bwd.preact} & {t.data_ptr() for t in back}
