"""The recurrence under what records or differentiates a program (engine.gated_recurrence*,
torch.ops.mst.gated_recurrence*), on the CPU with the kernels' wrappers replaced by plain torch."""
import pytest
import torch
from torch.autograd import forward_ad as fwAD

from ml_music_style_transfer_amd import engine as E
from ml_music_style_transfer_amd import kernels as K
from oracle import gated_ref as R


def _plain(x, gate, h0, reverse=False):
    s, out = h0, []
    a = torch.sigmoid(gate)
    for t in (range(x.shape[2] - 1, -1, -1) if reverse else range(x.shape[2])):
        s = a[..., t] * s + (1 - a[..., t]) * x[..., t]
        out.append(s)
    return torch.stack(out[::-1] if reverse else out, -1), s


@pytest.fixture(autouse=True)
def kernels(monkeypatch):
    """As the kernels' wrappers do it: outputs allocated and then filled by a call that no tracer sees."""
    def fill(out, values):
        out.numpy()[...] = values.numpy()
        return out

    def fwd(x, gate, h0, lengths, reverse):
        x, gate = x.detach(), gate.detach()
        h0 = torch.zeros(x.shape[:2]) if h0 is None else h0.detach()
        h, last = _plain(x, gate, h0, reverse)
        return fill(torch.empty(x.shape), h), fill(torch.empty(x.shape[:2]), last), torch.empty(*x.shape[:2], 0)

    def bwd(gh, gl, x, gate, h0, lengths, carry, reverse, need_dh0=True):
        x, gate, gh, gl = (None if t is None else t.detach() for t in (x, gate, gh, gl))
        f = R.forward(x, gate, None if h0 is None else h0.detach(), lengths, reverse)
        g = R.backward(f, torch.zeros_like(x) if gh is None else gh, gl, reverse)
        return tuple(g[k].float() for k in ("dx", "dgate", "dh0"))

    def step(x, gate, state):
        a = torch.sigmoid(gate.detach())
        state.detach().copy_(a * state.detach() + (1 - a) * x.detach())
        return fill(torch.empty(x.shape), state.detach())
    for name, f in (("gated_fwd", fwd), ("gated_bwd", bwd), ("gated_step", step)):
        monkeypatch.setattr(K, name, f)


def _data(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 3, 7, generator=g), torch.randn(2, 3, 7, generator=g), torch.randn(2, 3, generator=g)]


def test_traced_call_is_recorded():
    """torch.jit.trace records the operator, not the memory that a direct call returned."""
    traced = torch.jit.trace(lambda x, gate, h0: E.gated_recurrence(x, gate, h0, None, True), _data(1))
    assert any(n.kind() == "mst::gated_recurrence" for n in traced.graph.nodes())
    fresh = _data(2)
    for got, want in zip(traced(*fresh), _plain(*fresh, reverse=True)):
        assert torch.equal(got, want)


def test_traced_frame_is_recorded():
    x, gate, h0 = _data(3)
    traced = torch.jit.trace(E.gated_recurrence_step, (x[..., 0], gate[..., 0], h0.clone()), check_trace=False)
    assert any(n.kind() == "mst::gated_recurrence_step" for n in traced.graph.nodes())
    state, want = h0.clone(), _plain(x[..., 1:2], gate[..., 1:2], h0)[1]
    assert torch.equal(traced(x[..., 1], gate[..., 1], state), want) and torch.equal(state, want)


def _forms(x, gate, h0):
    """Each public form as a function of one input, with that input's value."""
    op = torch.ops.mst.gated_recurrence
    step = torch.ops.mst.gated_recurrence_step
    carry = torch.empty(2, 3, 0)
    return {
        "x": (lambda v: E.gated_recurrence(v, gate, h0)[0], x),
        "gate": (lambda v: E.gated_recurrence(x, v, h0)[0], gate),
        "h0": (lambda v: E.gated_recurrence(x, gate, v)[1], h0),
        "frame": (lambda v: E.gated_recurrence_step(v, gate[..., 0], h0.clone()), x[..., 0]),
        "operator": (lambda v: op(v, gate, h0, None, False)[0], x),
        "operator frame": (lambda v: step(x[..., 0], v, h0.clone()), gate[..., 0]),
        "operator backward": (lambda v: torch.ops.mst.gated_recurrence_backward(v, None, x, gate, h0, None, carry,
                                                                                False)[0], x),
    }


@pytest.mark.parametrize("form", list(_forms(*_data(0))))
def test_forward_mode_is_refused(form):
    """A tangent is refused, not dropped: dual tensors, torch.func.jvp and jacfwd."""
    f, at = _forms(*_data(4))[form]
    words = "no forward-mode derivative"
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match=words):
        f(fwAD.make_dual(at, torch.ones_like(at)))
    with pytest.raises(NotImplementedError, match=words):
        torch.func.jvp(f, (at,), (torch.ones_like(at),))


@pytest.mark.parametrize("call", [E.gated_recurrence, lambda *a: torch.ops.mst.gated_recurrence(*a, None, False)])
def test_dual_gradients_are_refused(call):
    leaves = [t.requires_grad_() for t in _data(5)]
    h = call(*leaves)[0]
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.autograd.grad(h, leaves, fwAD.make_dual(torch.ones_like(h), torch.ones_like(h)))


def test_constants_inside_forward_mode():
    """Without a tangent among its own inputs the call is an ordinary one, gradients included."""
    x, gate, h0 = _data(6)
    want = _plain(x, gate, h0)[0]
    frame = _plain(x[..., :1], gate[..., :1], h0)[1]

    def f(v):
        assert torch.equal(E.gated_recurrence_step(x[..., 0], gate[..., 0], h0.clone()), frame)
        return v * E.gated_recurrence(x, gate, h0)[0]
    y, t = torch.func.jvp(f, (x,), (torch.ones_like(x),))
    assert torch.equal(y, x * want) and torch.equal(t, want)
    leaves = [v.clone().requires_grad_() for v in (x, gate, h0)]
    grads = torch.autograd.grad(_plain(*leaves)[0].sum(), leaves)
    with fwAD.dual_level():
        assert torch.equal(fwAD.unpack_dual(f(fwAD.make_dual(x, torch.ones_like(x)))).tangent, want)
        for a, b in zip(torch.autograd.grad(E.gated_recurrence(*leaves)[0].sum(), leaves), grads):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
        h = E.gated_recurrence(*leaves)[0]
    for a, b in zip(torch.autograd.grad(h.sum(), leaves), grads):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
