"""Gated linear recurrence (engine.gated_recurrence, torch.ops.mst.gated_recurrence*, gated.hip).

CPU: the oracle's gradients against torch's autograd and against differences; fake shapes; refusals.
GPU: outputs and gradients against the float64 oracle within its float32 error bounds plus half a step
of the output type; masked frames, empty clips, views, streams, chunks, single frames, graphs.
"""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ml_music_style_transfer_amd import _lib as L
from ml_music_style_transfer_amd import engine as E
from ml_music_style_transfer_amd import kernels as K
from oracle import gated_ref as R

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def _data(B, C, T, dtype=torch.float32, seed=0, shift=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, C, T, generator=g).to(dtype)
    gate = (2 * torch.randn(B, C, T, generator=g) + shift).to(dtype)
    gh = torch.randn(B, C, T, generator=g).to(dtype)
    h0, gl = torch.randn(B, C, generator=g), torch.randn(B, C, generator=g)
    return x, gate, gh, h0, gl


# ------------------------------------------------------------------------------ CPU
def _by_torch(x, gate, h0, lengths, reverse):
    s, out = h0, [None] * x.shape[2]
    a = torch.sigmoid(gate)
    for t in (range(x.shape[2] - 1, -1, -1) if reverse else range(x.shape[2])):
        on = (t < lengths)[:, None]
        s = torch.where(on, a[..., t] * s + (1 - a[..., t]) * x[..., t], s)
        out[t] = torch.where(on, s, torch.zeros_like(s))
    return torch.stack(out, -1), s


@pytest.mark.parametrize("reverse", [False, True])
def test_oracle_gradients(reverse):
    x, gate, gh, h0, gl = (t.double() for t in _data(3, 4, 9, seed=1))
    n = torch.tensor([9, 4, 0])
    leaves = [t.clone().requires_grad_() for t in (x, gate, h0)]
    h, last = _by_torch(leaves[0], leaves[1], leaves[2], n, reverse)
    want = torch.autograd.grad((h, last), leaves, (gh, gl))
    f = R.forward(x, gate, h0, n, reverse)
    b = R.backward(f, gh, gl, reverse)
    assert torch.allclose(f["h"], h, atol=1e-13) and torch.allclose(f["last"], last, atol=1e-13)
    for got, ref in zip((b["dx"], b["dgate"], b["dh0"]), want):
        assert torch.allclose(got, ref, rtol=1e-11, atol=1e-13)
    # differences: central, error O(step^2) and the rounding's 1e-16 / step
    g = torch.Generator().manual_seed(2)
    d = [torch.randn(t.shape, generator=g).double() for t in (x, gate, h0)]

    def value(k):
        y = R.forward(x + k * d[0], gate + k * d[1], h0 + k * d[2], n, reverse)
        return (y["h"] * gh).sum() + (y["last"] * gl).sum()
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    along = sum((u * v).sum() for u, v in zip(d, (b["dx"], b["dgate"], b["dh0"])))
    assert abs(slope - along) <= 1e-7 * max(1.0, abs(float(along)))


def test_fake_shapes_and_tiles():
    lib = L.load()
    for T in (1, 512, 513, 1024, 1025, 100000):
        for dtype, code in L.TYPES.items():
            assert lib.mst_gated_tiles(code, T) == K.gated_tiles(dtype, T)
    with FakeTensorMode():
        x = torch.empty(2, 5, 1600, device="cuda", dtype=torch.bfloat16)
        h, last, carry = torch.ops.mst.gated_recurrence(x, x, None, None, False)
        assert h.shape == x.shape and h.dtype == x.dtype
        assert last.shape == (2, 5) and last.dtype == torch.float32 and carry.shape == (2, 5, K.gated_tiles(x.dtype, 1600))
        dx, dg, dh0 = torch.ops.mst.gated_recurrence_backward(h, last, x, x, None, None, carry, False)
        assert dx.shape == dg.shape == x.shape and dh0.shape == (2, 5)
        s = torch.empty(2, 5, device="cuda")
        y = torch.ops.mst.gated_recurrence_step(x[..., 0], x[..., 1], s)
        assert y.shape == (2, 5) and y.dtype == torch.bfloat16


def test_refusals():
    def z(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype)
    bad = [
        (ValueError, "one shape", (z(2, 3, 4), z(2, 3, 5))),
        (ValueError, "one shape", (z(3, 4), z(3, 4))),
        (TypeError, "both float32", (z(2, 3, 4), z(2, 3, 4, dtype=torch.bfloat16))),
        (TypeError, "both float32", (z(2, 3, 4, dtype=torch.float64), z(2, 3, 4, dtype=torch.float64))),
        (ValueError, "h0 must be", (z(2, 3, 4), z(2, 3, 4), z(3))),
        (TypeError, "floating h0", (z(2, 3, 4), z(2, 3, 4), z(2, 3, dtype=torch.int32))),
        (ValueError, "lengths must be", (z(2, 3, 4), z(2, 3, 4), None, z(3, dtype=torch.int32))),
        (TypeError, "int32 or int64", (z(2, 3, 4), z(2, 3, 4), None, z(2))),
        (RuntimeError, "no CPU path", (z(2, 3, 4), z(2, 3, 4))),
    ]
    for err, words, args in bad:
        with pytest.raises(err, match=words):
            E.gated_recurrence(*args)
    x, back = z(2, 3, 2000), torch.ops.mst.gated_recurrence_backward
    for gh, gl, carry, words in ((x, None, z(2, 3, 3), "carry must be"), (x, None, z(2, 4, 3).transpose(1, 2), "carry must be"),
                                 (x, None, z(2, 3, 4, dtype=torch.float16), "carry must be"),
                                 (z(2, 3, 1999), None, z(2, 3, 4), "a gradient of"),
                                 (x, z(3, 2), z(2, 3, 4), "a gradient of")):
        with pytest.raises(ValueError, match=words):
            back(gh, gl, x, x, None, None, carry, False)
    for err, words, args in [
            (ValueError, "one shape", (z(2, 3), z(2, 3), z(3, 2))),
            (TypeError, "both float32", (z(2, 3), z(2, 3, dtype=torch.float16), z(2, 3))),
            (TypeError, "contiguous float32 state", (z(2, 3), z(2, 3), z(2, 3, dtype=torch.float16))),
            (TypeError, "contiguous float32 state", (z(2, 3), z(2, 3), z(3, 2).t())),
            (RuntimeError, "no CPU path", (z(2, 3), z(2, 3), z(2, 3)))]:
        with pytest.raises(err, match=words):
            E.gated_recurrence_step(*args)
    with FakeTensorMode(), pytest.raises(ValueError, match="one device"):
        E.gated_recurrence(torch.zeros(1, 1, 2, device="cuda"), torch.zeros(1, 1, 2, device="cuda"),
                           torch.zeros(1, 1))


def test_c_entries_refuse():
    """Bad arguments return MST_EINVAL before anything is launched (no device is needed)."""
    lib = L.load()
    p, q = 4096, None  # never dereferenced on the host
    ok = dict(type=0, B=2, C=3, T=4, x=p, gate=p, h=p, last=p, carry=q)
    for change in (dict(type=3), dict(type=-1), dict(B=0), dict(C=0), dict(T=0), dict(T=2 ** 31 - 1),
                   dict(B=2 ** 16, C=2 ** 16), dict(x=q), dict(gate=q), dict(h=q), dict(last=q),
                   dict(T=1025, carry=q)):
        a = dict(ok, **change)
        assert lib.mst_gated_fwd(a["type"], a["x"], 12, 4, a["gate"], 12, 4, None, None, a["B"], a["C"],
                                 a["T"], 0, a["h"], a["last"], a["carry"], None, 0, None) == L.MST_EINVAL, change
        if "last" not in change:
            assert lib.mst_gated_bwd(a["type"], a["x"], 12, 4, a["gate"], 12, 4, None, None, a["carry"],
                                     None, None, a["B"], a["C"], a["T"], 0, a["h"], p, None, None,
                                     0, None) == L.MST_EINVAL, change
    for a in ((5, p, p, p, p, 2), (0, q, p, p, p, 2), (0, p, q, p, p, 2), (0, p, p, q, p, 2),
              (0, p, p, p, q, 2), (0, p, p, p, p, 0)):
        assert lib.mst_gated_step(a[0], a[1], 3, a[2], 3, a[5], 3, a[3], a[4], None) == L.MST_EINVAL


# ------------------------------------------------------------------------------ GPU
def _within(got, ref, err, what):
    got = got.detach().cpu()
    fi = torch.finfo(got.dtype)
    own = 0.0 if got.dtype == torch.float32 else fi.eps / 2  # the result's own rounding is in err
    # half a step of the type, or of its smallest steps; float32 terms below the normal range
    tol = err + own * (ref.abs() + err) + fi.smallest_normal * fi.eps / 2 + 2.0 ** -120
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((off / tol)[bad].max()):.3g} x bound"


def _run(cuda, x, gate, gh, h0=None, gl=None, lengths=None, reverse=False):
    """The framework's forward and gradients on device copies (views are kept as they are)."""
    xd, gd = (t.to(cuda).detach().requires_grad_() for t in (x, gate))
    hd = h0.to(cuda).detach().requires_grad_() if h0 is not None else None
    n = lengths.to(cuda) if lengths is not None else None
    h, last = E.gated_recurrence(xd, gd, hd, n, reverse)
    grads = torch.autograd.grad((h, last), [t for t in (xd, gd, hd) if t is not None],
                                (gh.to(cuda), gl.to(cuda) if gl is not None else torch.zeros_like(last)))
    return h, last, grads


def _check(cuda, x, gate, gh, h0=None, gl=None, lengths=None, reverse=False, got=None):
    h, last, grads = got or _run(cuda, x, gate, gh, h0, gl, lengths, reverse)
    f = R.forward(x, gate, h0, lengths, reverse)
    b = R.backward(f, gh, gl, reverse)
    _within(h, f["h"], f["h_err"], "h")
    _within(last, f["last"], f["last_err"], "last")
    _within(grads[0], b["dx"], b["dx_err"], "dx")
    _within(grads[1], b["dgate"], b["dgate_err"], "dgate")
    if h0 is not None:
        _within(grads[2], b["dh0"], b["dh0_err"], "dh0")


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True], ids=["fwd", "rev"])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 127, 129, 252, 256, 257, 511, 512, 513,
                               1000, 1024, 1025, 2049])
def test_lengths_of_the_axis(cuda, T, reverse):
    x, gate, gh, h0, gl = _data(3, 7, T, seed=T)
    _check(cuda, x, gate, gh, h0, gl, None, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("T", [1, 6, 7, 8, 9, 17, 63, 252, 257, 513, 860, 1024, 1025])
def test_types(cuda, T, dtype):
    x, gate, gh, h0, gl = _data(2, 5, T, dtype, seed=T + 1)
    for reverse in (False, True):
        _check(cuda, x, gate, gh, h0, gl, None, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [9, 100, 700])
def test_padded_clips(cuda, T, dtype):
    """Frames past a clip's length hold NaN: nothing of them comes through, h and the gradients
    are 0 there; an empty clip hands its state on; lengths outside [0, T] are taken into it."""
    x, gate, gh, h0, gl = _data(6, 3, T, dtype, seed=T)
    n = torch.tensor([T, T - 1, 1, 0, -5, T + 9], dtype=torch.int32)
    past = (torch.arange(T) >= n.clamp(0, T)[:, None])[:, None].expand(6, 3, T)
    xn, gn, ghn = (t.masked_fill(past, float("nan")) for t in (x, gate, gh))
    for reverse in (False, True):
        got = _run(cuda, xn, gn, ghn, h0, gl, n, reverse)
        _check(cuda, x, gate, gh, h0, gl, n, reverse, got)
        for t in (got[0], got[2][0], got[2][1]):
            assert (t.detach().cpu()[past] == 0).all()
        assert torch.equal(got[1][3].cpu(), h0[3]) and torch.equal(got[2][2][3].cpu(), gl[3])
    a = _run(cuda, x, gate, gh, h0, gl, n.long(), False)
    assert torch.equal(a[0], _run(cuda, x, gate, gh, h0, gl, n, False)[0])


@pytest.mark.gpu
def test_empty_shapes(cuda):
    for B, C, T in ((2, 3, 0), (0, 3, 5), (2, 0, 5)):
        x, gate, gh, h0, gl = _data(B, C, T)
        h, last, (dx, dg, dh0) = _run(cuda, x, gate, gh, h0, gl)
        assert h.shape == dx.shape == dg.shape == x.shape
        assert torch.equal(last.cpu(), h0) and torch.equal(dh0.cpu(), gl)
    x = torch.zeros(2, 3, 0, device=cuda)
    assert torch.equal(E.gated_recurrence(x, x)[1], torch.zeros(2, 3, device=cuda))


@pytest.mark.gpu
def test_views(cuda):
    """Halves of one layer's output, slices that start anywhere, other orders, expanded inputs and
    incoming gradients: the values are those of contiguous copies."""
    x, gate, gh, h0, gl = _data(3, 8, 301, seed=5)
    want = _run(cuda, x, gate, gh, h0, gl)
    z = torch.cat((x, gate), 1).to(cuda)
    wide = torch.zeros(3, 8, 311, device=cuda)
    wide[..., 7:308] = x.to(cuda)
    time_first = gate.permute(2, 0, 1).contiguous().to(cuda).permute(1, 2, 0)
    for a, b in ((z[:, :8], z[:, 8:]), (wide[..., 7:308], time_first)):
        got = _run(cuda, a.detach(), b.detach(), gh.transpose(0, 1).contiguous().transpose(0, 1), h0, gl)
        for u, v in zip((got[0], got[1], *got[2]), (want[0], want[1], *want[2])):
            assert torch.equal(u, v)
    # one clip for all, one gate for all channels, one incoming gradient for all frames
    x1, g1 = x[:1].clone(), gate[:, :1].clone()
    xd, gd = x1.to(cuda).requires_grad_(), g1.to(cuda).requires_grad_()
    h, _ = E.gated_recurrence(xd.expand(3, 8, 301), gd.expand(3, 8, 301))
    one = gh[..., :1].to(cuda)
    dx, dg = torch.autograd.grad(h, (xd, gd), one.expand(3, 8, 301))
    f = R.forward(x1.expand(3, 8, 301), g1.expand(3, 8, 301))
    b = R.backward(f, gh[..., :1].expand(3, 8, 301))
    _within(h, f["h"], f["h_err"], "h")
    # torch adds the copies' gradients: 8 terms, each addition half a step of the partial sums
    for got, ref, err, k in ((dx, b["dx"], b["dx_err"], 0), (dg, b["dgate"], b["dgate_err"], 1)):
        _within(got, ref.sum(k, keepdim=True), (err + 8 * R.U * ref.abs()).sum(k, keepdim=True), "sum")


@pytest.mark.gpu
def test_only_some_gradients(cuda):
    x, gate, gh, h0, gl = _data(2, 3, 300, seed=6)
    xd, gd, hd = x.to(cuda), gate.to(cuda).requires_grad_(), h0.to(cuda)
    h, last = E.gated_recurrence(xd, gd, hd)
    (a,) = torch.autograd.grad(h, gd, gh.to(cuda), retain_graph=True)
    (b,) = torch.autograd.grad(last, gd, gl.to(cuda))
    f = R.forward(x, gate, h0)
    for got, ref in ((a, R.backward(f, gh)), (b, R.backward(f, torch.zeros_like(gh), gl))):
        _within(got, ref["dgate"], ref["dgate_err"], "dgate")
    half = h0.bfloat16().to(cuda).requires_grad_()  # the gradient has the state's own type
    h, _ = E.gated_recurrence(xd, gate.to(cuda), half)
    assert torch.autograd.grad(h.sum(), half)[0].dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_extreme_gates_and_values(cuda, reverse):
    """Gates of the type's lowest and highest values and infinities hold or replace the state exactly;
    a value that is not finite reaches no frame before it."""
    lowest = torch.finfo(torch.float32).min
    x, gate, gh, h0, gl = _data(5, 2, 300, seed=7)
    gate[0], gate[1], gate[2], gate[3] = lowest, -lowest, float("-inf"), float("inf")
    gate[4] = torch.where(torch.arange(300) % 3 == 0, lowest, 50.0)
    h, last, grads = _run(cuda, x, gate, gh, h0, gl, None, reverse)
    for b in (0, 2):
        assert torch.equal(h[b].cpu(), x[b]) and torch.equal(grads[0][b].cpu(), _replaced(gh[b], gl[b], reverse))
    for b in (1, 3):
        assert torch.equal(h[b].cpu(), h0[b][:, None].expand(2, 300))
        assert (grads[0][b] == 0).all()
    assert (grads[1][:4] == 0).all()
    _check(cuda, x[4:], gate[4:], gh[4:], h0[4:], gl[4:], None, reverse)
    at = 137
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[4, 0, at] = bad
        hb = E.gated_recurrence(y.to(cuda), gate.to(cuda), h0.to(cuda), None, reverse)[0]
        before = slice(at + 1, None) if reverse else slice(0, at)
        assert torch.equal(hb[4, :, before], h[4, :, before]) and torch.equal(hb[4, 1], h[4, 1])
        assert torch.equal(hb[:4], h[:4])
        assert not torch.isfinite(hb[4, 0, at])
    gn = gate.clone()
    gn[4, 0, at] = float("nan")
    hb = E.gated_recurrence(x.to(cuda), gn.to(cuda), h0.to(cuda), None, reverse)[0]
    assert torch.equal(hb[4, 0, before], h[4, 0, before]) and torch.equal(hb[4, 1], h[4, 1])
    after = slice(0, at + 1) if reverse else slice(at, None)
    assert hb[4, 0, after].isnan().all()


def _replaced(gh, gl, reverse):
    """d x where every frame replaces the state: gh, and the last frame's state gradient."""
    d = gh.clone()
    d[:, 0 if reverse else -1] += gl
    return d


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,T,dtype,reverse,padded", [
    (1, 2, 33501, torch.float32, False, False),   # 66 segments of one tile
    (1, 2, 33501, torch.bfloat16, True, False),
    (2, 250, 10301, torch.float32, True, True),   # segments of two tiles, the last of one
    (2, 40, 10301, torch.float16, False, True),
    (1, 3, 5000, torch.float16, True, True),      # one wave a row
    (3, 100, 3001, torch.float32, False, False),
    (1, 300, 1500, torch.bfloat16, True, True)])
def test_long_axis(cuda, B, C, T, dtype, reverse, padded):
    x, gate, gh, h0, gl = _data(B, C, T, dtype, seed=T, shift=3.0)
    n = torch.tensor([T - 700, T // 3][:B], dtype=torch.int32) if padded else None
    _check(cuda, x, gate, gh, h0, gl, n, reverse)


@pytest.mark.gpu
def test_many_rows(cuda):
    x, gate, gh, h0, gl = _data(70, 1025, 3, seed=8)
    _check(cuda, x, gate, gh, h0, gl)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """h has more than 2^31 elements; every clip is the same expanded one."""
    T, B = 1000003, 2200
    x, gate, _, _, _ = _data(1, 1, T, torch.bfloat16, seed=9)
    xd, gd = x.to(cuda), gate.to(cuda)
    one = E.gated_recurrence(xd, gd)[0][0]
    h, last = E.gated_recurrence(xd.expand(B, 1, T), gd.expand(B, 1, T))
    assert h.numel() > 2 ** 31
    # the rows may be cut elsewhere than a single one: both within the bound of one oracle row
    f = R.forward(x[..., :4000], gate[..., :4000])
    for row in (one, h[0], h[B // 2], h[B - 1]):
        _within(row[None, :, :4000], f["h"], f["h_err"], "h")
    assert torch.equal(h[B - 1], h[0]) and (last == last[0]).all()
    del h


@pytest.mark.gpu
def test_chunks_and_single_frames_continue(cuda):
    """A recording in chunks, each from the state of the one before, and frame by frame, against the
    oracle's run over the whole: each piece is the same recurrence, so the same bounds hold."""
    x, gate, _, h0, _ = _data(2, 9, 400, seed=10)
    f = R.forward(x, gate, h0)
    xd, gd = x.to(cuda), gate.to(cuda)
    s, out = h0.to(cuda), []
    for a, b in ((0, 1), (1, 130), (130, 131), (131, 400)):
        h, s = E.gated_recurrence(xd[..., a:b], gd[..., a:b], s)
        out.append(h)
    _within(torch.cat(out, -1), f["h"], f["h_err"], "chunks")
    _within(s, f["last"], f["last_err"], "state")
    s = h0.to(cuda)
    frames = []
    for t in range(400):
        frames.append(E.gated_recurrence_step(xd[..., t], gd[..., t], s))
    _within(torch.stack(frames, -1), f["h"], f["h_err"], "frames")
    _within(s, f["last"], f["last_err"], "state")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,C", [(1, 1), (1, 1025), (3, 64), (257, 129)])
def test_step(cuda, B, C, dtype):
    x, gate, _, h0, _ = _data(B, C, 1, dtype, seed=B + C)
    f = R.forward(x, gate, h0)
    z = torch.cat((x[..., 0], gate[..., 0]), 1).to(cuda)
    for a, b in ((x[..., 0].to(cuda), gate[..., 0].to(cuda)), (z[:, :C], z[:, C:]),
                 (x[..., 0].t().contiguous().to(cuda).t(), gate[..., 0].to(cuda))):
        s = h0.to(cuda)
        y = E.gated_recurrence_step(a, b, s)
        assert y.dtype == dtype
        _within(y, f["last"], f["last_err"], "y")
        _within(s, f["last"], f["last_err"], "state")
    s = torch.zeros(0, C, device=cuda)
    assert E.gated_recurrence_step(z[:0, :C], z[:0, C:], s).shape == (0, C)


@pytest.mark.gpu
def test_another_stream_and_two_calls_at_once(cuda):
    x, gate, gh, h0, gl = _data(2, 64, 5000, seed=11)
    want = _run(cuda, x, gate, gh, h0, gl)
    dev = [t.to(cuda) for t in (x, gate, gh, h0, gl)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_run(cuda, *dev[:3], h0=dev[3].detach(), gl=dev[4]))
    torch.cuda.synchronize()
    for h, last, grads in got:
        for u, v in zip((h, last, *grads), (want[0], want[1], *want[2])):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_captured_forward_and_backward(cuda):
    """Replays give the eager results, with eager calls and other work between them."""
    x, gate, gh, h0, gl = _data(1, 16, 6000, seed=12)
    static = [t.to(cuda) for t in (x, gate, gh, h0, gl)]

    def program():
        a, b, c = (t.detach().requires_grad_() for t in (static[0], static[1], static[3]))
        h, last = E.gated_recurrence(a, b, c)
        return (h, last, *torch.autograd.grad((h, last), (a, b, c), (static[2], static[4])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        program()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs with a workspace each
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, program()))
    for k in range(3):
        fresh = _data(1, 16, 6000, seed=20 + k)
        for s, t in zip(static, fresh):
            s.copy_(t)
        for graph, _ in graphs:
            graph.replay()
        want = program()
        torch.cuda.synchronize()
        for _, out in graphs:
            for u, v in zip(out, want):
                assert torch.equal(u, v)


@pytest.mark.gpu
def test_step_captured(cuda):
    x, gate, _, h0, _ = _data(4, 33, 3, torch.bfloat16, seed=13)
    xs, gs, s = x[..., 0].to(cuda), gate[..., 0].to(cuda), h0.to(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        E.gated_recurrence_step(xs, gs, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = E.gated_recurrence_step(xs, gs, s)
    s.copy_(h0)
    e = h0.to(cuda)
    for t in range(3):
        xs.copy_(x[..., t])
        gs.copy_(gate[..., t])
        graph.replay()
        assert torch.equal(y, E.gated_recurrence_step(x[..., t].to(cuda), gate[..., t].to(cuda), e))
    assert torch.equal(s, e)


@pytest.mark.gpu
def test_operator_and_direct_call_agree(cuda):
    """engine's direct calls and the registered operator are the same kernels; inference mode; the
    in-place update counts in the state's version."""
    x, gate, gh, h0, _ = (t.to(cuda) for t in _data(2, 5, 700, seed=15))
    leaves = [t.clone().requires_grad_() for t in (x, gate, h0)]
    want = torch.ops.mst.gated_recurrence(*leaves, None, True)
    grads = torch.autograd.grad(want[0], leaves, gh)
    h, last = E.gated_recurrence(*leaves, None, True)
    assert torch.equal(h, want[0]) and torch.equal(last, want[1])
    for a, b in zip(torch.autograd.grad(h, leaves, gh), grads):
        assert torch.equal(a, b)
    with torch.inference_mode():
        h, last = E.gated_recurrence(x, gate, h0, None, True)
        assert torch.equal(h, want[0]) and torch.equal(last, want[1])
        s = h0.clone()
        y = E.gated_recurrence_step(x[..., 0], gate[..., 0], s)
    s2 = h0.clone()
    version = s2._version
    assert torch.equal(torch.ops.mst.gated_recurrence_step(x[..., 0], gate[..., 0], s2), y)
    assert torch.equal(s, s2) and s2._version > version
    s3 = h0.clone()
    version = s3._version
    E.gated_recurrence_step(x[..., 0], gate[..., 0], s3)
    assert s3._version > version


@pytest.mark.gpu
def test_traced_and_differentiated_twice(cuda):
    """A traced call goes through the registered operators and gives the direct call's values; a
    second derivative is refused."""
    x, gate, _, h0, _ = (t.to(cuda) for t in _data(2, 5, 700, seed=16))

    def value(x, gate, h0):
        h, last = E.gated_recurrence(x, gate, h0, None, True)
        return (h * h).sum() + last.sum()

    def frame(x, gate, state):
        return E.gated_recurrence_step(x, gate, state) + 1
    a, b = ([t.clone().requires_grad_() for t in (x, gate, h0)] for _ in range(2))
    value(*a).backward()
    torch.compile(value, backend="aot_eager", fullgraph=True)(*b).backward()
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad)
    s, t = h0.clone(), h0.clone()
    with torch.no_grad():
        y = torch.compile(frame, backend="aot_eager", fullgraph=True)(x[..., 0], gate[..., 0], t)
        assert torch.equal(frame(x[..., 0], gate[..., 0], s), y) and torch.equal(s, t)
    grads = torch.autograd.grad(value(*a), a, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].sum().backward()


@pytest.mark.gpu
def test_opcheck(cuda):
    x, gate, _, h0, _ = _data(2, 3, 300, seed=14)
    args = (x.to(cuda).requires_grad_(), gate.to(cuda).requires_grad_(), h0.to(cuda).requires_grad_(),
            torch.tensor([300, 17], dtype=torch.int32, device=cuda), True)
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.mst.gated_recurrence, args, test_utils=checks)
    torch.library.opcheck(torch.ops.mst.gated_recurrence_step,
                          (x[..., 0].to(cuda), gate[..., 0].to(cuda), h0.to(cuda)), test_utils=checks)
