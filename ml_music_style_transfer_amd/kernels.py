"""Thin tensor-level wrappers over libmst_hip's C ABI (include/mst.h).

Every function enqueues HIP kernels on torch's current stream and returns
without synchronising. Tensors must be contiguous float32 CUDA tensors; there
is deliberately no CPU fallback (see _lib.ptr).

Layer geometry (all implicit GEMMs of gemm.hip; reference model/model.py):
  conv3   nn.Conv1d(k=3, p=1)                       model.py:14-22
  convT2  nn.ConvTranspose1d(k, s=2, p=1)           model.py:24-31   (two sub-pixel phases)
  convT1  nn.ConvTranspose1d(k=3, s=1, p=1)         model.py:242     (lastconv)
  linear  nn.Linear over channels of an NCL tensor  model.py:98-99,104-107
Sources are (tensor, time_offset) pairs forming a virtual channel concat; the
offset implements crop_and_concat (model.py:71-78).
"""
import ctypes
import os
import threading
from array import array

import torch
from torch.autograd import forward_ad

from . import _lib as L

SLOPE = 0.01
IN_EPS = 1e-5
# dev-only A/B knob: force one K schedule on every GEMM (mst_conv_desc.splitk semantics)
_FORCE_SPLITK = int(os.environ.get("MST_FORCE_SPLITK", "0"))


def _lib():
    return L.load()


def empty(*shape, like=None, device=None):
    dev = like.device if like is not None else device
    return torch.empty(shape, device=dev, dtype=torch.float32)


def _src(spec):
    s = L.MstSrc()
    if spec is None:
        return s
    t, off = spec
    # any NCL view with unit time stride works (e.g. the channel halves of torch.split, train.py:130)
    assert t.dim() == 3 and t.stride(2) == 1 and t.dtype == torch.float32 and t.is_cuda
    s.p = t.data_ptr()
    s.sb = t.stride(0)
    s.sc = t.stride(1)
    s.C = t.shape[1]
    s.T = t.shape[2]
    s.off = off
    return s


def _dst(spec):
    d = L.MstDst()
    if spec is None:
        return d
    t, off, gate, gscale = spec
    assert t.is_contiguous() and t.dim() == 3
    d.p = t.data_ptr()
    d.sb = t.shape[1] * t.shape[2]
    d.sc = t.shape[2]
    d.C = t.shape[1]
    d.T = t.shape[2]
    d.off = off
    if gate is not None:
        assert gate.shape == t.shape
        d.gate = gate.data_ptr()
        d.gate_scale = gscale
    return d


# Workspace arena: one grow-only scratch buffer per (host thread, device, launch stream). Launches on
# one stream are ordered, so consecutive GEMM split-K slabs and loss partials share it instead of
# paying an allocator round trip each. Threads do not share: the launches of one call leave data for
# each other there, and another thread's launches may come between them (autograd's thread has its
# own, so a training step holds two). An outgrown buffer is simply dropped: torch's caching
# allocator hands its block out again only in this stream's order, after the launches already
# queued on it. Under stream capture the arena is bypassed (each launch takes a fresh buffer
# from the graph's private pool, torch's capture semantics), so no graph names an arena
# buffer. Requests above ARENA_MAX_BYTES (Griffin-Lim's multi-GB clip chunks) are one-off
# allocations that return to the allocator after the call instead of staying pinned here.
class _Arena(threading.local):
    def __init__(self):
        self.buffers = {}


_ARENA = _Arena()
ARENA_MAX_BYTES = 256 << 20


def workspace(nbytes, device):
    """(float32 buffer of >= nbytes, its byte size) for one launch on the current stream."""
    if nbytes == 0:
        return None, 0
    n = (nbytes + 3) // 4
    if torch.cuda.is_current_stream_capturing() or nbytes > ARENA_MAX_BYTES:
        return torch.empty(n, device=device, dtype=torch.float32), 4 * n
    key, arena = (device.index, L.stream().value), _ARENA.buffers
    buf = arena.get(key)
    if buf is None or buf.numel() < n:
        if buf is not None:
            n = min(max(n, 2 * buf.numel()), ARENA_MAX_BYTES // 4)
        arena[key] = None  # release the outgrown block before taking the larger one
        buf = arena[key] = torch.empty(n, device=device, dtype=torch.float32)
    return buf, 4 * buf.numel()


_workspace = workspace


# Optional per-launch GEMM timing (bench.py's roofline leg): when a list is installed, every
# GEMM launch is bracketed by HIP events on torch's current stream (the launch stream).
_GEMM_LOG = None


def gemm_timing(log):
    """Install (list) or remove (None) the GEMM timing log; entries are (start, end, flops, tag)."""
    global _GEMM_LOG
    _GEMM_LOG = log


def _timed(launch, flops, tag, shape=None):
    if _GEMM_LOG is None:
        launch()
        return
    s = torch.cuda.Event(enable_timing=True)
    e = torch.cuda.Event(enable_timing=True)
    s.record()
    launch()
    e.record()
    _GEMM_LOG.append((s, e, flops, tag, shape))


def conv_like(*, B, M, Tn, srcs, Tv, taps, a, beta, g, A, A_off=0, sAm, sAc, sAt, dsts, ostride=1,
              ophase=0, alpha=1.0, bias=None, act=L.ACT_NONE, drop_p=0.0, seed=0, splitk=0,
              seed_dev=None):
    lib = _lib()
    d = L.MstConvDesc()
    d.B, d.M, d.Tn, d.taps = B, M, Tn, taps
    d.Ctot = sum(s[0].shape[1] for s in srcs)
    d.a, d.beta, d.g, d.Tv = a, beta, g, Tv
    d.A = A.data_ptr() + 4 * A_off
    d.sAm, d.sAc, d.sAt = sAm, sAc, sAt
    d.src[0] = _src(srcs[0])
    d.src[1] = _src(srcs[1] if len(srcs) > 1 else None)
    d.ostride, d.ophase = ostride, ophase
    d.dst[0] = _dst(dsts[0])
    d.dst[1] = _dst(dsts[1] if len(dsts) > 1 else None)
    d.alpha = alpha
    d.bias = bias.data_ptr() if bias is not None else None
    d.act = act
    d.drop_p = drop_p
    d.seed = seed
    d.seed_dev = seed_dev.data_ptr() if seed_dev is not None else None
    d.splitk = splitk or _FORCE_SPLITK
    ref = ctypes.byref(d)
    need = lib.mst_conv_fwd_workspace_size(ref)  # split-K: splits * M * N * 4 bytes
    ws, nb = _workspace(need, A.device)
    _timed(lambda: L.check(lib.mst_conv_fwd_f32(ref, L.ptr(ws), nb, L.stream()), "mst_conv_fwd_f32"),
           2.0 * M * B * Tn * d.Ctot * taps, "conv", (M, B * Tn, d.Ctot * taps, taps, a, need))


def wgrad_like(*, P, srcs, Tv, taps, a, beta, g, out, ldo, ldc=0, ldt=0, scale=1.0, accumulate=False,
               splitk=0):
    """out[m*ldo + c*ldc + tap*ldt] (+)= scale * sum_{b,t} P[b][m][t] X(b, c, a*t+beta+g*tap);
    ldc = ldt = 0 means the torch layout (ldc = taps, ldt = 1)."""
    lib = _lib()
    d = L.MstWgradDesc()
    B, M, Tk = P.shape
    d.B, d.M, d.Tk, d.taps = B, M, Tk, taps
    d.Ctot = sum(s[0].shape[1] for s in srcs)
    d.a, d.beta, d.g, d.Tv = a, beta, g, Tv
    d.P = P.data_ptr()
    d.sPb = M * Tk
    d.sPc = Tk
    d.src[0] = _src(srcs[0])
    d.src[1] = _src(srcs[1] if len(srcs) > 1 else None)
    d.out = out.data_ptr()
    d.ldo = ldo
    d.ldc, d.ldt = ldc, ldt
    d.scale = scale
    d.accumulate = 1 if accumulate else 0
    d.splitk = splitk or _FORCE_SPLITK
    ref = ctypes.byref(d)
    need = lib.mst_wgrad_workspace_size(ref)  # split-K: splits * M * (source's C * taps) * 4 bytes
    ws, nb = _workspace(need, P.device)
    _timed(lambda: L.check(lib.mst_conv_wgrad_f32(ref, L.ptr(ws), nb, L.stream()),
                           "mst_conv_wgrad_f32"), 2.0 * M * B * Tk * d.Ctot * taps, "wgrad",
           (M, d.Ctot * taps, B * Tk, taps, a, need))


def _wgrad_out(dW):
    """(ldo, ldc, ldt) of a (d0, C, taps) weight-gradient tensor in any layout."""
    return dW.stride(0), dW.stride(1), dW.stride(2)


# ---------------------------------------------------------------- Conv1d k3 p1
# Weights may be in the torch layout or tap-major (model.slot_view): every A operand takes
# its strides from the tensor.
def conv3_fwd(srcs, W, bias, out, act=L.ACT_NONE):
    B, Cout, T = out.shape
    conv_like(B=B, M=Cout, Tn=T, srcs=srcs, Tv=T, taps=3, a=1, beta=-1, g=1, A=W, sAm=W.stride(0),
              sAc=W.stride(1), sAt=W.stride(2), dsts=[(out, 0, None, 1.0)], bias=bias, act=act)


def conv3_dgrad(dY, W, dsts):
    B, Cout, T = dY.shape
    Cin = W.shape[1]
    conv_like(B=B, M=Cin, Tn=T, srcs=[(dY, 0)], Tv=T, taps=3, a=1, beta=1, g=-1, A=W,
              sAm=W.stride(1), sAc=W.stride(0), sAt=W.stride(2), dsts=dsts)


def conv3_wgrad(dY, srcs, dW, accumulate):
    ldo, ldc, ldt = _wgrad_out(dW)
    wgrad_like(P=dY, srcs=srcs, Tv=dY.shape[2], taps=3, a=1, beta=-1, g=1, out=dW, ldo=ldo, ldc=ldc,
               ldt=ldt, accumulate=accumulate)


# ------------------------------------------------- ConvTranspose1d(k, s=2, p=1)
def convT2_out_len(Tin, k):
    return (Tin - 1) * 2 - 2 + k


def convT2_fwd(x, W, bias, out):
    Cin, Cout, k = W.shape
    B, _, Tin = x.shape
    Tout = out.shape[2]
    for p in (0, 1):
        nq = k // 2 if p == 0 else (k + 1) // 2
        Tn = (Tout - p + 1) // 2
        if nq == 0 or Tn <= 0:
            continue
        conv_like(B=B, M=Cout, Tn=Tn, srcs=[(x, 0)], Tv=Tin, taps=nq, a=1, beta=p, g=-1, A=W,
                  A_off=(1 - p) * W.stride(2), sAm=W.stride(1), sAc=W.stride(0), sAt=2 * W.stride(2),
                  dsts=[(out, 0, None, 1.0)], ostride=2, ophase=p, bias=bias)


def convT2_dgrad(dY, W, dsts):
    Cin, Cout, k = W.shape
    B, _, Tout = dY.shape
    Tin = dsts[0][0].shape[2]
    conv_like(B=B, M=Cin, Tn=Tin, srcs=[(dY, 0)], Tv=Tout, taps=k, a=2, beta=-1, g=1, A=W,
              sAm=W.stride(0), sAc=W.stride(1), sAt=W.stride(2), dsts=dsts)


def convT2_wgrad(x, dY, dW, accumulate):
    Cin, Cout, k = dW.shape
    ldo, ldc, ldt = _wgrad_out(dW)
    wgrad_like(P=x, srcs=[(dY, 0)], Tv=dY.shape[2], taps=k, a=2, beta=-1, g=1, out=dW, ldo=ldo,
               ldc=ldc, ldt=ldt, accumulate=accumulate)


# ------------------------------------------- ConvTranspose1d(k=3, s=1, p=1) (lastconv)
def convT1_fwd(x, W, bias, out, alpha=1.0, act=L.ACT_NONE):
    Cin, Cout, k = W.shape
    B, _, T = x.shape
    conv_like(B=B, M=Cout, Tn=T, srcs=[(x, 0)], Tv=T, taps=k, a=1, beta=1, g=-1, A=W,
              sAm=W.stride(1), sAc=W.stride(0), sAt=W.stride(2), dsts=[(out, 0, None, 1.0)],
              alpha=alpha, bias=bias, act=act)


def convT1_dgrad(dY, W, dx, alpha=1.0):
    Cin, Cout, k = W.shape
    B, _, T = dY.shape
    conv_like(B=B, M=Cin, Tn=T, srcs=[(dY, 0)], Tv=T, taps=k, a=1, beta=-1, g=1, A=W,
              sAm=W.stride(0), sAc=W.stride(1), sAt=W.stride(2), dsts=[(dx, 0, None, 1.0)],
              alpha=alpha)


def convT1_wgrad(x, dY, dW, accumulate, scale=1.0):
    ldo, ldc, ldt = _wgrad_out(dW)
    wgrad_like(P=x, srcs=[(dY, 0)], Tv=dY.shape[2], taps=dW.shape[2], a=1, beta=-1, g=1, out=dW,
               ldo=ldo, ldc=ldc, ldt=ldt, scale=scale, accumulate=accumulate)


# ------------------------------------------------------- Linear over NCL channels
def linear_fwd(srcs, W, bias, out, act=L.ACT_NONE, drop_p=0.0, seed=0, seed_dev=None):
    B, Cout, T = out.shape
    Cin = W.shape[1]
    conv_like(B=B, M=Cout, Tn=T, srcs=srcs, Tv=T, taps=1, a=1, beta=0, g=0, A=W, sAm=Cin, sAc=1,
              sAt=1, dsts=[(out, 0, None, 1.0)], bias=bias, act=act, drop_p=drop_p, seed=seed,
              seed_dev=seed_dev)


def linear_dgrad(dY, W, dsts):
    B, Cout, T = dY.shape
    Cin = W.shape[1]
    conv_like(B=B, M=Cin, Tn=T, srcs=[(dY, 0)], Tv=T, taps=1, a=1, beta=0, g=0, A=W, sAm=1,
              sAc=Cin, sAt=1, dsts=dsts)


def linear_wgrad(dY, srcs, dW, accumulate):
    wgrad_like(P=dY, srcs=srcs, Tv=dY.shape[2], taps=1, a=1, beta=0, g=0, out=dW,
               ldo=dW.shape[1], accumulate=accumulate)


# ---------------------------------------------------------- norm / elementwise
def in_lrelu_fwd(y, pool):
    B, C, T = y.shape
    a = torch.empty_like(y)
    pooled = empty(B, C, T // 2, like=y) if pool else None
    mean = empty(B * C, like=y)
    rstd = empty(B * C, like=y)
    L.check(_lib().mst_instnorm_lrelu_fwd_f32(L.ptr(y), B * C, T, IN_EPS, SLOPE, L.ptr(a),
                                              L.ptr(pooled), L.ptr(mean), L.ptr(rstd), L.stream()),
            "instnorm_fwd")
    return a, pooled, mean, rstd


def in_lrelu_bwd(y, mean, rstd, d_a=None, d_pool0=None, d_pool1=None, rowsum=False):
    """IN + LeakyReLU (+ maxpool) backward. rowsum=True also returns the (B, C) per-row sums of
    dy (the producing conv's bias gradient before the batch reduction, bias_grad_rows)."""
    B, C, T = y.shape
    dy = torch.empty_like(y)
    rs = empty(B, C, like=y) if rowsum else None
    L.check(_lib().mst_instnorm_lrelu_bwd_f32(L.ptr(y), L.ptr(mean), L.ptr(rstd), B * C, T, SLOPE,
                                              L.ptr(d_a), L.ptr(d_pool0), L.ptr(d_pool1), L.ptr(dy),
                                              L.ptr(rs), L.stream()), "instnorm_bwd")
    return (dy, rs) if rowsum else dy


def bias_grad_rows(rs, db, accumulate):
    """db (+)= sum over the batch of per-(b, c) row sums (from in_lrelu_bwd(rowsum=True))."""
    B, C = rs.shape
    L.check(_lib().mst_bias_grad_rows_f32(L.ptr(rs), B, C, 1.0, L.ptr(db), 1 if accumulate else 0,
                                          L.stream()), "bias_grad_rows")


def bias_grad(dy, db, accumulate):
    if not dy.is_contiguous() or not db.is_contiguous():
        raise ValueError("bias_grad: contiguous (B, C, T) dy and (C,) db required")
    B, C, T = dy.shape
    L.check(_lib().mst_bias_grad_f32(L.ptr(dy), B, C, T, 1.0, L.ptr(db), 1 if accumulate else 0,
                                     L.stream()), "bias_grad")


def lrelu_bwd(dy, y):
    dx = torch.empty_like(y)
    L.check(_lib().mst_lrelu_bwd_f32(L.ptr(dy), L.ptr(y), y.numel(), SLOPE, L.ptr(dx), L.stream()),
            "lrelu_bwd")
    return dx


def relu_gate_bwd(d, h, scale):
    out = torch.empty_like(h)
    L.check(_lib().mst_relu_gate_bwd_f32(L.ptr(d), L.ptr(h), h.numel(), scale, L.ptr(out),
                                         L.stream()), "relu_gate_bwd")
    return out


def _loss(fn, pred, target):
    lib = _lib()
    n = pred.numel()
    ws, _ = workspace(lib.mst_l1_workspace_size(n) + 8, pred.device)
    loss = torch.empty((), device=pred.device, dtype=torch.float32)
    L.check(getattr(lib, fn)(L.ptr(pred), L.ptr(target), n, L.ptr(loss), L.ptr(ws), L.stream()), fn)
    return loss


def l1_fwd(pred, target):
    return _loss("mst_l1_fwd_f32", pred, target)


def mse_fwd(pred, target):
    return _loss("mst_mse_fwd_f32", pred, target)


def l1_bwd(pred, target, gscale):
    dx = torch.empty_like(pred)
    L.check(_lib().mst_l1_bwd_f32(L.ptr(pred), L.ptr(target), pred.numel(), L.ptr(gscale), L.ptr(dx),
                                  L.stream()), "l1_bwd")
    return dx


def adam(p, g, m, v, lr_step, b1, b2, eps, bc2_sqrt, max_blocks=None):
    """torch.optim.Adam's update (mst_adam_f32). 1 - b1 and 1 - b2 are formed in double here and
    rounded, as torch forms them; max_blocks caps the grid (a background launch)."""
    args = (L.ptr(p), L.ptr(g), L.ptr(m), L.ptr(v), p.numel(), lr_step, b2, 1.0 - b1, 1.0 - b2, eps,
            bc2_sqrt)
    if max_blocks is None:
        L.check(_lib().mst_adam_f32(*args, L.stream()), "adam")
    else:
        L.check(_lib().mst_adam_ex_f32(*args, max_blocks, L.stream()), "adam")


def adam_dev(p, g, m, v, hyper, b1, b2, eps):
    """adam() with (lr_step, bc2_sqrt) read from the 2-float device tensor `hyper`."""
    assert hyper.dtype == torch.float32 and hyper.numel() >= 2 and hyper.is_cuda
    L.check(_lib().mst_adam_dev_f32(L.ptr(p), L.ptr(g), L.ptr(m), L.ptr(v), p.numel(), L.ptr(hyper),
                                    b2, 1.0 - b1, 1.0 - b2, eps, L.stream()), "adam_dev")


# ------------------------------------------- gradient norm, clipping, clipped Adam
def memory_order(t):
    """Dimension permutation that lists t's dims from the largest stride to the smallest: for a
    dense tensor, t.permute(perm) is contiguous (a tap-major slot view (d0, d1, k) of (d0, k, d1)
    memory gives perm (0, 2, 1))."""
    return sorted(range(t.dim()), key=lambda d: (-t.stride(d), d))


def _is_dense(t):
    return t.is_contiguous() or t.permute(memory_order(t)).is_contiguous()


def check_max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number >= 0, got {max_norm}")
    return max_norm


def _address(a):
    return a.buffer_info()[0]


class GradTable:
    """Gradients as the host arrays that mst_grad_norm and mst_grad_scale take (addresses, sizes,
    element types). A gradient with gaps between its elements goes in as a dense copy, which is
    copied back after a change."""

    def __init__(self, ts, what, writes=False):
        # one property of all tensors at a time: a list of hundreds is bound by these loops
        self.device = dev = ts[0].device
        types = [L.TYPES.get(t.dtype) for t in ts]
        if None in types or {t.layout for t in ts} != {torch.strided}:
            bad = next(t for t in ts if t.dtype not in L.TYPES or t.layout != torch.strided)
            raise TypeError(f"{what}: dense float32, bfloat16 or float16 gradients, got {bad.dtype} "
                            f"({bad.layout})")
        if not dev.type == "cuda":
            raise RuntimeError(f"{what}: CUDA (HIP) tensors only; there is no CPU path")
        if {t.get_device() for t in ts} != {dev.index}:
            raise ValueError(f"{what}: gradients on one device, got {sorted({str(t.device) for t in ts})}")
        self.tensors, self.count, self.copies = ts, len(ts), []
        if not all([t.is_contiguous() for t in ts]):
            ts = [t if _is_dense(t) else self._copy(t, what, writes) for t in ts]
        self.arrays = (array("Q", [t.data_ptr() for t in ts]), array("q", [t.numel() for t in ts]),
                       array("i", types))

    def _copy(self, t, what, writes):
        if writes and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise ValueError(f"{what}: an expanded gradient holds several elements in one place; clone it "
                             "first")
        d = t.contiguous()
        self.copies.append((t, d))
        return d

    def args(self):
        return (*(_address(a) for a in self.arrays), self.count)

    def norm(self, out=None):
        dev, lib = self.device, _lib()
        norm = torch.empty((), device=dev, dtype=torch.float32) if out is None else out
        ws, nb = workspace(lib.mst_grad_norm_workspace_size(self.count), dev)
        L.check(lib.mst_grad_norm(*self.args(), L.ptr(norm), L.ptr(ws), nb, L.stream()), "grad_norm")
        return norm

    def scale(self, norm, max_norm):
        L.check(_lib().mst_grad_scale(*self.args(), L.ptr(norm), max_norm, L.stream()),
                "clip_grad_norm_ (gradients that share memory?)")
        torch.autograd.graph.increment_version(self.tensors)
        for t, d in self.copies:
            t.copy_(d)


def grad_norm(ts, out=None):
    """L2 norm over every element of the tensors (0-d float32 on their device; sums in double, in
    an order that depends on the sizes alone), written to `out` if given."""
    table = GradTable(ts, "grad_norm")
    with L.device_of(table.device):
        return table.norm(out)


def clip_grad_norm_(ts, max_norm, check=None):
    """g *= min(1, max_norm / (norm + 1e-6)) for every tensor, in place; returns the norm before.
    check(norm), if given, runs before anything is changed."""
    table = GradTable(ts, "clip_grad_norm_", writes=True)
    with L.device_of(table.device):
        norm = table.norm()
        if check is not None:
            check(norm)
        table.scale(norm, max_norm)
    return norm


def adam_clip(ps, gs, ms, vs, norm, max_norm, lr_step, b1, b2, eps, bc2_sqrt, hyper=None):
    """adam() over lists of float32 tensors, gradients taken times min(1, max_norm / (norm + 1e-6));
    hyper as in adam_dev(). The four tensors of an entry are dense, in one element order."""
    n = len(ps)
    if not len(gs) == len(ms) == len(vs) == n:
        raise ValueError("adam_clip: as many gradients and moments as parameters")
    if n == 0:
        return
    assert hyper is None or (hyper.dtype == torch.float32 and hyper.numel() >= 2 and hyper.is_cuda)
    dev = ps[0].device
    numel = [t.numel() for t in ps]
    for ts in (ps, gs, ms, vs):
        if {t.dtype for t in ts} != {torch.float32} or dev.type != "cuda" or \
                {t.get_device() for t in ts} != {dev.index}:
            raise TypeError("adam_clip: float32 CUDA tensors on one device, got "
                            f"{sorted({f'{t.dtype} on {t.device}' for t in ts})}")
        if [t.numel() for t in ts] != numel:
            raise ValueError("adam_clip: sizes differ")
    with L.device_of(dev):
        arrays = [array("Q", [t.data_ptr() for t in ts]) for ts in (ps, gs, ms, vs)] + [array("q", numel)]
        L.check(_lib().mst_adam_clip_f32(*(_address(a) for a in arrays), n, L.ptr(norm), max_norm, lr_step,
                                         b2, 1.0 - b1, 1.0 - b2, eps, bc2_sqrt, L.ptr(hyper), L.stream()),
                "adam_clip (parameters or moments that share memory?)")


# ---------------------------------------------------------- gated linear recurrence
GATED_TILE = 512  # frames between two kept states (gated.hip)


def gated_tiles(dtype, T):
    """States that the backward needs of a row of T frames (mst_gated_tiles): none in one tile, of
    512 frames in float32 and up to 1024 in 16 bits."""
    one = GATED_TILE if dtype == torch.float32 else 2 * GATED_TILE
    return (T + GATED_TILE - 1) // GATED_TILE if T > one else 0


def refuse_tangents(what, *ts):
    """The recurrence has no forward-mode derivative: a tensor that carries a tangent (a dual tensor,
    torch.func.jvp) is refused, where the kernels would drop the tangent without a word."""
    if in_forward_mode() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError(f"{what}: no forward-mode derivative (reverse mode only)")


def in_forward_mode():
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()


def gated_check(x, gate, h0, lengths):
    """Shapes and types of the recurrence's arguments (real and fake tensors alike)."""
    if x.dim() != 3 or gate.shape != x.shape:
        raise ValueError(f"gated_recurrence: x and gate of one shape (B, C, T), got {tuple(x.shape)} "
                         f"and {tuple(gate.shape)}")
    if x.dtype not in L.TYPES or gate.dtype != x.dtype:
        raise TypeError("gated_recurrence: x and gate both float32, bfloat16 or float16, got "
                        f"{x.dtype} and {gate.dtype}")
    B, C, T = x.shape
    if h0 is not None:
        if tuple(h0.shape) != (B, C):
            raise ValueError(f"gated_recurrence: h0 must be ({B}, {C}), got {tuple(h0.shape)}")
        if h0.dtype not in L.TYPES:
            raise TypeError(f"gated_recurrence: floating h0, got {h0.dtype}")
    if lengths is not None:
        if tuple(lengths.shape) != (B,):
            raise ValueError(f"gated_recurrence: lengths must be ({B},), got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"gated_recurrence: int32 or int64 lengths, got {lengths.dtype}")
    for t in (gate, h0, lengths):
        if t is not None and t.device != x.device:
            raise ValueError(f"gated_recurrence: tensors on one device, got {x.device} and {t.device}")


def gated_bwd_check(gh, glast, x, gate, h0, lengths, carry):
    gated_check(x, gate, h0, lengths)
    B, C, T = x.shape
    want = (B, C, gated_tiles(x.dtype, T))
    if tuple(carry.shape) != want or carry.dtype != torch.float32 or not carry.is_contiguous():
        raise ValueError(f"gated_recurrence_backward: carry must be the forward's, {want} float32, got "
                         f"{tuple(carry.shape)} {carry.dtype}")
    for t, shape in ((gh, (B, C, T)), (glast, (B, C))):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"gated_recurrence_backward: a gradient of {shape}, got {tuple(t.shape)}")
    for t in (gh, glast, carry):
        if t is not None and t.device != x.device:
            raise ValueError("gated_recurrence_backward: tensors on one device")


def _unit_time(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _gated_inputs(x, gate, h0, lengths):
    if not x.is_cuda:
        raise RuntimeError("gated_recurrence: CUDA (HIP) tensors only; there is no CPU path")
    if lengths is not None:
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, x.shape[2]).to(torch.int32)
        lengths = lengths.contiguous()
    return _unit_time(x), _unit_time(gate), h0.float().contiguous() if h0 is not None else None, lengths


def _gated_workspace(x, carry):
    if carry.numel() == 0:  # rows of one tile need none
        return None, 0
    return workspace(_lib().mst_gated_workspace_size(L.TYPES[x.dtype], *x.shape), x.device)


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def gated_fwd(x, gate, h0, lengths, reverse):
    """(h, last, carry) of mst_gated_fwd; carry (B, C, gated_tiles(x.dtype, T)) goes to gated_bwd."""
    gated_check(x, gate, h0, lengths)
    x, gate, h0, lengths = _gated_inputs(x, gate, h0, lengths)
    B, C, T = x.shape
    dev = x.device
    h = torch.empty(B, C, T, device=dev, dtype=x.dtype)
    carry = torch.empty(B, C, gated_tiles(x.dtype, T), device=dev, dtype=torch.float32)
    if h.numel() == 0:  # no frame: the state stays
        return h, h0.clone() if h0 is not None else torch.zeros(B, C, device=dev), carry
    last = torch.empty(B, C, device=dev, dtype=torch.float32)
    with L.device_of(dev):
        ws, nb = _gated_workspace(x, carry)
        L.check(_lib().mst_gated_fwd(L.TYPES[x.dtype], _p(x), x.stride(0), x.stride(1), _p(gate),
                                     gate.stride(0), gate.stride(1), _p(h0), _p(lengths), B, C, T,
                                     1 if reverse else 0, _p(h), _p(last), _p(carry), _p(ws), nb,
                                     L.stream()),
                "gated_recurrence")
    return h, last, carry


def gated_bwd(gh, glast, x, gate, h0, lengths, carry, reverse, need_dh0=True):
    """(dx, dgate, dh0) of mst_gated_bwd; gh and glast may be None (zeros), dh0 is None if not needed."""
    gated_bwd_check(gh, glast, x, gate, h0, lengths, carry)
    x, gate, h0, lengths = _gated_inputs(x, gate, h0, lengths)
    B, C, T = x.shape
    dev = x.device
    dx = torch.empty(B, C, T, device=dev, dtype=x.dtype)
    dgate = torch.empty(B, C, T, device=dev, dtype=x.dtype)
    gh = gh.to(x.dtype).contiguous() if gh is not None else None
    glast = glast.float().contiguous() if glast is not None else None
    if dx.numel() == 0:
        return dx, dgate, glast.clone() if glast is not None else torch.zeros(B, C, device=dev)
    dh0 = torch.empty(B, C, device=dev, dtype=torch.float32) if need_dh0 else None
    with L.device_of(dev):
        ws, nb = _gated_workspace(x, carry)
        L.check(_lib().mst_gated_bwd(L.TYPES[x.dtype], _p(x), x.stride(0), x.stride(1), _p(gate),
                                     gate.stride(0), gate.stride(1), _p(h0), _p(lengths), _p(carry),
                                     _p(gh), _p(glast), B, C, T, 1 if reverse else 0, _p(dx),
                                     _p(dgate), _p(dh0), _p(ws), nb, L.stream()),
                "gated_recurrence_backward")
    return dx, dgate, dh0


def gated_step_check(x, gate, state):
    if x.dim() != 2 or gate.shape != x.shape or state.shape != x.shape:
        raise ValueError("gated_recurrence_step: x, gate and state of one shape (B, C), got "
                         f"{tuple(x.shape)}, {tuple(gate.shape)} and {tuple(state.shape)}")
    if x.dtype not in L.TYPES or gate.dtype != x.dtype:
        raise TypeError("gated_recurrence_step: x and gate both float32, bfloat16 or float16, got "
                        f"{x.dtype} and {gate.dtype}")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise TypeError("gated_recurrence_step: a contiguous float32 state (it is updated in place)")
    if gate.device != x.device or state.device != x.device:
        raise ValueError("gated_recurrence_step: tensors on one device")


def gated_step(x, gate, state):
    """One frame: state (B, C) updated in place, its new values returned in x's type."""
    gated_step_check(x, gate, state)
    if not x.is_cuda:
        raise RuntimeError("gated_recurrence_step: CUDA (HIP) tensors only; there is no CPU path")
    x, gate = _unit_time(x), _unit_time(gate)
    B, C = x.shape
    h = torch.empty(B, C, device=x.device, dtype=x.dtype)
    if h.numel():
        with L.device_of(x.device):
            L.check(_lib().mst_gated_step(L.TYPES[x.dtype], _p(x), x.stride(0), _p(gate),
                                          gate.stride(0), B, C, _p(state), _p(h), L.stream()),
                    "gated_recurrence_step (x or gate in the state's memory?)")
        torch.autograd.graph.increment_version(state)
    return h


def scale_(x, s):
    L.check(_lib().mst_scale_f32(L.ptr(x), x.numel(), s, L.stream()), "scale")


def fill_(x, v):
    L.check(_lib().mst_fill_f32(L.ptr(x), x.numel(), v, L.stream()), "fill")
