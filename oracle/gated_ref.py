"""Gated linear recurrence in float64 on the CPU, frame by frame, with its gradients and with a bound
on what a float32 evaluation of the same formulas, in any order of composition, may be off.

  a_t = sigmoid(gate_t), c_t = 1 - a_t, h_t = a_t h_{t-1} + c_t x_t; frames t >= length are the identity

Error model, u = 2^-24 (half a float32 step): e = e^-|gate| within 3u + |gate| u / 20 (an exponential and its
correction, ln 2 in float32), 7.4u before it underflows; 1 + e one rounding, a quotient r within 2u (exact
where e < u), e r one rounding. r passes on at most half of e's error (|gate| near 0), so r is within 4.5u,
e r within 8.5u: a and c to 9u; c x to 10u. A state of magnitude M (the recurrence run on |x|, |h0|)
that passes a frame gains at most a's 9u and two roundings, 11u a M in all; the frame's own term its 10u
and the sum's rounding; composing maps in a tree rounds a term at most once a level, and a term has
passed at least as many frames as levels. With M_t = a_t M_{t-1} + c_t |x_t| both are within
  E_t = a_t (E_{t-1} + 8u M_{t-1}) + 12u c_t |x_t| + 4u M_t
and what is handed back, u_t = a_t (gh_t + u_{t+1}), is of the same form.
"""
import torch

U = 2.0 ** -24


def _order(T, reverse):
    return range(T - 1, -1, -1) if reverse else range(T)


def forward(x, gate, h0=None, lengths=None, reverse=False):
    """x, gate (B, C, T) of any type -> dict of float64 h (0 past the lengths), last, and the bounds
    h_err, last_err; a, c, states before each frame (prev), their magnitudes and bounds."""
    x, gate = x.double(), gate.double()
    B, C, T = x.shape
    s = torch.zeros(B, C, dtype=torch.float64) if h0 is None else h0.double()
    n = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    live = (torch.arange(T) < n[:, None])[:, None]
    a = torch.where(live, torch.sigmoid(gate), torch.ones(()).double())
    c = torch.where(live, torch.sigmoid(-gate), torch.zeros(()).double())
    x = torch.where(live, x, torch.zeros(()).double())
    h, h_err, prev = torch.zeros(B, C, T).double(), torch.zeros(B, C, T).double(), torch.zeros(B, C, T).double()
    prev_mag, prev_err = torch.zeros(B, C, T).double(), torch.zeros(B, C, T).double()
    M, E = s.abs(), torch.zeros(B, C).double()
    for t in _order(T, reverse):
        prev[..., t], prev_mag[..., t], prev_err[..., t] = s, M, E
        on = live[..., t]
        b = c[..., t] * x[..., t]
        s2 = a[..., t] * s + b
        M2 = a[..., t] * M + b.abs()
        E2 = a[..., t] * (E + 8 * U * M) + 12 * U * b.abs() + 4 * U * M2
        s, M, E = torch.where(on, s2, s), torch.where(on, M2, M), torch.where(on, E2, E)
        h[..., t] = torch.where(on, s, torch.zeros(()).double())
        h_err[..., t] = torch.where(on, E, torch.zeros(()).double())
    return dict(h=h, last=s, h_err=h_err, last_err=E, a=a, c=c, x=x, live=live, prev=prev,
                prev_mag=prev_mag, prev_err=prev_err)


def backward(f, gh, glast=None, reverse=False):
    """Gradients of sum(h gh) + sum(last glast) given forward()'s dict: dx, dgate, dh0 and bounds."""
    a, c, x, live = f["a"], f["c"], f["x"], f["live"]
    B, C, T = a.shape
    gh = torch.where(live, gh.double(), torch.zeros(()).double())
    u = torch.zeros(B, C).double() if glast is None else glast.double()
    M, E = u.abs(), torch.zeros(B, C).double()
    out = {k: torch.zeros(B, C, T).double() for k in ("dx", "dgate", "dx_err", "dgate_err")}
    for t in reversed(list(_order(T, reverse))):
        on = live[..., t]
        d = gh[..., t] + u
        dm = gh[..., t].abs() + M
        de = E + 2 * U * dm
        ct, at = c[..., t], a[..., t]
        diff = f["prev"][..., t] - x[..., t]
        mag = f["prev_mag"][..., t] + x[..., t].abs()
        out["dx"][..., t] = torch.where(on, ct * d, 0 * d)
        out["dx_err"][..., t] = torch.where(on, ct * (de + 8 * U * dm), 0 * d)
        out["dgate"][..., t] = torch.where(on, at * ct * d * diff, 0 * d)
        out["dgate_err"][..., t] = torch.where(
            on, at * ct * (de * mag + dm * f["prev_err"][..., t] + 20 * U * dm * mag), 0 * d)
        E = torch.where(on, at * (de + 10 * U * dm), E)
        u, M = torch.where(on, at * d, u), torch.where(on, at * dm, M)
    return dict(out, dh0=u, dh0_err=E)
