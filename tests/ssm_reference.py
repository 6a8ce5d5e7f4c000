"""The state-space operators by their definition, step by step in float64 on the CPU, with hand-written gradients, and bounds
on what float32 arithmetic may be off.

Bounds.  Let eps = 2^-24, half a step of float32.  One step of the recurrence multiplies the state by exp(dt A), computed
as exp2 of a product: two roundings of the exponent x = dt A / ln 2 and about ten half steps of dt itself (softplus: an exp2,
a reciprocal, a series, a sum), so relatively 12 |dt A| eps from the exponent, 2 eps from exp2 and 1 eps from the
multiply-add.  A contribution that is k steps old therefore carries at most (3 k + 12 k x e^{-k x}) eps <= (3 k + 5) eps of
its size at that time, T steps at most.  The input and output products, the two or three sigmoids of a gate (each about
20 half steps at |v| <= 8) and the sum over the states stay below 64 eps.  Errors are relative to the sum of the ABSOLUTE
values of all contributions, which `absolute=True` returns.  Gradients pass through the forward states and through the same
recurrence backwards: twice the forward bound, plus one eps for each term of a sum over steps, sequences or channels that is
not already below (blocks of 16 steps are summed first).  `bound` uses (8 T + B + D / 16 + 64) eps for all of them, and half
a step of the output's type on top, relative to the value.
"""
import math

import torch

EPS = 2.0 ** -24


def silu(v):
    return v * torch.sigmoid(v)


def silu_slope(v, absolute=False):
    """sigmoid(v) (1 + v (1 - sigmoid(v))).  Its two terms cancel near v = -1.28, so the size that rounding errors go by is
    the sum of their absolute values."""
    s = torch.sigmoid(v)
    return s * (1 + (v.abs() if absolute else v) * (1 - s))


def conv(x, weight, bias=None, act=True, initial=None, lengths=None, dy=None, dfinal=None, absolute=False):
    """(y, state, gradients): gradients None without dy / dfinal, else a dict by name."""
    B, T, D = x.shape
    K = weight.shape[1]
    mag = torch.abs if absolute else (lambda v: v)
    x, weight = x.double(), weight.double()
    bias = torch.zeros(D, dtype=torch.float64) if bias is None else bias.double()
    initial = torch.zeros(B, K - 1, D, dtype=torch.float64) if initial is None else initial.double()
    lengths = [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]
    y, state = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, K - 1, D, dtype=torch.float64)
    grads = None
    if dy is not None or dfinal is not None:
        grads = dict(x=torch.zeros(B, T, D, dtype=torch.float64), weight=torch.zeros(D, K, dtype=torch.float64),
                     bias=torch.zeros(D, dtype=torch.float64), initial=torch.zeros(B, K - 1, D, dtype=torch.float64))
    for b, n in enumerate(lengths):
        ext = torch.cat([initial[b], x[b, :n]])
        pre = bias.repeat(n, 1)
        size = mag(bias).repeat(n, 1)
        for k in range(K):
            pre = pre + ext[k:k + n] * weight[:, k]
            size = size + mag(ext[k:k + n] * weight[:, k])
        if absolute:     # |d act / d pre| <= 1.1
            y[b, :n] = size * 1.1 if act else size
        else:
            y[b, :n] = silu(pre) if act else pre
        state[b] = ext[n:n + K - 1]
        if grads is None:
            continue
        g = torch.zeros(n, D, dtype=torch.float64) if dy is None else dy[b, :n].double()
        if act:
            # the slope moves with the pre-activation by at most half its error
            g = mag(g) * (silu_slope(pre, True) + size) if absolute else g * silu_slope(pre)
        g = mag(g)
        dext = torch.zeros(n + K - 1, D, dtype=torch.float64)
        for k in range(K):
            dext[k:k + n] += mag(g * weight[:, k])
            grads["weight"][:, k] += mag(g * ext[k:k + n]).sum(0)
        if dfinal is not None:
            dext[n:n + K - 1] += mag(dfinal[b].double())
        grads["bias"] += g.sum(0)
        grads["x"][b, :n] = dext[K - 1:]
        grads["initial"][b] = dext[:K - 1]
    return y, state, grads


def scan(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, softplus=True, initial=None, lengths=None, dy=None, dfinal=None,
         absolute=False):
    """(y, state, gradients) as above."""
    mag = torch.abs if absolute else (lambda v: v)
    Bn, T, Dn = u.shape
    G, N = Bm.shape[2:]
    f64 = lambda v, *shape: torch.zeros(*shape, dtype=torch.float64) if v is None else v.double()  # noqa: E731
    u, A, raw = u.double(), A.double(), delta.double() + f64(delta_bias, Dn)
    D_, lens = f64(D, Dn), torch.tensor([T] * Bn if lengths is None else [min(max(int(n), 0), T) for n in lengths])
    dt = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    on = torch.arange(T)[None, :] < lens[:, None]
    zero = torch.zeros((), dtype=torch.float64)
    u, dt = torch.where(on[..., None], u, zero), torch.where(on[..., None], dt, zero)
    wide = lambda m: torch.where(on[..., None, None], m.double(), zero).repeat_interleave(Dn // G, 2)  # noqa: E731
    Bw, Cw = wide(Bm), wide(Cm)
    gate = torch.ones_like(u) if z is None else silu(torch.where(on[..., None], z.double(), zero))
    decay = torch.exp(dt[..., None] * A)
    decay = torch.where(on[..., None, None], decay, torch.ones((), dtype=torch.float64))
    h = mag(f64(initial, Bn, Dn, N))
    states, out = [h], torch.zeros_like(u)
    for t in range(T):
        h = decay[:, t] * h + mag((dt[:, t] * u[:, t])[..., None] * Bw[:, t])
        states.append(h)
        out[:, t] = mag(Cw[:, t] * h).sum(-1) + mag(D_ * u[:, t])
    y = mag(out * gate)
    if dy is None and dfinal is None:
        return y, h, None
    dout = torch.zeros_like(u) if dy is None else torch.where(on[..., None], dy.double(), zero)
    grads = {}
    if z is not None:
        zz = torch.where(on[..., None], z.double(), zero)
        grads["z"] = mag(dout * out * silu_slope(zz, absolute))
    d = mag(dout * gate)
    if absolute and softplus:
        slope = torch.sigmoid(raw)
    else:
        slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    dB, dC = torch.zeros(Bn, T, G, N, dtype=torch.float64), torch.zeros(Bn, T, G, N, dtype=torch.float64)
    dA = torch.zeros_like(A)
    g = mag(f64(dfinal, Bn, Dn, N))
    share = lambda m: m.view(Bn, G, Dn // G, N).sum(2)  # noqa: E731
    for t in reversed(range(T)):
        live = on[:, t, None, None]
        gt = torch.where(live, g + mag(d[:, t, :, None] * Cw[:, t]), zero)
        dC[:, t] = share(mag(d[:, t, :, None] * states[t + 1]) * live)
        dB[:, t] = share(mag(gt * (dt[:, t] * u[:, t])[..., None]))
        gB = mag(gt * Bw[:, t]).sum(-1)
        du[:, t] = mag(gB * dt[:, t]) + mag(D_ * d[:, t])
        w = gt * decay[:, t] * states[t]
        ddt[:, t] = mag(gB * u[:, t]) + mag(w * A).sum(-1)
        dA += mag(w * dt[:, t, :, None]).sum(0)
        g = torch.where(live, gt * decay[:, t], g)
    ddelta = torch.where(on[..., None], ddt * slope, zero)
    grads |= dict(u=du, delta=ddelta, A=dA, B=dB, C=dC, D=mag(d * u).sum((0, 1)), delta_bias=mag(ddelta).sum((0, 1)), initial=g)
    return y, h, grads


def bound(ref, size, dtype, T, B=1, D=1):
    """Allowed distance from `ref`, element by element; `size`: the same with absolute=True."""
    half = 0.0 if dtype in (torch.float32, torch.float64) else torch.finfo(dtype).eps / 2
    tiny = 0.0 if half == 0.0 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return (8 * T + B + D / 16 + 64) * EPS * (size.abs() + 2.0 ** -100) * (1 + half) + half * ref.abs() + tiny


def close(got, ref, size, T, B=1, D=1, what=""):
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    off = (got.detach().cpu().double() - ref).abs()
    allowed = bound(ref, size, got.dtype, T, B, D)
    bad = ~(off <= allowed)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / allowed).nan_to_num(math.inf).max()):.3g} "
                           f"times the bound, first at {bad.nonzero()[0].tolist()}")
