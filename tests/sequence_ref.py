"""Plain restatements of the operators on sequences and of the optimiser step in 64 bits, one row after another, on the CPU.

With ``magnitudes`` the same formulas run on absolute values, every term added: what bounds on rounding errors are multiples of."""
import torch


def causal_conv(x, weight, bias, silu, initial=None, dout=None, dfinal=None, magnitudes=False):
    """One sequence: x [rows, channels], weight [channels, taps], initial [taps - 1, channels].  (out, final) or, with `dout`, the gradients
    (dx, dweight, dbias, dinitial)."""
    a = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    n, K = x.shape[0], weight.shape[1]
    ext = torch.cat([torch.zeros(K - 1, x.shape[1], dtype=torch.float64) if initial is None else initial.double(), x.double()])
    bias = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias.double()
    w = weight.double()
    s = bias + sum(ext[k:k + n] * w[:, k] for k in range(K))
    sig = torch.sigmoid(s)
    size = bias.abs() + sum((ext[k:k + n] * w[:, k]).abs() for k in range(K))
    if dout is None:
        if magnitudes:
            return size, ext[n:].abs()
        return (s * sig if silu else s), ext[n:]
    slope = sig * (1 + s * (1 - sig)) if silu else torch.ones_like(s)
    if magnitudes and silu:
        # (the slope is a sum of two terms of either sign, and off by what s is off by times its own slope, which is below 1)
        slope = sig * (1 + s.abs() * (1 - sig)) + size
    ds = a(dout.double() * slope)
    dext = torch.zeros_like(ext)
    for k in range(K):
        dext[k:k + n] += a(ds * w[:, k])
    if dfinal is not None:
        dext[n:] += a(dfinal.double())
    dweight = torch.stack([a(ds * ext[k:k + n]).sum(0) for k in range(K)], 1)
    return dext[K - 1:], dweight, ds.sum(0), dext[:K - 1]


def scan(u, delta, A, B, C, D=None, delta_bias=None, z=None, softplus=False, initial=None, dout=None, dfinal=None, magnitudes=False):
    """One sequence: u, delta, z [rows, channels], B, C [rows, groups, states].  (out, final), or with `dout` a dict of gradients."""
    a = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    rows, channels = u.shape
    groups, states = B.shape[1], A.shape[1]
    A, B, C, u = A.double(), B.double().repeat_interleave(channels // groups, 1), C.double().repeat_interleave(channels // groups, 1), u.double()
    raw = delta.double() + (0 if delta_bias is None else delta_bias.double())
    dt = torch.nn.functional.softplus(raw, threshold=700) if softplus else raw
    skip = torch.zeros(channels, dtype=torch.float64) if D is None else D.double()
    h = torch.zeros(channels, states, dtype=torch.float64) if initial is None else a(initial.double())
    first, hs, ys = h, [], []
    for t in range(rows):
        h = torch.exp(dt[t, :, None] * A) * h + a((dt[t] * u[t])[:, None] * B[t])
        hs.append(h)
        ys.append(a(h * C[t]).sum(-1) + a(skip * u[t]))
    y = torch.stack(ys) if rows else torch.zeros(0, channels, dtype=torch.float64)
    gate = torch.ones_like(y) if z is None else z.double() * torch.sigmoid(z.double())
    if dout is None:
        return y * a(gate), h
    dout = dout.double()
    sig = torch.sigmoid(z.double()) if z is not None else None
    g = {"z": None if z is None else a(dout * (sig * (1 + a(z.double()) * (1 - sig)))) * y}
    gy = a(dout * gate)
    dh = torch.zeros(channels, states, dtype=torch.float64) if dfinal is None else a(dfinal.double())
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    dA, dB, dC = torch.zeros_like(A), torch.zeros(rows, groups, states, dtype=torch.float64), torch.zeros(rows, groups, states, dtype=torch.float64)
    for t in reversed(range(rows)):
        dh = dh + a(gy[t, :, None] * C[t])
        dC[t] = a(gy[t, :, None] * hs[t]).view(groups, -1, states).sum(1)
        dB[t] = a(dh * (dt[t] * u[t])[:, None]).view(groups, -1, states).sum(1)
        q = a(dh * B[t]).sum(-1)
        dh = dh * torch.exp(dt[t, :, None] * A)
        x = dh * (hs[t - 1] if t else first)
        dA += a(x * dt[t, :, None])
        du[t] = a(dt[t] * q) + a(skip * gy[t])
        ddt[t] = a(u[t] * q) + a(x * A).sum(-1)
    ddelta = ddt * torch.sigmoid(raw) if softplus else ddt
    g.update(u=du, delta=ddelta, A=dA, B=dB, C=dC, D=a(gy * u).sum(0), delta_bias=ddelta.sum(0), initial_state=dh)
    return g


_code = torch.arange(127)
E4M3 = torch.where(_code >= 8, torch.exp2((_code // 8 - 7).double()) * (1 + (_code % 8).double() / 8), (_code % 8).double() * 2.0 ** -9)


def e4m3_codes(r):
    """Number of the nearest value to each r >= 0, ties to the even code."""
    between = (E4M3[1:] + E4M3[:-1]) / 2
    low = torch.bucketize(r, between)                  # (a value on a border goes to the code below it, which is right if that is even)
    high = torch.bucketize(r, between, right=True)
    return torch.where(low % 2 == 0, low, high)


def adamw(w, g, m, v, step, rate, beta1, beta2, epsilon, decay):
    """New (weights, m, v) in 64 bits; `step` counts from 1."""
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    return w * (1 - rate * decay) - rate * (m / (1 - beta1 ** step)) / (torch.sqrt(v / (1 - beta2 ** step)) + epsilon), m, v
