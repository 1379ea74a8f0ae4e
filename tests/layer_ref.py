"""Plain restatements of the gated delta rule, layer norm and dropout in 64 bits, on the CPU, the first one row after another.

They also say how large what is added up on the way is (``sizes``): what bounds on rounding errors are multiples of."""
import math

import torch

import philox_ref


def unit(x, epsilon):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + epsilon)


def delta(q, k, v, g, beta, scale, normalise=True, epsilon=1e-6, initial=None, dout=None, dfinal=None):
    """One sequence: q, k [rows, key heads, keys], v [rows, heads, values], g, beta [rows, heads], initial [heads, keys, values].
    (out, final, sizes), or with `dout` also the gradients: (dict of gradients, dict of sizes)."""
    rows, heads, values = v.shape
    keys, group = q.shape[2], heads // q.shape[1]
    raw = {"q": q.double(), "k": k.double()}
    hat = {n: (unit(x, epsilon) if normalise else x).repeat_interleave(group, 1) for n, x in raw.items()}
    v, g, beta = v.double(), g.double(), beta.double()
    s = torch.zeros(heads, keys, values, dtype=torch.float64) if initial is None else initial.double()
    states, errors, out = [s], [], torch.zeros(rows, heads, values, dtype=torch.float64)
    for t in range(rows):
        s = torch.exp(g[t])[:, None, None] * s
        w = v[t] - torch.einsum("hkv,hk->hv", s, hat["k"][t])
        s = s + torch.einsum("hk,hv->hkv", hat["k"][t], beta[t][:, None] * w)
        out[t] = scale * torch.einsum("hkv,hk->hv", s, hat["q"][t])
        states.append(s)
        errors.append(w)
    column = torch.stack(states).norm(dim=2).amax(0) + (v.abs().amax(0) if rows else 0.0)        # [heads, values]: of a state's column, or a value
    queries = hat["q"].norm(dim=-1).amax(0) if rows else torch.zeros(heads, dtype=torch.float64)
    lengths = hat["k"].norm(dim=-1).amax(0) if rows else torch.ones(heads, dtype=torch.float64)
    if dout is None:
        return out, s, dict(out=scale * queries[:, None] * column, final=(column * lengths[:, None].clamp(min=1.0))[:, None, :].expand_as(s))
    dout = dout.double()
    ds = torch.zeros_like(s) if dfinal is None else dfinal.double()
    dq, dk, dv, dg, dbeta = (torch.zeros_like(x) for x in (hat["q"], hat["k"], v, g, beta))
    behind, dr = [ds], torch.zeros_like(v)
    for t in reversed(range(rows)):
        a = torch.exp(g[t])[:, None, None]
        dq[t] = scale * torch.einsum("hkv,hv->hk", states[t + 1], dout[t])
        ds = ds + scale * torch.einsum("hk,hv->hkv", hat["q"][t], dout[t])
        behind.append(ds)
        dr[t] = torch.einsum("hkv,hk->hv", ds, hat["k"][t])
        dbeta[t] = (dr[t] * errors[t]).sum(-1)
        dv[t] = beta[t][:, None] * dr[t]
        dk[t] = torch.einsum("hkv,hv->hk", ds, beta[t][:, None] * errors[t]) - torch.einsum("hkv,hv->hk", a * states[t], dv[t])
        ds = ds - torch.einsum("hk,hv->hkv", hat["k"][t], dv[t])
        dg[t] = (ds * a * states[t]).sum((1, 2))
        ds = a * ds
    behind.append(ds)
    # the largest of states, errors and their gradients, by head
    state, dstate = torch.stack(states).norm(dim=(2, 3)).amax(0), torch.stack(behind).norm(dim=(2, 3)).amax(0)
    error = torch.stack(errors).norm(dim=-1).amax(0) if rows else torch.zeros(heads, dtype=torch.float64)
    most = lambda x: x.amax(0) if rows else torch.zeros(heads, dtype=torch.float64)  # noqa: E731
    step, give, beta, value = most(dr.norm(dim=-1)), scale * most(dout.norm(dim=-1)), most(beta.abs()), most(v.norm(dim=-1))
    size = dict(dv=beta * (torch.stack(behind).norm(dim=2).amax(0).amax(-1) * lengths + give * queries), dbeta=error * step,
                dq=give * (state + error), dk=beta * (dstate * error + step * state + error * step) + give * queries * error * beta,
                dinitial=dstate * lengths.clamp(min=1.0) + give * queries, dg=state * dstate + give * queries * (state + error) + beta * step * (value + error))
    found = dict(dv=dv, dg=dg, dbeta=dbeta, dinitial=ds)
    for name, grad in (("q", dq), ("k", dk)):
        grad, large = grad.view(rows, heads // group, group, keys).sum(2), size["d" + name].view(-1, group).sum(1)
        if normalise:
            length = torch.sqrt((raw[name] ** 2).sum(-1, keepdim=True) + epsilon)
            unitary = raw[name] / length
            grad = (grad - unitary * (unitary * grad).sum(-1, keepdim=True)) / length
            large = large[None, :, None] / length
        else:
            large = large[None, :, None].expand(rows, -1, 1)
        found["d" + name], size["d" + name] = grad, large.expand_as(grad)
    size.update(dv=size["dv"][None, :, None].expand_as(dv), dbeta=size["dbeta"][None].expand_as(dbeta), dg=size["dg"][None].expand_as(dg),
                dinitial=size["dinitial"][:, None, None].expand_as(ds))
    return found, size


def layer_norm(x, weight=None, bias=None, gate=None, epsilon=1e-5, rms=False, dout=None):
    """x, gate [rows, channels].  (out, sizes), or with `dout` (dict of gradients, dict of sizes)."""
    x = x.double()
    mean = 0.0 if rms else x.mean(-1, keepdim=True)
    length = torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + epsilon)
    hat = (x - mean) / length
    # x - mean is off by roundings of x and of the mean's sum, of x' the length's too
    off = (x.abs() + (0.0 if rms else x.abs().mean(-1, keepdim=True))) / length + hat.abs()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    z = None if gate is None else gate.double()
    sig = None if z is None else torch.sigmoid(z)
    s = 1.0 if z is None else z * sig
    y, ysize = hat * w + b, off * w.abs() + b.abs()
    if dout is None:
        return y * s, ysize * (1.0 if z is None else s.abs())
    d = dout.double()
    found, size = {}, {}
    if z is not None:
        slope, slopes = sig * (1 + z * (1 - sig)), sig * (1 + z.abs() * (1 - sig))
        found["dgate"], size["dgate"] = d * y * slope, d.abs() * ysize * slopes
    d = d * s
    found["dweight"], size["dweight"] = (d * hat).sum(0), (d.abs() * off).sum(0)
    found["dbias"], size["dbias"] = d.sum(0), d.abs().sum(0)
    v = d * w
    along, alongsize = (v * hat).mean(-1, keepdim=True), (v.abs() * off).mean(-1, keepdim=True)
    found["dx"] = (v - (0.0 if rms else v.mean(-1, keepdim=True)) - hat * along) / length
    size["dx"] = (v.abs() + (0.0 if rms else v.abs().mean(-1, keepdim=True)) + off * alongsize) / length
    return found, size


def kept(rows, channels, probability, seed, call):
    """Which elements dropout keeps, [rows, channels], and what they are multiplied with."""
    import numpy as np
    groups = -(-channels // 8)
    n = np.arange(rows * groups, dtype=np.uint64)
    low = np.uint64(0xffffffff)
    same = np.ones_like(n)
    words = philox_ref.philox4x32(n & low, n >> np.uint64(32), same * np.uint64(call & 0xffffffff), same * np.uint64(call >> 32), seed & 0xffffffff, seed >> 32)
    halves = np.stack([np.asarray(part, dtype=np.int64) for w in words for part in (np.asarray(w, dtype=np.uint64) & np.uint64(0xffff), np.asarray(w, dtype=np.uint64) >> np.uint64(16))], -1)
    dropped = math.floor(probability * 65536 + 0.5)
    return torch.from_numpy(halves.reshape(rows, groups * 8)[:, :channels] >= dropped), 65536 / (65536 - dropped) if dropped < 65536 else 0.0
