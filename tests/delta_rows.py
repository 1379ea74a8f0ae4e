"""How large what is added up for each row's gradients of the gated delta rule is, from norms of that row's own operands, in 64 bits.

Rows forget: what a row of a decay a[t] = exp(g[t]) has of the rows before it is a[t] times that.  With unit keys and 0 <= beta <= 1 no row's transition makes an error
longer, so that the error of the state behind row t is at most what the rows up to it left of their own ("held"), and that of the state's gradient in front of the decay what those from it on did
("behind"):
  held[t] = a[t] held[t-1] + beta |k| (|v[t]| + a[t] |S[t-1]|),   behind[t] = scale |q| |dout[t]| + a[t+1] asked[t+1],   asked[t] = behind[t] + beta |k|^2 |dS[t]|
with S and dS as they are, lengths of matrices by the root of their squares.  A gradient is a product of a sum of the one kind and a sum of the other; a gate's carries a[t] itself."""
import torch

import layer_ref as ref


def sizes(q, k, v, g, beta, scale, normalise=True, epsilon=1e-6, initial=None, dout=None, dfinal=None):
    """Of arrays as ref.delta takes them: per row and head (q, k: and key head), the length of the vector that holds its gradient is off by a few units of fp32 of these."""
    rows, heads, values = v.shape
    keys, group = q.shape[2], heads // q.shape[1]
    raw = {"q": q.double(), "k": k.double()}
    hat = {n: (ref.unit(x, epsilon) if normalise else x).repeat_interleave(group, 1) for n, x in raw.items()}
    v, a, beta, dout = v.double(), torch.exp(g.double()), beta.double(), dout.double()
    s = torch.zeros(heads, keys, values, dtype=torch.float64) if initial is None else initial.double()
    length = lambda x: x.norm(dim=(1, 2))  # noqa: E731
    lq, lk, lv, lo = hat["q"].norm(dim=-1), hat["k"].norm(dim=-1), v.norm(dim=-1), dout.norm(dim=-1)
    held, front, state = [length(s)], [length(s)], s
    for t in range(rows):
        state = a[t][:, None, None] * state
        held.append(a[t] * held[-1] + beta[t] * lk[t] * (lv[t] + a[t] * front[-1] * lk[t]))
        w = v[t] - torch.einsum("hkv,hk->hv", state, hat["k"][t])
        state = state + torch.einsum("hk,hv->hkv", hat["k"][t], beta[t][:, None] * w)
        front.append(length(state))
    ds = torch.zeros_like(s) if dfinal is None else dfinal.double()
    ahead = length(ds)
    size = {n: torch.zeros(rows, heads, dtype=torch.float64) for n in ("q", "k", "v", "g", "beta")}
    for t in reversed(range(rows)):
        ds = ds + scale * torch.einsum("hk,hv->hkv", hat["q"][t], dout[t])
        behind = scale * lq[t] * lo[t] + ahead
        asked = behind + beta[t] * lk[t] ** 2 * length(ds)
        error = lv[t] + a[t] * held[t] * lk[t]
        size["q"][t] = scale * lo[t] * held[t + 1]
        size["k"][t] = beta[t] * (error * behind + a[t] * held[t] * lk[t] * behind)
        size["v"][t] = beta[t] * lk[t] * behind
        size["beta"][t] = error * lk[t] * behind
        size["g"][t] = a[t] * held[t] * asked
        dv = beta[t][:, None] * torch.einsum("hkv,hk->hv", ds, hat["k"][t])
        ds = a[t][:, None, None] * (ds - torch.einsum("hk,hv->hkv", hat["k"][t], dv))
        ahead = a[t] * asked
    size["initial"] = ahead
    for n, x in raw.items():
        size[n] = size[n].view(rows, heads // group, group).sum(2)
        if normalise:
            size[n] = size[n] / torch.sqrt((x ** 2).sum(-1) + epsilon)
    return size
