"""The gated delta rule through the C ABI against its restatement in 64 bits, one row after another.

Tolerances.  A result is one rounding to its type (half a step: eps / 2 of the value) of sums in fp32.  With unit keys and 0 <= beta <= 1 no row's
transition makes an error longer, so that what each row adds to it stays as it is at most.  On the way from an input to a result lie the keys of a
dot product, the rows of a chunk (64) twice (their dot products with one another, and the solution of a triangle of them) and once more for each row of the sequence; each
operation is off by at most half a step of fp32, of what is added up there (``sizes``: the largest lengths of states, errors and their gradients).  Such
errors are independent of each other and add up like their root: five standard deviations of sqrt(keys + 2 * 64 + rows) of them, and four operations for each (product, sum,
decay, length) as 4 x 2^-24 = 2^-22."""
import math

import numpy as np
import pytest
import torch

import layer_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def close(name, got, want, size, keys, rows, dtype=torch.float32):
    got = got.detach().cpu().double().reshape(want.shape)
    assert torch.isfinite(got).all(), name
    limit = torch.finfo(dtype).eps / 2 * want.abs() + 5 * 2.0 ** -22 * math.sqrt(keys + 2 * 64 + rows) * size * (1 + torch.finfo(dtype).eps)
    limit = limit + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - want).abs() - limit
    worst = int(off.argmax()) if off.numel() else 0
    assert not off.numel() or off.max() <= 0, (name, worst, float(got.reshape(-1)[worst]), float(want.reshape(-1)[worst]), float(limit.reshape(-1)[worst]))


def generator(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen)


def split(lengths):
    first = np.concatenate([[0], np.cumsum(lengths)])
    return [slice(int(a), int(b)) for a, b in zip(first, first[1:])], torch.tensor(first, dtype=torch.int32).cuda()


class Inputs:
    """Of sequences of those lengths, on the host: q, k, v as rows, some more behind the last."""

    def __init__(self, lengths, heads, key_heads, keys, values, dtype, spare=0, seed=0, places=0):
        r, T, rows = generator(seed), TYPES[dtype], sum(lengths) + spare
        self.q, self.k = r(rows, key_heads * keys).to(T), (r(rows, key_heads * keys) + 0.3).to(T)
        self.v = r(rows, heads * values).to(T)
        self.g = -torch.exp(r(rows, heads) - 2)
        self.beta = torch.sigmoid(2 * r(rows, heads))
        self.initial = r(max(places, len(lengths)), heads, keys, values)
        self.dout, self.dfinal = r(rows, heads * values).to(T), r(len(lengths), heads, keys, values)
        self.sizes = (heads, key_heads, keys, values)

    def of(self, part):
        heads, key_heads, keys, values = self.sizes
        n = part.stop - part.start
        return (self.q[part].view(n, key_heads, keys), self.k[part].view(n, key_heads, keys), self.v[part].view(n, heads, values), self.g[part], self.beta[part])


CASES = [
    # lengths, heads, key heads, keys, values, type, normalise, packed, slots, initial state
    ([1], 2, 1, 16, 16, "float32", True, False, False, True),
    ([1, 1, 1], 4, 2, 128, 128, "bfloat16", True, False, True, True),
    ([1, 1], 3, 3, 37, 21, "float16", False, False, False, True),
    ([1] * 5, 2, 2, 64, 1024, "bfloat16", True, False, False, False),
    ([2], 1, 1, 1, 1, "float32", True, False, False, True),
    ([5], 2, 1, 16, 8, "bfloat16", True, False, False, True),
    ([32, 32], 2, 2, 64, 64, "float32", True, False, False, True),
    ([64], 2, 1, 128, 128, "bfloat16", True, False, False, False),
    ([65, 65], 3, 1, 128, 96, "bfloat16", True, False, True, True),
    ([200], 4, 2, 64, 80, "bfloat16", True, False, False, True),
    ([301], 3, 1, 33, 47, "float32", True, False, False, True),
    ([137], 6, 3, 100, 72, "float16", True, False, False, True),
    ([150], 2, 2, 128, 200, "float32", True, False, False, True),
    ([97], 2, 2, 128, 128, "float16", False, False, False, True),
    ([0, 150, 1, 0, 64, 65, 8, 0], 2, 1, 40, 24, "bfloat16", True, True, True, True),
    ([0, 33, 1, 0, 32, 31, 128, 0, 2], 4, 2, 128, 64, "float32", True, True, False, True),
    ([100, 2], 2, 1, 72, 16, "float16", True, True, True, False),
    ([513], 1, 1, 128, 256, "bfloat16", True, False, False, True),
]


@pytest.mark.parametrize("lengths, heads, key_heads, keys, values, dtype, normalise, packed, slots, initial", CASES)
def test_delta_rule(lengths, heads, key_heads, keys, values, dtype, normalise, packed, slots, initial):
    from genn_amd.sequence import GatedDeltaRule
    T, S = TYPES[dtype], len(lengths)
    parts, offsets = split(lengths)
    rows, spare = sum(lengths), 3 if packed else 0
    places = S + 2 if slots else S
    i = Inputs(lengths, heads, key_heads, keys, values, dtype, spare, seed=len(lengths) * 100 + keys, places=places)
    if not normalise:
        i.q, i.k = ((x.float() / math.sqrt(2 * keys)).to(T) for x in (i.q, i.k))         # (shorter than 1, as the bound asks for)
    where = torch.randperm(places, generator=torch.Generator().manual_seed(1))[:S] if slots else torch.arange(S)
    state, out = i.initial.clone().cuda(), torch.full((rows + spare, heads * values), 7.0, dtype=T).cuda()
    # (keys, queries and values side by side in one array's rows, as a projection leaves them)
    wide = torch.cat([i.q, i.k, i.v], 1).cuda()
    a, b = i.q.shape[1], i.q.shape[1] + i.k.shape[1]
    op = GatedDeltaRule(S, max(lengths), heads, keys, values, key_heads=key_heads, dtype=dtype, normalise=normalise)
    arrays = dict(q=wide[:, :a], k=wide[:, a:b], v=wide[:, b:], g=i.g.cuda(), beta=i.beta.cuda(), offsets=offsets if packed else None)
    op.bind(out=out, initial_state=state if initial else None, final_state=state, slots=where.to(torch.int32).cuda() if slots else None, **arrays)
    op.run()
    torch.cuda.synchronize()
    for n, part in enumerate(parts):
        want, final, size = ref.delta(*i.of(part), keys ** -0.5, normalise, initial=i.initial[where[n]] if initial else None)
        close(f"out of {n}", out[part], want.reshape(-1, heads * values), size["out"].reshape(-1).expand(want.shape[0], -1), keys, lengths[n], T)
        close(f"final of {n}", state[where[n]], final, size["final"], keys, lengths[n])
    assert torch.all(out[rows:] == 7.0)
    others = [p for p in range(places) if p not in where.tolist()]
    assert torch.equal(state[others].cpu(), i.initial[others])
    if slots:
        return
    dq, dk, dv = (torch.full((rows + spare, n), 7.0, dtype=T).cuda() for n in (key_heads * keys, key_heads * keys, heads * values))
    dg, dbeta = (torch.full((rows + spare, heads), 7.0).cuda() for _ in range(2))
    dinitial = torch.full((S, heads, keys, values), 7.0).cuda()
    op.bind(initial_state=i.initial.cuda() if initial else None, **arrays)
    op.bind_gradients(out=i.dout.cuda(), final_state=i.dfinal.cuda(), q=dq, k=dk, v=dv, g=dg, beta=dbeta, initial_state=dinitial)
    op.backward()
    torch.cuda.synchronize()
    for n, part in enumerate(parts):
        found, size = ref.delta(*i.of(part), keys ** -0.5, normalise, initial=i.initial[n] if initial else None,
                                dout=i.dout[part].view(-1, heads, values), dfinal=i.dfinal[n])
        for name, got, t in (("dv", dv, T), ("dbeta", dbeta, torch.float32), ("dg", dg, torch.float32), ("dq", dq, T), ("dk", dk, T)):
            close(f"{name} of {n}", got[part], found[name].reshape(lengths[n], got.shape[1]), size[name].reshape(lengths[n], got.shape[1]), keys, lengths[n], t)
        close(f"dinitial of {n}", dinitial[n], found["dinitial"], size["dinitial"], keys, lengths[n])
    for x in (dq, dk, dv, dg, dbeta):
        assert torch.all(x[rows:] == 7.0)
