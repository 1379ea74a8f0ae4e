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


def arrays(i, heads, key_heads, keys, values):
    return dict(q=i.q.cuda(), k=i.k.cuda(), v=i.v.cuda(), g=i.g.cuda(), beta=i.beta.cuda())


@pytest.mark.parametrize("lengths, heads, key_heads, keys, values, dtype", [
    ([1500], 2, 1, 128, 64, "bfloat16"),
    ([1200, 3, 64, 0, 700, 1], 2, 2, 64, 40, "float32"),
    ([900, 900], 2, 1, 96, 128, "float16"),
])
def test_long_sequences_are_cut_and_joined(lengths, heads, key_heads, keys, values, dtype):
    from genn_amd.sequence import GatedDeltaRule
    T, S = TYPES[dtype], len(lengths)
    parts, offsets = split(lengths)
    i = Inputs(lengths, heads, key_heads, keys, values, dtype, 3, seed=7)
    out, final = torch.full((sum(lengths) + 3, heads * values), 7.0, dtype=T).cuda(), torch.zeros(S, heads, keys, values).cuda()
    op = GatedDeltaRule(S, max(lengths), heads, keys, values, key_heads=key_heads, dtype=dtype, normalise=True)
    op.bind(out=out, initial_state=i.initial.cuda(), final_state=final, offsets=offsets, **arrays(i, heads, key_heads, keys, values))
    op.run()
    for n, part in enumerate(parts):
        want, last, size = ref.delta(*i.of(part), keys ** -0.5, True, initial=i.initial[n])
        close(f"out of {n}", out[part], want.reshape(-1, heads * values), size["out"].reshape(-1).expand(want.shape[0], -1), keys, lengths[n], T)
        close(f"final of {n}", final[n], last, size["final"], keys, lengths[n])
    assert torch.all(out[sum(lengths):] == 7.0)


def test_gates_and_rates_at_their_ends():
    """Gates that forget everything, nothing, or grow; rates of zero and one; two rows with the same key."""
    from genn_amd.sequence import GatedDeltaRule
    n, H, K, V = 150, 3, 24, 20
    i = Inputs([n], H, H, K, V, "float32", seed=3)
    i.g[::7, 0], i.g[3::11, 1], i.g[:, 2] = -math.inf, 0.0, 0.01
    i.g[5, 1] = -1e30
    i.beta[::3], i.beta[1::5] = 0.0, 1.0
    i.k[40:60] = i.k[39]
    finite = torch.clamp(i.g, min=-1e6)
    out, final = torch.zeros(n, H * V).cuda(), torch.zeros(1, H, K, V).cuda()
    grads = dict(q=torch.zeros(n, H * K).cuda(), k=torch.zeros(n, H * K).cuda(), v=torch.zeros(n, H * V).cuda(), g=torch.zeros(n, H).cuda(), beta=torch.zeros(n, H).cuda())
    dinitial = torch.zeros(1, H, K, V).cuda()
    op = GatedDeltaRule(1, n, H, K, V, normalise=True)
    op.bind(out=out, initial_state=i.initial.cuda(), final_state=final, **arrays(i, H, H, K, V))
    op.run()
    op.bind_gradients(out=i.dout.cuda(), final_state=i.dfinal.cuda(), initial_state=dinitial, **grads)
    op.backward()
    q, k, v, _, beta = i.of(slice(0, n))
    want, last, size = ref.delta(q, k, v, finite, beta, K ** -0.5, True, initial=i.initial[0])
    # (the third head's state grows: exp(1.5) over all rows, an error as well)
    grow = math.exp(0.01 * n)
    close("out", out, want.reshape(n, -1), grow * size["out"].reshape(-1).expand(n, -1), K, n)
    close("final", final[0], last, grow * size["final"], K, n)
    found, size = ref.delta(q, k, v, finite, beta, K ** -0.5, True, initial=i.initial[0], dout=i.dout.view(n, H, V), dfinal=i.dfinal[0])
    for name, x in grads.items():
        close("d" + name, x, found["d" + name].reshape(x.shape), grow * grow * size["d" + name].reshape(x.shape), K, n)
    close("dinitial", dinitial[0], found["dinitial"], grow * size["dinitial"], K, n)


def test_tokens_continue_a_prompt_and_padding_is_left_alone():
    from genn_amd.sequence import GatedDeltaRule
    n, at, H, G, K, V = 90, 70, 4, 2, 64, 48
    i = Inputs([n], H, G, K, V, "bfloat16", seed=5)
    whole = torch.zeros(n, H * V, dtype=torch.bfloat16).cuda()
    sizes = dict(heads=H, keys=K, values=V, key_heads=G, dtype="bfloat16", normalise=True)
    op = GatedDeltaRule(1, n, **sizes)
    op.bind(out=whole, **arrays(i, H, G, K, V))
    op.run()
    pool, slots = torch.full((5, H, K, V), 9.0).cuda(), torch.tensor([3], dtype=torch.int32).cuda()
    got = torch.zeros(n, H * V, dtype=torch.bfloat16).cuda()
    op = GatedDeltaRule(1, at, **sizes)
    op.bind(q=i.q[:at].cuda(), k=i.k[:at].cuda(), v=i.v[:at].cuda(), g=i.g[:at].cuda(), beta=i.beta[:at].cuda(), out=got[:at], final_state=pool, slots=slots)
    op.run()
    slots = torch.tensor([-1, 3, 5], dtype=torch.int32).cuda()
    wide = lambda t, k: torch.stack([torch.full_like(t[k], math.nan), t[k], torch.full_like(t[k], math.nan)]).cuda()  # noqa: E731
    out = torch.full((3, H * V), 4.0, dtype=torch.bfloat16).cuda()
    op = GatedDeltaRule(3, 1, **sizes)
    for t in range(at, n):
        op.bind(q=wide(i.q, t), k=wide(i.k, t), v=wide(i.v, t), g=wide(i.g, t), beta=wide(i.beta, t), out=out, initial_state=pool, final_state=pool, slots=slots)
        op.run()
        got[t] = out[1]
    want, _, size = ref.delta(*i.of(slice(0, n)), K ** -0.5, True)
    for x in (whole, got):
        close("out", x, want.reshape(n, -1), size["out"].reshape(-1).expand(n, -1), K, n, torch.bfloat16)
    assert torch.all(out[[0, 2]] == 4.0) and torch.all(pool[[0, 1, 2, 4]] == 9.0)
    # a prompt's batch with padding in it: nothing of the padding's rows is read or written
    x, out = torch.full((2, 40, H * V), 4.0, dtype=torch.bfloat16).cuda(), torch.full((2, 40, H * V), 4.0, dtype=torch.bfloat16).cuda()
    two = lambda t: torch.stack([torch.full_like(t[:40], math.nan), t[:40]]).cuda()  # noqa: E731
    op = GatedDeltaRule(2, 40, **sizes)
    op.bind(q=two(i.q), k=two(i.k), v=two(i.v), g=two(i.g), beta=two(i.beta), out=out, final_state=pool, slots=torch.tensor([7, 2], dtype=torch.int32).cuda())
    op.run()
    assert torch.equal(out[0], x[0]) and torch.isfinite(out[1]).all() and torch.all(pool[[0, 1, 4]] == 9.0)


@pytest.mark.parametrize("dtype, heads", [("bfloat16", 2), ("float32", 2), ("bfloat16", 300)])
def test_what_is_not_finite_stays_where_it_belongs(dtype, heads):
    """In a sequence that is cut into segments and in one that is not (of enough heads for the whole chip)."""
    from genn_amd.sequence import GatedDeltaRule
    n, H, K, V, T = 200, heads, 40, 33, TYPES[dtype]
    i = Inputs([n], H, H, K, V, dtype, seed=8)

    def run(change, tokens=False):
        a = {k: x.clone() for k, x in dict(q=i.q, k=i.k, v=i.v, g=i.g, beta=i.beta, initial=i.initial).items()}
        change(a)
        out, final = torch.zeros(n, H * V, dtype=T).cuda(), torch.zeros(1, H, K, V).cuda()
        op = GatedDeltaRule(1, n, H, K, V, dtype=dtype, normalise=True)
        op.bind(out=out, initial_state=a["initial"].cuda(), final_state=final, **{k: a[k].cuda() for k in ("q", "k", "v", "g", "beta")})
        op.run()
        return out.view(n, H, V).cpu(), final[0].cpu()

    clean, last = run(lambda a: None)
    assert torch.isfinite(clean).all() and torch.isfinite(last).all()

    def check(change, rows, head, columns, state=True):
        out, final = run(change)
        bad = torch.zeros(n, H, V, dtype=torch.bool)
        bad[rows, head, columns] = True
        assert torch.equal(~torch.isfinite(out), bad)
        assert torch.equal(out[~bad], clean[~bad])
        bad = torch.zeros(H, K, V, dtype=torch.bool)
        bad[head, :, columns] = state
        assert torch.equal(~torch.isfinite(final), bad)
        assert torch.equal(final[~bad], last[~bad])

    every = slice(None)
    check(lambda a: a["v"].view(n, H, V)[70, 1].__setitem__(5, math.inf), slice(70, None), 1, 5)
    check(lambda a: a["v"].view(n, H, V)[0, 0].__setitem__(32, math.nan), slice(0, None), 0, 32)
    check(lambda a: a["q"].view(n, H, K)[10, 1].__setitem__(3, math.nan), 10, 1, every, state=False)
    check(lambda a: a["k"].view(n, H, K)[101, 0].__setitem__(39, math.nan), slice(101, None), 0, every)
    check(lambda a: a["k"].view(n, H, K)[0, 1].__setitem__(0, math.inf), slice(0, None), 1, every)
    check(lambda a: a["beta"][131].__setitem__(1, math.nan), slice(131, None), 1, every)
    check(lambda a: a["g"][63].__setitem__(0, math.nan), slice(63, None), 0, every)
    check(lambda a: a["initial"][0, 1, 7].__setitem__(9, math.inf), slice(0, None), 1, 9)


def test_nothing_to_do():
    from genn_amd.sequence import GatedDeltaRule
    H, K, V = 2, 8, 4
    e = lambda w: torch.zeros(0, w).cuda()  # noqa: E731
    state, final = torch.randn(3, H, K, V).cuda(), torch.zeros(3, H, K, V).cuda()
    a = dict(q=e(H * K), k=e(H * K), v=e(H * V), g=e(H), beta=e(H))
    for offsets in (None, torch.zeros(4, dtype=torch.int32).cuda()):
        for length in (0,) if offsets is None else (0, 5):
            final.zero_()
            op = GatedDeltaRule(3, length, H, K, V, normalise=True)
            op.bind(out=e(H * V), initial_state=state, final_state=final, offsets=offsets, **a)
            op.run()
            assert torch.equal(final, state)
            dinitial = torch.zeros_like(state)
            op.bind_gradients(out=e(H * V), q=e(H * K), final_state=state, initial_state=dinitial)
            op.backward()
            assert torch.equal(dinitial, state)
    op = GatedDeltaRule(0, 7, H, K, V)
    op.bind(out=e(H * V), final_state=torch.zeros(0, H, K, V).cuda(), **a)
    op.run()
    op.bind_gradients(out=e(H * V), q=e(H * K))
    op.backward()
    # states that begin at nothing
    final.fill_(5.0)
    op = GatedDeltaRule(3, 0, H, K, V)
    op.bind(out=e(H * V), final_state=final, **a)
    op.run()
    assert torch.all(final == 0.0)


def test_rows_behind_the_longest_that_is_allowed_are_left_alone():
    from genn_amd.sequence import GatedDeltaRule
    H, K, V, lengths = 2, 16, 8, [70, 5, 90]
    parts, offsets = split(lengths)
    i = Inputs(lengths, H, H, K, V, "float32", seed=4)
    for length in (33, 1):
        out = torch.full((sum(lengths), H * V), 7.0).cuda()
        op = GatedDeltaRule(3, length, H, K, V, normalise=True)
        op.bind(out=out, offsets=offsets, **arrays(i, H, H, K, V))
        op.run()
        for part in parts:
            used = slice(part.start, min(part.stop, part.start + length))
            want, _, size = ref.delta(*i.of(used), K ** -0.5, True)
            close("out", out[used], want.reshape(-1, H * V), size["out"].reshape(-1).expand(want.shape[0], -1), K, length)
            assert torch.all(out[used.stop:part.stop] == 7.0)


@pytest.mark.parametrize("shift", [1, 3, 4])
def test_any_alignment_gives_the_same(shift):
    from genn_amd.sequence import GatedDeltaRule
    n, H, K, V = 130, 2, 64, 32
    i = Inputs([n], H, H, K, V, "bfloat16", seed=2)

    def placed(t):
        room = torch.empty(t.numel() + 8, dtype=t.dtype).cuda()
        view = room[shift:shift + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    results = []
    for place in (lambda t: t.cuda(), placed):
        out, token = place(torch.zeros(n, H * V).bfloat16()), place(torch.zeros(1, H * V).bfloat16())
        state, kept = place(i.initial), place(i.initial)
        a = {k: place(x) for k, x in dict(q=i.q, k=i.k, v=i.v, g=i.g, beta=i.beta).items()}
        op = GatedDeltaRule(1, n, H, K, V, dtype="bfloat16", normalise=True)
        op.bind(out=out, initial_state=state, final_state=state, **a)
        op.run()
        grads = {k: place(torch.zeros_like(x)) for k, x in dict(q=i.q, k=i.k, v=i.v, g=i.g, beta=i.beta).items()}
        op.bind_gradients(out=place(i.dout), final_state=place(i.dfinal), **grads)
        op.backward()
        t = GatedDeltaRule(1, 1, H, K, V, dtype="bfloat16", normalise=True)
        t.bind(out=token, initial_state=kept, final_state=kept, **{k: x[:1] for k, x in a.items()})
        t.run()
        results.append([x.float().cpu() for x in (out, state, token, kept, *grads.values())])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_states_and_sequences_beyond_32_bits():
    """A pool of states of more than 2^32 elements, and sequences more than 2^32 elements apart, rows the most that is allowed."""
    from genn_amd.sequence import GatedDeltaRule
    H, K, V, n, stride = 2, 16, 16, 40, (1 << 25) - 1
    i = Inputs([n], H, H, K, V, "bfloat16", seed=6)
    places = (1 << 32) // (H * K * V) + 2
    pool = torch.empty(places, H, K, V, device="cuda")
    pool[places - 1] = i.initial[0].cuda()
    room = torch.empty(2 * n * stride + 4096, dtype=torch.bfloat16, device="cuda")
    used = [0]

    def far(t, width):
        at = torch.as_strided(room, (1, n, width), (0, stride, 1), used[0] + n * stride)
        used[0] += width
        if t is not None:
            at[0].copy_(t)
        return at

    a = dict(q=far(i.q, H * K), k=far(i.k, H * K), v=far(i.v, H * V), g=i.g.cuda(), beta=i.beta.cuda())
    out = far(None, H * V)
    op = GatedDeltaRule(1, n, H, K, V, dtype="bfloat16", normalise=True)
    op.bind(out=out, initial_state=pool, final_state=pool, slots=torch.tensor([places - 1], dtype=torch.int32).cuda(), **a)
    op.run()
    want, last, size = ref.delta(*i.of(slice(0, n)), K ** -0.5, True, initial=i.initial[0])
    close("out", out[0].clone(), want.reshape(n, -1), size["out"].reshape(-1).expand(n, -1), K, n, torch.bfloat16)
    close("final", pool[places - 1], last, size["final"], K, n)
    grads = {k: far(None, w) for k, w in (("q", H * K), ("k", H * K), ("v", H * V))}
    op.bind(initial_state=i.initial.cuda(), **a)
    op.bind_gradients(out=far(i.dout, H * V), **grads)
    op.backward()
    found, size = ref.delta(*i.of(slice(0, n)), K ** -0.5, True, initial=i.initial[0], dout=i.dout.view(n, H, V))
    for k, x in grads.items():
        close("d" + k, x[0].clone(), found["d" + k].reshape(n, -1), size["d" + k].reshape(n, -1), K, n, torch.bfloat16)


def test_gradients_asked_for_one_by_one():
    from genn_amd.sequence import GatedDeltaRule
    for H, G in ((2, 2), (4, 2)):
        n, K, V = 100, 24, 16
        i = Inputs([n], H, G, K, V, "float32", seed=9)
        make = lambda: dict(q=torch.zeros(n, G * K).cuda(), k=torch.zeros(n, G * K).cuda(), v=torch.zeros(n, H * V).cuda(), g=torch.zeros(n, H).cuda(), beta=torch.zeros(n, H).cuda(),  # noqa: E731
                            initial_state=torch.zeros(1, H, K, V).cuda())
        op = GatedDeltaRule(1, n, H, K, V, key_heads=G, normalise=True)
        op.bind(initial_state=i.initial.cuda(), **arrays(i, H, G, K, V))
        every = make()
        op.bind_gradients(out=i.dout.cuda(), final_state=i.dfinal.cuda(), **every)
        op.backward()
        for name in every:
            one = make()[name]
            op.bind_gradients(out=i.dout.cuda(), final_state=i.dfinal.cuda(), **{name: one})
            op.backward()
            assert torch.equal(one, every[name]) and float(one.abs().sum()) > 0, name
        # the gradient of the state in front over that of the state behind
        both = i.dfinal.cuda()
        op.bind_gradients(out=i.dout.cuda(), final_state=both, initial_state=both)
        op.backward()
        assert torch.equal(both, every["initial_state"])


def test_another_current_device_is_refused():
    from genn_amd import _abi
    from genn_amd.sequence import Dropout, GatedDeltaRule, LayerNorm
    x, g = torch.zeros(2, 8).cuda(), torch.zeros(2, 1).cuda()
    rule, norm, drop = GatedDeltaRule(1, 2, 1, 8, 8), LayerNorm(1, 2, 8), Dropout(1, 2, 8, 0.5)
    out = torch.zeros(2, 8).cuda()
    rule.bind(q=x, k=x, v=x, g=g, beta=g, out=out)
    norm.bind(x=x, out=out)
    drop.bind(x=x, out=out)
    # (the descriptors say that their arrays are on a device that is not the current one)
    rule._descriptor.sequences.device = norm._descriptor.sequences.device = drop._forward.sequences.device = 9
    for run in (rule.run, norm.run, lambda: drop.run(1)):
        with pytest.raises(_abi.GennmiError, match="current device"):
            run()


def test_a_layer_of_them_together_on_a_stream_and_in_a_graph():
    """Convolution, gated delta rule, norm of its heads with a gate, dropout onto the residual, a norm: forwards and back, against formulas in 64 bits, eagerly and replayed.

    What may differ: every stage's result is off by at most its own bound (5 x 2^-22 sqrt(keys + 2 * 64 + rows) relative to the largest of its array).  The same formulas are run with every stage's
    result off by that much at random; what that makes of the gradients, eight times, is the limit."""
    from genn_amd.sequence import CausalConvolution, Dropout, GatedDeltaRule, LayerNorm
    n, H, G, K, V, taps = 260, 4, 2, 32, 32, 4
    D = 2 * G * K + H * V
    gen = torch.Generator().manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    x, weight, bias, z, res = r(n, D), r(D, taps) / 2, r(D) / 4, r(n, H * V), r(n, H * V)
    g, beta, w1, w2, b2, loss = -torch.exp(r(n, H) - 2), torch.sigmoid(r(n, H)), 1 + r(V) / 8, 1 + r(H * V) / 8, r(H * V) / 8, r(n, H * V)
    keep, factor = ref.kept(n, H * V, 0.2, 77, 5)

    def formulas(noise, seed=0):
        rng = torch.Generator().manual_seed(seed)
        off = lambda t: t + noise * t.detach().abs().max() * (2 * torch.rand(t.shape, generator=rng, dtype=torch.float64) - 1)  # noqa: E731
        leaves = [t.double().requires_grad_() for t in (x, weight, bias, z, res, g, beta, w1, w2, b2)]
        X, W, B, Z, R, g_, b_, W1, W2, B2 = leaves
        ext = torch.cat([torch.zeros(taps - 1, D, dtype=torch.float64), X])
        s = B + sum(ext[k:k + n] * W[:, k] for k in range(taps))
        c = off(s * torch.sigmoid(s))
        unit = lambda t: ref.unit(t.view(n, G, K), 1e-6).repeat_interleave(H // G, 1)  # noqa: E731
        q, k, v = unit(c[:, :G * K]), unit(c[:, G * K:2 * G * K]), c[:, 2 * G * K:].view(n, H, V)
        S, rows = torch.zeros(H, K, V, dtype=torch.float64), []
        for t in range(n):
            S = torch.exp(g_[t])[:, None, None] * S
            S = S + k[t][:, :, None] * (b_[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1)))[:, None]
            rows.append(K ** -0.5 * (S * q[t][:, :, None]).sum(1))
        o = off(torch.stack(rows))
        o = off((o / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-5) * W1).reshape(n, H * V) * Z * torch.sigmoid(Z))
        h = off(R + torch.where(keep, o, 0.0) * factor)
        m = h - h.mean(-1, keepdim=True)
        y = off(m / torch.sqrt((m * m).mean(-1, keepdim=True) + 1e-5) * W2 + B2)
        return [y.detach()] + list(torch.autograd.grad((y * loss.double()).sum(), leaves))

    want = formulas(0.0)
    bound = 5 * 2.0 ** -22 * math.sqrt(K + 2 * 64 + n)
    limits = [8 * max(float((a - b).norm()) for a in (formulas(bound, s)[k] for s in (1, 2))) + bound * float(b.norm()) for k, b in enumerate(want)]

    on = lambda t: t.cuda()  # noqa: E731
    empty = lambda *shape: torch.zeros(*shape).cuda()  # noqa: E731
    a = dict(x=on(x), weight=on(weight), bias=on(bias), z=on(z), res=on(res), g=on(g), beta=on(beta), w1=on(w1), w2=on(w2), b2=on(b2), loss=on(loss))
    c, o, p, h, y = empty(n, D), empty(n, H * V), empty(n, H * V), empty(n, H * V), empty(n, H * V)
    dy = {k: torch.zeros_like(t) for k, t in a.items()}
    dc, do, dp, dh = empty(n, D), empty(n, H * V), empty(n, H * V), empty(n, H * V)
    call = torch.tensor([5], dtype=torch.int64).cuda()
    conv, rule, head, drop, norm = CausalConvolution(1, n, D, taps, silu=True), GatedDeltaRule(1, n, H, K, V, key_heads=G, normalise=True), LayerNorm(n, H, V, rms=True), \
        Dropout(1, n, H * V, 0.2, seed=77), LayerNorm(1, n, H * V)
    conv.bind(x=a["x"], weight=a["weight"], bias=a["bias"], out=c)
    rule.bind(q=c[:, :G * K], k=c[:, G * K:2 * G * K], v=c[:, 2 * G * K:], g=a["g"], beta=a["beta"], out=o)
    head.bind(x=o.view(n, H, V), weight=a["w1"], gate=a["z"].view(n, H, V), out=p.view(n, H, V))
    drop.bind(x=p, residual=a["res"], out=h)
    norm.bind(x=h, weight=a["w2"], bias=a["b2"], out=y)
    norm.bind_gradients(out=a["loss"], x=dh, weight=dy["w2"], bias=dy["b2"])
    drop.bind_gradients(out=dh, x=dp)
    head.bind_gradients(out=dp.view(n, H, V), x=do.view(n, H, V), weight=dy["w1"], gate=dy["z"].view(n, H, V))
    rule.bind_gradients(out=do, q=dc[:, :G * K], k=dc[:, G * K:2 * G * K], v=dc[:, 2 * G * K:], g=dy["g"], beta=dy["beta"])
    conv.bind_gradients(out=dc, x=dy["x"], weight=dy["weight"], bias=dy["bias"])
    sizes = [rule.workspace_bytes, norm.backward_workspace_bytes, head.backward_workspace_bytes, rule.backward_workspace_bytes, conv.backward_workspace_bytes]
    assert all(sizes)
    spaces = [torch.empty(b, dtype=torch.uint8).cuda() for b in sizes]

    def run(stream, w=(None,) * 5):
        conv.run(stream)
        rule.run(stream, w[0])
        head.run(stream)
        drop.run(call, stream)
        norm.run(stream)
        norm.backward(stream, w[1])
        drop.backward(call, stream)
        head.backward(stream, w[2])
        rule.backward(stream, w[3])
        conv.backward(stream, w[4])

    results = [y] + [dh if k == "res" else dy[k] for k in ("x", "weight", "bias", "z", "res", "g", "beta", "w1", "w2", "b2")]
    run(0)
    torch.cuda.synchronize()
    for k, (got, b, limit) in enumerate(zip(results, want, limits)):
        assert float((got.cpu().double() - b).norm()) <= limit, (k, float((got.cpu().double() - b).norm()), limit, float(b.norm()))
    first = [t.clone() for t in results]
    side = torch.cuda.Stream()
    for t in results:
        t.zero_()
    side.wait_stream(torch.cuda.current_stream())
    run(side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(results, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        stream = torch.cuda.current_stream().cuda_stream
        for refused in (rule.run, rule.backward, norm.backward):
            with pytest.raises(ValueError, match="captured"):
                refused(stream)
        run(stream, spaces)
    for k in range(4):
        for t in results:
            t.zero_()
        if k % 2:
            run(0)          # (eager, on workspaces of its own)
            for t in results:
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(results, first)), k
    # another call's number: other elements are dropped
    call.fill_(6)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(results[0], first[0])
    got = [t.clone() for t in results]
    run(0)
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(results, got))
