"""Causal convolution and selective scan through the C ABI against their restatements in 64 bits.

Tolerances.  A result is one rounding to its type (half a step: eps / 2 of the value) of a sum in fp32.  Every operation of that sum is off by at most half a step
of fp32, 2^-24, an exponential or logistic function by a few: counted as 4 x 2^-24 for each operation on the way from an input to the result, of
which there are K + 4 in a convolution and 2 (a decay and a sum) for every row that lies between them in a scan, relative to the sum of all terms' absolute
values (``magnitudes``).  Decays exp(dt A) add what their exponent is off by, |dt A| x 2^-22, over a run of rows at most
(sum |dt A|) exp(-sum |dt A|) < 1 in all: one more operation."""
import numpy as np
import pytest
import torch

import sequence_ref as ref
from genn_amd import _abi
from genn_amd.genn_model import Array

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
U = 2.0 ** -22


def close(name, got, want, size, operations, dtype=torch.float32):
    """Within half a step of the type and `operations` roundings of the magnitudes; smallest subnormals of the type count as well."""
    got = got.detach().cpu().double().reshape(want.shape)
    limit = torch.finfo(dtype).eps / 2 * want.abs() + operations * U * size * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - want).abs() - limit
    assert torch.isfinite(got).all(), name
    worst = int(off.argmax()) if off.numel() else 0
    assert not off.numel() or off.max() <= 0, (name, worst, float(got.reshape(-1)[worst]), float(want.reshape(-1)[worst]), float(limit.reshape(-1)[worst]))


def generator(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen)


def split(lengths):
    first = np.concatenate([[0], np.cumsum(lengths)])
    return [slice(int(a), int(b)) for a, b in zip(first, first[1:])], torch.tensor(first, dtype=torch.int32).cuda()


CONV = [
    # lengths, channels, taps, type, silu, bias, packed, slots, initial state
    ([5], 8, 4, "float32", True, True, False, False, False),
    ([1, 1, 1], 12, 4, "bfloat16", True, True, False, True, True),
    ([33, 33], 64, 4, "bfloat16", True, True, False, False, True),
    ([17], 3, 1, "float32", False, False, False, False, True),
    ([40], 7, 2, "float16", False, True, False, False, True),
    ([16, 16], 260, 3, "float32", True, False, False, False, False),
    ([64], 129, 8, "bfloat16", True, True, False, False, True),
    ([2, 2], 20, 8, "float16", True, True, False, False, True),
    ([0, 3, 50, 1, 0, 16, 17, 0], 36, 4, "bfloat16", True, True, True, True, True),
    ([0, 3, 50, 1, 0, 16, 17, 0], 5, 5, "float32", False, True, True, False, True),
    ([100, 2], 24, 6, "float16", True, True, True, False, False),
    ([31], 12, 7, "float32", True, True, False, False, True),
]


@pytest.mark.parametrize("lengths, channels, taps, dtype, silu, bias, packed, slots, initial", CONV)
def test_causal_conv(lengths, channels, taps, dtype, silu, bias, packed, slots, initial):
    from genn_amd.sequence import CausalConvolution
    T, r, S, K = TYPES[dtype], generator(len(lengths) * 100 + channels), len(lengths), taps
    parts, offsets = split(lengths)
    rows, spare = sum(lengths), 3 if packed else 0
    x = r(rows + spare, channels).to(T)
    weight, b = r(channels, K) * K ** -0.5, r(channels) if bias else None
    places = S + 2 if slots else S
    where = torch.randperm(places, generator=torch.Generator().manual_seed(1))[:S] if slots else torch.arange(S)
    before = r(places, K - 1, channels).to(T)
    state, out = before.clone().cuda(), torch.full((rows + spare, channels), 7.0, dtype=T).cuda()
    op = CausalConvolution(S, max(lengths), channels, K, dtype=dtype, silu=silu)
    # (initial and final state are the same array where there is an initial one)
    op.bind(x=x.cuda(), weight=weight.cuda(), bias=None if b is None else b.cuda(), out=out, initial_state=state if initial else None, final_state=state,
            offsets=offsets if packed else None, slots=where.to(torch.int32).cuda() if slots else None)
    op.run()
    torch.cuda.synchronize()
    for k, part in enumerate(parts):
        args = (x[part], weight, b, silu, before[where[k]] if initial else None)
        want, final = ref.causal_conv(*args)
        close(f"out of {k}", out[part], want, ref.causal_conv(*args, magnitudes=True)[0], K + 8, T)
        assert torch.equal(state[where[k]].cpu().double(), final)
    assert torch.all(out[rows:] == 7.0)
    others = [p for p in range(places) if p not in where.tolist()]
    assert torch.equal(state[others].cpu(), before[others])
    if slots:
        return
    dout, dfinal = r(rows + spare, channels).to(T), r(S, K - 1, channels).to(T)
    dx = torch.full((rows + spare, channels), 7.0, dtype=T).cuda()
    dw, db, dinitial = torch.full((channels, K), 7.0).cuda(), torch.full((channels,), 7.0).cuda(), torch.full((S, K - 1, channels), 7.0, dtype=T).cuda()
    op.bind(x=x.cuda(), weight=weight.cuda(), bias=None if b is None else b.cuda(), initial_state=before.cuda() if initial else None, offsets=offsets if packed else None)
    op.bind_gradients(out=dout.cuda(), final_state=dfinal.cuda(), x=dx, weight=dw, bias=db, initial_state=dinitial)
    op.backward()
    torch.cuda.synchronize()
    sums, sizes = [0, 0], [0, 0]
    for k, part in enumerate(parts):
        args = (x[part], weight, b, silu, before[k] if initial else None, dout[part], dfinal[k])
        want, size = ref.causal_conv(*args), ref.causal_conv(*args, magnitudes=True)
        close(f"dx of {k}", dx[part], want[0], size[0], 2 * K + 16, T)
        close(f"dinitial of {k}", dinitial[k], want[3], size[3], 2 * K + 16, T)
        for i in (0, 1):
            sums[i], sizes[i] = sums[i] + want[i + 1], sizes[i] + size[i + 1]
    close("dweight", dw, sums[0], sizes[0], K + 16 + 20)       # (sums of 16 rows, then in 64 bits)
    close("dbias", db, sums[1], sizes[1], K + 16 + 20)
    assert torch.all(dx[rows:] == 7.0)


SCAN = [
    # lengths, channels, states, groups, type, softplus, z, D, bias, packed, slots, initial state
    ([1], 5, 16, 1, "float32", True, True, True, True, False, False, True),
    ([1, 1, 1], 66, 5, 3, "bfloat16", True, True, True, True, False, True, True),
    ([1, 1], 20, 128, 2, "float16", False, False, False, False, False, False, True),
    ([1] * 9, 4, 3, 1, "bfloat16", True, False, True, False, False, False, False),
    ([7, 7], 64, 16, 1, "bfloat16", True, True, True, True, False, False, True),
    ([9], 65, 1, 1, "float32", False, False, False, False, False, False, True),
    ([40], 3, 8, 1, "float16", True, True, False, True, False, False, False),
    ([200, 200], 70, 16, 2, "bfloat16", True, True, True, True, False, False, True),
    ([301], 33, 7, 3, "float32", True, True, True, True, False, False, True),
    ([137], 130, 17, 1, "float32", True, True, True, True, False, False, True),
    ([150], 65, 128, 1, "bfloat16", True, True, True, True, False, False, False),
    ([33], 128, 33, 2, "float16", False, True, True, False, False, False, True),
    ([0, 150, 1, 0, 64, 65, 8, 0], 40, 16, 1, "bfloat16", True, True, True, True, True, True, True),
    ([0, 150, 1, 0, 64, 65, 8, 0], 24, 20, 2, "float32", True, True, True, True, True, False, True),
    ([1, 0, 1, 1], 12, 16, 1, "float32", True, True, True, True, True, True, True),
    ([20] * 100, 1024, 16, 1, "bfloat16", True, True, True, True, False, False, False),
]


@pytest.mark.parametrize("lengths, channels, states, groups, dtype, softplus, gate, skip, bias, packed, slots, initial", SCAN)
def test_selective_scan(lengths, channels, states, groups, dtype, softplus, gate, skip, bias, packed, slots, initial):
    from genn_amd.sequence import SelectiveScan
    T, r, S, D, N, G = TYPES[dtype], generator(sum(lengths) + channels), len(lengths), channels, states, groups
    parts, offsets = split(lengths)
    rows, spare = sum(lengths), 3 if packed else 0
    # (rows of three arrays side by side: their stride is not their width)
    wide = r(rows + spare, D + 2 * G * N).to(T)
    wide[:, :D] = (wide[:, :D].float() if softplus else wide[:, :D].float().abs() * 0.3).to(T)
    device = wide.cuda()
    cut = lambda a: (a[:, :D], a[:, D:D + G * N], a[:, D + G * N:])
    (delta, B, C), (ddelta_, dB_, dC_) = cut(wide), cut(device)
    u, z = r(rows + spare, D).to(T), r(rows + spare, D).to(T) if gate else None
    A = -torch.exp(r(D, N) * 0.5) * 0.7
    skips, b = r(D) if skip else None, r(D) - 2 if bias else None
    places = S + 2 if slots else S
    where = torch.randperm(places, generator=torch.Generator().manual_seed(1))[:S] if slots else torch.arange(S)
    before = r(places, D, N)
    state, out = before.clone().cuda(), torch.full((rows + spare, D), 7.0, dtype=T).cuda()
    on = lambda t: None if t is None else t.cuda()
    op = SelectiveScan(S, max(lengths), D, N, groups=G, dtype=dtype, softplus=softplus)
    op.bind(u=on(u), delta=ddelta_, A=on(A), B=dB_, C=dC_, out=out, D=on(skips), delta_bias=on(b), z=on(z), initial_state=state if initial else None,
            final_state=state, offsets=offsets if packed else None, slots=where.to(torch.int32).cuda() if slots else None)
    op.run()
    torch.cuda.synchronize()

    def of(k):
        p = parts[k]
        return dict(u=u[p], delta=delta[p], A=A, B=B[p].reshape(-1, G, N), C=C[p].reshape(-1, G, N), D=skips, delta_bias=b, z=None if z is None else z[p],
                    softplus=softplus, initial=before[where[k]] if initial else None)

    some = range(S) if S < 20 else (0, S // 2, S - 1)
    for k in some:
        want, final = ref.scan(**of(k))
        size, most = ref.scan(**of(k), magnitudes=True)
        operations = 2 * lengths[k] + N + 12
        close(f"out of {k}", out[parts[k]], want, size, operations, T)
        close(f"final state of {k}", state[where[k]], final, most, operations)
    assert torch.all(out[rows:] == 7.0)
    others = [p for p in range(places) if p not in where.tolist()]
    assert torch.equal(state[others].cpu(), before[others])
    again = out.clone()
    state.copy_(before)
    op.run()
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    if slots or S >= 20:
        return
    dout, dfinal = r(rows + spare, D).to(T), r(S, D, N)
    grads = {n: torch.full((rows + spare, w), 7.0, dtype=T).cuda() for n, w in (("u", D), ("delta", D), ("z", D), ("B", G * N), ("C", G * N))}
    if not gate:
        del grads["z"]
    grads.update(A=torch.full((D, N), 7.0).cuda(), D=torch.full((D,), 7.0).cuda(), delta_bias=torch.full((D,), 7.0).cuda(), initial_state=torch.full((S, D, N), 7.0).cuda())
    op.bind(u=on(u), delta=ddelta_, A=on(A), B=dB_, C=dC_, D=on(skips), delta_bias=on(b), z=on(z), initial_state=before.cuda() if initial else None,
            offsets=offsets if packed else None)
    op.bind_gradients(out=on(dout), final_state=on(dfinal), **grads)
    op.backward()
    torch.cuda.synchronize()
    sums, sizes = dict(A=0, D=0, delta_bias=0), dict(A=0, D=0, delta_bias=0)
    for k, p in enumerate(parts):
        want, size = (ref.scan(**of(k), dout=dout[p], dfinal=dfinal[k], magnitudes=m) for m in (False, True))
        operations = 4 * lengths[k] + N + 40
        for n in ("u", "delta", "z", "B", "C"):
            if n in grads:
                # (B's and C's are sums over a group's channels as well: 6 levels in a wavefront, then tile by tile)
                more = 6 + -(-D // (64 * G)) if n in "BC" else 0
                close(f"d{n} of {k}", grads[n][p], want[n].reshape(-1, grads[n].shape[1]), size[n].reshape(-1, grads[n].shape[1]), operations + more, T)
        close(f"dinitial of {k}", grads["initial_state"][k], want["initial_state"], size["initial_state"], operations)
        for n in sums:
            sums[n], sizes[n] = sums[n] + want[n], sizes[n] + size[n]
    for n in sums:
        close(f"d{n}", grads[n], sums[n], sizes[n], 4 * max(lengths) + N + 80)      # (32 rows in 32 bits, then in 64)
    for n in ("u", "delta", "z", "B", "C"):
        if n in grads:
            assert torch.all(grads[n][rows:] == 7.0), n
    first = {n: g.clone() for n, g in grads.items()}
    op.backward()
    torch.cuda.synchronize()
    assert all(torch.equal(first[n], g) for n, g in grads.items())


@pytest.mark.parametrize("lengths, channels, states, groups, dtype, packed", [
    ([40, 40], 130, 16, 2, "bfloat16", False),          # (65 channels a group: a whole tile and one of a single lane)
    ([150], 390, 5, 3, "float32", False), ([70, 0, 1, 90], 260, 16, 2, "float32", True), ([33], 260, 20, 2, "float16", False),
    ([1, 1], 390, 16, 3, "bfloat16", False), ([300], 258, 33, 2, "float32", False)])
def test_groups_of_several_tiles_of_channels(lengths, channels, states, groups, dtype, packed):
    test_selective_scan(lengths, channels, states, groups, dtype, True, True, True, True, packed, False, True)


@pytest.mark.parametrize("states", [7, 16, 40])
def test_gradients_asked_for_one_by_one(states):
    """Whichever are asked for, they are the same, and nothing else is written."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, S, n, D, N, K = generator(states), 2, 75, 66, states, 4
    on = lambda *shape: r(*shape).cuda()
    s = SelectiveScan(S, n, D, N, softplus=True)
    s.bind(u=on(S, n, D), delta=on(S, n, D), A=-torch.rand(D, N).cuda(), B=on(S, n, N), C=on(S, n, N), D=on(D), delta_bias=on(D), z=on(S, n, D), initial_state=on(S, D, N))
    c = CausalConvolution(S, n, D, K, silu=True)
    c.bind(x=on(S, n, D), weight=on(D, K), bias=on(D), initial_state=on(S, K - 1, D))
    row = (S, n, D)
    for op, shapes in ((s, dict(u=row, delta=row, z=row, A=(D, N), B=(S, n, N), C=(S, n, N), D=(D,), delta_bias=(D,), initial_state=(S, D, N))),
                       (c, dict(x=row, weight=(D, K), bias=(D,), initial_state=(S, K - 1, D)))):
        dout = on(S, n, D)
        every = {k: torch.zeros(shape).cuda() for k, shape in shapes.items()}
        op.bind_gradients(out=dout, **every)
        op.backward()
        torch.cuda.synchronize()
        for name, shape in shapes.items():
            one = torch.zeros(shape).cuda()
            op.bind_gradients(out=dout, **{name: one})
            op.backward()
            torch.cuda.synchronize()
            assert torch.equal(one, every[name]) and one.abs().sum() > 0, name
        op.bind_gradients(out=dout)
        op.backward()
        torch.cuda.synchronize()


def test_tokens_continue_a_prompt_and_padding_is_left_alone():
    """A prompt's state, then one row at a time, gives what the whole sequence gives; sequences whose slot is none are neither read nor written."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, n, D, N, K = generator(5), 90, 72, 16, 4
    x, delta, B, C, z = r(n, D), r(n, D), r(n, N), r(n, N), r(n, D)
    weight, bias, A = r(D, K), r(D), -torch.exp(r(D, N) * 0.3)
    whole, conv = torch.empty(n, D).cuda(), torch.empty(n, D).cuda()
    c = CausalConvolution(1, n, D, K, silu=True)
    c.bind(x=x.cuda(), weight=weight.cuda(), bias=bias.cuda(), out=conv)
    c.run()
    s = SelectiveScan(1, n, D, N, softplus=True)
    s.bind(u=conv, delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), z=z.cuda(), out=whole)
    s.run()
    pool, window = torch.full((5, D, N), 9.0).cuda(), torch.full((5, K - 1, D), 9.0).cuda()
    slots = torch.tensor([3], dtype=torch.int32).cuda()
    at, got, mid = 70, torch.empty(n, D).cuda(), torch.empty(n, D).cuda()
    c = CausalConvolution(1, at, D, K, silu=True)
    c.bind(x=x[:at].cuda(), weight=weight.cuda(), bias=bias.cuda(), out=mid[:at], final_state=window, slots=slots)
    c.run()
    s = SelectiveScan(1, at, D, N, softplus=True)
    s.bind(u=mid[:at], delta=delta[:at].cuda(), A=A.cuda(), B=B[:at].cuda(), C=C[:at].cuda(), z=z[:at].cuda(), out=got[:at], final_state=pool, slots=slots)
    s.run()
    # a padded batch: the running sequence between two that are none
    slots = torch.tensor([-1, 3, 5], dtype=torch.int32).cuda()
    wide = lambda t, i: torch.stack([torch.full_like(t[i], float("nan")), t[i], torch.full_like(t[i], float("nan"))]).cuda()
    one, two = torch.full((3, D), 4.0).cuda(), torch.full((3, D), 4.0).cuda()
    c, s = CausalConvolution(3, 1, D, K, silu=True), SelectiveScan(3, 1, D, N, softplus=True)
    for t in range(at, n):
        c.bind(x=wide(x, t), weight=weight.cuda(), bias=bias.cuda(), out=one, initial_state=window, final_state=window, slots=slots)
        c.run()
        s.bind(u=one, delta=wide(delta, t), A=A.cuda(), B=wide(B, t), C=wide(C, t), z=wide(z, t), out=two, initial_state=pool, final_state=pool, slots=slots)
        s.run()
        mid[t], got[t] = one[1], two[1]
    torch.cuda.synchronize()
    assert torch.equal(mid, conv)
    size = ref.scan(conv.cpu(), delta, A, B.reshape(n, 1, N), C.reshape(n, 1, N), z=z, softplus=True, magnitudes=True)[0]
    close("tokens", got, whole.cpu().double(), size, 2 * (2 * n + N + 12))          # (both sides are off by as much)
    assert torch.all(one[[0, 2]] == 4.0) and torch.all(two[[0, 2]] == 4.0)
    assert torch.all(pool[[0, 1, 2, 4]] == 9.0) and torch.all(window[[0, 1, 2, 4]] == 9.0)


def test_what_is_not_finite_stays_where_it_belongs():
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, n, D, N, K = generator(8), 40, 70, 9, 3
    x, weight = r(n, D), r(D, K)
    x[20, 5], x[11, 66] = float("inf"), float("nan")
    out = torch.empty(n, D).cuda()
    c = CausalConvolution(1, n, D, K)
    c.bind(x=x.cuda(), weight=weight.cuda(), out=out)
    c.run()
    bad = torch.zeros(n, D, dtype=torch.bool)
    bad[20:23, 5] = bad[11:14, 66] = True
    assert torch.equal(~torch.isfinite(out.cpu()), bad)
    s = SelectiveScan(1, n, D, N, softplus=True)
    args = dict(u=x.cuda(), delta=r(n, D).cuda(), A=-torch.rand(D, N).cuda(), B=torch.rand(n, N).cuda() + 0.1, C=torch.rand(n, N).cuda() + 0.1)
    s.bind(out=out, **args)
    s.run()
    bad[:] = False
    bad[20:, 5] = bad[11:, 66] = True
    assert torch.equal(~torch.isfinite(out.cpu()), bad)
    # a step in time that closes a unit (exp(dt A) = 0) and one that leaves it as it is (dt = 0)
    args["u"] = r(n, D).cuda()
    args["delta"] = torch.tensor([0.0, 1e4]).repeat(n * D // 2).view(n, D).cuda()
    s = SelectiveScan(1, n, D, N)
    final = torch.empty(1, D, N).cuda()
    s.bind(out=out, final_state=final, initial_state=torch.ones(1, D, N).cuda(), **args)
    s.run()
    assert torch.all(final[0, 0::2] == 1.0) and torch.isfinite(out).all()


@pytest.mark.parametrize("length", [1, 30, 500])
@pytest.mark.parametrize("states", [1, 5, 8, 11, 20, 40])
def test_what_is_infinite_stays_infinite(states, length):
    """An infinite input or state gives the infinities of the formula, whatever the number of states (a wavefront has registers for 8 or 16 of them)."""
    from genn_amd.sequence import SelectiveScan
    r, D, N = generator(states + length), 70, states
    u, delta, B, C = r(length, D), torch.rand(length, D) * 0.02 + 0.01, torch.rand(length, N) + 0.1, torch.rand(length, N) + 0.1
    A, initial = -torch.rand(D, N), r(D, N)
    u[min(12, length - 1), 3], u[0, 65], delta[length // 2, 68], u[length // 2, 68] = float("inf"), float("-inf"), float("inf"), 1.0
    initial[7, 0], initial[9, N - 1] = float("inf"), float("-inf")
    out, final = torch.empty(length, D).cuda(), torch.empty(1, D, N).cuda()
    s = SelectiveScan(1, length, D, N)
    s.bind(u=u.cuda(), delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), D=torch.ones(D).cuda(), out=out, initial_state=initial.cuda().view(1, D, N), final_state=final)
    s.run()
    torch.cuda.synchronize()
    args = dict(u=u, delta=delta, A=A, B=B.view(length, 1, N), C=C.view(length, 1, N), D=torch.ones(D), initial=initial)
    want = ref.scan(**args)
    sizes = ref.scan(magnitudes=True, **args)
    assert torch.isinf(want[0][-1, [3, 7, 9, 65, 68]]).all() and torch.isfinite(want[0][:, 10:60]).all()
    for got, w, size in ((out, want[0], sizes[0]), (final[0], want[1], sizes[1])):
        got, odd = got.cpu().double(), ~torch.isfinite(w)
        assert torch.allclose(got[odd], w[odd], rtol=0, atol=0, equal_nan=True)
        assert torch.isfinite(got[~odd]).all()
        close("finite ones", got[~odd], w[~odd], size[~odd], 2 * length + N + 12)


@pytest.mark.parametrize("length", [1, 30, 500])
@pytest.mark.parametrize("states", [8, 20])
def test_an_infinite_input_without_a_direct_path(states, length):
    """Without D the outputs have no share of u but by the states, which are infinite from there on."""
    from genn_amd.sequence import SelectiveScan
    r, D, N = generator(states + length), 70, states
    u, delta, B, C = r(length, D), torch.rand(length, D) * 0.02 + 0.01, torch.rand(length, N) + 0.1, torch.rand(length, N) + 0.1
    A = -torch.rand(D, N)
    at = min(12, length - 1)
    u[at, 3], u[at, 66] = float("inf"), float("-inf")
    out = torch.empty(length, D).cuda()
    s = SelectiveScan(1, length, D, N)
    s.bind(u=u.cuda(), delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), out=out)
    s.run()
    torch.cuda.synchronize()
    got = out.cpu()
    assert torch.all(got[at:, 3] == float("inf")) and torch.all(got[at:, 66] == float("-inf"))
    got[at:, [3, 66]] = 0.0
    assert torch.isfinite(got).all()


def test_an_infinite_state_outlasts_decays_that_round_to_zero():
    """A row's decay is e^-16, that of a chunk of rows is none in 32 bits: what is infinite stays so row by row, and over chunks."""
    from genn_amd.sequence import SelectiveScan
    n, D, N = 600, 64, 16
    initial = torch.ones(1, D, N)
    initial[0, 5, 3], initial[0, 6, 0] = float("inf"), float("-inf")
    one = lambda *shape: torch.ones(*shape).cuda()
    out, final = torch.empty(1, n, D).cuda(), torch.empty(1, D, N).cuda()
    s = SelectiveScan(1, n, D, N)
    s.bind(u=one(1, n, D), delta=one(1, n, D), A=-16 * one(D, N), B=one(1, n, N), C=one(1, n, N), out=out, initial_state=initial.cuda(), final_state=final)
    assert s.workspace_bytes > 0            # (in chunks)
    s.run()
    torch.cuda.synchronize()
    out, final = out[0].cpu(), final[0].cpu()
    assert torch.all(out[:, 5] == float("inf")) and torch.all(out[:, 6] == float("-inf"))
    assert final[5, 3] == float("inf") and final[6, 0] == float("-inf")
    out[:, 5:7], final[5, 3], final[6, 0] = 0.0, 0.0, 0.0
    assert torch.isfinite(out).all() and torch.isfinite(final).all()


@pytest.mark.parametrize("largest", [1e20, 3e38])
def test_a_large_state_that_is_forgotten_leaves_nothing(largest):
    """The decay of the first chunk is none in 32 bits: what was there before is not in the states behind it, however large."""
    from genn_amd.sequence import SelectiveScan
    n, D, N = 600, 64, 16
    r = generator(15)
    u, B, C, A, delta, initial = r(n, D) * 1e-5, r(n, N), r(n, N), -8 - torch.rand(D, N), torch.full((n, D), 1e-3), torch.full((D, N), largest)
    delta[:24] = 1.0            # (e^-192 and less, and then hardly any)
    out, final = torch.empty(1, n, D).cuda(), torch.empty(1, D, N).cuda()
    s = SelectiveScan(1, n, D, N)
    s.bind(u=u.cuda(), delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), out=out, initial_state=initial.cuda().view(1, D, N), final_state=final)
    assert s.workspace_bytes > 0
    s.run()
    torch.cuda.synchronize()
    args = dict(u=u, delta=delta, A=A, B=B.view(n, 1, N), C=C.view(n, 1, N), initial=initial)
    want, size = ref.scan(**args), ref.scan(magnitudes=True, **args)
    close("final state", final[0], want[1], size[1], 2 * n + N + 12)
    close("out", out[0], want[0], size[0], 2 * n + N + 12)


@pytest.mark.parametrize("lengths", [[5], [0, 13, 0], [0, 500, 3, 0]])
def test_units_that_forget_everything(lengths):
    """A = -infinity: a row's state is what comes in with it; sequences without rows keep theirs.  Also one whose product with log2(e) is infinite."""
    from genn_amd.sequence import SelectiveScan
    S, D, N = len(lengths), 20, 5
    parts, offsets = split(lengths)
    rows, r = sum(lengths), generator(sum(lengths))
    u, delta, B, C, dout = r(rows, D), torch.rand(rows, D) + 0.1, r(rows, N), r(rows, N), r(rows, D)
    A, initial, dfinal = -torch.rand(D, N), r(S, D, N), r(S, D, N)
    A[3], A[7, 2], A[11, 4] = float("-inf"), float("-inf"), -3e38
    grads = {k: torch.empty(rows, w).cuda() for k, w in (("u", D), ("B", N), ("C", N))}
    grads.update(A=torch.empty(D, N).cuda(), initial_state=torch.empty(S, D, N).cuda())
    out, final = torch.empty(rows, D).cuda(), torch.empty(S, D, N).cuda()
    s = SelectiveScan(S, max(lengths), D, N)
    s.bind(u=u.cuda(), delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), out=out, initial_state=initial.cuda(), final_state=final, offsets=offsets)
    s.run()
    s.bind_gradients(out=dout.cuda(), final_state=dfinal.cuda(), **grads)
    s.backward()
    torch.cuda.synchronize()
    dA, sizeA = 0, 0
    for k, p in enumerate(parts):
        args = dict(u=u[p], delta=delta[p], A=A, B=B[p].view(-1, 1, N), C=C[p].view(-1, 1, N), initial=initial[k])
        want, size = (ref.scan(magnitudes=m, **args) for m in (False, True))
        close(f"out of {k}", out[p], want[0], size[0], 2 * lengths[k] + N + 12)
        close(f"final state of {k}", final[k], want[1], size[1], 2 * lengths[k] + N + 12)
        want, size = (ref.scan(magnitudes=m, dout=dout[p], dfinal=dfinal[k], **args) for m in (False, True))
        for name in ("u", "B", "C"):
            close(f"d{name} of {k}", grads[name][p], want[name].reshape(-1, grads[name].shape[1]), size[name].reshape(-1, grads[name].shape[1]), 4 * lengths[k] + N + 48)
        close(f"dinitial of {k}", grads["initial_state"][k], want["initial_state"], size["initial_state"], 4 * lengths[k] + N + 40)
        dA, sizeA = dA + want["A"], sizeA + size["A"]
    close("dA", grads["A"], dA, sizeA, 4 * max(lengths) + N + 80)


@pytest.mark.parametrize("sequences, length", [(0, 5), (3, 0)])
def test_nothing_to_do_leaves_states_and_gives_zero_gradients(sequences, length):
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    D, N, K = 6, 4, 3
    rows = lambda w: torch.zeros(sequences, length, w).cuda()
    first, last, window, moved = torch.rand(sequences, D, N).cuda(), torch.zeros(sequences, D, N).cuda(), torch.rand(sequences, K - 1, D).cuda(), torch.zeros(sequences, K - 1, D).cuda()
    weight, A, grads = torch.rand(D, K).cuda(), -torch.rand(D, N).cuda(), {}
    c, s = CausalConvolution(sequences, length, D, K), SelectiveScan(sequences, length, D, N)
    c.bind(x=rows(D), weight=weight, out=rows(D), initial_state=window, final_state=moved)
    s.bind(u=rows(D), delta=rows(D), A=A, B=rows(N), C=rows(N), out=rows(D), initial_state=first, final_state=last)
    c.run()
    s.run()
    dlast, dmoved, dfirst, dwindow = torch.rand(sequences, D, N).cuda(), torch.rand(sequences, K - 1, D).cuda(), torch.zeros(sequences, D, N).cuda(), torch.zeros(sequences, K - 1, D).cuda()
    dA, dw = torch.ones(D, N).cuda(), torch.ones(D, K).cuda()
    c.bind_gradients(out=rows(D), x=rows(D), weight=dw, final_state=dmoved, initial_state=dwindow)
    s.bind_gradients(out=rows(D), u=rows(D), A=dA, B=rows(N), final_state=dlast, initial_state=dfirst)
    c.backward()
    s.backward()
    torch.cuda.synchronize()
    for got, want in ((last, first), (moved, window), (dfirst, dlast), (dwindow, dmoved)):
        assert torch.equal(got, want)
    assert torch.all(dA == 0) and torch.all(dw == 0)


@pytest.mark.parametrize("length", [4, 500])
def test_packed_arrays_without_sequences(length):
    """Rows that belong to no sequence are left alone, and sums over sequences are zero."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    rows, D, N, K = 300, 20, 6, 3
    full = lambda *shape: torch.full(shape, 7.0).cuda()
    offsets = torch.zeros(1, dtype=torch.int32).cuda()
    c, s = CausalConvolution(0, length, D, K), SelectiveScan(0, length, D, N)
    out = {k: full(rows, D) for k in ("c", "s", "x", "u", "delta", "z")}
    sums = {k: full(*shape) for k, shape in (("weight", (D, K)), ("bias", (D,)), ("A", (D, N)), ("D", (D,)), ("delta_bias", (D,)))}
    dB, dC = full(rows, N), full(rows, N)
    c.bind(x=full(rows, D), weight=full(D, K), bias=full(D), out=out["c"], offsets=offsets)
    s.bind(u=full(rows, D), delta=full(rows, D), A=full(D, N), B=full(rows, N), C=full(rows, N), D=full(D), delta_bias=full(D), z=full(rows, D), out=out["s"], offsets=offsets)
    c.bind_gradients(out=full(rows, D), x=out["x"], weight=sums["weight"], bias=sums["bias"])
    s.bind_gradients(out=full(rows, D), u=out["u"], delta=out["delta"], z=out["z"], B=dB, C=dC, A=sums["A"], D=sums["D"], delta_bias=sums["delta_bias"])
    for op in (c, s):
        op.run()
        op.backward()
    torch.cuda.synchronize()
    assert all(torch.all(t == 7.0) for t in (*out.values(), dB, dC))
    assert all(torch.all(t == 0.0) for t in sums.values())


def test_another_current_device_is_refused():
    """(the descriptors say that their arrays are the second device's, while the first is current)"""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    t, A = torch.ones(1, 3, 4).cuda(), -torch.ones(4, 4).cuda()
    out = torch.zeros(1, 3, 4).cuda()
    c, s = CausalConvolution(1, 3, 4, 4), SelectiveScan(1, 3, 4, 4)
    c.bind(x=t, weight=A, out=out)
    s.bind(u=t, delta=t, A=A, B=t, C=t, out=out)
    for op in (c, s):
        op.bind_gradients(out=t)
        assert op._descriptor.sequences.device == 1
        op._descriptor.sequences.device = 2
        for call in (op.run, op.backward):
            with pytest.raises(_abi.GennmiError, match="on device 1"):
                call()
    torch.cuda.synchronize()
    assert torch.all(out == 0)


def test_a_state_of_nothing_stays_nothing_however_fast_units_grow():
    """Units with A > 0, no input for 500 rows and then some: a chunk's growth is infinite in fp32, a state of zero stays zero."""
    from genn_amd.sequence import SelectiveScan
    n, D, N = 520, 64, 16
    u = torch.zeros(1, n, D)
    u[:, 500:] = 1.0
    B, A, delta, out, final = torch.ones(1, n, N).cuda(), torch.ones(D, N).cuda(), torch.full((1, n, D), 3.0).cuda(), torch.empty(1, n, D).cuda(), torch.empty(1, D, N).cuda()
    delta[:, 500:] = 0.5
    s = SelectiveScan(1, n, D, N)
    s.bind(u=u.cuda(), delta=delta, A=A, B=B, C=B, out=out, final_state=final)
    assert s.workspace_bytes > 0
    s.run()
    torch.cuda.synchronize()
    args = dict(u=u[0], delta=delta[0].cpu(), A=A.cpu(), B=B[0].cpu().view(n, 1, N), C=B[0].cpu().view(n, 1, N))
    want, last = ref.scan(**args)
    close("out", out[0], want, want, 2 * 20 + N + 12 + 4 * 10)             # (growth e^0.5 a row, 20 rows: what exponents of up to 10 are off by as well)
    close("final state", final[0], last, last, 2 * 20 + N + 12 + 4 * 10)


def test_rows_behind_the_longest_that_is_allowed_are_left_alone():
    """Packed sequences of 70 and 3 rows where `length` is 40: the first is cut."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, rows, D, N, K, most = generator(12), 73, 20, 16, 4, 40
    x, delta, B, C, dout = r(rows, D), r(rows, D).abs(), r(rows, N), r(rows, N), r(rows, D)
    A, weight = -torch.rand(D, N), r(D, K)
    offsets = torch.tensor([0, 70, 73], dtype=torch.int32).cuda()
    mine, left = [slice(0, 40), slice(70, 73)], slice(40, 70)
    full = lambda w: torch.full((rows, w), 7.0).cuda()
    out, dx, dB, dC, dw, dA = full(D), full(D), full(N), full(N), torch.empty(D, K).cuda(), torch.empty(D, N).cuda()
    c, s = CausalConvolution(2, most, D, K), SelectiveScan(2, most, D, N)
    c.bind(x=x.cuda(), weight=weight.cuda(), out=out, offsets=offsets)
    c.bind_gradients(out=dout.cuda(), x=dx, weight=dw)
    c.run()
    c.backward()
    torch.cuda.synchronize()
    want = [ref.causal_conv(x[p], weight, None, False)[0] for p in mine]
    size = [ref.causal_conv(x[p], weight, None, False, magnitudes=True)[0] for p in mine]
    grads, sizes = ([ref.causal_conv(x[p], weight, None, False, dout=dout[p], magnitudes=m) for p in mine] for m in (False, True))
    for k, p in enumerate(mine):
        close("conv", out[p], want[k], size[k], K + 8)
        close("dx", dx[p], grads[k][0], sizes[k][0], K + 8)
    close("dweight", dw, grads[0][1] + grads[1][1], sizes[0][1] + sizes[1][1], K + 64 + 20)
    assert torch.all(out[left] == 7.0) and torch.all(dx[left] == 7.0)
    out.fill_(7.0)
    dx.fill_(7.0)
    s.bind(u=x.cuda(), delta=delta.cuda(), A=A.cuda(), B=B.cuda(), C=C.cuda(), out=out, offsets=offsets)
    s.bind_gradients(out=dout.cuda(), u=dx, A=dA, B=dB, C=dC)
    s.run()
    s.backward()
    torch.cuda.synchronize()
    of = lambda p: dict(u=x[p], delta=delta[p], A=A, B=B[p].view(-1, 1, N), C=C[p].view(-1, 1, N))
    grads, sizes = ([ref.scan(**of(p), dout=dout[p], magnitudes=m) for p in mine] for m in (False, True))
    for k, p in enumerate(mine):
        close("scan", out[p], ref.scan(**of(p))[0], ref.scan(**of(p), magnitudes=True)[0], 2 * most + N + 12)
        close("du", dx[p], grads[k]["u"], sizes[k]["u"], 4 * most + N + 40)
        for name, got in (("B", dB), ("C", dC)):
            close(f"d{name}", got[p], grads[k][name].view(-1, N), sizes[k][name].view(-1, N), 4 * most + N + 47)
    close("dA", dA, grads[0]["A"] + grads[1]["A"], sizes[0]["A"] + sizes[1]["A"], 4 * most + N + 80)
    for t in (out, dx, dB, dC):
        assert torch.all(t[left] == 7.0)


def test_gradients_of_a_long_convolution():
    """Enough rows for the longest chunks; a few channels of it against the restatement."""
    from genn_amd.sequence import CausalConvolution
    S, n, D, K = 4, 2100, 2048, 4
    x, dout, dx = (torch.randn(S, n, D, device="cuda").to(torch.bfloat16) for _ in range(3))
    weight, bias, dw, db = torch.randn(D, K, device="cuda"), torch.randn(D, device="cuda"), torch.empty(D, K, device="cuda"), torch.empty(D, device="cuda")
    c = CausalConvolution(S, n, D, K, dtype="bfloat16", silu=True)
    c.bind(x=x, weight=weight, bias=bias)
    c.bind_gradients(out=dout, x=dx, weight=dw, bias=db)
    c.backward()
    torch.cuda.synchronize()
    some = torch.tensor([0, 1, 777, 2047])
    take = lambda t: t[..., some.cuda()].cpu()
    w, b, sums, sizes = weight[some.cuda()].cpu(), bias[some.cuda()].cpu(), [0, 0], [0, 0]
    for k in range(S):
        args = (take(x[k]), w, b, True, None, take(dout[k]))
        want, size = ref.causal_conv(*args), ref.causal_conv(*args, magnitudes=True)
        close(f"dx of {k}", take(dx[k]), want[0], size[0], 2 * K + 16, torch.bfloat16)
        for i in (0, 1):
            sums[i], sizes[i] = sums[i] + want[i + 1], sizes[i] + size[i + 1]
    close("dweight", dw[some.cuda()], sums[0], sizes[0], K + 64 + 20)        # (sums of 64 rows, then in 64 bits)
    close("dbias", db[some.cuda()], sums[1], sizes[1], K + 64 + 20)


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_any_alignment_gives_the_same(shift):
    """Rows that begin anywhere take the element-wise accesses: same sums."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, n, D, N, K = generator(2), 35, 68, 12, 4

    def placed(t, dtype=torch.bfloat16):
        room = torch.empty(t.numel() + 8, dtype=dtype).cuda()
        view = room[shift:shift + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    x, delta, B, C, weight, A, state = r(n, D), r(n, D), r(n, N), r(n, N), r(D, K), -torch.rand(D, N), r(1, D, N)
    results = []
    for place in (lambda t, dtype=torch.bfloat16: t.to(dtype).cuda(), placed):
        out, final, scanned = place(torch.zeros(n, D)), place(torch.zeros(1, K - 1, D)), place(torch.zeros(n, D))
        c = CausalConvolution(1, n, D, K, dtype="bfloat16", silu=True)
        c.bind(x=place(x), weight=place(weight, torch.float32), out=out, final_state=final)
        c.run()
        s = SelectiveScan(1, n, D, N, dtype="bfloat16", softplus=True)
        h = place(state, torch.float32)
        s.bind(u=out, delta=place(delta), A=place(A, torch.float32), B=place(B), C=place(C), out=scanned, initial_state=h, final_state=h)
        s.run()
        token, g = place(torch.zeros(1, D)), place(state, torch.float32)
        t = SelectiveScan(1, 1, D, N, dtype="bfloat16", softplus=True)
        t.bind(u=out[:1], delta=place(delta[:1]), A=place(A, torch.float32), B=place(B[:1]), C=place(C[:1]), out=token, initial_state=g, final_state=g)
        t.run()
        results.append([a.float().cpu() for a in (out, final, scanned, h, token, g)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_offsets_beyond_32_bits():
    """The third row of a sequence, and the second sequence, lie more than 2^32 elements behind the first."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    D, N, K, stride = 64, 4, 3, (1 << 31) + 64
    room = torch.empty(2 * stride + 1024, dtype=torch.bfloat16, device="cuda")
    r = generator(4)
    x = r(3, D).to(torch.bfloat16)
    far = torch.as_strided(room, (1, 3, D), (0, stride, 1))
    far[0].copy_(x)
    weight, out = r(D, K).cuda(), torch.empty(3, D, dtype=torch.bfloat16).cuda()
    c = CausalConvolution(1, 3, D, K, dtype="bfloat16")
    c.bind(x=far, weight=weight, out=out)
    c.run()
    want, _ = ref.causal_conv(x, weight.cpu(), None, False)
    close("conv", out, want, ref.causal_conv(x, weight.cpu(), None, False, magnitudes=True)[0], K + 8, torch.bfloat16)
    A, B = -torch.rand(D, N), r(3, N).to(torch.bfloat16)
    out.copy_(torch.zeros(3, D))
    s = SelectiveScan(1, 3, D, N, dtype="bfloat16")
    s.bind(u=far, delta=far, A=A.cuda(), B=B.cuda(), C=B.cuda(), out=out)
    s.run()
    args = dict(u=x, delta=x, A=A, B=B.view(3, 1, N), C=B.view(3, 1, N))
    close("scan", out, ref.scan(**args)[0], ref.scan(**args, magnitudes=True)[0], 2 * 3 + N + 12, torch.bfloat16)


def test_rows_and_sequences_beyond_32_bits_forwards_and_back():
    """Two sequences of three rows, more than 2^31 elements from row to row and 2^32 from sequence to sequence, all arrays side by side in one."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    S, n, D, N, K, stride = 2, 3, 64, 16, 3, (1 << 31) + 64
    room = torch.empty(S * n * stride, dtype=torch.bfloat16, device="cuda")
    r, used = generator(14), [0]

    def far(width, values=None):
        at = torch.as_strided(room, (S, n, width), (n * stride, stride, 1), used[0])
        used[0] += width
        if values is not None:
            for k in range(S):
                at[k].copy_(values[k])
        return at

    give = {k: r(S, n, w).to(torch.bfloat16) for k, w in (("x", D), ("delta", D), ("B", N), ("C", N), ("z", D), ("dout", D))}
    on = {k: far(v.shape[-1], v) for k, v in give.items()}
    weight, A, initial = r(D, K), -torch.rand(D, N), r(S, D, N)
    back = lambda t: torch.stack([t[k].clone() for k in range(S)]).cpu()
    c, s = CausalConvolution(S, n, D, K, dtype="bfloat16", silu=True), SelectiveScan(S, n, D, N, dtype="bfloat16", softplus=True)
    out, dx, dw = far(D), far(D), torch.empty(D, K).cuda()
    c.bind(x=on["x"], weight=weight.cuda(), out=out)
    c.bind_gradients(out=on["dout"], x=dx, weight=dw)
    scanned, final, dA = far(D), torch.empty(S, D, N).cuda(), torch.empty(D, N).cuda()
    grads = {k: far(w) for k, w in (("u", D), ("delta", D), ("z", D), ("B", N), ("C", N))}
    s.bind(u=on["x"], delta=on["delta"], A=A.cuda(), B=on["B"], C=on["C"], z=on["z"], out=scanned, initial_state=initial.cuda(), final_state=final)
    s.bind_gradients(out=on["dout"], A=dA, **grads)
    for op in (c, s):
        op.run()
        op.backward()
    torch.cuda.synchronize()
    got = {k: back(v) for k, v in dict(out=out, dx=dx, scanned=scanned, **grads).items()}
    dws, dAs = [0, 0], [0, 0]
    for k in range(S):
        args = (give["x"][k], weight, None, True)
        close("conv", got["out"][k], ref.causal_conv(*args)[0], ref.causal_conv(*args, magnitudes=True)[0], K + 8, torch.bfloat16)
        args = (*args, None, give["dout"][k])
        want, size = (ref.causal_conv(*args, magnitudes=m) for m in (False, True))
        close("dx", got["dx"][k], want[0], size[0], 2 * K + 16, torch.bfloat16)
        dws = [dws[0] + want[1], dws[1] + size[1]]
        args = dict(u=give["x"][k], delta=give["delta"][k], A=A, B=give["B"][k].view(n, 1, N), C=give["C"][k].view(n, 1, N), z=give["z"][k], softplus=True, initial=initial[k])
        want, size = (ref.scan(**args, magnitudes=m) for m in (False, True))
        close("scan", got["scanned"][k], want[0], size[0], 2 * n + N + 12, torch.bfloat16)
        close("final state", final[k], want[1], size[1], 2 * n + N + 12)
        want, size = (ref.scan(**args, dout=give["dout"][k], magnitudes=m) for m in (False, True))
        for name in grads:
            close(f"d{name}", got[name][k], want[name].reshape(n, -1), size[name].reshape(n, -1), 4 * n + N + 47, torch.bfloat16)
        dAs = [dAs[0] + want["A"], dAs[1] + size["A"]]
    close("dweight", dw, *dws, K + 16 + 20)
    close("dA", dA, *dAs, 4 * n + N + 80)


def test_streams_graphs_and_workspaces():
    """On a stream of the caller's, and captured there: every replay gives the eager call's bits, with eager work of the same operator between the
    replays.  A captured call needs a workspace of its own."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, n, D, N, K = generator(6), 300, 130, 16, 4
    make = lambda *shape: r(*shape).to(torch.bfloat16).cuda()
    x, delta, B, C, z, dout = make(n, D), make(n, D), make(n, N), make(n, N), make(n, D), make(n, D)
    weight, A = r(D, K).cuda(), -torch.rand(D, N).cuda()
    mid, out, du, dx = (torch.zeros(n, D, dtype=torch.bfloat16).cuda() for _ in range(4))
    dA, dw = torch.zeros(D, N).cuda(), torch.zeros(D, K).cuda()
    c, s = CausalConvolution(1, n, D, K, dtype="bfloat16", silu=True), SelectiveScan(1, n, D, N, dtype="bfloat16", softplus=True)
    c.bind(x=x, weight=weight, out=mid)
    s.bind(u=mid, delta=delta, A=A, B=B, C=C, z=z, out=out)
    assert s.workspace_bytes > 0
    s.bind_gradients(out=dout, u=du, A=dA)
    c.bind_gradients(out=du, x=dx, weight=dw)
    spaces = [torch.empty(b, dtype=torch.uint8).cuda() for b in (s.workspace_bytes, s.backward_workspace_bytes, c.backward_workspace_bytes)]

    def run(stream, workspaces=(None, None, None)):
        c.run(stream)
        s.run(stream, workspaces[0])
        s.backward(stream, workspaces[1])
        c.backward(stream, workspaces[2])

    results = (mid, out, du, dx, dA, dw)
    run(0)
    torch.cuda.synchronize()
    want = [t.clone() for t in results]
    assert all(float(t.float().abs().sum()) > 0 for t in want)
    side = torch.cuda.Stream()
    for t in results:
        t.zero_()
    side.wait_stream(torch.cuda.current_stream())
    run(side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        stream = torch.cuda.current_stream().cuda_stream
        with pytest.raises(ValueError, match="captured"):
            s.run(stream)
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
        assert all(torch.equal(a, b) for a, b in zip(results, want)), k
    # other inputs in the same place
    x.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in results]
    run(0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results, got)) and not torch.equal(got[1], want[1])


def test_a_bind_that_is_refused_leaves_the_one_before():
    """Also where the refused arrays were packed and those before are not: gradients are bound to those before."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    r, S, n, D, N, K = generator(3), 2, 9, 6, 4, 3
    on = lambda *shape: r(*shape).cuda()
    offsets = torch.tensor([0, 9, 18], dtype=torch.int32).cuda()
    args = dict(u=on(S, n, D), delta=on(S, n, D).abs(), A=-torch.rand(D, N).cuda(), B=on(S, n, N), C=on(S, n, N), out=on(S, n, D))
    flat = {k: v.view(S * n, -1) if v.dim() == 3 else v for k, v in args.items()}
    dout = on(S, n, D)
    for op, good, packed, wrong, name, shape in (
            (SelectiveScan(S, n, D, N), args, flat, dict(A=on(D, N + 1)), "A", (D, N)),
            (CausalConvolution(S, n, D, K), dict(x=args["u"], weight=on(D, K), out=on(S, n, D)), dict(x=flat["u"], weight=on(D, K)), dict(weight=on(D, K + 1)), "weight", (D, K))):
        grads = [torch.empty(shape).cuda() for _ in range(2)]
        for k, g in enumerate(grads):
            op.bind(**good)
            if k:
                with pytest.raises(ValueError, match="shape"):
                    op.bind(**{**packed, **wrong}, offsets=offsets)
            op.run()
            op.bind_gradients(out=dout, **{name: g})
            op.backward()
        torch.cuda.synchronize()
        assert torch.equal(*grads) and grads[0].abs().sum() > 0
    # ... and where the library refuses it
    s = SelectiveScan(S, n, D, N)
    s.bind(**args)
    with pytest.raises(_abi.GennmiError, match="sequences overlap"):
        s.bind(**{**args, "out": torch.zeros(n, D).cuda().expand(S, n, D)})
    args["out"].zero_()
    s.run()
    torch.cuda.synchronize()
    assert args["out"].abs().sum() > 0


def test_arrays_of_the_package_and_what_the_layer_refuses():
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    n, D, N, K = 6, 10, 4, 3
    rng = np.random.default_rng(1)
    arrays = {k: Array(int(np.prod(shape)), np.float32) for k, shape in dict(x=(2, n, D), weight=(D, K), out=(2, n, D), final=(2, K - 1, D)).items()}
    for k in ("x", "weight"):
        arrays[k].view[:] = rng.normal(size=arrays[k].count)
        arrays[k].push_to_device()
    c = CausalConvolution(2, n, D, K)
    c.bind(x=arrays["x"], weight=arrays["weight"], out=arrays["out"], final_state=arrays["final"])
    c.run()
    x = torch.from_numpy(arrays["x"].view.copy()).view(2, n, D)
    weight = torch.from_numpy(arrays["weight"].view.copy()).view(D, K)
    got = torch.from_numpy(arrays["out"].pull_from_device().copy()).view(2, n, D)
    for k in range(2):
        close("out", got[k], ref.causal_conv(x[k], weight, None, False)[0], ref.causal_conv(x[k], weight, None, False, magnitudes=True)[0], K + 8)
    assert np.array_equal(arrays["final"].pull_from_device().reshape(2, K - 1, D), x[:, n - K + 1:].numpy())
    t = torch.zeros(2, n, D).cuda()
    w = torch.zeros(D, K).cuda()
    for wrong, error in ((dict(x=t[:, :, :9]), "shape"), (dict(x=t.half()), "holds"), (dict(weight=w.t()), "shape"), (dict(out=t.permute(0, 2, 1)), "shape"),
                         (dict(x=torch.zeros(2, n, 2 * D).cuda()[:, :, ::2]), "neighbours"), (dict(final_state=torch.zeros(2, K, D).cuda()), "shape"),
                         (dict(slots=torch.zeros(2).cuda()), "holds"), (dict(offsets=torch.zeros(2, dtype=torch.int32).cuda()), "shape")):
        with pytest.raises((ValueError, TypeError), match=error):
            c.bind(**{**dict(x=t, weight=w, out=torch.zeros_like(t)), **wrong})
    with pytest.raises(_abi.GennmiError, match="same array"):
        c.bind(x=t, weight=w, out=t)
        c.run()
    for wrong in (dict(length=1 << 31), dict(sequences=-1), dict(channels=1 << 40), dict(taps=-2)):
        with pytest.raises(ValueError, match="below 2"):
            CausalConvolution(**{**dict(sequences=2, length=n, channels=D, taps=K), **wrong})
    s = SelectiveScan(2, n, D, N)
    with pytest.raises(RuntimeError, match="bind"):
        s.run()
    with pytest.raises(ValueError, match="B has shape"):
        s.bind(u=t, delta=t, A=torch.zeros(D, N).cuda(), B=t, C=t, out=torch.zeros_like(t))
    for a in arrays.values():
        a.free()
    with pytest.raises(ValueError, match="freed"):
        c.bind(x=arrays["x"], weight=w, out=torch.zeros_like(t))
