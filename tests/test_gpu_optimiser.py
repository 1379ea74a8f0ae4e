"""The AdamW step through the C ABI against its restatement in 64 bits.

Tolerances: m and v in fp32 are two products and a sum, three roundings of at most 2^-24 of the terms (constants rounded to fp32 add one each): 6 x 2^-24.  A change
of a weight is a quotient of such values with a root, some 16 roundings, and is added to a weight that was scaled: 2^-24 x (2 |w| + 24 |change|), then one
rounding to the weights' type.  Codes and scales of the states in 8 bits are the nearest to the formula's values in 64 bits; where such a value lies as near to the
border between two as the order of its operations moves it (a few 2^-53; 10^-14 is allowed), either."""
import numpy as np
import pytest
import torch

import sequence_ref as ref
from genn_amd.genn_model import Array, GeNNModel, init_postsynaptic, init_weight_update
from genn_amd.optimiser import AdamW

pytestmark = pytest.mark.gpu
BETA1, BETA2, EPS = 0.9, 0.99, 1e-8
U = 2.0 ** -24


def within(name, got, want, limit):
    """What is not finite (gradients in 16 bits are now and then) is so on both sides."""
    got, fine = got.detach().cpu().double(), torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), name
    off = ((got - want).abs() - limit)[fine]
    assert not off.numel() or off.max() <= 0, (name, float(off.max()))


def scales_close(name, got, want):
    """The nearest fp32 value, or its neighbour where `want` lies halfway between the two."""
    within(name, got, want, want.abs() * U * (1 + 1e-7) + 2.0 ** -150)


def codes_close(name, got, r):
    """The nearest code to each r, or its neighbour where r lies on the border."""
    got, want = got.long(), ref.e4m3_codes(r)
    border = (ref.E4M3[torch.minimum(got, want).clamp(max=126)] + ref.E4M3[torch.maximum(got, want).clamp(max=126)]) / 2
    assert torch.all((got == want) | (((got - want).abs() == 1) & ((r - border).abs() <= 1e-14 * r))), name


def weights_close(name, got, w, want, decay, rate, dtype):
    limit = U * (2 * w.abs() + 24 * (want - w).abs() + 24 * rate * decay * w.abs()) + torch.finfo(dtype).eps / 2 * want.abs()
    within(name, got, want, limit + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)


def tensors(sizes, weight, gradient, shift=0, seed=0):
    """Weights and gradients of several tensors, each `shift` elements into memory of its own."""
    gen = torch.Generator().manual_seed(seed)
    made = []
    for n in sizes:
        w, g = torch.randn(n, generator=gen) * 0.1, torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen))
        room = [torch.full((n + 8,), 5.0, dtype=t).cuda() for t in (weight, gradient)]
        for r, v in zip(room, (w, g)):
            r[shift:shift + n].copy_(v)
        made.append((room, [r[shift:shift + n] for r in room]))
    return made


SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 10000, 4, 0, 70001]


@pytest.mark.parametrize("weight, gradient, copy, shift", [
    (torch.float32, torch.float32, None, 0), (torch.float32, torch.bfloat16, torch.bfloat16, 0), (torch.float32, torch.float16, torch.float16, 1),
    (torch.bfloat16, torch.bfloat16, None, 0), (torch.float16, torch.float32, torch.bfloat16, 3)])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_against_the_formula(weight, gradient, copy, shift, bits):
    rate, decays = 1e-2, [0.1 * (k % 3) for k in range(len(SIZES))]
    made = tensors(SIZES, weight, gradient, shift)
    opt = AdamW(learning_rate=rate, beta1=BETA1, beta2=BETA2, epsilon=EPS, state_bits=bits)
    copies = [None if copy is None else torch.zeros(n + shift, dtype=copy).cuda()[shift:] for n in SIZES]
    states = []
    for (_, (w, g)), c, decay in zip(made, copies, decays):
        n = w.numel()
        s = dict(m=torch.zeros(n).cuda(), v=torch.zeros(n).cuda()) if bits == 32 else \
            dict(m=torch.zeros(n, dtype=torch.uint8).cuda(), v=torch.zeros(n, dtype=torch.uint8).cuda(), m_scale=torch.zeros(-(-n // 256)).cuda(), v_scale=torch.zeros(-(-n // 256)).cuda())
        states.append(s)
        opt.add(w, g, copy=c, weight_decay=decay, **s)
    opt.build()
    blocks = lambda t: torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)
    for step in range(1, 5):
        for k, (_, (w, g)) in enumerate(made):           # new gradients, some of them nothing at all
            g.mul_(-0.7)
            if step == 3 and k % 2:
                g.zero_()
        before = [[w.cpu().double(), g.cpu().double()] + [t.clone().cpu() for t in s.values()] for (_, (w, g)), s in zip(made, states)]
        opt.step()
        torch.cuda.synchronize()
        assert opt.steps == step
        for k, (room, (w, g)) in enumerate(made):
            n = w.numel()
            w0, g0, m0, v0 = before[k][:4]
            if bits == 8 and n:
                M, V = before[k][4].double(), before[k][5].double()
                value = blocks(m0.view(torch.float8_e4m3fn).double()) * (M / 448)[:, None]
                root = blocks(v0.view(torch.float8_e4m3fn).double()) / 448
                m0, v0 = value.view(-1)[:n], (root * root * V[:, None]).view(-1)[:n]
            want, m, v = ref.adamw(w0, g0, m0.double(), v0.double(), step, rate, BETA1, BETA2, EPS, decays[k])
            weights_close(f"weights of {k}", w, w0, want, decays[k], rate, weight)
            if copy is not None:
                weights_close(f"copy of {k}", copies[k], w0, want, decays[k], rate, copy)
                if weight == torch.float32:
                    assert torch.allclose(copies[k], w.to(copy), rtol=0, atol=0, equal_nan=True)
            s = states[k]
            if bits == 32:
                within(f"m of {k}", s["m"], m, 6 * U * (BETA1 * m0.abs() + (1 - BETA1) * g0.abs()) + 1e-44)
                within(f"v of {k}", s["v"], v, 6 * U * v + 1e-44)
            elif n:
                scales_close(f"scale of m of {k}", s["m_scale"], blocks(m).abs().amax(1))
                scales_close(f"scale of v of {k}", s["v_scale"], blocks(v).amax(1))
                M, V = (s[name].cpu().double().repeat_interleave(256)[:n] for name in ("m_scale", "v_scale"))
                fine = torch.isfinite(M) & torch.isfinite(V)
                codes = s["m"].cpu().long()
                codes_close(f"m of {k}", (codes & 127)[fine], torch.where(M > 0, m.abs() * 448 / M, 0.0)[fine])
                assert torch.all(((codes >= 128) == (m < 0))[fine & (codes & 127 > 0)]), k
                codes, root = s["v"].cpu().long()[fine], torch.where(V > 0, torch.sqrt(v / V) * 448, 0.0)[fine]
                raised = (v[fine] > 0) & (ref.e4m3_codes(root) == 0)
                assert torch.all(codes[raised] == 1), k
                codes_close(f"v of {k}", codes[~raised], root[~raised])
            assert all(torch.all(r[:shift] == 5.0) and torch.all(r[shift + n:] == 5.0) for r in room)


@pytest.mark.parametrize("bits, gradient", [(32, torch.float32), (32, torch.bfloat16), (8, torch.bfloat16)])
def test_a_step_that_passes_the_caches_by(bits, gradient):
    """A step of more than 64 MiB takes streaming accesses: the same bits as optimisers of a tensor each, which do not, and the formula's values.  The last tensor
    begins in the middle of an access."""
    sizes, rate, decay = [3000001, 2600003, 1027, 5], 1e-2, 0.1
    step = sum(sizes) * (8 + 4 * bits // 8 + torch.finfo(gradient).bits // 8)
    most = max(sizes) * (8 + 4 * bits // 8 + torch.finfo(gradient).bits // 8)
    if bits == 32:
        sizes, step, most = [s // 2 for s in sizes], step // 2, most // 2
    assert step > 64 << 20 > most
    made, again = ([w_g for _, w_g in tensors(sizes, torch.float32, gradient, seed=8)] for _ in range(2))
    room = torch.zeros(1000 + 3).cuda()
    first = [w.cpu().double() for w, _ in made]
    one, several = AdamW(learning_rate=rate, beta1=BETA1, beta2=BETA2, epsilon=EPS, state_bits=bits), []
    copies = [[torch.zeros(n, dtype=torch.bfloat16).cuda() for n in sizes] for _ in range(2)]
    for k in range(len(sizes)):
        one.add(*made[k], copy=copies[0][k], weight_decay=decay)
        several.append(AdamW(learning_rate=rate, beta1=BETA1, beta2=BETA2, epsilon=EPS, state_bits=bits))
        several[k].add(*again[k], copy=copies[1][k], weight_decay=decay)
    odd = [torch.cat([room.clone(), torch.zeros(8).cuda()])[3:][:1000] for _ in range(2)]
    ones = torch.ones(1000).cuda()
    one.add(odd[0], ones)
    several.append(AdamW(learning_rate=rate, beta1=BETA1, beta2=BETA2, epsilon=EPS, state_bits=bits))
    several[-1].add(odd[1], ones)
    for o in (one, *several):
        o.build()
    for k in range(2):
        for o in (one, *several):
            o.step()
        torch.cuda.synchronize()
        if k == 0:
            for n, (w, g) in enumerate(made):
                want, m, v = ref.adamw(first[n], g.cpu().double(), 0.0, 0.0, 1, rate, BETA1, BETA2, EPS, decay)
                weights_close(f"weights of {n}", w, first[n], want, decay, rate, torch.float32)
                got = {s: torch.from_numpy(a.pull_from_device().copy()) for s, a in one.states[n].items()}
                if bits == 32:
                    within(f"m of {n}", got["m"], m, 6 * U * m.abs() + 1e-44)
                    within(f"v of {n}", got["v"], v, 6 * U * v + 1e-44)
                else:
                    M, V = (got[s].double().repeat_interleave(256)[:sizes[n]] for s in ("m_scale", "v_scale"))
                    codes_close(f"m of {n}", got["m"].long() & 127, m.abs() * 448 / M)
                    codes, root = got["v"].long(), torch.sqrt(v / V) * 448
                    raised = (v > 0) & (ref.e4m3_codes(root) == 0)
                    assert torch.all(codes[raised] == 1)
                    codes_close(f"v of {n}", codes[~raised], root[~raised])
    assert torch.equal(odd[0], odd[1]) and odd[0].abs().sum() > 0
    for n in range(len(sizes)):
        assert torch.equal(made[n][0], again[n][0]) and torch.equal(copies[0][n], copies[1][n])
        for s in one.states[n]:
            assert np.array_equal(one.states[n][s].pull_from_device(), several[n].states[0][s].pull_from_device()), (n, s)


def test_a_positive_second_moment_never_becomes_zero():
    """A weight whose gradients are 10^-8 of its block's largest keeps a second moment: its next step is no division by epsilon."""
    g = torch.full((256,), 1e-8).cuda()
    g[7] = 1.0
    w = torch.zeros(256).cuda()
    opt = AdamW(learning_rate=1e-3, epsilon=1e-12, state_bits=8)
    opt.add(w, g)
    opt.build()
    opt.step()
    assert int((opt.states[0]["v"].pull_from_device() == 0).sum()) == 0
    g[:] = 0.0
    for _ in range(5):
        opt.step()
    assert float(w.abs().max()) < 0.02


@pytest.mark.parametrize("largest", [1e-20, 1.0, 1e15, 3e19, 5e19, 8e19])
def test_codes_of_any_size(largest):
    """Codes do not depend on how large a block's gradients are, up to second moments (here 3.2e38) at the end of fp32's range."""
    gen = torch.Generator().manual_seed(4)
    g = torch.rand(512, generator=gen) * largest
    g[100], g[300] = largest, largest
    # (first moments of up to 3e38 as well, from a state that was that large)
    codes, scale = torch.full((512,), 126, dtype=torch.uint8).cuda(), torch.tensor([1.0, 3e38]).cuda()
    w, m, v, V = torch.zeros(512).cuda(), torch.zeros(512, dtype=torch.uint8).cuda(), torch.zeros(512, dtype=torch.uint8).cuda(), torch.zeros(2).cuda()
    other, zero = torch.zeros(512).cuda(), torch.zeros(512).cuda()
    opt = AdamW(beta1=0.9, beta2=0.95, epsilon=EPS, state_bits=8)
    opt.add(w, g.cuda(), m=m, v=v, m_scale=torch.zeros(2).cuda(), v_scale=V)
    opt.add(other, zero, m=codes, v=torch.zeros(512, dtype=torch.uint8).cuda(), m_scale=scale, v_scale=torch.zeros(2).cuda())
    opt.build()
    opt.step()
    torch.cuda.synchronize()
    second = (1 - 0.95) * g.double() ** 2
    scales_close("scale of v", V, second.view(2, 256).amax(1))
    codes_close("v", v.cpu(), torch.sqrt(second / V.cpu().double().repeat_interleave(256)) * 448)
    assert torch.all(codes == 126)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_finite_stays_in_its_block(bits):
    gen = torch.Generator().manual_seed(1)
    g = torch.randn(1024, generator=gen).cuda()
    g[300], g[1000] = float("nan"), float("inf")
    w, other = torch.ones(1024).cuda(), torch.ones(100).cuda()
    opt = AdamW(learning_rate=1e-3, state_bits=bits)
    opt.add(w, g)
    opt.add(other, torch.ones(100).cuda())
    opt.build()
    opt.step()
    opt.step()
    assert torch.isfinite(other).all()
    bad = ~torch.isfinite(w.cpu())
    assert bad[300]
    assert not bad[:256].any() and not bad[512:768].any()
    if bits == 32:
        assert bad.sum() <= 2


def test_rate_scale_and_skip_on_the_device_and_a_captured_step():
    """A captured step counts, and reads its rate, its scale and whether to skip when it is replayed."""
    def build(stream_of):
        (_, (w, g)), = tensors([5000], torch.float32, torch.float32, seed=3)
        opt = AdamW(beta1=BETA1, beta2=BETA2)
        opt.add(w, g, weight_decay=0.1)
        opt.build()
        return w, opt
    rates, scales, skips = [1e-2, 3e-3, 1e-3, 5e-4, 2e-4], [1.0, 0.5, 2.0, 0.25, 1.0], [0, 0, 1, 0, 0]
    w, opt = build(None)
    for rate, scale, skip in zip(rates, scales, skips):
        if not skip:
            opt.step(rate, gradient_scale=torch.tensor([scale]).cuda())
            torch.cuda.synchronize()
    captured, other = build(None)
    rate, scale, skip = torch.zeros(1).cuda(), torch.zeros(1).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        other.step(rate, gradient_scale=scale, skip=skip, stream=torch.cuda.current_stream().cuda_stream)
    assert other.steps == 0
    for k, values in enumerate(zip(rates, scales, skips)):
        for t, v in zip((rate, scale, skip), values):
            t.fill_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert other.steps == sum(not s for s in skips[:k + 1])
    # (a rate as a double, and the same rounded to fp32: the change differs by its last bit)
    assert torch.allclose(w, captured, rtol=2 ** -22, atol=2 ** -22 * 1e-2)
    assert opt.steps == 4


def test_a_checkpoint_continues_where_it_was_taken():
    def build(states=None):
        made = tensors([3000, 77], torch.float32, torch.float32, seed=5)
        opt = AdamW(learning_rate=1e-2, state_bits=8)
        for k, (_, (w, g)) in enumerate(made):
            opt.add(w, g, **(states[k] if states else {}))
        opt.build()
        return [w for _, (w, _) in made], opt
    w, opt = build()
    for _ in range(3):
        opt.step()
    saved = [{k: torch.from_numpy(a.pull_from_device().copy()).cuda() for k, a in s.items()} for s in opt.states]
    weights, steps = [x.clone() for x in w], opt.steps
    opt.step()
    again, other = build(saved)
    for a, b in zip(again, weights):
        a.copy_(b)
    other.steps = steps
    other.step()
    assert other.steps == 4 and all(torch.equal(a, b) for a, b in zip(again, w))


def test_rates_of_any_kind_of_number():
    import numpy as np
    results = []
    for rate in (0.5, np.float32(0.5), np.float64(0.5), torch.tensor(0.5).cuda()):
        w, g = torch.ones(10).cuda(), torch.ones(10).cuda()
        opt = AdamW()
        opt.add(w, g)
        opt.build()
        opt.step(rate)
        torch.cuda.synchronize()
        results.append(w.clone())
    assert all(torch.equal(results[0], r) for r in results) and float(results[0][0]) < 0.6


def test_another_current_device_is_refused():
    """(an optimiser that says it belongs to the second device, while the first is current)"""
    w = torch.ones(10).cuda()
    opt = AdamW()
    opt.add(w, w.clone())
    opt.device = 1
    with pytest.raises(ValueError, match="current device is 0"):
        opt.add(w.clone(), w.clone())
    with pytest.raises(ValueError, match="current device is 0"):
        opt.build()


def test_what_the_layer_refuses():
    opt = AdamW()
    w = torch.zeros(10).cuda()
    for wrong, error in ((dict(weights=w, gradients=torch.zeros(9).cuda()), "elements"), (dict(weights=w.double(), gradients=w), "holds"),
                         (dict(weights=torch.zeros(20).cuda()[::2], gradients=w), "contiguous"), (dict(weights=w, gradients=w.clone(), m_scale=w), "no scales"),
                         (dict(weights=w, gradients=w.clone(), copy=torch.zeros(10).cuda()), "holds")):
        with pytest.raises((ValueError, TypeError), match=error):
            opt.add(**wrong)
    opt.add(w, w.clone())
    from genn_amd._abi import GennmiError
    with pytest.raises(GennmiError, match="not finalised"):
        opt.step()
    opt.build()
    with pytest.raises(GennmiError, match="learning rate"):
        opt.step(float("nan"))
    with pytest.raises(ValueError, match="one value"):
        opt.step(gradient_scale=w)
    with pytest.raises(GennmiError, match="finalised"):
        opt.add(torch.zeros(3).cuda(), torch.zeros(3).cuda())
    opt.free()
    with pytest.raises(RuntimeError, match="freed"):
        opt.add(w, w.clone())


@pytest.mark.parametrize("matrix", ["SPARSE", "DENSE"])
def test_a_network_steps_with_the_weights_that_were_trained(make_model, matrix):
    """The runner keeps copies of a projection's weights: a step of the optimiser reaches them, in front of queued and resident steps alike."""
    n, steps = 300, 20
    rng = np.random.default_rng(2)
    i, j = np.nonzero(rng.random((n, n)) < 0.1)
    g0 = rng.random(n * n if matrix == "DENSE" else len(i)).astype(np.float32) * 0.05
    lif = dict(C=1.0, TauM=20.0, Vrest=-60.0, Vreset=-60.0, Vthresh=-50.0, Ioffset=0.6, TauRefrac=5.0)

    def build(weights):
        m = make_model("float", "trained", dt=1.0)
        src = m.add_neuron_population("S", n, "LIF", lif, {"V": np.linspace(-60, -50, n, dtype=np.float32), "RefracTime": 0.0})
        trg = m.add_neuron_population("T", n, "LIF", dict(lif, Vthresh=1e9, Ioffset=0.0), {"V": -60.0, "RefracTime": 0.0})
        s = m.add_synapse_population("ST", matrix, src, trg, init_weight_update("StaticPulse", {}, {"g": weights}), init_postsynaptic("DeltaCurr"))
        if matrix == "SPARSE":
            s.set_sparse_connections(i, j)
            s.set_var_coo("g", weights)
        m.build()
        m.load()
        return m, src, trg, s

    m, src, trg, s = build(g0)
    first = {v: (p, p.vars[v].pull_from_device().copy()) for p, v in ((src, "V"),)}
    m.run_steps(steps) if hasattr(m, "run_steps") else [m.step_time() for _ in range(steps)]
    unchanged = trg.vars["V"].pull_from_device().copy()
    g = s.vars["g"]
    gradients = Array(g.count, np.float32, fill=np.sin(np.arange(g.count)).astype(np.float32))
    opt = AdamW(learning_rate=0.02)
    opt.add(g, gradients)
    opt.build()
    old = g.pull_from_device().copy()
    opt.step()
    new = g.pull_from_device().copy()
    assert np.allclose(new, old - 0.02 * np.sign(np.sin(np.arange(g.count))), atol=1e-4)

    def again(m, src, trg):
        for p in (src, trg):
            for v, value in (("V", np.linspace(-60, -50, n, dtype=np.float32) if p is src else -60.0), ("RefracTime", 0.0)):
                p.vars[v].view[:] = value
                p.vars[v].push_to_device()
        [m.step_time() for _ in range(steps)]
        return trg.vars["V"].pull_from_device().copy()

    got = again(m, src, trg)
    other, src2, trg2, s2 = build(g0)
    [other.step_time() for _ in range(steps)]
    s2.vars["g"].view[:] = new
    s2.vars["g"].push_to_device()
    want = again(other, src2, trg2)
    # (sums of at most 300 inputs in an order of their own: 300 x 2^-24 of a few ten millivolts)
    assert np.allclose(got, want, rtol=0, atol=300 * 2 ** -24 * 80)
    assert not np.allclose(got, unchanged, rtol=0, atol=1e-2)
    opt.free()


def test_a_layer_is_trained_by_the_operators_together():
    """Convolution, scan, a quadratic loss, their gradients, and the step: gradients along a direction are those of differences of the loss in 64 bits, and
    the steps run."""
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    gen = torch.Generator().manual_seed(9)
    r = lambda *shape: torch.randn(*shape, generator=gen)
    S, n, D, N, K = 3, 70, 40, 8, 4
    x, delta, B, C, target = r(S, n, D), r(S, n, D), r(S, n, N), r(S, n, N), r(S, n, D)
    p = dict(weight=r(D, K) * 0.5, bias=r(D) * 0.1, A=-torch.exp(r(D, N) * 0.3), skip=r(D), delta_bias=r(D) - 1)
    on = {k: v.clone().cuda() for k, v in p.items()}
    g = {k: torch.zeros_like(v) for k, v in on.items()}
    mid, out, dmid, dx = (torch.zeros(S, n, D).cuda() for _ in range(4))
    conv, scan = CausalConvolution(S, n, D, K, silu=True), SelectiveScan(S, n, D, N, softplus=True)
    conv.bind(x=x.cuda(), weight=on["weight"], bias=on["bias"], out=mid)
    scan.bind(u=mid, delta=delta.cuda(), A=on["A"], B=B.cuda(), C=C.cuda(), D=on["skip"], delta_bias=on["delta_bias"], out=out)
    dout = torch.zeros(S, n, D).cuda()
    scan.bind_gradients(out=dout, u=dmid, A=g["A"], D=g["skip"], delta_bias=g["delta_bias"])
    conv.bind_gradients(out=dmid, x=dx, weight=g["weight"], bias=g["bias"])
    opt = AdamW(learning_rate=1e-2)
    for k in on:
        opt.add(on[k], g[k])
    opt.build()

    def gradients():
        conv.run()
        scan.run()
        torch.sub(out, target.cuda(), out=dout)
        scan.backward()
        conv.backward()

    def loss(q):
        total = 0.0
        for s in range(S):
            m, _ = ref.causal_conv(x[s], q["weight"], q["bias"], True)
            y, _ = ref.scan(m, delta[s], q["A"], B[s].view(n, 1, N), C[s].view(n, 1, N), D=q["skip"], delta_bias=q["delta_bias"], softplus=True)
            total += float(((y - target[s].double()) ** 2).sum()) / 2
        return total

    gradients()
    torch.cuda.synchronize()
    for k in p:
        d = torch.sign(g[k].cpu().double())           # (along which every entry's error counts)
        up, down = ({**{m: v.double() for m, v in p.items()}, k: p[k].double() + e * d} for e in (1e-5, -1e-5))
        want = (loss(up) - loss(down)) / 2e-5
        got = float((g[k].cpu().double() * d).sum())
        # fp32 sums over 70 rows and two operators, their terms of either sign: 1e-4 of the absolute sum is 1,700 half steps
        assert abs(got - want) < 1e-4 * abs(want) + 1e-6, (k, got, want)
    before = {k: v.clone() for k, v in on.items()}
    for _ in range(3):
        gradients()
        opt.step()
    assert opt.steps == 3
    assert all(torch.isfinite(v).all() and not torch.equal(v, before[k]) for k, v in on.items())
