"""The sequence operators and the optimiser step, as cases that can be prepared, run and compared.

A case is one pass of a user's program through one operator: a short causal convolution or a selective state space scan over
prompts, its gradients in training, or one token of every running sequence; or an AdamW step over all weights of a model.
Arrays of sequences are rows of channels; sequences of different lengths lie one behind another in packed rows.
"""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256             # weights that share a scale of the states in 8 bits
BETA1, BETA2, EPS, DECAY, RATE = 0.9, 0.95, 1e-8, 0.1, 1e-3


def listed():
    return [
        # A prompt through the convolution of one layer; the last inputs stay as the state that tokens continue from.
        dict(name="conv_prompt", op="conv", sequences=1, length=4096, channels=4096, taps=4, type="bfloat16"),
        # The convolution's gradients in a training step.
        dict(name="conv_training", op="conv_backward", sequences=8, length=2048, channels=2048, taps=4, type="bfloat16"),
        # One token of sixteen running sequences whose states lie scattered in a pool: nothing but latency.
        dict(name="conv_token", op="conv_token", sequences=16, channels=2048, taps=4, type="bfloat16"),
        # One prompt through the scan: few channels, so that only a split over time fills the chip.
        dict(name="scan_prompt", op="scan", sequences=1, length=4096, channels=2048, states=16, groups=1, type="bfloat16"),
        # Prompts of very different lengths (none and one row among them), two groups, an odd number of channels in each.
        dict(name="scan_ragged_prompts", op="scan_ragged", sequences=33, rows=8011, channels=1002, states=16, groups=2, type="float16"),
        # The scan's gradients in a training step: the largest.
        dict(name="scan_training", op="scan_backward", sequences=8, length=2048, channels=2048, states=16, groups=1, type="bfloat16"),
        # Gradients of a small experiment in 32 bits; no size is even.
        dict(name="scan_training_small", op="scan_backward", sequences=3, length=301, channels=511, states=7, groups=1, type="float32"),
        # One token of one sequence.
        dict(name="scan_token_one", op="scan_token", sequences=1, channels=2048, states=16, groups=1, type="bfloat16"),
        # One token of many sequences: reads and writes all their states.
        dict(name="scan_token_batch", op="scan_token", sequences=256, channels=4096, states=16, groups=1, type="bfloat16"),
        # The weights of a small network: many short tensors, nothing but latency.
        dict(name="adamw_small", op="adamw", tensors=20, weights=60011, bits=32, gradient="float32", copy=False),
        # A model's weights in 32 bits with a working copy in 16, gradients in 16.
        dict(name="adamw_32", op="adamw", tensors=60, weights=80000000, bits=32, gradient="bfloat16", copy=True),
        # The same step with its states in 8 bits.
        dict(name="adamw_8", op="adamw", tensors=60, weights=130000000, bits=8, gradient="bfloat16", copy=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every operator alike, sizes over the range of the listed ones and below."""
    op = rng.choice(["conv", "conv_backward", "conv_token", "scan", "scan_ragged", "scan_backward", "scan_token", "adamw"])
    if op == "adamw":
        return dict(op=op, tensors=rng.randint(1, 60), weights=_log(rng, 1000, 80000000), bits=rng.choice([8, 32]),
                    gradient=rng.choice(["float32", "bfloat16"]), copy=rng.choice([False, True]))
    case = dict(op=op, type=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]))
    if op.startswith("conv"):
        case["taps"] = rng.choice([2, 3, 4, 4, 4])
    else:
        case["states"] = rng.choice([4, 8, 16, 16, 16, 24, 32])
        case["groups"] = rng.choice([1, 1, 2])
    case["channels"] = case.get("groups", 1) * _log(rng, 60, 4000 // case.get("groups", 1))
    if op.endswith("token"):
        return dict(case, sequences=_log(rng, 1, 200))
    most = 24000000 // case["channels"]         # rows: an eighth and more below the largest listed case in all
    most = most if op.startswith("conv") else most * 16 // max(16, case["states"])
    if op == "scan_ragged":
        return dict(case, sequences=rng.randint(1, 40), rows=_log(rng, 50, min(most, 10000)))
    sequences = _log(rng, 1, 16)
    return dict(case, sequences=sequences, length=_log(rng, 2, min(8000, most // sequences)))


def _lengths(case):
    """Rows of each sequence: of the packed ones as cut at random places, so that some are long, some short and now and then one empty."""
    if case["op"] != "scan_ragged":
        return [case.get("length", 1)] * case["sequences"]
    rng = random.Random(case["sequences"] * 7919 + case["rows"])
    cuts = sorted(rng.randint(0, case["rows"]) for _ in range(case["sequences"] - 1))
    if len(cuts) > 3:
        cuts[1], cuts[3] = cuts[0], cuts[2] + 1 if cuts[2] + 1 <= cuts[4 if len(cuts) > 4 else 3] else cuts[2]      # one without rows, one of one
    ends = [0] + cuts + [case["rows"]]
    return [b - a for a, b in zip(ends, ends[1:])]


def _shapes(case):
    """Weights of each tensor: matrices of a model with short vectors between them."""
    rng = random.Random(case["tensors"] * 31 + case["weights"])
    share = [math.exp(rng.uniform(0.0, 3.0)) * (0.002 if k % 3 == 2 else 1.0) for k in range(case["tensors"])]
    return [max(1, int(case["weights"] * s / sum(share))) for s in share]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    state = dict(case=case)
    if case["op"] == "adamw":
        sizes = _shapes(case)
        # (every tensor begins at a block of its own in one buffer)
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        decay = torch.zeros(total, device="cuda")
        for k, (a, n) in enumerate(zip(starts, sizes)):
            used[a:a + n] = True
            decay[a:a + n] = 0.0 if k % 3 == 2 else DECAY       # no decay of biases and gains
        state.update(sizes=sizes, starts=starts, used=used, decay=decay, steps=0)
        state["w"] = normal(total, scale=0.02) * used
        # gradients whose size differs from tensor to tensor and from weight to weight
        state["g"] = (normal(total, scale=1e-3) * torch.exp(normal(total)) * used).to(TYPES[case["gradient"]])
        state["copy"] = state["w"].to(torch.bfloat16) if case["copy"] else None
        if case["bits"] == 32:
            state["m"], state["v"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
        else:
            state["m"], state["v"] = (torch.zeros(total, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
            state["M"], state["V"] = torch.zeros(total // BLOCK, device="cuda"), torch.zeros(total // BLOCK, device="cuda")
        if own:
            from genn_amd.optimiser import AdamW
            opt = AdamW(learning_rate=RATE, beta1=BETA1, beta2=BETA2, epsilon=EPS, state_bits=case["bits"])
            for k, (a, n) in enumerate(zip(starts, sizes)):
                part = dict(weights=state["w"][a:a + n], gradients=state["g"][a:a + n], m=state["m"][a:a + n], v=state["v"][a:a + n],
                            weight_decay=0.0 if k % 3 == 2 else DECAY)
                if case["copy"]:
                    part["copy"] = state["copy"][a:a + n]
                if case["bits"] == 8:
                    blocks = slice(a // BLOCK, a // BLOCK + -(-n // BLOCK))
                    part.update(m_scale=state["M"][blocks], v_scale=state["V"][blocks])
                opt.add(**part)
            opt.build()
            state["plan"] = opt
        return state

    T, D, lengths = TYPES[case["type"]], case["channels"], _lengths(case)
    S, rows = len(lengths), sum(lengths)
    token, ragged, backward = case["op"].endswith("token"), case["op"] == "scan_ragged", case["op"].endswith("backward")
    spare = 5 if ragged else 0          # rows behind the last sequence
    first = torch.tensor([0] + lengths).cumsum(0)
    state.update(lengths=lengths, first=first.cuda(), longest=max(lengths))
    at = torch.repeat_interleave(torch.arange(S), torch.tensor(lengths))
    state["at"] = at.cuda()                                             # the sequence of each row
    state["place"] = (torch.arange(rows) - first[at]).cuda()            # its place in it
    state["offsets"] = first.to(torch.int32).cuda() if ragged else None
    state["slots"] = None
    states = S
    if token or ragged:
        states = S + 3
        state["slots"] = torch.randperm(states, generator=gen, device="cuda")[:S].to(torch.int32)
    where = state["slots"].long() if state["slots"] is not None else torch.arange(S, device="cuda")
    state["where"] = where
    state["out"] = torch.zeros(rows + spare, D, dtype=T, device="cuda")
    if case["op"].startswith("conv"):
        K = case["taps"]
        state["x"] = normal(rows, D, dtype=T)
        state["weight"] = uniform(-1, 1, D, K) * K ** -0.5
        state["bias"] = uniform(-1, 1, D) * K ** -0.5
        state["initial"] = normal(states, K - 1, D, dtype=T) if token or backward else None
        state["final"] = state["initial"] if token else torch.zeros(states, K - 1, D, dtype=T, device="cuda")
        if backward:
            state["dout"] = normal(rows, D, dtype=T)
            state["dfinal"] = normal(states, K - 1, D, dtype=T)
            state["dx"] = torch.zeros(rows, D, dtype=T, device="cuda")
            state["dweight"], state["dbias"] = torch.zeros(D, K, device="cuda"), torch.zeros(D, device="cuda")
            state["dinitial"] = torch.zeros(states, K - 1, D, dtype=T, device="cuda")
        if own:
            from genn_amd.sequence import CausalConvolution
            plan = CausalConvolution(S, state["longest"], D, K, dtype=case["type"], silu=True)
            plan.bind(x=state["x"], weight=state["weight"], bias=state["bias"], out=state["out"], initial_state=state["initial"],
                      final_state=state["final"], slots=state["slots"])
            if backward:
                plan.bind_gradients(out=state["dout"], final_state=state["dfinal"], x=state["dx"], weight=state["dweight"], bias=state["dbias"],
                                    initial_state=state["dinitial"])
            state["plan"] = plan
        return state

    N, G = case["states"], case["groups"]
    # the projections that a layer's input gives: time steps, input and output weights side by side in one row
    wide = normal(rows + spare, D + 2 * G * N, dtype=T)
    state["u"] = normal(rows + spare, D, dtype=T)
    state["delta"], state["B"], state["C"] = wide[:, :D], wide[:, D:D + G * N], wide[:, D + G * N:]
    state["z"] = normal(rows + spare, D, dtype=T)
    state["A"] = -torch.arange(1, N + 1, device="cuda") * torch.exp(normal(D, N, scale=0.1))
    state["D"] = 1 + normal(D, scale=0.1)
    state["bias"] = torch.log(torch.expm1(torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))))
    state["initial"] = normal(states, D, N) if token or ragged or backward else None
    state["final"] = state["initial"] if token else torch.zeros(states, D, N, device="cuda")
    if backward:
        state["dout"] = normal(rows, D, dtype=T)
        state["dfinal"] = normal(states, D, N)
        state["du"], state["ddelta"], state["dz"] = (torch.zeros(rows, D, dtype=T, device="cuda") for _ in range(3))
        state["dB"], state["dC"] = (torch.zeros(rows, G * N, dtype=T, device="cuda") for _ in range(2))
        state["dA"], state["dD"], state["dbias"] = torch.zeros(D, N, device="cuda"), torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda")
        state["dinitial"] = torch.zeros(states, D, N, device="cuda")
    if own:
        from genn_amd.sequence import SelectiveScan
        plan = SelectiveScan(S, state["longest"], D, N, groups=G, dtype=case["type"], softplus=True)
        plan.bind(u=state["u"], delta=state["delta"], A=state["A"], B=state["B"], C=state["C"], D=state["D"], delta_bias=state["bias"], z=state["z"],
                  out=state["out"], initial_state=state["initial"], final_state=state["final"], offsets=state["offsets"], slots=state["slots"])
        if backward:
            plan.bind_gradients(out=state["dout"], final_state=state["dfinal"], u=state["du"], delta=state["ddelta"], A=state["dA"], B=state["dB"],
                                C=state["dC"], D=state["dD"], delta_bias=state["dbias"], z=state["dz"], initial_state=state["dinitial"])
        state["plan"] = plan
    return state


def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        if own:
            state["plan"].step()
        else:
            _adamw(state)
        return {k: state[k] for k in ("w", "m", "v", "M", "V", "copy") if state.get(k) is not None}
    if op.endswith("backward"):
        if own:
            state["plan"].backward()
        else:
            (_conv_backward if op.startswith("conv") else _scan_backward)(state)
        return {k: state[k] for k in ("dx", "dweight", "du", "ddelta", "dz", "dB", "dC", "dA", "dD", "dbias", "dinitial") if k in state}
    if own:
        state["plan"].run()
    else:
        (_conv if op.startswith("conv") else _scan)(state)
    return {"out": state["out"], "final": state["final"]}


# ---- plain forms: elementary operations on all rows at once, in 32 bits

def _e4m3(r):
    """The nearest values of the 8-bit format with 4 bits of exponent and 3 of mantissa, ties to the even one."""
    step = torch.exp2(torch.frexp(r)[1].clamp(min=-5).double() - 4)
    return (torch.round(r / step) * step).clamp(-448, 448)


def _adamw(s):
    s["steps"] += 1
    g = s["g"].float()
    eight = s["case"]["bits"] == 8
    if eight:           # (in 64 bits: values next to the border between two codes)
        g = g.double()
        m = s["m"].double().view(-1, BLOCK) * (s["M"].double() / 448)[:, None]
        v = (s["v"].double().view(-1, BLOCK) / 448).square() * s["V"].double()[:, None]
        m, v = m.view(-1) * BETA1 + (1 - BETA1) * g, v.view(-1) * BETA2 + (1 - BETA2) * g * g
        M, V = m.view(-1, BLOCK).abs().amax(1).float(), v.view(-1, BLOCK).amax(1).float()
        s["M"].copy_(M)
        s["V"].copy_(V)
        scaled = m.view(-1, BLOCK) * (448 / M.double().clamp(min=1e-45))[:, None]
        s["m"].copy_(_e4m3(scaled).view(-1).float().to(torch.float8_e4m3fn))
        root = (v.view(-1, BLOCK) / V.double().clamp(min=1e-45)[:, None]).sqrt() * 448
        code = _e4m3(root).view(-1)
        s["v"].copy_(torch.where(v > 0, code.clamp(min=2.0 ** -9), code).float().to(torch.float8_e4m3fn))
        m, v = m.float(), v.float()
    else:
        m, v = s["m"].mul_(BETA1).add_(g * (1 - BETA1)), s["v"].mul_(BETA2).add_(g * g * (1 - BETA2))
    root = (v / (1 - BETA2 ** s["steps"])).sqrt() + EPS
    w = s["w"] * (1 - RATE * s["decay"]) - RATE * (m / (1 - BETA1 ** s["steps"])) / root
    s["w"].copy_(w)
    if s["copy"] is not None:
        s["copy"].copy_(w)


def _taps(s):
    """x[t - (K - 1) + k] of every row as [rows, K, channels]: before a sequence's first row lies its initial state."""
    K, rows = s["case"]["taps"], s["x"].shape[0]
    back = torch.arange(K, device="cuda") - (K - 1)
    at = torch.arange(rows, device="cuda")[:, None] + back
    inside = s["place"][:, None] + back >= 0
    got = s["x"].float()[at.clamp(min=0)] * inside[..., None]
    if s["initial"] is not None:
        before = (K - 1 + s["place"][:, None] + back).clamp(0, K - 2)
        got = got + s["initial"].float()[s["where"][s["at"]][:, None], before] * ~inside[..., None]
    return got


def _last(s):
    """Rows that the final state holds: [sequences, K - 1] places in a sequence, negative ones in its initial state."""
    K = s["case"]["taps"]
    return (s["first"][1:] - s["first"][:-1])[:, None] + torch.arange(K - 1, device="cuda") - (K - 1)


def _conv(s):
    K = s["case"]["taps"]
    lin = (_taps(s) * s["weight"].t()).sum(1) + s["bias"]
    s["out"][:lin.shape[0]].copy_(lin * torch.sigmoid(lin))
    last = _last(s)
    rows = s["x"][(s["first"][:-1, None] + last).clamp(min=0)]
    if s["initial"] is not None:
        rows = torch.where((last >= 0)[..., None], rows, s["initial"][s["where"][:, None], (last + K - 1).clamp(0, K - 2)])
    else:
        rows = rows * (last >= 0)[..., None]
    s["final"][s["where"]] = rows


def _conv_backward(s):
    K, (rows, D) = s["case"]["taps"], s["x"].shape
    taps = _taps(s)
    lin = (taps * s["weight"].t()).sum(1) + s["bias"]
    sig = torch.sigmoid(lin)
    ds = s["dout"].float() * (sig * (1 + lin * (1 - sig)))
    s["dbias"].copy_(ds.double().sum(0))
    s["dweight"].copy_((taps * ds[:, None]).sum(0, dtype=torch.float64).t())
    part = ds[:, None] * s["weight"].t()
    # (rows with the K - 1 of each sequence's initial state before them)
    S = len(s["lengths"])
    back = torch.arange(K, device="cuda")
    at = (torch.arange(rows, device="cuda") + s["at"] * (K - 1))[:, None] + back
    dx = torch.zeros(rows + S * (K - 1), D, device="cuda")
    for k in range(K):          # (one tap after another: the rows of one are all different)
        dx[at[:, k]] += part[:, k]
    ends = (s["first"][1:] + torch.arange(S, device="cuda") * (K - 1))[:, None] + torch.arange(K - 1, device="cuda")
    dx[ends] += s["dfinal"].float()[s["where"]]
    s["dx"].copy_(dx[at[:, K - 1]])
    starts = (s["first"][:-1] + torch.arange(S, device="cuda") * (K - 1))[:, None] + torch.arange(K - 1, device="cuda")
    s["dinitial"][s["where"]] = dx[starts].to(s["dinitial"].dtype)


def _recur(a, b, longest):
    """h[t] = a[t] h[t - 1] + b[t] along the first axis, by doubling; a is 0 where a sequence begins. Both are overwritten."""
    step = 1
    while step < longest:
        b[step:] += a[step:] * b[:-step]
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def _grouped(x, rows, s):
    G, N = s["case"]["groups"], s["case"]["states"]
    return x[:rows].float().reshape(rows, G, N).repeat_interleave(s["case"]["channels"] // G, 1)


def _scan_parts(s):
    rows = s["at"].shape[0]
    raw = s["delta"][:rows].float() + s["bias"]
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    u = s["u"][:rows].float()
    decay = torch.exp(dt[..., None] * s["A"])
    b = (dt * u)[..., None] * _grouped(s["B"], rows, s)
    starts = torch.nonzero(s["place"] == 0)[:, 0]
    if s["initial"] is not None:
        b[starts] += decay[starts] * s["initial"][s["where"][s["at"][starts]]]
    a = decay.clone()
    a[starts] = 0
    return rows, raw, dt, u, decay, starts, _recur(a, b, s["longest"])


def _scan(s):
    rows, raw, dt, u, decay, starts, h = _scan_parts(s)
    z = s["z"][:rows].float()
    y = (h * _grouped(s["C"], rows, s)).sum(-1) + s["D"] * u
    s["out"][:rows].copy_(y * z * torch.sigmoid(z))
    full = s["first"][1:] > s["first"][:-1]
    kept = s["initial"][s["where"]] if s["initial"] is not None else torch.zeros_like(s["final"][s["where"]])
    s["final"][s["where"]] = torch.where(full[:, None, None], h[(s["first"][1:] - 1).clamp(min=0)], kept)


def _scan_backward(s):
    G, N, D = s["case"]["groups"], s["case"]["states"], s["case"]["channels"]
    rows, raw, dt, u, decay, starts, h = _scan_parts(s)
    z, dout = s["z"].float(), s["dout"].float()
    C = _grouped(s["C"], rows, s)
    sig = torch.sigmoid(z)
    y = (h * C).sum(-1) + s["D"] * u
    s["dz"].copy_(dout * y * (sig * (1 + z * (1 - sig))))
    gy = dout * z * sig
    s["dC"].copy_((gy[..., None] * h).view(rows, G, D // G, N).sum(2).view(rows, G * N))
    s["dD"].copy_((gy * u).double().sum(0))
    # dh[t] = C gy + decay[t + 1] dh[t + 1]: the same recurrence from the other end
    b = gy[..., None] * C
    del C
    full = s["first"][1:] > s["first"][:-1]
    ends = s["first"][1:][full] - 1
    b[ends] += s["dfinal"][s["where"][full]]
    a = torch.zeros_like(decay)
    a[:-1] = decay[1:]
    a[ends] = 0
    dh = _recur(a.flip(0), b.flip(0), s["longest"]).flip(0)
    del a, b
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[starts] = s["initial"][s["where"][s["at"][starts]]]
    s["dB"].copy_((dh * (dt * u)[..., None]).view(rows, G, D // G, N).sum(2).view(rows, G * N))
    q = (dh * _grouped(s["B"], rows, s)).sum(-1)
    x = dh * decay * before
    s["du"].copy_(dt * q + s["D"] * gy)
    draw_ = (u * q + (x * s["A"]).sum(-1)) * torch.sigmoid(raw)
    s["ddelta"].copy_(draw_)
    s["dbias"].copy_(draw_.double().sum(0))
    s["dA"].copy_((x * dt[..., None]).sum(0, dtype=torch.float64))
    s["dinitial"][s["where"][full]] = (decay * dh)[s["first"][:-1][full]]
    s["dinitial"][s["where"][~full]] = s["dfinal"][s["where"][~full]]


# ---- what a pass cannot do without

def work(case):
    if case["op"] == "adamw":
        n = sum(_shapes(case))
        size = 4 if case["gradient"] == "float32" else 2
        return {"bytes": n * (8 + size + (16 if case["bits"] == 32 else 4) + (2 if case["copy"] else 0)), "flops": 16 * n}
    size = 4 if case["type"] == "float32" else 2
    lengths, D = _lengths(case), case["channels"]
    rows, S = sum(lengths), len(lengths)
    token, backward = case["op"].endswith("token"), case["op"].endswith("backward")
    if case["op"].startswith("conv"):
        K = case["taps"]
        state = S * (K - 1) * D * size
        moved = rows * D * size * (3 if backward else 2) + state * (3 if backward else 2 if token else 1) + D * (K + 1) * 4 * (2 if backward else 1)
        return {"bytes": moved, "flops": rows * D * (2 * K + 4) * (3 if backward else 1)}
    N, G = case["states"], case["groups"]
    state = S * D * N * 4
    moved = rows * size * ((7 * D + 4 * G * N) if backward else (4 * D + 2 * G * N)) + D * (N + 2) * 4 * (2 if backward else 1)
    moved += state * (3 if backward else 2 if token or case["op"] == "scan_ragged" else 1)
    return {"bytes": moved, "flops": rows * D * (N * (24 if backward else 8) + 20)}


# ---- the definitions in 64 bits, one row after another

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    lengths, first = s["lengths"], [0]
    for n in lengths:
        first.append(first[-1] + n)
    same = len(set(lengths)) == 1
    # sequences of one length together, others one by one
    parts = [(torch.arange(len(lengths), device="cuda"), lengths[0])] if same else [(torch.tensor([k], device="cuda"), n) for k, n in enumerate(lengths)]
    out = {}
    for seqs, n in parts:
        begin = s["first"][:-1][seqs]
        rows = begin[None, :] + torch.arange(n, device="cuda")[:, None]            # [n, sequences]
        (_exact_conv if case["op"].startswith("conv") else _exact_scan)(s, out, rows, s["where"][seqs])
    return out


def _like(s, out, key):
    if key not in out:
        out[key] = torch.zeros_like(s[key], dtype=torch.float64) if key != "final" else s["final"].double()
    return out[key]


def _exact_conv(s, out, rows, where):
    K, n = s["case"]["taps"], rows.shape[0]
    x = s["x"].double()[rows]
    begin = s["initial"].double()[where].transpose(0, 1) if s["initial"] is not None else x.new_zeros((K - 1,) + x.shape[1:])
    x = torch.cat([begin, x])
    w = s["weight"].double()
    lin = s["bias"].double() + sum(x[k:k + n] * w[:, k] for k in range(K))
    if not s["case"]["op"].endswith("backward"):
        _like(s, out, "out")[rows] = lin / (1 + torch.exp(-lin))
        _like(s, out, "final")[where] = x[n:].transpose(0, 1)
        return
    sig = 1 / (1 + torch.exp(-lin))
    ds = s["dout"].double()[rows] * (sig + lin * sig * (1 - sig))
    dx = torch.zeros_like(x)
    for k in range(K):
        dx[k:k + n] += ds * w[:, k]
    dx[n:] += s["dfinal"].double()[where].transpose(0, 1)
    _like(s, out, "dx")[rows] = dx[K - 1:]
    _like(s, out, "dinitial")[where] = dx[:K - 1].transpose(0, 1)
    out["dbias"] = out.get("dbias", 0) + ds.sum((0, 1))
    out["dweight"] = out.get("dweight", 0) + torch.stack([(ds * x[k:k + n]).sum((0, 1)) for k in range(K)], 1)


def _exact_scan(s, out, rows, where):
    G, N, D, n = s["case"]["groups"], s["case"]["states"], s["case"]["channels"], rows.shape[0]
    A, skip = s["A"].double(), s["D"].double()
    group = torch.arange(D, device="cuda") // (D // G)
    raw = s["delta"].double()[rows] + s["bias"].double()
    dt = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
    u, z = s["u"].double()[rows], s["z"].double()[rows]
    B, C = (s[k].double()[rows].view(n, rows.shape[1], G, N) for k in "BC")
    h = s["initial"].double()[where] if s["initial"] is not None else A.new_zeros((rows.shape[1], D, N))
    backward = s["case"]["op"].endswith("backward")
    y, kept = torch.zeros_like(u), [h]
    for t in range(n):
        h = torch.exp(dt[t][..., None] * A) * h + (dt[t] * u[t])[..., None] * B[t][:, group]
        y[t] = (h * C[t][:, group]).sum(-1) + skip * u[t]
        if backward:
            kept.append(h)
    gate = 1 / (1 + torch.exp(-z))
    if not backward:
        _like(s, out, "out")[rows] = y * z * gate
        _like(s, out, "final")[where] = h
        return
    dout = s["dout"].double()[rows]
    _like(s, out, "dz")[rows] = dout * y * (gate + z * gate * (1 - gate))
    gy = dout * z * gate
    dh = s["dfinal"].double()[where]
    dA = torch.zeros_like(dh)
    du, ddt, dB, dC = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(B), torch.zeros_like(C)
    for t in reversed(range(n)):
        dh = dh + gy[t][..., None] * C[t][:, group]
        dC[t] = (gy[t][..., None] * kept[t + 1]).view(-1, G, D // G, N).sum(2)
        dB[t] = (dh * (dt[t] * u[t])[..., None]).view(-1, G, D // G, N).sum(2)
        q = (dh * B[t][:, group]).sum(-1)
        dh = dh * torch.exp(dt[t][..., None] * A)           # with respect to the state before
        x = dh * kept[t]
        dA += x * dt[t][..., None]
        du[t], ddt[t] = dt[t] * q + skip * gy[t], u[t] * q + (x * A).sum(-1)
    _like(s, out, "du")[rows] = du
    ddelta = ddt / (1 + torch.exp(-raw))
    _like(s, out, "ddelta")[rows] = ddelta
    _like(s, out, "dB")[rows] = dB.flatten(2)
    _like(s, out, "dC")[rows] = dC.flatten(2)
    _like(s, out, "dinitial")[where] = dh
    out["dA"] = out.get("dA", 0) + dA.sum(0)
    out["dD"] = out.get("dD", 0) + (gy * u).sum((0, 1))
    out["dbias"] = out.get("dbias", 0) + ddelta.sum((0, 1))


def _exact_adamw(s):
    g, w = s["g"].double(), s["w"].double()
    m, v = (1 - BETA1) * g, (1 - BETA2) * g * g         # (the first step: the states are zero)
    new = w - RATE * (s["decay"].double() * w + (m / (1 - BETA1)) / (torch.sqrt(v / (1 - BETA2)) + EPS))
    out = {"w": new}
    if s["case"]["bits"] == 32:
        out.update(m=m, v=v)
    else:
        codes = torch.arange(127, device="cuda")
        top, low = codes // 8, codes % 8
        values = torch.where(top > 0, torch.exp2(top.double() - 7) * (1 + low / 8), low * 2.0 ** -9)
        between = (values[1:] + values[:-1]) / 2
        M, V = m.abs().view(-1, BLOCK).max(1).values.float(), v.view(-1, BLOCK).max(1).values.float()

        def coded(x):
            return values[torch.bucketize(x, between)]

        wide = M.double().repeat_interleave(BLOCK)
        out["m"] = torch.sign(m) * torch.where(wide > 0, coded(m.abs() / wide.clamp(min=1e-300) * 448), 0.0)
        wide = V.double().repeat_interleave(BLOCK)
        out["v"] = torch.where(v > 0, coded(torch.sqrt(v / wide.clamp(min=1e-300)) * 448).clamp(min=2.0 ** -9), 0.0)
        out.update(M=M.double(), V=V.double())
    if s["copy"] is not None:
        out["copy"] = new
    return out
