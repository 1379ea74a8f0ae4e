"""The gated delta rule, layer norm and dropout, as cases that can be prepared, run and compared.

A case is one pass of a user's program through one operator: a gated delta rule over prompts, its gradients in training, or one token of every
running sequence; layer norm (of whole rows, or of a row's heads with a gate) or its gradients; or dropout, onto a residual or as its gradient.
"""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CHUNK = 64              # rows that the plain form of the delta rule takes together
EPS_KEYS, EPS_NORM = 1e-6, 1e-5


def listed():
    return [
        # A prompt through one layer: heads that share keys two by two; few enough that only a split over time fills the chip.
        dict(name="delta_prompt", op="delta", sequences=1, length=4096, heads=32, key_heads=16, keys=128, values=128, type="bfloat16"),
        # Prompts of very different lengths (none and one row among them) whose states lie in a pool; sizes that no tile divides.
        dict(name="delta_ragged_prompts", op="delta_ragged", sequences=33, rows=8011, heads=6, key_heads=3, keys=100, values=72, type="float16"),
        # Gradients in a training step: the largest.
        dict(name="delta_training", op="delta_backward", sequences=8, length=2048, heads=16, key_heads=16, keys=128, values=128, type="bfloat16"),
        # Gradients of a small experiment in 32 bits; no size is even.
        dict(name="delta_training_small", op="delta_backward", sequences=3, length=301, heads=3, key_heads=1, keys=33, values=47, type="float32"),
        # One token of one sequence: nothing but latency.
        dict(name="delta_token_one", op="delta_token", sequences=1, heads=32, key_heads=16, keys=128, values=128, type="bfloat16"),
        # One token of many sequences: reads and writes all their states.
        dict(name="delta_token_batch", op="delta_token", sequences=256, heads=32, key_heads=16, keys=128, values=128, type="bfloat16"),
        # The rows of a prompt in front of a layer.
        dict(name="norm_prompt", op="norm", rows=4096, heads=1, width=4096, rms=False, bias=True, gate=False, type="bfloat16"),
        # Every head of a token's few rows, times the gate, behind the recurrence.
        dict(name="norm_heads_token", op="norm", rows=16, heads=32, width=128, rms=True, bias=False, gate=True, type="float16"),
        # Gradients in a training step: rows, and sums over rows for weights.
        dict(name="norm_training", op="norm_backward", rows=16384, heads=1, width=2048, rms=False, bias=True, gate=False, type="bfloat16"),
        # Gradients of the heads with their gate, in 32 bits, of an odd size.
        dict(name="norm_heads_training", op="norm_backward", rows=2407, heads=6, width=333, rms=True, bias=False, gate=True, type="float32"),
        # What a layer found, dropped at random, onto the residual in a training step.
        dict(name="dropout_training", op="dropout", rows=16384, width=2048, probability=0.1, residual=True, type="bfloat16"),
        # The same of a small experiment in 32 bits, as its gradient draws it again.
        dict(name="dropout_gradient_small", op="dropout_backward", rows=903, width=141, probability=0.25, residual=False, type="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every operator alike, sizes over the range of the listed ones and below."""
    op = rng.choice(["delta", "delta_ragged", "delta_backward", "delta_token", "norm", "norm_backward", "dropout"])
    case = dict(op=op, type=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]))
    if op == "dropout":
        width = _log(rng, 5, 5000)
        op = rng.choice([op, "dropout_backward"])
        return dict(case, op=op, rows=_log(rng, 1, 30000000 // width), width=width, probability=round(rng.uniform(0.02, 0.6), 3),
                    residual=op == "dropout" and rng.choice([False, True]))
    if op.startswith("norm"):
        heads = rng.choice([1, 1, rng.randint(2, 32)])
        width = _log(rng, 9, 8000) if heads == 1 else _log(rng, 30, 256)
        rms = rng.choice([False, True])
        return dict(case, rows=_log(rng, 1, 30000000 // (heads * width)), heads=heads, width=width, rms=rms, bias=not rms, gate=rng.choice([False, True]))
    case["key_heads"] = rng.randint(1, 16)
    case["heads"] = case["key_heads"] * rng.choice([1, 1, 2, 3])
    case["keys"], case["values"] = rng.choice([rng.randint(8, 128), 64, 128, 128]), rng.choice([rng.randint(8, 256), 64, 128, 128])
    if op == "delta_token":
        return dict(case, sequences=_log(rng, 1, 250))
    most = 150000000 // (case["heads"] * case["keys"] * case["values"] // 20)       # rows: a third and more below the largest listed case in all
    if op == "delta_ragged":
        return dict(case, sequences=rng.randint(1, 40), rows=_log(rng, 50, min(most, 8000)))
    sequences = _log(rng, 1, 12)
    return dict(case, sequences=sequences, length=_log(rng, 2, max(3, min(6000, most // sequences))))


def _lengths(case):
    """Rows of each sequence: of the packed ones as cut at random places, so that some are long, some short and now and then one empty."""
    if case["op"] != "delta_ragged":
        return [case.get("length", 1)] * case["sequences"]
    rng = random.Random(case["sequences"] * 7919 + case["rows"])
    cuts = sorted(rng.randint(0, case["rows"]) for _ in range(case["sequences"] - 1))
    if len(cuts) > 3:
        cuts[1], cuts[3] = cuts[0], min(cuts[2] + 1, cuts[4] if len(cuts) > 4 else cuts[3])      # one without rows, one of one
    ends = [0] + cuts + [case["rows"]]
    return [b - a for a, b in zip(ends, ends[1:])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    T = TYPES[case["type"]]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    def room(*shape, dtype=T):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    state = dict(case=case, training=case["op"].endswith("backward"))
    if case["op"].startswith("dropout"):
        rows, width = case["rows"], case["width"]
        state.update(x=normal(rows, width, dtype=T), residual=normal(rows, width, dtype=T) if case["residual"] else None, out=room(rows, width))
        # the seed of the run, and the number of the step and layer
        state.update(key=random.Random(seed).getrandbits(64), call=random.Random(seed + 1).getrandbits(40))
        if own:
            from genn_amd.sequence import Dropout
            plan = Dropout(1, rows, width, case["probability"], seed=state["key"], dtype=case["type"])
            if state["training"]:
                plan.bind_gradients(out=state["x"], x=state["out"])
            else:
                plan.bind(x=state["x"], residual=state["residual"], out=state["out"])
            state["plan"] = plan
        return state
    if case["op"].startswith("norm"):
        rows, heads, width = case["rows"], case["heads"], case["width"]
        # activations with an offset and a spread of their own for each row
        state["x"] = (normal(rows, heads, width) * torch.exp(normal(rows, heads, 1)) + normal(rows, heads, 1)).to(T)
        # the gate lies beside other projections of the same rows
        state["gate"] = normal(rows, heads * width + 24, dtype=T)[:, :heads * width].view(rows, heads, width) if case["gate"] else None
        state["weight"] = 1 + normal(width, scale=0.1)
        state["bias"] = normal(width, scale=0.1) if case["bias"] else None
        state["out"] = room(rows, heads, width)
        if state["training"]:
            state["dout"] = normal(rows, heads, width, dtype=T)
            state["dx"], state["dgate"] = room(rows, heads, width), room(rows, heads, width) if case["gate"] else None
            state["dweight"], state["dbias"] = room(width, dtype=torch.float32), room(width, dtype=torch.float32) if case["bias"] else None
        if own:
            from genn_amd.sequence import LayerNorm
            plan = LayerNorm(rows, heads, width, epsilon=EPS_NORM, rms=case["rms"], dtype=case["type"])
            plan.bind(x=state["x"], weight=state["weight"], bias=state["bias"], gate=state["gate"], out=state["out"])
            if state["training"]:
                plan.bind_gradients(out=state["dout"], x=state["dx"], weight=state["dweight"], bias=state["dbias"], gate=state["dgate"])
            state["plan"] = plan
        return state

    H, G, K, V = case["heads"], case["key_heads"], case["keys"], case["values"]
    lengths = _lengths(case)
    S, rows = len(lengths), sum(lengths)
    token, ragged, backward = case["op"] == "delta_token", case["op"] == "delta_ragged", state["training"]
    spare = 5 if ragged else 0          # rows behind the last sequence
    first = torch.tensor([0] + lengths).cumsum(0)
    longest = max(lengths)
    state.update(lengths=lengths, first=first.cuda(), longest=longest)
    # where each row lies among [sequences, longest], and back
    at = torch.repeat_interleave(torch.arange(S), torch.tensor(lengths))
    state["place"] = (at * longest + torch.arange(rows) - first[at]).cuda()
    state["offsets"] = first.to(torch.int32).cuda() if ragged else None
    places = S + 3 if token or ragged else S
    state["slots"] = torch.randperm(places, generator=gen, device="cuda")[:S].to(torch.int32) if places > S else None
    state["where"] = state["slots"].long() if places > S else torch.arange(S, device="cuda")
    # queries, keys and values as one projection gives them, side by side in a row
    wide = normal(rows + spare, 2 * G * K + H * V, dtype=T)
    state["q"], state["k"], state["v"] = wide[:, :G * K], wide[:, G * K:2 * G * K], wide[:, 2 * G * K:]
    # decays as a head's own rate times a softplus of the input, from a few rows to thousands of them
    step = torch.nn.functional.softplus(normal(rows + spare, H) + torch.log(torch.expm1(torch.exp(uniform(math.log(1e-3), math.log(1e-1), H)))))
    state["g"] = -uniform(1, 16, H) * step
    state["beta"] = torch.sigmoid(normal(rows + spare, H))
    state["out"] = room(rows + spare, H * V)
    state["initial"] = normal(places, H, K, V, scale=0.3) if token or ragged or backward else None
    state["final"] = state["initial"] if token else room(places, H, K, V, dtype=torch.float32)
    if backward:
        state["dout"], state["dfinal"] = normal(rows, H * V, dtype=T), normal(places, H, K, V, scale=0.3)
        state["dq"], state["dk"], state["dv"] = room(rows, G * K), room(rows, G * K), room(rows, H * V)
        state["dg"], state["dbeta"] = room(rows, H, dtype=torch.float32), room(rows, H, dtype=torch.float32)
        state["dinitial"] = room(places, H, K, V, dtype=torch.float32)
    if own:
        from genn_amd.sequence import GatedDeltaRule
        plan = GatedDeltaRule(S, longest, H, K, V, key_heads=G, dtype=case["type"], normalise=True, epsilon=EPS_KEYS)
        plan.bind(q=state["q"], k=state["k"], v=state["v"], g=state["g"], beta=state["beta"], out=state["out"], initial_state=state["initial"],
                  final_state=state["final"], offsets=state["offsets"], slots=state["slots"])
        if backward:
            plan.bind_gradients(out=state["dout"], final_state=state["dfinal"], q=state["dq"], k=state["dk"], v=state["dv"], g=state["dg"],
                                beta=state["dbeta"], initial_state=state["dinitial"])
        state["plan"] = plan
    return state


def run(state):
    op = state["case"]["op"]
    if op.startswith("dropout"):
        if own:
            (state["plan"].backward if state["training"] else state["plan"].run)(state["call"])
        else:
            _dropout(state)
        return {"out": state["out"]}
    if state["training"]:
        if own:
            state["plan"].backward()
        else:
            (_norm_backward if op.startswith("norm") else _delta_backward)(state)
        return {k: state[k] for k in ("dx", "dgate", "dweight", "dbias", "dq", "dk", "dv", "dg", "dbeta", "dinitial") if state.get(k) is not None}
    if own:
        state["plan"].run()
    else:
        (_norm if op == "norm" else _delta_token if op == "delta_token" else _delta)(state)
    return {k: state[k] for k in ("out", "final") if k in state}


# ---- plain forms: elementary operations in 32 bits

def _philox(c0, c1, c2, c3, key):
    """Philox4x32-10 on int64 tensors of 32-bit words: its four words."""
    k0, k1 = key & 0xffffffff, key >> 32
    for _ in range(10):
        p = [_product(0xD2511F53, c0), _product(0xCD9E8D57, c2)]
        c0, c1, c2, c3 = p[1][0] ^ c1 ^ k0, p[1][1], p[0][0] ^ c3 ^ k1, p[0][1]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c0, c1, c2, c3


def _product(a, x):
    """The upper and the lower 32 bits of a * x, by halves of a: 63 bits hold each."""
    low, high = (a & 0xffff) * x, (a >> 16) * x
    total = low + ((high & 0xffff) << 16)
    return (high >> 16) + (total >> 32), total & 0xffffffff


def _dropout(s):
    case, x = s["case"], s["x"]
    rows, width = x.shape
    groups = -(-width // 8)         # eight elements share a draw: 16 bits each, the lower half of a word first; a row begins a new group
    group = torch.arange(rows * groups, device="cuda")
    words = torch.stack(_philox(group & 0xffffffff, group >> 32, torch.full_like(group, s["call"] & 0xffffffff), torch.full_like(group, s["call"] >> 32), s["key"]), 1)
    halves = torch.stack([words & 0xffff, words >> 16], 2).view(rows, groups * 8)[:, :width]
    dropped = round(case["probability"] * 65536)
    y = torch.where(halves >= dropped, x.float() * (65536 / (65536 - dropped)), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["out"].copy_(y)


def _normed(s):
    x = s["x"].float()
    if not s["case"]["rms"]:
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS_NORM)
    return x * r, r


def _norm(s):
    y = _normed(s)[0] * s["weight"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gate"] is not None:
        z = s["gate"].float()
        y = y * z * torch.sigmoid(z)
    s["out"].copy_(y)


def _norm_backward(s):
    hat, r = _normed(s)
    d = s["dout"].float()
    if s["gate"] is not None:
        z = s["gate"].float()
        sig = torch.sigmoid(z)
        y = hat * s["weight"]
        if s["bias"] is not None:
            y = y + s["bias"]
        s["dgate"].copy_(d * y * sig * (1 + z * (1 - sig)))
        d = d * z * sig
    if s["bias"] is not None:
        s["dbias"].copy_(d.sum((0, 1), dtype=torch.float64))
    s["dweight"].copy_((d * hat).sum((0, 1), dtype=torch.float64))
    d = d * s["weight"]
    dx = d - hat * (d * hat).mean(-1, keepdim=True)
    if not s["case"]["rms"]:
        dx = dx - d.mean(-1, keepdim=True)
    s["dx"].copy_(dx * r)


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS_KEYS)


def _delta_token(s):
    c = s["case"]
    S, H, G, K, V = c["sequences"], c["heads"], c["key_heads"], c["keys"], c["values"]
    q, k = (_unit(s[n].float().view(S, G, K)).repeat_interleave(H // G, 1) for n in "qk")
    h = torch.exp(s["g"])[..., None, None] * s["final"][s["where"]]
    u = s["beta"][..., None] * (s["v"].float().view(S, H, V) - (h * k[..., None]).sum(2))
    h = h + k[..., None] * u[..., None, :]
    s["final"][s["where"]] = h
    s["out"].copy_(((h * q[..., None]).sum(2) * K ** -0.5).view(S, H * V))


def _laid(s, x, heads, width):
    """Packed rows as [sequences, heads, chunks, CHUNK, width], zero where a sequence has no row."""
    S, n = len(s["lengths"]), -(-s["longest"] // CHUNK)
    wide = x.new_zeros(S * s["longest"], heads * width, dtype=torch.float32)
    wide[s["place"]] = x[:s["place"].shape[0]].float()
    whole = x.new_zeros(S, n * CHUNK, heads, width, dtype=torch.float32)
    whole[:, :s["longest"]] = wide.view(S, s["longest"], heads, width)
    return whole.view(S, n, CHUNK, heads, width).permute(0, 3, 1, 2, 4).contiguous()


def _packed(s, x, out):
    """The other way round."""
    S, heads, n, _, width = x.shape
    whole = x.permute(0, 2, 3, 1, 4).reshape(S, n * CHUNK, heads * width)[:, :s["longest"]].reshape(S * s["longest"], heads * width)
    out[:s["place"].shape[0]] = whole[s["place"]].to(out.dtype)


def _swap(x):
    return x.transpose(-1, -2).contiguous()


def _delta_parts(s):
    """All chunks at once: everything that does not need a state."""
    c = s["case"]
    H, G, K, V = c["heads"], c["key_heads"], c["keys"], c["values"]
    p = dict(qraw=_laid(s, s["q"], G, K), kraw=_laid(s, s["k"], G, K), v=_laid(s, s["v"], H, V))
    p["q"], p["k"] = (_unit(p[n]).repeat_interleave(H // G, 1) for n in ("qraw", "kraw"))
    p["q"] = p["q"] * K ** -0.5
    p["beta"] = _laid(s, s["beta"], H, 1)
    sums = _laid(s, s["g"], H, 1)[..., 0].double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device="cuda").tril()
    p["decay"] = torch.exp((sums[..., :, None] - sums[..., None, :]).masked_fill(lower == 0, -math.inf)).float()
    p["kk"], p["qk"] = p["k"] @ _swap(p["k"]), p["q"] @ _swap(p["k"])
    p["before"] = torch.exp(sums).float()[..., None]                              # since the chunk's beginning
    p["behind"] = torch.exp(sums[..., -1:] - sums).float()[..., None]             # until its end
    p["strict"] = lower.tril(-1)
    p["L"] = p["beta"] * p["kk"] * p["decay"] * p["strict"]
    p["P"] = p["qk"] * p["decay"]
    # (I + L)^-1 by halves: of a block [[A, 0], [B, D]] it is [[A', 0], [-D' B A', D']]
    t = torch.eye(CHUNK, device="cuda").expand_as(p["L"]).contiguous()
    size = 1
    at = torch.arange(CHUNK, device="cuda")
    while size < CHUNK:
        block = ((at[:, None] // size == at[None, :] // size + 1) & (at[None, :] // size % 2 == 0)).float()
        t = t - t @ (p["L"] * block) @ t
        size *= 2
    p["T"] = t
    return p


def _states(s, p):
    """The state in front of every chunk and behind the last one, and U."""
    H, K, V = s["case"]["heads"], s["case"]["keys"], s["case"]["values"]
    h = s["initial"][s["where"]] if s["initial"] is not None else torch.zeros(len(s["lengths"]), H, K, V, device="cuda")
    W, U = p["T"] @ (p["beta"] * p["before"] * p["k"]), p["T"] @ (p["beta"] * p["v"])
    keys = _swap(p["behind"] * p["k"])
    states = []
    for n in range(U.shape[2]):
        states.append(h)
        U[:, :, n] -= W[:, :, n] @ h
        h = p["before"][:, :, n, -1:] * h + keys[:, :, n] @ U[:, :, n]
    return (torch.stack(states, 2) if states else h[:, :, None][:, :, :0]), U, h


def _delta(s):
    p = _delta_parts(s)
    h, U, last = _states(s, p)
    _packed(s, p["before"] * (p["q"] @ h) + p["P"] @ U, s["out"])
    s["final"][s["where"]] = last


def _delta_backward(s):
    c = s["case"]
    H, G, K, V = c["heads"], c["key_heads"], c["keys"], c["values"]
    p = _delta_parts(s)
    h, U, last = _states(s, p)
    dout = _laid(s, s["dout"], H, V)
    Tt, dU = _swap(p["T"]), _swap(p["P"]) @ dout
    direct = _swap(p["before"] * p["q"]) @ dout
    keys, kt = p["behind"] * p["k"], _swap(p["k"])
    d = s["dfinal"][s["where"]]
    behind, dR = [], torch.zeros_like(dU)
    for n in reversed(range(dU.shape[2])):
        behind.append(d)
        dU[:, :, n] += keys[:, :, n] @ d
        dR[:, :, n] = Tt[:, :, n] @ dU[:, :, n]
        d = p["before"][:, :, n, -1:] * d + direct[:, :, n] - kt[:, :, n] @ (p["beta"] * p["before"])[:, :, n].mul(dR[:, :, n])
    s["dinitial"][s["where"]] = d
    d = torch.stack(behind[::-1], 2)
    dv = p["beta"] * dR
    dX = -dv * p["before"]
    dL, dP = -(dR @ _swap(U)) * p["strict"], (dout @ _swap(U)) * p["decay"]
    dbeta = (dR * (p["v"] - p["before"] * (p["k"] @ h))).sum(-1) + (dL * p["decay"] * p["kk"]).sum(-1)
    dkk = dL * p["beta"] * p["decay"]
    dq = p["before"] * (dout @ _swap(h)) + dP @ p["k"]
    dk = dX @ _swap(h) + p["behind"] * (U @ _swap(d)) + _swap(dP) @ p["q"] + (dkk + _swap(dkk)) @ p["k"]
    # (with states and errors measured in units of the decay so far, outputs grow with it and values shrink)
    dsums = ((p["q"] * dq).sum(-1) - (p["v"] * dv).sum(-1)).double()
    after = torch.cat([h[:, :, 1:], last[:, :, None]], 2)
    dsums[..., -1] += (after * d).sum((-1, -2), dtype=torch.float64)
    dg = dsums.flip(-1).cumsum(-1).flip(-1)
    _packed(s, dv, s["dv"])
    _packed(s, dg[..., None].float(), s["dg"])
    _packed(s, dbeta[..., None], s["dbeta"])
    for name, raw, grad in (("dq", p["qraw"], dq * K ** -0.5), ("dk", p["kraw"], dk)):
        grad = grad.view(grad.shape[0], G, H // G, *grad.shape[2:]).sum(2)
        r = torch.rsqrt((raw * raw).sum(-1, keepdim=True) + EPS_KEYS)
        hat = raw * r
        _packed(s, r * (grad - hat * (hat * grad).sum(-1, keepdim=True)), s[name])


# ---- what a pass cannot do without

def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"].startswith("dropout"):
        n = case["rows"] * case["width"]
        return {"bytes": n * size * (3 if case["residual"] else 2), "flops": 12 * n}
    if case["op"].startswith("norm"):
        n, backward = case["rows"] * case["heads"] * case["width"], case["op"].endswith("backward")
        moved = n * size * ((3 if backward else 2) + case["gate"] * (2 if backward else 1))
        return {"bytes": moved + case["width"] * 4 * (1 + case["bias"]) * (2 if backward else 1), "flops": n * (24 if backward else 10)}
    H, G, K, V = case["heads"], case["key_heads"], case["keys"], case["values"]
    lengths = _lengths(case)
    rows, S = sum(lengths), len(lengths)
    row = (2 * G * K + 2 * H * V) * size + 2 * H * 4
    state = S * H * K * V * 4
    if case["op"] == "delta_backward":
        return {"bytes": rows * (row + (2 * G * K + H * V) * size + 2 * H * 4) + 3 * state, "flops": 21 * rows * H * K * V}
    return {"bytes": rows * row + state * (1 if case["op"] == "delta" else 2), "flops": 7 * rows * H * K * V}


# ---- the definitions in 64 bits, one row after another

def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_dropout if case["op"].startswith("dropout") else _exact_norm if case["op"].startswith("norm") else _exact_delta)(s)


def _exact_dropout(s):
    import numpy as np
    rows, width = s["x"].shape
    groups = -(-width // 8)
    u = np.uint64
    n = np.arange(rows * groups, dtype=u)
    low = u(0xffffffff)
    call, key = u(s["call"]), [u(s["key"] & 0xffffffff), u(s["key"] >> 32)]
    x = [n & low, n >> u(32), np.full_like(n, call & low), np.full_like(n, call >> u(32))]
    for _ in range(10):
        a, b = u(0xD2511F53) * x[0], u(0xCD9E8D57) * x[2]          # (32 bits times 32: 64 hold them)
        x = [(b >> u(32)) ^ x[1] ^ key[0], b & low, (a >> u(32)) ^ x[3] ^ key[1], a & low]
        key = [(key[0] + u(0x9E3779B9)) & low, (key[1] + u(0xBB67AE85)) & low]
    draws = np.stack([part for word in x for part in (word & u(0xffff), word >> u(16))], 1).reshape(rows, groups * 8)[:, :width]
    dropped = int(math.floor(s["case"]["probability"] * 65536 + 0.5))
    kept = torch.from_numpy((draws >= u(dropped)).astype(np.float64)).cuda()
    out = s["x"].double() * kept / (1 - dropped / 65536)
    return {"out": out if s["residual"] is None else out + s["residual"].double()}


def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    n = x.shape[-1]
    mean = 0.0 if s["case"]["rms"] else x.sum(-1, keepdim=True) / n
    deviation = torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / n + EPS_NORM)
    hat = (x - mean) / deviation
    plain = hat * w + (0.0 if s["bias"] is None else s["bias"].double())
    z = None if s["gate"] is None else s["gate"].double()
    gate = 1.0 if z is None else z / (1 + torch.exp(-z))
    if not s["training"]:
        return {"out": plain * gate}
    d = s["dout"].double()
    out = {}
    if z is not None:
        e = torch.exp(-z)
        out["dgate"] = d * plain * (1 + e + z * e) / (1 + e) ** 2
    inner = d * gate
    out["dweight"] = (inner * hat).sum((0, 1))
    if s["bias"] is not None:
        out["dbias"] = inner.sum((0, 1))
    v = inner * w
    centre = 0.0 if s["case"]["rms"] else v.sum(-1, keepdim=True) / n
    out["dx"] = (v - centre - hat * ((v * hat).sum(-1, keepdim=True) / n)) / deviation
    return out


def _exact_delta(s):
    c = s["case"]
    H, G, K, V, S, longest = c["heads"], c["key_heads"], c["keys"], c["values"], len(s["lengths"]), s["longest"]
    rows = s["place"].shape[0]

    def laid(x, heads, width):              # [rows of a sequence, sequences, heads, width]; no row: zero
        y = torch.zeros(S * longest, heads * width, dtype=torch.float64, device="cuda")
        y[s["place"]] = x[:rows].double()
        return y.view(S, longest, heads, width).transpose(0, 1).contiguous()

    def back(y, like):
        out = torch.zeros(like.shape, dtype=torch.float64, device="cuda")
        out[:rows] = y.transpose(0, 1).reshape(S * longest, -1)[s["place"]]
        return out

    raw = {n: laid(s[n], G, K) for n in "qk"}
    size = {n: torch.sqrt((raw[n] ** 2).sum(-1, keepdim=True) + EPS_KEYS) for n in "qk"}
    q, k = ((raw[n] / size[n]).repeat_interleave(H // G, 2) for n in "qk")
    v, g, beta = laid(s["v"], H, V), laid(s["g"], H, 1)[..., 0], laid(s["beta"], H, 1)
    scale = 1 / math.sqrt(K)
    h = s["initial"][s["where"]].double() if s["initial"] is not None else torch.zeros(S, H, K, V, dtype=torch.float64, device="cuda")

    def step(h, t):
        h = torch.exp(g[t])[..., None, None] * h
        error = v[t] - (k[t][..., None, :] @ h)[..., 0, :]
        return h, error, torch.addcmul(h, k[t][..., None], (beta[t] * error)[..., None, :])

    every = 64
    kept, out = [], torch.zeros_like(v)
    for t in range(longest):
        if t % every == 0:
            kept.append(h)
        h = step(h, t)[2]
        if not s["training"]:
            out[t] = scale * (q[t][..., None, :] @ h)[..., 0, :]
    if not s["training"]:
        final = s["final"].double()
        final[s["where"]] = h
        return {"out": back(out, s["out"]), "final": final}
    dout = laid(s["dout"], H, V)
    d = s["dfinal"][s["where"]].double()
    dq, dk, dv, dg, dbeta = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    for n in reversed(range(len(kept))):
        h, inside = kept.pop(), []
        last = min(longest, (n + 1) * every)
        for t in range(n * every, last):
            before, error, after = step(h, t)
            inside.append((before, error, after))
            h = after
        for t in reversed(range(n * every, last)):
            before, error, after = inside.pop()         # (the state times the decay, the error, the new state)
            dq[t] = scale * (after @ dout[t][..., None])[..., 0]
            d = torch.addcmul(d, scale * q[t][..., None], dout[t][..., None, :])
            du = (k[t][..., None, :] @ d)[..., 0, :]
            derror = beta[t] * du
            dbeta[t] = (du * error).sum(-1, keepdim=True)
            dv[t] = derror
            dk[t] = (d @ (beta[t] * error)[..., None])[..., 0] - (before @ derror[..., None])[..., 0]
            d = torch.addcmul(d, k[t][..., None], derror[..., None, :], value=-1.0)
            dg[t] = (d * before).sum((-1, -2))
            d = torch.exp(g[t])[..., None, None] * d
    found = dict(dv=back(dv, s["dv"]), dg=back(dg, s["dg"]), dbeta=back(dbeta, s["dbeta"]))
    for name, hat, grad in (("q", q, dq), ("k", k, dk)):
        grad = (grad - hat * (hat * grad).sum(-1, keepdim=True)).view(longest, S, G, H // G, K).sum(3) / size[name]
        found["d" + name] = back(grad, s["d" + name])
    dinitial = s["dinitial"].double()
    dinitial[s["where"]] = d
    return dict(found, dinitial=dinitial)
