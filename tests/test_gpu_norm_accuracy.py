"""Layer norm where a row's statistics are hard: rows far from zero, gates far from it and at their ends, more rows than work-groups, very many for one weight.

Tolerances, in half steps of fp32 (2^-24), of operations as test_gpu_layers.py counts them (64 for a row's sum and what follows).  A row's mean is found, then the mean of what is left of it: the first
is off by at most 64 of them of the mean size of the elements, what is left by half a step of itself, and the second mean by 64 of the mean size of what is left.  So x - mean is off by
64 x 2^-24 (|x - mean| + mean |x - mean| + 64 x 2^-24 mean |x|), and not by steps of x itself."""
import math

import pytest
import torch

import layer_ref as ref

pytestmark = pytest.mark.gpu
STEP, OPERATIONS = 2.0 ** -24, 64


def rows_far_from_zero(channels, seed):
    """Constant rows; rows that lie close around 1500 and 10,000; one that is 1000 in one place only; an ordinary one."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    constant = torch.tensor([0.1, 132.7, 1234.567, 1e4 + 1 / 3, -771.3]).repeat(4) * (1 + torch.rand(20, generator=gen) / 8)
    single = r(1, channels) / 16
    single[0, channels // 2] = 1000.0
    return torch.cat([constant[:, None].expand(20, channels), 1500 + r(4, channels) / 100, 1e4 + r(4, channels) / 16, single, r(3, channels)]), 20


def left(x, epsilon=1e-5):
    """x' in 64 bits, what x - mean and the length are off by together, relative to the length, and the length."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    d, most = x - mean, x.abs().mean(-1, keepdim=True)
    length = torch.sqrt((d * d).mean(-1, keepdim=True) + epsilon)
    # (the squares are of elements less the first mean, and what that adds to them is taken off again)
    off = (d.abs() + d.abs().mean(-1, keepdim=True) + OPERATIONS * STEP * most) / length + (d / length).abs() * (1 + (OPERATIONS * STEP * most / length) ** 2)
    return d / length, off, length


# 16 lanes a row, a wavefront, several wavefronts (gradients: a wavefront with 16 and 32 elements a lane, several with 8 and 16); of sizes that a 16-byte access fits and others
CHANNELS = [3, 100, 128, 132, 300, 336, 500, 512, 700, 1001, 1024, 1500, 2048, 2050, 5000, 8200, 16383]


@pytest.mark.parametrize("channels", CHANNELS)
def test_rows_far_from_zero(channels):
    from genn_amd.sequence import LayerNorm
    x, constant = rows_far_from_zero(channels, channels)
    gen = torch.Generator().manual_seed(1)
    w, b, dout = (torch.randn(*s, generator=gen) for s in ((channels,), (channels,), x.shape))
    out, dx, dw = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda(), torch.zeros(channels).cuda()
    op = LayerNorm(1, x.shape[0], channels)
    op.bind(x=x.cuda(), weight=w.cuda(), bias=b.cuda(), out=out)
    op.run()
    op.bind_gradients(out=dout.cuda(), x=dx, weight=dw)
    op.backward()
    out, dx, dw = (t.cpu().double() for t in (out, dx, dw))
    hat, off, length = left(x)
    w, b, dout = w.double(), b.double(), dout.double()
    unit = OPERATIONS * STEP
    far = (out - (hat * w + b)).abs() - (STEP * (hat * w + b).abs() + unit * (off * w.abs()) + 2 * STEP * ((hat * w).abs() + b.abs()))
    assert (far <= 0).all(), (int(far.argmax()) // channels, float(far.max()))
    # (a row whose elements are all the same is nothing but the bias, to what steps of steps leave)
    assert ((out - b)[:constant].abs() <= STEP * b.abs() + 2 * STEP * b.abs() + unit * unit * 2 * x[:constant].double().abs() / math.sqrt(1e-5) * w.abs()).all()
    want, size = (dout * hat).sum(0), (dout.abs() * off).sum(0)
    assert ((dw - want).abs() <= STEP * want.abs() + 2 * unit * size).all()
    v = dout * w
    along, alongsize = (v * hat).mean(-1, keepdim=True), (v.abs() * off).mean(-1, keepdim=True)
    want = (v - v.mean(-1, keepdim=True) - hat * along) / length
    # (the length is off by x - mean's errors squared and more: counted with off, which has them relative to x')
    size = (v.abs() + v.abs().mean(-1, keepdim=True) + off * alongsize) / length
    size = size * (1 + (OPERATIONS * STEP * x.double().abs().mean(-1, keepdim=True) / length) ** 2)
    assert ((dx - want).abs() <= STEP * want.abs() + 2 * unit * size).all()


@pytest.mark.parametrize("rows, channels, dtype", [(70000, 64, "bfloat16"), (20000, 300, "float32"), (9000, 512, "float16"), (5000, 2048, "bfloat16"), (2500, 8200, "bfloat16"), (9000, 1000, "bfloat16")])
def test_more_rows_than_work_groups_take_at_once(rows, channels, dtype):
    """Each work-group has several rows one after another, of which the next is on its way."""
    from genn_amd.sequence import LayerNorm
    T = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}[dtype]
    gen = torch.Generator().manual_seed(rows)
    x, z, d = (torch.randn(rows, channels, generator=gen).to(T) for _ in range(3))
    w, b = (torch.randn(channels, generator=gen) for _ in range(2))
    for gate in (None, z):
        out, dx = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda()
        dz, dw, db = torch.zeros_like(x).cuda(), torch.zeros(channels).cuda(), torch.zeros(channels).cuda()
        op = LayerNorm(1, rows, channels, dtype=dtype)
        op.bind(x=x.cuda(), weight=w.cuda(), bias=b.cuda(), gate=None if gate is None else gate.cuda(), out=out)
        op.run()
        op.bind_gradients(out=d.cuda(), x=dx, weight=dw, bias=db, gate=None if gate is None else dz)
        op.backward()
        want, size = ref.layer_norm(x, w, b, gate)
        found, sizes = ref.layer_norm(x, w, b, gate, dout=d)
        least = torch.finfo(T).smallest_normal * torch.finfo(T).eps
        for name, got, value, most, t, n in (("out", out, want, size, T, OPERATIONS), ("dx", dx, found["dx"], sizes["dx"], T, 2 * OPERATIONS),
                                             ("dweight", dw, found["dweight"], sizes["dweight"], torch.float32, 2 * OPERATIONS + rows // 512), ("dbias", db, found["dbias"], sizes["dbias"], torch.float32, 2 * OPERATIONS + rows // 512)):
            off = (got.cpu().double() - value).abs() - (torch.finfo(t).eps / 2 * value.abs() + n * STEP * most * (1 + torch.finfo(t).eps) + least)
            assert (off <= 0).all(), (name, float(off.max()), int((off > 0).sum()))
        if gate is not None:
            off = (dz.cpu().double() - found["dgate"]).abs() - (torch.finfo(T).eps / 2 * found["dgate"].abs() + 2 * OPERATIONS * STEP * sizes["dgate"] * (1 + torch.finfo(T).eps) + least)
            assert (off <= 0).all()


def test_gates_far_from_zero():
    """Rows of which x' is 1 exactly (all elements 1, rms, no epsilon), so that out is the gate's own z sigmoid(z).

    Steps of fp32 relative to it: the exponential one step (2 x 2^-24) and half a step of its argument, which is below one half; the sum with 1, a reciprocal of one step, and two
    products: 1 + 2 + 1/2 x 1/2 + 2 + 2, counted as 8 x 2^-24; and one rounding less than that for each of the products of the slope, s (1 + z (1 - s)), that adds up terms of either sign."""
    from genn_amd.sequence import LayerNorm
    z = torch.cat([torch.linspace(-80, 80, 4001), torch.linspace(-3, 3, 1000), torch.tensor([0.0, -0.0, -1.2784645])])
    n = z.numel()
    z, x = z.repeat_interleave(8).view(n, 8), torch.ones(n, 8)
    out, dz, dout = torch.zeros(n, 8).cuda(), torch.zeros(n, 8).cuda(), torch.full((n, 8), 0.7)
    op = LayerNorm(1, n, 8, epsilon=0.0, rms=True)
    op.bind(x=x.cuda(), gate=z.cuda(), out=out)
    op.run()
    op.bind_gradients(out=dout.cuda(), gate=dz)
    op.backward()
    z = z.double()
    s = torch.sigmoid(z)
    want = z * s
    off = (out.cpu().double() - want).abs() / (want.abs() + 2.0 ** -126)
    assert (off <= 8 * STEP).all(), (float(z.reshape(-1)[int(off.argmax())]), float(off.max() / STEP))
    want, size = dout.double() * s * (1 + z * torch.sigmoid(-z)), dout.double() * s * (1 + z.abs() * torch.sigmoid(-z))
    off = (dz.cpu().double() - want).abs() / size
    assert (off <= 16 * STEP).all(), (float(z.reshape(-1)[int(off.argmax())]), float(off.max() / STEP))


@pytest.mark.parametrize("gate", [False, True])
def test_gates_and_rows_at_their_ends(gate):
    """Gates of an infinity and of none; what they give is what the formulas give."""
    from genn_amd.sequence import LayerNorm
    for dtype in ("float32", "bfloat16"):
        T = torch.float32 if dtype == "float32" else torch.bfloat16
        z = torch.tensor([math.inf, -math.inf, math.nan, 1e30, -1e30, 200.0, -200.0, 0.0])
        x, out = torch.ones(1, 8).to(T), torch.zeros(1, 8).to(T).cuda()
        op = LayerNorm(1, 1, 8, epsilon=0.0, rms=True, dtype=dtype)
        op.bind(x=x.cuda(), gate=z.to(T).view(1, 8).cuda() if gate else None, out=out)
        op.run()
        got = out.cpu().double()[0]
        if not gate:
            assert torch.all(got == 1.0)
            continue
        assert got[0] == math.inf and torch.isnan(got[1]) and torch.isnan(got[2]) and got[3] == float(z.to(T)[3]) and got[4] == 0.0 and got[5] == 200.0 and got[6].abs() < 1e-37 and got[7] == 0.0


def test_weights_of_very_many_rows():
    """A lane adds up at most 256 rows in 32 bits and a work-group 16 lanes' behind that, each addition off by at most half a step of the sum; then 64 bits.  Equal values of one sign lose most."""
    from genn_amd.sequence import LayerNorm
    rows = 64_000_000
    value = 0.901
    x = torch.zeros(rows, 1, device="cuda")
    d = torch.full((rows, 1), value, device="cuda")
    db = torch.zeros(1, device="cuda")
    op = LayerNorm(1, rows, 1)
    op.bind(x=x)
    op.bind_gradients(out=d, bias=db)
    op.backward()
    want = rows * float(torch.tensor(value).double())
    assert abs(float(db.double()) - want) <= want * STEP * (1 + 256 + 16), (float(db), want)


def test_gradients_in_fp32_are_as_exact_as_elementary_operations_in_fp32():
    """Against the same formulas of torch in 32 bits (weights' sums in 64): root mean squares of the errors, from 64 bits, of 19 million elements and 1332 weights.

    Weights: a product is off by some 8e-8 of itself, as theirs.  A lane adds up five rows in fp32: nine half steps squared a row and lane of a partial sum, 36 in 19 rows of four lanes, and one rounding of
    their sum, 19 in 19: 0.41 x 2^-24 sqrt(36 / 19 + 1) = 4.2e-8 beside the 8e-8, 1.13 of them.  Gates: the exponential and the reciprocal are off by a step each instead of half of one.  1.2 is above both."""
    from genn_amd.sequence import LayerNorm
    rows, channels, total = 14442, 333, {}
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        x, z, d, w = r(rows, channels) * torch.exp(r(rows, 1)) + r(rows, 1), r(rows, channels), r(rows, channels), 1 + r(channels) / 8
        got = dict(dx=torch.zeros_like(x), dgate=torch.zeros_like(x), dweight=torch.zeros_like(w))
        op = LayerNorm(1, rows, channels, rms=True)
        op.bind(x=x, weight=w, gate=z)
        op.bind_gradients(out=d, x=got["dx"], gate=got["dgate"], weight=got["dweight"])
        op.backward()

        def form(x, z, d, w):
            s = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
            hat, sig = x * s, torch.sigmoid(z)
            dgate, d = d * (hat * w) * sig * (1 + z * (1 - sig)), d * z * sig
            dweight, d = (d * hat).sum(0, dtype=torch.float64), d * w
            return dict(dx=(d - hat * (d * hat).mean(-1, keepdim=True)) * s, dgate=dgate, dweight=dweight)

        plain, exact = form(x, z, d, w), form(*(t.double() for t in (x, z, d, w)))
        for k in exact:
            off = total.setdefault(k, [0.0, 0.0])
            off[0] += float(((got[k].double() - exact[k]) ** 2).sum())
            off[1] += float(((plain[k].float().double() - exact[k]) ** 2).sum())
    for k, (own, plain) in total.items():
        assert math.sqrt(own / plain) <= 1.2, (k, math.sqrt(own / plain))
