"""Layer norm, its gradients and dropout through the C ABI against their restatements in 64 bits.

Tolerances.  A result is one rounding to its type (half a step) of what is computed in fp32.  The sums of a row are made of at most 16 elements a lane, 6 steps over
lanes and 16 wavefronts, one behind another: 40 operations, half a step of fp32 (2^-24) each at most, then some 20 more to the result, counted as 2^-24 of ``sizes``
each; exponential and division count among them.  Weights' gradients add what a lane adds up over its rows, and no more than 64 steps over the rows of a
work-group; the sums behind that are in 64 bits."""
import math

import pytest
import torch

import layer_ref as ref
from genn_amd import _abi
from genn_amd.genn_model import Array

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
OPERATIONS = 64


def close(name, got, want, size, dtype=torch.float32, operations=OPERATIONS):
    got = got.detach().cpu().double().reshape(want.shape)
    assert torch.isfinite(got).all(), name
    limit = torch.finfo(dtype).eps / 2 * want.abs() + operations * 2.0 ** -24 * size * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - want).abs() - limit
    worst = int(off.argmax()) if off.numel() else 0
    assert not off.numel() or off.max() <= 0, (name, worst, float(got.reshape(-1)[worst]), float(want.reshape(-1)[worst]), float(limit.reshape(-1)[worst]))


def generator(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen)


NORM = [
    # rows, heads, channels, type, rms, weight, bias, gate
    (1, 1, 1, "float32", False, True, True, False),
    (5, 1, 3, "float32", False, False, False, False),
    (7, 1, 8, "bfloat16", False, True, True, True),
    (33, 3, 128, "bfloat16", True, True, False, True),
    (17, 1, 129, "float16", False, True, True, True),
    (9, 2, 333, "float32", True, True, False, True),
    (300, 1, 512, "float16", False, True, True, False),
    (20, 1, 1000, "bfloat16", False, True, False, True),
    (3, 1, 1024, "float32", True, True, True, True),
    (6, 1, 1025, "float32", False, True, True, True),
    (40, 1, 2048, "bfloat16", False, True, True, False),
    (3, 1, 5000, "float16", False, True, True, True),
    (2, 1, 16384, "bfloat16", False, True, True, True),
    (2, 1, 16383, "float32", True, True, True, False),
    (5000, 1, 64, "float32", False, True, True, True),
]


@pytest.mark.parametrize("rows, heads, channels, dtype, rms, weight, bias, gate", NORM)
def test_layer_norm(rows, heads, channels, dtype, rms, weight, bias, gate):
    from genn_amd.sequence import LayerNorm
    T, r = TYPES[dtype], generator(rows + channels)
    x = (r(rows, heads, channels) * torch.exp(r(rows, heads, 1)) + r(rows, heads, 1)).to(T)
    z = r(rows, heads * channels + 24).to(T) if gate else None
    w, b = 1 + 0.3 * r(channels) if weight else None, 0.3 * r(channels) if bias else None
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    zc = None if z is None else z.cuda()[:, :heads * channels].view(rows, heads, channels)
    flat = None if z is None else z[:, :heads * channels].reshape(-1, channels)
    op = LayerNorm(rows, heads, channels, rms=rms, dtype=dtype)
    out = torch.full((rows, heads, channels), 7.0, dtype=T).cuda()
    op.bind(x=x.cuda(), weight=cuda(w), bias=cuda(b), gate=zc, out=out)
    op.run()
    torch.cuda.synchronize()
    want, size = ref.layer_norm(x.view(-1, channels), w, b, flat, 1e-5, rms)
    close("out", out, want, size, T)
    dout = r(rows, heads, channels).to(T)
    dx, dz = torch.full((rows, heads, channels), 7.0, dtype=T).cuda(), torch.full((rows, heads, channels), 7.0, dtype=T).cuda()
    dw, db = torch.full((channels,), 7.0).cuda(), torch.full((channels,), 7.0).cuda()
    op.bind_gradients(out=dout.cuda(), x=dx, weight=dw, bias=db, gate=dz if gate else None)
    op.backward()
    torch.cuda.synchronize()
    found, size = ref.layer_norm(x.view(-1, channels), w, b, flat, 1e-5, rms, dout=dout.view(-1, channels))
    close("dx", dx, found["dx"], size["dx"], T, 2 * OPERATIONS)
    close("dweight", dw, found["dweight"], size["dweight"], operations=2 * OPERATIONS)
    close("dbias", db, found["dbias"], size["dbias"], operations=2 * OPERATIONS)
    if gate:
        close("dgate", dz, found["dgate"], size["dgate"], T, 2 * OPERATIONS)
    # only some of them
    dx2, dw2 = torch.zeros_like(dx), torch.zeros_like(dw)
    op.bind_gradients(out=dout.cuda(), weight=dw2)
    op.backward()
    assert torch.equal(dw2, dw)
    op.bind_gradients(out=dout.cuda(), x=dx2)
    assert op.backward_workspace_bytes == 0
    op.backward()
    assert torch.equal(dx2, dx)


DROPOUT = [
    # sequences, length, channels, probability, type, residual
    (1, 1, 1, 0.5, "float32", False),
    (1, 3, 7, 0.3, "float16", True),
    (2, 5, 16, 0.1, "bfloat16", True),
    (1, 301, 141, 0.25, "float32", True),
    (3, 40, 1000, 0.9, "bfloat16", False),
    (1, 64, 24, 0.0, "float16", True),
    (1, 64, 24, 1.0, "bfloat16", True),
]


@pytest.mark.parametrize("sequences, length, channels, probability, dtype, residual", DROPOUT)
def test_dropout(sequences, length, channels, probability, dtype, residual):
    from genn_amd.sequence import Dropout
    T, r, seed, call = TYPES[dtype], generator(channels), 0x9876543212345678, 0x1234567890
    x, more = r(sequences, length, channels).to(T), r(sequences, length, channels).to(T) if residual else None
    x.view(-1)[::5] = math.inf
    keep, factor = ref.kept(sequences * length, channels, probability, seed, call)
    keep = keep.view(x.shape)
    x[keep & torch.isinf(x)] = 2.0             # (what is dropped leaves nothing, also of infinities)
    out = torch.full_like(x, 7.0).cuda()
    op = Dropout(sequences, length, channels, probability, seed=seed, dtype=dtype)
    op.bind(x=x.cuda(), residual=None if more is None else more.cuda(), out=out)
    op.run(call)
    kept = torch.where(keep, x.double(), 0.0) * factor
    want = kept + (0.0 if more is None else more.double())
    # (the factor, the product and the sum: three operations of fp32 behind one rounding)
    close("out", out, want, kept.abs() + want.abs(), T, 3)
    before = out.clone()
    number = torch.tensor([call], dtype=torch.int64).cuda()
    out.fill_(7.0)
    op.run(number)
    assert torch.equal(out, before)
    # the gradient, in place, of rows that lie apart: the same elements
    wide = torch.full((sequences, length, channels + 3), 7.0, dtype=T).cuda()
    wide[..., :channels] = x.cuda()
    op.bind_gradients(out=wide[..., :channels], x=wide[..., :channels])
    op.backward(call)
    close("dx", wide[..., :channels], kept, kept.abs(), T, 3)
    assert torch.all(wide[..., channels:] == 7.0)


def test_norm_in_place_and_of_strided_heads():
    from genn_amd.sequence import LayerNorm
    r = generator(4)
    wide = r(12, 5 * 32 + 8).bfloat16().cuda()
    gate = r(12, 5, 32).bfloat16().cuda()
    want, size = ref.layer_norm(wide[:, 4:164].reshape(-1, 32).cpu(), gate=gate.view(-1, 32).cpu(), rms=True)
    kept = wide.clone()
    heads = wide[:, 4:164].view(12, 5, 32)
    op = LayerNorm(12, 5, 32, rms=True, dtype="bfloat16")
    op.bind(x=heads, gate=gate, out=heads)
    op.run()
    close("out", heads.reshape(-1, 32), want, size, torch.bfloat16)
    assert torch.equal(wide[:, :4], kept[:, :4]) and torch.equal(wide[:, 164:], kept[:, 164:])
    op.bind(x=kept[:, 4:164].view(12, 5, 32), gate=gate, out=gate)
    op.run()
    assert torch.equal(gate, heads)


def test_rows_that_are_not_numbers_stay_alone_and_constant_rows_are_zero():
    from genn_amd.sequence import LayerNorm
    for channels in (24, 700, 3000):
        x = generator(channels)(6, channels)
        x[1, 3], x[3, channels - 1], x[4] = math.nan, math.inf, 2.5
        out = torch.zeros(6, channels).cuda()
        op = LayerNorm(1, 6, channels)
        op.bind(x=x.cuda(), out=out)
        op.run()
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all() and torch.all(out[4] == 0.0)
        rest = [0, 2, 5]
        close("out", out[rest], *ref.layer_norm(x[rest]))


def test_nothing_to_do():
    from genn_amd.sequence import Dropout, LayerNorm
    x = torch.ones(4, 8).cuda()
    dw, db = torch.full((8,), 7.0).cuda(), torch.full((8,), 7.0).cuda()
    for sequences, length in ((0, 4), (3, 0)):
        op = LayerNorm(sequences, length, 8)
        op.bind(x=x[:0], out=x[:0])
        op.run()
        op.bind_gradients(out=x[:0], weight=dw, bias=db)
        op.backward()
        assert torch.all(dw == 0.0) and torch.all(db == 0.0)
        drop = Dropout(sequences, length, 8, 0.5)
        drop.bind(x=x[:0], out=x[:0])
        drop.run(0)
    assert torch.all(x == 1.0)


def test_arrays_of_the_package_and_what_the_layer_refuses():
    from genn_amd.sequence import Dropout, LayerNorm
    x = generator(1)(6, 10)
    a, b, call = Array(60, "float32"), Array(60, "float32"), Array(1, "uint64")
    a.view[:] = x.reshape(-1).numpy()
    a.push_to_device()
    op = LayerNorm(2, 3, 10)
    op.bind(x=a, out=b)
    op.run()
    b.pull_from_device()
    close("out", torch.from_numpy(b.view.copy()), *ref.layer_norm(x))
    drop = Dropout(2, 3, 10, 0.5, seed=3)
    drop.bind(x=a, out=b)
    call.view[:] = 9
    call.push_to_device()
    drop.run(call)
    b.pull_from_device()
    assert torch.equal(torch.from_numpy(b.view.copy()).view(6, 10), torch.where(ref.kept(6, 10, 0.5, 3, 9)[0], x * 2, 0.0))
    for wrong in (lambda: Dropout(1, 1, 1, 1.5), lambda: Dropout(1, 1, 1, 0.5, seed=-1), lambda: drop.run(-1), lambda: drop.run(torch.zeros(2, dtype=torch.int64).cuda()),
                  lambda: op.bind(x=a, out=b, weight=torch.ones(9).cuda())):
        with pytest.raises(ValueError):
            wrong()
    with pytest.raises(TypeError):
        drop.run(torch.zeros(1).cuda())
    with pytest.raises(TypeError):
        op.bind(x=torch.zeros(6, 10).half().cuda(), out=b)
    with pytest.raises(RuntimeError):
        LayerNorm(2, 3, 10).run()
    with pytest.raises(RuntimeError):
        drop.backward(3)
    with pytest.raises(_abi.GennmiError):
        broken = LayerNorm(2, 3, 20000)
        broken.bind(x=torch.zeros(6, 20000).cuda(), out=torch.zeros(6, 20000).cuda())
        broken.run()


@pytest.mark.parametrize("channels", [64, 520, 2048, 5000])
def test_any_alignment_gives_the_same(channels):
    from genn_amd.sequence import Dropout, LayerNorm
    r, rows = generator(channels), 9
    x, z, d = (r(rows, channels).bfloat16() for _ in range(3))
    w, b = 1 + r(channels) / 8, r(channels) / 8
    results = []
    for shift in (0, 1, 3, 4):
        def placed(t):
            room = torch.empty(t.numel() + 8, dtype=t.dtype).cuda()
            view = room[shift:shift + t.numel()].view(t.shape)
            view.copy_(t)
            return view
        out, dx, dz, dw, db, kept = placed(x), placed(x), placed(x), placed(w), placed(w), placed(x)
        op = LayerNorm(1, rows, channels, dtype="bfloat16")
        op.bind(x=placed(x), weight=placed(w), bias=placed(b), gate=placed(z), out=out)
        op.run()
        op.bind_gradients(out=placed(d), x=dx, gate=dz, weight=dw, bias=db)
        op.backward()
        drop = Dropout(1, rows, channels, 0.3, seed=1, dtype="bfloat16")
        drop.bind(x=placed(x), residual=placed(z), out=kept)
        drop.run(2)
        results.append([t.double().cpu() for t in (out, dx, dz, dw, db, kept)])
    want, size = ref.layer_norm(x, w, b, z)
    for other in results:
        close("out", other[0], want, size, torch.bfloat16)
        assert torch.equal(other[5], results[0][5])
        # (another alignment may give a row to other lanes: the last bit of a sum)
        for a, c in zip(other[:5], results[0][:5]):
            assert float((a - c).norm()) <= 2.0 ** -8 * float(c.norm())


def test_rows_and_calls_at_their_ends():
    """Sequences more than 2^32 elements apart, the largest seed and numbers of calls, a number on the device that is added to none."""
    from genn_amd.sequence import Dropout, LayerNorm
    r, far, channels = generator(5), (1 << 32) + 64, 136
    room = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    x = r(2, 3, channels).bfloat16()
    there = torch.as_strided(room, (2, 3, channels), (far, channels + 8, 1))
    there.copy_(x)
    out = torch.zeros(2, 3, channels, dtype=torch.bfloat16).cuda()
    op = LayerNorm(2, 3, channels, dtype="bfloat16")
    op.bind(x=there, out=out)
    op.run()
    close("out", out.view(6, channels), *ref.layer_norm(x.view(6, channels)), torch.bfloat16)
    op.bind(x=x.cuda(), out=there)
    op.run()
    assert torch.equal(there, out)
    seed = (1 << 64) - 1
    drop = Dropout(2, 3, channels, 0.5, seed=seed, dtype="bfloat16")
    drop.bind(x=x.cuda(), out=there)
    for call in (0, (1 << 32) - 1, 1 << 32, (1 << 64) - 1):
        drop.run(call)
        keep, factor = ref.kept(6, channels, 0.5, seed, call)
        want = torch.where(keep.view(x.shape), x.double(), 0.0) * factor
        close("out", there.contiguous(), want, want.abs(), torch.bfloat16, 3)
    last = torch.tensor([-1], dtype=torch.int64).cuda()         # (all 64 bits)
    before = there.clone()
    there.zero_()
    drop.run(last)
    assert torch.equal(there, before)


@pytest.mark.parametrize("channels, rows", [(48, 700), (1024, 40), (6000, 5)])
def test_a_row_that_is_no_number_leaves_the_others_gradients_alone(channels, rows):
    from genn_amd.sequence import LayerNorm
    r = generator(channels)
    x, z, d = r(rows, channels), r(rows, channels), r(rows, channels)
    grads = []
    for bad in (False, True):
        if bad:
            x[rows // 2, 7] = math.nan
        dx, dz = torch.zeros(rows, channels).cuda(), torch.zeros(rows, channels).cuda()
        op = LayerNorm(1, rows, channels, rms=True)
        op.bind(x=x.cuda(), gate=z.cuda())
        op.bind_gradients(out=d.cuda(), x=dx, gate=dz)
        op.backward()
        grads.append((dx.cpu(), dz.cpu()))
    rest = torch.arange(rows) != rows // 2
    for a, b in zip(*grads):
        assert torch.equal(a[rest], b[rest]) and torch.isnan(b[rows // 2]).all()


def test_a_bind_that_is_refused_leaves_what_was_bound():
    from genn_amd.sequence import Dropout, GatedDeltaRule, LayerNorm
    x = generator(2)(2, 8).cuda()
    for op, more in ((GatedDeltaRule(1, 2, 1, 8, 8), ("q", "k", "v")), (LayerNorm(1, 2, 8), ("x",)), (Dropout(1, 2, 8, 0.5), ("x",))):
        def arrays(t):
            given = {name: t for name in more}
            return dict(given, g=t[:, :1], beta=t[:, :1]) if len(more) > 1 else given
        call = (lambda: op.run(3)) if isinstance(op, Dropout) else op.run
        first, second = torch.zeros_like(x), torch.zeros_like(x)
        op.bind(out=first, **arrays(x))
        call()
        first.zero_()
        with pytest.raises((ValueError, TypeError)):
            op.bind(out=second, **arrays(x[:1]))
        with pytest.raises((ValueError, TypeError)):
            op.bind(out=second, **arrays(x.cpu()))
        call()
        assert float(first.abs().sum()) > 0 and float(second.abs().sum()) == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("channels, gate, rows", [(8200, True, 2100), (8200, False, 700), (8193, True, 60)])
def test_gradients_of_the_longest_rows(channels, gate, rows, dtype):
    """Of rows for more work-groups than the chip holds: each adds up several."""
    from genn_amd.sequence import LayerNorm
    T, r = TYPES[dtype], generator(channels + rows)
    x, d, w, b = r(rows, channels).to(T), r(rows, channels).to(T), 1 + r(channels) / 8, r(channels) / 8
    z = r(rows, channels).to(T) if gate else None
    dx, dz, dw, db = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda(), torch.zeros(channels).cuda(), torch.zeros(channels).cuda()
    op = LayerNorm(1, rows, channels, dtype=dtype)
    op.bind(x=x.cuda(), weight=w.cuda(), bias=b.cuda(), gate=z.cuda() if gate else None)
    op.bind_gradients(out=d.cuda(), x=dx, weight=dw, bias=db, gate=dz if gate else None)
    op.backward()
    found, size = ref.layer_norm(x, w, b, z, dout=d)
    close("dx", dx, found["dx"], size["dx"], T, 2 * OPERATIONS)
    # (a lane adds up rows / 512 rows before the sums in 64 bits)
    close("dweight", dw, found["dweight"], size["dweight"], operations=2 * OPERATIONS + rows // 512)
    close("dbias", db, found["dbias"], size["dbias"], operations=2 * OPERATIONS + rows // 512)
    if gate:
        close("dgate", dz, found["dgate"], size["dgate"], T, 2 * OPERATIONS)
