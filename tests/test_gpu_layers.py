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
