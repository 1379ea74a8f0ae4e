"""Gradients of the gated delta rule row by row: each row's own vector against the formulas in 64 bits, bounded by what is added up for that row, so that a wrong row cannot hide behind a larger one.

Tolerances.  One rounding to the result's type (half a step), and of what is added up in fp32 for that row (``delta_rows.sizes``) five standard deviations of sqrt(keys + 2 * 64 + rows) independent errors
of 2^-24 each, four operations for each: keys of a dot product, the rows of a chunk twice, the rows of the sequence.  The bounds of every head's rows together have to be below a quarter of its
gradient, so that an array of zeros does not pass."""
import math

import pytest
import torch

import delta_rows
import layer_ref as ref
from test_gpu_delta import TYPES, Inputs, arrays, split

pytestmark = pytest.mark.gpu


def gates(i, kind, seed):
    """Decays that a row keeps most of, of a few rows, and of nothing but the row (exp(-20) of what was before it)."""
    r = torch.rand(i.g.shape, generator=torch.Generator().manual_seed(seed))
    if kind == "strong":
        i.g = -3 - 17 * r
    elif kind == "mixed":
        i.g = torch.where(r < 0.2, -40 * r, i.g)


def gradients(lengths, i, heads, key_heads, keys, values, dtype, normalise=True):
    from genn_amd.sequence import GatedDeltaRule
    T, S, rows = TYPES[dtype], len(lengths), sum(lengths)
    got = dict(q=torch.full((rows, key_heads * keys), 7.0, dtype=T).cuda(), k=torch.full((rows, key_heads * keys), 7.0, dtype=T).cuda(), v=torch.full((rows, heads * values), 7.0, dtype=T).cuda(),
               g=torch.full((rows, heads), 7.0).cuda(), beta=torch.full((rows, heads), 7.0).cuda(), initial_state=torch.full((S, heads, keys, values), 7.0).cuda())
    op = GatedDeltaRule(S, max(lengths), heads, keys, values, key_heads=key_heads, dtype=dtype, normalise=normalise)
    op.bind(initial_state=i.initial.cuda(), offsets=split(lengths)[1], **arrays(i, heads, key_heads, keys, values))
    op.bind_gradients(out=i.dout.cuda(), final_state=i.dfinal.cuda(), **got)
    op.backward()
    torch.cuda.synchronize()
    return {n: x.cpu().double() for n, x in got.items()}


def compare(lengths, i, got, heads, key_heads, keys, values, dtype, normalise=True):
    eps, tiny = torch.finfo(TYPES[dtype]).eps / 2, torch.finfo(TYPES[dtype]).smallest_normal * torch.finfo(TYPES[dtype]).eps
    for n, part in enumerate(split(lengths)[0]):
        more = dict(initial=i.initial[n], dout=i.dout[part].view(-1, heads, values), dfinal=i.dfinal[n])
        found, _ = ref.delta(*i.of(part), keys ** -0.5, normalise, **more)
        size = delta_rows.sizes(*i.of(part), keys ** -0.5, normalise, **more)
        unit = 5 * 2.0 ** -22 * math.sqrt(keys + 2 * 64 + lengths[n])
        for name in ("q", "k", "v", "g", "beta"):
            want = found["d" + name]
            have = got[name][part].view(want.shape)
            if want.dim() == 2:
                want, have = want[..., None], have[..., None]
            e, least = (eps, tiny) if name in "qkv" else (2.0 ** -24, 2.0 ** -126)
            off, limit = (have - want).norm(dim=-1), e * want.norm(dim=-1) + unit * (1 + 2 * e) * size[name] + least * math.sqrt(want.shape[-1])
            worst = int((off / limit).argmax())
            assert (off <= limit).all(), (name, n, worst, float(off.reshape(-1)[worst]), float(limit.reshape(-1)[worst]), float((off / limit).max()), int((off > limit).sum()))
            whole = want.norm(dim=(0, 2))
            assert (unit * size[name].norm(dim=0) < whole / 4).all(), (name, unit * size[name].norm(dim=0), whole)
        off = (got["initial_state"][n] - found["dinitial"]).norm(dim=(1, 2))
        assert (off <= 2.0 ** -24 * found["dinitial"].norm(dim=(1, 2)) + unit * size["initial"] + 2.0 ** -126 * math.sqrt(keys * values)).all(), (n, off, size["initial"])


@pytest.mark.parametrize("lengths, heads, key_heads, keys, values, dtype, normalise, kind", [
    ([513], 1, 1, 128, 256, "bfloat16", True, "slow"),
    ([301], 3, 1, 33, 47, "float32", True, "slow"),
    ([137, 64], 6, 3, 100, 72, "float16", True, "mixed"),
    ([256], 2, 2, 128, 128, "bfloat16", True, "strong"),
    ([200, 1, 33], 2, 1, 64, 80, "float32", True, "strong"),
    ([97], 2, 2, 128, 40, "float16", True, "strong"),
    ([190], 2, 1, 48, 64, "bfloat16", False, "mixed"),
    ([70], 3, 3, 16, 8, "float32", False, "mixed"),
    # (more work-groups than the chip has compute units, and several chunks of each)
    ([130] * 5, 26, 26, 128, 48, "bfloat16", True, "mixed"),
    ([75] * 6, 46, 23, 64, 20, "float32", True, "mixed"),
    ([70] * 5, 26, 26, 72, 33, "float16", True, "slow"),
])
def test_gradients_row_by_row(lengths, heads, key_heads, keys, values, dtype, normalise, kind):
    i = Inputs(lengths, heads, key_heads, keys, values, dtype, seed=sum(lengths) + keys)
    gates(i, kind, sum(lengths))
    if not normalise:
        i.q, i.k = ((x.float() / math.sqrt(2 * keys)).to(TYPES[dtype]) for x in (i.q, i.k))          # (shorter than 1, as the bound asks for)
    sizes = (heads, key_heads, keys, values, dtype, normalise)
    compare(lengths, i, gradients(lengths, i, *sizes), *sizes)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_gates_that_forget_everything_have_no_gradient(dtype):
    """The gradient of a gate is a multiple of the decay: nothing, where that is nothing; and the same gates of the rows around it are not disturbed by it."""
    lengths, heads, keys, values = [150], 3, 40, 24
    i = Inputs(lengths, heads, heads, keys, values, dtype, seed=12)
    i.g[::9, 0], i.g[3:80, 1], i.g[:, 2] = -math.inf, -1e30, -500.0
    got = gradients(lengths, i, heads, heads, keys, values, dtype)
    assert torch.all(got["g"][::9, 0] == 0.0) and torch.all(got["g"][3:80, 1] == 0.0) and torch.all(got["g"][:, 2] == 0.0)
    i.g = torch.clamp(i.g, min=-1e6)
    found, _ = ref.delta(*i.of(slice(0, 150)), keys ** -0.5, initial=i.initial[0], dout=i.dout.view(-1, heads, values), dfinal=i.dfinal[0])
    size = delta_rows.sizes(*i.of(slice(0, 150)), keys ** -0.5, initial=i.initial[0], dout=i.dout.view(-1, heads, values), dfinal=i.dfinal[0])
    unit = 5 * 2.0 ** -22 * math.sqrt(keys + 2 * 64 + 150)
    assert torch.all((got["g"] - found["dg"]).abs() <= 2.0 ** -24 * found["dg"].abs() + unit * size["g"] + 2.0 ** -126)
