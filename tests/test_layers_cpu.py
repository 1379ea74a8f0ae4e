"""The gated delta rule, layer norm and dropout as far as they go without a GPU: layouts of the descriptors, what the entry points refuse before
they touch the device, and the 64-bit restatements that the GPU tests compare with, against differences."""
import ctypes as C

import pytest
import torch

import layer_ref as ref
from genn_amd import _abi

F32, F16, BF16 = (_abi.FLOAT_TYPES[t] for t in ("float32", "float16", "bfloat16"))
AT = 1 << 20            # an address that nothing may follow


def changed(c, changes):
    for name, value in changes.items():
        at = c
        *path, last = name.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, value)
    return c


def delta(**changes):
    c = _abi.DeltaRule(type=BF16, heads=4, keyHeads=2, keys=16, values=24, normalise=1, scale=0.25, epsilon=1e-6)
    c.sequences = _abi.Sequences(count=2, length=5)
    for k, (name, width) in enumerate((("q", 32), ("k", 32), ("v", 96), ("out", 96), ("g", 4), ("beta", 4))):
        setattr(c, name, _abi.Rows(AT + 16384 * k, width, 5 * width))
    return changed(c, changes)


def norm(**changes):
    c = _abi.LayerNorm(type=BF16, channels=24, epsilon=1e-5, weight=AT + 65536, bias=AT + 131072)
    c.sequences = _abi.Sequences(count=2, length=5)
    c.x, c.out = _abi.Rows(AT, 24, 120), _abi.Rows(AT + 4096, 24, 120)
    return changed(c, changes)


def dropout(**changes):
    c = _abi.Dropout(type=BF16, channels=24, probability=0.1, seed=1, call=2)
    c.sequences = _abi.Sequences(count=2, length=5)
    c.x, c.out, c.residual = _abi.Rows(AT, 24, 120), _abi.Rows(AT + 4096, 24, 120), _abi.Rows(AT + 8192, 24, 120)
    return changed(c, changes)


def refused(rc, code, text):
    said = _abi.load().gennmi_last_error().decode()
    assert rc == code and text in said, (rc, said)


def test_descriptors_have_the_librarys_layout():
    sizes = (C.c_size_t * 5)()
    assert _abi.load().gennmi_abi_layer_sizes(C.byref(sizes)) == 0
    assert list(sizes) == [C.sizeof(s) for s in _abi.LAYER_STRUCTS]


@pytest.mark.parametrize("change, code, text", [
    (dict(type=1), -3, "element type"), (dict(keys=0), -3, "keys"), (dict(keys=129), -3, "keys"), (dict(values=0), -3, "values"), (dict(values=1025), -3, "values"),
    (dict(heads=0), -2, "heads"), (dict(keyHeads=0), -2, "heads"), (dict(keyHeads=3), -2, "heads"), (dict(heads=1 << 17, keyHeads=1), -2, "heads"),
    (dict(q__data=None), -2, "q is missing"), (dict(k__data=AT + 1), -2, "aligned"), (dict(v__data=None), -2, "v is missing"), (dict(out__data=None), -2, "out is missing"),
    (dict(g__data=None), -2, "g is missing"), (dict(g__data=AT + 2), -2, "aligned"), (dict(beta__rowStride=3), -2, "rows overlap"), (dict(q__rowStride=31), -2, "rows overlap"),
    (dict(out__sequenceStride=95), -2, "sequences overlap"), (dict(initialState=AT + 2), -2, "state"), (dict(finalState=AT + 1), -2, "state"),
    (dict(sequences__slots=AT, sequences__numSlots=0), -2, "numSlots"), (dict(sequences__offsets=AT + 2, sequences__rows=9), -2, "offsets"),
    (dict(sequences__count=1 << 12, sequences__length=1 << 19), -2, "more sequences or rows"),
    (dict(sequences__count=1 << 24, sequences__length=1, heads=1 << 16, keyHeads=1, v__rowStride=24 << 16, out__rowStride=24 << 16, out__sequenceStride=24 << 16, g__rowStride=1 << 16,
          beta__rowStride=1 << 16), -2, "one launch"),
    (dict(out__data=AT + 32768), -2, "out overlaps v"), (dict(finalState=AT + 16384), -2, "overlaps"),
])
def test_delta_rule_refuses(change, code, text):
    room = AT + (1 << 30)
    refused(_abi.load().gennmi_delta_rule(C.byref(delta(**change)), room, 1 << 40, None), code, text)


@pytest.mark.parametrize("change, code, text", [
    (dict(type=7), -3, "element type"), (dict(channels=0), -3, "channels"), (dict(channels=16385), -3, "channels"), (dict(epsilon=-1.0), -2, "epsilon"), (dict(epsilon=float("nan")), -2, "epsilon"),
    (dict(x__data=None), -2, "x is missing"), (dict(out__data=None), -2, "out is missing"), (dict(x__rowStride=23), -2, "rows overlap"), (dict(weight=AT + 2), -2, "aligned"),
    (dict(sequences__offsets=AT, sequences__rows=9), -2, "not packed"), (dict(sequences__slots=AT, sequences__numSlots=3), -2, "not packed"), (dict(out__data=AT + 48), -2, "out overlaps x"),
    (dict(out__data=AT, out__sequenceStride=240), -2, "out overlaps x"), (dict(weight=AT + 4096), -2, "out overlaps weight"), (dict(gate__data=AT + 1), -2, "aligned"),
])
def test_layer_norm_refuses(change, code, text):
    refused(_abi.load().gennmi_layer_norm(C.byref(norm(**change)), None), code, text)


@pytest.mark.parametrize("change, code, text", [
    (dict(type=7), -3, "element type"), (dict(channels=0), -2, "channels"), (dict(probability=-0.1), -2, "probability"), (dict(probability=1.1), -2, "probability"),
    (dict(probability=float("nan")), -2, "probability"), (dict(x__data=None), -2, "x is missing"), (dict(out__data=AT + 8192 + 2), -2, "out overlaps residual"),
    (dict(sequences__offsets=AT, sequences__rows=9), -2, "not packed"), (dict(callDevice=AT + 4), -2, "callDevice"), (dict(callDevice=AT + 4096), -2, "out overlaps callDevice"),
    (dict(sequences__count=1, sequences__length=(1 << 31) - 1, channels=1 << 24, x__rowStride=1 << 24, out__rowStride=1 << 24, residual__rowStride=1 << 24), -2, "one launch"),
])
def test_dropout_refuses(change, code, text):
    refused(_abi.load().gennmi_dropout(C.byref(dropout(**change)), None), code, text)


def test_gradients_and_workspaces_that_are_refused():
    lib = _abi.load()
    size = C.c_size_t()
    assert lib.gennmi_delta_rule_workspace(C.byref(delta()), C.byref(size)) == 0 and size.value > 0
    refused(lib.gennmi_delta_rule(C.byref(delta()), None, 0, None), -2, "workspace")
    refused(lib.gennmi_delta_rule(C.byref(delta()), AT + (1 << 30) + 8, size.value, None), -2, "16-byte")
    refused(lib.gennmi_delta_rule(C.byref(delta()), AT, size.value, None), -2, "overlaps")
    assert lib.gennmi_delta_rule_workspace(C.byref(delta(sequences__length=1)), C.byref(size)) == 0 and size.value == 0
    refused(lib.gennmi_delta_rule_workspace(C.byref(delta()), None), -2, "null result")
    refused(lib.gennmi_delta_rule_backward(C.byref(delta()), None, None, 0, None), -2, "null gradient")
    refused(lib.gennmi_delta_rule(None, None, 0, None), -2, "null descriptor")
    g = _abi.DeltaRuleGradient()
    refused(lib.gennmi_delta_rule_backward(C.byref(delta()), C.byref(g), None, 0, None), -2, "the gradient of out is missing")
    g.out = _abi.Rows(AT + (1 << 21), 96, 480)
    g.q = _abi.Rows(AT, 32, 160)
    refused(lib.gennmi_delta_rule_backward(C.byref(delta()), C.byref(g), AT + (1 << 30), 1 << 40, None), -2, "the gradient of q overlaps q")
    refused(lib.gennmi_delta_rule_backward(C.byref(delta(sequences__slots=AT, sequences__numSlots=3)), C.byref(g), AT + (1 << 30), 1 << 40, None), -2, "slots are not for gradients")
    n = _abi.LayerNormGradient()
    refused(lib.gennmi_layer_norm_backward(C.byref(norm()), C.byref(n), None, 0, None), -2, "the gradient of out is missing")
    n.out, n.weight = _abi.Rows(AT + (1 << 21), 24, 120), AT + (1 << 22)
    refused(lib.gennmi_layer_norm_backward(C.byref(norm()), C.byref(n), None, 0, None), -2, "workspace")
    n.gate = _abi.Rows(AT + (1 << 23), 24, 120)
    refused(lib.gennmi_layer_norm_backward(C.byref(norm()), C.byref(n), AT + (1 << 30), 1 << 40, None), -2, "without gate")
    n.gate, n.x = _abi.Rows(), _abi.Rows(AT + (1 << 21), 24, 120)
    refused(lib.gennmi_layer_norm_backward(C.byref(norm()), C.byref(n), AT + (1 << 30), 1 << 40, None), -2, "the gradient of x overlaps the gradient of out")
    refused(lib.gennmi_layer_norm(None, None), -2, "null descriptor")
    refused(lib.gennmi_dropout(None, None), -2, "null descriptor")


def test_strides_of_the_delta_rule_are_limited():
    lib, size = _abi.load(), C.c_size_t()
    most = 1 << 25
    for name in ("q", "k", "v", "out"):
        far = {name + "__data": 1 << 40, name + "__rowStride": most, name + "__sequenceStride": 5 * most}
        refused(lib.gennmi_delta_rule_workspace(C.byref(delta(**far)), C.byref(size)), -2, "stride of q, k, v or out")
        far.update({name + "__rowStride": most - 1})
        assert lib.gennmi_delta_rule_workspace(C.byref(delta(**far)), C.byref(size)) == 0
        far.update({name + "__rowStride": most, "sequences__length": 1})        # (no second row)
        assert lib.gennmi_delta_rule_workspace(C.byref(delta(**far)), C.byref(size)) == 0
    g = _abi.DeltaRuleGradient(out=_abi.Rows(1 << 40, most, 5 * most))
    refused(lib.gennmi_delta_rule_backward(C.byref(delta()), C.byref(g), AT + (1 << 30), 1 << 40, None), -2, "stride of the gradients")
    g = _abi.DeltaRuleGradient(out=_abi.Rows(1 << 40, 96, 480), v=_abi.Rows(1 << 41, most, 5 * most))
    refused(lib.gennmi_delta_rule_backward(C.byref(delta()), C.byref(g), AT + (1 << 30), 1 << 40, None), -2, "stride of the gradients")


def test_gradients_of_the_restatements_are_those_of_differences():
    gen = torch.Generator().manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)  # noqa: E731
    n, H, G, K, V = 7, 4, 2, 5, 3
    for normalise in (True, False):
        arrays = dict(q=r(n, G, K), k=r(n, G, K) / 3, v=r(n, H, V), g=-r(n, H).abs(), beta=torch.sigmoid(r(n, H)), initial=r(H, K, V))
        dout, dfinal = r(n, H, V), r(H, K, V)

        def value(**a):
            out, final, _ = ref.delta(a["q"], a["k"], a["v"], a["g"], a["beta"], 0.4, normalise, initial=a["initial"])
            return float((out * dout).sum() + (final * dfinal).sum())

        found, _ = ref.delta(*(arrays[k] for k in ("q", "k", "v", "g", "beta")), 0.4, normalise, initial=arrays["initial"], dout=dout, dfinal=dfinal)
        for name, x in arrays.items():
            d = r(*x.shape)
            got = (value(**{**arrays, name: x + 1e-5 * d}) - value(**{**arrays, name: x - 1e-5 * d})) / 2e-5
            assert abs(got - float((found["d" + name] * d).sum())) < 1e-6, name
    for rms in (True, False):
        arrays = dict(x=r(6, 9), weight=r(9), bias=r(9), gate=r(6, 9))
        dout = r(6, 9)
        found, _ = ref.layer_norm(rms=rms, dout=dout, **arrays)
        for name, x in arrays.items():
            d = r(*x.shape)
            ends = [float((ref.layer_norm(rms=rms, **{**arrays, name: x + s * d})[0] * dout).sum()) for s in (1e-5, -1e-5)]
            assert abs((ends[0] - ends[1]) / 2e-5 - float((found["d" + name] * d).sum())) < 1e-6, name


def test_draws_of_the_restatement():
    kept, factor = ref.kept(1000, 37, 0.25, 12345, 6)
    assert factor == 65536 / 49152 and abs(float(kept.double().mean()) - 0.75) < 5 * (0.75 * 0.25 / 37000) ** 0.5
    assert torch.equal(kept[:10], ref.kept(10, 37, 0.25, 12345, 6)[0])
    assert not torch.equal(kept, ref.kept(1000, 37, 0.25, 12345, 7)[0])
    assert ref.kept(3, 8, 0.0, 1, 1)[0].all() and not ref.kept(3, 8, 1.0, 1, 1)[0].any()
