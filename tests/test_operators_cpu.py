"""Operators on sequences and the optimiser, as far as they go without a GPU: layouts of the descriptors, sizes of workspaces, and what the
entry points refuse before they touch the device.  Also the 64-bit restatements that the GPU tests compare with, against differences."""
import ctypes as C
import json
import os
import random
import subprocess
import sys

import pytest
import torch

import sequence_ref as ref
from genn_amd import _abi

F32, F16, BF16 = (_abi.FLOAT_TYPES[t] for t in ("float32", "float16", "bfloat16"))
AT = 1 << 20            # an address that nothing may follow


def conv(**changes):
    c = _abi.CausalConv(type=BF16, channels=24, taps=4, silu=1, weight=AT, bias=AT, initialState=None, finalState=None)
    c.sequences = _abi.Sequences(count=2, length=5)
    c.x, c.out = _abi.Rows(AT, 24, 120), _abi.Rows(AT + 4096, 24, 120)
    return changed(c, changes)


def scan(**changes):
    c = _abi.Scan(type=BF16, channels=24, states=16, groups=2, softplus=1, A=AT, D=AT, deltaBias=AT)
    c.sequences = _abi.Sequences(count=2, length=5)
    for k, name in enumerate(("u", "delta", "z", "out")):
        setattr(c, name, _abi.Rows(AT + 4096 * k, 24, 120))
    c.B, c.C = _abi.Rows(AT + 4096 * 5, 32, 160), _abi.Rows(AT + 4096 * 6, 32, 160)
    return changed(c, changes)


def changed(c, changes):
    for name, value in changes.items():
        at = c
        *path, last = name.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, value)
    return c


def refused(rc, code, text):
    said = _abi.load().gennmi_last_error().decode()
    assert rc == code and text in said, (rc, said)


def test_descriptors_have_the_librarys_layout():
    sizes = (C.c_size_t * 9)()
    assert _abi.load().gennmi_abi_operator_sizes(C.byref(sizes)) == 0
    assert list(sizes) == [C.sizeof(s) for s in _abi.OPERATOR_STRUCTS]


@pytest.mark.parametrize("change, code, text", [
    (dict(type=1), -3, "element type"), (dict(type=7), -3, "element type"), (dict(taps=0), -3, "taps"), (dict(taps=9), -3, "taps"),
    (dict(channels=0), -2, "channels"), (dict(weight=None), -2, "weight"), (dict(weight=AT + 2), -2, "aligned"), (dict(bias=AT + 1), -2, "aligned"),
    (dict(x__data=None), -2, "x is missing"), (dict(x__data=AT + 1), -2, "aligned"), (dict(out__data=AT), -2, "same array"), (dict(out__data=None), -2, "out is missing"),
    (dict(x__rowStride=23), -2, "rows overlap"), (dict(out__sequenceStride=0), -2, "sequences overlap"), (dict(out__rowStride=1 << 41), -2, "stride"), (dict(x__rowStride=1 << 32), -2, "stride"),
    (dict(initialState=AT + 1), -2, "state"), (dict(finalState=AT + 1), -2, "state"),
    (dict(sequences__count=(1 << 24) + 1), -2, "more sequences"), (dict(sequences__length=1 << 31), -2, "more sequences"),
    (dict(sequences__offsets=AT + 2, sequences__rows=10), -2, "offsets"), (dict(sequences__slots=AT, sequences__numSlots=0), -2, "numSlots"),
    (dict(sequences__offsets=AT, sequences__rows=1 << 31), -2, "more sequences or rows"),
    (dict(sequences__count=1 << 12, sequences__length=1 << 19), -2, "more sequences or rows"),
    (dict(sequences__count=1, sequences__length=(1 << 31) - 1, channels=1 << 24, x__rowStride=1 << 24, out__rowStride=1 << 24), -2, "one launch"),
])
def test_causal_conv_refuses(change, code, text):
    refused(_abi.load().gennmi_causal_conv(C.byref(conv(**change)), None), code, text)


@pytest.mark.parametrize("change, code, text", [
    (dict(type=2), -3, "element type"), (dict(states=0), -3, "states"), (dict(states=129), -3, "states"), (dict(channels=0), -2, "channels"),
    (dict(groups=0), -2, "groups"), (dict(groups=5), -2, "groups"), (dict(A=None), -2, "A is missing"), (dict(A=AT + 1), -2, "aligned"),
    (dict(D=AT + 2), -2, "aligned"), (dict(initialState=AT + 2), -2, "aligned"), (dict(out__data=AT), -2, "array of its own"),
    (dict(out__data=None), -2, "out is missing"), (dict(delta__data=None), -2, "delta is missing"), (dict(z__rowStride=1), -2, "rows overlap"),
    (dict(B__rowStride=31), -2, "rows overlap"), (dict(C__data=None), -2, "C is missing"), (dict(out__sequenceStride=23), -2, "sequences overlap"),
    (dict(sequences__slots=AT + 2, sequences__numSlots=3), -2, "slots"), (dict(sequences__count=1 << 12, sequences__length=1 << 19), -2, "more sequences or rows"),
])
def test_selective_scan_refuses(change, code, text):
    c = scan(**change)
    refused(_abi.load().gennmi_selective_scan(C.byref(c), C.c_void_p(AT), 1 << 60, None), code, text)


def test_calls_without_arguments_and_workspaces_are_refused():
    lib = _abi.load()
    size = C.c_size_t()
    refused(lib.gennmi_causal_conv(None, None), -2, "null descriptor")
    refused(lib.gennmi_selective_scan(None, None, 0, None), -2, "null descriptor")
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), None, None, 0, None), -2, "null gradient")
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), None, None, 0, None), -2, "null gradient")
    refused(lib.gennmi_selective_scan_workspace(C.byref(scan()), None), -2, "null result")
    refused(lib.gennmi_stream_is_capturing(None, None), -2, "null result")
    refused(lib.gennmi_current_device(None), -2, "null result")
    # the gradients' checks
    g = _abi.CausalConvGradient(out=_abi.Rows(AT + 8192, 24, 120), x=_abi.Rows(AT + 16384, 24, 120), weight=AT)
    need = lib.gennmi_causal_conv_backward_workspace
    assert need(C.byref(conv()), C.byref(size)) == 0 and size.value > 0
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), C.byref(g), None, 0, None), -2, "workspace")
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), C.byref(g), AT, size.value - 1, None), -2, "workspace")
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), C.byref(g), AT + 4, size.value, None), -2, "16-byte")
    refused(lib.gennmi_causal_conv_backward(C.byref(conv(sequences__slots=AT, sequences__numSlots=4)), C.byref(g), AT, size.value, None), -2, "slots")
    g.x = _abi.Rows(AT, 24, 120)
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), C.byref(g), AT, size.value, None), -2, "array of its own")
    g = _abi.CausalConvGradient(out=_abi.Rows(AT + 8192, 24, 120), initialState=AT, finalState=AT)
    refused(lib.gennmi_causal_conv_backward(C.byref(conv()), C.byref(g), AT, size.value, None), -2, "array of its own")
    g = _abi.ScanGradient(out=_abi.Rows(AT + 4096 * 7, 24, 120), u=_abi.Rows(AT + 4096 * 8, 24, 120), delta=_abi.Rows(AT + 4096 * 8, 24, 120))
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), C.byref(g), AT, 1 << 60, None), -2, "array of its own")
    g = _abi.ScanGradient(out=_abi.Rows(AT + 4096 * 7, 24, 120), B=_abi.Rows(AT + 4096 * 8, 32, 160), C=_abi.Rows(AT + 4096 * 8, 32, 160))
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), C.byref(g), AT, 1 << 60, None), -2, "array of its own")
    g = _abi.ScanGradient(out=_abi.Rows(AT + 4096 * 7, 24, 120), u=_abi.Rows(AT + 4096 * 8, 24, 120))
    assert lib.gennmi_selective_scan_backward_workspace(C.byref(scan()), C.byref(size)) == 0 and size.value > 0
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), C.byref(g), AT, size.value - 1, None), -2, "workspace")
    refused(lib.gennmi_selective_scan_backward(C.byref(scan(z__data=None)), C.byref(changed(g, dict(z=_abi.Rows(AT + 4096 * 9, 24, 120)))), AT, size.value, None), -2, "without z")
    g.z = _abi.Rows()
    g.B = _abi.Rows(AT + 4096 * 5, 32, 160)
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), C.byref(g), AT, size.value, None), -2, "array of its own")
    g.B = _abi.Rows()
    wide = scan(sequences__count=1, sequences__length=(1 << 31) - 1, channels=1 << 24, groups=1, z__data=None)
    for name in ("u", "delta", "out"):
        getattr(wide, name).rowStride = 1 << 24
    large = changed(_abi.ScanGradient(out=_abi.Rows(AT + 4096 * 7, 1 << 24, 0)), {})
    refused(lib.gennmi_selective_scan_backward(C.byref(wide), C.byref(large), AT, 1 << 62, None), -2, "one launch")
    g.out = _abi.Rows()
    refused(lib.gennmi_selective_scan_backward(C.byref(scan()), C.byref(g), AT, size.value, None), -2, "gradient of out is missing")


def test_workspaces_of_packed_sequences_go_by_their_rows():
    """Not by the number of sequences times the longest one, which may be far more than there are rows."""
    lib, size = _abi.load(), C.c_size_t()
    for entry in (lib.gennmi_selective_scan_workspace, lib.gennmi_selective_scan_backward_workspace):
        c = scan(sequences__count=1000, sequences__length=8000, sequences__offsets=AT, sequences__rows=10000)
        assert entry(C.byref(c), C.byref(size)) == 0
        assert size.value < (10000 // 8 + 1000) * 24 * (16 * 3 + 4) * 4 + 10000 * 2 * 16 * 2 * 4 + 4096
    c = scan(sequences__length=1, u__rowStride=1 << 33)         # (the stride of rows that are not there)
    assert lib.gennmi_selective_scan_workspace(C.byref(c), C.byref(size)) == 0 and size.value == 0     # (a token needs none)


def test_packed_arrays_without_sequences_have_no_chunks():
    """Rows that belong to no sequence: there is nothing to sum over, and nothing to keep for it (offsets has one element)."""
    lib, size = _abi.load(), C.c_size_t()
    none = dict(sequences__count=0, sequences__offsets=AT, sequences__rows=10000)
    assert lib.gennmi_causal_conv_backward_workspace(C.byref(conv(sequences__length=100, **none)), C.byref(size)) == 0 and size.value == 0
    for length in (4, 8000):
        assert lib.gennmi_selective_scan_workspace(C.byref(scan(sequences__length=length, **none)), C.byref(size)) == 0 and size.value == 0
        assert lib.gennmi_selective_scan_backward_workspace(C.byref(scan(sequences__length=length, **none)), C.byref(size)) == 0
        assert size.value <= 2 * 10000 * 2 * 16 * 4 + 256           # (only what goes by rows)


def reaches_the_device(rc):
    """(the descriptors name a device that is not there, so nothing is launched)"""
    said = _abi.load().gennmi_last_error().decode()
    assert rc not in (0, -2) and "current device" in said, (rc, said)


WIDE = 1 << 24          # channels
FAR = 1 << 50           # between the addresses of arrays of that size


def wide(make, count, length, channels=WIDE, states=None, **changes):
    rows = {f"{r}__{k}": v for n, r in enumerate(("x", "out") if states is None else ("u", "delta", "z", "out"))
            for k, v in (("rowStride", channels), ("sequenceStride", channels * length), ("data", (n + 1) * FAR))}
    if states is not None:
        rows.update({f"{r}__{k}": v for r in "BC" for k, v in (("rowStride", states), ("sequenceStride", states * length))}, states=states, groups=1)
    return make(**rows, channels=channels, sequences__count=count, sequences__length=length, sequences__device=78, **changes)


def test_launches_of_2_to_the_32_threads_are_refused_before_anything_runs():
    """The last size that every launch of a call covers, and the first that one of them does not."""
    lib, size, space = _abi.load(), C.c_size_t(), (C.c_void_p(60 * FAR), 1 << 62)
    many = "more rows than one launch covers"
    # convolution: four channels a thread, 16 rows; gradients: two, 64 rows
    reaches_the_device(lib.gennmi_causal_conv(C.byref(wide(conv, 1, 1023 * 16)), None))
    refused(lib.gennmi_causal_conv(C.byref(wide(conv, 1, 1023 * 16 + 1)), None), -2, many)
    g = _abi.CausalConvGradient(out=_abi.Rows(20 * FAR, WIDE, 0))
    reaches_the_device(lib.gennmi_causal_conv_backward(C.byref(wide(conv, 1, 511 * 64)), C.byref(g), None, 0, None))
    refused(lib.gennmi_causal_conv_backward(C.byref(wide(conv, 1, 511 * 64 + 1)), C.byref(g), None, 0, None), -2, many)
    # scan: a wavefront for 64 channels of a sequence and 16 states; a token: a lane for four states
    for count, length, states in ((255, 2, 16), (31, 2, 128), (63, 1, 16), (7, 1, 128)):
        for more in (0, 1):
            c = wide(scan, count + more, length, states=states)
            rc = lib.gennmi_selective_scan(C.byref(c), *space, None)
            refused(rc, -2, many) if more else reaches_the_device(rc)
            rc = lib.gennmi_selective_scan_workspace(C.byref(c), C.byref(size))
            refused(rc, -2, many) if more else None
            assert more or rc == 0
    # gradients: the walk over chunks, a wavefront for a state of a sequence; then the sums of B and C, and those over chunks
    for count, length, channels, states, gradients in (((1 << 22) - 1, 33, 1, 16, {}), (1, 134217720, 1, 16, dict(B=_abi.Rows(30 * FAR, 16, 0))),
                                                       (1, 2, 64 * 32767, 126, dict(A=30 * FAR))):
        g = _abi.ScanGradient(out=_abi.Rows(20 * FAR, channels, channels * length), **gradients)
        for more in (0, 1):
            at = dict(count=count + (more if count > 1 else 0), length=length + (more if length > 100 else 0), channels=channels + (more if channels > 1 else 0), states=states)
            g.out.rowStride, g.out.sequenceStride = at["channels"], at["channels"] * at["length"]
            rc = lib.gennmi_selective_scan_backward(C.byref(wide(scan, **at)), C.byref(g), *space, None)
            refused(rc, -2, many) if more else reaches_the_device(rc)
    c = wide(scan, 1 << 22, 33, channels=1, states=16)
    refused(lib.gennmi_selective_scan_backward_workspace(C.byref(c), C.byref(size)), -2, many)
    # an optimiser: a work-group of 256 threads for 1024 weights
    o, at = C.c_void_p(), 1 << 50
    for count, more in ((((1 << 24) - 1) * 1024, False), (((1 << 24) - 1) * 1024 + 1, True)):
        assert lib.gennmi_optimiser_create(C.byref(o), C.byref(_abi.AdamWSettings(beta1=0.9, beta2=0.99, epsilon=1e-8, stateBits=32))) == 0
        assert lib.gennmi_optimiser_push(o, C.byref(parameter(weight=at, gradient=2 * at, m=3 * at, v=4 * at, count=count)), None) == 0
        rc = lib.gennmi_optimiser_finalise(o)
        refused(rc, -2, "one launch") if more else None
        assert more or rc != -2
        lib.gennmi_optimiser_destroy(o)


def parameter(**changes):
    p = _abi.Parameter(weight=AT, gradient=AT + 8192, m=AT + 16384, v=AT + 32768, count=100, weightType=F32, gradientType=BF16)
    return changed(p, changes)


@pytest.mark.parametrize("change, code, text", [
    (dict(weightType=1), -3, "element type"), (dict(gradientType=4), -3, "element type"), (dict(copy=AT + 65536, copyType=F32), -3, "element type"),
    (dict(weight=None), -2, "missing"), (dict(gradient=None), -2, "missing"), (dict(v=None), -2, "missing"), (dict(weight=AT + 2), -2, "aligned"),
    (dict(m=AT + 16385), -2, "aligned"), (dict(weightDecay=float("nan")), -2, "decay"), (dict(count=1 << 41), -2, "number of weights"),
    (dict(m=AT + 4), -2, "arrays of their own"), (dict(v=AT + 16384), -2, "arrays of their own"), (dict(copy=AT + 100, copyType=BF16), -2, "arrays of their own"),
    (dict(gradient=AT + 200), -2, "arrays of their own"), (dict(gradient=AT + 16384 + 396), -2, "arrays of their own"),
])
def test_optimiser_refuses_tensors(change, code, text):
    lib, o = _abi.load(), C.c_void_p()
    assert lib.gennmi_optimiser_create(C.byref(o), C.byref(_abi.AdamWSettings(beta1=0.9, beta2=0.99, epsilon=1e-8, stateBits=32))) == 0
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter(**change)), None), code, text)
    lib.gennmi_optimiser_destroy(o)


def test_optimiser_refuses_settings_order_and_overlaps():
    lib, o = _abi.load(), C.c_void_p()
    for wrong in (dict(stateBits=16), dict(beta1=1.0), dict(beta2=-0.1), dict(epsilon=float("nan")), dict(epsilon=-1.0), dict(beta1=float("nan"))):
        s = changed(_abi.AdamWSettings(beta1=0.9, beta2=0.99, epsilon=1e-8, stateBits=8), wrong)
        assert lib.gennmi_optimiser_create(C.byref(o), C.byref(s)) < 0 and not o
    assert lib.gennmi_optimiser_create(C.byref(o), C.byref(_abi.AdamWSettings(beta1=0.9, beta2=0.99, epsilon=0.0, stateBits=8))) == 0
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter()), None), -2, "missing")          # (no scales)
    eight = dict(mScale=AT + (1 << 17), vScale=AT + (1 << 18))
    idx = C.c_uint32(7)
    assert lib.gennmi_optimiser_push(o, C.byref(parameter(**eight)), C.byref(idx)) == 0 and idx.value == 0
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter(**eight)), None), -2, "pushed before")
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter(weight=AT + 396, m=AT + (1 << 21), v=AT + (1 << 22), **eight)), None), -2, "pushed before")
    scales = dict(mScale=AT + (1 << 19), vScale=AT + (1 << 20))
    assert lib.gennmi_optimiser_push(o, C.byref(parameter(weight=AT + 400, m=AT + (1 << 21), v=AT + (1 << 22), **scales)), C.byref(idx)) == 0 and idx.value == 1
    third = dict(weight=AT + (1 << 23), m=AT + (1 << 24), v=AT + (1 << 25))
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter(**{**eight, **third})), None), -2, "pushed before")              # (the scales of the first)
    own = dict(mScale=AT + (1 << 26), vScale=AT + (1 << 27))
    refused(lib.gennmi_optimiser_push(o, C.byref(parameter(**{**own, **third, "gradient": AT + 4})), None), -2, "pushed before")     # (weights of the first)
    assert lib.gennmi_optimiser_push(o, C.byref(parameter(**{**own, **third})), C.byref(idx)) == 0 and idx.value == 2       # (the gradient of the first)
    refused(lib.gennmi_optimiser_step(o, C.byref(_abi.AdamWStep(rate=1e-3)), None), -4, "not finalised")
    refused(lib.gennmi_optimiser_step(None, None, None), -2, "null")
    n = C.c_uint64()
    refused(lib.gennmi_optimiser_get_step(o, C.byref(n)), -4, "not finalised")
    refused(lib.gennmi_optimiser_set_step(o, 3), -4, "not finalised")
    assert lib.gennmi_optimiser_destroy(o) == 0 and lib.gennmi_optimiser_destroy(None) == 0


def places(rows, count, length, width):
    """Elements that an array of 16 bits holds, one set a row."""
    return [set(range(rows.data // 2 + s * rows.sequenceStride + t * rows.rowStride, rows.data // 2 + s * rows.sequenceStride + t * rows.rowStride + width))
            for s in range(count) for t in range(length)]


def test_arrays_that_overlap_in_part_are_refused():
    """Any two layouts of rows, against their elements one by one: accepted are those of which no two rows that are written, and none that is written
    and another that is read, share an element."""
    rng, lib, said = random.Random(5), _abi.load(), {True: 0, False: 0}
    for k in range(4000):
        count, length, width = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 4)
        stride = lambda: rng.choice([width, 2 * width, 3 * width, count * width, length * width, (length + 1) * width, rng.randint(width, 40)])
        a = _abi.Rows(AT, stride(), stride())
        b = _abi.Rows(AT + 2 * rng.choice([width, length * width, count * length * width, rng.randint(0, 120)]), *((a.rowStride, a.sequenceStride) if k % 2 else (stride(), stride())))
        x, out = (a, b) if k % 3 else (b, a)
        held, written = places(x, count, length, width), places(out, count, length, width)
        apart = sum(map(len, written)) == len(set().union(*written)) and not set().union(*written) & set().union(*held)
        c = conv(channels=width, taps=1, silu=0, weight=FAR, bias=None, x=x, out=out, sequences__count=count, sequences__length=length, sequences__device=78)
        rc = lib.gennmi_causal_conv(C.byref(c), None)
        if apart:
            reaches_the_device(rc)
        else:
            assert rc == -2 and any(t in lib.gennmi_last_error().decode() for t in ("overlap", "same array")), (lib.gennmi_last_error(), count, length, width, x, out)
        said[apart] += 1
    assert min(said.values()) > 500


def test_states_gradients_and_workspaces_that_overlap_are_refused():
    lib, size = _abi.load(), C.c_size_t()
    far = dict(weight=FAR, bias=2 * FAR, sequences__device=78)
    state = 2 * 3 * 24 * 2              # bytes of the convolution's states
    at = AT + (1 << 16)
    for change, text in ((dict(finalState=at, initialState=at), None), (dict(finalState=at, initialState=at + 2), "the final state overlaps the initial state"),
                         (dict(finalState=at, initialState=at + state), None), (dict(finalState=AT + 470), "the final state overlaps x"), (dict(finalState=AT + 4096 + 470), "out overlaps the final state"),
                         (dict(finalState=FAR + 380), "the final state overlaps weight"), (dict(out__data=AT + 48), "out overlaps x"),
                         (dict(sequences__slots=AT + 4096, sequences__numSlots=2, finalState=at), "out overlaps slots")):
        rc = lib.gennmi_causal_conv(C.byref(conv(**far, **change)), None)
        refused(rc, -2, text) if text else reaches_the_device(rc)
    c = conv(**far, initialState=at)
    assert lib.gennmi_causal_conv_backward_workspace(C.byref(c), C.byref(size)) == 0
    for change, text in ((dict(), None), (dict(initialState=at), None), (dict(initialState=at + 4), "the gradient of the initial state overlaps the initial state"),
                         (dict(x__data=AT + 8192 + 24 * 2), "the gradient of x overlaps the gradient of out"), (dict(weight=AT + 16384), "the gradient of weight overlaps the gradient of x"),
                         (dict(weight=4 * FAR, bias=4 * FAR + 380), "the gradient of weight overlaps the gradient of bias"), (dict(weight=FAR), None),
                         (dict(bias=3 * FAR + 16), "the gradient of bias overlaps the workspace"), (dict(x__data=3 * FAR + 16), "the gradient of x overlaps the workspace")):
        g = changed(_abi.CausalConvGradient(out=_abi.Rows(AT + 8192, 24, 120), x=_abi.Rows(AT + 16384, 24, 120), weight=4 * FAR), change)
        rc = lib.gennmi_causal_conv_backward(C.byref(c), C.byref(g), 3 * FAR, size.value, None)
        refused(rc, -2, text) if text else reaches_the_device(rc)
    far = dict(A=FAR, D=2 * FAR, deltaBias=3 * FAR, sequences__device=78)
    state = 2 * 24 * 16 * 4
    space = 4 * FAR
    for change, text in ((dict(), None), (dict(finalState=at, initialState=at), None), (dict(finalState=at, initialState=at + state - 4), "the final state overlaps the initial state"),
                         (dict(out__data=AT + 4096 * 5 + 2), "out overlaps B"), (dict(out__data=FAR + 1024), "out overlaps A"), (dict(finalState=AT + 4096 * 6), "the final state overlaps C"),
                         # rows of one wide array, side by side, and one element too near
                         (dict(u__rowStride=48, u__sequenceStride=240, out__data=AT + 48, out__rowStride=48, out__sequenceStride=240), None),
                         (dict(u__rowStride=48, u__sequenceStride=240, out__data=AT + 46, out__rowStride=48, out__sequenceStride=240), "out overlaps u"),
                         # time outside, sequences inside
                         (dict(u__rowStride=96, u__sequenceStride=48, out__data=AT + 48, out__rowStride=96, out__sequenceStride=48), None),
                         # sequences that hold all rows of one array, then all of another's, which are not as far apart
                         (dict(u__rowStride=24, u__sequenceStride=400, out__data=AT + 240, out__rowStride=30, out__sequenceStride=400), None),
                         (dict(u__rowStride=24, u__sequenceStride=400, out__data=AT + 238, out__rowStride=30, out__sequenceStride=400), "out overlaps u"),
                         (dict(out__rowStride=24, out__sequenceStride=60), "out: sequences overlap"), (dict(out__rowStride=24, out__sequenceStride=24), "out: sequences overlap")):
        rc = lib.gennmi_selective_scan(C.byref(scan(**far, **change)), space, 1 << 20, None)
        refused(rc, -2, text) if text else reaches_the_device(rc)
    c = scan(**far, sequences__length=100, **{f"{n}__{k}": v for n, w, p in (("u", 24, 10), ("delta", 24, 11), ("z", 24, 12), ("out", 24, 13), ("B", 32, 14), ("C", 32, 15))
                                              for k, v in (("data", p * FAR), ("sequenceStride", 100 * w))})
    assert lib.gennmi_selective_scan_backward_workspace(C.byref(c), C.byref(size)) == 0
    rows = lambda data, width=24, wide=None: _abi.Rows(data, wide or width, 100 * (wide or width))
    for gradients, text in ((dict(u=rows(21 * FAR)), None), (dict(u=rows(10 * FAR + 24)), "the gradient of u overlaps u"), (dict(delta=rows(space + 48)), "the gradient of delta overlaps the workspace"),
                            (dict(u=rows(21 * FAR), delta=rows(21 * FAR + 24)), "the gradient of u overlaps the gradient of delta"),
                            (dict(B=rows(21 * FAR, 32, 64), C=rows(21 * FAR + 64, 32, 64)), None), (dict(B=rows(21 * FAR, 32, 64), C=rows(21 * FAR + 62, 32, 64)), "the gradient of B overlaps the gradient of C"),
                            (dict(A=21 * FAR, D=21 * FAR + 4 * 24 * 16 - 4), "the gradient of A overlaps the gradient of D"), (dict(A=21 * FAR, D=21 * FAR + 4 * 24 * 16), None),
                            (dict(A=FAR, D=2 * FAR, deltaBias=3 * FAR), None), (dict(deltaBias=space + 64), "the gradient of delta's bias overlaps the workspace"),
                            (dict(initialState=21 * FAR, finalState=21 * FAR), None), (dict(initialState=21 * FAR, finalState=21 * FAR + 4), "the gradient of the initial state overlaps the gradient of the final state")):
        g = _abi.ScanGradient(out=rows(20 * FAR), **gradients)
        rc = lib.gennmi_selective_scan_backward(C.byref(c), C.byref(g), space, size.value, None)
        refused(rc, -2, text) if text else reaches_the_device(rc)


# The runtime's calls that an optimiser's table takes, on host memory: copy number `failing` (counted from 1) fails
RUNTIME = r"""
#include <stdlib.h>
#include <string.h>
int failing = 0, copies = 0, live = 0;
struct { void *ptr; size_t bytes; } block[64];
int hipMalloc(void **p, size_t n) { *p = calloc(1, n); block[live].ptr = *p; block[live++].bytes = n; return 0; }
int hipFree(void *p)
{
    for(int k = 0; k < live; k++) { if(block[k].ptr == p) { for(live--; k < live; k++) { block[k] = block[k + 1]; } free(p); return 0; } }
    return p ? 1 : 0;
}
int hipMemcpy(void *to, const void *from, size_t n, int kind) { (void)kind; if(++copies == failing) { return 2; } memcpy(to, from, n); return 0; }
int hipGetDevice(int *device) { *device = 0; return 0; }
"""
FINALISE = """
import ctypes as C, json, sys
runtime = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from genn_amd import _abi
lib, said = _abi.load(), []
for tensors in (2, 0):
    for failing in range(4):
        o = C.c_void_p()
        C.c_int.in_dll(runtime, "copies").value, C.c_int.in_dll(runtime, "failing").value = 0, failing
        assert lib.gennmi_optimiser_create(C.byref(o), C.byref(_abi.AdamWSettings(beta1=0.9, beta2=0.99, epsilon=1e-8, stateBits=32))) == 0
        for k in range(tensors):
            at = (k + 1) << 30
            p = _abi.Parameter(weight=at, gradient=at + 65536, m=2 * at + (1 << 20), v=at + 262144, count=3000 + k, weightDecay=0.5)
            assert lib.gennmi_optimiser_push(o, C.byref(p), None) == 0
        first = lib.gennmi_optimiser_finalise(o)
        live = C.c_int.in_dll(runtime, "live").value
        assert (first != 0) == (failing > 0) and (first == 0 or live == 0), (first, live)
        assert first == 0 or lib.gennmi_optimiser_finalise(o) == 0
        blocks = (C.c_size_t * 128).in_dll(runtime, "block")
        said.append([tensors] + [C.string_at(blocks[2 * k], blocks[2 * k + 1]).hex() for k in range(C.c_int.in_dll(runtime, "live").value)])
        lib.gennmi_optimiser_destroy(o)
        assert C.c_int.in_dll(runtime, "live").value == 0
print(json.dumps(said))
"""


def test_a_table_whose_copy_failed_is_made_anew(tmp_path):
    """Whichever copy of finalise fails, the next attempt uploads what a first one would have, and nothing else is kept."""
    source, shared = tmp_path / "runtime.c", tmp_path / "runtime.so"
    source.write_text(RUNTIME)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(shared), str(source)])
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FINALISE, str(shared), root], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr
    said = json.loads(done.stdout)
    assert len(said) == 8 and all(len(s) == 4 for s in said)
    for k in range(8):
        assert said[k] == said[k // 4 * 4], k


def test_python_layer_refuses_before_it_touches_the_device():
    from genn_amd.operands import Operand
    from genn_amd.sequence import CausalConvolution, SelectiveScan
    for make in (lambda t: CausalConvolution(1, 1, 4, 4, dtype=t), lambda t: SelectiveScan(1, 1, 4, 4, dtype=t)):
        with pytest.raises(NotImplementedError):
            make("float64")
    with pytest.raises(ValueError, match="not on the device"):
        Operand(torch.zeros(3), "x")
    with pytest.raises(TypeError, match="neither"):
        Operand([1.0], "x")


class Elsewhere:
    """What a tensor on a device says of itself."""
    is_cuda, dtype = True, torch.uint8

    def __init__(self, shape, strides, index):
        self.shape, self.strides, self.device = shape, strides, torch.device("cuda", index)

    def data_ptr(self):
        return AT

    def stride(self):
        return self.strides


def test_workspaces_are_looked_at_as_other_arrays_are():
    """On the operator's device, and its bytes one behind another."""
    from genn_amd.sequence import SelectiveScan
    op = SelectiveScan.__new__(SelectiveScan)
    op.device, op._workspaces = 0, {}
    assert op._workspace("forward", Elsewhere((4096,), (1,), 0), 4096, 0) == (AT, 4096)
    with pytest.raises(ValueError, match="on device 1"):
        op._workspace("forward", Elsewhere((4096,), (1,), 1), 4096, 0)
    with pytest.raises(ValueError, match="workspace is not contiguous"):
        op._workspace("forward", Elsewhere((4096,), (2,), 0), 4096, 0)


def test_gradients_of_the_restatements_are_those_of_differences():
    """Along random directions, by central differences: off by a third derivative times step^2 (1e-10 here) and rounding over step (1e-16 / 1e-5)."""
    gen = torch.Generator().manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)
    n, D, N, G, K = 9, 6, 3, 2, 4
    arrays = dict(u=r(n, D), delta=r(n, D) * 0.5, A=-torch.rand(D, N, generator=gen, dtype=torch.float64), B=r(n, G, N), C=r(n, G, N), D=r(D),
                  delta_bias=r(D), z=r(n, D), initial=r(D, N))
    dout, dfinal = r(n, D), r(D, N)

    def value(**a):
        out, final = ref.scan(softplus=True, **a)
        return float((out * dout).sum() + (final * dfinal).sum())

    g = ref.scan(softplus=True, dout=dout, dfinal=dfinal, **arrays)
    for name, x in arrays.items():
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        got = (value(**{**arrays, name: x + 1e-5 * d}) - value(**{**arrays, name: x - 1e-5 * d})) / 2e-5
        assert abs(got - float((g[{"initial": "initial_state"}.get(name, name)] * d).sum())) < 1e-7, name
    arrays = dict(x=r(n, D), weight=r(D, K), bias=r(D), initial=r(K - 1, D))
    dfinal = r(K - 1, D)

    def value(**a):
        out, final = ref.causal_conv(silu=True, **a)
        return float((out * dout).sum() + (final * dfinal).sum())

    g = dict(zip(("x", "weight", "bias", "initial"), ref.causal_conv(silu=True, dout=dout, dfinal=dfinal, **arrays)))
    for name, x in arrays.items():
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        got = (value(**{**arrays, name: x + 1e-5 * d}) - value(**{**arrays, name: x - 1e-5 * d})) / 2e-5
        assert abs(got - float((g[name] * d).sum())) < 1e-7, name


def test_codes_of_the_restatement_are_the_formats():
    values = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(ref.E4M3, values)
    assert torch.equal(ref.e4m3_codes(values), torch.arange(127))
    between = (values[1:] + values[:-1]) / 2                # ties go to the even code
    assert torch.equal(ref.e4m3_codes(between) % 2, torch.zeros(126, dtype=torch.int64))
