"""Refusals and host-side parts of the token operators (no GPU): rotary plans, argument
checks of s2s_rotary_apply and s2s_masked_attention. Every refused call names addresses
that are never read: the checks come before any device work."""
import ctypes
import importlib
import math

import pytest

from s2s_testlib import pkg


def binding():
    pkg()
    return importlib.import_module("swin2sr_b200.capi")


ADDR = 1 << 20  # aligned, never dereferenced


def refused(fn, text, *args, **kw):
    C = binding()
    with pytest.raises(C.S2SError) as e:
        fn(*args, **kw)
    assert e.value.code == C.S2S_ERR_INVALID and text in str(e.value), str(e.value)


@pytest.mark.parametrize("cap", [1e-30, 9e-13, 1.1e12, 3e38])
def test_caps_whose_quotients_leave_32_bits(cap):
    refused(attention, "cap must be", cap=cap, scale=1e12 if cap < 1 else 1e-12)


def test_rotary_plan_series_and_axes():
    C = binding()
    r = C.rotary_plan([2, 3, 1], 100.0)
    assert (r.axes, r.pairs, r.interleaved) == (3, 6, 0)
    assert list(r.axis[:6]) == [0, 0, 1, 1, 1, 2]
    for p in range(6):
        assert r.frequency[p] == pytest.approx(100.0 ** (-p / 6), rel=1e-15)
    r = C.rotary_plan([2, 0, 3], 100.0, per_axis=True, interleaved=True)
    assert r.interleaved == 1 and list(r.axis[:5]) == [0, 0, 2, 2, 2]
    want = [1.0, 100.0 ** -0.5, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]
    assert list(r.frequency[:5]) == pytest.approx(want, rel=1e-15)


@pytest.mark.parametrize("sections,base,text", [
    ([], 1e4, "axes must be"), ([1, 1, 1, 1], 1e4, "axes must be"), ([0], 1e4, "sum to"),
    ([-1, 4], 1e4, "a section must be"), ([129], 1e4, "a section must be"),
    ([100, 100], 1e4, "sum to"), ([4], 0.0, "base"), ([4], -2.0, "base"),
    ([4], math.nan, "base"), ([4], math.inf, "base")])
def test_rotary_plan_refusals(sections, base, text):
    refused(binding().rotary_plan, text, sections, base)


@pytest.mark.parametrize("change,text", [
    (dict(head_dim=15), "head_dim"), (dict(tokens=-1), "tokens"), (dict(d_pos=0), "d_pos"),
    (dict(d_pos=ADDR + 2), "d_pos"), (dict(pos_stride=9), "pos_stride"), (dict(n=0), "n must be"),
    (dict(n=5), "n must be"), (dict(x=(0, 64, 16, 4)), "null data"),
    (dict(x=(ADDR + 1, 64, 16, 4)), "aligned"), (dict(x=(ADDR, 0, 16, 4)), "token_stride"),
    (dict(x=(ADDR, 64, -16, 4)), "head_stride"), (dict(x=(ADDR, 64, 16, 3)), "differ in heads"),
    (dict(y=(ADDR, 64, 8, 4)), "head_stride is less"), (dict(y=(ADDR, 8, 16, 4)), "token_stride is less"),
    (dict(x=(ADDR, 64, 16, 0)), "heads must be"), (dict(x=(ADDR, 1 << 50, 16, 4)), "token_stride"),
    (dict(axis=7), "axis is out of range"), (dict(frequency=math.inf), "not finite"),
    (dict(pairs=0), "out of range"), (dict(pairs=200), "out of range"), (dict(axes=0), "out of range")])
def test_rotary_refusals(change, text):
    C = binding()
    r = C.rotary_plan([4, 4])
    if "axis" in change:
        r.axis[3] = change["axis"]
    if "frequency" in change:
        r.frequency[7] = change["frequency"]
    for f in ("pairs", "axes"):
        if f in change:
            setattr(r, f, change[f])
    x, y = C.heads(*change.get("x", (ADDR, 64, 16, 4))), C.heads(*change.get("y", (ADDR, 64, 16, 4)))
    refused(C.rotary, text, r, "float16", change.get("head_dim", 16), change.get("tokens", 10),
            change.get("d_pos", ADDR), change.get("pos_stride", 10), [(x, y)] * change.get("n", 1))


def test_dtype_names():
    C = binding()
    with pytest.raises(ValueError, match="dtype must be one of"):
        C.rotary(C.rotary_plan([4]), "float64", 8, 0, 0, 0, [(C.heads(0, 8, 8, 1),) * 2])


BASE = dict(dtype="float16", head_dim=32, scale=0.2, q=(ADDR, 128, 32, 4), k=(ADDR, 64, 32, 2),
            v=(ADDR, 64, 32, 2), out=(ADDR, 128, 32, 4), q_tokens=10, kv_tokens=20, documents=2)


def attention(**change):
    C = binding()
    a = {**BASE, **change}
    for f in ("q", "k", "v", "out"):
        a[f] = C.heads(*a[f])
    C.attention(**a)


@pytest.mark.parametrize("change,text", [
    (dict(dtype="float32"), "dtype"), (dict(head_dim=0), "head_dim"), (dict(head_dim=12), "head_dim"),
    (dict(head_dim=136), "head_dim"), (dict(q_tokens=-1), "must be >= 0"),
    (dict(kv_tokens=-1), "must be >= 0"), (dict(documents=-1), "must be >= 0"),
    (dict(d_q_offsets=ADDR), "come together"), (dict(d_kv_offsets=ADDR), "come together"),
    (dict(documents=3), "must divide"), (dict(d_prefix=ADDR), "causal"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=math.nan), "cap"),
    (dict(cap=math.inf), "cap"), (dict(axes=-1), "axes"), (dict(axes=4), "axes"),
    (dict(axes=1), "axes need"), (dict(axes=1, d_slopes=ADDR, d_q_pos=ADDR), "axes need"),
    (dict(q=(ADDR + 8, 128, 32, 4)), "16-byte"), (dict(k=(ADDR, 68, 32, 2)), "token_stride"),
    (dict(v=(ADDR, 64, 36, 2)), "head_stride"), (dict(out=(ADDR, 128, 24, 4)), "head_stride"),
    (dict(out=(ADDR, 128, 24, 4)), "less than head_dim"), (dict(q=(0, 128, 32, 4)), "null data"),
    (dict(v=(ADDR, 64, 32, 1)), "same heads"), (dict(k=(ADDR, 96, 32, 3), v=(ADDR, 96, 32, 3)), "multiple"),
    (dict(out=(ADDR, 128, 32, 2)), "same heads"), (dict(d_lse=ADDR + 1), "4-byte"),
    (dict(k=(ADDR, 0, 32, 2)), "token_stride")])
def test_attention_refusals(change, text):
    refused(attention, text, **change)


@pytest.mark.parametrize("tensors,text", [
    ([((1, 64, 16, 4), (2, 63, 16, 4))], "run into"), ([((1, 64, 16, 4), (2, 16, 159, 4))], "run into"),
    ([((1, 64, 16, 4), (2, 16, 16, 4))], "run into"),
    ([((1, 64, 16, 4), (2, 64, 16, 4)), ((3, 64, 16, 4), (2, 64, 16, 4))], "another tensor"),
    ([((1, 64, 16, 4), (2, 64, 16, 4)), ((2, 64, 16, 4), (3, 64, 16, 4))], "another tensor"),
    ([((1, 64, 16, 4), (1, 128, 16, 4))], "same strides")])
def test_rotary_outputs_over_other_tensors(tensors, text):
    C = binding()
    rows = [tuple(C.heads(ADDR * x[0], *x[1:]) for x in pair) for pair in tensors]
    refused(C.rotary, text, C.rotary_plan([4, 4]), "float16", 16, 10, ADDR, 10, rows)


@pytest.mark.parametrize("change,text", [
    (dict(out=(2 * ADDR, 120, 32, 4)), "run into"), (dict(out=(2 * ADDR, 32, 312, 4)), "run into"),
    (dict(out=(ADDR, 128, 32, 4)), "one another"), (dict(out=(2 * ADDR, 128, 32, 4), d_lse=ADDR), "one another"),
    (dict(out=(2 * ADDR, 128, 32, 4), d_lse=2 * ADDR), "one another"),
    (dict(q=(3 * ADDR, 128, 32, 4), out=(ADDR, 128, 32, 4)), "one another")])
def test_attention_outputs_over_other_tensors(change, text):
    refused(attention, text, **change)


def test_nothing_to_do_is_no_error():
    C = binding()
    attention(q_tokens=0, kv_tokens=0)
    attention(documents=0)
    x = C.heads(0, 16, 16, 1)
    C.rotary(C.rotary_plan([4]), "bfloat16", 8, 0, 0, 0, [(x, x)])


def test_struct_sizes_match_the_header():
    """The ctypes mirrors against the C layout (x86-64): 8-byte aligned members."""
    C = binding()
    assert ctypes.sizeof(C.S2SHeads) == 32
    assert ctypes.sizeof(C.S2SRotary) == 12 + 128 + 4 + 128 * 8
    assert C.S2SAttention.scale.offset == 48 and C.S2SAttention.q.offset == 88
    assert ctypes.sizeof(C.S2SAttention) == 88 + 4 * 32 + 8
