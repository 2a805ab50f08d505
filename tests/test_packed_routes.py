"""Routes attention_masked, rotary and linear_f16 without a GPU: the launches the runtime's methods
make, the calls they refuse, and the host helpers of packed rows and rotation tables."""

import math
from types import SimpleNamespace

import numpy as np
import pytest

from tessery_amd import batching, rotary
from tessery_amd.errors import InferenceError
from tessery_amd.runtime import HipRuntime


def recorder():
    calls = []
    return calls, SimpleNamespace(_dispatch=lambda *a, **kw: calls.append((a, kw)))


ATTENTION = dict(tokens=48, seq=24, heads=8, kv_heads=2, dim=64)
ROTARY = dict(tokens=48, seq=24, heads=8, kv_heads=2, dim=64, rotary_dim=32)
LINEAR = dict(rows=5, cols=7, k=9)


def attention(buffers="qkvlo", **changes):
    calls, fake = recorder()
    HipRuntime._attention_masked(fake, list(buffers), **{**ATTENTION, **changes})
    (args, kw), = calls
    return args, kw


def rotate(buffers="qktQK", **changes):
    calls, fake = recorder()
    HipRuntime._rotary(fake, list(buffers), **{**ROTARY, **changes})
    (args, kw), = calls
    return args, kw


def linear(buffers="xwo", **changes):
    calls, fake = recorder()
    HipRuntime._linear_f16(fake, list(buffers), **{**LINEAR, **changes})
    (args, kw), = calls
    return args, kw


def test_attention_launch():
    (name, bufs), kw = attention()
    assert name == "attention_masked" and bufs == list("qkvlolll")
    assert kw["threads"] == 48 and kw["group_size"] == 256
    assert kw["scale"] == 0.125 and kw["theta"] == 0.0 and kw["n"] == 0
    assert kw["bidirectional"] == 0 and kw["flags"] == 1
    (_, bufs), kw = attention(mask="prefix", prefix="p", spans="s", table="t", radius=5, window=9,
                              cap=30, scale=0.5, precision="f32", packed=True)
    assert bufs == list("qkvlostp") and kw["bidirectional"] == 2
    assert kw["flags"] == 2 + 8 + 16 + 32 and kw["rows"] == 5 and kw["n"] == 9
    assert kw["theta"] == 30.0 and kw["scale"] == 0.5
    (_, bufs), kw = attention(slopes="a", packed="v", mask="bidirectional")
    assert bufs == list("qkvlolal") and kw["flags"] == 1 + 4 + 32 and kw["bidirectional"] == 1


@pytest.mark.parametrize("changes", [
    dict(tokens=47), dict(tokens=0), dict(seq=0), dict(heads=3), dict(heads=0), dict(kv_heads=0),
    dict(dim=60), dict(dim=264), dict(dim=0), dict(dim=64.0), dict(mask="other"),
    dict(mask="prefix"), dict(prefix="p"), dict(precision="bf16"), dict(packed="k"),
    dict(window=-1), dict(window=2**32), dict(window=1.5), dict(radius=4), dict(table="t", radius=-1),
    dict(table="t", radius=2**20 + 1), dict(slopes="s", table="t"), dict(cap=-1.0), dict(cap=1e-31),
    dict(cap=math.inf), dict(cap=math.nan), dict(scale=math.inf), dict(scale=math.nan)])
def test_attention_refusals(changes):
    with pytest.raises(InferenceError):
        attention(**changes)


def test_attention_takes_five_buffers():
    with pytest.raises(InferenceError):
        attention("qkvl")


def test_rotary_launch():
    (name, bufs), kw = rotate()
    assert name == "rotary" and bufs == list("qktttt") + ["Q", "K"] and kw["flags"] == 1
    assert kw["k"] == 32 and kw["bidirectional"] == 0 and kw["threads"] == 48
    (_, bufs), kw = rotate(positions="p", q_norm="a", k_norm="b", layout="interleaved",
                           precision="f32", eps=1e-5)
    assert bufs == list("qkptabQK") and kw["flags"] == 6 and kw["bidirectional"] == 1
    assert kw["eps"] == 1e-5
    (_, bufs), kw = rotate(["p", "p", "t", "p", "p"], packed=True)
    assert kw["flags"] == 1 + 8 + 16  # in place
    (_, bufs), kw = rotate(["p", "p", "t", "Q", "K"], packed=True)
    assert kw["flags"] == 1 + 8
    (_, bufs), kw = rotate(["q", None, "t", "Q", None], kv_heads=0, q_norm="a")
    assert bufs == ["q", "t", "t", "t", "a", "t", "Q", "t"] and kw["flags"] == 5


@pytest.mark.parametrize("changes", [
    dict(tokens=47), dict(seq=0), dict(heads=0), dict(kv_heads=-1), dict(dim=0), dict(dim=1026),
    dict(rotary_dim=31), dict(rotary_dim=66), dict(rotary_dim=0), dict(layout="other"),
    dict(precision="bf16"), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
    dict(q_norm="a"), dict(k_norm="a"), dict(kv_heads=0, k_norm="a"),
    dict(kv_heads=0, packed=True)])
def test_rotary_refusals(changes):
    with pytest.raises(InferenceError):
        rotate(**changes)


@pytest.mark.parametrize("kw", [dict(positions=0, rotary_dim=8), dict(positions=4, rotary_dim=7),
                                dict(positions=4, rotary_dim=0),
                                dict(positions=4, rotary_dim=8, factor=math.nan)])
def test_rotary_table_refusals(kw):
    with pytest.raises(InferenceError):
        HipRuntime._rotary_table(recorder()[1], ["f", "t"], **kw)


def test_linear_launch():
    (name, bufs), kw = linear()
    assert name == "linear_f16" and bufs == list("xwxxo") and kw["flags"] == 0
    assert (kw["rows"], kw["cols"], kw["k"], kw["threads"]) == (5, 7, 9, 5)
    (_, bufs), kw = linear(bias="b", residual="r", activation="silu", out_dtype="f32")
    assert bufs == list("xwbro") and kw["flags"] == 7 and kw["bidirectional"] == 4


@pytest.mark.parametrize("changes", [dict(rows=0), dict(cols=0), dict(k=0), dict(rows=2.0),
                                     dict(activation="tanh"), dict(out_dtype="bf16")])
def test_linear_refusals(changes):
    with pytest.raises(InferenceError):
        linear(**changes)


def test_document_spans_and_positions():
    spans = batching.document_spans([[3, 0, 2], [6], []], 6)
    assert spans.dtype == np.uint32 and spans.shape == (3, 6, 2)
    assert spans[0].tolist() == [[0, 3]] * 3 + [[3, 5]] * 2 + [[0, 0]]
    assert spans[1].tolist() == [[0, 6]] * 6 and not spans[2].any()
    positions = batching.document_positions([[3, 0, 2], [6], []], 6)
    assert positions.tolist() == [[0, 1, 2, 0, 1, 0], [0, 1, 2, 3, 4, 5], [0] * 6]
    for bad in ([[4, 3]], [[-1]]):
        with pytest.raises(InferenceError):
            batching.document_spans(bad, 6)


def test_frequencies():
    base, one = rotary.frequencies(64, 1e4)
    np.testing.assert_allclose(base, 1e4 ** (-np.arange(32) / 32), rtol=1e-15)
    assert one == 1.0
    squeezed, _ = rotary.frequencies(64, 1e4, scaling="linear", factor=4.0)
    np.testing.assert_allclose(squeezed, base / 4, rtol=1e-15)
    ntk, _ = rotary.frequencies(64, 1e4, scaling="ntk", factor=4.0)
    np.testing.assert_allclose(ntk[[0, -1]], [base[0], base[-1] / 4], rtol=1e-13)
    yarn, factor = rotary.frequencies(64, 1e4, scaling="yarn", factor=4.0, trained=4096)
    turns = 4096 * base / (2 * math.pi)
    np.testing.assert_array_equal(yarn[turns >= 32], base[turns >= 32])
    np.testing.assert_allclose(yarn[turns <= 1], base[turns <= 1] / 4, rtol=1e-15)
    assert np.all((yarn <= base) & (yarn >= base / 4)) and (turns <= 1).any() and (turns >= 32).any()
    assert math.isclose(factor, 1.0 + 0.1 * math.log(4.0))


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(theta=0.0), dict(theta=math.inf),
                                dict(scaling="other"), dict(factor=0.5), dict(factor=math.inf),
                                dict(scaling="yarn"), dict(scaling="yarn", trained=8, slow=4, fast=2)])
def test_frequencies_refusals(kw):
    with pytest.raises(InferenceError):
        rotary.frequencies(**{**dict(dim=8, theta=1e4), **kw})
