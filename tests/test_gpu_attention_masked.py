"""Route attention_masked against the float64 oracle, within the oracle's bound: masks, windows, spans,
prefixes, caps, slopes and tables, both types, head sizes from 8 to 256, rows packed or apart, tokens
that attend nothing, values that are not finite behind a mask, and the calls it refuses."""

import math

import numpy as np
import pytest

from oracle import encoder as ref
from tessery_amd import batching
from tessery_amd.errors import InferenceError

pytestmark = pytest.mark.gpu

TYPES = {"f16": np.float16, "f32": np.float32}


def operands(seed, b, s, h, kv, d, precision, std=1.0):
    rng = np.random.default_rng(seed)
    return [(std * rng.standard_normal((b, s, n, d))).astype(TYPES[precision]) for n in (h, kv, kv)]


def run(rt, q, k, v, lengths, *, packed=False, guard=True, replays=0, **kw):
    """The call on fresh buffers; the output buffer starts as NaN. Extra keyword arrays become
    buffers."""
    b, s, h, d = q.shape
    precision = "f16" if q.dtype == np.float16 else "f32"
    arrays = {n: kw.pop(n) for n in ("prefix", "spans", "slopes", "table") if kw.get(n) is not None}
    for n in ("prefix", "spans"):
        if n in arrays:
            arrays[n] = np.ascontiguousarray(arrays[n], np.uint32)
    for n in ("slopes", "table"):
        if n in arrays:
            arrays[n] = np.ascontiguousarray(arrays[n], np.float32)
    if "table" in arrays:
        kw["radius"] = arrays["table"].shape[1] // 2
    bufs = {n: rt.upload(a) for n, a in arrays.items()}
    rows = rt.upload(np.concatenate((q, k, v), axis=2))
    apart = [rt.upload(x) for x in (q, k, v)]
    qkv = {False: apart, True: [rows] * 3, "v": [apart[0], apart[1], rows]}[packed]
    lens = rt.upload(np.asarray(lengths, np.uint32))
    out = rt.upload(np.full(q.shape, np.nan, q.dtype))
    held = [*bufs.values(), rows, *apart, lens, out]

    def call():
        rt._attention_masked([*qkv, lens, out], tokens=b * s, seq=s, heads=h, kv_heads=k.shape[2],
                             dim=d, precision=precision, packed=packed, **bufs, **kw)

    try:
        with rt.command():
            call()
        return rt.read(out, q.shape, q.dtype)
    finally:
        for buf in held:
            buf.close()


def check(rt, q, k, v, lengths, **kw):
    options = {n: x for n, x in kw.items() if n != "packed"}
    want, bound = ref.attention_masked(q, k, v, np.asarray(lengths), **options)
    got = run(rt, q, k, v, lengths, **kw).astype(np.float64)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    assert over.max() <= 0, (float(over.max()), float(np.abs(got - want).max()))
    return got


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 80, 96, 128, 136, 256])
@pytest.mark.parametrize("mask", ["causal", "bidirectional"])
def test_head_sizes(runtime, precision, dim, mask):
    q, k, v = operands(dim, 2, 75, 4, 2, dim, precision)
    check(runtime, q, k, v, [75, 33], mask=mask)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("seq", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 321])
def test_lengths(runtime, precision, seq):
    q, k, v = operands(seq, 2, seq, 3, 1, 64, precision)
    for mask in ("causal", "bidirectional"):
        check(runtime, q, k, v, [seq, (seq + 1) // 2], mask=mask)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (6, 2), (8, 1), (16, 8)])
@pytest.mark.parametrize("packed", [False, True, "v"])
def test_heads_and_rows(runtime, precision, heads, kv_heads, packed):
    q, k, v = operands(heads, 2, 90, heads, kv_heads, 32, precision)
    check(runtime, q, k, v, [90, 41], mask="causal", packed=packed)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 2**31, 2**32 - 1])
@pytest.mark.parametrize("mask", ["causal", "bidirectional", "prefix"])
def test_windows(runtime, precision, window, mask):
    q, k, v = operands(window % 97, 2, 150, 2, 2, 64, precision)
    prefix = np.array([40, 149]) if mask == "prefix" else None
    check(runtime, q, k, v, [150, 70], mask=mask, window=window, prefix=prefix)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [(0, 1), (64, 150), (2**32 - 1, 77)])
def test_prefixes(runtime, precision, prefix):
    q, k, v = operands(7, 2, 150, 4, 2, 64, precision)
    check(runtime, q, k, v, [150, 70], mask="prefix", prefix=np.array(prefix, np.uint32))


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("mask", ["causal", "bidirectional"])
@pytest.mark.parametrize("documents", [[[64, 64, 72], [1, 1, 198]], [[200], [3, 0, 30, 5, 90]],
                                       [[], [7] * 28]])
def test_documents(runtime, precision, mask, documents):
    """Documents that end at, before and inside a tile; tokens behind the documents attend nothing and
    get zeros."""
    q, k, v = operands(8, 2, 200, 4, 4, 64, precision)
    got = check(runtime, q, k, v, [200, 200], mask=mask,
                spans=batching.document_spans(documents, 200))
    for b, lengths in enumerate(documents):
        assert not got[b, sum(lengths):].any()


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_spans_of_any_values(runtime, precision):
    """Spans are ranges, whatever they hold: empty, turned round, past the row, away from the token."""
    q, k, v = operands(9, 1, 140, 2, 2, 64, precision)
    spans = np.random.default_rng(9).integers(0, 220, size=(1, 140, 2)).astype(np.uint32)
    spans[0, 3], spans[0, 4], spans[0, 5] = (2**32 - 1, 2**32 - 1), (0, 2**32 - 1), (139, 140)
    check(runtime, q, k, v, [131], mask="bidirectional", spans=spans)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("cap", [0.5, 30.0, 50.0])
@pytest.mark.parametrize("std", [0.05, 1.0, 6.0])
def test_caps(runtime, precision, cap, std):
    q, k, v = operands(10, 2, 100, 4, 2, 64, precision, std)
    v = (v / std).astype(v.dtype)
    check(runtime, q, k, v, [100, 64], mask="causal", cap=cap)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("cap", [256.0, 300.0, 1e5])
@pytest.mark.parametrize("biased", [False, True])
def test_wide_caps(runtime, precision, cap, biased):
    """Caps far above the scores leave them as exact as they were (the fp32 bound holds that of every
    cap: it goes with the score, not with the cap)."""
    q, k, v = operands(30, 2, 100, 4, 2, 64, precision)
    slopes = np.array([0.1, 0.02, 0.3, 0.0], np.float32) if biased else None
    check(runtime, q, k, v, [100, 64], mask="bidirectional", cap=cap, slopes=slopes)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("mask", ["causal", "bidirectional"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_slopes(runtime, precision, mask, cap):
    q, k, v = operands(11, 2, 170, 6, 3, 64, precision)
    check(runtime, q, k, v, [170, 90], mask=mask, cap=cap,
          slopes=(2.0 ** (-8 * np.arange(1, 7) / 6)).astype(np.float32))


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("radius", [0, 1, 20, 128, 1000])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_tables(runtime, precision, radius, cap):
    q, k, v = operands(12, 2, 170, 4, 2, 64, precision)
    table = np.random.default_rng(12).standard_normal((4, 2 * radius + 1)).astype(np.float32)
    check(runtime, q, k, v, [170, 90], mask="bidirectional", cap=cap, table=table)


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_tables_that_mask(runtime, precision):
    """A table may hide distances with -inf (a token left with nothing else gets zeros) or with the
    type's lowest value (one left with nothing else attends its keys alike)."""
    q, k, v = operands(13, 1, 100, 2, 2, 32, precision)
    table = np.zeros((2, 41), np.float32)
    table[0, :21] = -np.inf     # head 0: only keys behind the token
    table[1, :21] = np.finfo(np.float32).min
    want, bound = ref.attention_masked(q, k, v, np.array([100]), mask="bidirectional", table=table)
    got = run(runtime, q, k, v, [100], mask="bidirectional", table=table).astype(np.float64)
    assert not got[0, 99, 0].any()  # the last token of head 0 has no key behind it
    np.testing.assert_allclose(got[0, 99, 1], v[0, :, 1].astype(np.float64).mean(0),
                               atol=2e-3 if precision == "f16" else 2e-6)
    assert np.all(np.abs(got - want)[0, :, 0] <= bound[0, :, 0])
    assert np.all(np.abs(got - want)[0, :99, 1] <= bound[0, :99, 1])


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_behind_a_mask_do_not_reach(runtime, precision, dim, bad):
    """Keys and values past the length, of other documents, later in the row: what they hold changes no
    token that does not attend them, to the bit or within the bound (a row recomputed on its own)."""
    q, k, v = operands(14, 2, 150, 4, 2, dim, precision)
    spans = batching.document_spans([[50, 45, 55], [150]], 150)
    lengths = [150, 101]
    want, bound = ref.attention_masked(q, k, v, np.array(lengths), mask="causal", spans=spans)
    k2, v2 = k.copy(), v.copy()
    for x in (k2, v2):
        x[0, 60] = bad   # in the second document: tokens 60 .. 94 see it
        x[1, 101:] = bad  # past the length
    got = run(runtime, q, k2, v2, lengths, mask="causal", spans=spans).astype(np.float64)
    clean = np.ones(150, bool)
    clean[60:95] = False
    assert np.all(np.abs(got - want)[0, clean] <= bound[0, clean])
    assert np.all(np.abs(got - want)[1] <= bound[1])
    assert np.isnan(got[0, 60:95]).all()


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_a_query_that_is_not_finite_stays_alone(runtime, precision):
    q, k, v = operands(15, 1, 70, 2, 2, 64, precision)
    want, bound = ref.attention_masked(q, k, v, np.array([70]), mask="bidirectional")
    q[0, 33, 1, 5] = np.nan
    got = run(runtime, q, k, v, [70], mask="bidirectional").astype(np.float64)
    keep = np.ones((70, 2), bool)
    keep[33, 1] = False
    assert np.all(np.abs(got - want)[0][keep] <= bound[0][keep])
    assert np.isnan(got[0, 33, 1]).all()


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_infinite_values_that_are_attended(runtime, precision):
    q, k, v = operands(16, 1, 40, 1, 1, 64, precision)
    v[0, 10, 0, 3] = np.inf
    got = run(runtime, q, k, v, [40], mask="causal")
    assert np.isposinf(got[0, 10:, 0, 3]).all() and np.isfinite(got[0, :10]).all()
    assert np.isfinite(np.delete(got[0, 10:, 0], 3, axis=-1)).all()


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_empty_rows_and_zero_lengths(runtime, precision):
    q, k, v = operands(17, 3, 66, 2, 1, 64, precision)
    got = check(runtime, q, k, v, [0, 66, 1], mask="bidirectional")
    assert not got[0].any()
    # a window that ends before the keys do leaves the padded tokens far behind them nothing
    got = check(runtime, q, k, v, [10, 66, 1], mask="causal", window=5)
    assert not got[0, 14:].any() and got[0, 13].any()


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_large_scores(runtime, precision):
    """Scores of hundreds: the running maximum carries them."""
    q, k, v = operands(18, 1, 300, 2, 2, 64, precision, std=5.0)
    check(runtime, q, k, v, [300], mask="causal", scale=1.0)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("cap", [0.0, 3.0])
@pytest.mark.parametrize("biased", [False, True])
def test_scales_that_are_not_positive(runtime, precision, scale, cap, biased):
    q, k, v = operands(22, 1, 100, 2, 2, 64, precision)
    slopes = np.array([0.1, 0.02], np.float32) if biased else None
    check(runtime, q, k, v, [100], mask="causal", scale=scale, cap=cap, slopes=slopes)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("b,s,h,kv,d", [(70, 40, 2, 1, 32), (3, 700, 12, 12, 64), (1, 1500, 2, 2, 128),
                                        (2, 600, 3, 1, 256), (6, 130, 16, 8, 96), (1, 900, 1, 1, 32)])
def test_many_and_few_workgroups(runtime, precision, b, s, h, kv, d):
    """Batches on either side of every rule that shares the keys of a block out, and more rows than
    are put in order of length."""
    q, k, v = operands(23, b, s, h, kv, d, precision)
    lengths = np.random.default_rng(23).integers(1, s + 1, size=b)
    rows = np.unique(np.random.default_rng(24).integers(0, s, size=12))
    for kw in (dict(mask="causal"), dict(mask="bidirectional", cap=9.0),
               dict(mask="causal", slopes=np.full(h, 0.05, np.float32))):
        got = run(runtime, q, k, v, lengths, **kw).astype(np.float64)
        assert np.isfinite(got).all()
        for n in {0, b // 2, b - 1}:  # a few tokens of a few batch rows
            one = slice(n, n + 1)
            want, bound = ref.attention_masked(q[one], k[one], v[one], lengths[one], tokens=rows, **kw)
            assert np.all(np.abs(got[n, rows] - want[0, rows]) <= bound[0, rows])


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("d", [8, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("s", [1, 2, 4, 5, 8, 9])
def test_a_few_tokens(runtime, precision, d, s):
    """Batch rows on either side of the lengths that go without tiles."""
    q, k, v = operands(31, 7, s, 6, 2, d, precision)
    lengths = np.random.default_rng(31).integers(0, s + 1, size=7)
    check(runtime, q, k, v, lengths, mask="causal")
    check(runtime, q, k, v, lengths, mask="prefix", prefix=lengths[::-1].copy(), cap=5.0, packed=True)
    check(runtime, q, k, v, lengths, mask="bidirectional", window=2,
          slopes=np.array([0.1, 0.02, 0.3, 0.0, 1.0, 0.5], np.float32))
    table = np.random.default_rng(32).standard_normal((6, 7)).astype(np.float32)
    check(runtime, q, k, v, lengths, mask="causal", table=table,
          spans=batching.document_spans([[s // 2, s - s // 2] if s > 1 else [1]] * 7, s))


def test_very_many_single_tokens(runtime):
    """The weight of a lone key is one: a row is its value, to the last of 2^24."""
    many, v = 2**19, np.random.default_rng(33).standard_normal((2**19, 1, 1, 8)).astype(np.float16)
    q = np.ones((many, 1, 32, 8), np.float16)
    got = run(runtime, q, v, v, np.ones(many, np.uint32), mask="causal")
    np.testing.assert_array_equal(got, np.broadcast_to(v, got.shape))


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_all_at_once(runtime, precision):
    q, k, v = operands(19, 2, 260, 8, 4, 128, precision)
    table = np.random.default_rng(19).standard_normal((8, 65)).astype(np.float32)
    check(runtime, q, k, v, [260, 131], mask="prefix", prefix=np.array([30, 200]), window=90,
          cap=25.0, table=table, packed=True,
          spans=batching.document_spans([[100, 160], [131]], 260))


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("mask", ["causal", "bidirectional"])
@pytest.mark.parametrize("spans", ["documents", "anything"])
def test_many_blocks_of_documents(runtime, precision, mask, spans):
    """So many workgroups that blocks of long documents come first: each block is one's, whatever the
    spans hold."""
    q, k, v = operands(34, 2, 1090, 48, 24, 8, precision)
    if spans == "documents":
        at = batching.document_spans([[7, 500, 64, 1, 128, 300, 90], [1, 1, 700, 20]], 1090)
    else:
        at = np.random.default_rng(35).integers(0, 1300, size=(2, 1090, 2)).astype(np.uint32)
        at[0, ::64], at[1, 63::64] = (0, 2**32 - 1), (2**32 - 1, 0)
    check(runtime, q, k, v, [1090, 722], mask=mask, spans=at)


def test_a_long_row_of_documents(runtime):
    rng = np.random.default_rng(20)
    lengths = []
    while sum(lengths) < 2000:
        lengths.append(int(rng.integers(1, 300)))
    q, k, v = operands(20, 1, 2500, 1, 1, 64, "f16")
    check(runtime, q, k, v, [2500], mask="bidirectional",
          spans=batching.document_spans([lengths], 2500))


def test_same_bits_every_time(runtime):
    q, k, v = operands(21, 2, 300, 4, 2, 64, "f16")
    first = run(runtime, q, k, v, [300, 222], mask="causal")
    for _ in range(3):
        np.testing.assert_array_equal(run(runtime, q, k, v, [300, 222], mask="causal"), first)


def test_refusals(runtime):
    shape = dict(tokens=48, seq=24, heads=4, kv_heads=2, dim=64, precision="f16")
    q, out = runtime.buffer(48 * 4 * 64 * 2), runtime.buffer(48 * 4 * 64 * 2)
    k, v = runtime.buffer(48 * 2 * 64 * 2), runtime.buffer(48 * 2 * 64 * 2)
    lens, small = runtime.buffer(8), runtime.buffer(16)
    rows = runtime.buffer(48 * 8 * 64 * 2)

    def refused(buffers, **kw):
        with pytest.raises(InferenceError):
            with runtime.command():
                runtime._attention_masked(buffers, **{**shape, **kw})

    refused([small, k, v, lens, out])
    refused([q, small, v, lens, out])
    refused([q, k, small, lens, out])
    refused([q, k, v, lens, small])
    refused([q, k, v, lens, q])             # the output is an input
    refused([q, k, v, lens, lens])
    refused([q, k, v, lens, out], precision="f32")
    refused([q, k, v, lens, out], packed=True)
    refused([rows, k, rows, lens, out], packed=True)
    refused([q, k, v, lens, out], packed="v")
    refused([q, k, v, lens, out], spans=small)
    refused([q, k, v, lens, out], table=small, radius=10)
    refused([q, k, v, lens, out], slopes=lens)
    refused([q, k, v, lens, out], tokens=24 * 5, mask="prefix", prefix=lens)
    with runtime.command():
        runtime._attention_masked([rows, rows, rows, lens, out], **{**shape, "packed": True})
    assert math.prod((48, 8, 64)) * 2 == rows.size
