"""Routes rotary and rotary_table against the float64 oracle, within the oracle's bound: layouts, parts
of the head, norms, types, packed rows in place and out of them, positions of documents and beyond the
table, scaled frequencies, and the calls it refuses."""

import numpy as np
import pytest

from oracle import encoder as ref
from tessery_amd import batching, rotary
from tessery_amd.errors import InferenceError
from tessery_amd.workloads import bf16_values, bf16_words

pytestmark = pytest.mark.gpu

TYPES = {"f16": np.float16, "f32": np.float32}


def run(rt, q, k, *, seq, rot, layout, table, packed=False, place=False, positions=None, norms=None,
        eps=1e-6):
    """Rotated q and k, and v (random) of packed rows as it was left."""
    tokens, h, d = q.shape
    kv = 0 if k is None else k.shape[1]
    dtype = q.dtype
    held = []

    def up(x):
        held.append(rt.upload(x))
        return held[-1]

    v = np.random.default_rng(1).standard_normal((tokens, kv, d)).astype(dtype)
    try:
        if packed:
            rows = up(np.concatenate((q, k, v), axis=1))
            bufs = [rows, rows]
            outs = bufs if place else [up(np.full_like(q, np.nan)), up(np.full_like(k, np.nan))]
        else:
            bufs = [up(q), None if k is None else up(k)]
            outs = bufs if place else [up(np.full_like(q, np.nan)),
                                       None if k is None else up(np.full_like(k, np.nan))]
        extra = {}
        if positions is not None:
            extra["positions"] = up(np.ascontiguousarray(positions, np.uint32))
        if norms is not None:
            extra["q_norm"] = up(norms[0])
            if kv:
                extra["k_norm"] = up(norms[1])
        with rt.command():
            rt._rotary([*bufs, table, *outs], tokens=tokens, seq=seq, heads=h, kv_heads=kv, dim=d,
                       rotary_dim=rot, layout=layout, packed=packed, eps=eps,
                       precision="f16" if dtype == np.float16 else "f32", **extra)
        if packed and place:
            got = rt.read(rows, (tokens, h + 2 * kv, d), dtype)
            np.testing.assert_array_equal(got[:, h + kv:], v)
            return got[:, :h], got[:, h:h + kv]
        return (rt.read(outs[0], q.shape, dtype),
                None if k is None else rt.read(outs[1], k.shape, dtype))
    finally:
        for b in held:
            b.close()


def check(rt, seed, batch, seq, h, kv, d, rot, precision, *, layout="half", packed=False, place=False,
          norm=False, positions=None, values=None, factor=1.0, rows=None, eps=1e-6):
    rng = np.random.default_rng(seed)
    tokens, dtype = batch * seq, TYPES[precision]
    q = rng.standard_normal((tokens, h, d)).astype(dtype)
    k = rng.standard_normal((tokens, kv, d)).astype(dtype) if kv else None
    norms = [bf16_words(rng.uniform(0.5, 1.5, d)) for _ in range(2)] if norm else None
    if values is None:
        values, factor = rotary.frequencies(rot, 1e4)
    table = rotary.table(rt, positions=rows or seq, dim=rot, values=values, multiplier=factor)
    try:
        got = run(rt, q, k, seq=seq, rot=rot, layout=layout, table=table, packed=packed, place=place,
                  positions=positions, norms=norms, eps=eps)
    finally:
        table.close()
    at = np.tile(np.arange(seq), batch) if positions is None else np.asarray(positions).ravel()
    for i, x in enumerate((q, k)):
        if x is None:
            continue
        want, bound = ref.rotary(x, at, values, layout=layout, factor=factor, eps=eps,
                                 norm=None if norms is None else bf16_values(norms[i]))
        over = np.abs(got[i].astype(np.float64) - want) - bound
        assert over.max() <= 0, float(over.max())


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dim,rot", [(8, 8), (32, 32), (64, 32), (64, 16), (80, 40), (96, 96),
                                     (128, 128), (128, 64), (256, 64), (256, 256), (20, 10), (6, 2),
                                     (17, 16), (40, 10), (1024, 512)])
def test_heads(runtime, precision, layout, norm, dim, rot):
    check(runtime, dim + rot, 2, 13, 3, 2, dim, rot, precision, layout=layout, norm=norm)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("packed,place", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("h,kv,dim,rot", [(4, 2, 64, 64), (5, 5, 40, 20), (16, 8, 128, 128),
                                          (1, 1, 96, 48), (12, 4, 256, 128)])
def test_rows(runtime, precision, norm, packed, place, h, kv, dim, rot):
    for layout in ("half", "interleaved"):
        check(runtime, h, 2, 21, h, kv, dim, rot, precision, layout=layout, norm=norm, packed=packed,
              place=place)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("batch,seq", [(1, 1), (1, 2), (3, 1), (1, 77), (5, 130), (2, 515)])
def test_tokens(runtime, precision, batch, seq):
    check(runtime, seq, batch, seq, 4, 2, 64, 64, precision, norm=True)
    check(runtime, seq, batch, seq, 3, 0, 128, 128, precision)  # queries alone


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(4, 4), (24, 8), (36, 20), (40, 20), (80, 20), (132, 4), (252, 124)])
def test_pieces_of_two_channels(runtime, precision, layout, dim, rot):
    for norm, place in ((False, False), (True, True)):
        check(runtime, dim, 2, 19, 3, 2, dim, rot, precision, layout=layout, norm=norm, packed=True,
              place=place)


@pytest.mark.parametrize("precision", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(20, 20), (36, 4), (40, 8), (80, 80)])
def test_many_rows(runtime, precision, layout, dim, rot):
    """So many that a thread takes several heads, of which the last part of q and of k is not full."""
    for norm in (False, True):
        check(runtime, rot, 3, 1801, 26, 3, dim, rot, precision, layout=layout, norm=norm, packed=True,
              place=True)


@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_positions_of_documents(runtime, precision):
    at = batching.document_positions([[30, 50, 5], [90]], 90)
    for kv in (2, 0):
        check(runtime, 3, 2, 90, 4, kv, 64, 64, precision, positions=at, norm=True)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn"])
@pytest.mark.parametrize("precision", ["f16", "f32"])
def test_scaled_far_positions(runtime, scaling, precision):
    """Positions of a long context: the angles are those of float64."""
    values, factor = rotary.frequencies(64, 1e6, scaling=scaling, factor=8.0, trained=8192)
    at = np.random.default_rng(4).integers(0, 65536, size=50)
    at[0], at[1] = 65535, 0
    check(runtime, 5, 1, 50, 2, 1, 64, 64, precision, positions=at, values=values, factor=factor,
          rows=65536)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dim", [64, 20])
def test_positions_beyond_the_table_give_zeros(runtime, norm, dim):
    rng = np.random.default_rng(6)
    q = rng.standard_normal((4, 2, dim)).astype(np.float32)
    k = rng.standard_normal((4, 1, dim)).astype(np.float32)
    norms = [bf16_words(np.ones(dim))] * 2 if norm else None
    table = rotary.table(runtime, positions=10, dim=dim // 2)
    got = run(runtime, q, k, seq=4, rot=dim // 2, layout="half", table=table, norms=norms,
              positions=[9, 10, 2**32 - 1, 0])
    table.close()
    for y in got:
        assert not y[1:3].any() and np.isfinite(y).all() and y[0].any() and y[3].any()


def test_zero_rows_and_nan_stay_in_their_head(runtime):
    rng = np.random.default_rng(7)
    q = rng.standard_normal((3, 2, 64)).astype(np.float16)
    k = np.zeros((3, 1, 64), np.float16)
    q[1, 0, 5] = np.nan
    norms = [bf16_words(np.ones(64))] * 2
    table = rotary.table(runtime, positions=3, dim=64)
    qo, ko = run(runtime, q, k, seq=3, rot=64, layout="half", table=table, norms=norms)
    table.close()
    assert np.isnan(qo[1, 0]).all() and np.isfinite(qo[[0, 2]]).all() and np.isfinite(qo[1, 1]).all()
    assert not ko.any()


def test_table_is_float64_rounded_once(runtime):
    values, factor = rotary.frequencies(16, 1e6, scaling="yarn", factor=4.0, trained=1024)
    table = rotary.table(runtime, positions=5000, dim=16, values=values, multiplier=factor)
    got = runtime.read(table, (5000, 16))
    table.close()
    angle = np.arange(5000)[:, None] * values
    want = np.concatenate((np.cos(angle), np.sin(angle)), 1) * np.float64(np.float32(factor))
    assert np.abs(got - want).max() <= 2.0**-24 * 1.2 + 1e-12


def test_refusals(runtime):
    shape = dict(tokens=8, seq=4, heads=2, kv_heads=1, dim=32, rotary_dim=32, precision="f16")
    q, k, qo, ko = (runtime.buffer(8 * n * 32 * 2) for n in (2, 1, 2, 1))
    rows, small = runtime.buffer(8 * 4 * 32 * 2), runtime.buffer(16)
    table = rotary.table(runtime, positions=4, dim=32)

    def refused(buffers, **kw):
        with pytest.raises(InferenceError):
            with runtime.command():
                runtime._rotary(buffers, **{**shape, **kw})

    for i in range(5):
        refused([small if j == i else b for j, b in enumerate((q, k, table, qo, ko))])
    refused([q, k, table, qo, ko], seq=8)                 # more positions than the table holds
    refused([q, k, table, k, ko])                         # outputs over the other input
    refused([q, k, table, qo, qo])
    refused([q, k, table, qo, q])
    refused([q, k, table, table, ko])
    refused([q, k, table, qo, ko], packed=True)
    refused([rows, rows, table, rows, ko], packed=True)   # half in place
    refused([q, k, table, qo, ko], positions=small)
    refused([q, k, table, qo, ko], q_norm=small, k_norm=small)
    refused([q, k, table, qo, ko], precision="f32")
    with pytest.raises(InferenceError):
        rotary.table(runtime, positions=4, dim=32, values=np.full(16, np.nan))
    with pytest.raises(InferenceError):
        rotary.table(runtime, positions=2**25, dim=32)
    with runtime.command():
        runtime._rotary([rows, rows, table, rows, rows], **shape, packed=True)
