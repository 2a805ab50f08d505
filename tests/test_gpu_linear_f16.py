"""Route linear_f16 against the float64 oracle, within the oracle's bound: shapes around every tile,
odd widths, activations, bias, residual (in place too), both output types, rows left alone, values that
are not finite, and the calls it refuses."""

import numpy as np
import pytest

from oracle import encoder as ref
from tessery_amd.errors import InferenceError

pytestmark = pytest.mark.gpu


def operands(seed, m, n, k):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((m, k)).astype(np.float16),
            (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16),
            (0.5 * rng.standard_normal(n)).astype(np.float32),
            rng.standard_normal((m, n)).astype(np.float16))


def run(rt, x, w, *, bias=None, residual=None, place=False, out_dtype="f16", **kw):
    (m, k), n = x.shape, w.shape[0]
    dtype = np.float16 if out_dtype == "f16" else np.float32
    held = [rt.upload(a) for a in (x, w)]
    extra = {name: rt.upload(a) for name, a in (("bias", bias), ("residual", residual))
             if a is not None}
    if place:
        out, rows = extra["residual"], m
    else:
        out, rows = rt.upload(np.full((m + 1, n), np.nan, dtype)), m + 1
    try:
        with rt.command():
            rt._linear_f16([*held, out], rows=m, cols=n, k=k, out_dtype=out_dtype, **extra, **kw)
        got = rt.read(out, (rows, n), dtype)
    finally:
        for b in {*held, *extra.values(), out}:
            b.close()
    assert place or np.isnan(got[m:]).all()
    return got[:m]


def check(rt, seed, m, n, k, *, bias=False, residual=False, out_dtype="f16", activation="none",
          place=False):
    x, w, b, r = operands(seed, m, n, k)
    kw = dict(bias=b if bias else None, residual=r if residual else None, activation=activation)
    want, bound = ref.linear(x, w, half=out_dtype == "f16", **kw)
    got = run(rt, x, w, out_dtype=out_dtype, place=place, **kw).astype(np.float64)
    over = np.abs(got - want) - bound
    assert over.max() <= 0, (float(over.max()), float(np.abs(got - want).max()))


SHAPES = [(1, 1, 1), (1, 16, 8), (2, 7, 33), (5, 64, 64), (16, 32, 100), (17, 48, 72), (24, 256, 128),
          (31, 100, 40), (32, 384, 384), (33, 65, 256), (63, 130, 64), (64, 64, 1024), (65, 96, 520),
          (77, 1536, 384), (100, 72, 72), (127, 129, 31), (128, 128, 64), (129, 257, 192),
          (200, 384, 1536), (255, 256, 96), (256, 256, 256), (300, 520, 264), (513, 300, 80),
          (1000, 64, 2048), (520, 768, 1000), (600, 1032, 40)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(runtime, m, n, k):
    check(runtime, m + n + k, m, n, k)
    check(runtime, m + n + k, m, n, k, bias=True, residual=True, activation="gelu", out_dtype="f32")


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("out_dtype", ["f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (70, 136, 96), (300, 256, 128)])
def test_epilogues(runtime, activation, bias, residual, out_dtype, m, n, k):
    check(runtime, 3, m, n, k, bias=bias, residual=residual, out_dtype=out_dtype,
          activation=activation)


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (24, 512, 1024), (130, 200, 88), (512, 512, 512),
                                   (64, 64, 4096)])
def test_residual_in_place(runtime, m, n, k):
    check(runtime, 4, m, n, k, bias=True, residual=True, place=True)


@pytest.mark.parametrize("m,n,k", [(1, 8192, 64), (1, 64, 8192), (4, 1024, 4096), (2048, 1024, 256),
                                   (1536, 2048, 64)])
def test_long_sides(runtime, m, n, k):
    check(runtime, 5, m, n, k, bias=True)


@pytest.mark.parametrize("m,n,k", [(33, 65, 4096), (70, 96, 8000), (363, 68, 6479), (100, 130, 2561),
                                   (64, 64, 65536), (200, 37, 1000)])
@pytest.mark.parametrize("out_dtype", ["f16", "f32"])
def test_long_sums_of_few_outputs(runtime, m, n, k, out_dtype):
    """K shared out between workgroups, the parts added in order."""
    for place in (False, True) if out_dtype == "f16" else (False,):
        check(runtime, 9, m, n, k, bias=True, residual=True, activation="silu", out_dtype=out_dtype,
              place=place)


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 72), (2000, 2041, 128), (2048, 4096, 64),
                                   (2010, 4090, 200), (4096, 4096, 64), (4000, 4104, 200),
                                   (4001, 4099, 72)])
def test_many_outputs(runtime, m, n, k):
    """Products that fill the chip with tiles of 128 and 256."""
    check(runtime, 8, m, n, k, bias=True, residual=True, activation="relu")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_rows_and_columns_that_are_not_finite(runtime, m):
    """A row of x or of W that holds a NaN or an infinity reaches its own outputs alone."""
    x, w, b, _ = operands(6, m, 200, 160)
    want, bound = ref.linear(x, w, bias=b)
    x2, w2 = x.copy(), w.copy()
    x2[m // 2, 7] = np.nan
    w2[13, 159] = np.inf
    got = run(runtime, x2, w2, bias=b).astype(np.float64)
    keep = np.ones((m, 200), bool)
    keep[m // 2] = False
    keep[:, 13] = False
    assert np.all(np.abs(got - want)[keep] <= bound[keep])
    assert np.isnan(got[m // 2]).all() and not np.isfinite(got[:, 13]).any()


def test_outputs_that_leave_fp16(runtime):
    x = np.full((2, 64), 100.0, np.float16)
    w = np.full((3, 64), 100.0, np.float16)
    assert np.isposinf(run(runtime, x, w)).all()
    np.testing.assert_array_equal(run(runtime, x, w, out_dtype="f32"), np.full((2, 3), 640000.0))


def test_same_bits_every_time(runtime):
    for m, n, k in ((24, 512, 2048), (300, 300, 300), (512, 512, 1024)):
        x, w, b, r = operands(7, m, n, k)
        first = run(runtime, x, w, bias=b, residual=r)
        for _ in range(3):
            np.testing.assert_array_equal(run(runtime, x, w, bias=b, residual=r), first)


def test_refusals(runtime):
    x, w, out, small = (runtime.buffer(n) for n in (8 * 64 * 2, 16 * 64 * 2, 8 * 16 * 4, 16))
    shape = dict(rows=8, cols=16, k=64)

    def refused(buffers, **kw):
        with pytest.raises(InferenceError):
            with runtime.command():
                runtime._linear_f16(buffers, **{**shape, **kw})

    refused([small, w, out])
    refused([x, small, out])
    refused([x, w, small])
    refused([x, w, out], bias=small)
    refused([x, w, out], residual=small)
    refused([x, w, x])
    refused([x, w, w])
    refused([x, w, out], bias=out)
    refused([x, w, out], residual=out, out_dtype="f32")  # of another type than the output
    refused([x, w, out], rows=9)
    refused([x, w, out], k=70000)
    with runtime.command():
        runtime._linear_f16([x, w, out], **shape, residual=out)
