"""The float64 oracle of attention_masked, rotary and linear_f16 against closed forms and torch."""

import math

import numpy as np
import pytest
import torch

from oracle import attention as plain
from oracle import encoder as ref


def operands(seed, b, s, h, kv, d):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((b, s, n, d)) for n in (h, kv, kv)]


@pytest.mark.parametrize("bidirectional", [0, 1])
def test_plain_masks_are_the_attention_oracle(bidirectional):
    q, k, v = operands(0, 2, 9, 4, 2, 8)
    lengths = np.array([9, 4])
    got, _ = ref.attention_masked(q, k, v, lengths,
                                  mask="bidirectional" if bidirectional else "causal")
    want = plain.attention(q, k, v, lengths, bidirectional=bool(bidirectional))
    np.testing.assert_allclose(got, want, atol=1e-13)


def test_masks_bias_and_cap_match_torch():
    b, s, h, d = 2, 11, 3, 8
    q, k, v = operands(1, b, s, h, h, d)
    lengths, prefix = np.array([11, 7]), np.array([4, 9])
    spans = np.zeros((b, s, 2), int)
    spans[:, :5], spans[:, 5:9] = (0, 5), (5, 9)  # tokens 9 and 10 attend nothing
    table = np.random.default_rng(2).standard_normal((h, 7))
    got, _ = ref.attention_masked(q, k, v, lengths, mask="prefix", window=4, cap=2.0,
                                  prefix=prefix, spans=spans, table=table)
    i, j = torch.arange(s)[:, None], torch.arange(s)[None, :]
    for n in range(b):
        doc = torch.tensor([0] * 5 + [1] * 4 + [2, 3])
        seen = ((j <= i) | (j < int(prefix[n]))) & (j < int(lengths[n])) & ((i - j).abs() < 4)
        seen = seen & (doc[:, None] == doc[None, :]) & (j < 9)
        x = torch.einsum("ihd,jhd->hij", torch.tensor(q[n]), torch.tensor(k[n])) / math.sqrt(d)
        x = 2.0 * torch.tanh(x / 2.0) + torch.tensor(table)[:, (j - i).clamp(-3, 3) + 3]
        p = torch.softmax(x.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        want = torch.einsum("hij,jhd->ihd", p, torch.tensor(v[n]))
        np.testing.assert_allclose(got[n], want.numpy(), atol=1e-13)
    assert not got[:, 9:].any()


def test_slopes_are_a_table_of_distances():
    q, k, v = operands(3, 1, 10, 2, 1, 8)
    slopes = np.array([0.5, 0.25])
    table = -slopes[:, None] * np.abs(np.arange(-9, 10))
    kw = dict(mask="bidirectional")
    a, _ = ref.attention_masked(q, k, v, np.array([10]), slopes=slopes, **kw)
    c, _ = ref.attention_masked(q, k, v, np.array([10]), table=table, **kw)
    np.testing.assert_allclose(a, c, atol=1e-14)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_depends_on_distance_alone(layout):
    """Turned by p and p + n, the product of two vectors depends on n alone, and norms are kept."""
    rng = np.random.default_rng(4)
    freq = 1e4 ** (-np.arange(4) / 4.0)
    x = np.repeat(rng.standard_normal((1, 2, 12)), 4, axis=0)
    y, _ = ref.rotary(x, np.array([0, 7, 100, 107]), freq, layout=layout)
    np.testing.assert_allclose((y[0, 0] * y[1, 1]).sum(), (y[2, 0] * y[3, 1]).sum(), atol=1e-12)
    np.testing.assert_allclose((y * y).sum(-1), (x * x).sum(-1), atol=1e-12)
    np.testing.assert_array_equal(y[..., 8:], x[..., 8:])


def test_linear_matches_torch():
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((3, 5)), rng.standard_normal((4, 5))
    bias, res = rng.standard_normal(4), rng.standard_normal((3, 4))
    y = torch.tensor(x) @ torch.tensor(w).T + torch.tensor(bias)
    for name, f in dict(none=lambda t: t, relu=torch.relu, gelu=torch.nn.functional.gelu,
                        gelu_tanh=lambda t: torch.nn.functional.gelu(t, approximate="tanh"),
                        silu=torch.nn.functional.silu).items():
        got, _ = ref.linear(x, w, bias=bias, residual=res, activation=name)
        np.testing.assert_allclose(got, (f(y) + torch.tensor(res)).numpy(), atol=1e-13)
