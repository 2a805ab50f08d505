"""One encoder layer on fp16 activations of packed batches, as a program queues it: the q, k and v
projection, norms and rotation inside its rows, attention over the documents, the output projection added
to the layer's input, and the feed-forward. Each step's output is held to the float64 oracle on that
step's own inputs; one command, separate commands and plan replays (a HIP graph, between other work)
give the same bits."""

import numpy as np
import pytest

from oracle import encoder as ref
from tessery_amd import batching, rotary
from tessery_amd.workloads import bf16_values, bf16_words

pytestmark = pytest.mark.gpu

B, S, H, KV, D, WIDE = 2, 96, 6, 2, 64, 640
HIDDEN, ROWS = H * D, (H + 2 * KV) * D
DOCUMENTS = [[40, 17, 30], [96]]
TOKENS = B * S


class Layer:
    def __init__(self, rt, seed):
        rng = np.random.default_rng(seed)

        def weight(n, k):
            return (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16)

        self.rt = rt
        self.host = dict(
            x=rng.standard_normal((TOKENS, HIDDEN)).astype(np.float16),
            w_qkv=weight(ROWS, HIDDEN), w_o=weight(HIDDEN, HIDDEN), w_1=weight(WIDE, HIDDEN),
            w_2=weight(HIDDEN, WIDE),
            b_qkv=(0.1 * rng.standard_normal(ROWS)).astype(np.float32),
            b_1=(0.1 * rng.standard_normal(WIDE)).astype(np.float32),
            q_norm=bf16_words(rng.uniform(0.5, 1.5, D)),
            k_norm=bf16_words(rng.uniform(0.5, 1.5, D)),
            lengths=np.full(B, S, np.uint32), spans=batching.document_spans(DOCUMENTS, S),
            positions=batching.document_positions(DOCUMENTS, S))
        self.buf = {n: rt.upload(a) for n, a in self.host.items()}
        self.freq, self.factor = rotary.frequencies(D, 1e4, scaling="yarn", factor=2.0, trained=48)
        self.buf["table"] = rotary.table(rt, positions=S, dim=D, values=self.freq,
                                         multiplier=self.factor)
        self.shapes = dict(qkv=(TOKENS, ROWS), turned=(TOKENS, ROWS), o=(TOKENS, HIDDEN),
                           mid=(TOKENS, HIDDEN), wide=(TOKENS, WIDE), y=(TOKENS, HIDDEN))
        for n, shape in self.shapes.items():
            self.buf[n] = rt.buffer(2 * int(np.prod(shape)))

    def steps(self):
        """The layer's calls, in order."""
        rt, b = self.rt, self.buf
        heads = dict(tokens=TOKENS, seq=S, heads=H, kv_heads=KV, dim=D, packed=True)
        return [
            lambda: rt._linear_f16([b["x"], b["w_qkv"], b["qkv"]], rows=TOKENS, cols=ROWS, k=HIDDEN,
                                   bias=b["b_qkv"]),
            lambda: rt._dispatch("copy", [b["qkv"], b["turned"]], threads=2 * TOKENS * ROWS),
            lambda: rt._rotary([b["turned"], b["turned"], b["table"], b["turned"], b["turned"]],
                               rotary_dim=D, positions=b["positions"], q_norm=b["q_norm"],
                               k_norm=b["k_norm"], **heads),
            lambda: rt._attention_masked([b["turned"]] * 3 + [b["lengths"], b["o"]],
                                         mask="bidirectional", spans=b["spans"], **heads),
            lambda: rt._linear_f16([b["o"], b["w_o"], b["mid"]], rows=TOKENS, cols=HIDDEN, k=HIDDEN,
                                   residual=b["x"]),
            lambda: rt._linear_f16([b["mid"], b["w_1"], b["wide"]], rows=TOKENS, cols=WIDE, k=HIDDEN,
                                   bias=b["b_1"], activation="gelu"),
            lambda: rt._linear_f16([b["wide"], b["w_2"], b["y"]], rows=TOKENS, cols=HIDDEN, k=WIDE,
                                   residual=b["mid"])]

    def read(self):
        return {n: self.rt.read(self.buf[n], s, np.float16) for n, s in self.shapes.items()}

    def wipe(self):
        for n, s in self.shapes.items():
            self.rt.write(self.buf[n], np.full(s, np.nan, np.float16))

    def close(self):
        for b in self.buf.values():
            b.close()


def within(got, want, bound):
    assert np.max(np.abs(got.astype(np.float64) - want) - bound) <= 0


def test_steps_match_the_oracle_and_ways_to_run_them_each_other(runtime):
    layer = Layer(runtime, 1)
    h = layer.host
    try:
        layer.wipe()
        for step in layer.steps():  # a command each
            with runtime.command():
                step()
        got = layer.read()
        within(got["qkv"], *ref.linear(h["x"], h["w_qkv"], bias=h["b_qkv"]))
        rows = got["qkv"].reshape(TOKENS, H + 2 * KV, D)
        turned = got["turned"].reshape(TOKENS, H + 2 * KV, D)
        for name, part in (("q_norm", slice(0, H)), ("k_norm", slice(H, H + KV))):
            within(turned[:, part], *ref.rotary(
                rows[:, part], h["positions"].ravel(), layer.freq, layout="half",
                factor=layer.factor, norm=bf16_values(h[name])))
        np.testing.assert_array_equal(turned[:, H + KV:], rows[:, H + KV:])
        q, k, v = np.split(turned.reshape(B, S, H + 2 * KV, D), [H, H + KV], axis=2)
        want, bound = ref.attention_masked(q, k, v, h["lengths"], mask="bidirectional",
                                           spans=h["spans"])
        within(got["o"], want.reshape(TOKENS, HIDDEN), bound.reshape(TOKENS, HIDDEN))
        within(got["mid"], *ref.linear(got["o"], h["w_o"], residual=h["x"]))
        within(got["wide"], *ref.linear(got["mid"], h["w_1"], bias=h["b_1"], activation="gelu"))
        within(got["y"], *ref.linear(got["wide"], h["w_2"], residual=got["mid"]))

        layer.wipe()
        with runtime.command():  # one command
            for step in layer.steps():
                step()
        one = layer.read()
        for n in got:
            np.testing.assert_array_equal(one[n], got[n], err_msg=n)

        with runtime.profile_kernels() as profile:
            with runtime.command():
                for step in layer.steps():
                    step()
        assert [r["kernel"] for r in profile] == ["linear_f16", "copy", "rotary", "attention_masked"] + \
            3 * ["linear_f16"]
        assert all(r["gpu_seconds"] > 0 for r in profile)

        other = Layer(runtime, 2)  # eager work between the replays, on the same scratch
        builds = runtime.diagnostics()["graph_builds"]
        try:
            for replay in range(5):
                layer.wipe()
                with runtime._workspace(), runtime.command(), \
                        runtime._execution_plan(("layer",), list(layer.buf.values())) as replayed:
                    assert replayed == (replay > 0)
                    if not replayed:
                        for step in layer.steps():
                            step()
                planned = layer.read()
                for n in got:
                    np.testing.assert_array_equal(planned[n], got[n], err_msg=f"{replay} {n}")
                with runtime.command():
                    for step in other.steps():
                        step()
        finally:
            other.close()
        assert runtime.diagnostics()["graph_builds"] == builds + 1
    finally:
        layer.close()


def test_a_plan_replayed_over_other_buffers_refuses_outputs_that_are_inputs(runtime):
    """A plan checks sizes as it is made; which buffers its slots stand for is known at a replay."""
    from tessery_amd.errors import InferenceError

    x, w, out = (runtime.buffer(32 * 32 * 2) for _ in range(3))

    def queue(bufs):
        with runtime._workspace(), runtime.command(), \
                runtime._execution_plan(("one",), bufs) as replayed:
            if not replayed:
                runtime._linear_f16(bufs, rows=32, cols=32, k=32)
            return replayed

    assert queue([x, w, out]) is False
    assert queue([x, w, out]) is True
    with pytest.raises(InferenceError):
        queue([x, w, x])


def test_split_sums_share_their_scratch_with_the_other_projections(runtime):
    """Products whose K is shared out leave their sums where dense and uint4 projections keep theirs:
    queued together, each gives what it gives alone."""
    rng = np.random.default_rng(5)
    m, n, k = 40, 72, 4096
    x = rng.standard_normal((m, k)).astype(np.float16)
    w = (rng.standard_normal((n, k)) / 64).astype(np.float16)
    a = rng.standard_normal((64, 384)).astype(np.float32)
    bt = (rng.standard_normal((384, 384)) / 20).astype(np.float32)
    bufs = [runtime.upload(t) for t in (x, w)]
    dense = [runtime.upload(t) for t in (a, bt)]
    outs = [runtime.buffer(m * n * 2), runtime.buffer(64 * 384 * 4), runtime.buffer(m * n * 2)]

    def linear(out):
        runtime._linear_f16([*bufs, out], rows=m, cols=n, k=k)

    def matmul():
        runtime._matmul_f32([*dense, outs[1]], rows=64, cols=384, k=384)

    def read():
        return (runtime.read(outs[0], (m, n), np.float16), runtime.read(outs[1], (64, 384)),
                runtime.read(outs[2], (m, n), np.float16))

    for call in (lambda: linear(outs[0]), matmul, lambda: linear(outs[2])):
        with runtime.command():
            call()
    alone = read()
    within(alone[0], *ref.linear(x, w))
    for _ in range(3):
        with runtime.command():
            linear(outs[0])
            matmul()
            linear(outs[2])
            matmul()
        for got, want in zip(read(), alone):
            np.testing.assert_array_equal(got, want)
