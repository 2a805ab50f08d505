"""The operators of an encoder layer on fp16 (or fp32) activations and packed batches, as cases that
can be timed and compared: attention with score functions and masks, the rotation of queries and keys
with their norm, and the projection with its epilogue.

Kinds of cases:
  attention   softmax(scale q k^T, capped by a tanh, plus a bias that depends on the distance) v over
              the keys that a causal, bidirectional or prefix mask, a window and the documents of a
              packed row leave
  rotary      per-head RMSNorm of q and k and the rotation of their first channels by position
  linear      act(x W^T + bias) + residual

With `own` false a pass runs elementary torch operations in fp32, rounded once at the end; with
`own` true it makes the runtime's calls on device buffers.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

EPS, THETA = 1e-6, 1e6


def listed():
    return [
        # one search query behind an instruction that every token may read: launches and latency
        dict(name="attention_prefix_1x24", kind="attention", batch=1, seq=24, heads=16, kv_heads=8,
             dim=128, precision="f16", mask="prefix", window=0, cap=0.0, bias="none", radius=0,
             documents=False, packed=False, lengths="full", shape_seed=0),
        # a long row packed with whole documents of all lengths, read from the projection's rows
        dict(name="attention_documents_1x8192", kind="attention", batch=1, seq=8192, heads=12,
             kv_heads=12, dim=64, precision="f16", mask="bidirectional", window=0, cap=0.0,
             bias="none", radius=0, documents=True, packed=True, lengths="full", shape_seed=1),
        # long passages through a layer with capped scores and a sliding window
        dict(name="attention_capped_2x4096", kind="attention", batch=2, seq=4096, heads=16,
             kv_heads=8, dim=128, precision="f16", mask="causal", window=1024, cap=50.0,
             bias="none", radius=0, documents=False, packed=False, lengths="full", shape_seed=2),
        # an fp32 encoder whose only positions are slopes, a ragged batch
        dict(name="attention_slopes_f32_8x512", kind="attention", batch=8, seq=512, heads=12,
             kv_heads=12, dim=64, precision="f32", mask="bidirectional", window=0, cap=0.0,
             bias="slopes", radius=0, documents=False, packed=False, lengths="uniform",
             shape_seed=3),
        # relative positions from a table, a few passages of odd width
        dict(name="attention_table_3x181", kind="attention", batch=3, seq=181, heads=12,
             kv_heads=12, dim=32, precision="f16", mask="bidirectional", window=0, cap=0.0,
             bias="table", radius=128, documents=False, packed=False, lengths="uniform",
             shape_seed=4),
        # a decoder layer's q and k norms and rotation, a full batch, inside the projection's rows
        dict(name="rotary_norm_32x512", kind="rotary", batch=32, seq=512, heads=16, kv_heads=8,
             dim=128, rotary_dim=128, layout="half", norm=True, precision="f16", packed=True,
             positions="row", scaling="none", factor=1.0, shape_seed=0),
        # the same for one search query
        dict(name="rotary_norm_1x24", kind="rotary", batch=1, seq=24, heads=16, kv_heads=8,
             dim=128, rotary_dim=128, layout="half", norm=True, precision="f16", packed=False,
             positions="row", scaling="none", factor=1.0, shape_seed=0),
        # neighbouring channels of half a head, fp32, a few passages of odd width
        dict(name="rotary_pairs_f32_3x181", kind="rotary", batch=3, seq=181, heads=12, kv_heads=12,
             dim=64, rotary_dim=32, layout="interleaved", norm=False, precision="f32",
             packed=False, positions="row", scaling="none", factor=1.0, shape_seed=0),
        # a long row of packed documents, positions from each document's start, frequencies scaled
        # for four times the trained length
        dict(name="rotary_scaled_1x16384", kind="rotary", batch=1, seq=16384, heads=16, kv_heads=8,
             dim=128, rotary_dim=128, layout="half", norm=False, precision="f16", packed=False,
             positions="documents", scaling="yarn", factor=4.0, shape_seed=5),
        # the first product of an encoder's feed-forward over a full batch
        dict(name="linear_gelu_16384x4096x1024", kind="linear", rows=16384, cols=4096, k=1024,
             activation="gelu", bias=True, residual=False, out="f16"),
        # the second one, added to the layer's input
        dict(name="linear_residual_4096x1024x4096", kind="linear", rows=4096, cols=1024, k=4096,
             activation="none", bias=True, residual=True, out="f16"),
        # one search query: the weights are what is read
        dict(name="linear_silu_24x4096x1024", kind="linear", rows=24, cols=4096, k=1024,
             activation="silu", bias=True, residual=False, out="f16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "rotary", "linear"))
    if kind == "linear":
        while True:
            rows, cols, k = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
            if rng.random() < 0.6:  # most widths are multiples of 32, some are not even
                cols, k = (cols + 31) // 32 * 32, (k + 31) // 32 * 32
            if rows * cols * k <= 16384 * 4096 * 1024:
                break
        return dict(kind=kind, rows=rows, cols=cols, k=k,
                    activation=rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                    out=rng.choice(("f16", "f16", "f32")))
    dim = rng.choice((32, 40, 64, 64, 80, 96, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 3))
    if kind == "rotary":
        while True:
            seq, batch = _log_int(rng, 1, 16384), _log_int(rng, 1, 32)
            if batch * seq * heads * dim * 2 <= 16384 * 24 * 128:
                break
        return dict(kind=kind, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary_dim=rng.choice((dim, dim, dim // 2, dim // 4 // 2 * 2)),
                    layout=rng.choice(("half", "interleaved")), norm=rng.random() < 0.5,
                    precision=rng.choice(("f16", "f32")), packed=rng.random() < 0.5,
                    positions=rng.choice(("row", "documents")),
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                    factor=rng.choice((2.0, 4.0, 8.0)), shape_seed=rng.randrange(1 << 20))
    precision = rng.choice(("f16", "f16", "f32"))
    while True:
        seq, batch = _log_int(rng, 1, 8192 if precision == "f16" else 2048), _log_int(rng, 1, 32)
        if (batch * seq * seq * heads * dim <= 8192 * 8192 * 12 * 64 // 2
                and batch * seq <= 16384):
            break
    bias = rng.choice(("none", "none", "slopes", "table"))
    return dict(kind=kind, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                precision=precision, mask=rng.choice(("causal", "bidirectional", "prefix")),
                window=rng.choice((0, 0, _log_int(rng, 1, 2048))),
                cap=rng.choice((0.0, 0.0, 30.0, 50.0)), bias=bias,
                radius=_log_int(rng, 1, 1024) if bias == "table" else 0,
                documents=rng.random() < 0.4, packed=rng.random() < 0.5,
                lengths=rng.choice(("full", "uniform")), shape_seed=rng.randrange(1 << 20))


# ---- shapes of a batch: valid tokens, documents of a packed row, prefixes ----------------------


def _lengths(case):
    """Valid tokens of each row; one row has them all."""
    rng, seq = random.Random(case["shape_seed"]), case["seq"]
    got = [seq if case["lengths"] == "full" else rng.randint(1, seq)
           for _ in range(case["batch"])]
    got[rng.randrange(len(got))] = seq
    return got


def _document_bounds(case):
    """For each row the bounds of its documents: most short, a few long."""
    rng, seq = random.Random(case["shape_seed"] + 1), case["seq"]
    rows = []
    for _ in range(case["batch"]):
        at, bounds = 0, []
        while at < seq:
            end = min(seq, at + _log_int(rng, min(8, seq), min(2048, seq)))
            bounds.append((at, end))
            at = end
        rows.append(bounds)
    return rows


def _spans(case):
    """[batch, seq, 2]: the first key of each token's document and the one behind its last."""
    spans = np.zeros((case["batch"], case["seq"], 2), np.int32)
    for b, bounds in enumerate(_document_bounds(case)):
        for start, end in bounds:
            spans[b, start:end] = (start, end)
    return spans


def _positions(case):
    """[batch, seq]: a token's place in its row, or in its document."""
    pos = np.tile(np.arange(case["seq"], dtype=np.int32), (case["batch"], 1))
    if case["positions"] == "documents":
        for b, bounds in enumerate(_document_bounds(case)):
            for start, end in bounds:
                pos[b, start:end] -= start
    return pos


def _prefixes(case):
    rng = random.Random(case["shape_seed"] + 2)
    return [rng.randint(0, max(1, case["seq"] // 2)) for _ in range(case["batch"])]


def _intervals(case):
    """The half-open range of keys each token attends, [batch, seq] twice."""
    b, s, w = case["batch"], case["seq"], case["window"]
    i = np.arange(s)[None, :]
    lo = np.zeros((b, s), np.int64)
    hi = np.broadcast_to(np.array(_lengths(case))[:, None], (b, s)).astype(np.int64)
    if case["mask"] == "causal":
        hi = np.minimum(hi, i + 1)
    elif case["mask"] == "prefix":
        hi = np.minimum(hi, np.maximum(i + 1, np.array(_prefixes(case))[:, None]))
    if w:
        lo, hi = np.maximum(lo, i - w + 1), np.minimum(hi, i + w)
    if case["documents"]:
        spans = _spans(case)
        lo, hi = np.maximum(lo, spans[..., 0]), np.minimum(hi, spans[..., 1])
    return lo, hi


# ---- inputs, drawn by torch from the seed alone ------------------------------------------------


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _dtype(name):
    return {"f16": torch.float16, "f32": torch.float32}[name]


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["cols"], case["k"]
        t = {"x": _normal(g, m, k).half(), "w": _normal(g, n, k, std=k**-0.5).half()}
        if case["bias"]:
            t["bias"] = _normal(g, n, std=0.5)
        if case["residual"]:
            t["residual"] = _normal(g, m, n).half()
        return t
    b, s, h, kv, d = (case[x] for x in ("batch", "seq", "heads", "kv_heads", "dim"))
    dtype = _dtype(case["precision"])
    t = {}
    if case["packed"]:  # rows of the q, k and v heads, as one projection leaves them
        t["qkv"] = _normal(g, b, s, h + 2 * kv, d).to(dtype)
    else:
        t["q"], t["k"] = _normal(g, b, s, h, d).to(dtype), _normal(g, b, s, kv, d).to(dtype)
        if case["kind"] == "attention":
            t["v"] = _normal(g, b, s, kv, d).to(dtype)
    if case["kind"] == "rotary":
        if case["norm"]:
            for name in ("q_norm", "k_norm"):
                t[name] = (torch.rand(d, generator=g, device="cuda") + 0.5).bfloat16()
        if case["positions"] != "row":
            t["positions"] = torch.tensor(_positions(case), device="cuda")
        return t
    t["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if case["documents"]:
        t["spans"] = torch.tensor(_spans(case), device="cuda")
    if case["mask"] == "prefix":
        t["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
    if case["bias"] == "slopes":  # a geometric series over the heads, as such models have
        t["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda") / h)
    elif case["bias"] == "table":
        t["table"] = _normal(g, h, 2 * case["radius"] + 1)
    return t


def _split(state):
    """q, k and v of a state, whichever rows hold them."""
    t, case = state["t"], state["case"]
    if case["packed"]:
        return torch.split(t["qkv"], (case["heads"], case["kv_heads"], case["kv_heads"]), dim=2)
    return t["q"], t["k"], t.get("v")


# ---- the framework's side: device buffers, and torch tensors over them -------------------------

_runtime = None


def _rt():
    """The one runtime a process keeps."""
    global _runtime
    if _runtime is None:
        from tessery_amd import HipRuntime

        _runtime = HipRuntime()
    return _runtime


class _Memory:
    """A runtime buffer's device memory for torch: what the buffer's handle points at begins with
    the device address. A tensor over it holds this object, and so the buffer."""

    def __init__(self, buffer):
        self.buffer = buffer
        address = ctypes.c_void_p.from_address(buffer.pointer).value
        self.__cuda_array_interface__ = {"shape": (buffer.size,), "typestr": "|u1",
                                         "data": (address, False), "version": 2}


def _view(buffer, shape, dtype):
    return torch.as_tensor(_Memory(buffer), device="cuda").view(dtype).view(shape)


def _upload(tensor):
    buffer = _rt().buffer(tensor.numel() * tensor.element_size())
    _view(buffer, tensor.shape, tensor.dtype).copy_(tensor)
    return buffer


def _prepare_own(state):
    """Buffers of the inputs and outputs, and the rotation's table, which a program keeps."""
    case, t = state["case"], state["t"]
    state["bufs"] = bufs = {name: _upload(x) for name, x in t.items()}
    del state["t"]
    if case["kind"] == "linear":
        out = _dtype(case["out"])
        shapes = {"out": ((case["rows"], case["cols"]), out)}
    else:
        b, s, d, dtype = case["batch"], case["seq"], case["dim"], _dtype(case["precision"])
        shapes = {"out": ((b, s, case["heads"], d), dtype)}
        if case["kind"] == "rotary":
            shapes = {"q_out": ((b, s, case["heads"], d), dtype),
                      "k_out": ((b, s, case["kv_heads"], d), dtype)}
            from tessery_amd import rotary

            bufs["rotations"] = rotary.table(
                _rt(), positions=case["seq"], dim=case["rotary_dim"], theta=THETA,
                scaling=case["scaling"], factor=case["factor"], trained=_trained(case))
    state["outs"] = {}
    for name, (shape, dtype) in shapes.items():
        bufs[name] = _rt().buffer(math.prod(shape) * dtype.itemsize)
        state["outs"][name] = _view(bufs[name], shape, dtype)
    torch.cuda.synchronize()
    return state


def _run_own(state):
    rt, case, bufs = _rt(), state["case"], state["bufs"]
    get = bufs.get
    with rt.command():
        if case["kind"] == "linear":
            rt._linear_f16([bufs["x"], bufs["w"], bufs["out"]], rows=case["rows"],
                           cols=case["cols"], k=case["k"], bias=get("bias"),
                           residual=get("residual"), activation=case["activation"],
                           out_dtype=case["out"])
        else:
            packed, tokens = case["packed"], case["batch"] * case["seq"]
            qkv = [bufs["qkv"]] * 3 if packed else [bufs["q"], bufs["k"], get("v")]
            shape = dict(tokens=tokens, seq=case["seq"], heads=case["heads"],
                         kv_heads=case["kv_heads"], dim=case["dim"],
                         precision=case["precision"], packed=packed)
            if case["kind"] == "attention":
                rt._attention_masked([*qkv, bufs["lengths"], bufs["out"]], **shape,
                                     mask=case["mask"], window=case["window"], cap=case["cap"],
                                     prefix=get("prefix"), spans=get("spans"),
                                     slopes=get("slopes"), table=get("table"),
                                     radius=case["radius"])
            else:
                rt._rotary([*qkv[:2], bufs["rotations"], bufs["q_out"], bufs["k_out"]], **shape,
                           rotary_dim=case["rotary_dim"], layout=case["layout"],
                           positions=get("positions"), q_norm=get("q_norm"),
                           k_norm=get("k_norm"), eps=EPS)
    return state["outs"]


# ---- the plain form: elementary torch operations in fp32 ---------------------------------------


def _trained(case):
    """The length the unscaled frequencies were trained for."""
    return max(1, int(case["seq"] / case["factor"]))


def _frequencies(case):
    """Radians a position of each rotated pair, and the factor on the rotated channels."""
    r, f = case["rotary_dim"], case["factor"]
    c = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    kind, base = case["scaling"], THETA
    if kind == "ntk" and r > 2:
        base = THETA * f ** (r / (r - 2))
    freq = base ** (-2.0 * c / r)
    if kind == "linear":
        return freq / f, 1.0
    if kind == "yarn":  # turns within the trained length: kept from 32 on, divided up to 1
        turns = _trained(case) * freq / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        return freq * keep + freq / f * (1.0 - keep), 0.1 * math.log(f) + 1.0
    return freq, 1.0


def _prepare_plain(state):
    case, t = state["case"], state["t"]
    if case["kind"] == "rotary":
        freq, factor = _frequencies(case)
        angle = torch.arange(case["seq"], dtype=torch.float64, device="cuda")[:, None] * freq
        t["cos"] = (angle.cos() * factor).float()
        t["sin"] = (angle.sin() * factor).float()
    elif case["kind"] == "attention":
        lo, hi = _intervals(case)
        t["lo"], t["hi"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lo, hi))
    torch.cuda.synchronize()
    return state


def _erf_gelu(y):
    return 0.5 * y * (1.0 + torch.erf(y * 0.5**0.5))


def _tanh_gelu(y):
    return 0.5 * y * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))


ACTIVATIONS = {"none": lambda y: y, "relu": lambda y: torch.where(y > 0, y, torch.zeros_like(y)),
               "gelu": _erf_gelu, "gelu_tanh": _tanh_gelu, "silu": lambda y: y / (1.0 + torch.exp(-y))}


def _linear_plain(state):
    case, t = state["case"], state["t"]
    y = t["x"].float() @ t["w"].float().T
    if case["bias"]:
        y = y + t["bias"]
    y = ACTIVATIONS[case["activation"]](y)
    if case["residual"]:
        y = y + t["residual"].float()
    return {"out": y.to(_dtype(case["out"]))}


def _rotary_plain(state):
    case, t = state["case"], state["t"]
    q, k, _ = _split(state)
    r, outs = case["rotary_dim"], {}
    if case["positions"] == "row":
        cos, sin = t["cos"][None, :, None], t["sin"][None, :, None]
    else:
        at = t["positions"].long()
        cos, sin = t["cos"][at][:, :, None], t["sin"][at][:, :, None]
    for name, x in (("q", q), ("k", k)):
        y = x.float()
        if case["norm"]:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * t[name + "_norm"].float()
        turned, rest = y[..., :r], y[..., r:]
        if case["layout"] == "half":
            a, b = turned[..., :r // 2], turned[..., r // 2:]
            turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        outs[name + "_out"] = torch.cat((turned, rest), -1).to(x.dtype)
    return outs


def _attention_plain(state):
    case, t = state["case"], state["t"]
    q, k, v = _split(state)
    group, s = case["heads"] // case["kv_heads"], case["seq"]
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    j = torch.arange(s, device="cuda", dtype=torch.int32)
    for b in range(case["batch"]):
        ks = k[b].float().repeat_interleave(group, 1).permute(1, 2, 0).contiguous()
        vs = v[b].float().repeat_interleave(group, 1).permute(1, 0, 2).contiguous()
        for first in range(0, s, 2048):
            rows = slice(first, min(s, first + 2048))
            scores = (q[b, rows].float().permute(1, 0, 2).contiguous() @ ks) * case["dim"] ** -0.5
            if case["cap"]:
                scores = torch.tanh(scores / case["cap"]) * case["cap"]
            away = j[None, :] - j[rows, None]
            if case["bias"] == "slopes":
                scores = scores - t["slopes"][:, None, None] * away.abs()
            elif case["bias"] == "table":
                at = away.clamp(-case["radius"], case["radius"]) + case["radius"]
                scores = scores + t["table"][:, at.long()]
            seen = (j[None, :] >= t["lo"][b, rows, None]) & (j[None, :] < t["hi"][b, rows, None])
            scores = torch.where(seen, scores, float("-inf"))
            top = scores.amax(-1, keepdim=True)
            e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
            total = e.sum(-1, keepdim=True)
            y = (e @ vs) / torch.where(total == 0, 1.0, total)
            out[b, rows] = y.permute(1, 0, 2).to(out.dtype)
    return {"out": out}


PLAIN = {"attention": _attention_plain, "rotary": _rotary_plain, "linear": _linear_plain}


def prepare(case, seed):
    state = {"case": case, "t": _inputs(case, seed)}
    return _prepare_own(state) if own else _prepare_plain(state)


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["cols"], case["k"]
        size = _dtype(case["out"]).itemsize
        return {"bytes": 2 * (m * k + n * k) + m * n * size + 4 * n * case["bias"]
                + 2 * m * n * case["residual"], "flops": 2 * m * n * k}
    size = _dtype(case["precision"]).itemsize
    b, s, h, kv, d = (case[x] for x in ("batch", "seq", "heads", "kv_heads", "dim"))
    if case["kind"] == "rotary":
        values = b * s * (h + kv) * d
        return {"bytes": 2 * values * size + (4 * b * s if case["positions"] != "row" else 0)
                + 4 * s * case["rotary_dim"], "flops": values * (6 if case["norm"] else 3)}
    lo, hi = _intervals(case)
    pairs = int(np.maximum(hi - lo, 0).sum())
    return {"bytes": size * d * (2 * b * s * h + 2 * sum(_lengths(case)) * kv)
            + (8 * b * s if case["documents"] else 0), "flops": 4 * d * h * pairs}


# ---- the same in 64 bits -----------------------------------------------------------------------


def _exact_linear(case, t):
    out = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
    w = t["w"].double().t().contiguous()
    for first in range(0, case["rows"], 4096):
        rows = slice(first, first + 4096)
        y = torch.mm(t["x"][rows].double(), w)
        if "bias" in t:
            y += t["bias"].double()
        name = case["activation"]
        if name == "relu":
            y = y.clamp(min=0.0)
        elif name == "gelu":  # y times the normal distribution's integral up to y
            y = y * torch.special.ndtr(y)
        elif name == "gelu_tanh":
            u = math.sqrt(2.0 / math.pi) * y * (1.0 + 0.044715 * y**2)
            y = y * torch.sigmoid(2.0 * u)
        elif name == "silu":
            y = y * torch.sigmoid(y)
        if "residual" in t:
            y = y + t["residual"][rows].double()
        out[rows] = y
    return {"out": out}


def _exact_rotary(case, t):
    """Each pair as a complex number, multiplied by factor * exp(i pos freq)."""
    h, kv, r = case["heads"], case["kv_heads"], case["rotary_dim"]
    c = torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r
    f, factor = case["factor"], 1.0
    base = math.log(THETA)
    if case["scaling"] == "ntk" and r > 2:
        base += r / (r - 2) * math.log(f)
    freq = torch.exp(-base * c)
    if case["scaling"] == "linear":
        freq = freq / f
    elif case["scaling"] == "yarn":
        share = torch.clamp((_trained(case) / (2 * math.pi / freq) - 1) / (32 - 1), min=0, max=1)
        freq = (1 - share) * (freq / f) + share * freq
        factor = 1 + math.log(f) / 10
    pos = torch.tensor(_positions(case), device="cuda").double()
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda").expand(
        *pos.shape, 1, r // 2).contiguous(), (pos[..., None] * freq)[:, :, None])
    outs = {}
    for name, at, heads in (("q", 0, h), ("k", h, kv)):
        x = (t["qkv"][:, :, at:at + heads] if case["packed"] else t[name]).double()
        if case["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            x = x * t[name + "_norm"].double()
        y = x.clone()
        if case["layout"] == "half":
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        outs[name + "_out"] = y
    return outs


def _exact_attention(case, t):
    """Row block by row block of each head, only over the keys that some row of it attends."""
    b, s, h, kv, d = (case[x] for x in ("batch", "seq", "heads", "kv_heads", "dim"))
    lo, hi = _intervals(case)
    out = torch.zeros(b, s, h, d, dtype=torch.float64, device="cuda")
    block = 1024
    for row in range(b):
        if case["packed"]:
            parts = t["qkv"][row].double().split((h, kv, kv), dim=1)
        else:
            parts = (t["q"][row].double(), t["k"][row].double(), t["v"][row].double())
        q, k, v = (x.transpose(0, 1).contiguous() for x in parts)
        for first in range(0, s, block):
            last = min(s, first + block)
            some = hi[row, first:last] > lo[row, first:last]
            if not some.any():
                continue
            k0 = int(lo[row, first:last][some].min())
            k1 = int(hi[row, first:last][some].max())
            i = torch.arange(first, last, device="cuda")[:, None]
            j = torch.arange(k0, k1, device="cuda")[None, :]
            low = torch.tensor(lo[row, first:last], device="cuda")[:, None]
            high = torch.tensor(hi[row, first:last], device="cuda")[:, None]
            hidden = (j < low) | (j >= high)
            empty = (high <= low)
            for g in range(kv):
                heads = slice(g * (h // kv), (g + 1) * (h // kv))
                x = torch.einsum("hid,jd->hij", q[heads, first:last], k[g, k0:k1]) / math.sqrt(d)
                if case["cap"]:
                    x = case["cap"] * (x / case["cap"]).tanh()
                if case["bias"] == "slopes":
                    x = x - t["slopes"].double()[heads, None, None] * (i - j).abs()
                elif case["bias"] == "table":
                    edge = case["radius"]
                    away = torch.minimum(torch.maximum(j - i, torch.full_like(j, -edge)),
                                         torch.full_like(j, edge)) + edge
                    x = x + t["table"].double()[heads][:, away]
                x = x.masked_fill(hidden, -math.inf).masked_fill(empty, 0.0)
                p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)).masked_fill(empty, 0.0)
                out[row, first:last, heads] = torch.einsum("hij,jd->ihd", p, v[g, k0:k1])
    return {"out": out}


def exact(case, seed):
    t = _inputs(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary,
            "linear": _exact_linear}[case["kind"]](case, t)
