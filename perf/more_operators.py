"""Performance cases of the operators between an attention decoder's attention calls.

  norm    a block's output normalised, gated and added to the residual stream, and the stream normalised for the next block
  linear  tokens quantised to 8 bits and multiplied with 8-bit weights: a scale for each token and each output channel
  rotary  rotary positions of queries and keys: interleaved or half pairs, the whole head or a part of it
  rules   penalties for repeated tokens, biases and grammar masks on logits, the histories read through beams' tables

run() with own = False states the operators in elementary torch operations; with own = True it calls the framework
(pkx.BlockNorm, pkx.LinearI8, pkx.Rotary, pkx.LogitRules).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_PY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_amd", "python")
_TYPES = {"f16": torch.float16, "f32": torch.float32}
_LARGEST_NORM, _LARGEST_LINEAR, _LARGEST_ROTARY, _LARGEST_RULES = 670e6, 549e9, 235e6, 200e6    # bytes, operations, bytes, bytes


def listed():
    return [
        # one token of a greedy decode: latency
        {"name": "norm_f16_r1", "kind": "norm", "type": "f16", "x32": False, "rows": 1, "d": 1024, "post": "none", "pre": "rms",
         "gate": "none", "fn": "linear", "alpha": 1.0},
        # 16 clips of 125 frames: norms on both sides, half a residual step, a gate vector for each clip
        {"name": "norm_f16_r2000_layer", "kind": "norm", "type": "f16", "x32": True, "rows": 2000, "d": 1024, "post": "layer",
         "pre": "layer", "gate": "item", "fn": "linear", "alpha": 0.5},
        # a large batch in exact precision, odd width, a gate value for every element
        {"name": "norm_f32_r8192_gated", "kind": "norm", "type": "f32", "x32": True, "rows": 8192, "d": 4090, "post": "rms",
         "pre": "rms", "gate": "row", "fn": "sigmoid", "alpha": 1.0},
        # one token through a feed-forward's first product: latency and the weights' bytes
        {"name": "linear_f16_m1", "kind": "linear", "type": "f16", "M": 1, "N": 4096, "K": 1024, "act": "silu", "bias": True, "add": False},
        # 16 items x 4 beams through the second one, added to the residual stream
        {"name": "linear_f16_m64", "kind": "linear", "type": "f16", "M": 64, "N": 1024, "K": 4096, "act": "none", "bias": True, "add": True},
        # 16 clips of 125 frames through the first one
        {"name": "linear_f16_m2000", "kind": "linear", "type": "f16", "M": 2000, "N": 4096, "K": 1024, "act": "silu", "bias": True, "add": False},
        # a large batch of prompts in a wide model
        {"name": "linear_f16_m16384", "kind": "linear", "type": "f16", "M": 16384, "N": 4096, "K": 4096, "act": "none", "bias": False, "add": False},
        # 16 items x 8 beams, the next token
        {"name": "rotary_f16_r128", "kind": "rotary", "type": "f16", "R": 128, "n": 1, "H": 8, "Hkv": 8, "dk": 64, "rot": 64,
         "pairs": "half", "far": 448, "scaled": False, "ragged": False},
        # four long prompts late in a long context, half of each head turned, frequencies scaled, ragged lengths
        {"name": "rotary_f16_r4_long", "kind": "rotary", "type": "f16", "R": 4, "n": 8192, "H": 16, "Hkv": 4, "dk": 128, "rot": 64,
         "pairs": "interleaved", "far": 1000000, "scaled": True, "ragged": True},
        # one utterance, 4 beams over the transducer's vocabulary
        {"name": "rules_f32_r4", "kind": "rules", "type": "f32", "R": 4, "V": 1025, "len": 18, "window": 0, "table": False, "bias": "one",
         "mask": False},
        # a serving batch on a wordpiece vocabulary, each beam's grammar state names its mask
        {"name": "rules_f16_r128_grammar", "kind": "rules", "type": "f16", "R": 128, "V": 8193, "len": 448, "window": 0, "table": True,
         "bias": "none", "mask": True},
        # the widest search: 32 items x 16 beams, 32k words, long histories of which the last 1024 tokens count
        {"name": "rules_f32_r512", "kind": "rules", "type": "f32", "R": 512, "V": 32769, "len": 4096, "window": 1024, "table": True,
         "bias": "rows", "mask": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "rotary", "rules"])
    typ = rng.choice(["f16", "f16", "f32"])
    if kind == "norm":
        d = rng.choice([512, 1024, 8 * _log_int(rng, 4, 1024), _log_int(rng, 32, 8192)])
        rows = max(1, min(_log_int(rng, 1, 32768), int(_LARGEST_NORM / (20.0 * d))))
        return {"kind": kind, "type": typ, "x32": typ == "f32" or rng.random() < 0.5, "rows": rows, "d": d,
                "post": rng.choice(["none", "layer", "rms"]), "pre": rng.choice(["layer", "rms"]),
                "gate": rng.choice(["none", "item", "row"]), "fn": rng.choice(["linear", "sigmoid"]), "alpha": rng.choice([0.5, 1.0])}
    if kind == "linear":
        N, K = (rng.choice([1024, 4096, 16 * _log_int(rng, 1, 512), _log_int(rng, 17, 8192)]) for _ in range(2))
        M = max(1, min(rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 1, 16384)]), int(_LARGEST_LINEAR / (2.0 * N * K))))
        return {"kind": kind, "type": typ, "M": M, "N": N, "K": K, "act": rng.choice(["none", "silu"]), "bias": rng.random() < 0.5,
                "add": rng.random() < 0.4}
    if kind == "rotary":
        dk = rng.choice([32, 64, 64, 80, 128])
        rot = rng.choice([dk, dk, dk // 2, 2 * rng.randint(1, dk // 2)])
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 1, 2, 4])
        n = rng.choice([1, 1, _log_int(rng, 2, 8192)])
        R = max(1, min(_log_int(rng, 1, 256), int(_LARGEST_ROTARY / (8.0 * n * (H + Hkv) * dk))))
        return {"kind": kind, "type": typ, "R": R, "n": n, "H": H, "Hkv": Hkv, "dk": dk, "rot": rot,
                "pairs": rng.choice(["half", "interleaved"]), "far": _log_int(rng, n, 1000000), "scaled": rng.random() < 0.4,
                "ragged": n > 1 and rng.random() < 0.4}
    V, n = _log_int(rng, 33, 65537), _log_int(rng, 1, 8192)
    R = max(1, min(_log_int(rng, 1, 512), int(_LARGEST_RULES / (16.0 * V + 8.0 * n))))
    return {"kind": kind, "type": typ, "R": R, "V": V, "len": n, "window": rng.choice([0, 0, _log_int(rng, 1, 1024)]),
            "table": rng.random() < 0.5, "bias": rng.choice(["none", "one", "rows"]), "mask": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _spread(n, full, least):
    """Lengths from `full` down to a fifth of it, at least `least`."""
    return [max(least, full - (full * 4 * i) // (5 * n)) for i in range(n)]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _items(rows):
    """Rows of an item: 125 frames where there are enough of them."""
    return max(1, min(rows, 125))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)
    order = np.random.default_rng(int(seed))
    dt = _TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)

    st = {"case": case}
    if case["kind"] == "norm":
        M, d = case["rows"], case["d"]
        dx = torch.float32 if case["x32"] else torch.float16
        # a residual stream: a few channels far larger than the others, a mean apart from zero
        loud = torch.where(rand(d) < 0.01, torch.full((d,), 20.0, device="cuda"), torch.ones(d, device="cuda"))
        st.update(x=(2 * randn(M, d) * loud + 0.3).to(dx), y=(randn(M, d) * (0.5 + rand(M, 1))).to(dt), gate=None,
                  x_out=torch.zeros((M, d), device="cuda", dtype=dx), h=torch.zeros((M, d), device="cuda", dtype=dt),
                  per=_items(M) if case["gate"] == "item" else 1, eps=1e-5)
        for side in ("post", "pre"):
            st[side + "_w"] = 1 + 0.2 * randn(d) if case[side] != "none" else None
            st[side + "_b"] = 0.1 * randn(d) if case[side] == "layer" else None
        if case["gate"] != "none":
            st["gate"] = randn(-(-M // st["per"]), d).to(dt)
    elif case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        st.update(x=(randn(M, K) * (0.5 + rand(M, 1))).to(dt), w=(40 * randn(N, K)).round().clamp(-127, 127).to(torch.int8),
                  w_scale=0.0005 + 0.0005 * rand(N), bias=0.1 * randn(N) if case["bias"] else None,
                  add=randn(M, N).to(dt) if case["add"] else None, y=torch.zeros((M, N), device="cuda", dtype=dt))
    elif case["kind"] == "rotary":
        R, n, H, Hkv, dk, rot = (case[x] for x in ("R", "n", "H", "Hkv", "dk", "rot"))
        f = torch.pow(torch.full((rot // 2,), 10000.0, device="cuda", dtype=torch.float64),
                      -torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
        if case["scaled"]:      # eight times the context of 8192: what turns less than once in it is interpolated, more than 32 times kept
            keep = ((8192 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
            f = f * (keep + (1 - keep) / 8)
        lens = _spread(R, n, 1) if case["ragged"] else [n] * R
        # the projection's output: queries, keys and values of a token side by side
        st.update(qkv=randn(R, n, H + 2 * Hkv, dk).to(dt), freq=f, start=_ints(order.integers(0, case["far"] - n + 1, R).tolist()),
                  count=_ints(order.permutation(lens).tolist()), q_out=torch.zeros((R, n, H, dk), device="cuda", dtype=dt),
                  k_out=torch.zeros((R, n, Hkv, dk), device="cuda", dtype=dt))
    else:
        R, V, n = case["R"], case["V"], case["len"]
        x = 2.5 * randn(R, V)
        at = torch.randint(0, V, (R, 6), generator=g, device="cuda")
        x.scatter_add_(1, at, 6 + 4 * rand(R, 6))
        # words of a text: few frequent ones, many rare ones
        words = (V * rand(R, n) ** 4).long().clamp(0, V - 1).to(torch.int32)
        st.update(logits=x.to(dt), out=torch.zeros((R, V), device="cuda", dtype=dt), words=words,
                  len=_ints(order.permutation(_spread(R, n, 0)).tolist()), slot=_ints(order.permutation(R).tolist()), table=None,
                  repetition=1 + 0.3 * rand(R), presence=0.5 * rand(R), frequency=0.2 * rand(R), bias=None, bias_index=None,
                  mask=None, mask_index=None)
        if case["table"]:   # 8 beams an item, each position of a beam's history in one of its item's slots
            st["slot"] = None
            first = torch.arange(R, device="cuda")[:, None] // 8 * 8
            size = (R - first).clamp(max=8)
            st["table"] = (first + (rand(R, n) * size).long().minimum(size - 1)).to(torch.int32).contiguous()
        if case["bias"] != "none":
            many = 1 if case["bias"] == "one" else min(R, 8)
            st["bias"] = torch.where(rand(many, V) < 0.02, 4 * randn(many, V), torch.zeros(many, V, device="cuda"))
            st["bias_index"] = _ints(order.integers(-1 if many > 1 else 0, many, R).tolist())
        if case["mask"]:    # grammar states: most let few words through, one lets all through (row -1)
            many = min(R, 32)
            share = 0.02 + 0.5 * rand(many, 1) ** 2
            bits = (rand(many, (V + 31) // 32 * 32) < share).reshape(many, -1, 32).long()
            bits = (bits << torch.arange(32, device="cuda")).sum(2)
            st["mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32).contiguous()
            st["mask_index"] = _ints(order.integers(-1, many, R).tolist())
    if own:     # the plan that a program keeps: the buffers' addresses bound to the calls, the weights laid out once
        st["plan"] = _plan(st)
    return st


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
class _Dev:
    """A torch tensor as the binding's device array (address, shape, dtype, strides in elements)."""

    def __init__(self, t):
        self.t, self.ptr, self.shape, self.strides = t, t.data_ptr(), tuple(t.shape), tuple(t.stride())
        self.dtype = np.dtype(str(t.dtype).replace("torch.", ""))


def _plan(st):
    if _PY not in sys.path:
        sys.path.insert(0, _PY)
    import pkx

    case = st["case"]
    d = {k: _Dev(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "norm":
        return [pkx.BlockNorm(d["x"], d["h"], y=d["y"], x_out=d["x_out"], post=case["post"], post_w=d.get("post_w"), post_b=d.get("post_b"),
                              gate=d.get("gate"), rows_per_gate=st["per"], gate_fn=case["fn"], alpha=case["alpha"], pre=case["pre"],
                              pre_w=d.get("pre_w"), pre_b=d.get("pre_b"), eps=st["eps"])]
    if case["kind"] == "linear":
        w = pkx.WeightI8(d["w"], d["w_scale"])      # laid out once; the call quantises the tokens
        return [pkx.LinearI8(d["x"], w, d["y"], bias=d.get("bias"), act=case["act"], add=d.get("add"))]
    if case["kind"] == "rotary":
        H, Hkv = case["H"], case["Hkv"]
        return [pkx.Rotary(d["freq"], [(_Dev(st["qkv"][:, :, :H]), d["q_out"]), (_Dev(st["qkv"][:, :, H:H + Hkv]), d["k_out"])],
                           start=d["start"], count=d["count"], interleaved=case["pairs"] == "interleaved")]
    return [pkx.LogitRules(d["logits"], d["out"], tokens=d["words"], length=d["len"], slot=d.get("slot"), table=d.get("table"),
                           window=case["window"], repetition=d["repetition"], presence=d["presence"], frequency=d["frequency"],
                           bias=d.get("bias"), bias_index=d.get("bias_index"), mask=d.get("mask"), mask_index=d.get("mask_index"))]


def _outputs(st):
    kind = st["case"]["kind"]
    return {n: st[n] for n in {"norm": ("x_out", "h"), "linear": ("y",), "rotary": ("q_out", "k_out"), "rules": ("out",)}[kind]}


def _own(st):
    for call in st["plan"]:
        call()
    return _outputs(st)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_normalised(x, kind, w, b, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return x if b is None else x + b


def _plain_norm(st):
    case = st["case"]
    x, y = st["x"].float(), st["y"].float()
    u = _plain_normalised(y, case["post"], st["post_w"], st["post_b"], st["eps"])
    if st["gate"] is not None:
        gate = st["gate"].float()
        if case["fn"] == "sigmoid":
            gate = 1 / (1 + torch.exp(-gate))
        u = u * gate.repeat_interleave(st["per"], 0)[:x.shape[0]]
    x = x + case["alpha"] * u
    h = _plain_normalised(x, case["pre"], st["pre_w"], st["pre_b"], st["eps"])
    return {"x_out": x.to(st["x"].dtype), "h": h.to(st["y"].dtype)}


def _plain_linear(st):
    x = st["x"].float()
    top = x.abs().amax(1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    q = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale)).clamp(-127, 127)
    y = torch.matmul(q, st["w"].float().t()) * (scale * st["w_scale"])
    if st["bias"] is not None:
        y = y + st["bias"]
    if st["case"]["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    if st["add"] is not None:
        y = st["add"].float() + y
    return {"y": y.to(st["x"].dtype)}


def _plain_turned(x, cos, sin, rot, pairs):
    """x [R][n][H][dk] in 32 bits, cos and sin [R][n][1][rot / 2]."""
    x, rest = x[..., :rot], x[..., rot:]
    if pairs == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_rotary(st):
    case, n = st["case"], st["case"]["n"]
    at = torch.arange(n, device="cuda")
    angle = (st["start"].double()[:, None] + at)[:, :, None] * st["freq"]       # in 64 bits: far positions
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    live = (at < st["count"][:, None])[:, :, None, None]
    H, Hkv = case["H"], case["Hkv"]
    q, k = (_plain_turned(x.float(), cos, sin, case["rot"], case["pairs"]).to(x.dtype)
            for x in (st["qkv"][:, :, :H], st["qkv"][:, :, H:H + Hkv]))
    return {"q_out": torch.where(live, q, st["q_out"]), "k_out": torch.where(live, k, st["k_out"])}


def _plain_rules(st):
    case, n = st["case"], st["case"]["len"]
    R, V = case["R"], case["V"]
    x = st["logits"].float()
    pos = torch.arange(n, device="cuda")
    rows = torch.arange(R, device="cuda")[:, None].expand(-1, n)
    where = st["table"].long() if st["table"] is not None else st["slot"].long()[:, None].expand(-1, n)
    words = st["words"][where, pos].long()
    last = st["len"].long()[:, None]
    counted = pos < last
    if case["window"]:
        counted = counted & (pos >= last - case["window"])
    times = torch.zeros((R, V), device="cuda")
    times.index_put_((rows, words), counted.float(), accumulate=True)
    rep, pres, freq = (st[k][:, None] for k in ("repetition", "presence", "frequency"))
    seen = times > 0
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep) - pres - freq * times, x)
    if st["bias"] is not None:
        i = st["bias_index"].long()[:, None]
        x = x + torch.where(i >= 0, st["bias"][i[:, 0].clamp(min=0)], torch.zeros_like(x))
    if st["mask"] is not None:
        i, v = st["mask_index"].long(), torch.arange(V, device="cuda")
        bit = (st["mask"][i.clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        x = torch.where((bit != 0) | (i < 0)[:, None], x, torch.full_like(x, -math.inf))
    return {"out": x.to(st["logits"].dtype)}


def run(st):
    if own:
        return _own(st)
    return {"norm": _plain_norm, "linear": _plain_linear, "rotary": _plain_rotary, "rules": _plain_rules}[st["case"]["kind"]](st)


# ---------------------------------------------------------------------------
# work, and the operators from their definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = 2.0 if case["type"] == "f16" else 4.0
    if case["kind"] == "norm":
        M, d = float(case["rows"]), case["d"]
        gates = {"none": 0.0, "row": M, "item": float(-(-case["rows"] // _items(case["rows"])))}[case["gate"]]
        vectors = sum({"none": 0, "rms": 1, "layer": 2}[case[s]] for s in ("post", "pre"))
        return {"bytes": d * (M * (2 * (4.0 if case["x32"] else 2.0) + 2 * e) + gates * e + 4.0 * vectors), "flops": 20.0 * M * d}
    if case["kind"] == "linear":
        M, N, K = float(case["M"]), case["N"], case["K"]
        return {"bytes": M * K * e + N * K + M * N * e * (2 if case["add"] else 1) + 4.0 * (M + N * (2 if case["bias"] else 1)),
                "flops": 2.0 * M * N * K}
    if case["kind"] == "rotary":
        tokens = float(sum(_spread(case["R"], case["n"], 1))) if case["ragged"] else float(case["R"] * case["n"])
        heads = case["H"] + case["Hkv"]
        return {"bytes": 2 * e * tokens * heads * case["dk"] + 8.0 * case["R"], "flops": tokens * (3.0 * heads * case["rot"] + 20.0 * case["rot"])}
    R, V = float(case["R"]), case["V"]
    seen = sum(min(n, case["window"] or n) for n in _spread(case["R"], case["len"], 0))
    by = 2 * e * R * V + seen * (8.0 if case["table"] else 4.0) + 16.0 * R
    by += {"none": 0.0, "one": 4.0 * V, "rows": 4.0 * V * min(case["R"], 8)}[case["bias"]]
    by += min(case["R"], 32) * V / 8.0 if case["mask"] else 0.0
    return {"bytes": by, "flops": 4.0 * R * V}


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "rotary": _exact_rotary, "rules": _exact_rules}[case["kind"]](st)


def _exact_normalised(x, kind, w, b, eps):
    if kind == "none":
        return x
    mean = x.sum(1) / x.shape[1] if kind == "layer" else torch.zeros(x.shape[0], device="cuda", dtype=torch.float64)
    var = ((x - mean[:, None]) ** 2).sum(1) / x.shape[1]
    out = (x - mean[:, None]) / torch.sqrt(var + eps)[:, None] * w.double()[None]
    return out if b is None else out + b.double()[None]


def _exact_norm(st):
    case = st["case"]
    u = _exact_normalised(st["y"].double(), case["post"], st["post_w"], st["post_b"], st["eps"])
    if st["gate"] is not None:
        i = torch.arange(case["rows"], device="cuda") // st["per"]
        gate = st["gate"].double()[i]
        u = u * (torch.sigmoid(gate) if case["fn"] == "sigmoid" else gate)
    x = st["x"].double() + case["alpha"] * u
    return {"x_out": x, "h": _exact_normalised(x, case["pre"], st["pre_w"], st["pre_b"], st["eps"])}


def _exact_linear(st):
    # what is held in 8 bits, and its scale, are defined by 32-bit steps; the rest is in 64
    out, w = [], st["w"].double()
    for x in st["x"].float().split(2048):
        s = (x.abs().max(1).values / torch.tensor(127.0, device="cuda"))[:, None]
        q = torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-127, 127)
        out.append((q.double() @ w.t()) * s.double() * st["w_scale"].double()[None])
    y = torch.cat(out)
    if st["bias"] is not None:
        y = y + st["bias"].double()[None]
    if st["case"]["act"] == "silu":
        y = y * torch.sigmoid(y)
    return {"y": y if st["add"] is None else y + st["add"].double()}


def _exact_rotary(st):
    case, out = st["case"], {}
    rot, R, n = case["rot"], case["R"], case["n"]
    # a pair as a complex number times e^(i angle)
    pos = st["start"].double()[:, None] + torch.arange(n, device="cuda", dtype=torch.float64)[None]
    turn = torch.polar(torch.ones((R, n, rot // 2), device="cuda", dtype=torch.float64), pos[:, :, None] * st["freq"])
    first = torch.arange(rot // 2, device="cuda") * (2 if case["pairs"] == "interleaved" else 1)
    second = first + (1 if case["pairs"] == "interleaved" else rot // 2)
    gone = torch.arange(n, device="cuda")[None] >= st["count"][:, None]
    for name, lo, hi in (("q_out", 0, case["H"]), ("k_out", case["H"], case["H"] + case["Hkv"])):
        x = st["qkv"][:, :, lo:hi].double()
        z = torch.complex(x[..., first], x[..., second]) * turn[:, :, None]
        x[..., first], x[..., second] = z.real, z.imag
        x[gone] = 0
        out[name] = x
    return out


def _exact_rules(st):
    case = st["case"]
    R, V = case["R"], case["V"]
    words, lens = st["words"].cpu().numpy(), st["len"].tolist()
    table = st["table"].cpu().numpy() if st["table"] is not None else None
    slots = st["slot"].tolist() if table is None else None
    out = st["logits"].cpu().numpy().astype(np.float64)
    bias = None if st["bias"] is None else st["bias"].cpu().numpy().astype(np.float64)
    for r in range(R):
        t = np.arange(max(0, lens[r] - case["window"]) if case["window"] else 0, lens[r])
        ids, times = np.unique(words[table[r, t], t] if table is not None else words[slots[r], t], return_counts=True)
        rep, pres, freq = (float(st[k][r]) for k in ("repetition", "presence", "frequency"))
        v = out[r, ids]
        out[r, ids] = np.where(v > 0, v / rep, v * rep) - pres - freq * times
        if bias is not None and int(st["bias_index"][r]) >= 0:
            out[r] += bias[int(st["bias_index"][r])]
    out = torch.from_numpy(out).cuda()
    if st["mask"] is not None:
        bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V] > 0
        bits = torch.from_numpy(bits).cuda()
        for r, i in enumerate(st["mask_index"].tolist()):
            if i >= 0:
                out[r, ~bits[i]] = -math.inf
    return {"out": out}
