"""Performance cases of the decoder operators: what an attention decoder under beam search calls per step.

  cross  attention of a decoder's queries to an encoder's states of another length (f16, f32)
  cache  new tokens appended to an 8-bit key/value cache (a scale for each block of 32 tokens and head),
         attention over it, and the touched tokens read back as values
  beam   selection of the W best of W x V candidates per item, and the beams' states reordered

run() with own = False states the operators in elementary torch operations; with own = True it calls the framework
(pkx.CrossAttention, pkx.CacheAppend, pkx.CacheAttention, pkx.CacheRead, pkx.BeamSelect, pkx.BeamReorder).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32      # tokens that share a scale in the cache
_PY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_amd", "python")
_TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one utterance of 10 s (125 frames), the next token of a greedy decode: latency
        {"name": "cross_f16_b1_10s", "kind": "cross", "type": "f16", "B": 1, "nq": 1, "T": 125, "H": 8, "Hkv": 8, "dk": 64,
         "ragged": False, "mask": False},
        # a batch of 16 ragged clips up to 30 s, 4 beams each
        {"name": "cross_f16_b16_w4_30s", "kind": "cross", "type": "f16", "B": 16, "nq": 4, "T": 375, "H": 8, "Hkv": 8, "dk": 128,
         "ragged": True, "mask": False},
        # four recordings of 5 minutes, 8 beams, two query heads to a key head
        {"name": "cross_f16_b4_w8_300s", "kind": "cross", "type": "f16", "B": 4, "nq": 8, "T": 3750, "H": 16, "Hkv": 8, "dk": 64,
         "ragged": False, "mask": False},
        # transcripts scored against their audio in one pass: many queries
        {"name": "cross_f16_b16_q448", "kind": "cross", "type": "f16", "B": 16, "nq": 448, "T": 750, "H": 8, "Hkv": 8, "dk": 128,
         "ragged": False, "mask": False},
        # the exact-precision path, odd sizes, silent frames masked out
        {"name": "cross_f32_b3_masked", "kind": "cross", "type": "f32", "B": 3, "nq": 37, "T": 211, "H": 8, "Hkv": 8, "dk": 64,
         "ragged": True, "mask": True},
        # one dictation, 18th token: latency
        {"name": "cache_f16_r1", "kind": "cache", "type": "f16", "R": 1, "nq": 1, "new": 1, "len": 18, "H": 8, "Hkv": 8, "dk": 64,
         "table": False, "causal": True},
        # 16 items x 8 beams, the next token, each beam's history spread over its item's slots
        {"name": "cache_f16_r128_beams", "kind": "cache", "type": "f16", "R": 128, "nq": 1, "new": 1, "len": 448, "H": 8, "Hkv": 8,
         "dk": 64, "table": True, "causal": True},
        # four long documents, four query heads to a key head
        {"name": "cache_f16_r4_long", "kind": "cache", "type": "f16", "R": 4, "nq": 1, "new": 1, "len": 32768, "H": 16, "Hkv": 4,
         "dk": 128, "table": False, "causal": True},
        # prompts of 200 tokens after histories of different lengths, exact-precision activations
        {"name": "cache_f32_r8_prompt", "kind": "cache", "type": "f32", "R": 8, "nq": 200, "new": 200, "len": 1025, "H": 8, "Hkv": 8,
         "dk": 64, "table": False, "causal": True},
        # one utterance, 4 beams over the transducer's vocabulary, the prediction network's states moved along
        {"name": "beam_f32_b1_w4", "kind": "beam", "type": "f32", "B": 1, "W": 4, "V": 1025, "states": 4, "row": 2560, "done": False},
        # a serving batch on a wordpiece vocabulary of 8192 and its end token, some beams finished
        {"name": "beam_f16_b16_w8", "kind": "beam", "type": "f16", "B": 16, "W": 8, "V": 8193, "states": 4, "row": 2560, "done": True},
        # the widest search: 32 items x 16 beams, 32k words, a cache's history table among the states
        {"name": "beam_f32_b32_w16", "kind": "beam", "type": "f32", "B": 32, "W": 16, "V": 32769, "states": 2, "row": 4096, "done": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cross", "cache", "beam"])
    if kind == "beam":
        W, V = _log_int(rng, 1, 16), _log_int(rng, 33, 65537)
        B = min(_log_int(rng, 1, 64), max(1, (16 << 20) // (W * V)))
        return {"kind": kind, "type": rng.choice(["f16", "f32"]), "B": B, "W": W, "V": V, "states": rng.randint(1, 8),
                "row": 4 * _log_int(rng, 16, 2048), "done": rng.random() < 0.5}
    kind_type = rng.choice(["f16", "f16", "f32"])
    dk = rng.choice([32, 64, 64, 80, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 1, 2, 4])
    if kind == "cross":
        nq, T, B = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 512)]), _log_int(rng, 1, 3750), _log_int(rng, 1, 32)
        most = 22e9 if kind_type == "f16" else 1.4e9
        B = max(1, min(B, int(most / (4.0 * nq * T * H * dk))))
        nq = max(1, min(nq, int(most / (4.0 * B * T * H * dk))))
        return {"kind": kind, "type": kind_type, "B": B, "nq": nq, "T": T, "H": H, "Hkv": Hkv, "dk": dk,
                "ragged": rng.random() < 0.5, "mask": rng.random() < 0.3}
    new = rng.choice([1, 1, _log_int(rng, 2, 256)])
    n = max(new, _log_int(rng, 1, 16384))
    causal = rng.random() < 0.75
    nq = new if causal else rng.choice([1, 4, 8])       # without it: queries of beams over an encoder's states
    most = 128e6 if nq <= 16 else 16e6
    R = max(1, min(_log_int(rng, 1, 256), int(most / (2.0 * n * Hkv * dk)), int(4e9 / (4.0 * nq * n * H * dk))))
    return {"kind": kind, "type": kind_type, "R": R, "nq": nq, "new": new, "len": n, "H": H, "Hkv": Hkv, "dk": dk,
            "table": nq == 1 and rng.random() < 0.5, "causal": causal}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _spread(n, full, least):
    """Lengths from `full` down to a fifth of it, at least `least`."""
    return [max(least, full - (full * 4 * i) // (5 * n)) for i in range(n)]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    order = np.random.default_rng(int(seed))
    dt = _TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    st = {"case": case}
    if case["kind"] == "cross":
        B, nq, T, H, Hkv, dk = (case[x] for x in ("B", "nq", "T", "H", "Hkv", "dk"))
        lens = _spread(B, T, 1) if case["ragged"] else [T] * B
        st.update(q=(2 * randn(B, nq, H, dk)).to(dt), k=randn(B, T, Hkv, dk).to(dt), v=randn(B, T, Hkv, dk).to(dt),
                  k_len=_ints(order.permutation(lens).tolist()), k_mask=None,
                  out=torch.zeros((B, nq, H, dk), device="cuda", dtype=dt))
        if case["mask"]:    # stretches of silence: a fifth of the frames, in runs
            runs = torch.rand((B, T // 7 + 1), generator=g, device="cuda") > 0.2
            st["k_mask"] = runs.repeat_interleave(7, 1)[:, :T].contiguous().to(torch.uint8)
    elif case["kind"] == "cache":
        R, nq, new, n, H, Hkv, dk = (case[x] for x in ("R", "nq", "new", "len", "H", "Hkv", "dk"))
        cap = (n + BLOCK - 1) // BLOCK * BLOCK + BLOCK
        lens = _ints(order.permutation(_spread(R, n, new)).tolist())
        kv = [(36 * randn(R, Hkv, cap, dk)).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
        sc = [0.02 + 0.02 * torch.rand((R, Hkv, cap // BLOCK), generator=g, device="cuda") for _ in range(2)]
        st.update(q=(1.5 * randn(R, nq, H, dk)).to(dt), k_new=randn(R, new, Hkv, dk).to(dt), v_new=randn(R, new, Hkv, dk).to(dt),
                  k=kv[0], v=kv[1], k_scale=sc[0], v_scale=sc[1], len=lens, start=lens - new, read_from=lens - new - (BLOCK - 1),
                  slot=_ints(order.permutation(R).tolist()), table=None,
                  out=torch.zeros((R, nq, H, dk), device="cuda", dtype=dt))
        st["k_read"], st["v_read"] = (torch.zeros((R, new + BLOCK - 1, Hkv, dk), device="cuda") for _ in range(2))
        if case["table"]:   # 8 beams an item: one common history, apart over the last 16 tokens; rows are slots
            st["slot"] = torch.arange(R, dtype=torch.int32, device="cuda")
            first = st["slot"].long() // 8 * 8
            size = (R - first).clamp(max=8)[:, None]
            common = torch.rand((R // 8 + 1, cap), generator=g, device="cuda")[first // 8]
            apart = torch.rand((R, cap), generator=g, device="cuda")
            late = torch.arange(cap, device="cuda")[None, :] >= st["start"].long()[:, None] - 16
            pick = (torch.where(late, apart, common) * size).long().minimum(size - 1)
            # an item's slots hold as many tokens as its shortest beam has
            st["table"] = (first[:, None] + pick).to(torch.int32).contiguous()
    else:
        B, W, V = case["B"], case["W"], case["V"]
        x = 2.5 * randn(B, W, V)
        # a sharp distribution as a trained model's: a few words stand out in each row
        at = torch.randint(0, V, (B, W, 6), generator=g, device="cuda")
        x.scatter_add_(2, at, 6 + 4 * torch.rand((B, W, 6), generator=g, device="cuda"))
        scores = -20 + 3 * randn(B, W)
        done = torch.rand((B, W), generator=g, device="cuda") < (0.15 if case["done"] else -1.0)
        st.update(logits=x.to(dt), scores=scores, done=done.to(torch.uint8), end=V - 1)
        st.update({n: torch.zeros((B, W), device="cuda", dtype=d) for n, d in
                   (("parent", torch.int32), ("token", torch.int32), ("new_scores", torch.float32), ("new_done", torch.uint8))})
        st["src"] = [randn(B * W, case["row"] // 4) for _ in range(case["states"])]
        st["dst"] = [torch.zeros_like(s) for s in st["src"]]
    if own:     # the plan that a program keeps: the buffers' addresses bound to the calls, no data touched
        st["plan"] = _plan(st)
    return st


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
class _Dev:
    """A torch tensor as the binding's device array (address, shape, dtype)."""

    def __init__(self, t):
        self.t, self.ptr, self.shape = t, t.data_ptr(), tuple(t.shape)
        self.dtype = np.dtype(str(t.dtype).replace("torch.", ""))


def _plan(st):
    if _PY not in sys.path:
        sys.path.insert(0, _PY)
    import pkx

    d = {k: _Dev(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
    if st["case"]["kind"] == "cross":
        return [pkx.CrossAttention(d["q"], d["k"], d["v"], d["out"], k_len=d["k_len"], k_mask=d.get("k_mask"))]
    if st["case"]["kind"] == "cache":
        c = pkx.Cache8.wrap(d["k"], d["v"], d["k_scale"], d["v_scale"])
        return [pkx.CacheAppend(c, d["k_new"], d["v_new"], start=d["start"], slot=d["slot"], table=d.get("table")),
                pkx.CacheAttention(c, d["q"], d["out"], length=d["len"], slot=d["slot"], table=d.get("table"),
                                   causal=st["case"]["causal"]),
                pkx.CacheRead(c, d["k_read"], d["v_read"], start=d["read_from"], slot=d["slot"])]
    return [pkx.BeamSelect(d["logits"], d["scores"], d["parent"], d["token"], d["new_scores"], done=d["done"],
                           new_done=d["new_done"], end_id=st["end"]),
            pkx.BeamReorder(d["parent"], [(_Dev(a), _Dev(b)) for a, b in zip(st["src"], st["dst"])])]


def _own(st):
    for call in st["plan"]:
        call()
    if st["case"]["kind"] == "cross":
        return {"out": st["out"]}
    if st["case"]["kind"] == "cache":
        return {"out": st["out"], "k": st["k_read"], "v": st["v_read"], "table": st["table"]}
    return {"parent": st["parent"], "token": st["token"], "scores": st["new_scores"], "done": st["new_done"], "states": st["dst"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _softmax_values(s, keep, v):
    """softmax over the kept last places of s (none kept: zeros), times v."""
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    z = p.sum(-1, keepdim=True)
    return torch.matmul(p / torch.where(z == 0, torch.ones_like(z), z), v)


def _heads(x, times):
    """[N][T][Hkv][dk] -> [N][Hkv * times][T][dk] in 32 bits."""
    return x.float().transpose(1, 2).repeat_interleave(times, 1).contiguous()


def _plain_cross(st):
    q, k, v = st["q"], st["k"], st["v"]
    G, T = q.shape[2] // k.shape[2], k.shape[1]
    keep = torch.arange(T, device=q.device)[None, :] < st["k_len"][:, None]
    if st["k_mask"] is not None:
        keep = keep & (st["k_mask"] != 0)
    s = torch.matmul(_heads(q, 1), _heads(k, G).transpose(2, 3).contiguous()) / math.sqrt(q.shape[3])
    return {"out": _softmax_values(s, keep[:, None, None, :], _heads(v, G)).transpose(1, 2).to(q.dtype).contiguous()}


def _plain_append(st, ints, scales, x):
    """Appends x [R][new][Hkv][dk] at positions start .. of the rows' slots, block by block (all within the capacity)."""
    R, new, Hkv, dk = x.shape
    start, slot = st["start"].long(), st["slot"].long()
    b0, NB = start // BLOCK, (new + 2 * BLOCK - 2) // BLOCK
    blocks = b0[:, None] + torch.arange(NB, device=x.device)                                     # [R][NB]
    pos = (b0 * BLOCK)[:, None] + torch.arange(NB * BLOCK, device=x.device)                      # [R][NB * BLOCK]
    is_new = (pos >= start[:, None]) & (pos < start[:, None] + new)
    is_old = pos < start[:, None]
    at = (pos - start[:, None]).clamp(0, new - 1)[:, :, None, None].expand(-1, -1, Hkv, dk)
    xn = torch.gather(x.float(), 1, at)
    amax = (xn.abs() * is_new[:, :, None, None]).reshape(R, NB, BLOCK, Hkv, dk).amax((2, 4))      # [R][NB][Hkv]
    held = scales[slot[:, None], :, blocks]
    begun = ((start % BLOCK != 0)[:, None] & (blocks == b0[:, None]))[:, :, None]
    before = torch.where(begun, held, torch.zeros_like(held))
    touched = is_new.reshape(R, NB, BLOCK).any(2)[:, :, None]
    scale = torch.maximum(before, amax / torch.full_like(amax, 127.0))
    div = torch.where(scale == 0, torch.ones_like(scale), scale)
    ratio = (before / div).repeat_interleave(BLOCK, 1)[:, :, :, None]
    div = div.repeat_interleave(BLOCK, 1)[:, :, :, None]
    old = ints[slot[:, None], :, pos]
    q_old = torch.round(old.float() * ratio)
    q_new = torch.round(xn / div).clamp(-127, 127)
    q = torch.where(is_new[:, :, None, None], q_new, torch.where(is_old[:, :, None, None], q_old, old.float())).to(torch.int8)
    heads = torch.arange(Hkv, device=x.device)
    ints[slot[:, None, None], heads, pos[:, :, None]] = q
    scales[slot[:, None, None], heads, blocks[:, :, None]] = torch.where(touched, scale, held)


def _plain_values(ints, scales, slot, pos):
    """The values of tokens pos [R][n] of slots [R][n]: [R][n][Hkv][dk]; zeros before a slot's first token."""
    p = pos.clamp(0, ints.shape[2] - 1)
    x = ints[slot, :, p].float() * scales[slot, :, p // BLOCK][..., None]
    return torch.where((pos >= 0)[:, :, None, None], x, torch.zeros_like(x))


def _plain_cache(st):
    case, new = st["case"], st["k_new"].shape[1]
    R, slot, n = case["R"], st["slot"].long(), st["len"].long()
    _plain_append(st, st["k"], st["k_scale"], st["k_new"])
    _plain_append(st, st["v"], st["v_scale"], st["v_new"])
    pos = torch.arange(case["len"], device=slot.device)[None, :].expand(R, -1)
    where = slot[:, None].expand(-1, case["len"])
    if st["table"] is not None:
        mine = st["start"].long()[:, None] + torch.arange(new, device=slot.device)
        st["table"].scatter_(1, mine, st["slot"][:, None].expand(-1, new))
        where = st["table"][:, :case["len"]].long()
    q = st["q"]
    k, v = (_heads(_plain_values(st[a], st[b], where, pos), case["H"] // case["Hkv"]) for a, b in (("k", "k_scale"), ("v", "v_scale")))
    last = n[:, None].expand(-1, q.shape[1])
    if case["causal"]:
        last = last - (q.shape[1] - 1) + torch.arange(q.shape[1], device=slot.device)
    keep = pos[:, None, :] < last[:, :, None]
    s = torch.matmul(_heads(q, 1), k.transpose(2, 3).contiguous()) / math.sqrt(q.shape[3])
    out = _softmax_values(s, keep[:, None], v).transpose(1, 2).to(q.dtype).contiguous()
    back = st["read_from"].long()[:, None] + torch.arange(new + BLOCK - 1, device=slot.device)
    k, v = (_plain_values(st[a], st[b], slot[:, None].expand_as(back), back) for a, b in (("k", "k_scale"), ("v", "v_scale")))
    return {"out": out, "k": k, "v": v, "table": st["table"]}


def _plain_beam(st):
    B, W, V = st["logits"].shape
    # in 64 bits: candidates of different beams lie as close as their sums' rounding
    x, score = st["logits"].double(), st["scores"].double()
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    c = score[:, :, None] + (x - lse)
    c = torch.where(torch.isnan(c), torch.full_like(c, -math.inf), c)
    done = (st["done"] != 0)[:, :, None]
    at_end = (torch.arange(V, device=x.device) == st["end"])[None, None, :]
    c = torch.where(done & at_end, score[:, :, None], c)
    # a finished beam's other words come after every candidate, those of no probability too
    rank = torch.where(done & ~at_end, torch.full_like(c, -math.inf), c.clamp(min=-1e300))
    best = torch.sort(rank.reshape(B, W * V), dim=1, descending=True, stable=True)[1][:, :W]
    parent, token = best // V, best % V
    scores = torch.gather(c.reshape(B, W * V), 1, best).float()
    ended = torch.gather(done[:, :, 0], 1, parent) | (token == st["end"])
    rows = (parent + W * torch.arange(B, device=x.device)[:, None]).reshape(-1)
    return {"parent": parent.to(torch.int32), "token": token.to(torch.int32), "scores": scores, "done": ended.to(torch.uint8),
            "states": [s[rows] for s in st["src"]]}


def run(st):
    if own:
        return _own(st)
    return {"cross": _plain_cross, "cache": _plain_cache, "beam": _plain_beam}[st["case"]["kind"]](st)


# ---------------------------------------------------------------------------
# work, and the operators from their definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = 2.0 if case["type"] == "f16" else 4.0
    if case["kind"] == "beam":
        rows = case["B"] * case["W"]
        return {"bytes": rows * (case["V"] * e + 4 + 1 + 13) + 2.0 * rows * case["states"] * case["row"],
                "flops": 4.0 * rows * case["V"]}
    H, Hkv, dk, nq = case["H"], case["Hkv"], case["dk"], case["nq"]
    if case["kind"] == "cross":
        lens = _spread(case["B"], case["T"], 1) if case["ragged"] else [case["T"]] * case["B"]
        mask = float(case["B"] * case["T"]) if case["mask"] else 0.0
        return {"bytes": e * (2.0 * case["B"] * nq * H * dk + 2.0 * sum(lens) * Hkv * dk) + mask, "flops": 4.0 * nq * sum(lens) * H * dk}
    R, new = case["R"], case["new"]
    lens = _spread(R, case["len"], new)
    seen = sum(n - (nq - 1) / 2.0 for n in lens) if case["causal"] else float(sum(lens))
    values = R * (new + BLOCK - 1) * Hkv * dk
    by = 2.0 * sum(lens) * Hkv * (dk + 4.0 / BLOCK) + (4.0 * sum(lens) if case["table"] else 0.0)
    by += e * 2.0 * R * nq * H * dk + 2.0 * (e + 1) * R * new * Hkv * dk + 2.0 * (1 + 4) * values
    return {"bytes": by, "flops": 4.0 * nq * seen * H * dk}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "beam":
        return _exact_beam(st)
    if case["kind"] == "cross":
        B, nq, H, dk = st["q"].shape
        G, o = H // case["Hkv"], torch.zeros((B, nq, H, dk), device="cuda", dtype=torch.float64)
        for b in range(B):
            at = torch.arange(case["T"], device="cuda") < st["k_len"][b]
            at = at if st["k_mask"] is None else at & (st["k_mask"][b] > 0)
            for h in range(H):
                o[b, :, h] = _exact_attention(st["q"][b, :, h], st["k"][b, at, h // G], st["v"][b, at, h // G], None)
        return {"out": o}
    R, H, G, new = case["R"], case["H"], case["H"] // case["Hkv"], case["new"]
    if R * H > 4096:
        return None
    for x, ints, scales in ((st["k_new"], st["k"], st["k_scale"]), (st["v_new"], st["v"], st["v_scale"])):
        _exact_append(st, x.float(), ints, scales)
    o = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
    starts, lens, slots = (st[x].tolist() for x in ("start", "len", "slot"))
    for r in range(R):
        if st["table"] is not None:
            st["table"][r, starts[r]:lens[r]] = slots[r]
        t = torch.arange(lens[r], device="cuda")
        where = torch.full_like(t, slots[r]) if st["table"] is None else st["table"][r, :lens[r]].long()
        k, v = (st[a][where, :, t].double() * st[b][where, :, t // BLOCK].double()[..., None] for a, b in (("k", "k_scale"), ("v", "v_scale")))
        for h in range(H):
            o[r, :, h] = _exact_attention(st["q"][r, :, h], k[:, h // G], v[:, h // G], case["causal"])
    # the values held in 8 bits are defined by 32-bit steps: they have no other value in 64
    return {"out": o, "k": None, "v": None, "table": st["table"]}


def _exact_attention(q, k, v, causal):
    if not len(k):
        return torch.zeros_like(q, dtype=torch.float64)
    s = q.double() @ k.double().t() / math.sqrt(q.shape[1])
    if causal:
        n, t = s.shape
        s = s.masked_fill(torch.ones((n, t), device="cuda", dtype=torch.bool).triu(t - n + 1), -math.inf)
    return torch.softmax(s, 1) @ v.double()


def _exact_append(st, x, ints, scales):
    """Token block by token block, all rows that touch one at a time."""
    new = x.shape[1]
    starts, slots = st["start"].tolist(), st["slot"].tolist()
    c127 = torch.tensor(127.0, device="cuda")
    for r, (s, slot) in enumerate(zip(starts, slots)):
        for b in range(s // BLOCK, (s + new - 1) // BLOCK + 1):
            lo, hi = max(s, b * BLOCK), min(s + new, (b + 1) * BLOCK)
            part = x[r, lo - s:hi - s].transpose(0, 1)                       # [Hkv][n][dk]
            top = part.abs().amax((1, 2)) / c127
            if lo > b * BLOCK:
                was = scales[slot, :, b].clone()
                top = torch.maximum(top, was)
                f = torch.where(top > 0, was / top, torch.zeros_like(top))
                old = ints[slot, :, b * BLOCK:lo]
                ints[slot, :, b * BLOCK:lo] = torch.round(old.float() * f[:, None, None]).to(torch.int8)
            scales[slot, :, b] = top
            ints[slot, :, lo:hi] = torch.where(top[:, None, None] > 0, torch.round(part / top[:, None, None]),
                                               torch.zeros_like(part)).clamp(-127, 127).to(torch.int8)


def _exact_beam(st):
    B, W, V = st["logits"].shape
    parent, token = (torch.zeros((B, W), dtype=torch.int32) for _ in range(2))
    scores, done, states = torch.zeros((B, W), dtype=torch.float64), torch.zeros((B, W), dtype=torch.uint8), []
    ended = st["done"].cpu().numpy()
    logits, old = st["logits"].cpu().numpy(), st["scores"].cpu().numpy().astype(np.float64)
    for b in range(B):
        found = []
        for w in range(W):
            if ended[b, w]:
                found.append((-old[b, w], w, st["end"]))
                continue
            x = logits[b, w].astype(np.float64)
            top = np.argsort(-x, kind="stable")[:W]
            z = x.max() + np.log(np.exp(x - x.max()).sum())
            found += [(-(old[b, w] + (x[i] - z)), w, int(i)) for i in top]
        for i, (c, w, t) in enumerate(sorted(found)[:W]):
            parent[b, i], token[b, i], scores[b, i], done[b, i] = w, t, -c, int(bool(ended[b, w]) or t == st["end"])
    rows = (parent.long() + W * torch.arange(B)[:, None]).reshape(-1).cuda()
    states = [s[rows].double() for s in st["src"]]
    return {"parent": parent, "token": token, "scores": scores, "done": done, "states": states}
