"""Refusals and size queries of the attention decoder operators, which need no
GPU: every check comes before the first device call.  The library is exercised
in a subprocess so this process never loads a HIP runtime."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import decoder_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "parakeet.cpp_amd", "build", "libpkx.so")


def _run(code):
    if not os.path.exists(LIB):
        pytest.skip("libpkx.so not built")
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "parakeet.cpp_amd", "python"))
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(PRE) + textwrap.dedent(code)], capture_output=True, text=True,
                       env=env, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout.strip().split("\n")


# addresses that nothing may follow: the calls have to fail (or do nothing) before the device
PRE = """
import ctypes as C, pkx
L = pkx.lib()
A = 1 << 20
def said(rc):
    print(rc, L.pkx_last_error().decode())
def cross(**kw):
    a = pkx.CrossAttnArgs(1, 2, 3, 40, 4, 2, 64, 0.125, A, 768, 256, 64, A, 5120, 128, 64, A, 5120, 128, 64, A, 768, 256, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a
def cache(**kw):
    c = pkx.Cache8Args(3, 2, 64, 96, A, A, A, A)
    for k, v in kw.items():
        setattr(c, k, v)
    return c
def toks(**kw):
    a = pkx.Cache8Tokens(1, 2, 5, A, 640, 128, 64, A, 640, 128, 64, None, A, None, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a
def attn(**kw):
    a = pkx.Cache8AttnArgs(1, 2, 1, 4, 1, 0.125, A, 256, 256, 64, A, 256, 256, 64, None, A, None, None, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a
def beam(**kw):
    a = pkx.BeamSelectArgs(1, 2, 4, 100, 5, A, 100, A, None, A, A, A, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a
"""


def test_cross_attention_refusals():
    out = _run("""
        for kw in (dict(type=8), dict(n_items=-1), dict(n_heads=3), dict(n_kv_heads=0), dict(d_head=60), dict(d_head=136),
                   dict(n_k=(1 << 30) + 1), dict(out_row=56), dict(out_head=0), dict(q=None), dict(k=A + 8), dict(v_row=132), dict(out_head=-64), dict(k_row=1 << 22), dict(type=0, q_head=66)):
            said(L.pkx_cross_attention(cross(**kw), None, 0, None))
        said(L.pkx_cross_attention(None, None, 0, None))
        said(L.pkx_cross_attention_workspace(cross(), None))
        n = C.c_size_t()
        said(L.pkx_cross_attention_workspace(cross(n_items=1, n_q=1, n_k=100000), C.byref(n)))
        said(L.pkx_cross_attention(cross(n_items=1, n_q=1, n_k=100000), A, n.value - 1, None))
        said(L.pkx_cross_attention(cross(n_items=1, n_q=1, n_k=100000), A + 4, n.value, None))
        said(L.pkx_cross_attention(cross(n_items=1 << 30, n_q=1 << 20), A, 1 << 60, None))
        for kw in (dict(n_items=0), dict(n_q=0, q=None), dict(n_items=0, k=None)):
            said(L.pkx_cross_attention(cross(**kw), None, 0, None))
    """)
    words = ["type", "negative", "n_heads", "n_heads", "d_head", "d_head", "2^30", "overlap", "overlap", "q must", "k must", "v must", "out must", "2^22", "q must",
             "null", "null"]
    for line, w in zip(out[:17], words):
        assert line.startswith("1 ") and w in line, (line, w)
    assert out[17].strip() == "0"
    for line, w in zip(out[18:21], ("workspace", "aligned", "at most")):
        assert line.startswith("1 ") and w in line, (line, w)
    assert [x.strip() for x in out[21:]] == ["0"] * 3


def test_cache_refusals():
    out = _run("""
        for c, t in ((cache(n_slots=0), toks()), (cache(d_head=72), toks()), (cache(d_head=144), toks()), (cache(capacity=100), toks()),
                     (cache(capacity=0), toks()), (cache(k=None), toks()), (cache(v=A + 4), toks()), (cache(), toks(type=2)),
                     (cache(), toks(n_new=-1)), (cache(), toks(k_tok=130)), (cache(), toks(start=None)), (cache(), toks(n_rows=4)),
                     (cache(), toks(table=A, table_row=95)), (cache(), toks(n_rows=3 << 20, slot=A))):
            said(L.pkx_cache8_append(c, t, None))
        for a in (attn(type=3), attn(n_heads=3), attn(n_q=-1), attn(max_len=-1), attn(len=None), attn(n_rows=4), attn(q=None),
                  attn(out_tok=100), attn(table=A, table_row=95)):
            said(L.pkx_cache8_attention(cache(), a, None, 0, None))
        said(L.pkx_cache8_read(cache(), 1, 1, None, None, A, A, None))
        said(L.pkx_cache8_read(cache(), 1, 1, None, A, A + 4, A, None))
        for a in (toks(n_rows=0), toks(n_new=0)):
            said(L.pkx_cache8_append(cache(), a, None))
        said(L.pkx_cache8_attention(cache(), attn(n_rows=0), None, 0, None))
        said(L.pkx_cache8_attention(cache(), attn(n_q=0), None, 0, None))
        said(L.pkx_cache8_read(cache(), 1, 0, None, None, None, None, None))
    """)
    words = ["no slots", "d_head", "d_head", "capacity", "capacity", "null", "aligned", "type", "negative", "k must", "null start",
             "more rows", "shorter", "2^22", "type", "n_heads", "negative", "max_len", "null len", "more rows", "q must", "out must",
             "shorter", "null start", "aligned"]
    for line, w in zip(out[:25], words):
        assert line.startswith("1 ") and w in line, (line, w)
    assert [x.strip() for x in out[25:]] == ["0"] * 5


def test_beam_refusals():
    out = _run("""
        for kw in (dict(type=8), dict(n_beams=0), dict(n_beams=33), dict(vocab=0), dict(end_id=100), dict(end_id=-2),
                   dict(done=A, end_id=-1), dict(logits=None), dict(token=None), dict(logits=A + 1), dict(logits_row=-1)):
            said(L.pkx_beam_select(beam(**kw), A, 1 << 30, None))
        n, many = C.c_size_t(), beam(vocab=100000, logits_row=100000)
        said(L.pkx_beam_select_workspace(many, C.byref(n)))
        said(L.pkx_beam_select(many, A, n.value - 1, None))
        said(L.pkx_beam_select(many, None, 0, None))
        said(L.pkx_beam_select(beam(n_items=0), None, 0, None))
        S = pkx.BeamState
        def order(states, B=2, W=2, n=None):
            a = (S * max(len(states), 1))(*states)
            said(L.pkx_beam_reorder(A, B, W, a, len(states) if n is None else n, None))
        order([S(A, A + 64, 16, 16, 17)])
        order([S(A, A + 60, 16, 16, 16)])
        order([S(A, A + 64, 16, 16, 16), S(A + 1000, A + 50, 16, 16, 16)])
        order([S(None, A, 16, 16, 16)])
        order([], n=33)
        order([], W=0)
        order([S(A, A + 64, 16, 16, -1)])
        order([])
        order([S(None, None, 0, 0, 0)], B=0)
    """)
    words = ["type", "n_beams", "n_beams", "end_id", "end_id", "end_id", "end_id", "null", "null", "misaligned", "misaligned"]
    for line, w in zip(out[:11], words):
        assert line.startswith("1 ") and w in line, (line, w)
    assert out[11].strip() == "0" and "workspace" in out[12] and "workspace" in out[13] and out[14].strip() == "0"
    for line, w in zip(out[15:22], ("at least", "overlaps", "overlaps", "null", "at most", "bad size", "at least")):
        assert line.startswith("1 ") and w in line, (line, w)
    assert [x.strip() for x in out[22:]] == ["0"] * 2


def test_refusals_of_values_and_of_sizes_whose_products_wrap():
    """A scale that is not finite, rows of an output that lie in each other, and sizes whose products pass 64 bits."""
    out = _run("""
        top = (1 << 31) - 1
        for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(k_mask=A, k_mask_item=-1),
                   dict(out_item=64, out_row=64, out_head=64), dict(out_item=256, out_row=256, out_head=64), dict(out_row=192),
                   dict(n_items=top, n_q=top, n_heads=top, n_kv_heads=top, out_item=1 << 62, out_row=1 << 40)):
            said(L.pkx_cross_attention(cross(**kw), None, 0, None))
        n = C.c_size_t()
        said(L.pkx_cross_attention_workspace(cross(n_items=top, n_q=top, n_heads=top, n_kv_heads=top), C.byref(n)))
        for kw in (dict(scale=float("nan")), dict(out_row=64, out_tok=64, out_head=64)):
            said(L.pkx_cache8_attention(cache(), attn(n_q=2, **kw), None, 0, None))
        said(L.pkx_cache8_append(cache(), toks(n_rows=1, n_new=top), None))
        said(L.pkx_cache8_read(cache(), top, top, A, A, A, A, None))
        said(L.pkx_cache8_read(cache(n_kv_heads=top, n_slots=1), 1, top, A, A, A, A, None))
        said(L.pkx_beam_reorder(A, top, top, (pkx.BeamState * 1)(pkx.BeamState(A, A, 1 << 60, 1 << 60, 16)), 1, None))
    """)
    words = ["scale", "scale", "scale", "k_mask", "overlap", "overlap", "overlap", "2^22", "2^22", "scale", "overlap", "2^22", "2^30",
             "2^30", "too many"]
    assert len(out) == len(words)
    for line, w in zip(out, words):
        assert line.startswith("1 ") and w in line, (line, w)


def test_binding_refuses_strides_it_would_not_pass_on():
    out = _run("""
        import numpy as np
        class V:
            def __init__(self, shape, dtype=np.float32, strides=None):
                self.ptr, self.shape, self.dtype, self.strides = A, shape, np.dtype(dtype), strides
        q, kv, n = V((2, 1, 4, 64)), V((2, 9, 2, 64)), V((2,), np.int32)
        cache = pkx.Cache8.wrap(*(V((2, 2, 96, 64), np.int8) for _ in range(2)), *(V((2, 2, 3)) for _ in range(2)))
        sel = lambda x, s=None: pkx.BeamSelect(x, s or V((2, 4)), *(V((2, 4), np.int32) for _ in range(2)), V((2, 4)))
        for f in (lambda: pkx.CrossAttention(q, kv, kv, V((2, 1, 4, 64), strides=(512, 512, 128, 2))),
                  lambda: pkx.CrossAttention(q, kv, kv, q, k_len=V((2,), np.int32, (2,))),
                  lambda: sel(V((2, 4, 50), strides=(400, 50, 1))),
                  lambda: sel(V((2, 4, 50)), V((2, 4), strides=(8, 1))),
                  lambda: pkx.CacheAppend(cache, q, q, n),
                  lambda: pkx.CacheAttention(cache, q, q, n, table=V((2, 95), np.int32, (200, 1))),
                  lambda: pkx.BeamReorder(V((1, 2), np.int32), [(V((2, 6)), V((2, 6), strides=(8, 1)))])):
            try:
                f()
                print("taken")
            except pkx.PkxError as e:
                print("refused", e)
        a = pkx.CrossAttention(q, kv, kv, q, k_mask=V((2, 9), np.uint8, (16, 1)))._keep[0]
        b = sel(V((2, 4, 50), strides=(256, 64, 1)))._keep[0]
        c = pkx.CacheAttention(cache, q, q, n, table=V((2, 50), np.int32, (77, 1)), max_len=50)._keep[1]
        print(a.k_mask_item, b.logits_row, c.table_row)
    """)
    assert len(out) == 8 and all(x.startswith("refused") for x in out[:7]), out
    assert out[7] == "16 64 77"


def test_workspace_follows_the_sizes():
    """No workspace where the rows fill the chip; with few rows and many keys partial sums for every split."""
    out = _run("""
        n = C.c_size_t()
        for kw in (dict(n_items=1, n_q=1, n_k=100), dict(n_items=1, n_q=1, n_k=40000), dict(n_items=64, n_q=400, n_k=40000)):
            L.pkx_cross_attention_workspace(cross(**kw), C.byref(n)); print(n.value)
    """)
    assert int(out[0]) == 0 and int(out[1]) > 0 and int(out[2]) == 0


def test_restated_append_keeps_the_values():
    """The restatement itself: a value is at most half a step of its final block scale off per requantisation."""
    rng = np.random.default_rng(1)
    ints, sc = np.zeros((1, 1, 64, 16), np.int8), np.zeros((1, 1, 2), np.float32)
    x = (rng.standard_normal((1, 40, 1, 16)) * np.linspace(0.1, 3, 40)[None, :, None, None]).astype(np.float32)
    for t in range(40):
        ref.append(ints, sc, x[:, t:t + 1], [0], [t], [1])
    y = ref.values(ints, sc, np.zeros(40, int), np.arange(40))
    # the scale rises at most 31 times in a block, each time half a step of the new scale
    step = sc[0, 0][np.arange(40) // 32][:, None, None]
    assert np.all(np.abs(y - x[0]) <= step * 16)
    assert np.abs(y - x[0]).mean() < step.max()
