"""Refusals and host functions of the operators around a decoder's attention, which
need no GPU: every check comes before the first device call.  The library is
exercised in a subprocess so this process never loads a HIP runtime."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import block_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "parakeet.cpp_amd", "build", "libpkx.so")

# addresses that nothing may follow: the calls have to fail (or do nothing) before the device
PRE = """
import ctypes as C, math, pkx
L = pkx.lib()
MB = 1 << 20
def said(rc):
    print(rc, L.pkx_last_error().decode())
def make(cls, base, kw):
    a = cls()
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return a
def norm(**kw):
    return make(pkx.BlockNormArgs, dict(type=1, x_type=0, d=64, n_rows=4, x=MB, x_row=64, y=2 * MB, y_row=64, rows_per_gate=1, alpha=1.0,
                pre=2, pre_eps=1e-5, x_out=3 * MB, x_out_row=64, h=4 * MB, h_row=64), kw)
def lin(**kw):
    return make(pkx.LinearI8Args, dict(x_type=24, type=1, n_rows=4, n_out=64, n_in=48, x=MB, x_row=48, x_scale=2 * MB, w=3 * MB, w_scale=4 * MB,
                alpha=1.0, y=5 * MB, y_row=64), kw)
def rot(parts, **kw):
    a = make(pkx.RotaryArgs, dict(type=1, n_rows=2, n_tok=3, d_head=64, rot=32, mult=1.0, freq=9 * MB, n_parts=len(parts)), kw)
    for i, p in enumerate(parts[:4]):
        a.part[i] = pkx.RotaryPart(*p)
    return a
def part(src=MB, dst=2 * MB, **kw):
    p = dict(zip(("src", "src_row", "src_tok", "src_head", "dst", "dst_row", "dst_tok", "dst_head", "n_heads"),
                 (src, 768, 256, 64, dst, 768, 256, 64, 4)), **kw)
    return tuple(p.values())
def rules(**kw):
    return make(pkx.LogitRulesArgs, dict(type=0, n_rows=4, vocab=100, logits=MB, logits_row=100, out=2 * MB, out_row=100, tokens=3 * MB, n_slots=4,
                capacity=50, len=4 * MB), kw)
"""


def _run(code, **env):
    if not os.path.exists(LIB):
        pytest.skip("libpkx.so not built")
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "parakeet.cpp_amd", "python"), **env)
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(PRE) + textwrap.dedent(code)], capture_output=True, text=True,
                       env=env, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout.strip("\n").split("\n")


def _refused(lines, words):
    assert len(lines) == len(words), lines
    for line, w in zip(lines, words):
        assert line.startswith("1 ") and w in line, (line, w)


def test_block_norm_refusals():
    out = _run("""
        nan = float("nan")
        cases = [dict(type=8), dict(x_type=24), dict(type=0, x_type=1), dict(n_rows=-1), dict(n_rows=1 << 22), dict(d=0), dict(d=16385), dict(post=3),
                 dict(pre=-1), dict(gate_fn=2), dict(pre_eps=-1.0), dict(post_eps=nan), dict(alpha=math.inf), dict(x=None, y=None),
                 dict(x_out=None, h=None, pre=0), dict(gate=5 * MB, gate_row=64, rows_per_gate=0), dict(y=None, gate=5 * MB, gate_row=64),
                 dict(post_w=5 * MB), dict(pre=0, pre_b=5 * MB), dict(y=None, post=1), dict(h=None), dict(h_i8=1), dict(x=MB + 2),
                 dict(y_row=-1), dict(h_row=63), dict(x_out_row=0),
                 # overlaps: shifted by a row, an output on a weight, the outputs on each other, h in 8 bits over y
                 dict(x_out=MB + 64 * 4), dict(h=2 * MB + 2), dict(pre_w=4 * MB), dict(h=3 * MB), dict(h_i8=1, h_scale=5 * MB, h=2 * MB),
                 dict(h=MB, h_row=128), dict(h_i8=1, h_scale=MB + 8)]
        for kw in cases:
            said(L.pkx_block_norm(norm(**kw), None))
        said(L.pkx_block_norm(None, None))
        for kw in (dict(n_rows=0), dict(n_rows=0, x=None, x_out=None)):
            said(L.pkx_block_norm(norm(**kw), None))
    """)
    words = ["type", "x_type", "f16 x", "negative", "2^22", "d must", "d must", "post and pre", "post and pre", "gate_fn", "eps", "eps", "alpha",
             "neither x", "neither x_out", "gate needs", "gate needs", "post without", "pre without", "post without", "pre without", "8 bits",
             "x is", "y is", "h is", "x_out is", "overlaps an input", "overlaps an input", "overlaps a weight", "outputs overlap",
             "overlaps an input", "overlaps an input", "overlaps an input", "null"]
    _refused(out[:-2], words)
    assert [x.strip() for x in out[-2:]] == ["0"] * 2


def test_quantise_and_weight_refusals():
    out = _run("""
        q = lambda type=1, x=MB, xr=64, M=4, n=64, o=2 * MB, qr=64, s=3 * MB: said(L.pkx_quantize_rows(type, x, xr, M, n, o, qr, s, None))
        q(type=8); q(M=-1); q(M=1 << 22); q(n=-1); q(x=None); q(x=MB + 1); q(xr=-64); q(qr=63); q(o=None); q(s=None); q(s=3 * MB + 2); q(o=MB + 100); q(s=MB)
        q(s=2 * MB + 64)
        n = C.c_size_t()
        said(L.pkx_i8_weight_bytes(8, 0, C.byref(n))); said(L.pkx_i8_weight_bytes(8, 131072, C.byref(n))); said(L.pkx_i8_weight_bytes(-1, 8, C.byref(n)))
        said(L.pkx_i8_weight_bytes(1 << 22, 8, C.byref(n))); said(L.pkx_i8_weight_bytes(4000000, 131071, C.byref(n))); said(L.pkx_i8_weight_bytes(8, 8, None))
        w = lambda w=MB, r=64, N=8, K=64, p=2 * MB: said(L.pkx_i8_weight_pack(w, r, N, K, p, None))
        w(w=None); w(r=-1); w(p=None); w(p=2 * MB + 8); w(p=MB + 64)
        q(M=0, x=None, o=None, s=None); w(N=0, w=None)
        for N, K in ((1, 1), (32, 128), (33, 129), (0, 5)):
            L.pkx_i8_weight_bytes(N, K, C.byref(n)); print(n.value)
    """)
    _refused(out[:25], ["type", "negative", "2^22", "negative", "x is", "x is", "x is", "q is", "q is", "scale is", "scale is", "overlaps", "overlaps",
                        "overlaps", "n_in", "n_in", "n_out", "n_out", "32 GiB", "null", "w is", "w is", "packed is", "packed is", "overlaps"])
    assert [x.strip() for x in out[25:27]] == ["0"] * 2
    assert [int(x) for x in out[27:]] == [32 * 128, 32 * 128, 64 * 256, 0]


def test_linear_refusals():
    out = _run("""
        nan = float("nan")
        cases = [dict(x_type=8), dict(type=24), dict(n_rows=-1), dict(n_in=0), dict(n_in=131072), dict(n_out=1 << 22), dict(n_rows=1 << 20, n_out=1 << 20),
                 dict(act=2), dict(alpha=nan), dict(w=None), dict(w=MB + 8), dict(w_scale=None), dict(bias=MB + 2), dict(y=None), dict(y=5 * MB + 1),
                 dict(y_row=63), dict(add=6 * MB + 1, add_row=64), dict(add=5 * MB + 64, add_row=64), dict(add=5 * MB, add_row=0), dict(y=3 * MB), dict(y=4 * MB),
                 dict(bias=5 * MB), dict(x=None), dict(x=MB + 8), dict(x_row=40), dict(x_row=32), dict(x_row=1 << 22), dict(x_scale=None), dict(y=MB), dict(y=2 * MB)]
        for kw in cases:
            said(L.pkx_linear_i8(lin(**kw), None, 0, None))
        said(L.pkx_linear_i8(None, None, 0, None))
        n = C.c_size_t()
        f = dict(x_type=1, x_scale=None, n_rows=100, n_in=4000, x_row=4000)
        said(L.pkx_linear_i8_workspace(lin(**f), C.byref(n)))
        said(L.pkx_linear_i8(lin(x_type=1), 7 * MB, 1 << 20, None))
        said(L.pkx_linear_i8(lin(**f), None, 0, None))
        said(L.pkx_linear_i8(lin(**f), 7 * MB + 4, 1 << 20, None))
        said(L.pkx_linear_i8(lin(**f), 7 * MB, n.value - 1, None))
        said(L.pkx_linear_i8(lin(x=MB + 1, **f), 7 * MB, 1 << 20, None))
        said(L.pkx_linear_i8(lin(y=MB, **f), 7 * MB, 1 << 20, None))
        said(L.pkx_linear_i8_workspace(lin(), None))
        for kw in (dict(n_rows=0), dict(n_out=0, y=None)):
            said(L.pkx_linear_i8(lin(**kw), None, 0, None))
        print(n.value)
        L.pkx_linear_i8_workspace(lin(), C.byref(n)); print(n.value)
    """)
    _refused(out[:31], ["x_type", "type", "negative", "n_in", "n_in", "n_out", "2^36", "act", "alpha", "w is", "w is", "w_scale", "bias", "y is", "y is",
                        "y is", "add is", "overlaps add", "overlaps add", "overlaps the weights", "overlaps the weights", "overlaps the weights", "x is", "x is",
                        "x is", "x is", "x_row", "x_scale", "overlaps x", "overlaps x", "null"])
    assert out[31].strip() == "0"
    _refused(out[32:39], ["x_scale", "workspace", "workspace", "workspace", "x is", "overlaps x", "null"])
    assert [x.strip() for x in out[39:41]] == ["0"] * 2
    assert int(out[41]) >= 100 * 4000 + 400 and int(out[42]) == 0


def test_rotary_refusals():
    out = _run("""
        S = 24 * 64
        qkv = lambda i, o=MB: dict(src=o + i * 2 * 64 * 2, src_row=3 * 3 * 2 * 64, src_tok=3 * 2 * 64, src_head=64, n_heads=2)
        dst = lambda i, o=MB: dict(dst=o + i * 2 * 64 * 2, dst_row=3 * 3 * 2 * 64, dst_tok=3 * 2 * 64, dst_head=64)
        for p, kw in (([part()], dict(type=24)), ([part()], dict(n_rows=-1)), ([part()], dict(d_head=0)), ([part()], dict(d_head=513)), ([part()], dict(rot=31)),
                      ([part()], dict(rot=66)), ([part()] * 5, {}), ([part()], dict(mult=math.nan)), ([part()], dict(pos=MB, pos_row=-1)),
                      ([part(n_heads=-1)], {}), ([part(n_heads=4097)], {}), ([part()], dict(freq=None)), ([part()], dict(freq=9 * MB + 4)),
                      ([part(src=None)], {}), ([part(dst=2 * MB + 1)], {}), ([part(src_tok=-1)], {}), ([part(dst_tok=192)], {}),
                      ([part(dst=MB + 128)], {}), ([part(), part(src=3 * MB)], {}), ([part(dst=9 * MB)], {}), ([part()], dict(start=2 * MB)),
                      # queries turned onto the keys beside them
                      ([part(**qkv(0), **dst(1)), part(**qkv(1), **dst(2))], {}),
                      ([part(dst_row=768, dst=MB, src_row=1536)], {}),
                      # in place, but transposed
                      ([part(dst=MB, src_row=192, src_tok=64, src_head=576, dst_row=64, dst_tok=192, dst_head=576)], dict(n_rows=3, n_tok=3))):
            said(L.pkx_rotary(rot(p, **kw), None))
        said(L.pkx_rotary(None, None))
        f = (C.c_double * 8)()
        for a in ((0.0, 16, 1, 0, 1, 32), (1e4, 15, 1, 0, 1, 32), (1e4, 514, 1, 0, 1, 32), (1e4, 16, 0, 0, 1, 32), (1e4, 16, 2, -1, 1, 32), (1e4, 16, 2, 100, 3, 3),
                  (math.inf, 16, 1, 0, 1, 32)):
            said(L.pkx_rotary_frequencies(*a, f))
        said(L.pkx_rotary_frequencies(1e4, 16, 1, 0, 1, 32, None))
        for kw in (dict(n_rows=0), dict(n_tok=0), dict(n_rows=0, freq=None)):
            said(L.pkx_rotary(rot([part()], **kw), None))
    """)
    _refused(out[:33], ["type", "negative", "d_head", "d_head", "rot must", "rot must", "at most", "mult", "pos", "heads", "heads", "freq", "freq", "null or", "null or",
                        "negative stride", "overlap", "overlaps a src", "two dsts", "overlaps freq", "overlaps start", "overlaps a src", "overlaps a src", "overlaps a src", "null",
                        "base", "rot must", "rot must", "factor", "context", "high", "base", "null"])
    assert [x.strip() for x in out[33:]] == ["0"] * 3


def test_logit_rules_refusals():
    out = _run("""
        cases = [dict(type=24), dict(n_rows=-1), dict(vocab=-1), dict(window=-1), dict(vocab=(1 << 22) + 1), dict(logits=None), dict(logits=MB + 2), dict(logits_row=-1),
                 dict(out=None), dict(out_row=99), dict(out=MB + 4), dict(out=MB, out_row=200), dict(n_slots=0), dict(capacity=-1), dict(capacity=(1 << 30) + 1), dict(len=None), dict(n_slots=3),
                 dict(table=5 * MB, table_row=49), dict(out=3 * MB), dict(out=4 * MB), dict(slot=2 * MB), dict(repetition=2 * MB + 400),
                 dict(bias=5 * MB + 2, bias_row=100, n_bias=1), dict(bias=5 * MB, bias_row=-1, n_bias=1), dict(bias=2 * MB, bias_row=100, n_bias=1),
                 dict(bias=5 * MB, bias_row=100, n_bias=1, bias_index=2 * MB), dict(mask=5 * MB, mask_row=4, n_mask=-1), dict(mask=2 * MB, mask_row=4, n_mask=1),
                 dict(mask=5 * MB, mask_row=4, n_mask=1, mask_index=2 * MB), dict(n_slots=(1 << 31) - 1, capacity=1 << 30)]
        for kw in cases:
            said(L.pkx_logit_rules(rules(**kw), None))
        said(L.pkx_logit_rules(None, None))
        for kw in (dict(n_rows=0), dict(vocab=0, logits=None)):
            said(L.pkx_logit_rules(rules(**kw), None))
    """)
    _refused(out[:31], ["type", "negative", "negative", "negative", "2^22", "logits are", "logits are", "logits are", "out is", "out is", "overlaps logits", "overlaps logits",
                        "no slots", "no slots", "2^30", "null len", "more rows", "shorter", "overlaps the tokens", "overlaps the tokens", "overlaps the tokens", "overlaps a penalty",
                        "bias is", "bias is", "overlaps bias", "overlaps bias_index", "mask is", "overlaps mask", "overlaps mask_index", "address space", "null"])
    assert [x.strip() for x in out[31:]] == ["0"] * 2


def test_operands_side_by_side_are_taken():
    """Columns of the same rows and in-place operands are no overlaps: the calls get past every check, to the missing device."""
    out = _run("""
        qkv = lambda i: dict(src=MB + i * 256, src_row=1152, src_tok=384, src_head=64, n_heads=2, dst=MB + i * 256, dst_row=1152, dst_tok=384, dst_head=64)
        s = None
        print(L.pkx_rotary(rot([part(**qkv(0)), part(**qkv(1))]), s), "overlap" in L.pkx_last_error().decode())
        print(L.pkx_block_norm(norm(x_out=MB, h=2 * MB), s), "overlap" in L.pkx_last_error().decode())
        print(L.pkx_block_norm(norm(x_type=1, x_row=192, y=MB + 128, y_row=192, x_out=MB, x_out_row=192, h=MB + 256, h_row=192), s), "overlap" in L.pkx_last_error().decode())
        print(L.pkx_linear_i8(lin(add=5 * MB, add_row=64), None, 0, s), "overlap" in L.pkx_last_error().decode())
        print(L.pkx_logit_rules(rules(out=MB), s), "overlap" in L.pkx_last_error().decode())
    """, HIP_VISIBLE_DEVICES="-1")
    assert out == ["1 False"] * 5


def test_binding_refusals():
    out = _run("""
        import numpy as np
        class V:
            def __init__(self, shape, dtype=np.float32, strides=None):
                self.ptr, self.shape, self.dtype, self.strides = MB, shape, np.dtype(dtype), strides
        x, i8, s = V((4, 64)), V((4, 64), np.int8), V((4,))
        w = pkx.WeightI8.__new__(pkx.WeightI8)
        w.shape, w.scale, w.packed = (32, 64), V((32,)), V((4096,), np.uint8)
        q = V((2, 3, 4, 64))
        for f in (lambda: pkx.BlockNorm(), lambda: pkx.BlockNorm(x, V((4, 63))), lambda: pkx.BlockNorm(x, x, pre="batch"), lambda: pkx.BlockNorm(x, i8),
                  lambda: pkx.BlockNorm(x, x, h_scale=s), lambda: pkx.BlockNorm(x, x, y=x, gate=V((3, 64))), lambda: pkx.BlockNorm(x, x, pre="rms", pre_w=V((63,))),
                  lambda: pkx.BlockNorm(x, x, y=x, gate=x, gate_fn="tanh"), lambda: pkx.QuantizeRows(x, V((4, 65), np.int8), s), lambda: pkx.QuantizeRows(i8, i8, s),
                  lambda: pkx.LinearI8(x, w, V((4, 31))), lambda: pkx.LinearI8(i8, w, V((4, 32))), lambda: pkx.LinearI8(x, w, V((4, 32)), x_scale=s),
                  lambda: pkx.LinearI8(V((4, 60)), w, V((4, 32))), lambda: pkx.LinearI8(x, w, V((4, 32)), act="relu"),
                  lambda: pkx.Rotary(V((16,)), [(q, q)]), lambda: pkx.Rotary(V((16,), np.float64), []),
                  lambda: pkx.Rotary(V((16,), np.float64), [(q, V((2, 3, 3, 64)))]), lambda: pkx.Rotary(V((16,), np.float64), [(q, q)], start=V((3,), np.int32)),
                  lambda: pkx.LogitRules(x, V((4, 60))), lambda: pkx.LogitRules(x, x, mask=V((2, 3), np.int32)), lambda: pkx.LogitRules(x, x, bias=V((2, 60))),
                  lambda: pkx.LogitRules(x, x, tokens=V((4, 9), np.int32), length=V((4,), np.int32), table=V((4, 8), np.int32))):
            try:
                f()
                print("taken")
            except pkx.PkxError as e:
                print("refused", e)
        a = pkx.LinearI8(V((4, 64), np.int8, (80, 1)), w, V((4, 32), np.float16, (48, 1)), x_scale=s)._keep[0]
        print(a.x_row, a.y_row, a.x_type, a.type)
    """)
    assert len(out) == 24 and all(x.startswith("refused") for x in out[:23]), out
    assert out[23] == "80 48 24 1"


def test_rotary_frequencies():
    out = _run("""
        for kw in (dict(), dict(factor=4.0), dict(factor=8.0, context=8192, low=1.0, high=32.0)):
            print(*(x.hex() for x in pkx.rotary_frequencies(64, 5e5, **kw).tolist()))
    """)
    got = [np.array([float.fromhex(x) for x in line.split()]) for line in out]
    f = 5e5 ** (-np.arange(32) / 32.0)
    keep = np.clip((8192 * f / (2 * np.pi) - 1) / 31, 0, 1)
    for g, want in zip(got, (f, f / 4, f * (keep + (1 - keep) / 8))):
        assert np.allclose(g, want, rtol=1e-14, atol=0)
    assert got[2][0] == f[0] and np.isclose(got[2][-1], f[-1] / 8, rtol=1e-14)


def test_restated_quantising():
    """The restatement: a held value is at most half a step off, and what is not finite does not set the scale."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 40)).astype(np.float32)
    x[1] = 0
    x[2, :3] = np.nan, np.inf, -np.inf
    q, s = ref.quantised(x)
    fine = np.isfinite(x)
    assert np.all(np.abs(q * s[:, None] - x)[fine] <= (0.5 + 2.0 ** -16) * np.broadcast_to(s[:, None], x.shape)[fine])
    assert s[1] == 0 and not q[1].any() and q[2, :3].tolist() == [0, 127, -127]
