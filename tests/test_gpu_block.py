"""The operators around a decoder's attention (block norm, 8-bit rows and products,
rotary positions, rules on logits) against float64 restatements (block_ref.py):
every element within a bound derived from the roundings the kernels make; what is
held in 8 bits exactly."""
import ctypes as C

import numpy as np
import pytest

import block_ref as ref
import decoder_ref

pytestmark = pytest.mark.gpu
NAN = float("nan")
DT = {"f16": np.float16, "f32": np.float32}


def dev(gpu, a, stream):
    return None if a is None else gpu.DeviceArray.from_numpy(np.ascontiguousarray(a), stream)


def i32(x):
    return np.asarray(x, np.int32)


class View:
    """A strided part of a device array, for the binding: strides in elements."""

    def __init__(self, base, offset, shape, strides):
        self.base, self.shape, self.dtype, self.strides = base, tuple(shape), base.dtype, tuple(strides)
        self.ptr = base.ptr + offset * base.dtype.itemsize


def check(got, want, err, f16, label):
    """Within the bound; infinities and NaN where the restatement has them."""
    want, got = np.asarray(want, np.float64), got.astype(np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), label
    bound = ref.rounded(np.asarray(err)[fine], want[fine], f16)
    off = np.abs(got[fine] - want[fine])
    worst = float((off / bound).max(initial=0))
    print(f"[{label}] largest error {off.max(initial=0):.2e}, {worst:.2f} of its bound", flush=True)
    assert np.isfinite(got[fine]).all() and worst <= 1.0, label


# ---- block norm -----------------------------------------------------------------
NORM = [
    # type, x type, rows, d, post, pre, gate rows (0: none), gate fn
    ("f16", "f16", 1, 1024, "none", "rms", 0, "linear"), ("f16", "f32", 5, 1000, "layer", "layer", 2, "linear"),
    ("f32", "f32", 3, 4090, "rms", "rms", 1, "sigmoid"), ("f16", "f16", 7, 8, "rms", "layer", 3, "sigmoid"),
    ("f32", "f32", 2, 1, "none", "layer", 0, "linear"), ("f16", "f32", 2, 1, "rms", "rms", 1, "linear"),
    ("f32", "f32", 130, 7, "layer", "rms", 130, "linear"), ("f16", "f32", 9, 63, "none", "none", 4, "sigmoid"),
    ("f16", "f16", 4, 512, "layer", "rms", 1, "linear"), ("f32", "f32", 6, 513, "rms", "layer", 0, "linear"),
    ("f16", "f32", 3, 1025, "layer", "rms", 1, "sigmoid"), ("f32", "f32", 3, 2048, "layer", "layer", 3, "linear"),
    ("f16", "f16", 2, 2049, "rms", "rms", 0, "linear"), ("f16", "f32", 2, 4096, "rms", "layer", 1, "sigmoid"),
    ("f32", "f32", 2, 4097, "layer", "rms", 2, "linear"), ("f16", "f16", 3, 8192, "none", "layer", 1, "linear"),
    ("f32", "f32", 2, 8201, "layer", "layer", 1, "sigmoid"), ("f16", "f32", 2, 16383, "rms", "rms", 0, "linear"),
    ("f32", "f32", 2, 16384, "layer", "rms", 1, "linear"), ("f16", "f16", 1000, 257, "rms", "layer", 125, "sigmoid"),
    ("f16", "f32", 37, 128, "layer", "layer", 5, "sigmoid"), ("f32", "f32", 18, 129, "layer", "rms", 1, "linear"), ("f16", "f16", 5003, 64, "none", "rms", 0, "linear"),
    ("f16", "f16", 11, 256, "rms", "layer", 0, "linear"), ("f32", "f32", 2049, 150, "layer", "layer", 2049, "sigmoid"), ("f16", "f32", 6, 240, "layer", "layer", 1, "linear"),
    ("f32", "f32", 1100, 500, "rms", "layer", 1, "linear"), ("f16", "f32", 600, 1000, "layer", "rms", 600, "sigmoid"), ("f32", "f32", 300, 1030, "layer", "layer", 0, "linear"),
    ("f32", "f32", 300, 2100, "layer", "rms", 1, "linear"), ("f16", "f16", 257, 4096, "rms", "layer", 2, "linear"), ("f16", "f32", 140, 5001, "layer", "layer", 7, "sigmoid"),
]


@pytest.mark.parametrize("type,xtype,M,d,post,pre,per,fn", NORM)
@pytest.mark.parametrize("i8", [False, True])
def test_block_norm(gpu, stream, type, xtype, M, d, post, pre, per, fn, i8):
    """Every norm, gate and width, a mean far from zero, rows of a large stride, in place."""
    print(f"[norm] {type} {xtype} M={M} d={d} {post} {pre} per={per} {fn} i8={i8}", flush=True)
    rng = np.random.default_rng(M * 7 + d)
    dt, dx = DT[type], DT[xtype]
    x = (3 * rng.standard_normal((M, d)) + 40 * rng.standard_normal((M, 1))).astype(dx)
    y = (rng.standard_normal((M, d)) + rng.standard_normal((M, 1)) * 10).astype(dt)
    gate = rng.standard_normal((-(-M // per), d)).astype(dt) if per else None
    vec = lambda on: (1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if on else None  # noqa: E731
    w = dict(post_w=vec(post != "none"), post_b=vec(post == "layer"), pre_w=vec(pre == "layer"), pre_b=vec(pre == "rms"))
    alpha, eps = 0.5 if M % 2 else -1.25, 1e-5
    pad = 5                                             # rows further apart than they are long, at odd alignments
    bx, by = np.full((M, d + pad), 7, dx), np.full((M, d + pad), 9, dt)
    bx[:, :d], by[:, :d] = x, y
    bx, by = dev(gpu, bx, stream), dev(gpu, by, stream)
    vx, vy = (View(b, 0, (M, d), (d + pad, 1)) for b in (bx, by))
    h = gpu.DeviceArray((M, d), np.int8) if i8 else vy   # in place: x_out is x, h is y
    hs = gpu.DeviceArray((M,), np.float32) if i8 else None
    wd = {k: dev(gpu, v, stream) for k, v in w.items()}
    gpu.BlockNorm(vx, h, y=vy, x_out=vx, post=post, pre=pre, gate=dev(gpu, gate, stream), rows_per_gate=max(per, 1), gate_fn=fn,
                  alpha=alpha, eps=eps, h_scale=hs, **wd)(stream)
    r, er, hh, eh = ref.block_norm(x, y, gate, max(per, 1), fn, alpha, post, w["post_w"], w["post_b"], pre, w["pre_w"], w["pre_b"], eps, eps)
    gx = bx.numpy(stream)
    check(gx[:, :d], r, er, xtype == "f16", "x_out")
    assert (gx[:, d:] == 7).all()
    if not i8:
        gy = by.numpy(stream)
        check(gy[:, :d], hh, eh, type == "f16", "h")
        assert (gy[:, d:] == 9).all()
        return
    q, s = h.numpy(stream).astype(np.float64), hs.numpy(stream).astype(np.float64)[:, None]
    top = np.abs(hh).max(1, keepdims=True)
    assert (np.abs(s - top / 127) <= eh.max(1, keepdims=True) / 127 + 2 * ref.U * s).all()
    assert (np.abs(q * s - hh) <= 0.5 * s * (1 + 2.0 ** -15) + eh + 128 * 2 * ref.U * s).all() and (np.abs(q) <= 127).all()


def test_block_norm_parts(gpu, stream):
    """Without a stream, without a block's output, without a norm, one output alone."""
    rng = np.random.default_rng(4)
    M, d = 3, 700
    x, y, g = (rng.standard_normal((M, d)).astype(np.float32) for _ in range(3))
    dx, dy, dg = (dev(gpu, a, stream) for a in (x, y, g))
    o, h = gpu.DeviceArray((M, d), np.float32), gpu.DeviceArray((M, d), np.float32)
    none = (None, None)
    for kw, args in ((dict(x=dx, h=h, pre="layer"), (x, None, None, 1, "linear", 1.0, "none", *none, "layer", *none)),
                     (dict(h=h, y=dy, post="rms", gate=dg, alpha=2.0), (None, y, g, 1, "linear", 2.0, "rms", *none, "none", *none)),
                     (dict(x=dx, y=dy, x_out=o, gate=dg, gate_fn="sigmoid"), (x, y, g, 1, "sigmoid", 1.0, "none", *none, "none", *none))):
        gpu.BlockNorm(**kw)(stream)
        r, er, hh, eh = ref.block_norm(*args, 1e-5, 1e-5)
        if "x_out" in kw:
            check(o.numpy(stream), r, er, False, "x_out")
        else:
            check(h.numpy(stream), hh, eh, False, "h")


@pytest.mark.parametrize("d", [1500, 100, 200, 500])
def test_block_norm_hard_rows(gpu, stream, d):
    """Rows of one value, of zeros, with a first element far out, of a mean 10^5 deviations away, of values whose squares pass f32,
    with a NaN or an infinity: each row by itself."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((8, d)).astype(np.float32)
    x[0], x[1] = 3.25, 0
    x[2, 0] = 1e6
    x[3] = x[3] + np.float32(1e5)
    x[4] *= np.float32(1e25)
    x[5] *= np.float32(1e-30)
    x[6, 77], x[7, 3] = NAN, np.inf
    for kind in ("layer", "rms"):
        h = gpu.DeviceArray(x.shape, np.float32)
        gpu.BlockNorm(dev(gpu, x, stream), h, pre=kind, eps=1e-5)(stream)
        got = h.numpy(stream)
        want = ref.normalised(x[:6].astype(np.float64), np.zeros((6, d)), kind, None, None, 1e-5)
        check(got[:6], *want, False, kind)
        assert np.isnan(got[6]).all() and np.isnan(got[7, 3])
    q, s = gpu.DeviceArray(x.shape, np.int8), gpu.DeviceArray((8,), np.float32)
    gpu.BlockNorm(dev(gpu, x, stream), q, h_scale=s)(stream)
    want = ref.quantised(x)
    assert np.array_equal(q.numpy(stream), want[0]) and np.array_equal(s.numpy(stream), want[1])


# ---- 8-bit rows and products ----------------------------------------------------
@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("M,n", [(1, 1), (5, 7), (3, 512), (9, 513), (2, 2048), (3, 2049), (2, 4100), (1, 16384), (2, 16385), (1, 50001), (2000, 24), (3, 8192), (2, 8193), (300, 5003)])
def test_quantize_rows(gpu, stream, type, M, n):
    """Bit for bit, with NaN, infinities, rows of zeros and of subnormal values; what lies between the rows stays."""
    rng = np.random.default_rng(M + n)
    x = (rng.standard_normal((M, n + 3)) * np.exp(rng.standard_normal((M, 1)))).astype(DT[type])
    if M > 2:
        x[1], x[2] = 0, x[2] * DT[type](2.0 ** -20)
    if n > 20:
        x[0, [1, 5, n - 1]] = NAN, np.inf, -np.inf
    q = dev(gpu, np.full((M, n + 2), 99, np.int8), stream)
    s = gpu.DeviceArray((M,), np.float32)
    gpu.QuantizeRows(View(dev(gpu, x, stream), 1, (M, n), (n + 3, 1)), View(q, 0, (M, n), (n + 2, 1)), s)(stream)
    want = ref.quantised(x[:, 1:n + 1])
    got = q.numpy(stream)
    assert np.array_equal(got[:, :n], want[0]) and (got[:, n:] == 99).all()
    assert np.array_equal(s.numpy(stream), want[1])


LINEAR = [
    # type, M, N, K, act, bias, add
    ("f16", 1, 4096, 1024, "silu", True, False), ("f32", 1, 1, 1, "none", False, False), ("f16", 3, 33, 17, "none", True, True),
    ("f32", 16, 64, 128, "silu", False, True), ("f16", 17, 50, 130, "none", True, False), ("f32", 2, 1025, 700, "none", True, True),
    ("f16", 64, 1024, 4096, "none", True, True), ("f16", 65, 100, 300, "silu", True, False), ("f32", 100, 33, 1000, "none", False, False),
    ("f16", 128, 256, 64, "none", False, True), ("f32", 129, 129, 129, "silu", True, True), ("f16", 300, 1000, 257, "none", True, False),
    ("f16", 700, 4096, 512, "silu", True, False), ("f32", 2000, 777, 96, "none", True, True), ("f16", 3500, 4100, 272, "none", False, False),
    ("f32", 4097, 4095, 16, "none", True, False), ("f16", 40, 8193, 320, "none", False, False), ("f16", 257, 2, 131071, "none", False, False),
    ("f32", 5, 3, 131071, "none", False, False), ("f16", 2000, 4096, 130, "silu", True, False), ("f32", 1990, 4000, 100, "none", False, True),
    ("f32", 6, 500, 1500, "silu", True, False), ("f16", 3, 40, 2048, "none", True, True), ("f32", 41, 100, 1000, "none", True, False), ("f16", 64, 500, 33, "silu", False, True), ("f16", 130, 1000, 640, "none", False, False),
]


@pytest.mark.parametrize("type,M,N,K,act,bias,add", LINEAR)
@pytest.mark.parametrize("tokens", ["f", "i8"])
def test_linear_i8(gpu, stream, type, M, N, K, act, bias, add, tokens):
    """Tokens quantised within the call and given in 8 bits (rows further apart, anything behind their ends), every tail."""
    print(f"[linear] {type} M={M} N={N} K={K} {act} bias={bias} add={add} {tokens}", flush=True)
    rng = np.random.default_rng(M + 3 * N + K)
    w, ws = rng.integers(-127, 128, (N, K)).astype(np.int8), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    a = rng.standard_normal((M, N + 1)).astype(DT[type]) if add else None
    wd = gpu.WeightI8(dev(gpu, w, stream), dev(gpu, ws, stream), stream)
    y = dev(gpu, np.full((M, N + 3), 5, DT[type]), stream)
    vy = View(y, 0, (M, N), (N + 3, 1))
    va = View(dev(gpu, a, stream), 1, (M, N), (N + 1, 1)) if add else None
    kw = dict(bias=dev(gpu, b, stream), act=act, add=va, alpha=0.5 if add else 1.0)
    if tokens == "f":
        x = rng.standard_normal((M, K)).astype(DT[type])
        q, s = ref.quantised(x)
        gpu.LinearI8(dev(gpu, x, stream), wd, vy, **kw)(stream)
    else:
        row = (K + 15) // 16 * 16 + (16 if M > 1 else 0)
        big = rng.integers(-128, 128, (M, row)).astype(np.int8)
        q, s = big[:, :K], rng.uniform(0.001, 0.05, M).astype(np.float32)
        gpu.LinearI8(View(dev(gpu, big, stream), 0, (M, K), (row, 1)), wd, vy, x_scale=dev(gpu, s, stream), **kw)(stream)
    want, err = ref.linear_i8(q, s, w, ws, b, act, kw["alpha"], a[:, 1:] if add else None, type == "f16")
    got = y.numpy(stream)
    check(got[:, :N], want, err, type == "f16", "y")
    assert (got[:, N:] == 5).all()


def test_linear_i8_extremes(gpu, stream):
    """The largest sums, in place over what is added, weights quantised by the binding, scales of zero."""
    K = 131071
    x, w = np.full((2, K), -128, np.int8), np.full((33, K), -128, np.int8)
    w[1::2] = 127
    x[1] = 127
    one = np.ones(33, np.float32)
    wd = gpu.WeightI8(dev(gpu, w, stream), dev(gpu, one, stream), stream)
    y = dev(gpu, np.ones((2, 33), np.float32), stream)
    xb = np.zeros((2, K + 1), np.int8)
    xb[:, :K] = x
    gpu.LinearI8(View(dev(gpu, xb, stream), 0, (2, K), (K + 1, 1)), wd, y, x_scale=dev(gpu, np.float32([1, 0]), stream), add=y)(stream)
    got = y.numpy(stream)
    sums = -128.0 * np.where(np.arange(33) % 2, 127, -128) * K
    assert np.array_equal(got[0], np.float32(1) + sums.astype(np.float32)) and (got[1] == 1).all()
    rng = np.random.default_rng(8)
    wf, xf = rng.standard_normal((70, 200)).astype(np.float32), rng.standard_normal((5, 200)).astype(np.float32)
    wq, ws = ref.quantised(wf)
    q, s = ref.quantised(xf)
    y = gpu.DeviceArray((5, 70), np.float32)
    gpu.LinearI8(dev(gpu, xf, stream), gpu.WeightI8.quantize(dev(gpu, wf, stream), stream), y)(stream)
    check(y.numpy(stream), *ref.linear_i8(q, s, wq, ws, None, "none", 1.0, None), False, "quantised weights")
    # SiLU of what f32 and f16 hold at their ends
    v = np.float32([np.inf, -np.inf, np.nan, 1e38, -1e38, 200, -200, 88.5, -88.5, 0, -0.0, 1e-30, -103, -87.4, -88.1, 60])
    wd = gpu.WeightI8(dev(gpu, np.zeros((16, 16), np.int8), stream), dev(gpu, np.ones(16, np.float32), stream), stream)
    for dt in (np.float32, np.float16):
        for rows in (1, 40):
            y = gpu.DeviceArray((rows, 16), dt)
            gpu.LinearI8(dev(gpu, np.ones((rows, 16), np.float32), stream), wd, y, bias=dev(gpu, v, stream), act="silu")(stream)
            got = y.numpy(stream)
            with np.errstate(all="ignore"):
                want = v.astype(np.float64) / (1 + np.exp(-v.astype(np.float64)))
                lost = np.abs(want) * 6 * ref.U + 1.2e-38        # subnormal results may be zeros
                if dt == np.float16:
                    want, lost = np.where(np.abs(want) > 65519, np.copysign(np.inf, want), want), lost + 2.0 ** -23 * np.abs(v * want)
            for r in range(rows):
                check(got[r], want, np.where(np.isfinite(want), lost, 0), dt == np.float16, "silu")


# ---- far apart ------------------------------------------------------------------
def _put(gpu, stream, base, at, a):
    a = np.ascontiguousarray(a)
    gpu.check(gpu.lib().pkx_memcpy_h2d(base.ptr + at * base.dtype.itemsize, a.ctypes.data, a.nbytes, stream.handle))


def _get(gpu, stream, base, at, shape):
    a = np.empty(shape, base.dtype)
    gpu.check(gpu.lib().pkx_memcpy_d2h(a.ctypes.data, base.ptr + at * base.dtype.itemsize, a.nbytes, stream.handle))
    return a


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_far_rows(gpu, stream, type):
    """Rows 2^31 elements apart: norm in place, quantised, products with what is added, logits."""
    rng = np.random.default_rng(40)
    dt, far, d, N = DT[type], 1 << 31, 300, 70
    big = gpu.DeviceArray((2 * far + d,), dt)
    x = rng.standard_normal((3, d)).astype(dt)
    view = lambda n: View(big, 0, (3, n), (far, 1))  # noqa: E731

    def fill(a):
        for r in range(3):
            _put(gpu, stream, big, r * far, a[r])

    def rows(n):
        return np.stack([_get(gpu, stream, big, r * far, (n,)) for r in range(3)])

    fill(x)
    h, y = gpu.DeviceArray((3, d), dt), rng.standard_normal((3, d)).astype(dt)
    gpu.BlockNorm(view(d), h, y=dev(gpu, y, stream), x_out=view(d), post="layer", pre="rms")(stream)
    r, er, hh, eh = ref.block_norm(x, y, None, 1, "linear", 1.0, "layer", None, None, "rms", None, None, 1e-5, 1e-5)
    check(rows(d), r, er, type == "f16", "far x_out")
    check(h.numpy(stream), hh, eh, type == "f16", "far h")
    fill(x)
    q, s = gpu.DeviceArray((3, d), np.int8), gpu.DeviceArray((3,), np.float32)
    gpu.QuantizeRows(view(d), q, s)(stream)
    want = ref.quantised(x)
    assert np.array_equal(q.numpy(stream), want[0]) and np.array_equal(s.numpy(stream), want[1])
    w, ws = rng.integers(-127, 128, (N, d)).astype(np.int8), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    wd = gpu.WeightI8(dev(gpu, w, stream), dev(gpu, ws, stream), stream)
    out = gpu.DeviceArray((3, N), dt)
    gpu.LinearI8(view(d), wd, out)(stream)
    check(out.numpy(stream), *ref.linear_i8(*want, w, ws, None, "none", 1.0, None, type == "f16"), type == "f16", "far x")
    gpu.LinearI8(dev(gpu, x, stream), wd, view(N), add=view(N))(stream)
    check(rows(N), *ref.linear_i8(*want, w, ws, None, "none", 1.0, x[:, :N], type == "f16"), type == "f16", "far y")
    fill(x)
    bias = rng.standard_normal((3, d)).astype(np.float32)
    gpu.LogitRules(view(d), view(d), bias=dev(gpu, bias, stream))(stream)
    for i, got in enumerate(rows(d)):
        check(got, *ref.rules(x[i], np.zeros(d), 1, 0, 0, bias[i], None), type == "f16", "far logits")


def test_repeated_rows(gpu, stream):
    """Inputs of stride 0 (one row for all, one head for all) and rows that overlap in what they are read from; names repeated."""
    rng = np.random.default_rng(44)
    M, d, N = 70, 200, 90
    flat = rng.standard_normal(M + d).astype(np.float32)
    base = dev(gpu, flat, stream)
    one, slide = View(base, 0, (M, d), (0, 1)), View(base, 0, (M, d), (1, 1))
    x1, xs = np.broadcast_to(flat[:d], (M, d)), np.stack([flat[i:i + d] for i in range(M)])
    o, h = gpu.DeviceArray((M, d), np.float32), gpu.DeviceArray((M, d), np.float32)
    gpu.BlockNorm(one, h, y=slide, x_out=o, gate=one, pre="layer")(stream)
    r, er, hh, eh = ref.block_norm(x1, xs, x1, 1, "linear", 1.0, "none", None, None, "layer", None, None, 1e-5, 1e-5)
    check(o.numpy(stream), r, er, False, "x_out")
    check(h.numpy(stream), hh, eh, False, "h")
    w, ws = rng.integers(-127, 128, (N, d)).astype(np.int8), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    wd = gpu.WeightI8(dev(gpu, w, stream), dev(gpu, ws, stream), stream)
    for x, rows in ((one, x1), (slide, xs)):
        for many in (M, 9):
            y, v = gpu.DeviceArray((many, N), np.float32), View(base, 0, (many, d), x.strides)
            gpu.LinearI8(v, wd, y, add=View(base, 3, (many, N), (0, 1)))(stream)
            q, s = ref.quantised(rows[:many])
            check(y.numpy(stream), *ref.linear_i8(q, s, w, ws, None, "none", 1.0, np.broadcast_to(flat[3:3 + N], (many, N))), False, "y")
    f, out = dev(gpu, 10000.0 ** (-np.arange(16) / 16), stream), gpu.DeviceArray((2, 5, 3, 32), np.float32)
    gpu.Rotary(f, [(View(base, 0, (2, 5, 3, 32), (7, 32, 0)), out)])(stream)
    got = out.numpy(stream)
    for i in range(2):
        src = np.stack([np.broadcast_to(flat[7 * i + 32 * t:7 * i + 32 * t + 32], (3, 32)) for t in range(5)])
        check(got[i], *ref.rotary(src, np.arange(5), 10000.0 ** (-np.arange(16) / 16), 32, False, 1.0), False, "turned")
    words, out = i32(rng.integers(0, d, (2, 20))), gpu.DeviceArray((M, d), np.float32)
    slot, freq = i32(np.arange(M) % 2), dev(gpu, np.full(M, 0.3, np.float32), stream)
    gpu.LogitRules(one, out, tokens=dev(gpu, words, stream), length=dev(gpu, i32([20] * M), stream), slot=dev(gpu, slot, stream), frequency=freq,
                   bias=View(base, 1, (M, d), (0, 1)), mask=View(dev(gpu, np.full(7, 0x5555FFFF, np.uint32), stream), 0, (M, 7), (0, 1)))(stream)
    got = out.numpy(stream)
    for r in range(M):
        counts = np.bincount(words[slot[r]], minlength=d)
        check(got[r], *ref.rules(x1[r], counts, 1, 0, np.float32(0.3), flat[1:1 + d], (0x5555FFFF >> (np.arange(d) % 32) & 1) != 0), False, f"rules {r}")


def test_many_rows_graph(gpu, stream):
    """The forms for many rows captured and replayed on changed inputs, against the same calls made directly on another stream between the replays."""
    rng = np.random.default_rng(45)
    M, D, N, other = 700, 1000, 900, gpu.Stream()
    wd = gpu.WeightI8.quantize(dev(gpu, rng.standard_normal((N, D)).astype(np.float32), stream), stream)
    freq = dev(gpu, gpu.rotary_frequencies(90), stream)
    x = gpu.DeviceArray((M, D), np.float16)
    sides = []
    for _ in range(2):
        q8, sc = gpu.DeviceArray((M, D), np.int8), gpu.DeviceArray((M,), np.float32)
        h, y, z = (gpu.DeviceArray(s, np.float16) for s in ((M, D), (M, N), (M, N)))
        heads = View(y, 0, (1, M, 10, 90), (M * N, N, 90))
        calls = [gpu.BlockNorm(x, h, pre="layer"), gpu.LinearI8(h, wd, y), gpu.Rotary(freq, [(heads, heads)]), gpu.LogitRules(y, z), gpu.QuantizeRows(x, q8, sc)]
        sides.append((calls, (h, y, z, q8, sc)))
    x.upload(rng.standard_normal((M, D)).astype(np.float16), stream)
    for c in sides[0][0] + sides[1][0]:
        c(stream)
    stream.sync()
    hip, graph, ex = _hip(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream.handle, 1) == 0
    for c in sides[0][0]:
        c(stream)
    assert hip.hipStreamEndCapture(stream.handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for step in range(3):
        x.upload(rng.standard_normal((M, D)).astype(np.float16), stream)
        stream.sync()
        assert hip.hipGraphLaunch(ex, stream.handle) == 0
        for c in sides[1][0]:
            c(other)
        stream.sync()
        other.sync()
        for a, b in zip(sides[0][1], sides[1][1]):
            assert np.array_equal(a.numpy(stream), b.numpy(stream)), step
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("M,N", [(1100, 40), (2000, 4096)])
def test_far_tokens_8bit(gpu, stream, M, N):
    """8-bit tokens of the largest stride, together past 4 GiB; few channels and tiles of them."""
    rng = np.random.default_rng(41)
    K, row = 100, (1 << 22) - 16
    big = gpu.DeviceArray(((M - 1) * row + 112,), np.int8)
    x, s = rng.integers(-127, 128, (M, K)).astype(np.int8), rng.uniform(0.001, 0.05, M).astype(np.float32)
    for m in range(M):
        _put(gpu, stream, big, m * row, x[m])
    w, ws = rng.integers(-127, 128, (N, K)).astype(np.int8), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    y = gpu.DeviceArray((M, N), np.float32)
    gpu.LinearI8(View(big, 0, (M, K), (row, 1)), gpu.WeightI8(dev(gpu, w, stream), dev(gpu, ws, stream), stream), y, x_scale=dev(gpu, s, stream))(stream)
    check(y.numpy(stream), *ref.linear_i8(x, s, w, ws, None, "none", 1.0, None), False, "far tokens")


@pytest.mark.parametrize("M", [2, 200])
def test_far_weights_8bit(gpu, stream, M):
    """Weights of more than 4 GiB (rows that overlap in what they are packed from), few tokens and tiles of them; the last channels of each."""
    rng = np.random.default_rng(42)
    N, K = 33000, 131071
    flat = rng.integers(-127, 128, (N - 1) * 16 + K).astype(np.int8)
    base = dev(gpu, flat, stream)
    ws = rng.uniform(0.0005, 0.002, N).astype(np.float32)
    wd = gpu.WeightI8(View(base, 0, (N, K), (16, 1)), dev(gpu, ws, stream), stream)
    x = rng.standard_normal((M, K)).astype(np.float32)
    y = gpu.DeviceArray((M, N), np.float32)
    gpu.LinearI8(dev(gpu, x, stream), wd, y)(stream)
    got, (q, s) = y.numpy(stream), ref.quantised(x[-2:])
    for n0 in (0, 16350, N - 40):
        w = np.stack([flat[16 * n:16 * n + K] for n in range(n0, n0 + 40)])
        check(got[-2:, n0:n0 + 40], *ref.linear_i8(q, s, w, ws[n0:n0 + 40], None, "none", 1.0, None), False, f"channels from {n0}")


def test_far_histories(gpu, stream):
    """Histories 2^30 tokens long, the last of them counted, by slot and by table; masks and biases whose rows lie 2^31 bytes apart."""
    rng = np.random.default_rng(43)
    cap, V, n = 1 << 30, 90, 40
    words = gpu.DeviceArray((3, cap), np.int32)
    ids = i32(rng.integers(0, V, (3, n)))
    for s in range(3):
        _put(gpu, stream, words, (s + 1) * cap - n, ids[s])
    table = gpu.DeviceArray((2, cap), np.int32)
    who = i32(rng.integers(-1, 4, (2, n)))
    for r in range(2):
        _put(gpu, stream, table, (r + 1) * cap - n, who[r])
    rows = gpu.DeviceArray((1 << 29,), np.float32)           # bias at 0 and 2^29 - 128, mask words behind each
    bias, bits = rng.standard_normal((2, V)).astype(np.float32), rng.random((2, 96)) < 0.7
    step = (1 << 29) - 128
    for i in range(2):
        _put(gpu, stream, rows, i * step, np.concatenate([bias[i], np.packbits(bits[i], bitorder="little").view(np.float32)]))
    x = rng.standard_normal((2, V)).astype(np.float32)
    out, f = gpu.DeviceArray((2, V), np.float32), dev(gpu, np.float32([0.3, 0.4]), stream)
    sets = View(rows, 0, (2, V), (step, 1))
    keep = View(rows, V, (2, 3), (step, 1))
    keep.dtype = np.dtype(np.uint32)
    for by in ("slot", "table"):
        where = dict(slot=dev(gpu, i32([2, 1]), stream)) if by == "slot" else dict(table=table)
        gpu.LogitRules(dev(gpu, x, stream), out, tokens=words, length=dev(gpu, i32([cap, cap]), stream), window=n, frequency=f, bias=sets, mask=keep, **where)(stream)
        got = out.numpy(stream)
        for r in range(2):
            s = np.full(n, [2, 1][r]) if by == "slot" else who[r]
            fine = (s >= 0) & (s < 3)
            counts = np.bincount(ids[s[fine], np.arange(n)[fine]], minlength=V)
            check(got[r], *ref.rules(x[r], counts, 1, 0, [0.3, 0.4][r], bias[r], bits[r, :V]), False, f"far {by} {r}")


# ---- rotary ---------------------------------------------------------------------
ROTARY = [
    # type, R, n, heads, d, rot, interleaved, layout
    ("f16", 3, 1, (8, 8), 64, 64, False, "fused"), ("f16", 2, 37, (4, 1), 128, 64, True, "fused"), ("f32", 1, 5, (2, 2), 80, 80, False, "apart"),
    ("f32", 2, 9, (3,), 32, 10, True, "apart"), ("f16", 2, 3, (2, 1), 40, 26, False, "in place"), ("f32", 1, 130, (1, 1, 1), 7, 6, False, "in place"),
    ("f16", 4, 2, (1, 4), 8, 2, True, "head major"), ("f32", 2, 4, (16, 2), 256, 256, True, "in place"), ("f16", 1, 1, (1,), 512, 512, False, "apart"),
    ("f16", 2, 6, (2, 2), 64, 0, False, "apart"), ("f16", 5, 7, (2, 3), 80, 40, True, "head major"),
]


@pytest.mark.parametrize("type,R,n,heads,d,rot,inter,layout", ROTARY)
@pytest.mark.parametrize("mode", ["start", "pos"])
def test_rotary(gpu, stream, type, R, n, heads, d, rot, inter, layout, mode):
    """Pairs, widths and layouts; positions from a start or one for each token, far and negative ones; ragged counts, an empty row."""
    print(f"[rotary] {type} R={R} n={n} heads={heads} d={d} rot={rot} inter={inter} {layout} {mode}", flush=True)
    rng = np.random.default_rng(R * 100 + n + d)
    freq = 10000.0 ** (-np.arange(rot // 2) * 2 / max(rot, 1))
    all_heads, dt = sum(heads), DT[type]
    start = i32(rng.integers(0, 1000000, R))
    pos = i32(rng.integers(-3000, 1 << 24, (R, n + 2)))
    count = i32(([n, 0, max(n - 1, 0), n + 5, -3] * R)[:R])
    x = rng.standard_normal((R, n, all_heads, d)).astype(dt)
    x[np.arange(n)[None] >= count[:, None]] = NAN       # not read, or not written
    if layout == "head major":
        src = dev(gpu, x.transpose(0, 2, 1, 3), stream)
        strides = (all_heads * n * d, d, n * d)
        at = lambda h: h * n * d  # noqa: E731
    else:
        src = dev(gpu, x, stream)
        strides = (n * all_heads * d, all_heads * d, d)
        at = lambda h: h * d  # noqa: E731
    parts, outs, h0 = [], [], 0
    for H in heads:
        s = View(src, at(h0), (R, n, H, d), strides)
        o = s if layout == "in place" else dev(gpu, np.full((R, n, H, d), 3, dt), stream)
        parts.append((s, o))
        outs.append(o)
        h0 += H
    where = dict(start=dev(gpu, start, stream)) if mode == "start" else dict(pos=View(dev(gpu, pos, stream), 1, (R, n), (n + 2, 1)))
    mult = 1.0 if mode == "start" else 1.25
    f = gpu.DeviceArray((max(rot // 2, 1),), np.float64)
    f.upload(freq if rot else np.zeros(1), stream)
    gpu.Rotary(View(f, 0, (rot // 2,), (1,)), parts, count=dev(gpu, count, stream), interleaved=inter, mult=mult, **where)(stream)
    h0 = 0
    for o, H in zip(outs, heads):
        got = src.numpy(stream)[:, :, h0:h0 + H] if layout == "in place" else o.numpy(stream)
        for r in range(R):
            c = min(max(int(count[r]), 0), n)
            at_ = start[r] + np.arange(c, dtype=np.int64) if mode == "start" else pos[r, 1:1 + c]
            want, err = ref.rotary(x[r, :c, h0:h0 + H], at_, freq, rot, inter, mult)
            check(got[r, :c], want, err, type == "f16", f"row {r}")
            assert np.array_equal(got[r, :c, :, rot:], x[r, :c, h0:h0 + H, rot:])
            assert np.isnan(got[r, c:]).all() if layout == "in place" else (got[r, c:] == 3).all()
        h0 += H


def test_rotary_undone(gpu, stream):
    """Turned by a position and by its negative: what it was, within the roundings of both."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, 50, 2, 64)).astype(np.float32)
    d, f = dev(gpu, x, stream), dev(gpu, 10000.0 ** (-np.arange(32) / 32), stream)
    p = i32(rng.integers(0, 100000, (1, 50)))
    for sign in (1, -1):
        gpu.Rotary(f, [(d, d)], pos=dev(gpu, sign * p, stream))(stream)
    err = 2 * (9 * ref.U + 2.0 ** -51 * 1e5) * (np.abs(x[..., :32]) + np.abs(x[..., 32:])) * np.sqrt(2.0)
    assert (np.abs(d.numpy(stream) - x) <= np.concatenate([err, err], -1) * 1.01 + 2 * ref.U * np.abs(x)).all()


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("far", ["row", "token", "head"])
def test_rotary_far(gpu, stream, type, far):
    """Rows, tokens or heads 2^31 elements apart, in place and into packed ones."""
    rng = np.random.default_rng(9)
    dt, d, n, R, H = DT[type], 64, *{"row": (3, 2, 2), "token": (2, 2, 3), "head": (3, 2, 2)}[far]
    step = {"row": (1 << 31, H * d, d), "token": (H * d, 1 << 31, d), "head": (n * d, d, 1 << 31)}[far]
    big = gpu.DeviceArray(((1 << 31) + 4 * R * n * H * d,), dt)
    x = rng.standard_normal((R, n, H, d)).astype(dt)
    at = lambda r, i, h: r * step[0] + i * step[1] + h * step[2]  # noqa: E731
    every = [(r, i, h) for r in range(R) for i in range(n) for h in range(H)]
    for r, i, h in every:
        _put(gpu, stream, big, at(r, i, h), x[r, i, h])
    freq = 10000.0 ** (-np.arange(16) / 16)
    v, packed, f, start = View(big, 0, x.shape, step), gpu.DeviceArray(x.shape, dt), dev(gpu, freq, stream), i32(np.arange(R) * 1000)
    for dst in (packed, v):
        gpu.Rotary(f, [(v, dst)], start=dev(gpu, start, stream))(stream)
    got = packed.numpy(stream)
    for r in range(R):
        want, err = ref.rotary(x[r], start[r] + np.arange(n), freq, 32, False, 1.0)
        check(got[r], want, err, type == "f16", f"far {far} {r}")
    assert np.array_equal(np.stack([_get(gpu, stream, big, at(*e), (d,)) for e in every]).reshape(x.shape), got)


# ---- rules on logits ------------------------------------------------------------
RULES = [
    # type, R, V, capacity, window, table, bias rows, mask rows
    ("f32", 4, 1025, 18, 0, False, 1, 0), ("f16", 16, 8193, 448, 0, True, 0, 5), ("f32", 3, 1, 5, 0, False, 2, 2), ("f16", 2, 33, 70, 7, True, 3, 3),
    ("f32", 5, 32769, 3000, 1024, True, 4, 4), ("f16", 1, 65537, 9000, 0, False, 1, 1), ("f32", 7, 8192, 1, 1, False, 0, 7), ("f16", 3, 20000, 0, 0, False, 0, 0),
    ("f32", 2, 300000, 500, 100, True, 0, 2), ("f32", 130, 50, 200, 0, True, 9, 9), ("f16", 600, 1000, 40, 5, False, 3, 0),
]


@pytest.mark.parametrize("type,R,V,cap,window,table,nb,nm", RULES)
@pytest.mark.parametrize("in_place", [False, True])
def test_logit_rules(gpu, stream, type, R, V, cap, window, table, nb, nm, in_place):
    """Counts through slots and tables, tokens, slots, lengths and row names out of range, masks that leave nothing, -inf, infinities and NaN
    in masked and penalised places, words at the ends of rows, rows further apart."""
    print(f"[rules] {type} R={R} V={V} cap={cap} window={window} table={table} bias={nb} mask={nm}", flush=True)
    rng = np.random.default_rng(V + cap)
    dt = DT[type]
    x = (4 * rng.standard_normal((R, V + 5))).astype(dt)
    x[rng.random(x.shape) < 0.01] = -np.inf
    slots = R + 2
    words = np.where(rng.random((slots, cap)) < 0.7, (V * rng.random((slots, cap)) ** 4), rng.integers(-2, V + 3, (slots, cap))).astype(np.int32)
    if cap > 2:
        words[:, 0], words[:, 1] = 0, V - 1
    lens = i32(rng.integers(0, cap + 1, R))
    lens[0] = cap + 10
    if R > 2:
        lens[1], lens[2] = -4, cap
    slot = i32(rng.permutation(slots)[:R])
    tab = i32(rng.integers(0, slots, (R, cap + 3)))
    tab[rng.random(tab.shape) < 0.05] = slots
    if R > 3:
        slot[3] = -1
    rep, pres, freq = (rng.uniform(a, b, R).astype(np.float32) for a, b in ((0.5, 2), (-0.5, 1), (0, 0.3)))
    bias = np.where(rng.random((nb, V)) < 0.1, 3 * rng.standard_normal((nb, V)), 0).astype(np.float32)
    bi = i32(rng.integers(-1, nb + 1, R))
    keep = rng.random((nm, V)) < 0.4
    if nm:
        keep[0] = False
    bits = np.zeros((nm, (V + 31) // 32 * 32), bool)
    bits[:, :V] = keep
    mask = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
    mi = i32(rng.integers(-1, nm + 1, R))
    if nm and R > 1:
        mi[0], mi[1] = 0, -1
        x[0, rng.random(V + 5) < 0.1] = NAN                # hidden by a mask of nothing
    dx = dev(gpu, x, stream)
    vx = View(dx, 2, (R, V), (V + 5, 1))
    out = vx if in_place else dev(gpu, np.full((R, V), 9, dt), stream)
    kw = dict(bias=dev(gpu, bias, stream), bias_index=dev(gpu, bi, stream)) if nb else {}
    if nm:
        kw.update(mask=dev(gpu, mask, stream), mask_index=dev(gpu, mi, stream))
    if cap:
        kw.update(tokens=dev(gpu, words, stream), length=dev(gpu, lens, stream), window=window, repetition=dev(gpu, rep, stream),
                  presence=dev(gpu, pres, stream), frequency=dev(gpu, freq, stream))
        kw.update(table=View(dev(gpu, tab, stream), 1, (R, cap), (cap + 3, 1))) if table else kw.update(slot=dev(gpu, slot, stream))
    gpu.LogitRules(vx, out, **kw)(stream)
    got = dx.numpy(stream) if in_place else out.numpy(stream)
    if in_place:
        assert np.array_equal(got[:, :2], x[:, :2], equal_nan=True) and np.array_equal(got[:, V + 2:], x[:, V + 2:], equal_nan=True)
        got = got[:, 2:V + 2]
    for r in range(R):
        counts = np.zeros(V)
        if cap:
            n = min(max(int(lens[r]), 0), cap)
            t = np.arange(max(0, n - window) if window else 0, n)
            s = tab[r, 1 + t] if table else np.full(len(t), slot[r])
            t, s = t[(s >= 0) & (s < slots)], s[(s >= 0) & (s < slots)]
            ids = words[s, t]
            np.add.at(counts, ids[(ids >= 0) & (ids < V)], 1)
        want, err = ref.rules(x[r, 2:V + 2], counts, rep[r], pres[r], freq[r], bias[bi[r]] if 0 <= bi[r] < nb else None,
                              keep[mi[r]] if 0 <= mi[r] < nm else None)
        check(got[r], want, err, type == "f16", f"row {r}") if r < 8 else None
        if r >= 8:
            fine = np.isfinite(want)
            assert np.array_equal(got[r][~fine].astype(np.float64), want[~fine], equal_nan=True)
            assert (np.abs(got[r][fine].astype(np.float64) - want[fine]) <= ref.rounded(err[fine], want[fine], type == "f16")).all()


def test_logit_rules_defaults(gpu, stream):
    """Each part alone; row names left out: row r's own."""
    rng = np.random.default_rng(6)
    R, V = 3, 100
    x = rng.standard_normal((R, V)).astype(np.float32)
    words = i32(rng.integers(0, V, (R, 30)))
    n, dx, out = dev(gpu, i32([30, 3, 0]), stream), dev(gpu, x, stream), gpu.DeviceArray((R, V), np.float32)
    v = rng.uniform(0.5, 2, R).astype(np.float32)
    for name, base in (("repetition", (1, 0, 0)), ("presence", (1, 0, 0)), ("frequency", (1, 0, 0))):
        gpu.LogitRules(dx, out, tokens=dev(gpu, words, stream), length=n, **{name: dev(gpu, v, stream)})(stream)
        got = out.numpy(stream)
        for r, m in enumerate((30, 3, 0)):
            args = [v[r] if k == name else b for k, b in zip(("repetition", "presence", "frequency"), base)]
            check(got[r], *ref.rules(x[r], np.bincount(words[r, :m], minlength=V), *args, None, None), False, name)
    bias, keep = rng.standard_normal((R, V)).astype(np.float32), rng.random((R, 128)) < 0.5
    gpu.LogitRules(dx, out, bias=dev(gpu, bias, stream))(stream)
    assert np.array_equal(out.numpy(stream), x + bias)
    gpu.LogitRules(dx, out, mask=dev(gpu, np.packbits(keep, axis=1, bitorder="little").view(np.int32), stream))(stream)
    assert np.array_equal(out.numpy(stream), np.where(keep[:, :V], x, -np.inf))
    gpu.LogitRules(dx, out)(stream)
    assert np.array_equal(out.numpy(stream), x)


# ---- together -------------------------------------------------------------------
class Layer:
    """One layer of a decoder and its head on the operators, as a program would call them: bound once, run every step."""

    def __init__(self, gpu, stream, rng, B, W, V, H, d, cap, cache):
        D, R = H * d, B * W
        self.gpu, self.V, self.R = gpu, V, R
        mat = lambda n, k: (rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32)  # noqa: E731
        self.w = {n: mat(*s) for n, s in (("qkv", (3 * D, D)), ("out", (D, D)), ("up", (2 * D, D)), ("down", (D, 2 * D)), ("head", (V, D)))}
        w = {n: gpu.WeightI8.quantize(dev(gpu, a, stream), stream) for n, a in self.w.items()}
        new = lambda *s, t=np.float32: dev(gpu, np.zeros(s, t), stream)  # noqa: E731
        self.x, self.h, self.hs = new(R, D), new(R, D, t=np.int8), new(R)
        self.qkv, self.ctx, self.y, self.up = new(R, 3 * D), new(R, D), new(R, D), new(R, 2 * D)
        self.logits, self.ruled = new(R, V), new(R, V)
        self.start, self.len = new(R, t=np.int32), new(R, t=np.int32)
        self.words = new(R, cap, t=np.int32)
        self.tables, self.score = [new(R, cap, t=np.int32) for _ in range(2)], [new(B, W) for _ in range(2)]
        self.done = [new(B, W, t=np.uint8) for _ in range(2)]
        self.parent, self.token = new(B, W, t=np.int32), new(B, W, t=np.int32)
        self.cache = cache
        heads = lambda i: View(self.qkv, i * D, (R, 1, H, d), (3 * D, 3 * D, d))  # noqa: E731
        one = lambda a: View(a, 0, (R, 1, H, d), (D, D, d))  # noqa: E731
        freq = dev(gpu, gpu.rotary_frequencies(d, factor=4.0, context=64, low=1, high=8), stream)
        rep, pres = dev(gpu, np.full(R, 1.3, np.float32), stream), dev(gpu, np.full(R, 0.1, np.float32), stream)
        self.keep = rng.random((2, V)) < 0.7
        self.keep[:, V - 1] = True
        bits = np.zeros((2, (V + 31) // 32 * 32), bool)
        bits[:, :V] = self.keep
        masks = dev(gpu, np.packbits(bits, axis=1, bitorder="little").view(np.int32), stream)
        self.state = dev(gpu, i32(np.arange(R) % 3 - 1), stream)
        self.calls = []
        for i in (0, 1):
            t = self.tables[i]
            self.calls.append([
                gpu.BlockNorm(self.x, self.h, pre="rms", h_scale=self.hs),
                gpu.LinearI8(self.h, w["qkv"], self.qkv, x_scale=self.hs),
                gpu.Rotary(freq, [(heads(0), heads(0)), (heads(1), heads(1))], start=self.start),
                gpu.CacheAppend(cache, heads(1), heads(2), self.start, table=t),
                gpu.CacheAttention(cache, heads(0), one(self.ctx), self.len, table=t),
                gpu.LinearI8(self.ctx, w["out"], self.y),
                gpu.BlockNorm(self.x, self.h, y=self.y, x_out=self.x, post="rms", pre="layer", alpha=0.5, h_scale=self.hs),
                gpu.LinearI8(self.h, w["up"], self.up, x_scale=self.hs, act="silu"),
                gpu.LinearI8(self.up, w["down"], self.x, add=self.x),
                gpu.BlockNorm(self.x, self.y, pre="rms"),
                gpu.LinearI8(self.y, w["head"], self.logits),
                gpu.LogitRules(self.logits, self.ruled, tokens=self.words, length=self.start, table=t, repetition=rep, presence=pres,
                               mask=masks, mask_index=self.state),
                gpu.BeamSelect(View(self.ruled, 0, (B, W, V), (W * V, V, 1)), self.score[i], self.parent, self.token, self.score[1 - i],
                               done=self.done[i], new_done=self.done[1 - i], end_id=V - 1),
                gpu.BeamReorder(self.parent, [(self.tables[i], self.tables[1 - i])]),
            ])

    def outputs(self, i, stream):
        return {n: a.numpy(stream) for n, a in dict(x=self.x, qkv=self.qkv, ctx=self.ctx, logits=self.logits, ruled=self.ruled, parent=self.parent,
                                                    token=self.token, score=self.score[1 - i], table=self.tables[1 - i]).items()}


def _linear(x, w):
    """x [M][K] through weights quantised by output channel, tokens by row: the float64 value."""
    wq, ws = ref.quantised(w)
    q, s = ref.quantised(x)
    return ref.linear_i8(q, s, wq, ws, None, "none", 1.0, None)


def test_decoder_layer_steps(gpu, stream):
    """Beam steps of a whole layer and its head: norms into 8 bits, products, rotary in place, the 8-bit cache by table, rules over the beams' histories,
    selection and reordering; each operator's output against its restatement on what the calls before it gave."""
    rng = np.random.default_rng(31)
    B, W, V, H, d, cap, steps = 2, 3, 70, 2, 32, 64, 40
    R, D = B * W, H * d
    net = Layer(gpu, stream, rng, B, W, V, H, d, cap, gpu.Cache8(R, H, d, cap))
    embed = rng.standard_normal((V, D)).astype(np.float32)
    score = np.full((B, W), -np.inf, np.float32)
    score[:, 0] = 0
    net.score[0].upload(score, stream)
    tok, freq = np.zeros(R, int), gpu.rotary_frequencies(d, factor=4.0, context=64, low=1, high=8)
    words, hist = np.zeros((R, cap), np.int32), [[] for _ in range(R)]
    state = np.arange(R) % 3 - 1
    for step in range(steps):
        i = step & 1
        net.x.upload(embed[tok], stream)
        net.start.upload(np.full(R, step, np.int32), stream)
        net.len.upload(np.full(R, step + 1, np.int32), stream)
        net.words.upload(words, stream)
        c = net.calls[i]
        c[0](stream)
        h, hs = net.h.numpy(stream), net.hs.numpy(stream)
        c[1](stream)
        qkv = net.qkv.numpy(stream)
        wq, ws = ref.quantised(net.w["qkv"])
        check(qkv, *ref.linear_i8(h, hs, wq, ws, None, "none", 1.0, None), False, "qkv")
        c[2](stream)
        turned = net.qkv.numpy(stream)
        for r in range(R):
            for z in (0, 1):
                x = qkv[r, z * D:(z + 1) * D].reshape(1, H, d)
                check(turned[r, z * D:(z + 1) * D].reshape(1, H, d), *ref.rotary(x, [step], freq, d, False, 1.0), False, "turned")
        assert np.array_equal(turned[:, 2 * D:], qkv[:, 2 * D:])
        c[3](stream), c[4](stream), c[5](stream)
        ctx, y, x = net.ctx.numpy(stream), net.y.numpy(stream), net.x.numpy(stream)
        assert np.isfinite(ctx).all()
        check(y, *_linear(ctx, net.w["out"]), False, "out")
        c[6](stream)
        r6 = ref.block_norm(x, y, None, 1, "linear", 0.5, "rms", None, None, "layer", None, None, 1e-5, 1e-5)
        x1, h, hs = net.x.numpy(stream), net.h.numpy(stream), net.hs.numpy(stream)
        check(x1, r6[0], r6[1], False, "x_out")
        assert (np.abs(h * hs[:, None].astype(np.float64) - r6[2]) <= 0.51 * hs[:, None] + r6[3]).all()
        c[7](stream), c[8](stream), c[9](stream)
        up, x2 = net.up.numpy(stream), net.x.numpy(stream)
        want, err = _linear(up, net.w["down"])
        check(x2, want + x1, err + ref.U * np.abs(want + x1), False, "down")
        y = net.y.numpy(stream)
        c[10](stream), c[11](stream)
        logits, ruled = net.logits.numpy(stream), net.ruled.numpy(stream)
        check(logits, *_linear(y, net.w["head"]), False, "head")
        for r in range(R):
            counts = np.bincount([words[s, t] for s, t in hist[r]], minlength=V) if hist[r] else np.zeros(V)
            check(ruled[r], *ref.rules(logits[r], counts, 1.3, 0.1, 0, None, net.keep[state[r]] if state[r] >= 0 else None), False, f"rules {r}")
        done = net.done[i].numpy(stream)
        score = net.score[i].numpy(stream)
        c[12](stream), c[13](stream)
        want = decoder_ref.beam_select(ruled.reshape(B, W, V), score, done, V - 1)
        assert np.array_equal(net.parent.numpy(stream), want[0]) and np.array_equal(net.token.numpy(stream), want[1]), step
        src = (want[0] + W * np.arange(B)[:, None]).reshape(-1)
        # position `step` is the token that a beam took in at this step, as its keys and values are: its own slot, then by the reordered table
        words[:, step] = tok
        hist = [hist[s] + [(s, step)] for s in src]
        tok = want[1].reshape(-1)
    print(f"[layer] {steps} steps", flush=True)


def _hip():
    h = C.CDLL("libamdhip64.so.7")       # the runtime that libpkx.so has loaded
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
    h.hipGraphExecDestroy.argtypes = [C.c_void_p]
    h.hipGraphDestroy.argtypes = [C.c_void_p]
    return h


def test_decoder_layer_graph(gpu, stream):
    """A layer's step captured into a graph and replayed on changed inputs against the same calls made directly, on another stream between the replays."""
    B, W, V, H, d, cap = 2, 4, 3001, 4, 64, 256
    sides = [Layer(gpu, stream, np.random.default_rng(12), B, W, V, H, d, cap, gpu.Cache8(B * W, H, d, cap)) for _ in range(2)]
    R, other = B * W, gpu.Stream()
    kv = [np.random.default_rng(14).integers(-127, 128, (R, H, cap, d)).astype(np.int8) for _ in range(2)]
    for s in sides:
        s.cache.k.upload(kv[0], stream)         # lengths below jump: positions in between hold these
        s.cache.v.upload(kv[1], stream)
        s.len.upload(i32([1] * R), stream)
        for c in s.calls[0]:                   # first calls outside the capture load the kernels
            c(stream)
    stream.sync()
    hip, graph, ex = _hip(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream.handle, 1) == 0
    for c in sides[0].calls[0]:
        c(stream)
    assert hip.hipStreamEndCapture(stream.handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    rng = np.random.default_rng(13)
    for step in range(5):
        n = (0, 1, 31, 64, 200)[step]
        x, words = rng.standard_normal((R, H * d)).astype(np.float32), i32(rng.integers(0, V, (R, cap)))
        table, score = i32(rng.integers(0, R, (R, cap))), rng.standard_normal((B, W)).astype(np.float32)
        for s in sides:
            for a, v in ((s.x, x), (s.words, words), (s.tables[0], table), (s.score[0], score), (s.start, i32([n] * R)), (s.len, i32([n + 1] * R))):
                a.upload(v, stream)
        stream.sync()
        assert hip.hipGraphLaunch(ex, stream.handle) == 0
        for c in sides[1].calls[0]:
            c(other)
        stream.sync()
        other.sync()
        a, b = sides[0].outputs(0, stream), sides[1].outputs(0, other)
        for k in a:
            assert np.array_equal(a[k], b[k], equal_nan=True), (step, k)
        print(f"[graph] replay {step}, length {n}: the same", flush=True)
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


def test_two_streams_at_once(gpu, stream):
    """Calls of every operator on two streams with a workspace each give what they give alone."""
    rng = np.random.default_rng(21)
    other = gpu.Stream()
    M, D, N = 700, 1000, 900
    x = dev(gpu, rng.standard_normal((M, D)).astype(np.float16), stream)
    w = gpu.WeightI8.quantize(dev(gpu, rng.standard_normal((N, D)).astype(np.float32), stream), stream)
    outs = [gpu.DeviceArray((M, N), np.float16) for _ in range(3)]
    hs = [gpu.DeviceArray((M, D), np.float16) for _ in range(3)]
    calls = [(gpu.LinearI8(x, w, o), gpu.BlockNorm(x, h, pre="layer")) for o, h in zip(outs, hs)]
    for c in calls[2]:
        c(stream)
    stream.sync()
    for _ in range(10):
        for s, cs in zip((stream, other), calls):
            for c in cs:
                c(s)
    stream.sync()
    other.sync()
    for group in (outs, hs):
        want = group[2].numpy(stream)
        assert np.array_equal(group[0].numpy(stream), want) and np.array_equal(group[1].numpy(stream), want)
