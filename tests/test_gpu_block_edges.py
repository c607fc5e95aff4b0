"""The operators around a decoder's attention where their sizes, addresses or values are at an end, against block_ref.py."""
import numpy as np
import pytest

import block_ref as ref
import test_gpu_block as norm_rows
from test_gpu_block import View, _get, _put, check, dev

pytestmark = pytest.mark.gpu


def test_rotary_blocks_past_32_bits(gpu, stream):
    """A part of 513 heads takes a token a workgroup and one of a single head 1024: 2^21 + 1 workgroups for the first are 2^31 + 1024 tokens of
    the second, whose last ones have to end there."""
    n, d, heads = (1 << 21) + 1, 4, 513
    rng = np.random.default_rng(50)
    freq = np.float64([1.0, 0.01])
    many, one = gpu.DeviceArray((1, n, heads, d), np.float16), rng.standard_normal((1, n, 1, d)).astype(np.float16)
    ends = (0, 1, 77777, n - 2, n - 1)
    x = rng.standard_normal((len(ends), heads, d)).astype(np.float16)
    for a, i in zip(x, ends):
        _put(gpu, stream, many, i * heads * d, a)
    alone = dev(gpu, one, stream)
    gpu.Rotary(dev(gpu, freq, stream), [(many, many), (alone, alone)], interleaved=True)(stream)
    want, err = ref.rotary(one[0], np.arange(n), freq, d, True, 1.0)
    check(alone.numpy(stream)[0], want, err, True, "one head")
    want, err = ref.rotary(x, ends, freq, d, True, 1.0)
    check(np.stack([_get(gpu, stream, many, i * heads * d, (heads, d)) for i in ends]), want, err, True, "513 heads")


def test_quantize_longest_row(gpu, stream):
    """A row of 2^31 - 1 values, the last of them the largest: what a lane adds to its place past it is past 31 bits."""
    n, step = (1 << 31) - 1, 1 << 26
    rng = np.random.default_rng(51)
    part = rng.uniform(-2, 2, step).astype(np.float16)
    x, q, s = gpu.DeviceArray((1, n), np.float16), gpu.DeviceArray((1, n), np.int8), gpu.DeviceArray((1,), np.float32)
    for at in range(0, n, step):
        _put(gpu, stream, x, at, part[:min(step, n - at)])
    _put(gpu, stream, x, n - 1, np.float16([-3]))
    gpu.QuantizeRows(x, q, s)(stream)
    scale = np.float32(3) / np.float32(127)
    assert s.numpy(stream)[0] == scale
    want = np.rint(part.astype(np.float32) / scale).astype(np.int8)
    for at in range(0, n, step):
        got = _get(gpu, stream, q, at, (min(step, n - at),))
        if at + step >= n:
            assert got[-1] == -127
            got = got[:-1]
        assert np.array_equal(got, want[:len(got)]), at


# ---- the 8-bit product's tiles ---------------------------------------------------
TILES = [
    # tile, type, M, N, K (slabs of 128), act, bias, add, rows at whole lines, tokens
    ((32, 128), "f16", 300, 1030, 1000, "silu", True, True, True, "i8"), ((32, 128), "f32", 1001, 1000, 260, "none", True, False, True, "f"),
    ((64, 128), "f16", 2001, 1000, 700, "silu", True, True, True, "f"), ((64, 128), "f32", 2001, 1000, 700, "silu", True, True, False, "i8"),
    ((64, 128), "f16", 700, 2050, 1100, "none", True, False, False, "i8"), ((64, 128), "f32", 1000, 6000, 384, "none", False, True, True, "f"),
    ((64, 256), "f16", 2001, 3000, 1100, "silu", True, True, True, "f"), ((64, 256), "f16", 2001, 3000, 1100, "none", False, True, False, "i8"),
    ((64, 256), "f32", 1000, 4099, 2040, "silu", True, True, True, "i8"), ((64, 256), "f32", 520, 6000, 2050, "none", True, False, False, "f"),
    ((128, 256), "f16", 3000, 8200, 260, "silu", True, True, True, "f"), ((128, 256), "f16", 4100, 4099, 700, "none", True, True, False, "i8"),
    ((128, 256), "f32", 2001, 6000, 1100, "silu", True, True, True, "i8"), ((128, 256), "f32", 4100, 3000, 1100, "none", False, True, False, "f"),
    ((128, 256), "f32", 3000, 12300, 200, "silu", True, False, True, "f"), ((128, 256), "f16", 16400, 8200, 128, "none", True, False, True, "i8"),
]


@pytest.mark.parametrize("tile,type,M,N,K,act,bias,add,lines,tokens", TILES)
def test_linear_i8_tiles(gpu, stream, tile, type, M, N, K, act, bias, add, lines, tokens):
    """Every tile of the product, with rests in tokens, channels and inputs, even and odd numbers of slabs, results at whole lines and not: whole
    rows of the first tiles, of the last ones and of some in between."""
    print(f"[tiles] {tile} {type} M={M} N={N} K={K} {act} bias={bias} add={add} lines={lines} {tokens}", flush=True)
    rng = np.random.default_rng(M + 3 * N + K + lines)
    dt = np.dtype({"f16": np.float16, "f32": np.float32}[type])
    w, ws = rng.integers(-127, 128, (N, K)).astype(np.int8), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    row = -(-N * dt.itemsize // 64) * 64 // dt.itemsize + (64 // dt.itemsize if lines else 3)
    a = rng.standard_normal((M, N)).astype(dt) if add else None
    y = dev(gpu, np.full((M, row), 5, dt), stream)
    kw = dict(bias=dev(gpu, b, stream), act=act, add=dev(gpu, a, stream), alpha=-0.75 if add else 1.0)
    wd, vy = gpu.WeightI8(dev(gpu, w, stream), dev(gpu, ws, stream), stream), View(y, 0, (M, N), (row, 1))
    if tokens == "f":
        x = rng.standard_normal((M, K)).astype(dt)
        call = gpu.LinearI8(dev(gpu, x, stream), wd, vy, **kw)
    else:
        x, s = rng.integers(-128, 128, (M, (K + 15) // 16 * 16 + 16)).astype(np.int8), rng.uniform(0.001, 0.05, M).astype(np.float32)
        call = gpu.LinearI8(View(dev(gpu, x, stream), 0, (M, K), (x.shape[1], 1)), wd, vy, x_scale=dev(gpu, s, stream), **kw)
    assert call.tile()[0] == tile
    call(stream)
    got, r = y.numpy(stream), np.unique(np.r_[0:40, 60:70, 126:130, rng.integers(0, M, 40), M - 140:M])
    q, s = ref.quantised(x[r]) if tokens == "f" else (x[r, :K], s[r])
    want, err = ref.linear_i8(q, s, w, ws, b, act, kw["alpha"], a[r] if add else None, type == "f16")
    check(got[r, :N], want, err, type == "f16", "y")
    assert (got[:, N:] == 5).all()


# ---- forms that larger or odder sizes take ---------------------------------------
@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("R,V,table", [(1100, 70, True), (350, 8193, False), (130, 40001, True)])
def test_logit_rules_many_rows(gpu, stream, type, R, V, table):
    """More than 1024 tiles of 4096 words: tiles of up to 8192, one and several of them to a row; in place."""
    rng = np.random.default_rng(R + V)
    dt, cap, slots = {"f16": np.float16, "f32": np.float32}[type], 90, 40
    x = (4 * rng.standard_normal((R, V))).astype(dt)
    words = rng.integers(-1, V + 1, (slots, cap)).astype(np.int32)
    words[:, :6] = 0, V - 1, min(V - 1, 4095), min(V - 1, 4096), min(V - 1, 8191), min(V - 1, 8192)
    lens, slot, tab = (rng.integers(a, b, s).astype(np.int32) for a, b, s in ((0, cap + 2, R), (0, slots, R), (-1, slots + 1, (R, cap))))
    rep, pres, freq = (rng.uniform(a, b, R).astype(np.float32) for a, b in ((0.5, 2), (-0.5, 1), (0, 0.3)))
    bias, keep = rng.standard_normal((3, V)).astype(np.float32), rng.random((2, (V + 31) // 32 * 32)) < 0.5
    bi, mi = rng.integers(-1, 4, R).astype(np.int32), rng.integers(-1, 3, R).astype(np.int32)
    d = {k: dev(gpu, v, stream) for k, v in dict(tokens=words, length=lens, repetition=rep, presence=pres, frequency=freq, bias=bias, bias_index=bi, mask_index=mi,
                                                 mask=np.packbits(keep, axis=1, bitorder="little").view(np.uint32), **(dict(table=tab) if table else dict(slot=slot))).items()}
    y = dev(gpu, x, stream)
    gpu.LogitRules(y, y, **d)(stream)
    got = y.numpy(stream).astype(np.float64)
    for r in range(R):
        n = min(int(lens[r]), cap)
        s, t = tab[r, :n] if table else np.full(n, slot[r]), np.arange(n)
        fine = (s >= 0) & (s < slots)
        ids = words[s[fine], t[fine]]
        counts = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V)
        want, err = ref.rules(x[r], counts, rep[r], pres[r], freq[r], bias[bi[r]] if 0 <= bi[r] < 3 else None, keep[mi[r], :V] if 0 <= mi[r] < 2 else None)
        kept = np.isfinite(want)
        assert np.array_equal(got[r][~kept], want[~kept]), r
        assert (np.abs(got[r][kept] - want[kept]) <= ref.rounded(err[kept], want[kept], type == "f16")).all(), r


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("type,d,rot", [("f16", 80, 40), ("f16", 20, 12), ("f16", 24, 8), ("f16", 88, 88), ("f16", 100, 20), ("f32", 80, 20), ("f32", 12, 8), ("f16", 128, 0), ("f16", 26, 26)])
@pytest.mark.parametrize("place", ["apart", "in place"])
def test_rotary_pieces(gpu, stream, type, d, rot, inter, place):
    """Pairs and rests that divide by eight, by four and by neither, several tokens to a workgroup, two parts."""
    rng = np.random.default_rng(d + rot)
    dt, n, R, heads = {"f16": np.float16, "f32": np.float32}[type], 43, 2, (5, 1)
    x = rng.standard_normal((R, n, 6, d)).astype(dt)
    freq = 10000.0 ** (-np.arange(rot // 2) * 2 / max(rot, 1))
    src, f = dev(gpu, x, stream), dev(gpu, freq if rot else np.zeros(1), stream)
    out = src if place == "in place" else dev(gpu, np.full(x.shape, 3, dt), stream)
    part = lambda a, h0, H: View(a, h0 * d, (R, n, H, d), (n * 6 * d, 6 * d, d))  # noqa: E731
    gpu.Rotary(View(f, 0, (rot // 2,), (1,)), [(part(src, 0, 5), part(out, 0, 5)), (part(src, 5, 1), part(out, 5, 1))], start=dev(gpu, np.int32([3, 70000]), stream),
               interleaved=inter, mult=0.5)(stream)
    got = out.numpy(stream)
    for r, p in enumerate((3, 70000)):
        want, err = ref.rotary(x[r], p + np.arange(n), freq, rot, inter, 0.5)
        check(got[r], want, err, type == "f16", f"row {r}")
    assert np.array_equal(got[..., rot:], x[..., rot:])


# ---- block norm -----------------------------------------------------------------
@pytest.mark.parametrize("M,d", [(128, 2049), (129, 2049), (200, 4096), (256, 3001), (257, 2500)])
@pytest.mark.parametrize("type,xtype,post,pre,per,fn", [("f16", "f32", "layer", "rms", 7, "sigmoid"), ("f32", "f32", "rms", "layer", 0, "linear"),
                                                       ("f16", "f16", "none", "layer", 1, "linear")])
@pytest.mark.parametrize("i8", [False, True])
def test_block_norm_hundreds_of_rows(gpu, stream, type, xtype, post, pre, per, fn, M, d, i8):
    """Rows of 2049 to 4096 channels around the numbers of them at which the form changes."""
    norm_rows.test_block_norm(gpu, stream, type, xtype, M, d, post, pre, per, fn, i8)


@pytest.mark.parametrize("d", [100, 200, 500, 1000, 1500, 3000, 16000])
def test_block_norm_infinite_rows(gpu, stream, d):
    """RMS of a row with an infinity: over an infinite root, 0 where the row is finite (its bias then) and NaN at the infinity; a block's output with
    one leaves the other channels of the residual as they were."""
    rng = np.random.default_rng(d)
    x, b = rng.standard_normal((3, d)).astype(np.float32), rng.standard_normal(d).astype(np.float32)
    x[0, 7], x[2, [1, d - 1]] = np.inf, -np.inf
    lost = np.isinf(x)
    h = gpu.DeviceArray(x.shape, np.float32)
    gpu.BlockNorm(dev(gpu, x, stream), h, pre="rms", pre_b=dev(gpu, b, stream))(stream)
    got = h.numpy(stream)
    check(got[1:2], *ref.normalised(x[1:2].astype(np.float64), np.zeros((1, d)), "rms", None, b, 1e-5), False, "finite row")
    assert np.isnan(got[lost]).all() and all(np.array_equal(got[r][~lost[r]], b[~lost[r]]) for r in (0, 2))
    s, o = rng.standard_normal((3, d)).astype(np.float32), gpu.DeviceArray(x.shape, np.float32)
    gpu.BlockNorm(dev(gpu, s, stream), y=dev(gpu, x.astype(np.float16), stream), x_out=o, post="rms")(stream)
    got = o.numpy(stream)
    assert np.isnan(got[lost]).all() and all(np.array_equal(got[r][~lost[r]], s[r][~lost[r]]) for r in (0, 2))


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("d", [100, 200, 500, 1000, 1500, 3000, 16000])
def test_block_norm_ends_of_f32(gpu, stream, kind, d):
    """Rows whose values lie further apart than f32 reaches, rows at its end and rows of subnormal values without an eps."""
    rng = np.random.default_rng(d)
    x = rng.standard_normal((8, d)).astype(np.float32)
    x[0], x[0, d // 2] = -2e38, 2e38
    x[1] = np.where(np.arange(d) % 2, 1, -1) * np.float32(3.4e38)
    x[2] = np.where(np.arange(d) % 3, 1, -0.9) * np.float32(3.4e38)
    x[3] *= np.float32(1e37)
    x[4] *= np.float32(1e-40)
    x[5] = np.arange(d) % 2 * np.float32(1.5e-45)
    x[6] *= np.float32(1e-36)
    h = gpu.DeviceArray(x.shape, np.float32)
    gpu.BlockNorm(dev(gpu, x, stream), h, pre=kind, eps=0)(stream)
    check(h.numpy(stream), *ref.normalised(x.astype(np.float64), np.zeros(x.shape), kind, None, None, 0.0), False, kind)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_silu_to_the_end_of_f32(gpu, stream, M):
    """SiLU of values whose e^-v passes f32 while v e^v is still a normal number, and of those on both sides."""
    v = np.r_[np.linspace(-95, -80, 301), np.linspace(-45, -38, 141), np.linspace(-4, 4, 61)].astype(np.float32)
    wd = gpu.WeightI8(dev(gpu, np.zeros((len(v), 16), np.int8), stream), dev(gpu, np.ones(len(v), np.float32), stream), stream)
    y = gpu.DeviceArray((M, len(v)), np.float32)
    gpu.LinearI8(dev(gpu, np.ones((M, 16), np.float32), stream), wd, y, bias=dev(gpu, v, stream), act="silu")(stream)
    got, x = y.numpy(stream), v.astype(np.float64)
    want = x / (1 + np.exp(-x))
    for r in (0, M // 2, M - 1):
        check(got[r], want, np.abs(want) * 6 * ref.U + 2.0 ** -126, False, f"row {r}")       # what is below the normal numbers may be 0
