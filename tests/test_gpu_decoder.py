"""The attention decoder operators (cross attention, 8-bit cache, beam selection
and reordering) against float64 restatements (decoder_ref.py): every element
within a bound derived from the roundings the kernels make; what is held in 8
bits, token ids and parents exactly."""
import ctypes as C

import numpy as np
import pytest

import decoder_ref as ref

pytestmark = pytest.mark.gpu
NAN = float("nan")


def dev(gpu, a, stream):
    return gpu.DeviceArray.from_numpy(np.ascontiguousarray(a), stream)


def i32(x):
    return np.asarray(x, np.int32)


class View:
    """A strided part of a device array, for the binding: strides in elements."""

    def __init__(self, base, offset, shape, strides):
        self.base, self.shape, self.dtype, self.strides = base, tuple(shape), base.dtype, tuple(strides)
        self.ptr = base.ptr + offset * base.dtype.itemsize


def check_attention(got, want, f16, d, label):
    err, bound = np.abs(got.astype(np.float64) - want[0]), ref.attention_bound(want, f16, d)
    worst = float((err / bound).max(initial=0))
    print(f"[{label}] largest error {err.max(initial=0):.2e}, {worst:.2f} of its bound", flush=True)
    assert np.isfinite(got).all() and worst <= 1.0


CROSS = [
    # type, B, n_q, n_k, H, Hkv, d
    ("f16", 1, 1, 125, 8, 8, 64), ("f16", 3, 4, 33, 4, 2, 128), ("f16", 2, 1, 1, 2, 1, 32), ("f16", 2, 5, 7, 3, 3, 8),
    ("f16", 2, 17, 70, 2, 2, 80), ("f16", 1, 2, 3001, 2, 1, 64), ("f16", 1, 1, 4096, 1, 1, 128), ("f16", 2, 130, 97, 2, 2, 64),
    ("f16", 1, 65, 300, 4, 1, 128), ("f16", 1, 64, 1, 1, 1, 24), ("f16", 2, 300, 515, 1, 1, 32), ("f16", 1, 200, 130, 2, 2, 128),
    ("f32", 1, 1, 125, 8, 8, 64), ("f32", 3, 4, 33, 4, 2, 128), ("f32", 2, 5, 7, 3, 3, 8), ("f32", 2, 37, 211, 2, 2, 64),
    # enough rows and keys for the many-row kernel, every head width, rows and keys that end inside a tile
    ("f16", 3, 130, 300, 48, 24, 64), ("f16", 2, 200, 515, 32, 32, 32), ("f16", 1, 257, 700, 36, 9, 128), ("f16", 2, 150, 430, 40, 40, 80),
    ("f16", 1, 200, 3000, 16, 2, 40),
    # no keys at all
    ("f16", 2, 3, 0, 2, 1, 64), ("f16", 1, 70, 0, 1, 1, 64), ("f32", 2, 3, 0, 2, 1, 64), ("f32", 1, 70, 0, 1, 1, 32),
    ("f32", 1, 2, 2048, 2, 1, 32), ("f32", 1, 3, 900, 2, 2, 128), ("f32", 2, 130, 97, 2, 2, 80), ("f32", 1, 70, 64, 4, 1, 128),
]


@pytest.mark.parametrize("type,B,nq,nk,H,Hkv,d", CROSS)
@pytest.mark.parametrize("masked", [False, True])
def test_cross_attention(gpu, stream, type, B, nq, nk, H, Hkv, d, masked):
    """Ragged queries and keys (lengths 0 and n among them), key masks that leave rows empty, NaN wherever
    nothing may be read, rows behind q_len left as they were."""
    print(f"[cross] {type} B={B} nq={nq} nk={nk} H={H} Hkv={Hkv} d={d} masked={masked}", flush=True)
    rng = np.random.default_rng(nq * 1000 + nk + d)
    dt = np.float16 if type == "f16" else np.float32
    q, k, v = (rng.standard_normal(s).astype(dt) for s in ((B, nq, H, d), (B, nk, Hkv, d), (B, nk, Hkv, d)))
    q *= dt(2)
    klen, qlen, mask = np.full(B, nk), np.full(B, nq), np.ones((B, nk), np.uint8)
    if masked:
        klen = np.array([nk, 0, max(1, nk // 3)])[:B]
        qlen = np.array([nq, nq, max(0, nq - 1)])[:B]
        mask = (rng.random((B, nk)) < 0.6).astype(np.uint8) * 7
        if B > 2:
            mask[2] = 0
        gone = (mask == 0) | (np.arange(nk)[None] >= klen[:, None])
        k[gone], v[gone] = NAN, np.inf
        q[np.arange(nq)[None] >= qlen[:, None]] = NAN
    out0 = rng.standard_normal((B, nq, H, d)).astype(dt)
    bufs = [dev(gpu, x, stream) for x in (q, k, v, out0)]
    extra = dict(q_len=dev(gpu, i32(qlen), stream), k_len=dev(gpu, i32(klen), stream), k_mask=dev(gpu, mask, stream)) if masked else {}
    scale = 0.3 if masked else None
    gpu.CrossAttention(*bufs, scale=scale, **extra)(stream)
    got = bufs[3].numpy(stream)
    G = H // Hkv
    for b in range(B):
        n = qlen[b]
        assert np.array_equal(got[b, n:], out0[b, n:])
        keep = np.broadcast_to((mask[b] != 0) & (np.arange(nk) < klen[b]), (n, nk))
        if n == 0:
            continue
        for h in range(H):
            want = ref.attention(q[b, :n, h], k[b, :, h // G], v[b, :, h // G], scale or d ** -0.5, keep)
            check_attention(got[b, :n, h], want, type == "f16", d, f"cross b{b} h{h}")


def test_rows_of_masks_logits_and_tables_further_apart(gpu, stream):
    """The middle of larger buffers of masks, logits and tables gives what packed copies give."""
    rng = np.random.default_rng(12)
    q, k, v = (dev(gpu, rng.standard_normal((2, n, 2, 32)).astype(np.float16), stream) for n in (3, 50, 50))
    mask = (rng.random((2, 64)) < 0.5).astype(np.uint8)
    outs = [gpu.DeviceArray((2, 3, 2, 32), np.float16) for _ in range(2)]
    gpu.CrossAttention(q, k, v, outs[0], k_mask=View(dev(gpu, mask, stream), 5, (2, 50), (64, 1)))(stream)
    gpu.CrossAttention(q, k, v, outs[1], k_mask=dev(gpu, np.ascontiguousarray(mask[:, 5:55]), stream))(stream)
    assert np.array_equal(*(o.numpy(stream) for o in outs))
    c = HostCache(gpu, stream, 3, 2, 64, 32, rng)
    table = rng.integers(0, 3, (2, 90)).astype(np.int32)
    n = dev(gpu, i32([60, 33]), stream)
    gpu.CacheAttention(c.dev, q, outs[0], n, table=View(dev(gpu, table, stream), 7, (2, 64), (90, 1)))(stream)
    gpu.CacheAttention(c.dev, q, outs[1], n, table=dev(gpu, np.ascontiguousarray(table[:, 7:71]), stream))(stream)
    assert np.array_equal(*(o.numpy(stream) for o in outs))
    x = rng.standard_normal((2, 4, 128)).astype(np.float32)
    score = dev(gpu, rng.standard_normal((2, 4)).astype(np.float32), stream)
    got = []
    for logits in (View(dev(gpu, x, stream), 3, (2, 4, 101), (4 * 128, 128, 1)), dev(gpu, np.ascontiguousarray(x[..., 3:104]), stream)):
        o = [gpu.DeviceArray((2, 4), t) for t in (np.int32, np.int32, np.float32)]
        gpu.BeamSelect(logits, score, *o)(stream)
        got.append([a.numpy(stream) for a in o])
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_cross_attention_strides_and_streams(gpu, stream):
    """Head-major buffers, the middle of larger ones, two streams at once, and what surrounds the output kept."""
    rng = np.random.default_rng(5)
    B, nq, nk, H, d = 2, 6, 90, 4, 64
    q = rng.standard_normal((B, H, nq + 3, d + 8)).astype(np.float16)
    kv = rng.standard_normal((B, nk, 2, H, d)).astype(np.float16)
    out0 = rng.standard_normal((B, H, nq, d + 16)).astype(np.float16)
    dq, dkv, s2 = dev(gpu, q, stream), dev(gpu, kv, stream), gpu.Stream()
    outs = [dev(gpu, out0, stream) for _ in range(2)]
    qs = (H * (nq + 3) * (d + 8), d + 8, (nq + 3) * (d + 8))
    os_ = (H * nq * (d + 16), d + 16, nq * (d + 16))
    calls = [gpu.CrossAttention(View(dq, 8, (B, nq, H, d), qs), View(dkv, 0, (B, nk, H, d), (nk * 2 * H * d, 2 * H * d, d)),
                                View(dkv, H * d, (B, nk, H, d), (nk * 2 * H * d, 2 * H * d, d)),
                                View(o, 8, (B, nq, H, d), os_)) for o in outs]
    for _ in range(3):
        for c, s in zip(calls, (stream, s2)):
            c(s)
    s2.sync()
    got = [o.numpy(stream) for o in outs]
    assert np.array_equal(got[0], got[1])
    assert np.array_equal(got[0][..., :8], out0[..., :8]) and np.array_equal(got[0][..., d + 8:], out0[..., d + 8:])
    for b in range(B):
        for h in range(H):
            want = ref.attention(q[b, h, :nq, 8:8 + d], kv[b, :, 0, h], kv[b, :, 1, h], d ** -0.5, np.ones((nq, nk), bool))
            check_attention(got[0][b, h, :, 8:8 + d], want, True, d, f"strides b{b} h{h}")


@pytest.mark.parametrize("type,H,nq,nk,d", [("f16", 2, 5, 75, 64), ("f16", 64, 330, 250, 64), ("f32", 2, 5, 75, 64), ("f32", 2, 80, 75, 128)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_cross_attention_scales(gpu, stream, type, H, nq, nk, d, scale):
    """Any factor: negative, zero (the mean of the kept values), large, with keys left out."""
    rng = np.random.default_rng(nq)
    dt = np.float16 if type == "f16" else np.float32
    q, k, v = (rng.standard_normal((1, n, H, d)).astype(dt) for n in (nq, nk, nk))
    mask = (rng.random((1, nk)) < 0.7).astype(np.uint8)
    out = gpu.DeviceArray(q.shape, dt)
    gpu.CrossAttention(*(dev(gpu, x, stream) for x in (q, k, v)), out, k_mask=dev(gpu, mask, stream), scale=scale)(stream)
    got = out.numpy(stream)
    for h in (0, H - 1):
        want = ref.attention(q[0, :, h], k[0, :, h], v[0, :, h], scale, np.broadcast_to(mask[0] != 0, (nq, nk)))
        check_attention(got[0, :, h], want, type == "f16", d, f"scale {scale} h{h}")


def test_cross_attention_far_items(gpu, stream):
    """Items 2^31 elements apart."""
    rng = np.random.default_rng(6)
    nk, d, far = 40, 32, 1 << 31
    big = gpu.DeviceArray((far + nk * d,), np.float16)
    q, k, v = (rng.standard_normal((2, n, 1, d)).astype(np.float16) for n in (3, nk, nk))
    for b in range(2):
        x = np.ascontiguousarray(k[b])
        gpu.check(gpu.lib().pkx_memcpy_h2d(big.ptr + 2 * b * far, x.ctypes.data, x.nbytes, stream.handle))
    dq, dv, out = dev(gpu, q, stream), dev(gpu, v, stream), gpu.DeviceArray((2, 3, 1, d), np.float16)
    gpu.CrossAttention(dq, View(big, 0, (2, nk, 1, d), (far, d, d)), dv, out)(stream)
    got = out.numpy(stream)
    for b in range(2):
        want = ref.attention(q[b, :, 0], k[b, :, 0], v[b, :, 0], d ** -0.5, np.ones((3, nk), bool))
        check_attention(got[b, :, 0], want, True, d, f"far b{b}")


# ---- 8-bit cache ------------------------------------------------------------
class HostCache:
    """A cache on the device and its restatement."""

    def __init__(self, gpu, stream, S, H, cap, d, rng):
        shape = (S, H, cap, d)
        self.k, self.v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (rng.uniform(0.001, 0.05, (S, H, cap // 32)).astype(np.float32) for _ in range(2))
        self.dev = gpu.Cache8.wrap(*(dev(gpu, x, stream) for x in (self.k, self.v, self.ks, self.vs)))

    def same(self, stream):
        for a, b, n in ((self.dev.k, self.k, "k"), (self.dev.v, self.v, "v"), (self.dev.k_scale, self.ks, "k_scale"),
                        (self.dev.v_scale, self.vs, "v_scale")):
            got = a.numpy(stream)
            assert np.array_equal(got, b), (n, int((got != b).sum()))


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("d,new", [(64, 1), (128, 1), (16, 1), (48, 1), (80, 1), (112, 1), (16, 5), (80, 40), (128, 100), (48, 31), (32, 33)])
def test_cache_append(gpu, stream, type, d, new):
    """Bytes and scales equal to the restatement's, whatever the position in a block; rows out of range, past the
    capacity, of count 0 and naming a slot again; NaN, infinities and zeros among the values; the rest untouched."""
    print(f"[append] {type} d={d} new={new}", flush=True)
    rng = np.random.default_rng(d + new)
    S, H, cap, R = 9, 3, 160, 10
    c = HostCache(gpu, stream, S, H, cap, d, rng)
    slot, start = i32([3, 0, 8, 1, 1, 9, -1, 5, 6, 2]), i32([0, 31, cap - 2, 64, 0, 0, 0, -1, cap, 50])
    count = i32([new, new + 5, new, new, new, new, new, new, new, 0])
    dt = np.float16 if type == "f16" else np.float32
    x = [(rng.standard_normal((R, new, H, d)) * rng.choice([1e-3, 1.0, 30.0], (R, 1, H, 1))).astype(dt) for _ in range(2)]
    x[0][0, 0, 0, :4] = [NAN, np.inf, -np.inf, 0]
    x[1][3, :, 1] = 0
    table0 = rng.integers(0, 99, (R, cap + 4)).astype(np.int32)
    table = dev(gpu, table0, stream)
    call = gpu.CacheAppend(c.dev, *(dev(gpu, a, stream) for a in x), start=dev(gpu, start, stream), slot=dev(gpu, slot, stream),
                           count=dev(gpu, count, stream), table=table)
    for again in range(2):          # the same tokens at the same place again change nothing
        call(stream)
        if again == 0:
            ref.append(c.k, c.ks, x[0], slot, start, count)
            ref.append(c.v, c.vs, x[1], slot, start, count)
        c.same(stream)
    want = table0.copy()
    for r in (0, 1, 2, 3):
        want[r, start[r]:min(start[r] + min(new, count[r]), cap)] = slot[r]
    assert np.array_equal(table.numpy(stream), want)
    got = [gpu.DeviceArray((R, 70, H, d), np.float32) for _ in range(2)]
    first = i32([-3, 0, cap - 5, cap, 10, 0, 0, 90, 91, 92])
    gpu.CacheRead(c.dev, *got, start=dev(gpu, first, stream), slot=dev(gpu, slot, stream))(stream)
    for y, ints, sc in ((got[0], c.k, c.ks), (got[1], c.v, c.vs)):
        y = y.numpy(stream)
        for r in range(R):
            pos = first[r] + np.arange(70)
            ok = (pos >= 0) & (pos < cap) & (0 <= slot[r] < S)
            val = ref.values(ints, sc, np.where(ok, slot[r], 0), np.where(ok, pos, 0))
            assert np.array_equal(y[r], np.where(ok[:, None, None], val, 0)), r


CACHE = [
    # type, R, n_q, H, Hkv, d, len, causal, table
    ("f16", 1, 1, 8, 8, 64, 18, True, False), ("f16", 3, 1, 4, 2, 128, 300, True, False), ("f16", 6, 1, 4, 4, 64, 100, True, True),
    ("f16", 3, 7, 4, 2, 80, 65, True, False), ("f16", 2, 70, 2, 2, 64, 200, True, False), ("f16", 1, 1, 2, 1, 32, 5000, True, False),
    ("f16", 2, 8, 2, 2, 16, 333, False, False), ("f16", 2, 40, 4, 2, 128, 90, False, True), ("f16", 1, 2, 16, 1, 48, 1, True, False),
    ("f32", 1, 1, 8, 8, 64, 18, True, False), ("f32", 6, 1, 4, 4, 128, 100, True, True), ("f32", 2, 70, 2, 1, 64, 200, True, False),
    # many rows over few keys: a weight's two f16 terms that do not add up to it are seen
    ("f32", 4, 128, 8, 8, 64, 48, False, False), ("f32", 2, 1500, 64, 64, 128, 150, False, False),
    # the many-row kernel: causal and not, keys split and whole; sizes just short of it
    ("f16", 6, 150, 32, 16, 128, 1100, True, False), ("f16", 6, 130, 32, 8, 80, 1230, False, False),
    ("f32", 6, 150, 32, 16, 128, 1100, False, False), ("f32", 6, 130, 32, 8, 112, 1230, True, False),
    ("f16", 6, 200, 16, 16, 64, 900, True, False), ("f32", 6, 257, 16, 16, 32, 650, True, False),
    ("f32", 1, 3, 2, 1, 32, 3000, True, False), ("f32", 3, 5, 2, 2, 16, 64, False, False), ("f32", 2, 80, 2, 2, 80, 111, True, True),
]


@pytest.mark.parametrize("type,R,nq,H,Hkv,d,n,causal,table", CACHE)
def test_cache_attention(gpu, stream, type, R, nq, H, Hkv, d, n, causal, table):
    """Lengths from 0 to n, queries before the first token, ragged queries, slots and table entries out of range,
    block scales that differ by five orders of magnitude."""
    print(f"[cache] {type} R={R} nq={nq} H={H} Hkv={Hkv} d={d} len={n} causal={causal} table={table}", flush=True)
    rng = np.random.default_rng(n + nq + d)
    cap, S = (n + 95) // 32 * 32, R + 2
    c = HostCache(gpu, stream, S, Hkv, cap, d, rng)
    c.vs *= 10.0 ** rng.uniform(-4, 1, c.vs.shape).astype(np.float32)
    c.dev.v_scale.upload(c.vs, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = (rng.standard_normal((R, nq, H, d)) * 0.7).astype(dt)
    lens = i32([n, 0, max(1, n // 2), n + 10 ** 6, 3, n][:R])
    qlen = i32([nq, nq, max(0, nq - 2), nq, nq, 0][:R])
    slot = i32([(3 * r + 1) % S if S % 3 else (r + 2) % S for r in range(R)])
    if R > 2 and not table:
        slot[0] = S
    out0 = rng.standard_normal(q.shape).astype(dt)
    tab, extra = None, {}
    if table:
        tab = rng.integers(0, S, (R, n)).astype(np.int32)
        tab[:, ::7] = rng.choice([-1, S, 1 << 30], tab[:, ::7].shape)
        if n > 64:
            tab[0, 32:64] = -5
        extra = dict(table=dev(gpu, tab, stream))
    out = dev(gpu, out0, stream)
    call = gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, lens, stream), slot=dev(gpu, slot, stream),
                              q_len=dev(gpu, qlen, stream), causal=causal, max_len=n, **extra)
    call(stream)
    got = out.numpy(stream)
    pos = np.arange(n)
    for r in range(R):
        L, m = min(max(int(lens[r]), 0), n), int(qlen[r])
        assert np.array_equal(got[r, m:], out0[r, m:])
        where = tab[r] if table else np.full(n, slot[r])
        ok = (where >= 0) & (where < S) & (pos < L)
        safe = np.where(ok, where, 0)
        K, V = ref.values(c.k, c.ks, safe, pos), ref.values(c.v, c.vs, safe, pos)
        keep = np.broadcast_to(ok, (m, n))
        if causal:
            keep = keep & (pos[None] <= (L - m + np.arange(m))[:, None])
        for h in range(H if m else 0):
            want = ref.attention(q[r, :, h][:m], K[:, h // (H // Hkv)], V[:, h // (H // Hkv)], d ** -0.5, keep)
            check_attention(got[r, :m, h], want, type == "f16", d, f"cache r{r} h{h}")


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_cache_attention_unused_slots_may_hold_anything(gpu, stream, type):
    """Positions whose table entry is out of range, with NaN scales in every slot and block that no entry names."""
    rng = np.random.default_rng(3)
    S, H, cap, d, n = 4, 2, 160, 64, 150
    c = HostCache(gpu, stream, S, H, cap, d, rng)
    tab = np.full((2, n), 1, np.int32)
    tab[:, 70:] = 2
    tab[0, ::3], tab[1, 32:64], tab[1, 140:] = -1, S, 1 << 30
    for a in (c.ks, c.vs):
        a[[0, 3]], a[1, :, 3:], a[2, :, :2] = NAN, NAN, NAN
    c.dev.k_scale.upload(c.ks, stream)
    c.dev.v_scale.upload(c.vs, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = rng.standard_normal((2, 1, H, d)).astype(dt)
    out = gpu.DeviceArray(q.shape, dt)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n, n]), stream), max_len=n, table=dev(gpu, tab, stream))(stream)
    got = out.numpy(stream)
    for r in range(2):
        ok = (tab[r] >= 0) & (tab[r] < S)
        K, V = (np.nan_to_num(ref.values(x, y, np.where(ok, tab[r], 0), np.arange(n))) for x, y in ((c.k, c.ks), (c.v, c.vs)))
        for h in range(H):
            want = ref.attention(q[r, :, h], K[:, h], V[:, h], d ** -0.5, ok[None])
            check_attention(got[r, :, h], want, type == "f16", d, f"r{r} h{h}")


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("table", [False, True])
def test_cache_attention_weights_near_nothing(gpu, stream, type, table):
    """Blocks whose weights run from 1 down to below the least normal f32: what is added for them is finite."""
    rng = np.random.default_rng(4)
    d, n = 16, 32 * 24
    c = HostCache(gpu, stream, 1, 1, n, d, rng)
    c.k[:] = 0
    c.k[0, 0, :, 0] = 100 - np.arange(n) // 32 * 8       # block b: scores of 8 (12 - b) + a little, in units of log 2
    c.k[0, 0, :, 1] = np.arange(n) % 3
    c.ks[:] = 1
    c.vs[:] = 1e-3
    c.dev.k.upload(c.k, stream)
    c.dev.k_scale.upload(c.ks, stream)
    c.dev.v_scale.upload(c.vs, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = np.zeros((1, 1, 1, d), dt)
    q[..., :2] = np.log(2), 0.125
    out = gpu.DeviceArray(q.shape, dt)
    extra = dict(table=dev(gpu, np.zeros((1, n), np.int32), stream)) if table else {}
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n]), stream), scale=1.0, **extra)(stream)
    K, V = (ref.values(x, y, np.zeros(n, int), np.arange(n))[:, 0] for x, y in ((c.k, c.ks), (c.v, c.vs)))
    check_attention(out.numpy(stream)[0, :, 0], ref.attention(q[0, :, 0], K, V, 1.0, np.ones((1, n), bool)), type == "f16", d, "near nothing")


@pytest.mark.parametrize("kind", ["cross", "cache"])
def test_many_small_weights_are_kept(gpu, stream, kind):
    """One key far above 20000 others of weight 100.5 x 2^-24 each: rounded to f16 as they are they would be 0.5% off
    together; scaled into its normal range they are off by at most half a step, 2^-11, and the output by another."""
    n, d = 20032, 16
    s0 = float(-np.log2(100.5 * 2.0 ** -24))
    k, v = np.zeros((1, n, 1, d), np.float32), np.ones((1, n, 1, d), np.float32)
    k[0, 0, 0, 0], v[0, 0] = 1, 0
    out = gpu.DeviceArray((1, 1, 1, d), np.float16)
    q = np.zeros((1, 1, 1, d), np.float16)
    q[..., 0] = 16
    scale = s0 * np.log(2) / 16
    if kind == "cross":
        gpu.CrossAttention(dev(gpu, q, stream), *(dev(gpu, x.astype(np.float16), stream) for x in (k, v)), out, scale=scale)(stream)
    else:
        c = gpu.Cache8(1, 1, d, n)
        gpu.CacheAppend(c, dev(gpu, k, stream), dev(gpu, v, stream), start=dev(gpu, i32([0]), stream))(stream)
        gpu.CacheAttention(c, dev(gpu, q, stream), out, dev(gpu, i32([n]), stream), scale=scale)(stream)
    rest = (n - 1) * 2.0 ** -s0
    want = rest / (1 + rest)
    # (a factor of 2^-24 relative in f32 moves the score of 17.3 by 2e-6 nats: nothing beside 2^-11)
    err = np.abs(out.numpy(stream).astype(np.float64) - want).max()
    print(f"[{kind}] error {err:.2e} of {want:.4f}", flush=True)
    assert err <= 2.0 ** -10 * want


def test_cache_far_slots(gpu, stream):
    """A slot, and a position, whose byte offset passes 2^32."""
    rng = np.random.default_rng(8)
    S, cap, d = 3, 1 << 24, 128
    k, v = gpu.DeviceArray((S, 1, cap, d), np.int8), gpu.DeviceArray((S, 1, cap, d), np.int8)
    sc = [gpu.DeviceArray((S, 1, cap // 32), np.float32) for _ in range(2)]
    c = gpu.Cache8.wrap(k, v, *sc)
    x = [rng.standard_normal((2, 40, 1, d)).astype(np.float32) for _ in range(2)]
    start, slot = i32([cap - 64, 0]), i32([1, 2])
    dslot = dev(gpu, slot, stream)
    gpu.CacheAppend(c, *(dev(gpu, a, stream) for a in x), start=dev(gpu, start, stream), slot=dslot)(stream)
    back = [gpu.DeviceArray((2, 40, 1, d), np.float32) for _ in range(2)]
    gpu.CacheRead(c, *back, start=dev(gpu, start, stream), slot=dslot)(stream)
    got = [b.numpy(stream) for b in back]
    for a, b in zip(x, got):
        top = max(np.abs(a[r, t:u]).max() for r in range(2) for t, u in ((0, 32), (32, 40)))
        assert np.abs(a - b).max() <= 0.5001 * top / 127
    q, out = rng.standard_normal((1, 1, 1, d)).astype(np.float32), gpu.DeviceArray((1, 1, 1, d), np.float32)
    gpu.CacheAttention(c, dev(gpu, q, stream), out, dev(gpu, i32([40]), stream), slot=dev(gpu, i32([2]), stream), max_len=64)(stream)
    want = ref.attention(q[0, :, 0], got[0][1, :, 0], got[1][1, :, 0], d ** -0.5, np.ones((1, 40), bool))
    check_attention(out.numpy(stream)[0, :, 0], want, False, d, "far slot")


# ---- beams --------------------------------------------------------------------
def run_select(gpu, stream, logits, scores, done, end):
    B, W, V = logits.shape
    o = [gpu.DeviceArray((B, W), t) for t in (np.int32, np.int32, np.float32, np.uint8)]
    gpu.BeamSelect(dev(gpu, logits, stream), dev(gpu, scores, stream), *o[:3],
                   done=None if done is None else dev(gpu, done, stream), new_done=o[3], end_id=end)(stream)
    return [a.numpy(stream) for a in o]


def check_select(got, want, scores, label):
    assert np.array_equal(got[0], want[0]), label
    assert np.array_equal(got[1], want[1]), label
    assert np.array_equal(got[3], want[3]), label
    fin = np.isfinite(want[2])
    assert np.array_equal(fin, np.isfinite(got[2])), label
    # one f32 rounding of a 64-bit sum whose log-sum carries the f32 exponentials' error (at most 2^-22 each)
    err = np.abs(got[2][fin] - want[2][fin])
    assert (err <= 2.0 ** -24 * np.abs(want[2][fin]) + 2.0 ** -21).all(), (label, err.max())


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (2, 4, 1025), (1, 32, 33), (3, 8, 3), (2, 5, 2048), (1, 7, 2049), (2, 16, 9001),
                                   (1, 3, 70000), (5, 2, 64), (1, 32, 70001), (2, 17, 700), (1, 20, 1500), (1, 1, 32768), (1, 1, 32769)])
def test_beam_select(gpu, stream, type, B, W, V):
    """Random logits; then equal ones (ties to the lowest index), finished beams, dead beams, -inf words."""
    print(f"[beam] {type} B={B} W={W} V={V}", flush=True)
    rng = np.random.default_rng(B * 100 + W * 10 + V)
    dt = np.float16 if type == "f16" else np.float32
    x = (3 * rng.standard_normal((B, W, V))).astype(dt)
    scores = (-10 + 2 * rng.standard_normal((B, W))).astype(np.float32)
    end = V - 1
    check_select(run_select(gpu, stream, x, scores, None, -1), ref.beam_select(x, scores, None, -1), scores, "random")
    done = (rng.random((B, W)) < 0.4).astype(np.uint8)
    check_select(run_select(gpu, stream, x, scores, done, end), ref.beam_select(x, scores, done, end), scores, "finished")
    same = np.full((B, W, V), 0.25, dt)
    zero = np.zeros((B, W), np.float32)
    check_select(run_select(gpu, stream, same, zero, None, end), ref.beam_select(same, zero, None, end), zero, "equal")
    first = np.full((B, W), -np.inf, np.float32)
    first[:, 0] = 0
    check_select(run_select(gpu, stream, x, first, None, end), ref.beam_select(x, first, None, end), first, "first step")
    odd = x.copy()
    odd[0, 0, 0] = NAN
    odd[-1, -1, V // 2] = np.inf
    if W > 1:
        odd[0, 1] = -np.inf
    if W > 2:
        odd[0, 2, ::2] = -np.inf
    sc = scores.copy()
    sc[-1, 0] = NAN
    check_select(run_select(gpu, stream, odd, sc, done, end), ref.beam_select(odd, sc, done, end), sc, "odd values")
    every = np.ones((B, W), np.uint8)
    check_select(run_select(gpu, stream, odd, scores, every, end), ref.beam_select(odd, scores, every, end), scores, "all finished")


@pytest.mark.parametrize("widths", [[64], [16, 4, 1], [7, 13, 4096 + 4], [1 << 16, 20, 3]])
def test_beam_reorder(gpu, stream, widths):
    """Rows of any size and alignment by parent; rows of a parent out of range stay."""
    rng = np.random.default_rng(sum(widths))
    B, W = 3, 5
    parent = rng.integers(0, W, (B, W)).astype(np.int32)
    parent[1, 2], parent[2, 4] = -1, W
    src = [rng.integers(0, 256, (B * W, n)).astype(np.uint8) for n in widths]
    dst = [rng.integers(0, 256, (B * W, n)).astype(np.uint8) for n in widths]
    ds, dd = ([dev(gpu, a, stream) for a in x] for x in (src, dst))
    gpu.BeamReorder(dev(gpu, parent, stream), list(zip(ds, dd)))(stream)
    for s, d, o in zip(src, dst, dd):
        want = d.copy()
        for r in range(B * W):
            p = parent[r // W, r % W]
            if 0 <= p < W:
                want[r] = s[r // W * W + p]
        assert np.array_equal(o.numpy(stream), want)


# ---- together -------------------------------------------------------------------
class Decoder:
    """One attention layer of a decoder with fixed random tables: queries, keys and values of a token at a position."""

    def __init__(self, rng, V, H, d, steps):
        self.q, self.k, self.v = (rng.standard_normal((V, H, d)) for _ in range(3))
        self.pos = 0.5 * rng.standard_normal((steps, H, d))
        self.out = rng.standard_normal((2 * H * d, V)) * 0.4

    def qkv(self, tok, step, dt=np.float32):
        return [(t[tok] + self.pos[step])[:, None].astype(dt) for t in (self.q, self.k, self.v)]


def test_decoder_steps(gpu, stream):
    """A beam search of 70 steps over encoder states with every operator: cache append with the table, cache and cross
    attention, selection, reordering of the table and of a state.  Parents and tokens equal to a search in float64
    whose histories are copied outright."""
    rng = np.random.default_rng(77)
    B, W, V, H, d, T, steps = 2, 4, 50, 2, 32, 61, 70
    net = Decoder(rng, V, H, d, steps)
    enc_k, enc_v = (rng.standard_normal((B, T, H, d)).astype(np.float32) for _ in range(2))
    enc_len = i32([T, 40])
    R, cap, end = B * W, 96, V - 1
    cache = gpu.Cache8(R, H, d, cap)
    tables = [dev(gpu, np.zeros((R, cap), np.int32), stream) for _ in range(2)]
    counts = [dev(gpu, np.zeros((R, 3), np.int32), stream) for _ in range(2)]
    q, k, v, self_out, cross_out = (gpu.DeviceArray((R, 1, H, d), np.float32) for _ in range(5))
    start, length = gpu.DeviceArray((R,), np.int32), gpu.DeviceArray((R,), np.int32)
    rows = lambda a: View(a, 0, (B, W, H, d), (W * H * d, H * d, d))  # noqa: E731
    cross = gpu.CrossAttention(rows(q), dev(gpu, enc_k, stream), dev(gpu, enc_v, stream), rows(cross_out),
                               k_len=dev(gpu, enc_len, stream))
    append = [gpu.CacheAppend(cache, k, v, start, table=t) for t in tables]
    attend = [gpu.CacheAttention(cache, q, self_out, length, table=t) for t in tables]
    logits = gpu.DeviceArray((B, W, V), np.float32)
    sc = [gpu.DeviceArray((B, W), np.float32) for _ in range(2)]
    fin = [gpu.DeviceArray((B, W), np.uint8) for _ in range(2)]
    parent, token = gpu.DeviceArray((B, W), np.int32), gpu.DeviceArray((B, W), np.int32)
    select = [gpu.BeamSelect(logits, sc[i], parent, token, sc[1 - i], done=fin[i], new_done=fin[1 - i], end_id=end) for i in (0, 1)]
    reorder = [gpu.BeamReorder(parent, [(tables[i], tables[1 - i]), (counts[i], counts[1 - i])]) for i in (0, 1)]
    scores = np.full((B, W), -np.inf, np.float32)
    scores[:, 0] = 0
    sc[0].upload(scores, stream)
    fin[0].upload(np.zeros((B, W), np.uint8), stream)
    counts[0].upload(np.arange(R * 3).reshape(R, 3).astype(np.int32), stream)
    # the restatement: per beam its own copied history of (key, value) as held in 8 bits
    hist = [[] for _ in range(R)]
    ints = [np.zeros((R, H, cap, d), np.int8) for _ in range(2)]
    scale = [np.zeros((R, H, cap // 32), np.float32) for _ in range(2)]
    done, tok, ids = np.zeros((B, W), np.uint8), np.zeros(R, np.int64), np.arange(R * 3).reshape(R, 3)
    for step in range(steps):
        i = step & 1
        hq, hk, hv = net.qkv(tok, step)
        for a, x in ((q, hq), (k, hk), (v, hv)):
            a.upload(x, stream)
        start.upload(np.full(R, step, np.int32), stream)
        length.upload(np.full(R, step + 1, np.int32), stream)
        append[i](stream)
        attend[i](stream)
        cross(stream)
        a, c = self_out.numpy(stream), cross_out.numpy(stream)
        # values held: every beam's slot, blocks requantised as they fill
        for z, x in ((0, hk), (1, hv)):
            ref.append(ints[z], scale[z], x, np.arange(R), np.full(R, step), np.ones(R))
        want_logits = np.zeros((R, V))
        for r in range(R):
            hist[r] = hist[r] + [(r, step)]
            sl, ps = (np.array(t) for t in zip(*hist[r]))
            K, Vv = ref.values(ints[0], scale[0], sl, ps), ref.values(ints[1], scale[1], sl, ps)
            keep = np.ones((1, step + 1), bool)
            ck = (np.arange(T) < enc_len[r // W])[None]
            parts = []
            for h in range(H):
                w1 = ref.attention(hq[r, :, h], K[:, h], Vv[:, h], d ** -0.5, keep)
                w2 = ref.attention(hq[r, :, h], enc_k[r // W, :, h], enc_v[r // W, :, h], d ** -0.5, ck)
                check = np.abs(a[r, :, h] - w1[0]) <= ref.attention_bound(w1, False, d)
                assert check.all() and (np.abs(c[r, :, h] - w2[0]) <= ref.attention_bound(w2, False, d)).all(), (step, r, h)
                parts += [w1[0], w2[0]]
            want_logits[r] = np.concatenate(parts, 1)[0] @ net.out
        lg = want_logits.reshape(B, W, V).astype(np.float32)
        logits.upload(lg, stream)
        select[i](stream)
        reorder[i](stream)
        want = ref.beam_select(lg, scores, done, end)
        got_p, got_t = parent.numpy(stream), token.numpy(stream)
        assert np.array_equal(got_p, want[0]) and np.array_equal(got_t, want[1]), step
        src = (want[0] + W * np.arange(B)[:, None]).reshape(-1)
        hist = [list(hist[s]) for s in src]
        ids = ids[src]
        scores, done, tok = sc[1 - i].numpy(stream), want[3], want[1].reshape(-1)
        assert np.array_equal(fin[1 - i].numpy(stream), done)
    assert np.array_equal(counts[steps & 1].numpy(stream), ids)
    print(f"[decoder] {steps} steps, scores {scores.min():.2f} .. {scores.max():.2f}", flush=True)


def _hip():
    h = C.CDLL("libamdhip64.so.7")       # the runtime that libpkx.so has loaded
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
    h.hipGraphExecDestroy.argtypes = [C.c_void_p]
    h.hipGraphDestroy.argtypes = [C.c_void_p]
    return h


def test_decoder_graph(gpu, stream):
    """A step captured into a graph and replayed on changed inputs, lengths among them, against the same calls made
    directly, with direct calls between the replays."""
    rng = np.random.default_rng(9)
    B, W, V, H, d, T, cap = 2, 3, 5000, 2, 64, 700, 1024
    R = B * W

    def make(c):
        return dict(q=gpu.DeviceArray((R, 1, H, d), np.float16), k=gpu.DeviceArray((R, 1, H, d), np.float16),
                    v=gpu.DeviceArray((R, 1, H, d), np.float16), o=gpu.DeviceArray((R, 1, H, d), np.float16),
                    o2=gpu.DeviceArray((B, W, H, d), np.float16), start=gpu.DeviceArray((R,), np.int32),
                    len=gpu.DeviceArray((R,), np.int32), logits=gpu.DeviceArray((B, W, V), np.float16),
                    sc=gpu.DeviceArray((B, W), np.float32), p=gpu.DeviceArray((B, W), np.int32),
                    t=gpu.DeviceArray((B, W), np.int32), ns=gpu.DeviceArray((B, W), np.float32),
                    tab=dev(gpu, np.zeros((R, cap), np.int32), stream), tab2=dev(gpu, np.zeros((R, cap), np.int32), stream), c=c)

    enc = [dev(gpu, rng.standard_normal((B, T, H, d)).astype(np.float16), stream) for _ in range(2)]
    base = [rng.integers(-127, 128, (R, H, cap, d)).astype(np.int8) for _ in range(2)]
    bsc = [rng.uniform(0.01, 0.03, (R, H, cap // 32)).astype(np.float32) for _ in range(2)]
    sides = [make(gpu.Cache8.wrap(*(dev(gpu, x, stream) for x in base + bsc))) for _ in range(2)]
    calls = []
    for s in sides:
        q2 = View(s["q"], 0, (B, W, H, d), (W * H * d, H * d, d))
        calls.append([gpu.CacheAppend(s["c"], s["k"], s["v"], s["start"], table=s["tab"]),
                      gpu.CacheAttention(s["c"], s["q"], s["o"], s["len"], table=s["tab"]),
                      gpu.CrossAttention(q2, *enc, s["o2"]),
                      gpu.BeamSelect(s["logits"], s["sc"], s["p"], s["t"], s["ns"]),
                      gpu.BeamReorder(s["p"], [(s["tab"], s["tab2"])])])
    for s, cs in zip(sides, calls):       # first calls outside the capture load the kernels
        for n, shape in (("q", None), ("k", None), ("v", None), ("logits", None), ("sc", None)):
            s[n].upload(np.zeros(s[n].shape, s[n].dtype), stream)
        s["start"].upload(i32([0] * R), stream)
        s["len"].upload(i32([1] * R), stream)
        for c in cs:
            c(stream)
    stream.sync()
    hip, graph, ex = _hip(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream.handle, 1) == 0
    for c in calls[0]:
        c(stream)
    assert hip.hipStreamEndCapture(stream.handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for step, n in enumerate((1, 33, 700, 64, 1000)):
        x = {k: rng.standard_normal(sides[0][k].shape).astype(sides[0][k].dtype) for k in ("q", "k", "v", "logits", "sc")}
        x["start"], x["len"] = i32([n - 1] * R), i32([n] * R)
        for s in sides:
            for k, a in x.items():
                s[k].upload(a, stream)
        assert hip.hipGraphLaunch(ex, stream.handle) == 0
        for c in calls[1]:
            c(stream)
        for k in ("o", "o2", "p", "t", "ns", "tab", "tab2"):
            assert np.array_equal(sides[0][k].numpy(stream), sides[1][k].numpy(stream)), (step, k)
        assert np.array_equal(sides[0]["c"].k.numpy(stream), sides[1]["c"].k.numpy(stream))
        print(f"[graph] replay {step}, length {n}: the same", flush=True)
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


def test_graph_allocates_nothing(gpu, stream):
    """The calls take no device memory of their own."""
    q, k, v = (gpu.DeviceArray((1, n, 2, 64), np.float16) for n in (1, 5000, 5000))
    for a in (q, k, v):
        a.upload(np.zeros(a.shape, np.float16), stream)
    out = gpu.DeviceArray(q.shape, np.float16)
    call = gpu.CrossAttention(q, k, v, out)
    call(stream)
    stream.sync()
    free0 = gpu.mem_info()[0]
    for _ in range(20):
        call(stream)
    stream.sync()
    assert gpu.mem_info()[0] == free0
