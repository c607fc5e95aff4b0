"""The attention decoder operators where their arithmetic or their addresses are at an end, against decoder_ref.py."""
import numpy as np
import pytest

import decoder_ref as ref
from test_gpu_decoder import HostCache as DecoderCache, check_attention, dev, i32

pytestmark = pytest.mark.gpu


class HostCache(DecoderCache):
    def same_scales(self, stream):
        for a, b in ((self.dev.k_scale, self.ks), (self.dev.v_scale, self.vs)):
            assert np.array_equal(a.numpy(stream), b, equal_nan=True)


def small_weights(q, k, v, scale, keep, least):
    """sum over kept keys of min(p, least) |v|: what rounding weights to multiples of `least` may lose."""
    s = np.where(keep, np.asarray(q, np.float64) @ np.asarray(k, np.float64).T * scale, -np.inf)
    p = np.exp(s - s.max(1, keepdims=True))
    return np.minimum(p, least) @ np.abs(np.asarray(v, np.float64))


def check_scaled(got, q, k, v, scale, keep, f16, d, label):
    """Within the roundings of every key's own block, however large the other blocks' values are: the bound of
    decoder_ref with a weight's absolute error at most 2^-32 (a sixteen-bit term of 2^14 p r, r at least 2^-7, is
    off by 2^-25 at most where it is subnormal) and never more than the weight."""
    want = list(ref.attention(q, k, v, scale, keep))
    low = small_weights(q, k, v, scale, keep, 2.0 ** -32)
    want[2] = 0 * want[2]
    err, bound = np.abs(got.astype(np.float64) - want[0]), ref.attention_bound(want, f16, d) + low
    worst = float((err / bound).max())
    print(f"[{label}] largest error {err.max():.2e} of values up to {np.abs(want[0]).max():.2e}, {worst:.2f} of its bound", flush=True)
    assert np.isfinite(got).all() and worst <= 1.0


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("nq", [2, 256])
@pytest.mark.parametrize("d", [80, 128])
def test_cache_blocks_of_small_values_next_to_large_ones(gpu, stream, type, nq, d):
    """Rows whose weights all lie in one block with values 2^40 below the other blocks' (few rows, and enough for the
    many-row kernel): first, last, either half of a 64-key step."""
    print(f"[scales] {type} nq={nq} d={d}", flush=True)
    rng = np.random.default_rng(nq + d)
    R, H, n = 4, 16, 1920
    c = HostCache(gpu, stream, R, H, n, d, rng)
    wanted = [0, n // 32 - 1, 20, 33]
    c.k[:] = 0
    c.k[..., 1] = rng.integers(-127, 128, c.k.shape[:-1])
    c.ks[:] = 2.0 ** -7
    c.vs[:] = 2.0 ** 34 * rng.uniform(0.6, 1, c.vs.shape)
    for r, b in enumerate(wanted):
        c.k[r, :, 32 * b:32 * b + 32, 0] = 127
        c.vs[r, :, b] = 2.0 ** -6 * rng.uniform(0.6, 1, H)
    for a, x in ((c.dev.k, c.k), (c.dev.k_scale, c.ks), (c.dev.v_scale, c.vs)):
        a.upload(x, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = np.zeros((R, nq, H, d), dt)
    q[..., 0] = 101          # other blocks: weights e^-100
    q[..., 1] = rng.standard_normal(q.shape[:-1])
    out = gpu.DeviceArray(q.shape, dt)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream), causal=False, scale=1.0)(stream)
    got = out.numpy(stream)
    for r in range(R):
        K, V = (ref.values(x, y, np.full(n, r), np.arange(n)) for x, y in ((c.k, c.ks), (c.v, c.vs)))
        for h in (0, H - 1):
            check_scaled(got[r, :, h], q[r, :, h], K[:, h], V[:, h], 1.0, np.ones((nq, n), bool), type == "f16", d, f"r{r} h{h}")


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_cache_blocks_that_a_row_does_not_see(gpu, stream, type):
    """Causal rows in front of a block whose values are 2^40 times those that they see."""
    rng = np.random.default_rng(40)
    R, H, n, nq, d = 4, 16, 1920, 256, 128
    c = HostCache(gpu, stream, R, H, n, d, rng)
    first = [n - 32, n - 64, n - 128, n - 160]
    c.vs[:] = 2.0 ** -6 * rng.uniform(0.6, 1, c.vs.shape)
    for r, t in enumerate(first):
        c.vs[r, :, t // 32:] = 2.0 ** 34
    c.dev.v_scale.upload(c.vs, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = (rng.standard_normal((R, nq, H, d)) * 0.7).astype(dt)
    out = gpu.DeviceArray(q.shape, dt)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream))(stream)
    got = out.numpy(stream)
    for r in range(R):
        K, V = (ref.values(x, y, np.full(n, r), np.arange(n)) for x, y in ((c.k, c.ks), (c.v, c.vs)))
        m = first[r] - (n - nq)          # rows that see nothing of it
        keep = np.arange(n)[None] <= (n - nq + np.arange(m))[:, None]
        for h in (0, H - 1):
            check_scaled(got[r, :m, h], q[r, :m, h], K[:, h], V[:, h], d ** -0.5, keep, type == "f16", d, f"r{r} h{h}")


def test_new_cache_is_clear(gpu, stream):
    """The scales of a new cache are zeros, whatever the memory held."""
    old = [gpu.DeviceArray((3, 2, 64 // 32), np.float32) for _ in range(64)]
    for a in old:
        a.upload(np.full(a.shape, np.nan, np.float32), stream)
    del old, a
    for _ in range(8):
        c = gpu.Cache8(3, 2, 32, 64)
        assert not c.k_scale.numpy(stream).any() and not c.v_scale.numpy(stream).any()


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("prompt,d", [(50, 64), (33, 48), (31, 128)])
def test_beams_share_a_prompt_in_slots_that_held_another_sequence(gpu, stream, type, prompt, d):
    """A prompt in one slot that the beams' tables name, every beam's tokens from there on in its own slot, whose scales
    are another sequence's (large, NaN) until they are cleared; a slot of another item is left as it was."""
    print(f"[prompt] {type} {prompt} d={d}", flush=True)
    rng = np.random.default_rng(prompt)
    W, H, cap, steps = 4, 2, 128, 20
    c = HostCache(gpu, stream, W + 2, H, cap, d, rng)
    c.ks[:], c.vs[:] = 1e6, np.nan
    c.dev.k_scale.upload(c.ks, stream)
    c.dev.v_scale.upload(c.vs, stream)
    slots = i32([4, 0, 3, 1])
    gpu.CacheClear(c.dev, dev(gpu, i32([4, 0, -1, 3, 1, W + 2, 0]), stream))(stream)
    c.ks[slots], c.vs[slots] = 0, 0
    c.same_scales(stream)
    dt = np.float16 if type == "f16" else np.float32
    table, slot = dev(gpu, np.full((W, cap), -1, np.int32), stream), dev(gpu, slots, stream)
    where = np.full((W, cap), -1)
    where[:, :prompt] = slots[0]
    x = [rng.standard_normal((1, prompt, H, d)).astype(dt) for _ in range(2)]
    gpu.CacheAppend(c.dev, *(dev(gpu, a, stream) for a in x), start=dev(gpu, i32([0]), stream), slot=dev(gpu, slots[:1], stream))(stream)
    for ints, scale, a in ((c.k, c.ks, x[0]), (c.v, c.vs, x[1])):
        ref.append(ints, scale, a, slots[:1], [0], [prompt])
    table.upload(i32(where), stream)
    for t in range(prompt, prompt + steps):
        x = [rng.standard_normal((W, 1, H, d)).astype(dt) for _ in range(3)]
        gpu.CacheAppend(c.dev, *(dev(gpu, a, stream) for a in x[:2]), start=dev(gpu, i32([t] * W), stream), slot=slot, table=table)(stream)
        for ints, scale, a in ((c.k, c.ks, x[0]), (c.v, c.vs, x[1])):
            ref.append(ints, scale, a, slots, [t] * W, [1] * W)
        where[:, t] = slots
        out = gpu.DeviceArray((W, 1, H, d), dt)
        gpu.CacheAttention(c.dev, dev(gpu, x[2], stream), out, dev(gpu, i32([t + 1] * W), stream), table=table)(stream)
        got = out.numpy(stream)
        for r in range(W):
            K, V = (ref.values(a, b, where[r, :t + 1], np.arange(t + 1)) for a, b in ((c.k, c.ks), (c.v, c.vs)))
            for h in range(H):
                want = ref.attention(x[2][r, :, h], K[:, h], V[:, h], d ** -0.5, np.ones((1, t + 1), bool))
                check_attention(got[r, :, h], want, type == "f16", d, f"t{t} r{r} h{h}")
    c.same_scales(stream)
    assert np.array_equal(c.dev.k.numpy(stream), c.k) and np.array_equal(c.dev.v.numpy(stream), c.v)
    back = gpu.DeviceArray((W, steps, H, d), np.float32)
    gpu.CacheRead(c.dev, back, None, start=dev(gpu, i32([prompt] * W), stream), slot=slot)(stream)
    for r in range(W):
        assert np.array_equal(back.numpy(stream)[r], ref.values(c.k, c.ks, np.full(steps, slots[r]), prompt + np.arange(steps)))
    gpu.CacheClear(c.dev)(stream)
    assert not c.dev.k_scale.numpy(stream).any() and not c.dev.v_scale.numpy(stream).any()


@pytest.mark.parametrize("nq", [2, 256])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_f32_queries_with_large_scores_on_the_cache(gpu, stream, nq, scale):
    """Scores of 8128 nats whose keys differ by one at most, formed without a rounding but for the factors: a weight is
    off by the roundings of its exponent, its two terms and the sums, not by 2^-24 of the score."""
    rng = np.random.default_rng(nq)
    R, H, n, d = 4, 16, 1920, 128
    c = HostCache(gpu, stream, R, H, n, d, rng)
    c.k[:] = 0
    at = 32 * np.arange(n // 32) + rng.integers(0, 32, n // 32)      # one key a block
    c.k[:, :, at, 0] = 127
    c.ks[:] = 1 + rng.integers(0, 1 << 10, c.ks.shape) * 2.0 ** -23
    for a, x in ((c.dev.k, c.k), (c.dev.k_scale, c.ks)):
        a.upload(x, stream)
    q = np.zeros((R, nq, H, d), np.float32)
    q[..., 0] = 64 * scale
    out = gpu.DeviceArray(q.shape, np.float32)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream), causal=False, scale=scale)(stream)
    got, worst = out.numpy(stream).astype(np.float64), 0.0
    for r in range(R):
        K, V = (x[r].astype(np.float64) * np.repeat(y[r].astype(np.float64), 32, 1)[..., None] for x, y in ((c.k, c.ks), (c.v, c.vs)))
        for h in (0, H - 1):
            o, a = ref.attention(q[r, :, h], K[h], V[h], scale, np.ones((nq, n), bool))[:2]
            # a weight: 2^-22 of two terms, 2^-23 each of its exponential and of exponents below 1; n / 32 sums of
            # 2^-24 and rescalings of as much; all of it once more in the sum that divides
            bound = a * 2 * (2.0 ** -22 + 2 * 2.0 ** -23 + 2 * (n // 32) * 2.0 ** -24)
            worst = max(worst, float((np.abs(got[r, :, h] - o) / bound).max()))
    print(f"[large scores] nq={nq} {worst:.2f} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("nq", [2, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_one_dominating_key_of_the_cache_is_exact_in_f16(gpu, stream, nq, causal):
    """A weight of 1 (the others' sum is below 2^-100) is exact in f16, whatever the blocks' scales: the output is the
    key's value rounded to f16, half a step of 2^-11, and a few f32 roundings."""
    rng = np.random.default_rng(nq + causal)
    R, H, n, d = 4, 16, 1920, 128
    c = HostCache(gpu, stream, R, H, n, d, rng)
    c.k[:] = 0
    at = np.array([5, 32 * 7 + 31, 32 * 40, n - 257])
    c.k[np.arange(R), :, at, 0] = 127
    c.ks[:] = 1
    for a, x in ((c.dev.k, c.k), (c.dev.k_scale, c.ks)):
        a.upload(x, stream)
    q = np.zeros((R, nq, H, d), np.float16)
    q[..., 0] = 1
    out = gpu.DeviceArray(q.shape, np.float16)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream), causal=causal, scale=1.0)(stream)
    got = out.numpy(stream).astype(np.float64)
    for r in range(R):
        v = c.v[r, :, at[r]].astype(np.float64) * c.vs[r, :, at[r] // 32, None]
        assert (np.abs(got[r] - v[None]) <= (2.0 ** -11 + 2.0 ** -17) * np.abs(v) + 2.0 ** -25).all(), r


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("d", [32, 48, 128])
def test_cache_far_slots_by_table(gpu, stream, type, d):
    """Slots that together pass 2 GiB (3 of 2^30 bytes), rows that mix them by table up to the last position, entries out
    of range between; every width of the kernel's loads."""
    print(f"[far table] {type} d={d}", flush=True)
    rng = np.random.default_rng(d)
    S, H, G = 3, 2, 2
    cap = (1 << 29) // d // 32 * 32
    k, v = gpu.DeviceArray((S, H, cap, d), np.int8), gpu.DeviceArray((S, H, cap, d), np.int8)
    assert S * H * cap * d > 1 << 31
    sc = [rng.uniform(0.005, 0.02, (S, H, cap // 32)).astype(np.float32) for _ in range(2)]
    c = gpu.Cache8.wrap(k, v, *(dev(gpu, a, stream) for a in sc))
    pos = np.concatenate([a + np.arange(40) for a in (0, cap // 2 + 5, cap - 40)])
    ints = [rng.integers(-127, 128, (S, H, len(pos), d)).astype(np.int8) for _ in range(2)]
    for a, x in ((k, ints[0]), (v, ints[1])):
        for s in range(S):
            for h in range(H):
                for i in range(0, len(pos), 40):
                    run = np.ascontiguousarray(x[s, h, i:i + 40])
                    gpu.check(gpu.lib().pkx_memcpy_h2d(a.ptr + ((s * H + h) * cap + int(pos[i])) * d, run.ctypes.data, run.nbytes, stream.handle))
    table = np.full((2, cap), -1, np.int32)
    table[1] = S
    who = rng.integers(-1, S + 1, (2, len(pos)))
    who[:, ::5] = 2
    table[:, pos] = who
    dt = np.float16 if type == "f16" else np.float32
    q = rng.standard_normal((2, 1, H * G, d)).astype(dt)
    out = gpu.DeviceArray(q.shape, dt)
    lens = [cap, cap - 3]
    gpu.CacheAttention(c, dev(gpu, q, stream), out, dev(gpu, i32(lens), stream), table=dev(gpu, table, stream))(stream)
    got = out.numpy(stream)
    for r in range(2):
        keep = (who[r] >= 0) & (who[r] < S) & (pos < lens[r])
        sl = np.where(keep, who[r], 0)
        K, V = (x[sl, :, np.arange(len(pos))] * y[sl, :, pos // 32][..., None] for x, y in zip(ints, sc))
        for h in range(H * G):
            want = ref.attention(q[r, :, h], K[:, h // G], V[:, h // G], d ** -0.5, keep[None])
            check_attention(got[r, :, h], want, type == "f16", d, f"far table r{r} h{h}")


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("R,nq,H,n,d,table", [(2, 3, 4, 130, 64, False), (2, 3, 4, 130, 48, True), (4, 256, 16, 1920, 128, False)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("causal", [False, True])
def test_cache_attention_scales(gpu, stream, type, R, nq, H, n, d, table, scale, causal):
    """Any factor on 8-bit keys: negative, zero (the mean of the seen values), large; few rows, by table, many rows."""
    rng = np.random.default_rng(n + nq)
    c = HostCache(gpu, stream, R, H, (n + 31) // 32 * 32, d, rng)
    dt = np.float16 if type == "f16" else np.float32
    q = rng.standard_normal((R, nq, H, d)).astype(dt)
    out, tab = gpu.DeviceArray(q.shape, dt), rng.integers(-1, R, (R, n)).astype(np.int32)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream), causal=causal, scale=scale, max_len=n,
                       table=dev(gpu, tab, stream) if table else None)(stream)
    got, pos = out.numpy(stream), np.arange(n)
    for r in (0, R - 1):
        where = tab[r] if table else np.full(n, r)
        K, V = (ref.values(x, y, np.maximum(where, 0), pos) for x, y in ((c.k, c.ks), (c.v, c.vs)))
        keep = np.broadcast_to(where >= 0, (nq, n))
        if causal:
            keep = keep & (pos[None] <= (n - nq + np.arange(nq))[:, None])
        for h in (0, H - 1):
            # at scale 3 most weights are tiny, and some outputs are made of them alone.  A weight goes to f16 (f32: a
            # second term) as 2^14 p, or by table as 2^14 p v / (largest p v of the tile), v the block's value scale: where
            # that is subnormal the step is 2^-24 and half of it 2^-39 of the largest, times at most 50 by the
            # table for the scales of 0.001 to 0.05 here: below 2^-33, and check_scaled allows 2^-32
            check_scaled(got[r, :, h], q[r, :, h], K[:, h], V[:, h], scale, keep, type == "f16", d, f"scale {scale} r{r} h{h}")


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("nq", [2, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_cache_blocks_of_scale_zero(gpu, stream, type, nq, causal):
    """Blocks whose value or key scale is 0, whatever integers stand there: first ones, both or one half of a step, all;
    tiny and large scales between them."""
    rng = np.random.default_rng(nq)
    R, H, n, d = 4, 16, 1920, 128
    c = HostCache(gpu, stream, R, H, n, d, rng)
    c.vs[0] = 0
    c.vs[1, :, :5] = 0
    c.vs[2, :, ::2] = 0
    c.vs[2, :, 1::4] *= 2.0 ** -9
    c.vs[3, :, 2:] = 0
    c.ks[1, :, 7:20] = 0
    c.ks[2] = 0
    for a, x in ((c.dev.k_scale, c.ks), (c.dev.v_scale, c.vs)):
        a.upload(x, stream)
    dt = np.float16 if type == "f16" else np.float32
    q = (rng.standard_normal((R, nq, H, d)) * 0.7).astype(dt)
    out = gpu.DeviceArray(q.shape, dt)
    gpu.CacheAttention(c.dev, dev(gpu, q, stream), out, dev(gpu, i32([n] * R), stream), causal=causal)(stream)
    got, pos = out.numpy(stream), np.arange(n)
    assert not got[0].any()
    for r in range(R):
        K, V = (ref.values(x, y, np.full(n, r), pos) for x, y in ((c.k, c.ks), (c.v, c.vs)))
        keep = np.ones((nq, n), bool)
        if causal:
            keep = keep & (pos[None] <= (n - nq + np.arange(nq))[:, None])
        for h in (0, H - 1):
            check_scaled(got[r, :, h], q[r, :, h], K[:, h], V[:, h], d ** -0.5, keep, type == "f16", d, f"zero scales r{r} h{h}")
