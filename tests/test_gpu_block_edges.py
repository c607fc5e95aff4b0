"""The operators around a decoder's attention where their sizes, addresses or values are at an end, against block_ref.py."""
import numpy as np
import pytest

import block_ref as ref
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
