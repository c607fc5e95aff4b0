"""Size checks of the operators around a decoder's attention at the ends of their ranges, without a GPU."""
from test_block_cpu import _run

TILES = """
def tile(M, N, K, x_type=24):
    m, n, count = C.c_int(), C.c_int(), C.c_int64()
    a = lin(n_rows=M, n_out=N, n_in=K, x_type=x_type)
    assert L.pkx_linear_i8_tile(a, C.byref(m), C.byref(n), C.byref(count)) == 0
    return m.value, n.value, count.value
"""


def test_linear_tiles_can_be_launched():
    """Whatever sizes are taken, a launch has fewer than 2^32 threads."""
    out = _run(TILES + """
for M, N in ((262144, 262143), (262143, 262144), (1 << 14, (1 << 22) - 1), ((1 << 22) - 1, 1 << 14), ((1 << 22) - 1, 16257), (16383, 4194176), (200000, 300000), (1 << 20, 65535)):
    for K in (1, 16, 60, 100, 1000, 131071):
        for x_type in (24, 1, 0):
            m, n, count = tile(M, N, K, x_type)
            print(M, N, K, x_type, (m, n), count, count * (512 if m == 16 else 256) < 1 << 32 and count >= -(-M // m) * -(-N // n))
print(tile(0, 5, 5), tile(5, 0, 5), L.pkx_linear_i8_tile(lin(), None, None, None), L.pkx_linear_i8_tile(lin(n_rows=-1), *[C.byref(t()) for t in (C.c_int, C.c_int, C.c_int64)]))
""")
    assert len(out) == 8 * 6 * 3 + 1
    assert all(x.endswith("True") for x in out[:-1]), [x for x in out[:-1] if not x.endswith("True")]
    assert out[-1] == "(0, 0, 0) (0, 0, 0) 1 1"


def test_linear_tiles_are_all_tested():
    """The choice by sizes still sends each case of the GPU test to the tile that the case is there for, and no tile is without one."""
    from test_gpu_block_edges import TILES as cases
    sizes = [(c[2], c[3], c[4], {"i8": 24, "f": {"f16": 1, "f32": 0}[c[1]]}[c[9]]) for c in cases]
    out = _run(TILES + "for a in " + repr(sizes) + ": print(tile(*a)[:2])")
    assert out == [str(c[0]) for c in cases]
    assert {(c[0], c[1]) for c in cases} == {(t, d) for t in ((32, 128), (64, 128), (64, 256), (128, 256)) for d in ("f16", "f32")}
