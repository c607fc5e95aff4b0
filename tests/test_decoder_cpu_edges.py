"""Refusals and size checks of the attention decoder operators at the ends of their ranges, without a GPU."""
from test_decoder_cpu import _run


def test_clear_refusals():
    out = _run("""
        for c, n, slot in ((cache(n_slots=0), 1, None), (cache(k_scale=None), 1, None), (cache(capacity=100), 1, None), (cache(), -1, None),
                           (cache(), 4, None), (None, 1, None)):
            said(L.pkx_cache8_clear(c, n, slot, None))
        said(L.pkx_cache8_clear(cache(), 0, None, None))
        said(L.pkx_cache8_clear(cache(), 0, A, None))
    """)
    for line, w in zip(out[:6], ("no slots", "null", "capacity", "negative", "more rows", "null")):
        assert line.startswith("1 ") and w in line, (line, w)
    assert [x.strip() for x in out[6:]] == ["0"] * 2
