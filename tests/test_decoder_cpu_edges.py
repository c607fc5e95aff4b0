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


def test_reorder_refuses_rows_past_the_address_space_and_a_written_parent():
    """Strides whose span wraps 64 bits would hide an overlap; a destination over parent would be read while written."""
    out = _run("""
        S = pkx.BeamState
        def order(states, B=1, W=5):
            said(L.pkx_beam_reorder(A, B, W, (S * len(states))(*states), len(states), None))
        order([S(A + (1 << 30), A + (1 << 20), 16, 1 << 62, 16)])
        order([S(A + (1 << 30), A + (1 << 20), 1 << 62, 16, 16)])
        order([S(A + (1 << 30), A + (1 << 20), 16, 16, 16), S(A + (1 << 25), A + (1 << 26), 1 << 62, 16, 16)])
        order([S(A + (1 << 20), A, 16, 16, 16)])
        order([S(A + (1 << 20), A + 16, 16, 16, 4)])
        order([S(A + (1 << 20), A - 64, 16, 16, 16)])
        order([S(A, A + 20, 4, 4, 4)], B=0)
    """)
    for line, w in zip(out[:6], ["address space"] * 3 + ["parent"] * 3):
        assert line.startswith("1 ") and w in line, (line, w)
    assert out[6].strip() == "0"
