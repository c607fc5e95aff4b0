"""numpy restatements of the operators around a decoder's attention (block norm,
8-bit rows and products, rotary positions, rules on logits) in float64, with the
largest error that the kernels' roundings may add up to, element by element."""
import numpy as np

U = 2.0 ** -24          # half a step of f32
F32_MAX = np.finfo(np.float32).max


def rounded(err, value, f16):
    """err plus the rounding of value to the output's type (f16: 2^-11 of it, 2^-25 where it is subnormal)."""
    return err + (2.0 ** -11 * (np.abs(value) + err) + 2.0 ** -25 if f16 else U * (np.abs(value) + err)) + 1e-44


def normalised(x, ex, kind, w, b, eps):
    """The norm of rows x, known to within ex: (values, error)."""
    if kind == "none":
        return x, ex
    mean = x.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(x), 1))
    dx = x - mean
    var = (dx * dx).mean(1, keepdims=True) + eps
    inv = 1 / np.sqrt(var)
    w = np.ones(x.shape[1]) if w is None else np.asarray(w, np.float64)
    b = np.zeros(x.shape[1]) if b is None else np.asarray(b, np.float64)
    n = dx * inv * w
    # what comes in: through the value, the mean and (Cauchy-Schwarz) the variance
    rms = np.sqrt((ex * ex).mean(1, keepdims=True))
    err = np.abs(w) * inv * (ex + ex.mean(1, keepdims=True)) + np.abs(n) * inv * rms
    # what is added: the mean's f64 sums (2^-53 for each of up to 2^14 terms), x - mean in two subtractions, 1 / sqrt rounded to
    # f32 (from a variance that f64 keeps to 2^-25), two products and a sum
    spread = np.abs(dx).max(1, keepdims=True) + np.abs(x[:, :1] - mean)
    err = err + np.abs(w) * inv * 2.0 ** -38 * spread + 8 * U * np.abs(n) + U * np.abs(n + b) * (b != 0).any()
    return n + b, err


def block_norm(x, y, gate, per, fn, alpha, post, post_w, post_b, pre, pre_w, pre_b, post_eps, pre_eps):
    """-> (x', its f32 error, h, its f32 error), before any rounding to an output's type."""
    f = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
    x, y, gate = f(x), f(y), f(gate)
    if y is None:
        r, er = x, np.zeros_like(x)
    else:
        u, eu = normalised(y, np.zeros_like(y), post, post_w, post_b, post_eps)
        if gate is not None:
            g = gate[np.arange(len(y)) // per]
            eg = np.zeros_like(g)
            if fn == "sigmoid":     # exp to 2^-23, a sum and a division
                g = 1 / (1 + np.exp(-g))
                eg = 5 * U * g
            eu = np.abs(g) * eu + np.abs(u) * eg + U * np.abs(g * u)
            u = u * g
        r, er = alpha * u, abs(alpha) * eu + U * np.abs(alpha * u)
        if x is not None:
            r = r + x
            er = er + U * np.abs(r)
    h, eh = normalised(r, er, pre, pre_w, pre_b, pre_eps)
    return r, er, h, eh


def quantised(x):
    """Rows in 8 bits: (ints, scale), each step one f32 operation."""
    x = np.asarray(x, np.float32)
    a = np.where(np.abs(x) <= F32_MAX, np.abs(x), np.float32(0))
    s = (a.max(1, initial=0) / np.float32(127)).astype(np.float32)
    with np.errstate(all="ignore"):
        q = np.rint(x / np.where(s == 0, np.float32(1), s)[:, None])
    q = np.clip(np.nan_to_num(q, nan=0.0, posinf=127, neginf=-127), -127, 127)
    return np.where(s[:, None] == 0, 0, q).astype(np.int8), s


def linear_i8(q, s, w, ws, bias, act, alpha, add, f16=False):
    """-> (y, its f32 error) of ints q [M][K], w [N][K]; the sums are whole numbers."""
    acc = (q.astype(np.float64) @ w.astype(np.float64).T)
    v = acc * s.astype(np.float64)[:, None] * ws.astype(np.float64)[None]
    err = 4 * U * np.abs(v)
    if bias is not None:
        v = v + bias.astype(np.float64)
        err = err + U * np.abs(v)
    if act == "silu":
        y = v / (1 + np.exp(-v))
        # |d silu / dv| <= 1.1; then e^-v to 3 U (the hardware's exponential to a unit in the last place, 2 U, and a product), whose
        # share of 1 + e^-v is at most 1, that sum (U), its reciprocal (U after a Newton step) and the product (U).  An f16 result takes
        # the exponential of v log2 e rounded once (|v| U) and a reciprocal to a unit in the last place (2 U).
        err, v = 1.1 * err + (6 + (1 + np.abs(v) if f16 else 0)) * U * np.abs(y), y
    v, err = alpha * v, abs(alpha) * err + U * np.abs(alpha * v)
    if add is not None:
        v = v + add.astype(np.float64)
        err = err + U * np.abs(v)
    return v, err


def rotary(x, pos, freq, rot, interleaved, mult):
    """x [n][H][d] of tokens at pos [n] -> (values, f32 error)."""
    x = np.asarray(x, np.float64)
    angle = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freq)
    first = np.arange(rot // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rot // 2)
    y, err = x.copy(), np.zeros_like(x)
    a, b, c, s = x[..., first], x[..., second], np.cos(angle), np.sin(angle)
    y[..., first], y[..., second] = mult * (a * c - b * s), mult * (b * c + a * s)
    # sine and cosine: the reduced angle, five steps and the scale in f32, the angle's own f64 products; then two products and a sum
    e = (np.abs(a) + np.abs(b)) * abs(mult) * (9 * U + 2.0 ** -51 * (np.abs(angle) + 8))
    err[..., first] = err[..., second] = e
    return y, err


def rules(x, counts, rep, pres, freq, bias, mask):
    """One row: x [V], counts [V] -> (values, f32 error); mask [V] truth values."""
    x = np.asarray(x, np.float64)
    rep, pres, freq = (float(np.float32(a)) for a in (rep, pres, freq))
    with np.errstate(all="ignore"):
        pen = np.where(x > 0, x / rep, x * rep)
        y = np.where(counts > 0, pen - pres - freq * counts, x)
        err = np.where(counts > 0, U * (np.abs(pen) + np.abs(pen - pres) + np.abs(freq * counts) + np.abs(y)), 0)
        if bias is not None:
            y = y + bias.astype(np.float64)
            err = err + U * np.abs(y)
    if mask is not None:
        y = np.where(mask, y, -np.inf)
    return y, np.where(np.isfinite(y), err, 0)
