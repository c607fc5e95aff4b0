"""numpy restatements of the attention decoder operators: float64 for what is
computed, float32 step by step for what is held in 8 bits."""
import numpy as np

BLOCK = 32


def attention(q, k, v, scale, keep):
    """q [n][d], k, v [t][d], keep [n][t] -> (out [n][d], bound terms): float64, zeros for rows with nothing kept.

    The second value is (a, spread): a = sum p |v| and spread = sum over kept keys of |v|, per output element, and
    the largest |score| in nats, from which the tests derive their bounds."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    s = np.where(keep, q @ np.where(keep.any(0)[:, None], k, 0).T * scale, -np.inf)
    m = s.max(1, initial=-np.inf)[:, None]
    p = np.exp(s - np.where(np.isfinite(m), m, 0))
    l = p.sum(1, keepdims=True)
    p = p / np.where(l == 0, 1, l)
    v = np.where(keep.any(0)[:, None], v, 0)
    top = np.abs(np.where(np.isfinite(s), s, 0)).max(1, initial=0)[:, None]
    mass = np.abs(q) @ np.abs(np.where(keep.any(0)[:, None], k, 0)).T * abs(scale)
    mass = np.where(keep, mass, 0).max(1, initial=0)[:, None]
    return p @ v, p @ np.abs(v), np.where(keep, 1.0, 0.0) @ np.abs(v), top, mass


def attention_bound(ref, f16, d):
    """Largest error of the kernels per element, by arithmetic: see the terms."""
    o, a, spread, top, mass = ref
    u = 2.0 ** -24
    # a score is a sum of d products in f32 (d + 2 roundings of at most `mass`), scaled, minus a maximum that carries
    # the same error, through a 1-ulp exponential: the weight's relative error, doubled for the division by the sum
    w = 2 * (2 * (d + 4) * u * mass + 4 * u * top + 8 * u)
    err = a * w + 64 * u * a
    if f16:     # weights rounded to 11 bits (absolutely 2^-25 where they are subnormal), the output too
        err = err + 2.0 ** -11 * a + 2.0 ** -25 * spread + 2.0 ** -11 * np.abs(o) + 2.0 ** -25
    else:       # f32 queries on int8 keys: both factors carry 22 bits
        err = err + 2.0 ** -21 * a + 2 * 2.0 ** -21 * mass * a + 2.0 ** -24 * np.abs(o)
    return err + 1e-30


def append(ints, scales, x, slot, start, count):
    """ints [S][H][cap][d] int8, scales [S][H][cap/32], x [R][n][H][d]: appended in place."""
    f = np.float32
    seen = set()
    cap = ints.shape[2]
    for r in range(x.shape[0]):
        s0, sl = int(start[r]), int(slot[r])
        n = min(max(int(count[r]), 0), x.shape[1])
        first = sl not in seen
        seen.add(sl)
        if not (0 <= s0 < cap and 0 <= sl < ints.shape[0] and first):
            continue
        end = min(s0 + n, cap)
        for b in range(s0 // BLOCK, (end + BLOCK - 1) // BLOCK if end > s0 else 0):
            lo, hi = max(s0, b * BLOCK), min(end, (b + 1) * BLOCK)
            if lo >= hi:
                continue
            for h in range(ints.shape[1]):
                new = x[r, lo - s0:hi - s0, h].astype(f)
                a = np.abs(new)
                a = a[a <= np.finfo(f).max]
                top = f(a.max() if a.size else 0) / f(127)
                before = scales[sl, h, b] if lo > b * BLOCK else f(0)
                s = np.maximum(before, top)
                ratio = before / s if s != 0 else f(0)
                if lo > b * BLOCK and ratio != 1:
                    old = ints[sl, h, b * BLOCK:lo]
                    ints[sl, h, b * BLOCK:lo] = np.rint(old.astype(f) * ratio)
                with np.errstate(all="ignore"):
                    q = np.rint(new / s) if s != 0 else np.zeros_like(new)
                ints[sl, h, lo:hi] = np.clip(np.nan_to_num(q, nan=0.0, posinf=127, neginf=-127), -127, 127)
                scales[sl, h, b] = s


def values(ints, scales, slot, pos):
    """float32 values of positions pos of slots slot (same shapes) -> [...][H][d]."""
    return ints[slot, :, pos].astype(np.float32) * scales[slot, :, np.asarray(pos) // BLOCK][..., None]


def beam_select(logits, scores, done, end):
    """[B][W][V] -> parent, token, score (float64), done: [B][W]."""
    B, W, V = logits.shape
    out = [np.zeros((B, W), t) for t in (np.int32, np.int32, np.float64, np.uint8)]
    for b in range(B):
        cand = []
        for w in range(W):
            s = float(scores[b, w])
            s = s if s < np.inf else -np.inf
            if done is not None and done[b, w]:
                cand.append((-s, w, end))
                continue
            x = logits[b, w].astype(np.float64)
            dead = np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all() or s == -np.inf
            if dead:
                cand += [(np.inf, w, v) for v in range(min(V, W))]
                continue
            z = x.max() + np.log(np.exp(x - x.max()).sum())
            cand += [(-(s + (x[v] - z)), w, int(v)) for v in np.argsort(-x, kind="stable")[:W]]
        for i, (c, w, v) in enumerate(sorted(cand)[:W]):
            out[0][b, i], out[1][b, i], out[2][b, i] = w, v, -c
            out[3][b, i] = int(bool(done is not None and done[b, w]) or v == end)
    return out
