"""The 4-bit element from its definition, in numpy: what the tests of the device's rows and contexts compare with."""
import numpy as np

GROUP = 32
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def stored(rows, head_dim):
    """What rows [n, heads * head_dim] are worth once stored, in 64 bits: per group of 32 dims of a head the smallest power
    2^e with max |x| <= 7 * 2^e, e in [-125, 125], and x / 2^e at the nearest of LEVELS, ties to the even index; NaN for a group
    that is not finite."""
    x = np.asarray(rows, np.float32).astype(np.float64)
    n = x.shape[0]
    x = x.reshape(n, -1, head_dim)
    out = np.empty_like(x)
    for d in range(0, head_dim, GROUP):
        part = x[:, :, d:d + GROUP]
        top = np.abs(part).max(-1, keepdims=True)
        finite = np.isfinite(top)
        safe = np.where(finite, top, 1.0)
        m, e = np.frexp(safe / 7.0)  # in [1/2, 1) times 2^e: the power is 2^e, or 2^(e - 1) where m is 1/2
        e = np.clip(np.where(m == 0.5, e - 1, e), -125, 125)
        e = np.where(safe == 0.0, -125, e)
        scale = np.ldexp(1.0, e)
        y = np.where(finite, np.abs(part), 0.0) / scale
        far = np.abs(y[..., None] - LEVELS)
        best = far.min(-1, keepdims=True)
        near = far == best  # one level, or two at a tie: the even one
        idx = np.where(near.sum(-1) > 1, np.where(near, (np.arange(8) % 2 == 0) * 8 + 1, 0).argmax(-1), near.argmax(-1))
        value = np.copysign(LEVELS[idx] * scale, part)
        out[:, :, d:d + GROUP] = np.where(finite, value, np.nan)
    return out.reshape(n, -1)


def attention(q, keys, values, dims, first=None, window=0, window_start=0, attn_scalar=None):
    """Rows q [n, q_heads * hd] over stored rows [len, kv_dim] (64 bits): contexts, and the bound that `tolerance` gives each of
    their values. Row i is at position len - n + i (or first + i) and sees positions up to its own, through the window."""
    q_heads, kv_heads, hd = dims
    q = np.asarray(q, np.float32).reshape(-1, q_heads, hd)
    k = keys.reshape(-1, kv_heads, hd)
    v = values.reshape(-1, kv_heads, hd)
    n = q.shape[0]
    first = len(k) - n if first is None else first
    out, tol = np.empty(q.shape), np.empty(q.shape)
    scale = 1.0 / np.sqrt(attn_scalar or hd)
    pos = first + np.arange(n)
    at = np.arange(len(k))
    # rows of queries at a time; one where there are NaN, which are not to reach the rows in front of them
    block = 64 if np.isfinite(k).all() and np.isfinite(v).all() else 1
    for kh in range(kv_heads):
        heads = range(kh * q_heads // kv_heads, (kh + 1) * q_heads // kv_heads)
        for i0 in range(0, n, block):
            rows = slice(i0, min(i0 + block, n))
            lo = max(window_start, pos[i0] + 1 - window if window else 0)
            hi = pos[rows][-1] + 1
            kk, vv = k[lo:hi, kh], v[lo:hi, kh]
            seen = (at[None, lo:hi] <= pos[rows, None]) & (at[None, lo:hi] >= window_start)
            if window:
                seen &= at[None, lo:hi] > pos[rows, None] - window
            for h in heads:
                x = q[rows, h].astype(np.float64) * scale
                s = x @ kk.T
                m = np.where(seen, s, -np.inf).max(-1, keepdims=True)
                p = np.where(seen, np.exp(np.where(seen, s, m) - m), 0.0)
                total = p.sum(-1, keepdims=True)
                p /= total
                out[rows, h] = p @ vv
                tol[rows, h] = _bound(x, kk, s, seen, vv)[:, None] * (p @ np.abs(vv)) + 2.0 ** -29 * (seen @ np.abs(vv)) / total + 1e-37
    return out.reshape(n, -1), tol.reshape(n, -1)


def _bound(x, k, s, seen, v):
    """Relative to the weighted mean of |v|, how far a context may be off.

    A query value is five terms. The last of them leaves 2^-22 of the first term's power at most, a power that is at least the
    group's largest value over 7.5 and at most that over 3.75: 2^-23.9 of the largest value, one way or the other, so that dims are
    off independently of each other and a score by six of its standard deviations at most (the times log2(e) and back of base 2
    are in the 2^-24 below). Sums of at most 16 products and roundings of the score: 8 halves of a step of 32 bits of the sum of
    magnitudes. A score off by d moves the weights by 2 d relative to their sum. The weights are two terms of f16, off by half a step of
    half a step, 2^-22, or, where V has powers outside 2^-15 to 2^16 (largest values in 3.5 times the one to 7 times the other), of
    bf16, 2^-18. The exponential is off by 2^-22, sums of up to some thousand keys in partials of a few dozen by 2^-20 together.

    Beside that (`attention`): f16's steps end at 2^-24. A weight is held at 2^8 times itself, relative to a base that is at most 2^4
    above the largest, so that it is off by half of such a step over 2^8, 2^-33, times 2^4: 2^-29 of the largest weight."""
    top = np.stack([np.abs(v[:, d:d + GROUP]).max(-1) for d in range(0, v.shape[1], GROUP)])
    top = top[top > 0]
    far = top.size > 0 and (top.min() <= 3.5 * 2.0 ** -15 or top.max() > 6 * 2.0 ** 16)
    var = np.zeros(s.shape)
    for d in range(0, x.shape[1], GROUP):
        step = np.abs(x[:, d:d + GROUP]).max(-1) * 2.0 ** -23.9
        var += step[:, None] ** 2 / 3.0 * (k[:, d:d + GROUP] ** 2).sum(-1)[None]
    ds = 6.0 * np.sqrt(var) + (np.abs(x) @ np.abs(k).T + np.abs(s)) * 8 * 2.0 ** -24
    return 2.0 * np.where(seen, ds, 0.0).max(-1) + (2.0 ** -18 if far else 2.0 ** -22) + 2.0 ** -22 + 2.0 ** -20
