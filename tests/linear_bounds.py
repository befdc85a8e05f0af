"""Linear attention with a decay, token by token in 64 bits, and how far a kernel may be off whose factors have all of f32's 24 bits,
whatever lies beside them.

    S_t = exp(g_t) S_(t-1) + k_t v_t^T,   o_t = scale * S_t^T q_t

u = 2^-24, half a step of f32. A factor is the sum of three bf16 terms, exactly: the first leaves at most 2^-8 of it in 16 bits, the second 2^-16 of it in
8. Of a product of two, the three smallest of the nine products of terms are left out: 2 * 2^-24 and less, 3 u with the third. What a term holds below 2^-126
may count as 0: FLUSH, times the other factor.

A is the state of absolute values, E what the computed state may be off. `step` tokens apart (32: a chunk; 1: the recurrence) the old state is multiplied by an
exponential good to 4 u (two steps of f32, of an argument below one that is rounded once) and rounded twice: 8 u with what a sum over parts
adds. A new product k v: k times an exponential, 4 + 1 u, the terms left out, 3 u. An output: a score or the state times q, twice the terms left out,
6 u, the exponential and the product with it and the scale, 4 + 2 u, the terms left out of the weights' product with v, 3 u, the sum of both, 1 u: 16 u.

Sums: `additions` of a contraction of n, 6 n with six products each, round once each, u of the sum of magnitudes; where all but one of the products
are 0 (`single`), the sums are exact but for the six products' own: 6 u.
"""
import torch

U = 2.0 ** -24
FLUSH = 2.0 ** -126


def bounds(q, k, v, g, state, scale, single=False, step=32):
    """q, k [n, k_heads, dk], v [n, v_heads, dv], g [n, v_heads] (or [v_heads]), state [v_heads, dk, dv] or None, CPU tensors.
    Returns out [n, v_heads, dv], its bound, state, its bound."""
    n, vh, dv = v.shape
    dk = q.shape[2]
    q, k = (x.double().repeat_interleave(vh // x.shape[1], 1) for x in (q, k))
    v, g = v.double(), g.double().expand(n, vh)
    S = torch.zeros(vh, dk, dv, dtype=torch.float64) if state is None else state.double().clone()
    A, E = S.abs(), torch.zeros_like(S)
    out, tol = torch.empty(n, vh, dv, dtype=torch.float64), torch.empty(n, vh, dv, dtype=torch.float64)
    per_product = (8 + (6 if single else 6 * step)) * U
    per_output = (16 + (12 if single else 6 * (2 * dk + step))) * U
    for t in range(n):
        a = torch.exp(g[t])[:, None, None]
        kt, vt = k[t][:, :, None], v[t][:, None, :]
        S = a * S + kt * vt
        E = a * E + per_product * (kt * vt).abs() + FLUSH * (kt.abs() + vt.abs() + 1.0)
        A = a * A + (kt * vt).abs()
        if t % step == 0:
            E = E + 8 * U * A
        out[t] = scale * (q[t][:, :, None] * S).sum(1)
        tol[t] = abs(scale) * (q[t].abs()[:, :, None] * (E + per_output * A) + FLUSH * (q[t].abs()[:, :, None] + A)).sum(1) + FLUSH
    return out, tol, S, E + 8 * U * A + FLUSH
