"""Operands of the token mixers for which FP32 sums are whole numbers, so that every key and every token counts: with a
bound that grows with the number of terms, one of thousands could go missing unseen.

  * Windowed attention with Q = 0: every score is 0, every exponential 1, the sums are whole numbers below 2^24 and exact in
    any order.  Left are the division and the product with it.
  * Linear attention with g = 0: every power is 1, the results are whole numbers below 2^24 times a power of two.
"""
import numpy as np

U = 2.0 ** -24


def whole_values(rng, shape):
    """+-1 ... +-8: no value is zero, so that a key left out changes every column."""
    return (rng.integers(1, 9, shape) * rng.choice((-1, 1), shape)).astype(np.float32)


def uniform_window(V, head, QL, window, sinks, qlens, vlens):
    """V [N, G, VL, dv] of whole numbers -> Y and lse for Q = 0 as (value, bound): 1 / count and its product with the sum are
    rounded once each; the logarithm (base 2, one unit in its last place: 2 U) meets a rounded factor and a product."""
    N, G, VL, dv = V.shape
    Y, lse = np.zeros((N, head, QL, dv)), np.full((N, head, QL), -np.inf)
    for n in range(N):
        total = np.concatenate([np.zeros((G, 1, dv)), np.cumsum(V[n].astype(np.float64), 1)], 1)
        assert np.abs(V[n]).sum(1).max() < 2 ** 24
        for i in range(qlens[n]):
            pos = i + vlens[n] - qlens[n]
            low = max(pos - window + 1, 0) if window else 0
            first = min(sinks, low, vlens[n])
            count = max(pos + 1 - low, 0) + first
            if pos < 0 or count == 0:
                continue
            s = total[:, pos + 1] - total[:, low] + total[:, first]
            Y[n, :, i] = np.repeat(s / count, head // G, 0)
            lse[n, :, i] = np.log(count)
    return {"Y": (Y, 4 * U * np.abs(Y)), "lse": (lse, np.where(np.isfinite(lse), 6 * U * np.abs(np.where(np.isfinite(lse), lse, 0)), 0))}


def few(rng, shape):
    return rng.integers(-1, 2, shape).astype(np.float32)


def undecayed(Q, K, V, scale, lens, S0, dY, dS1):
    """g = 0, whole operands, scale a power of two: what every result is, exactly."""
    N, H, L, dk = Q.shape
    dv = V.shape[3]
    out = {"Y": np.zeros(V.shape), "S1": np.zeros((N, H, dk, dv)), "dQ": np.zeros(Q.shape), "dK": np.zeros(K.shape),
           "dV": np.zeros(V.shape), "dS0": np.zeros((N, H, dk, dv))}
    for n in range(N):
        T = lens[n]
        upto = np.tril(np.ones((T, T)))
        for h in range(H):
            q, k, v, dy = (x[n, h, :T].astype(np.float64) for x in (Q, K, V, dY))
            s0, ds1 = S0[n, h].astype(np.float64), dS1[n, h].astype(np.float64)
            out["Y"][n, h, :T] = scale * ((upto * (q @ k.T)) @ v + q @ s0)
            out["S1"][n, h] = s0 + k.T @ v
            out["dQ"][n, h, :T] = scale * ((upto * (dy @ v.T)) @ k + dy @ s0.T)
            out["dK"][n, h, :T] = scale * ((upto.T * (v @ dy.T)) @ q) + v @ ds1.T
            out["dV"][n, h, :T] = scale * ((upto.T * (k @ q.T)) @ dy) + k @ ds1
            out["dS0"][n, h] = ds1 + scale * (q.T @ dy)
    assert all(np.abs(x).max() / min(scale, 1.0) < 2 ** 24 for x in out.values())
    return out
