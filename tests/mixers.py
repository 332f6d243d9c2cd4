"""Windowed attention and linear attention with a decay in 64 bits, straight from their definitions, with the error
that FP32 arithmetic may leave in every element; and the plumbing to call the library's entries on numpy arrays.

U = 2^-24 is the half step of FP32.  The bounds count roundings, in the worst case and to first order:
  * a score is a sum of dk products of operands scaled beforehand: dk + 4 roundings of at most the sum of the products' sizes;
  * a probability moves by its own score's error and by the sum's, plus one rounding per term of the sum and a few for
    exp2, the rescalings and the division;
  * what is summed with these weights adds one rounding per term.
"""
import ctypes

import numpy as np

U = 2.0 ** -24


# ---------------------------------------------------------------- windowed attention
def sees(QL, VL, ql, vl, window, sinks):
    i, j = np.arange(QL)[:, None], np.arange(VL)[None]
    pos = i + vl - ql
    ok = (i < ql) & (j < vl) & (j <= pos)
    return ok & ((j > pos - window) | (j < sinks)) if window else ok


def window_reference(Q, K, V, scale, window, sinks, qlens, vlens, dY=None):
    """Q [N, H, QL, dk], K / V [N, G, VL, d] -> dict of (value, error bound) for Y, lse and, with dY, dQ, dK, dV."""
    N, H, QL, dk = Q.shape
    G, VL, dv = K.shape[1], K.shape[2], V.shape[3]
    shapes = {"Y": (N, H, QL, dv), "lse": (N, H, QL)}
    if dY is not None:
        shapes.update(dQ=Q.shape, dK=K.shape, dV=V.shape)
    out = {k: (np.zeros(s), np.zeros(s)) for k, s in shapes.items()}
    for n in range(N):
        ql, vl = qlens[n], vlens[n]
        on = sees(QL, VL, ql, vl, window, sinks)
        for hd in range(H):
            g = hd // (H // G)
            clean = lambda x, rows: np.where(np.arange(x.shape[0])[:, None] < rows, x, 0).astype(np.float64)
            q, k, v = clean(Q[n, hd], ql), clean(K[n, g], vl), clean(V[n, g], vl)
            s = np.where(on, scale * (q @ k.T), -np.inf)
            some = on.any(1)
            top = np.where(some, s.max(1), 0)
            e = np.where(on, np.exp(s - top[:, None]), 0)
            total = np.where(some, e.sum(1), 1)
            p = e / total[:, None]
            size = np.where(on, abs(scale) * (np.abs(q) @ np.abs(k).T), 0)
            ds = (dk + 4) * U * size.max(1)
            terms = on.sum(1)
            eps = 2 * ds + (terms + 20) * U
            out["Y"][0][n, hd] = y = p @ v
            out["Y"][1][n, hd] = ey = eps[:, None] * (p @ np.abs(v)) + 1e-37
            out["lse"][0][n, hd] = lse = np.where(some, top + np.log(total), -np.inf)
            out["lse"][1][n, hd] = np.where(some, ds + (terms + 20) * U + 4 * U * (np.abs(top) + np.abs(lse)), 0)
            if dY is None:
                continue
            dy = clean(dY[n, hd], ql)
            dp, D = dy @ v.T, (dy * y).sum(1)
            dS = scale * p * (dp - D[:, None])
            ep = eps + 6 * U * np.where(some, np.abs(lse) + np.abs(top), 0)
            edp = (dv + 4) * U * (np.abs(dy) @ np.abs(v).T)
            eD = (dv + 4) * U * (np.abs(dy) * np.abs(y)).sum(1) + (np.abs(dy) * ey).sum(1)
            edS = abs(scale) * p * ((ep[:, None] + 4 * U) * (np.abs(dp) + np.abs(D)[:, None]) + edp + eD[:, None])
            a = np.abs(dS)
            out["dQ"][0][n, hd] = dS @ k
            out["dQ"][1][n, hd] = edS @ np.abs(k) + (terms[:, None] + 4) * U * (a @ np.abs(k)) + 1e-37
            seen = on.sum(0)[:, None] * (H // G) + 20
            out["dK"][0][n, g] += dS.T @ q
            out["dK"][1][n, g] += edS.T @ np.abs(q) + seen * U * (a.T @ np.abs(q)) + 1e-37
            out["dV"][0][n, g] += p.T @ dy
            out["dV"][1][n, g] += (p * (ep[:, None] + 4 * U)).T @ np.abs(dy) + seen * U * (p.T @ np.abs(dy)) + 1e-37
    return out


# ---------------------------------------------------------------- linear attention with a decay
def decay_reference(Q, K, V, g, scale, lens, S0=None, dY=None, dS1=None):
    """[N, H, L, d] operands, token by token -> dict of (value, error bound) for Y, S1 and, with dY, dQ, dK, dV, dS0.
    A term meets at most dk or dv roundings in its own product, one per later token or sum it passes through and
    the error of its powers, 2 |g| per token."""
    N, H, L, dk = Q.shape
    dv = V.shape[3]
    shapes = {"Y": (N, H, L, dv), "S1": (N, H, dk, dv)}
    if dY is not None:
        shapes.update(dQ=Q.shape, dK=K.shape, dV=V.shape, dS0=(N, H, dk, dv))
    out = {k: (np.zeros(s), np.zeros(s)) for k, s in shapes.items()}
    for n in range(N):
        T = lens[n]
        for h in range(H):
            lam = np.exp(np.float64(g[h]))
            weight = (dk + dv + L + 32 + 4 * min(abs(float(g[h])), 100.0) * L) * U
            for sign in (0, 1):               # 0: the value; 1: the same sums over the operands' sizes, for the bound
                f = (lambda x: np.abs(x.astype(np.float64))) if sign else (lambda x: x.astype(np.float64))
                put = (lambda key, i, x: out[key][1][n, h].__setitem__(i, x * weight + 1e-37)) if sign else \
                      (lambda key, i, x: out[key][0][n, h].__setitem__(i, x))
                q, k, v = f(Q[n, h, :T]), f(K[n, h, :T]), f(V[n, h, :T])
                sc = abs(scale) if sign else scale
                S = f(S0[n, h]) if S0 is not None else np.zeros((dk, dv))
                dy = f(dY[n, h, :T]) if dY is not None else None
                for t in range(T):
                    S = lam * S + np.outer(k[t], v[t])
                    put("Y", t, sc * (q[t] @ S))
                    if dY is not None:
                        put("dQ", t, sc * (S @ dy[t]))
                put("S1", slice(None), S)
                if dY is None:
                    continue
                R = f(dS1[n, h]) if dS1 is not None else np.zeros((dk, dv))
                for t in range(T - 1, -1, -1):
                    R = R + sc * np.outer(q[t], dy[t])
                    put("dV", t, k[t] @ R)
                    put("dK", t, R @ v[t])
                    R = lam * R
                put("dS0", slice(None), R)
    return out


# ---------------------------------------------------------------- calls
def outer(x, head_inner):
    """[N, H, L, d] -> the layout in memory, d padded with zeros to a multiple of 4."""
    d4 = (x.shape[3] + 3) // 4 * 4
    y = np.zeros(x.shape[:3] + (d4,), np.float32)
    y[..., :x.shape[3]] = x
    return np.ascontiguousarray(y.transpose(0, 2, 1, 3)) if head_inner else y


def inner(x, shape, head_inner):
    N, H, L, d = shape
    d4 = (d + 3) // 4 * 4
    y = x.reshape(N, L, H, d4).transpose(0, 2, 1, 3) if head_inner else x.reshape(N, H, L, d4)
    return y[..., :d], y[..., d:]


def ints(dh, values):
    return None if values is None else dh.DeviceArray(np.asarray(values, np.int32).view(np.float32))


def at(x):
    return 0 if x is None else x.address


FILL = 7.5     # what outputs and buffers hold before a call: nothing of it may be left


def filled(dh, size):
    a = dh.DeviceArray(size=size, zero=False)
    a.fill(FILL)
    return a


def run_window(dh, Q, K, V, scale, window, sinks, qlens=None, vlens=None, dY=None, head_inner=0, stream=0):
    N, H, QL, dk = Q.shape
    G, VL, dv = K.shape[1], K.shape[2], V.shape[3]
    A = dh.Cuda_attention
    dk4, dv4 = (dk + 3) // 4 * 4, (dv + 3) // 4 * 4
    sizes = (N, H, G, QL, VL, dk4, dv4)
    need = A.window_bufsize(*sizes, window, sinks)
    buf = filled(dh, max(need // 4, 4))
    q, k, v = (dh.DeviceArray(outer(x, head_inner)) for x in (Q, K, V))
    y, lse = filled(dh, N * H * QL * dv4), filled(dh, N * H * QL)
    ql, vl = ints(dh, qlens), ints(dh, vlens)
    tail = sizes + (head_inner, scale, window, sinks)
    dh.Cuda.deviceSynchronize()
    A.window_forward([stream], 1, q.address, k.address, v.address, y.address, lse.address, at(ql), at(vl), buf.address, need, *tail)
    dh.Cuda.streamSynchronize(stream)
    out = {"lse": lse.get((N, H, QL))}
    out["Y"], pad = inner(y.get(), (N, H, QL, dv), head_inner)
    assert not pad.any(), "pad columns of Y"
    if dY is not None:
        g = dh.DeviceArray(outer(dY, head_inner))
        need = A.window_backward_bufsize(*sizes, window, sinks)
        buf2 = filled(dh, need // 4)
        dq, dk_, dv_ = filled(dh, q.size), filled(dh, k.size), filled(dh, v.size)
        dh.Cuda.deviceSynchronize()
        A.window_backward([stream], 1, q.address, k.address, v.address, y.address, lse.address, g.address, dq.address, dk_.address,
                          dv_.address, at(ql), at(vl), buf2.address, need, *tail)
        dh.Cuda.streamSynchronize(stream)
        for name, a, s in (("dQ", dq, Q.shape), ("dK", dk_, K.shape), ("dV", dv_, V.shape)):
            out[name], pad = inner(a.get(), s, head_inner)
            assert not pad.any(), "pad columns of " + name
    return out


def run_decay(dh, Q, K, V, g, scale, lens=None, S0=None, dY=None, dS1=None, head_inner=0, stream=0, in_place=False, want_state=True):
    N, H, L, dk = Q.shape
    dv = V.shape[3]
    A = dh.Cuda_linear_attention
    assert dk % 4 == 0 and dv % 4 == 0
    sizes = (N, H, L, dk, dv)
    need = A.bufsize(*sizes)
    buf = filled(dh, max(need // 4, 4))
    q, k, v = (dh.DeviceArray(outer(x, head_inner)) for x in (Q, K, V))
    dec = dh.DeviceArray(np.asarray(g, np.float32))
    s0 = dh.DeviceArray(S0) if S0 is not None else None
    s1 = s0 if in_place else (filled(dh, N * H * dk * dv) if want_state else None)
    y, ln = filled(dh, v.size), ints(dh, lens)
    tail = sizes + (head_inner, scale)
    dh.Cuda.deviceSynchronize()
    A.forward([stream], 1, q.address, k.address, v.address, dec.address, at(s0), y.address, at(s1), at(ln), buf.address, need, *tail)
    dh.Cuda.streamSynchronize(stream)
    out = {"Y": inner(y.get(), V.shape, head_inner)[0]}
    if s1 is not None:
        out["S1"] = s1.get((N, H, dk, dv))
    if dY is not None:
        gy = dh.DeviceArray(outer(dY, head_inner))
        d1 = dh.DeviceArray(dS1) if dS1 is not None else None
        need = A.backward_bufsize(*sizes)
        buf2 = filled(dh, max(need // 4, 4))
        dq, dk_, dv_ = filled(dh, q.size), filled(dh, k.size), filled(dh, v.size)
        d0 = filled(dh, N * H * dk * dv) if want_state else None
        dh.Cuda.deviceSynchronize()
        A.backward([stream], 1, q.address, k.address, v.address, dec.address, at(s0), gy.address, at(d1), dq.address, dk_.address,
                   dv_.address, at(d0), at(ln), buf2.address, need, *tail)
        dh.Cuda.streamSynchronize(stream)
        for name, a, s in (("dQ", dq, Q.shape), ("dK", dk_, K.shape), ("dV", dv_, V.shape)):
            out[name] = inner(a.get(), s, head_inner)[0]
        if d0 is not None:
            out["dS0"] = d0.get((N, H, dk, dv))
    return out


def check(got, want, what=""):
    for name, (value, bound) in want.items():
        if name not in got:
            continue
        x = np.asarray(got[name], np.float64)
        assert x.shape == value.shape, (what, name, x.shape, value.shape)
        same = (x == value) | (np.isneginf(x) & np.isneginf(value))
        off = np.where(same, 0, np.abs(np.where(same, 0, x) - np.where(same, 0, value)))
        bad = ~(off <= bound + np.abs(np.where(np.isfinite(value), value, 0)) * U)
        assert not bad.any(), "%s %s: %d of %d beyond the bound, first at %s: %r, should be %r within %.3g" % (
            what, name, bad.sum(), bad.size, tuple(np.argwhere(bad)[0]), x[bad][0], value[bad][0], bound[bad][0])
