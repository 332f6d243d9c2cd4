"""Windowed attention and linear attention with a decay on the GPU against their definitions in 64 bits
(tests/mixers.py derives the error that FP32 may leave in every element)."""
import os
import subprocess
import sys

import numpy as np
import pytest

from mixers import check, decay_reference, run_decay, run_window, window_reference

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def window_operands(rng, N, H, G, QL, VL, dk, dv):
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    return f(N, H, QL, dk), f(N, G, VL, dk), f(N, G, VL, dv), f(N, H, QL, dv)


# N, head, kv_head, QL, VL, dk, dv, window, sinks, qlens, vlens
WINDOW = [
    (1, 1, 1, 1, 1, 4, 4, 0, 0, None, None),                       # one token, one key
    (1, 2, 1, 1, 300, 64, 64, 100, 4, None, None),                 # single token, shared head, sinks apart from the window
    (2, 8, 2, 1, 700, 128, 128, 0, 0, None, [700, 13]),            # single token, everything visible, ragged caches
    (3, 6, 2, 1, 90, 36, 100, 33, 5, None, [90, 0, 1]),            # odd head dimensions, an empty cache, one key
    (2, 32, 1, 1, 65, 64, 32, 7, 70, None, [65, 64]),              # 32 rows on one head; more sinks than keys
    (1, 4, 4, 5, 40, 32, 32, 8, 2, None, None),                    # several last queries
    (2, 6, 3, 16, 17, 20, 24, 3, 1, [16, 9], [17, 9]),             # 32 rows in two blocks, ragged
    (1, 3, 1, 7, 3, 8, 8, 0, 0, None, None),                       # more queries than keys: the first see nothing
    (1, 16, 2, 1, 9000, 64, 64, 0, 0, None, None),                 # keys cut into parts
    (1, 2, 2, 17, 17, 16, 16, 0, 0, None, None),                   # the smallest tile
    (2, 2, 1, 200, 200, 64, 64, 50, 4, [200, 77], [200, 77]),
    (1, 4, 2, 257, 257, 128, 128, 64, 3, None, None),
    (2, 3, 3, 130, 333, 96, 96, 0, 0, [130, 100], [333, 100]),     # a piece on a cache
    (1, 2, 1, 129, 640, 32, 64, 1, 0, None, None),                 # a query sees itself alone
    (1, 2, 2, 150, 150, 64, 64, 1, 1, None, None),
    (3, 2, 1, 140, 140, 44, 12, 30, 140, [140, 0, 1], [140, 0, 1]),  # all keys are sinks; empty and single sequences
    (1, 1, 1, 190, 100, 16, 16, 20, 2, None, None),                # more queries than keys
    (1, 1, 1, 300, 2500, 64, 64, 0, 0, None, None),                # keys cut into parts, tiles
    (2, 4, 2, 300, 300, 80, 80, 128, 200, None, [300, 260]),       # fewer keys than queries in one; sinks in two key tiles
    (1, 6, 1, 520, 520, 128, 64, 33, 40, None, None),
    (2, 64, 1, 1, 430, 64, 64, 50, 3, None, [430, 31]),            # 64 rows on one head
    (2, 6, 2, 20, 300, 36, 100, 40, 2, [20, 7], [300, 299]),       # 60 rows, ragged
    (1, 13, 1, 5, 1000, 128, 128, 0, 3, None, None),               # 65 rows: a tile
    (1, 4, 2, 1, 400, 128, 128, 0, 0, None, None),                 # cut in three
    (1, 4, 4, 300, 2500, 96, 72, 0, 0, None, None),                # cut, and many rows to join
    (1, 2, 1, 150, 150, 32, 32, 1000, 5, None, None),              # a window beyond the sequence
    (5, 2, 1, 100, 3000, 32, 32, 0, 0, [100, 1, 50, 0, 100], [3000, 1, 200, 0, 64]),     # parts dealt by length
    (3, 1, 1, 200, 2000, 64, 64, 700, 20, [200, 150, 3], [2000, 900, 10]),               # and under a window
    (80, 1, 1, 70, 300, 16, 16, 0, 0, [70 - i % 71 for i in range(80)], [300 - 3 * i for i in range(80)]),   # 80 pairs
    (2, 4, 2, 700, 900, 128, 128, 0, 0, None, [900, 700]),         # lengths of keys alone; a triangle
    (12, 8, 8, 500, 500, 16, 16, 40, 2, None, None),               # many tiles: nothing is cut, in either direction
]


@pytest.mark.parametrize("head_inner", (0, 1))
@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(str(x) for x in c[:9]))
def test_window_forward_and_gradient(dh, gpu, case, head_inner):
    N, H, G, QL, VL, dk, dv, window, sinks, qlens, vlens = case
    rng = np.random.default_rng(QL * 31 + VL)
    Q, K, V, dY = window_operands(rng, N, H, G, QL, VL, dk, dv)
    ql, vl = qlens or [QL] * N, vlens or [VL] * N
    for n in range(N):                 # what lies behind the lengths is never looked at
        Q[n, :, ql[n]:], dY[n, :, ql[n]:] = np.nan, np.inf
        K[n, :, vl[n]:], V[n, :, vl[n]:] = np.inf, np.nan
    scale = 1.0 / np.sqrt(dk)
    got = run_window(dh, Q, K, V, scale, window, sinks, qlens, vlens, dY, head_inner)
    check(got, window_reference(Q, K, V, scale, window, sinks, ql, vl, dY), str(case))


def test_window_rows_that_no_query_sees_are_not_read(dh, gpu):
    # the last 5 queries of 400 under a window of 30 and 3 sinks: keys 3 .. 365 are seen by nobody
    rng = np.random.default_rng(3)
    for QL in (1, 5, 40):
        Q, K, V, dY = window_operands(rng, 1, 4, 2, QL, 400, 64, 64)
        K[:, :, 3:400 - QL - 29], V[:, :, 3:400 - QL - 29] = np.nan, np.nan
        got = run_window(dh, Q, K, V, 0.125, 30, 3)
        K, V = np.nan_to_num(K), np.nan_to_num(V)
        check(got, window_reference(Q, K, V, 0.125, 30, 3, [QL], [400]), "QL %d" % QL)


@pytest.mark.parametrize("QL", (1, 40))
def test_window_scores_far_apart(dh, gpu, QL):
    # scores that rise from key to key by far more than the lagging maximum, and large negative ones first
    Q, K, V, dY = window_operands(np.random.default_rng(5), 1, 2, 1, QL, 260, 32, 32)
    Q[...], K[...] = 1.0, 0.0
    K[0, 0, :, 0] = np.linspace(-3000.0, 3000.0, 260)
    for window in (0, 90):
        got = run_window(dh, Q, K, V, 1.0, window, 2, dY=dY)
        check(got, window_reference(Q, K, V, 1.0, window, 2, [QL], [260], dY), "window %d" % window)


def test_window_negative_and_zero_scale(dh, gpu):
    Q, K, V, dY = window_operands(np.random.default_rng(6), 1, 2, 2, 70, 70, 16, 16)
    for scale in (-0.5, 0.0):
        got = run_window(dh, Q, K, V, scale, 20, 1, dY=dY)
        check(got, window_reference(Q, K, V, scale, 20, 1, [70], [70], dY), "scale %g" % scale)


def test_window_gradient_against_differences(dh, gpu):
    rng = np.random.default_rng(7)
    Q, K, V, dY = window_operands(rng, 1, 4, 2, 150, 170, 24, 24)
    got = run_window(dh, Q, K, V, 0.2, 40, 3, dY=dY)
    loss = lambda q, k, v: (window_reference(q, k, v, 0.2, 40, 3, [150], [170])["Y"][0] * dY).sum()
    h = 1e-4
    for name, x in (("dQ", 0), ("dK", 1), ("dV", 2)):
        ops = [a.astype(np.float64) for a in (Q, K, V)]
        way = rng.standard_normal(ops[x].shape)
        up, down = list(ops), list(ops)
        up[x], down[x] = ops[x] + h * way, ops[x] - h * way
        slope = (loss(*up) - loss(*down)) / (2 * h)
        mine = (got[name].astype(np.float64) * way).sum()
        # the difference is off by h^2 times a third derivative, the gradient by its elements' bounds
        bound = window_reference(Q, K, V, 0.2, 40, 3, [150], [170], dY)[name][1]
        assert abs(mine - slope) <= (bound * np.abs(way)).sum() + 1e-6 * np.abs(got[name] * way).sum(), name


def test_window_bits_do_not_depend_on_the_run(dh, gpu):
    Q, K, V, dY = window_operands(np.random.default_rng(8), 2, 4, 1, 300, 300, 64, 64)
    a = run_window(dh, Q, K, V, 0.125, 64, 4, dY=dY)
    stream = dh.Cuda.newStream_NonBlocking()
    b = run_window(dh, Q, K, V, 0.125, 64, 4, dY=dY, stream=stream)
    dh.Cuda.deleteStream(stream)
    for name in a:
        assert np.array_equal(a[name], b[name]), name


def test_window_prompt_piece_and_step_agree(dh, gpu):
    """A prompt at once, in pieces on its cache, and its last token alone: the same attention."""
    rng = np.random.default_rng(9)
    Q, K, V, _ = window_operands(rng, 1, 8, 2, 400, 400, 64, 64)
    want = window_reference(Q, K, V, 0.125, 100, 4, [400], [400])
    whole = run_window(dh, Q, K, V, 0.125, 100, 4)
    check(whole, want, "whole")
    at = 0
    for n in (250, 100, 40, 9, 1):
        piece = run_window(dh, Q[:, :, at:at + n], K, V, 0.125, 100, 4, [n], [at + n])
        check(piece, {k: (v[:, :, at:at + n], b[:, :, at:at + n]) for k, (v, b) in want.items()}, "piece of %d" % n)
        at += n
    assert at == 400


# N, head, L, dk, dv, lens
DECAY = [
    (1, 1, 1, 4, 4, None), (2, 3, 1, 128, 128, None), (2, 2, 1, 36, 100, [1, 0]), (1, 2, 9, 64, 32, None),
    (3, 2, 16, 20, 64, [16, 5, 0]), (1, 2, 17, 16, 16, None), (2, 2, 100, 64, 64, [100, 31]), (1, 2, 128, 64, 64, None),
    (2, 1, 129, 32, 32, [129, 128]), (3, 2, 300, 64, 64, [300, 257, 0]), (1, 1, 256, 128, 128, None), (2, 2, 513, 128, 96, [513, 1]),
    (1, 2, 700, 96, 128, None), (2, 1, 600, 44, 12, [599, 256]),
]


@pytest.mark.parametrize("carried", (False, True))
@pytest.mark.parametrize("head_inner", (0, 1))
@pytest.mark.parametrize("case", DECAY, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_decay_forward_and_gradient(dh, gpu, case, head_inner, carried):
    N, H, L, dk, dv, lens = case
    rng = np.random.default_rng(L * 7 + dk)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, dY = f(N, H, L, dk), f(N, H, L, dk), f(N, H, L, dv), f(N, H, L, dv)
    ln = lens or [L] * N
    for n in range(N):
        for x in (Q, K, V, dY):
            x[n, :, ln[n]:] = np.nan
    g = np.array([-0.01, -0.7, 0.0][:H], np.float32)
    S0, dS1 = (f(N, H, dk, dv), f(N, H, dk, dv)) if carried else (None, None)
    scale = dk ** -0.5
    got = run_decay(dh, Q, K, V, g, scale, lens, S0, dY, dS1, head_inner)
    check(got, decay_reference(Q, K, V, g, scale, ln, S0, dY, dS1), str(case))
    bare = run_decay(dh, Q, K, V, g, scale, lens, S0, dY, dS1, head_inner, want_state=False)
    for name in bare:
        assert np.array_equal(bare[name], got[name]) or L <= 256, name     # one chunk: the state is not formed first


@pytest.mark.parametrize("g", (-float("inf"), -100.0, -20.0, -1e-6))
def test_decay_that_forgets_at_once_or_never(dh, gpu, g):
    rng = np.random.default_rng(11)
    for L in (1, 16, 40, 300):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)
        Q, K, V, dY = f(1, 1, L, 32), f(1, 1, L, 32), f(1, 1, L, 32), f(1, 1, L, 32)
        S0, dS1 = f(1, 1, 32, 32), f(1, 1, 32, 32)
        got = run_decay(dh, Q, K, V, [g], 0.5, None, S0, dY, dS1)
        check(got, decay_reference(Q, K, V, [g], 0.5, [L], S0, dY, dS1), "g %g, L %d" % (g, L))


@pytest.mark.parametrize("L", (3, 100, 700))
def test_decay_that_is_no_number(dh, gpu, L):
    rng = np.random.default_rng(L)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, S0 = f(1, 3, L, 32), f(1, 3, L, 32), f(1, 3, L, 32), f(1, 3, 32, 32)
    g = np.array([-0.1, np.nan, -0.2], np.float32)
    got = run_decay(dh, Q, K, V, g, 0.2, None, S0)
    assert np.isnan(got["Y"][:, 1]).all() and np.isnan(got["S1"][:, 1]).all()
    keep = [0, 2]
    want = decay_reference(Q[:, keep], K[:, keep], V[:, keep], g[keep], 0.2, [L], S0[:, keep])
    check({name: got[name][:, keep] for name in ("Y", "S1")}, want)


def test_decay_state_in_place(dh, gpu):
    rng = np.random.default_rng(12)
    for L in (1, 12, 200):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)
        Q, K, V, S0 = f(2, 2, L, 64), f(2, 2, L, 64), f(2, 2, L, 64), f(2, 2, 64, 64)
        a = run_decay(dh, Q, K, V, [-0.1, -0.2], 1.0, None, S0)
        b = run_decay(dh, Q, K, V, [-0.1, -0.2], 1.0, None, S0, in_place=True)
        assert np.array_equal(a["Y"], b["Y"]) and np.array_equal(a["S1"], b["S1"])


def test_decay_prompt_in_pieces_and_steps(dh, gpu):
    """A sequence at once, and in pieces down to single tokens with the state carried: the same outputs."""
    rng = np.random.default_rng(13)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    L = 700
    Q, K, V = f(2, 2, L, 64), f(2, 2, L, 64), f(2, 2, L, 64)
    g = [-0.02, -0.3]
    want = decay_reference(Q, K, V, g, 0.125, [L, L])
    check(run_decay(dh, Q, K, V, g, 0.125), want, "whole")
    state, at = np.zeros((2, 2, 64, 64), np.float32), 0
    for n in (400, 270, 17, 9, 1, 1, 1, 1):
        cut = slice(at, at + n)
        got = run_decay(dh, Q[:, :, cut], K[:, :, cut], V[:, :, cut], g, 0.125, None, state)
        state = got["S1"]
        check({"Y": got["Y"]}, {"Y": tuple(x[:, :, cut] for x in want["Y"])}, "piece of %d" % n)
        at += n
    assert at == L
    check({"S1": state}, want, "last state")


def test_decay_gradient_against_differences(dh, gpu):
    rng = np.random.default_rng(14)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    N, H, L, d = 1, 2, 300, 16
    Q, K, V, dY, S0, dS1 = f(N, H, L, d), f(N, H, L, d), f(N, H, L, d), f(N, H, L, d), f(N, H, d, d), f(N, H, d, d)
    g = np.array([-0.05, -0.5], np.float32)
    got = run_decay(dh, Q, K, V, g, 0.25, None, S0, dY, dS1)
    want = decay_reference(Q, K, V, g, 0.25, [L], S0, dY, dS1)

    def loss(q, k, v, s):
        r = decay_reference(q, k, v, g, 0.25, [L], s)
        return (r["Y"][0] * dY).sum() + (r["S1"][0] * dS1).sum()

    for x, name in enumerate(("dQ", "dK", "dV", "dS0")):
        ops = [a.astype(np.float64) for a in (Q, K, V, S0)]
        way = rng.standard_normal(ops[x].shape)
        up, down = list(ops), list(ops)
        up[x], down[x] = ops[x] + way, ops[x] - way       # the loss is linear in each operand: any step will do
        slope = (loss(*up) - loss(*down)) / 2
        mine = (got[name].astype(np.float64) * way).sum()
        assert abs(mine - slope) <= (want[name][1] * np.abs(way)).sum() + 1e-9 * abs(slope), name


def test_decay_bits_do_not_depend_on_the_run(dh, gpu):
    rng = np.random.default_rng(15)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, dY = f(2, 2, 500, 64), f(2, 2, 500, 64), f(2, 2, 500, 64), f(2, 2, 500, 64)
    a = run_decay(dh, Q, K, V, [-0.1, -0.2], 0.125, dY=dY)
    stream = dh.Cuda.newStream_NonBlocking()
    b = run_decay(dh, Q, K, V, [-0.1, -0.2], 0.125, dY=dY, stream=stream)
    dh.Cuda.deleteStream(stream)
    for name in a:
        assert np.array_equal(a[name], b[name]), name


def test_offsets_beyond_32_bits(dh, gpu):
    """The last tokens of caches of 4.9 GB: only the sinks and the window are filled, nothing else may be read."""
    G, d, VL, window, sinks = 8, 128, 1200000, 200, 3
    rng = np.random.default_rng(21)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    row = G * d
    A = dh.Cuda_attention
    caches = [dh.DeviceArray(size=VL * row, zero=False) for _ in "kv"]
    ends = []
    for c in caches:
        first, last = f(sinks, G, d), f(window + 64, G, d)
        dh.Cuda.set1D(0, c.address, first.reshape(-1), first.size)
        dh.Cuda.set1D(0, c.address + 4 * (VL - window - 64) * row, last.reshape(-1), last.size)
        ends.append(np.concatenate([first, last]).transpose(1, 0, 2)[None])
    for QL, head in ((1, 16), (40, 16)):
        Q = f(1, head, QL, d)
        q, y = dh.DeviceArray(np.ascontiguousarray(Q.transpose(0, 2, 1, 3))), dh.DeviceArray(size=Q.size)
        sizes = (1, head, G, QL, VL, d, d)
        need = A.window_bufsize(*sizes, window, sinks)
        buf = dh.DeviceArray(size=max(need // 4, 4))
        A.window_forward([0], 1, q.address, caches[0].address, caches[1].address, y.address, 0, 0, 0, buf.address, need, *sizes, 1,
                         0.1, window, sinks)
        dh.Cuda.deviceSynchronize()
        # the same with the hole closed: the keys between are seen by nobody in either
        want = window_reference(Q, *ends, 0.1, window, sinks, [QL], [sinks + window + 64])
        check({"Y": y.get((1, QL, head, d)).transpose(0, 2, 1, 3)}, want, "QL %d" % QL)


def test_states_too_large_for_the_caches(dh, gpu):
    """Two tokens on 84 x 32 states of 128 x 128 (176 MB, in and out): the form that reads and writes them non-temporally."""
    rng = np.random.default_rng(23)
    N, H, L, d = 84, 32, 2, 128
    f = lambda *s: rng.standard_normal(s, dtype=np.float32)
    Q, K, V, S = f(N, H, L, d), f(N, H, L, d), f(N, H, L, d), f(N, H, d, d)
    g = -np.exp2(-rng.uniform(0, 10, H)).astype(np.float32)
    got = run_decay(dh, Q, K, V, g, 0.25, None, S)
    for h in range(H):
        s, lam = S[:, h].astype(np.float64), np.exp(np.float64(g[h]))
        a = np.abs(s)
        for t in range(L):
            k, v, q = (x[:, h, t].astype(np.float64) for x in (K, V, Q))
            s = lam * s + k[:, :, None] * v[:, None]
            a = lam * a + np.abs(k)[:, :, None] * np.abs(v)[:, None]
            y, ya = 0.25 * np.einsum("nk,nkv->nv", q, s), 0.25 * np.einsum("nk,nkv->nv", np.abs(q), a)
            # as in decay_reference: dk + dv + L + 32 roundings and the powers'
            weight = (2 * d + L + 32 + 4 * abs(float(g[h])) * L) * 2.0 ** -24
            assert (np.abs(got["Y"][:, h, t] - y) <= weight * ya).all()
        assert (np.abs(got["S1"][:, h] - s) <= weight * a).all()


def test_a_cache_too_large_for_the_caches(dh, gpu):
    """A single token on 45000 keys of 8 heads of 128 (369 MB): the form that reads them non-temporally."""
    Q, K, V, _ = window_operands(np.random.default_rng(24), 1, 16, 8, 1, 45000, 128, 128)
    got = run_window(dh, Q, K, V, 128 ** -0.5, 0, 0, head_inner=1)
    check(got, window_reference(Q, K, V, 128 ** -0.5, 0, 0, [1], [45000]))


def test_calls_on_two_streams_at_once(dh, gpu):
    """Each with its own work buffer: nothing is shared between calls."""
    rng = np.random.default_rng(22)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    A, L, Cuda = dh.Cuda_attention, dh.Cuda_linear_attention, dh.Cuda
    N, H, S, d = 2, 4, 500, 64
    sizes, dsizes = (N, H, 2, S, S, d, d), (N, H, S, d, d)
    streams = [Cuda.newStream_NonBlocking() for _ in range(3)]
    jobs = []
    for i in range(3):
        ops = [dh.DeviceArray(x) for x in (f(N, H, S, d), f(N, 2, S, d), f(N, 2, S, d), f(N, H, S, d), f(N, H, S, d), f(N, H, S, d))]
        g = dh.DeviceArray(np.full(H, -0.1 * (i + 1), np.float32))
        outs = [dh.DeviceArray(size=N * H * S * d) for _ in range(2)] + [dh.DeviceArray(size=N * H * S)]
        grads = [dh.DeviceArray(size=a.size) for a in ops[:3]]
        need = max(A.window_bufsize(*sizes, 90, 3), A.window_backward_bufsize(*sizes, 90, 3))
        dneed = L.bufsize(*dsizes)
        bufs = [dh.DeviceArray(size=max(n // 4, 4)) for n in (need, dneed)]
        jobs.append((ops, g, outs, grads, bufs, need, dneed))
    Cuda.deviceSynchronize()

    def issue(i, stream):
        ops, g, outs, grads, bufs, need, dneed = jobs[i]
        q, k, v, dy, k2, v2 = (a.address for a in ops)
        A.window_forward([stream], 1, q, k, v, outs[0].address, outs[2].address, 0, 0, bufs[0].address, need, *sizes, 0, 0.125, 90, 3)
        A.window_backward([stream], 1, q, k, v, outs[0].address, outs[2].address, dy, *(a.address for a in grads), 0, 0,
                          bufs[0].address, need, *sizes, 0, 0.125, 90, 3)
        L.forward([stream], 1, q, k2, v2, g.address, 0, outs[1].address, 0, 0, bufs[1].address, dneed, *dsizes, 0, 0.125)

    def results(i):
        return [a.get() for a in jobs[i][2] + jobs[i][3]]

    alone = []
    for i in range(3):
        issue(i, 0)
        Cuda.deviceSynchronize()
        alone.append(results(i))
    for _ in range(5):
        for i in range(3):
            issue(i, streams[i])
    Cuda.deviceSynchronize()
    for i in range(3):
        for a, b in zip(alone[i], results(i)):
            assert np.array_equal(a, b)
    for s in streams:
        Cuda.deleteStream(s)


def test_captured_calls_replay():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "mixer_graph_check.py")], capture_output=True, text=True, timeout=110)
    if r.returncode == 77:
        pytest.skip(r.stdout.strip())
    assert r.returncode == 0, r.stdout + r.stderr


# ---------------------------------------------------------------- through the engine
@pytest.fixture()
def eg(dh, gpu):
    from dragon_hip import engine
    e = engine.cuda_float32(0, 8)
    yield e
    e.close()


def side_by_side(x):
    """[N, H, L, d] -> [N, L, H*d]"""
    N, H, L, d = x.shape
    return np.ascontiguousarray(x.transpose(0, 2, 1, 3)).reshape(N, L, H * d)


def apart(x, N, H, L, d):
    return np.asarray(x).reshape(N, L, H, d).transpose(0, 2, 1, 3)


@pytest.mark.parametrize("sync", (True, False))
@pytest.mark.parametrize("shape", [(2, 6, 2, 90, 130, 32, 64), (1, 1, 1, 40, 40, 30, 21), (3, 4, 4, 1, 77, 128, 128)], ids=str)
def test_engine_window_attention_and_gradient(eg, shape, sync):
    N, H, G, QL, VL, dk, dv = shape
    Q, K, V, dY = window_operands(np.random.default_rng(31), N, H, G, QL, VL, dk, dv)
    t = [eg.tensor(side_by_side(x), N, x.shape[2], x.shape[1] * x.shape[3]).c() for x in (Q, K, V, dY)]
    eg.sync(sync)
    y, lse = eg.attention_window(*t[:3], H, G, 25, 3, lse=True)
    y.c(), lse.c()
    grads = eg.attention_window_delta(t[3], y, *t[:3], lse, H, G, 25, 3)
    got = {"Y": apart(y.c().value(), N, H, QL, dv), "lse": lse.value().reshape(N, H, QL)}
    for name, x, like in zip(("dQ", "dK", "dV"), grads, (Q, K, V)):
        got[name] = apart(x.c().value(), *like.shape)
    check(got, window_reference(Q, K, V, np.float32(1) / np.sqrt(np.float32(dk)), 25, 3, [QL] * N, [VL] * N, dY), str(shape))
    eg.sync(True)
    eg.delete(y, lse, *grads, *t)


@pytest.mark.parametrize("sync", (True, False))
@pytest.mark.parametrize("L", (1, 40, 300))
def test_engine_linear_attention_and_gradient(eg, L, sync):
    rng = np.random.default_rng(32)
    N, H, dk, dv = 2, 3, 32, 64
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, dY, S0, dS1 = f(N, H, L, dk), f(N, H, L, dk), f(N, H, L, dv), f(N, H, L, dv), f(N, H, dk, dv), f(N, H, dk, dv)
    g = np.array([-0.5, -0.05, -0.005], np.float32)
    t = [eg.tensor(side_by_side(x), N, L, H * x.shape[3]).c() for x in (Q, K, V, dY)]
    dec, s0, ds1 = eg.tensor(g, H).c(), eg.tensor(S0, N, H, dk, dv).c(), eg.tensor(dS1, N, H, dk, dv).c()
    eg.sync(sync)
    y, s1 = eg.linear_attention(*t[:3], dec, H, s0, 0.2, state=True)
    grads = eg.linear_attention_delta(t[3], *t[:3], dec, H, s0, ds1, 0.2, state=True)
    got = {"Y": apart(y.c().value(), N, H, L, dv), "S1": s1.c().value().reshape(N, H, dk, dv)}
    for name, x, like in zip(("dQ", "dK", "dV"), grads, (Q, K, V)):
        got[name] = apart(x.c().value(), *like.shape)
    got["dS0"] = grads[3].c().value().reshape(N, H, dk, dv)
    check(got, decay_reference(Q, K, V, g, 0.2, [L] * N, S0, dY, dS1), "L %d" % L)
    eg.sync(True)
    eg.delete(y, s1, *grads, *t, dec, s0, ds1)


def test_engine_refuses(eg):
    from dragon_hip import engine
    z = lambda *d: eg.zeros(*d).c()
    q, k, v, dec = z(2, 9, 24), z(2, 11, 12), z(2, 11, 12), z(2)
    for bad in (lambda: eg.attention_window(q, k, v, 4, 3), lambda: eg.attention_window(q, k, v, 2, 2), lambda: eg.attention_window(q, k, v, 0),
                lambda: eg.attention_window(q, k, v, 2, 1, -1), lambda: eg.attention_window(z(3, 9, 24), k, v, 2, 1),
                lambda: eg.attention_window(z(1, 4, 300), z(1, 4, 300), z(1, 4, 300), 1),
                lambda: eg.attention_window_delta(q, q, q, k, v, z(5), 2, 1), lambda: eg.linear_attention(q, k, v, dec, 2),
                lambda: eg.linear_attention(q, q, q, z(3), 2), lambda: eg.linear_attention(q, q, q, dec, 2, State=z(2, 2, 12, 8)),
                lambda: eg.linear_attention_delta(k, q, q, q, dec, 2)):
        with pytest.raises(engine.IllegalArgumentException):
            bad()
    for bad in (lambda: eg.attention_window(None, k, v, 2), lambda: eg.linear_attention(q, q, q, None, 2),
                lambda: eg.attention_window_delta(q, q, q, k, v, None, 2, 1)):
        with pytest.raises(engine.NullPointerException):
            bad()


def test_two_mixers_of_a_decoder_together(eg):
    """What a decoder with both kinds of layers runs: projections, windowed attention on shared heads, linear attention on its
    output, an output projection; prompt at once against prompt and single tokens."""
    rng = np.random.default_rng(33)
    N, L, C, H, G, d = 1, 70, 64, 4, 2, 16
    f = lambda *s: (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)
    w = {n: f(C, m) for n, m in (("q", H * d), ("k", G * d), ("v", G * d), ("q2", H * d), ("k2", H * d), ("v2", H * d), ("o", C))}
    X = rng.standard_normal((L, C)).astype(np.float32)
    g = np.array([-0.02, -0.1, -0.3, -1.0], np.float32)
    W = {n: eg.tensor(a, *a.shape).c() for n, a in w.items()}
    dec = eg.tensor(g, H).c()

    def project(x, name, rows):
        a = eg.tensor(x, rows, C).c()
        return eg.matMul(a, W[name]).c().value().reshape(rows, -1)

    def layer(x, cache, state):
        rows = x.shape[0]
        t = lambda a: eg.tensor(a, 1, a.shape[0], a.shape[1]).c()
        k, v = (np.concatenate([c, project(x, n, rows)]) for c, n in zip(cache, "kv"))
        y = eg.attention_window(t(project(x, "q", rows)), t(k), t(v), H, G, 20, 2).c().value().reshape(rows, C)
        y2, s = eg.linear_attention(*(t(project(y, n, rows)) for n in ("q2", "k2", "v2")), dec, H, state, state=True)
        return project(y2.c().value().reshape(rows, C), "o", rows), (k, v), s.c()

    empty = (np.zeros((0, G * d), np.float32),) * 2
    whole, _, last = layer(X, empty, None)
    parts, cache, state = [], empty, None
    for a, b in ((0, 50), (50, 67), (67, 68), (68, 69), (69, 70)):
        y, cache, state = layer(X[a:b], cache, state)
        parts.append(y)
    # the same sums in other orders: the difference stays near the rounding of one value of each
    assert np.abs(np.concatenate(parts) - whole).max() <= 2e-5 * np.abs(whole).max()
    assert np.abs(state.value() - last.value()).max() <= 2e-5 * np.abs(last.value()).max()
