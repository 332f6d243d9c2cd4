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
