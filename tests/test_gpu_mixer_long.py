"""Long sequences of the token mixers, where a bound that counts roundings in the worst case would hide a missing key, a
missing token or an error that grows with the length."""
import numpy as np
import pytest

from mixers import check, decay_reference, run_decay, run_window
from mixers_exact import U, few, undecayed, uniform_window, whole_values
from test_gpu_mixers import DECAY

pytestmark = pytest.mark.gpu

# N, head, kv_head, QL, VL, d, window, sinks, qlens, vlens
UNIFORM = [
    (1, 16, 8, 1, 45000, 128, 0, 0, None, None),                    # 369 MB: read non-temporally, cut
    (1, 16, 8, 1, 46000, 128, 45001, 5, None, None),                # the same under a window, sinks in a step of their own
    (2, 8, 2, 1, 9001, 64, 0, 0, None, [9001, 4444]),               # cut, ragged
    (3, 8, 4, 1, 5000, 96, 3000, 20, None, [5000, 17, 0]),
    (1, 4, 2, 20, 7000, 64, 0, 0, None, None),                      # 40 rows: three blocks
    (1, 4, 2, 300, 6000, 128, 0, 0, None, None),                    # tiles, cut
    (1, 3, 1, 90, 9999, 32, 7000, 33, None, None),                  # tiles of 64 keys a step, cut, a window
    (3, 2, 1, 100, 8000, 64, 0, 0, [100, 60, 100], [8000, 500, 4001]),      # parts dealt by length
    (4, 4, 2, 70, 4000, 96, 2500, 9, [70, 1, 0, 33], [4000, 3999, 0, 40]),  # the same under a window
    (1, 8, 8, 1000, 3000, 64, 0, 0, None, None),                    # a triangle on a cache
]


@pytest.mark.parametrize("head_inner", (0, 1))
@pytest.mark.parametrize("case", UNIFORM, ids=lambda c: "-".join(str(x) for x in c[:8]))
def test_every_key_of_a_long_cache_counts(dh, gpu, case, head_inner):
    N, H, G, QL, VL, d, window, sinks, ql, vl = case
    rng = np.random.default_rng(VL)
    V, K = whole_values(rng, (N, G, VL, d)), rng.standard_normal((N, G, VL, d), dtype=np.float32)
    got = run_window(dh, np.zeros((N, H, QL, d), np.float32), K, V, 1.0, window, sinks, ql, vl, head_inner=head_inner)
    check(got, uniform_window(V, H, QL, window, sinks, ql or [QL] * N, vl or [VL] * N), str(case))


# N, head, L, dk, dv, lens: sequences whose segments are several runs of 32 tokens (in brackets: tokens x segments forward,
# and those of the gradient where they differ)
SEGMENTS = [
    (1, 2, 4200, 64, 64, None),                       # 96 x 44
    (3, 2, 2500, 64, 32, [2500, 1111, 70]),           # 64 x 40; ends in a segment's first and second run
    (4, 16, 1000, 64, 64, [1000, 750, 97, 0]),        # 64 x 16
    (4, 16, 1000, 32, 128, [1000, 513, 512, 129]),    # 128 x 8
    (2, 2, 3000, 128, 32, [3000, 2049]),              # 64 x 47
    (8, 16, 300, 100, 72, [300, 299, 192, 191, 97, 96, 95, 1]),     # 96 x 4
]


@pytest.mark.parametrize("head_inner", (0, 1))
@pytest.mark.parametrize("case", SEGMENTS, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_every_token_of_a_sequence_that_forgets_nothing_counts(dh, gpu, case, head_inner):
    N, H, L, dk, dv, lens = case
    rng = np.random.default_rng(L + dv)
    Q, K, V, dY = few(rng, (N, H, L, dk)), few(rng, (N, H, L, dk)), few(rng, (N, H, L, dv)), few(rng, (N, H, L, dv))
    S0, dS1 = few(rng, (N, H, dk, dv)), few(rng, (N, H, dk, dv))
    want = undecayed(Q, K, V, 0.5, lens or [L] * N, S0, dY, dS1)
    for n, T in enumerate(lens or []):
        for x in (Q, K, V, dY):
            x[n, :, T:] = np.nan
    got = run_decay(dh, Q, K, V, np.zeros(H, np.float32), 0.5, lens, S0, dY, dS1, head_inner)
    for name in want:
        assert np.array_equal(got[name], want[name]), name


@pytest.mark.parametrize("carried", (False, True))
@pytest.mark.parametrize("case", [(1, 2, 4200, 32, 36, None), (2, 3, 2100, 20, 64, [2100, 1313]), (4, 12, 500, 16, 68, [500, 130, 65, 31])],
                         ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_decay_over_segments_of_several_runs(dh, gpu, case, carried):
    N, H, L, dk, dv, lens = case
    rng = np.random.default_rng(L + dk)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, dY = f(N, H, L, dk), f(N, H, L, dk), f(N, H, L, dv), f(N, H, L, dv)
    S0, dS1 = (f(N, H, dk, dv), f(N, H, dk, dv)) if carried else (None, None)
    g = -np.exp2(-np.linspace(0.5, 9.0, H)).astype(np.float32)
    got = run_decay(dh, Q, K, V, g, 0.25, lens, S0, dY, dS1, head_inner=1)
    check(got, decay_reference(Q, K, V, g, 0.25, lens or [L] * N, S0, dY, dS1), str(case))


@pytest.mark.parametrize("case", DECAY, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_decay_results_do_not_depend_on_who_wants_the_states(dh, gpu, case):
    N, H, L, dk, dv, lens = case
    rng = np.random.default_rng(L)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    Q, K, V, dY, S0, dS1 = f(N, H, L, dk), f(N, H, L, dk), f(N, H, L, dv), f(N, H, L, dv), f(N, H, dk, dv), f(N, H, dk, dv)
    g = np.array([-0.01, -0.7, 0.0][:H], np.float32)
    a, b = (run_decay(dh, Q, K, V, g, 0.25, lens, S0, dY, dS1, want_state=w) for w in (True, False))
    assert set(b) == {"Y", "dQ", "dK", "dV"}
    for name in b:
        assert np.array_equal(a[name], b[name]), name


# Tokens a call, calls, multiplications of the state in all: 12 tokens multiply it each (decay_steps; the gradient at once), 192
# every 32 (decay_walk), 4096 in 64 segments once each (decay_scan).
@pytest.mark.parametrize("tokens, calls, forward, backward", [(12, 1500, 18000, 1500), (192, 300, 1800, 1800), (4096, 20, 1280, 1280)])
def test_a_slow_decay_does_not_drift(dh, gpu, tokens, calls, forward, backward):
    """A state that nothing is added to, e^{gT} of it after T tokens, call after call.  Every multiplication rounds an element
    by at most U, up or down as its digits happen to lie (a step takes hundreds of units in the last place off it), so the
    mean over E elements after M of them is off by U sqrt(M / E / 3) or so; six times that are allowed.  (Elements whole steps
    apart run through the same values and round alike, so no more count than a step has units.)  What is the same for all
    elements is the factor's own error, 4 U of what it takes off each time, |g| T of it in all.  A factor near 1 that is itself
    rounded to FP32 is off by up to U / 2 every time, in one direction, hundreds of U in the end."""
    H, d = 8, 64
    rng = np.random.default_rng(tokens)
    T = tokens * calls
    g = (-np.linspace(0.7, 2.0, H) / T).astype(np.float32)
    zero = dh.DeviceArray(size=tokens * H * d)
    out = [dh.DeviceArray(size=tokens * H * d) for _ in range(3)]
    dec = dh.DeviceArray(g)
    first = rng.uniform(0.5, 2.0, (H, d, d)).astype(np.float32)
    A = dh.Cuda_linear_attention
    sizes = (1, H, tokens, d, d)
    need, gneed = A.bufsize(*sizes), A.backward_bufsize(*sizes)
    buf = dh.DeviceArray(size=max(need, gneed, 16) // 4)
    state = dh.DeviceArray(first)
    grads = [dh.DeviceArray(first), dh.DeviceArray(size=first.size)]
    z = zero.address
    for i in range(calls):
        A.forward([0], 1, z, z, z, dec.address, state.address, out[0].address, state.address, 0, buf.address, need, *sizes, 1, 1.0)
        A.backward([0], 1, z, z, z, dec.address, 0, z, grads[i % 2].address, *(x.address for x in out), grads[1 - i % 2].address, 0,
                   buf.address, gneed, *sizes, 1, 1.0)
    dh.Cuda.deviceSynchronize()
    want = first * np.exp(g.astype(np.float64) * T)[:, None, None]
    for name, got, times in (("state", state, forward), ("gradient", grads[calls % 2], backward)):
        off = np.mean(got.get(first.shape) / want - 1.0, (1, 2))
        apart = np.minimum(np.abs(g) * T / times * 2.0 ** 23, d * d)
        bound = U * (4 * np.abs(g) * T + 6 * np.sqrt(times / (3 * apart)) + 4)
        assert (np.abs(off) <= bound).all(), "%s: off by %s U, %s U allowed" % (name, np.round(off / U, 1), np.round(bound / U, 1))
