"""The oracles of tests/mixers_exact.py see a single key or step go missing, at any place: mistakes planted in the oracle, on the
CPU."""
import numpy as np
import pytest

from mixers import check, decay_reference, window_reference
from mixers_exact import few, undecayed, uniform_window, whole_values


@pytest.mark.parametrize("case", [(2, 4, 2, 5, 40, 0, 0, [5, 3], [40, 31]), (1, 2, 1, 30, 90, 20, 3, [30], [90]), (1, 3, 3, 9, 4, 2, 2, [9], [4]),
                                  (2, 2, 1, 50, 50, 7, 60, [50, 0], [50, 0])], ids=str)
def test_uniform_attention_is_the_definition(case):
    N, H, G, QL, VL, window, sinks, ql, vl = case
    rng = np.random.default_rng(VL)
    V = whole_values(rng, (N, G, VL, 8))
    mine = uniform_window(V, H, QL, window, sinks, ql, vl)
    other = window_reference(np.zeros((N, H, QL, 4), np.float32), rng.standard_normal((N, G, VL, 4)).astype(np.float32), V, 0.5, window,
                             sinks, ql, vl)
    for name in ("Y", "lse"):
        assert np.array_equal(np.isneginf(mine[name][0]), np.isneginf(other[name][0]))
        ok = np.isfinite(mine[name][0])
        assert np.allclose(mine[name][0][ok], other[name][0][ok], rtol=1e-12, atol=1e-12)


def test_a_missing_or_repeated_key_of_a_long_cache_is_seen():
    rng = np.random.default_rng(24)
    G, VL, dv = 2, 45000, 16
    V = whole_values(rng, (1, G, VL, dv))
    want = uniform_window(V, 4, 1, 0, 0, [1], [VL])
    check({"Y": want["Y"][0].astype(np.float32), "lse": want["lse"][0].astype(np.float32)}, want)
    total = V.astype(np.float64).sum(2)
    cuts = sorted({VL * i // parts + d for parts in (2, 3, 32, 64) for i in range(parts) for d in (0, 15)} & set(range(VL)))
    for j in cuts:
        for lost, count in ((V[:, :, j], VL - 1), (-V[:, :, j], VL + 1), (V[:, :, j - j % 16:][:, :, :16].sum(2), VL - 16)):
            y = np.repeat((total - lost) / count, 2, 1)[:, :, None]
            with pytest.raises(AssertionError):
                check({"Y": y.astype(np.float32)}, want)
            with pytest.raises(AssertionError):      # the sum of the exponentials alone
                check({"Y": (np.repeat(total / count, 2, 1)[:, :, None]).astype(np.float32)}, want)


@pytest.mark.parametrize("lens", ([70, 70], [70, 33], [1, 0]))
def test_undecayed_is_the_definition(lens):
    rng = np.random.default_rng(3)
    Q, K, V, dY = few(rng, (2, 3, 70, 8)), few(rng, (2, 3, 70, 8)), few(rng, (2, 3, 70, 4)), few(rng, (2, 3, 70, 4))
    S0, dS1 = few(rng, (2, 3, 8, 4)), few(rng, (2, 3, 8, 4))
    mine = undecayed(Q, K, V, 0.5, lens, S0, dY, dS1)
    other = decay_reference(Q, K, V, np.zeros(3, np.float32), 0.5, lens, S0, dY, dS1)
    for name in mine:
        assert np.array_equal(mine[name], other[name][0]), name
