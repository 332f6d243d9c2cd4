"""What the engine's token mixers accept and refuse of operands that are read value after value."""
import numpy as np
import pytest

from mixers import check, decay_reference, window_reference
from test_gpu_mixers import apart, eg, side_by_side, window_operands  # noqa: F401  (eg: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head", (1, 2, 4))
def test_a_decay_whose_rows_are_padded_is_refused(eg, head):
    """[head, 1] holds its values 4 floats apart."""
    from dragon_hip import engine
    rng = np.random.default_rng(head)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    N, L, d = 1, 5, 8
    Q, K, V, dY = f(N, head, L, d), f(N, head, L, d), f(N, head, L, d), f(N, head, L, d)
    g = -np.arange(1, head + 1, dtype=np.float32) / 8
    t = [eg.tensor(side_by_side(x), N, L, head * d).c() for x in (Q, K, V, dY)]
    want = decay_reference(Q, K, V, g, 0.5, [L], None, dY)
    for shape in ((head,), (1, head), (1, 1, head)) + (((1, 4), (2, 2)) if head == 4 else ()) + ((head, 1),):
        dec = eg.tensor(g, *shape).c()
        if shape[-1] % 4 and shape[-1] != head:
            with pytest.raises(engine.IllegalArgumentException):
                eg.linear_attention(*t[:3], dec, head, scale=0.5)
            with pytest.raises(engine.IllegalArgumentException):
                eg.linear_attention_delta(t[3], *t[:3], dec, head, scale=0.5)
        else:
            y = eg.linear_attention(*t[:3], dec, head, scale=0.5)
            check({"Y": apart(y.c().value(), N, head, L, d)}, want, str(shape))
            grads = eg.linear_attention_delta(t[3], *t[:3], dec, head, scale=0.5)
            check({n: apart(x.c().value(), N, head, L, d) for n, x in zip(("dQ", "dK", "dV"), grads)}, want, str(shape))


@pytest.mark.parametrize("QL", (7, 8))
def test_an_lse_whose_rows_are_padded_is_refused(eg, QL):
    from dragon_hip import engine
    N, H, d = 2, 3, 8
    Q, K, V, dY = window_operands(np.random.default_rng(QL), N, H, H, QL, QL, d, d)
    t = [eg.tensor(side_by_side(x), N, QL, H * d).c() for x in (Q, K, V, dY)]
    y, lse = eg.attention_window(*t[:3], H, window=4, scale=0.5, lse=True)
    again = eg.tensor(lse.c().value().reshape(-1), N, H, QL).c()
    if QL % 4:
        with pytest.raises(engine.IllegalArgumentException):
            eg.attention_window_delta(t[3], y, *t[:3], again, H, window=4, scale=0.5)
    else:
        grads = eg.attention_window_delta(t[3], y, *t[:3], again, H, window=4, scale=0.5)
        want = window_reference(Q, K, V, 0.5, 4, 0, [QL] * N, [QL] * N, dY)
        check({n: apart(x.c().value(), N, H, QL, d) for n, x in zip(("dQ", "dK", "dV"), grads)}, want)


def test_no_key_value_heads_are_refused(eg):
    from dragon_hip import engine
    q, k = eg.zeros(1, 5, 16).c(), eg.zeros(1, 5, 16).c()
    y, lse = eg.attention_window(q, k, k, 2, lse=True)
    y.c(), lse.c()
    for bad in (0, -1):
        with pytest.raises(engine.IllegalArgumentException):
            eg.attention_window(q, k, k, 2, bad)
        with pytest.raises(engine.IllegalArgumentException):
            eg.attention_window_delta(y, y, q, k, k, lse, 2, bad)
