"""The closed form of linear attention with decay against the recurrence, on the CPU."""
import numpy as np
import pytest

import sequence_closed as closed
import sequence_reference as ref


@pytest.mark.parametrize("lengths", [None, [0, 5, 9, 12]], ids=str)
@pytest.mark.parametrize("given", [True, False])
def test_the_closed_form_is_the_recurrence(given, lengths):
    B, T, H, KH, dk, dv = 4, 9, 4, 2, 3, 5
    rng = np.random.default_rng(3)
    mk = lambda *s: rng.normal(size=s)
    q, k, v, go, state, gs = mk(B, T, H, dk), mk(B, T, KH, dk), mk(B, T, KH, dv), mk(B, T, H, dv), mk(B, H, dk, dv), mk(B, H, dk, dv)
    g = np.array([-0.1, -1.0, 0.0, -np.inf])
    n = None if lengths is None else np.array(lengths)
    if not given:
        state = gs = None
    got = closed.attention(q, k, v, g, state, n, 0.3) + closed.attention_backward(go, q, k, v, g, state, n, 0.3, gs)
    with np.errstate(invalid="ignore"):
        want = ref.attention(q, k, v, g, state, n, 0.3) + ref.attention_backward(go, q, k, v, g, state, n, 0.3, gs)
    for i, (a, b) in enumerate(zip(got, want)):
        assert np.abs(a - b).max() < 1e-13, i
