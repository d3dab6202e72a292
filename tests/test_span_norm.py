"""CPU check of the 2-norm bounds that the GPU tests of the attention hold its results to: mistakes planted in 64-bit attention (a window
or the sinks one key off, a lost third of the weights' bits, a lost half of the queries') stand out of them at least twofold in every case."""
import numpy as np
import pytest

import span_norm as norm
import span_ref as ref
from span_cases import CHAIN, NORM_WINDOWS, inputs


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", NORM_WINDOWS)
def test_planted_mistakes_stand_out(T, pos0, nHq, nKv, hd, window, sinks):
    q, (kc, ks, vc, vs) = inputs(T, pos0, nHq, nKv, hd)
    S = pos0 + T
    K, V, p = ref.values(kc, ks), ref.values(vc, vs), pos0 + np.arange(T)

    def seen(w, s):
        return ref.visible(p, np.arange(S), w, s)
    want, w, tol, wtol = norm.attend(q, K, V, seen(window, sinks), CHAIN)
    assert tol < 1e-5

    def stands_out(got):
        assert norm.off(got, want) > 2 * tol
    stands_out(norm.two_pieces(w, vc, vs))
    half = norm.softmax(norm.scores(norm.upper_half(q), K, None), seen(window, sinks))
    stands_out(norm.mix(half, V))
    assert norm.off(half, w) > 2 * wtol
    planted = 0
    for other in ((window + 1, sinks), (window - 1, sinks), (window, sinks + 1), (window, sinks - 1)):
        if window < 0 or min(other) < 0 or np.array_equal(seen(*other), seen(window, sinks)):
            continue
        stands_out(norm.attend(q, K, V, seen(*other))[0])
        planted += 1
    assert planted or window < 0 or window > S
    # one key of the future seen, one row's own key hidden
    if T > 1:
        more = seen(window, sinks).copy()
        more[0, pos0 + 1] = True
        stands_out(norm.attend(q, K, V, more)[0])
