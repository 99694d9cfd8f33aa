"""What a sequence gives up before its end, and verification, without a GPU: entry points without a cache, and the oracle that the GPU tests rest on."""

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from oracle.cache_steps_oracle import BAD_VALUE, Steps, verify


@pytest.fixture(scope="module")
def lib():
    _cabi.build()
    return _cabi.load()


def test_calls_without_a_cache(lib):
    assert lib.kb200_cache_attend_window(None, 0, None, None, 1, 1, None, None, None, None, 1.0, 4, 0, None, None, None, None, 0, None) == -1
    assert lib.kb200_cache_attend_window(None, 0, None, None, 1, 1, None, None, None, None, 1.0, -4, 0, None, None, None, None, 0, None) == -1
    assert lib.kb200_cache_release(None, 4, 0, None) == -1
    assert lib.kb200_cache_weigh(None, 0, None, None, None, 1, 1, None, None, None, None, 1.0, 0, None, 0, None, 0, None) == -1
    assert lib.kb200_cache_evict(None, None, 0, None, 0, 0, None, 0, None, 0, None) == -1
    assert lib.kb200_cache_verify(None, None, None, 1, 1, 1, None, None, 0, None, None, None, None, None, None, None, None, 0, None) == -1
    assert lib.kb200_cache_attend_window_workspace(None, 1, 1, 1, 4, 0) == lib.kb200_cache_evict_workspace(None) == lib.kb200_cache_verify_workspace(None, 1, 1, 1) == 0


def test_calls_of_a_closed_cache(lib):
    call = _cabi.load_call()
    with pytest.raises(ValueError, match="closed"):
        call.cache_release(None, 4, 0)
    with pytest.raises(ValueError, match="closed"):
        call.cache_weigh(*[None] * 11)
    with pytest.raises(ValueError, match="closed"):
        call.cache_evict(*[None] * 6)
    with pytest.raises(ValueError, match="closed"):
        call.cache_verify(*[None] * 9)
    with pytest.raises(TypeError):
        call.cache_verify(None)
    with pytest.raises(TypeError):
        call.cache_weigh(*[None] * 10)


def filled(lengths, drafted):
    generator = torch.Generator().manual_seed(1)
    o = Steps(2, len(lengths), 6, 40, 2, 16, 8, torch.float32)
    for n in (lengths, drafted):
        o.reserve(list(n))
        k, v = (torch.randn(len(n), max(n), 2, 16, generator=generator) for _ in range(2))
        for layer in range(2):
            o.append(layer, k, v, list(n))
        if n is lengths:
            o.accept(list(n))
    return o, torch.randn(len(lengths), max(drafted), 4, 16, generator=generator)


def test_oracle_of_windows():
    """A window that all tokens are in is no window; one of a single token is that token's value; released pages are not missed."""
    o, q = filled([30, 9], [3, 2])
    want, *_ = o.attend(0, q, None, [3, 2])
    for window, sinks in ((None, 0), (100, 0), (33, 0), (1, 100)):
        got, *_ = o.look(0, q, None, [3, 2], window=window, sinks=sinks)
        assert np.abs(got - want).max() < 1e-14
    got, _, _, lse = o.look(0, q, None, [3, 2], window=1)
    page, row = o._place(0, 31)
    assert np.allclose(got[0, 1, 0], o.pool[0, 1, page, 0, row]) and np.allclose(lse[0, 1, 0], o.pool[0, 0, page, 0, row] @ q[0, 1, 0].double().numpy() / 4)
    before, *_ = o.look(0, q, None, [3, 2], window=10, sinks=1)
    o.release(10, 1)
    assert o.rows[0][0] >= 0 and o.rows[0][1] == -1 and o.rows[0][2] >= 0 and -1 not in o.rows[1]      # (tokens 8 to 15 are gone)
    assert np.array_equal(o.look(0, q, None, [3, 2], window=10, sinks=1)[0], before)


def test_oracle_of_weights_and_evictions():
    o, q = filled([30, 9], [3, 2])
    *_, lse = o.look(0, q, None, [3, 2])
    weights, _ = o.weigh(0, q, lse, np.zeros((2, 48)), None, [3, 2])
    assert np.allclose(weights.sum(1), [12, 8]) and (weights[0, 33:] == 0).all() and weights[0, 32] < weights[0].max()
    o.accept([3, 2])
    marks = [[(o.pool[0, 0][o._place(s, j)[0], 0, o._place(s, j)[1]]).copy() for j in range(o.lengths[s])] for s in range(2)]
    weights = np.zeros((2, 48))
    weights[0, [5, 20, 21]] = 3, 5, 5
    weights[1] = np.nan
    after = o.evict(weights, [6, -1], recent=2, sinks=1)
    assert o.lengths == [6, 11] and after[0].tolist() == [0, 3, 5, 5, 0, 0] + [0] * 42 and np.isnan(after[1, :11]).all() and (after[1, 11:] == 0).all()
    for i, j in enumerate([0, 5, 20, 21, 31, 32]):
        page, row = o._place(0, i)
        assert np.array_equal(o.pool[0, 0, page, 0, row], marks[0][j])
    assert o.faults == 0


def test_oracle_of_verification():
    """By hand: three tokens of chances 1/2, 1/4 and 1/4."""
    p = torch.tensor([0.5, 0.25, 0.25]).log()
    logits = p.expand(1, 3, 3)

    def step(tokens, uniform, **kw):
        n, accepted, following, faults = verify(1, logits, torch.tensor([tokens]), torch.tensor([uniform]), **kw)
        assert faults == 0
        return accepted[0][:n[0]], following[0]

    assert step([0, 0, 1], [0.8, 0.4, 0.2]) == ([0, 1, 2], 2)              # both taken, and the last quarter drawn
    assert step([0, 0, 1], [0.8, 0.4, 0.3]) == ([0, 1], 2)                 # the second is not: of what is left, 1/2 and 1/4, 0.8 is in the last third
    assert step([0, 0, 1], [0.6, 0.6, 0.1]) == ([0], 2)                    # the first is not, and nobody asks for the second
    assert step([0, 0, 1], [0.6, 0.6, 0.4], parents=torch.tensor([-1, 0, 0])) == ([0, 2], 1)      # ... but for one that followed the same token: a half of what is left
    q = torch.tensor([0.25, 0.5, 0.25]).expand(1, 3, 3)
    assert step([0, 1, 2], [0.0, 0.4, 0.9], draft=q)[0] == [0, 1, 2]       # chances by the draft's: 1/2, and 1
    assert step([0, 1, 2], [0.9, 0.5, 0.9], draft=q) == ([0], 0)           # what is left is all the first token's
    assert step([0, 1, 2], [0.9, 0.0, 0.0], draft=q, temperature=torch.zeros(1)) == ([0], 0)
    n, accepted, following, faults = verify(2, torch.full((1, 3, 3), float("nan")), torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, 3), slots=[1])
    assert (n, accepted, following, faults) == ([0, 1], [[-1] * 3, [0, -1, -1]], [-1, -1], BAD_VALUE)
