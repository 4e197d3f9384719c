"""What an open block of the int8 cache costs: tokens that come one at a time are
rounded again each time that the block's scale grows.  The plain append of
tests/i8_ref.py, which the kernels match bit for bit, against that bound."""
import numpy as np
import pytest

from tests import i8_ref


def _filled(x, cuts):
    """One block filled with x [16, 128] in pieces that end at `cuts`: the values that it
    reads as, and its scale after each piece."""
    data = np.zeros((1, 1, 2, 1, 16, 128), np.int8)
    scale = np.zeros((1, 1, 2, 1, 1), np.float32)
    ptr, idx = np.array([0, 1], np.int32), np.zeros(1, np.int32)
    at, steps = 0, []
    for end in cuts:
        rows = x[at: end, None]
        i8_ref.append(data, scale, ptr, idx, np.array([end], np.int32), 0, rows, rows,
                      np.array([0, end - at]))
        steps.append(np.float64(scale[0, 0, 0, 0, 0]))
        at = end
    return data[0, 0, 0, 0].astype(np.float64) * steps[-1], steps


def _tokens(kind, rng):
    x = rng.standard_normal((16, 128))
    if kind == "grow":       # every token moves the scale by a little
        x[:, 5] = 3 * 1.01 ** np.arange(16) + 1
        x[:, 6:] = np.clip(x[:, 6:], -2.5, 2.5)
    if kind == "rise":
        x *= 1.5 ** np.arange(16)[:, None]
    return x.astype(np.float16)


@pytest.mark.parametrize("kind", ["normal", "grow", "rise"])
@pytest.mark.parametrize("cuts", [[16], [5, 16], [3, 4, 9, 16], list(range(1, 17))])
def test_error_is_half_a_step_for_each_growth(kind, cuts):
    """A token is rounded when it comes and whenever the scale has grown since, by at
    most half of the step of that time: |error| <= sum of s / 2 over those, so half a
    step for a block that came in one piece and never more than 8 steps."""
    for seed in range(20):
        x = _tokens(kind, np.random.default_rng(seed))
        got, steps = _filled(x, cuts)
        bound = np.zeros(16)
        at = 0
        for i, end in enumerate(cuts):
            if i and steps[i] != steps[i - 1]:
                bound[:at] += steps[i] / 2
            bound[at:end] += steps[i] / 2
            at = end
        err = np.abs(got - x.astype(np.float64)).max(1)
        assert (err <= bound * (1 + 1e-12)).all()
        assert bound.max() <= 8 * steps[-1]
        if len(cuts) == 1:
            assert bound.max() == steps[-1] / 2


def test_slow_growth_adds_up():
    """The bound is not one step: a scale that grows by 1% a token leaves codes below
    50 where they are each time, so that they grow with it."""
    x = _tokens("grow", np.random.default_rng(0))
    got, steps = _filled(x, list(range(1, 17)))
    assert np.abs(got - x.astype(np.float64)).max() > 2 * steps[-1]
