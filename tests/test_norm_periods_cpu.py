"""Periods of gradients that do not belong to them stay in Python."""
from types import SimpleNamespace

import pytest


def test_periods_of_another_number(pkg):
    h = object.__new__(pkg.Hemmer)
    h.lib = SimpleNamespace(slots=512)
    h._call = lambda *a: pytest.fail("reached the library")
    h._fn = lambda *a: pytest.fail("reached the library")
    g = pkg.CtxtTensor(SimpleNamespace(ptr=SimpleNamespace(value=1)), 16, 32, 32)
    for periods in ([], [32], [32] * 3, [2 ** 31, 32], [2 ** 40, None]):
        with pytest.raises(ValueError):
            h.grad_norm_squared([g, g], periods)
        with pytest.raises(ValueError):
            h.clip_grad_norm([g, g], 1.0, 2.0, periods=periods)
    assert list(h._periods([None, 32], 2)) == [512, 32] and h._periods(None, 2) is None
