"""Clipping with bounds up to the largest that is let through, beyond which it is refused.

The square of the norm is brought to [-1, 1] by 2 / bound^2, a whole number of units of 2^-42, of which a bound of 10^6 has nine.  What comes out has to be the
gradient times the factor to what the polynomial promises: for bound = 4 max_norm a degree of 15 is within 0.05 of min(1, max_norm / norm) up to the bound."""
import numpy as np
import pytest

from test_gpu_layer_norm import _decrypt, _encrypt, deep  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", [0.2, 0.5, 0.999])
@pytest.mark.parametrize("bound", [1e1, 1e3, 2000.0, 1e4, 1e5, 3.7e5, 7e5, 8.5e5, 1e6])
def test_large_bounds(deep, bound, place):  # noqa: F811
    h, rng = deep, np.random.default_rng(7)
    norm, limit = place * bound, bound / 4
    x = rng.normal(0, 1, (1, 2, 16, 32))
    x *= norm / np.sqrt((x ** 2).sum())
    outs, square = h.clip_grad_norm([_encrypt(h, x)], limit, bound, 15)
    assert abs(h.lib.decrypt(square)[0].real / norm ** 2 - 1) < 2.0 ** -14
    # the tile's imaginary parts are noise beside values of this size: 2^-14 of the largest is what a product has to meet
    z = h.lib.decrypt_many([(outs[0].ct, k) for k in range(2)])
    got, size = z.real.reshape(x.shape), np.abs(x).max()
    f = (got * x).sum() / (x * x).sum()
    assert np.abs(got - f * x).max() < size * 2.0 ** -14 and np.abs(z.imag).max() < size * 2.0 ** -14
    assert abs(f - min(1.0, limit / norm)) < 0.05


@pytest.mark.parametrize("bound", [1.1e6, 2e6, 3e6, 4.2e6, 1e7, 1e9, 1e150])
def test_bounds_that_are_refused(pkg, deep, bound):  # noqa: F811
    h = deep
    x = _encrypt(h, np.random.default_rng(1).uniform(-1, 1, (1, 1, 16, 32)))
    with pytest.raises(pkg.HBError) as e:
        h.clip_grad_norm([x], bound / 4, bound, 15)
    assert e.value.code == -1 and "bound" in str(e.value)
    outs, _ = h.clip_grad_norm([x], 10.0, 40.0, 3)   # and the handle goes on working
    assert h.lib.ct_meta(outs[0].ct)[1] == 2
