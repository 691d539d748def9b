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


@pytest.mark.parametrize("bound,sizes", [(4.0, [1] * 30), (1e5, [3, 1, 40, 2]), (1e6, [1])])
def test_recorded(deep, bound, sizes):  # noqa: F811
    """Clipping many handles as a graph, replayed on other gradients and again on the first."""
    h = deep

    def gradients(seed):
        rng = np.random.default_rng(seed)
        xs = [rng.normal(0, 1, (1, m, 16, 32)) for m in sizes]
        size = np.sqrt(sum((x ** 2).sum() for x in xs))
        return [_encrypt(h, x * (0.2 + 0.3 * seed) * bound / size, seed=10 * seed + k) for k, x in enumerate(xs)]

    first, other = gradients(1), gradients(2)
    periods = [512] * len(sizes)

    def run(grads):
        outs, square = h.clip_grad_norm(grads, bound / 4, bound, 7, periods=periods)
        return [*[o.ct for o in outs], square]

    want = [[h.lib.ct_export(o) for o in run(grads)] for grads in (first, other)]
    held = [h.lib.ct_export(x.ct) for x in first]
    h.lib.graph_begin()
    outs = run(first)
    graph = h.lib.graph_end()
    for words, res in ((None, want[0]), ([h.lib.ct_export(x.ct) for x in other], want[1]), (held, want[0])):
        for x, v in zip(first, words or ()):
            h.lib.ct_import(x.ct, v)
        h.lib.graph_launch(graph)
        for o, v in zip(outs, res):
            assert np.array_equal(h.lib.ct_export(o), v)
