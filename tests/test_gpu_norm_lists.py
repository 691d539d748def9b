"""Lists of tensors whose members fill their launches to the last: a launch takes 256 members."""
import numpy as np
import pytest

from test_gpu_layer_norm import TOL, _decrypt, _encrypt
from test_gpu_norms import _check, _objects, _pair
from test_gpu_tile_products import _ct, _points, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [[256], [512], [255, 1], [1] * 256, [128, 384], [100, 156, 256], [255], [257]], ids=lambda s: f"{len(s)}x{sum(s)}")
def test_products_of_full_launches(gpu_small, sizes):
    g, level = gpu_small, 1
    xs, f = [_rand(g, level, m, 10 + k) for k, m in enumerate(sizes)], _rand(g, level, 1, 9)
    at = _points(g, np.random.default_rng(len(sizes)), 12)
    handles, cf, fo = [_ct(g, x) for x in xs], _ct(g, f), _objects(f, at)[0]
    got = g.scale_many(handles, cf)
    assert len(got) == len(xs)
    for h, x in zip(got, xs):
        _check(g, h, [_pair(m, fo) for m in _objects(x, at)], at, level, 3, 2)
    _check(g, g.square_sum_many(handles), [sum(_pair(m, m) for x in xs for m in _objects(x, at))], at, level, 3, 2)


def test_clipping_256_members(pkg):
    """Gradients of 256 members in all, their norm twice the limit (degree 15 is off by less than 0.05 there)."""
    g = pkg.open_gpu(pkg.make_params(log_n=10, max_level=8, dnum=3, num_special=3, hamming_weight=32))
    g.keygen()
    h = pkg.open_hemmer(g)
    try:
        rng = np.random.default_rng(3)
        xs = [rng.normal(0, 1, (1, B, 16, 32)) for B in (250, 5, 1)]
        size = np.sqrt(sum((x ** 2).sum() for x in xs))
        xs = [x * 2.0 / size for x in xs]
        outs, square = h.clip_grad_norm([_encrypt(h, x, seed=k) for k, x in enumerate(xs)], 1.0, 4.0, 15)
        assert np.abs(g.decrypt(square) - 4.0).max() < 16 * TOL
        for o, x in zip(outs, xs):
            got = _decrypt(h, o, 1, x.shape[1])
            f = (got * x).sum() / (x * x).sum()
            assert abs(f - 0.5) < 0.05 and np.abs(got - f * x).max() < TOL
    finally:
        g.close()
