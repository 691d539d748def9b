"""Layer norm and its gradients one after the other at the benchmark's parameters, from what the forward pass kept: the degrees that leave it enough levels."""
import numpy as np
import pytest

from test_gpu_layer_norm import RANGE, TOL, _data, _decrypt, _encrypt, _model, _tiles, _whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,B,D,degree,weights", [(3, 2, 768, 14, True), (3, 1, 768, 7, False), (4, 2, 1001, 6, True)])
def test_forward_and_backward_in_the_full_ring(pkg, gpu_full, T, B, D, degree, weights):
    h = pkg.open_hemmer(gpu_full)
    w, rows, eps = 256, 128, 1e-3
    rng = np.random.default_rng(D + T)
    x, dy = _data(rng, B, rows, D), rng.uniform(-1, 1, (B, rows, D))
    gamma = rng.uniform(0.5, 1.5, D) if weights else None
    g1 = gamma if weights else np.ones(D)
    c, depth = h.polynomial("rsqrt", *RANGE, degree)
    y0, xhat0, r0 = _model(x, g1, 0.0, eps, RANGE, c)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, w)), D, RANGE, groups=T, gamma=gamma, eps=eps, degree=degree)
    assert np.abs(_whole(_decrypt(h, y, T, B), D) - y0).max() < TOL and h.lib.ct_meta(xhat.ct)[0] == 12 - 4 - depth
    dx, dgamma, dbeta = h.layer_norm_backward(_encrypt(h, _tiles(dy, T, w), seed=3), xhat, rstd, D, groups=T, gamma=gamma)
    g = dy * g1
    dx0 = r0 * (g - g.mean(-1, keepdims=True) - xhat0 * (g * xhat0).mean(-1, keepdims=True))
    assert np.abs(_whole(_decrypt(h, dx, T, B), D) - dx0).max() < TOL
    assert np.abs(_whole(_decrypt(h, dgamma, T, 1), D) - (dy * xhat0).sum((0, 1))).max() < B * rows * TOL / 8
    assert np.abs(_whole(_decrypt(h, dbeta, T, 1), D) - dy.sum((0, 1))).max() < B * rows * TOL / 8
    h.close()


@pytest.mark.parametrize("T,D,degree", [(3, 768, 15), (4, 1001, 7)])
def test_degrees_that_leave_too_few_levels(pkg, gpu_full, T, D, degree):
    """The forward pass is right; its gradients are refused, not wrong."""
    h = pkg.open_hemmer(gpu_full)
    rng = np.random.default_rng(D)
    x = _data(rng, 1, 128, D)
    c, _ = h.polynomial("rsqrt", *RANGE, degree)
    y, xhat, rstd = h.layer_norm(_encrypt(h, _tiles(x, T, 256)), D, RANGE, groups=T, degree=degree)
    assert np.abs(_whole(_decrypt(h, y, T, 1), D) - _model(x, 1.0, 0.0, 1e-5, RANGE, c)[0]).max() < TOL
    with pytest.raises(pkg.HBError) as e:
        h.layer_norm_backward(_encrypt(h, _tiles(x, T, 256), seed=2), xhat, rstd, D, groups=T)
    assert e.value.code == -1 and "level too low" in str(e.value)
    h.close()
