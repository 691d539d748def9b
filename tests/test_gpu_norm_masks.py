"""Layer norms with more ranges, levels and widths than masks are kept for."""
import numpy as np
import pytest

from test_gpu_layer_norm import RANGE, TOL, _data, _decrypt, _encrypt, _model, _tiles, _whole

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def full_cache(pkg):
    """Tiles of 16 x 32 after 70 ranges, and 31 widths at three levels."""
    g = pkg.open_gpu(pkg.make_params(log_n=10, max_level=12, dnum=4, num_special=3, hamming_weight=32))
    g.keygen()
    h = pkg.open_hemmer(g)
    x = np.random.default_rng(0).uniform(-1, 1, (1, 1, 16, 32))
    cx = _encrypt(h, x)
    for k in range(70):
        h.layer_norm(cx, 32, (0.1, 1.3 + 0.01 * k), degree=1)
    for level in (12, 11, 10):
        low = pkg.CtxtTensor(g.level_down(cx.ct, level), 16, 32, 32)
        for D in range(1, 32):
            h.layer_norm(low, D, RANGE, degree=1)
    yield h
    g.close()


@pytest.mark.parametrize("T,D", [(1, 32), (2, 64), (2, 45)])
def test_recorded(full_cache, T, D):
    h, B, w, rows, span = full_cache, 2, 32, 16, (0.1, 1.75 + T + D / 1000)
    rng = np.random.default_rng(D)
    x, dy = [_data(rng, B, rows, D) for _ in range(2)], rng.uniform(-1, 1, (B, rows, D))
    cx, other, cdy = _encrypt(h, _tiles(x[0], T, w)), _encrypt(h, _tiles(x[1], T, w), seed=7), _encrypt(h, _tiles(dy, T, w), seed=8)
    c, depth = h.polynomial("rsqrt", *span, 3)

    def step():
        y, xhat, rstd = h.layer_norm(cx, D, span, groups=T, degree=3)
        grads = h.layer_norm_backward(cdy, xhat, rstd, D, groups=T) if D == T * w else ()
        return [y.ct, xhat.ct, rstd.ct, *[t.ct for t in grads]], (y, xhat, rstd, grads)

    first = [h.lib.ct_export(o) for o in step()[0]]
    h.lib.graph_begin()
    try:
        outs, held = step()
    finally:
        graph = h.lib.graph_end()
    keep = h.lib.ct_export(cx.ct)
    h.lib.ct_import(cx.ct, h.lib.ct_export(other.ct))
    h.lib.graph_launch(graph)
    assert np.abs(_whole(_decrypt(h, held[0], T, B), D) - _model(x[1], 1.0, 0.0, 1e-5, span, c)[0]).max() < TOL
    h.lib.ct_import(cx.ct, keep)
    h.lib.graph_launch(graph)
    for o, want in zip(outs, first):
        assert np.array_equal(h.lib.ct_export(o), want)
    again = [h.lib.ct_export(o) for o in step()[0]]   # and without the graph, with masks made anew
    for a, b in zip(again, first):
        assert np.array_equal(a, b)


def test_the_same_as_in_a_cache_with_room(pkg, full_cache):
    """Bit for bit what a HEMMer over the same context gives that has kept no masks yet."""
    h, w, rows, D = full_cache, 32, 16, 45
    fresh = pkg.open_hemmer(h.lib)
    x = _data(np.random.default_rng(5), 1, rows, D)
    cx, span = _encrypt(h, _tiles(x, 2, w)), (0.1, 9.25)
    for a, b in zip(h.layer_norm(cx, D, span, groups=2, degree=3), fresh.layer_norm(cx, D, span, groups=2, degree=3)):
        assert np.array_equal(h.lib.ct_export(a.ct), h.lib.ct_export(b.ct))
    fresh.close()


@pytest.mark.parametrize("ring", ["gpu_small", "gpu_mid", "gpu_full"])
def test_masks_made_on_the_device(ring, request):
    """Bit for bit hb_encode of the same slots, again and again, recorded or not."""
    g = request.getfixturevalue(ring)
    for value, step, width, level in [(1.0, 32, 32, 3), (1.0 / 768, 256, 1, 8), (-0.3, 64, 23, 0), (2.5e-7, 2, 1, 5), (1e6, g.slots, 7, 2), (3.0, 1, 1, 1), (1.0, 16, 0, 4), (1e-30, 16, 3, 1)]:
        z = np.where(np.arange(g.slots) % step < width, value, 0.0)
        want = g.pt_export(g.encode(z, level))
        for _ in range(3):
            assert np.array_equal(g.pt_export(g.encode_mask(value, step, width, level)), want)
        g.graph_begin()
        pt = g.encode_mask(value, step, width, level)
        graph = g.graph_end()
        for _ in range(2):
            g.graph_launch(graph)
            assert np.array_equal(g.pt_export(pt), want)


def test_masks_that_are_refused(pkg, gpu_small):
    g = gpu_small
    for value, step, width, level in [(float("nan"), 16, 1, 1), (float("inf"), 16, 1, 1), (1.0, 0, 0, 1), (1.0, 24, 1, 1), (1.0, -16, 1, 1), (1.0, 2 * g.slots, 1, 1), (1.0, 16, 17, 1), (1.0, 16, -1, 1)]:
        with pytest.raises(pkg.HBError) as e:
            g.encode_mask(value, step, width, level)
        assert e.value.code == -1
    for level in (-1, g.L + 1):
        with pytest.raises(pkg.HBError):
            g.encode_mask(1.0, 16, 1, level)
    with pytest.raises(ValueError):
        g.encode_mask(1.0, 2 ** 32, 1, 1)
