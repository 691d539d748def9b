"""What the library keeps for later calls (masks, keys) does not lie in the buffers that a recorded graph writes to at every replay, even when it is made after the recording."""
import numpy as np
import pytest

from test_gpu_layer_norm import _data, _encrypt, _tiles

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ring(pkg):
    g = pkg.open_gpu(pkg.make_params(log_n=10, max_level=12, dnum=4, num_special=3, hamming_weight=32))
    g.keygen()
    yield g, pkg.open_hemmer(g)
    g.close()


@pytest.mark.parametrize("level", [12, 11, 10, 9])
@pytest.mark.parametrize("T,B,D", [(2, 1, 60), (2, 1, 64), (3, 2, 90)])
def test_masks_of_a_layer_norm(ring, T, B, D, level):
    """Two ranges: the second one's masks are made after a layer norm with the first was recorded, and used again after its replay."""
    g, h = ring
    x = _data(np.random.default_rng(2), B, 16, D)
    cx = _encrypt(h, _tiles(x, T, 32), level)

    def run(hi):
        return [o.ct for o in h.layer_norm(cx, D, (0.1, hi), groups=T, degree=3)]

    run(1.3)
    g.graph_begin()
    held = run(1.3)
    graph = g.graph_end()
    want = {hi: [g.ct_export(o) for o in run(hi)] for hi in (1.4, 1.5, 1.6, 1.7)}
    for _ in range(2):
        g.graph_launch(graph)
        for hi, res in want.items():
            for a, b in zip(run(hi), res):
                assert np.array_equal(g.ct_export(a), b), hi
    assert len(held) == 3


def test_plaintexts_and_keys(ring):
    """Plaintexts, extended ones and masked keys of many levels, and rotation keys, made after a product was recorded."""
    g, h = ring
    rng = np.random.default_rng(3)
    a, b = (h.encrypt2(rng.uniform(-1, 1, (16, 16)), rng.uniform(-1, 1, (16, 16)), nonce=k) for k in (1, 2))

    def product():
        return h.single_cc_matmul(a, b, 8).ct

    product()
    g.graph_begin()
    held = product()
    graph = g.graph_end()
    z = rng.uniform(-1, 1, g.slots)
    pts = [g.encode(z, level) for level in range(g.L + 1) for _ in range(4)]
    pts += [g.encode_ext(z, level) for level in range(g.L + 1) for _ in range(2)]
    words = [g.pt_export(p) for p in pts]
    steps = list(range(33, 45))
    g.gen_rot_keys(steps)
    keys = [g.evk_export(g.galois(k)) for k in steps]
    for _ in range(2):
        g.graph_launch(graph)
    for p, w in zip(pts, words):
        assert np.array_equal(g.pt_export(p), w)
    for k, w in zip(steps, keys):
        assert np.array_equal(g.evk_export(g.galois(k)), w)
    assert held is not None


def test_masks_of_products(ring):
    """Products of other levels and schedules, whose masks and masked keys are made after the first one was recorded."""
    g, h = ring
    rng = np.random.default_rng(4)
    a, b = (h.encrypt2(rng.uniform(-1, 1, (16, 16)), rng.uniform(-1, 1, (16, 16)), nonce=k) for k in (1, 2))
    wide = h.encrypt2(rng.uniform(-1, 1, (16, 16)), rng.uniform(-1, 1, (16, 16)), nonce=3)
    h.single_cc_matmul(a, b, 8)
    g.graph_begin()
    held = h.single_cc_matmul(a, b, 8)
    graph = g.graph_end()

    def others():
        return [g.ct_export(h.single_cc_matmul(a, wide, level).ct) for level in (3, 4, 5, 6, 7, 9)]

    want = others()
    for _ in range(2):
        g.graph_launch(graph)
        for x, y in zip(others(), want):
            assert np.array_equal(x, y)
    assert held is not None
