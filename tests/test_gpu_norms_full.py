"""The calls of test_gpu_norms at the benchmark's parameters, where a CTA takes several members one after the other, against Python's own integers at some coefficients."""
import numpy as np
import pytest

from test_gpu_norms import _check, _ct, _objects, _pair, _pt, _rand, _scale

pytestmark = pytest.mark.gpu

# column tiles, token tiles, level: chunks of two with one left, of eight with one left, of eight without a rest, of one; sums in parts and whole
SHAPES = [(2, 9, 2), (9, 4, 2), (3, 16, 1), (1, 33, 1), (12, 1, 0), (3, 4, 5), (40, 1, 0), (6, 2, 3), (7, 2, 3), (5, 2, 2), (8, 2, 2), (4, 9, 2)]


@pytest.mark.parametrize("T,B,level", SHAPES)
def test_all_calls(gpu_full, T, B, level):
    g = gpu_full
    at = np.array([0, 1, 2, 255, 256, 511, 512, 513, 32767, 32768, 65023, 65535])
    x, y, z, mean, r = _rand(g, level, T * B, 1), _rand(g, level, T * B, 2, edge=True), _rand(g, level, T * B, 3), _rand(g, level, B, 4), _rand(g, level, B, 5)
    gamma, beta = (_rand(g, level, T, s, polys=1)[:, 0] for s in (6, 7))
    xo, yo, zo, mo, ro, go, bo = (_objects(v, at) for v in (x, y, z, mean, r, gamma, beta))
    cx, cy, cz, cm, cr = (_ct(g, v) for v in (x, y, z, mean, r))
    pg, pb, K = [_pt(g, v) for v in gamma], [_pt(g, v) for v in beta], _scale(g, level)
    of = [(t * B + b, t, b) for t in range(T) for b in range(B)]
    _check(g, g.norm_squares(cx, T, mean=cm, pad=5), [sum(_pair(xo[t * B + b] - mo[b], xo[t * B + b] - mo[b]) for t in range(T)) - 5 * _pair(mo[b], mo[b]) for b in range(B)], at, level, 3, 2)
    _check(g, g.norm_squares(cy, T), [sum(_pair(yo[t * B + b], yo[t * B + b]) for t in range(T)) for b in range(B)], at, level, 3, 2)
    _check(g, g.norm_scale(cx, cr, T, mean=cm), [_pair(xo[k] - mo[b], ro[b]) for k, _, b in of], at, level, 3, 2)
    _check(g, g.norm_scale(cx, cy, T, mean=cm), [_pair(xo[k] - mo[b], yo[k]) for k, _, b in of], at, level, 3, 2)
    _check(g, g.norm_affine(cx, T, gamma=pg, beta=pb), [np.stack([xo[k][0] * go[t] + K * bo[t], xo[k][1] * go[t]]) for k, t, _ in of], at, level, 2, 2)
    _check(g, g.norm_affine(cx, T, beta=pb), [np.stack([xo[k][0] + bo[t], xo[k][1]]) for k, t, _ in of], at, level, 2, 1)
    for handle, q in ((cz, zo), (None, xo)):
        rows, rowsum, cols, colsum = g.norm_grad_sums(cx, cy, T, g=handle)
        _check(g, rows, [sum(_pair(q[t * B + b], yo[t * B + b]) for t in range(T)) for b in range(B)], at, level, 3, 2)
        _check(g, rowsum, [sum(q[t * B + b] for t in range(T)) for b in range(B)], at, level, 2, 1)
        _check(g, cols, [sum(_pair(xo[t * B + b], yo[t * B + b]) for b in range(B)) for t in range(T)], at, level, 3, 2)
        _check(g, colsum, [sum(xo[t * B + b] for b in range(B)) for t in range(T)], at, level, 2, 1)
    nothing = 0 * xo[0][:1]
    _check(g, g.norm_grad_input(cz, cm, cy, cr, T), [np.concatenate([K * (zo[k] - mo[b]), nothing]) - _pair(yo[k], ro[b]) for k, _, b in of], at, level, 3, 2)
    xs = [cx, cm, cy]
    _check(g, g.square_sum_many(xs), [sum(_pair(v, v) for v in [*xo, *mo, *yo])], at, level, 3, 2)
    f = g.batch_slice(cr, 0, 1)
    for h, v in zip(g.scale_many(xs, f), (xo, mo, yo)):
        _check(g, h, [_pair(k, ro[0]) for k in v], at, level, 3, 2)
    _check(g, g.combine([cx, cy], [0.5, -1.0], 2.0), [_two(xo[k], yo[k], g, level) for k, _, _ in of], at, level, 2, 2)


def _two(x, y, g, level):
    s = float(g.scales[level])
    v = int(np.rint(0.5 * s)) * x + int(np.rint(-s)) * y
    v[0] = v[0] + int(np.rint(2.0 * s)) * _scale(g, level)
    return v
