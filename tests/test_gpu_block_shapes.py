"""Products of all pairs of tiles and products grouped by expert in every block that the rules of dispatch choose, every coefficient against the calls that do the same pair by
pair and position by position.  tests/test_block_shapes_cpu.py holds these cases to reaching all of the blocks.  Whole numbers: equal or wrong."""
import ctypes as C

import numpy as np
import pytest

from conftest import FULL, MID, SMALL

pytestmark = pytest.mark.gpu

RINGS = {"small": SMALL, "mid": MID, "full": dict(FULL, log_n=16)}

# ring, level, groups, heads, query tiles, key tiles, all residues q - 1
PAIRS = [
    ("small", 1, 1, 1, 1, 1, False), ("small", 7, 3, 296, 1, 1, False), ("mid", 3, 1, 296, 1, 1, False), ("mid", 7, 5, 296, 1, 1, False), ("full", 1, 2, 148, 1, 1, False),
    ("small", 1, 2, 1, 1, 2, False), ("small", 7, 33, 296, 2, 1, True), ("mid", 3, 5, 296, 1, 2, False), ("mid", 7, 1, 296, 2, 1, False), ("full", 1, 1, 148, 2, 1, False),
    ("small", 1, 3, 1, 4, 1, False), ("small", 7, 1, 296, 3, 1, False), ("mid", 3, 2, 296, 1, 4, False), ("mid", 7, 3, 296, 4, 1, False), ("full", 1, 1, 148, 1, 3, False),
    ("small", 1, 1, 1, 2, 2, False), ("small", 7, 5, 296, 2, 2, False), ("mid", 3, 1, 296, 2, 2, False), ("mid", 7, 2, 296, 2, 2, False), ("full", 1, 1, 148, 2, 2, False),
    ("small", 1, 2, 1, 4, 2, False), ("small", 3, 1, 296, 2, 3, False), ("small", 7, 3, 296, 4, 2, False), ("mid", 3, 1, 296, 3, 2, False), ("mid", 7, 2, 296, 2, 4, False),
    ("small", 1, 3, 1, 4, 4, False), ("small", 1, 5, 296, 3, 4, False), ("small", 3, 33, 296, 4, 3, True), ("small", 7, 1, 296, 4, 4, False), ("mid", 3, 5, 296, 3, 3, False),
]

# ring, level, copies, inputs, K-groups, sizes, tiles, all residues q - 1
EXPERTS = [
    ("mid", 2, 5, 4, 2, [1], 1, False), ("mid", 2, 5, 4, 2, [4, 4, 1], 1, False), ("mid", 2, 5, 4, 2, [5, 4, 1], 1, False),
    ("mid", 2, 5, 4, 2, [2, 2, 1], 2, False), ("mid", 2, 5, 4, 2, [4, 4, 1], 2, False), ("mid", 2, 5, 4, 2, [5, 4, 1], 2, False), ("mid", 2, 3, 3, 1, [1, 1, 1], 3, False),
    ("mid", 2, 5, 4, 2, [2, 2, 1], 3, False), ("mid", 2, 5, 4, 2, [4, 4, 1], 3, False), ("mid", 2, 5, 4, 2, [5, 4, 1], 3, False), ("mid", 2, 3, 3, 1, [1, 1, 1], 4, False),
    ("mid", 2, 5, 4, 2, [2, 2, 1], 4, False), ("mid", 2, 5, 4, 2, [4, 4, 1], 4, False), ("mid", 2, 5, 4, 2, [5, 4, 1], 4, False), ("mid", 2, 3, 3, 1, [1, 1, 1], 5, False),
    ("mid", 2, 5, 4, 2, [3, 3, 1], 5, False), ("mid", 2, 5, 4, 2, [2, 2, 1], 7, False), ("mid", 2, 5, 4, 2, [3, 2, 1], 7, False), ("mid", 2, 5, 4, 2, [1, 1, 1], 10, False),
    ("full", 1, 6, 3, 1, [3, 2], 12, False), ("full", 5, 3, 3, 2, [3, 2, 1], 12, False), ("full", 2, 5, 2, 16, [2, 1], 6, False), ("full", 1, 2, 2, 3, [1], 8, False),
    # sums on both sides of the counts after which they are reduced, several positions at a time
    ("mid", 2, 127, 2, 1, [3, 3, 1], 5, True), ("mid", 2, 128, 2, 1, [3, 3, 1], 5, True), ("mid", 2, 129, 2, 1, [3, 3, 1], 5, True), ("mid", 2, 43, 2, 3, [3, 3, 1], 5, True),
    ("mid", 2, 127, 2, 1, [3, 2, 1], 7, True), ("mid", 2, 128, 2, 1, [3, 2, 1], 7, True), ("mid", 2, 129, 2, 1, [3, 2, 1], 7, True), ("mid", 2, 257, 2, 1, [3, 2, 1], 7, True),
]


@pytest.fixture(autouse=True)
def _memory_goes_back(request):
    """The cases are large, and tests that fill the GPU come after them."""
    import torch
    yield
    g = request.getfixturevalue("gpu_" + request.node.callspec.params["ring"])
    g._chk(g._fn("release_cached")(g.ctx))
    torch.cuda.empty_cache()


def _view(handle):
    """The device words of a handle, for torch."""
    import torch
    lib = handle.lib
    meta = lib.ct_meta(handle) if handle.kind == "ct" else lib.pt_meta(handle)
    address = lib._fn(handle.kind + "_device_ptr")
    address.restype = C.c_void_p

    class View:
        __cuda_array_interface__ = {"shape": (meta[2], meta[1], meta[0] + 1, lib.N) if handle.kind == "ct" else (meta[0] + 1, lib.N), "typestr": "<i8", "data": (address(handle.ptr), False), "version": 3,
                                    "strides": None}

    return torch.as_tensor(View(), device="cuda")


def _fill(handle, gen, largest):
    view, lib = _view(handle), handle.lib
    for l in range(view.shape[-2]):
        q = int(lib.primes[l])
        view[..., l, :].fill_(q - 1) if largest else view[..., l, :].random_(0, q, generator=gen)
    return handle


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _take(handle, members):
    """A ciphertext of some members of another."""
    import torch
    view = _view(handle)
    out = handle.lib.ct_create(view.shape[2] - 1, view.shape[1], len(members), 1)
    _view(out).copy_(view[torch.tensor(members, device="cuda")])
    torch.cuda.synchronize()
    return out


def _pair_by_pair(g, a, b, groups, heads, nq, nk, i, j):
    """[head]: the sums of one pair, up to eight groups a call"""
    out = C.c_void_p()
    for g0 in range(0, groups, 8):
        part = range(g0, min(groups, g0 + 8))
        x = _take(a, [(gr * heads + h) * nq + i for gr in part for h in range(heads)])
        y = _take(b, [(gr * heads + h) * nk + j for gr in part for h in range(heads)])
        g._chk(g.dll.hb_tensor_acc_groups(g.ctx, x.ptr, y.ptr, C.c_int(len(part)), C.byref(out)))
        g.sync()
    return type(a)(g, out, "ct")


@pytest.mark.parametrize("ring,level,groups,heads,nq,nk,largest", PAIRS)
def test_pairs(request, ring, level, groups, heads, nq, nk, largest):
    import torch
    g = request.getfixturevalue("gpu_" + ring)
    gen = _gen(groups + nq)
    a, b = (_fill(g.ct_create(level, 2, groups * heads * n, 1), gen, largest) for n in (nq, nk))
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    got = g.tensor_acc_cross(a, b, groups, heads=heads)
    g.sync()
    assert g.ct_meta(got) == (level, 3, heads * nq * nk, 2)
    out = _view(got).view(nk, heads, nq, 3, level + 1, g.N)
    for i, j in np.ndindex(nq, nk):
        assert torch.equal(out[j, :, i], _view(_pair_by_pair(g, a, b, groups, heads, nq, nk, i, j))), (i, j)
    # once more into the sums: twice of them
    primes = torch.tensor([int(q) for q in g.primes[: level + 1]], device="cuda")[:, None]
    want = _view(got) * 2
    want -= torch.where(want >= primes, primes, 0)
    torch.cuda.synchronize()
    assert g.tensor_acc_cross(a, b, groups, heads=heads, acc=got) is got
    g.sync()
    assert torch.equal(_view(got), want)


@pytest.mark.parametrize("ring,level,copies,inputs,bcount,sizes,tiles,largest", EXPERTS)
def test_experts(request, ring, level, copies, inputs, bcount, sizes, tiles, largest):
    import torch
    g = request.getfixturevalue("gpu_" + ring)
    gen, step = _gen(copies + tiles), 2 << ((g.N.bit_length() - 3) // 2)
    pre = _fill(g.ct_create(level, 2, copies * inputs * bcount, 1), gen, largest)
    pts = [[[_fill(g.encode(np.zeros(1), level), gen, largest) for _ in range(bcount)] for _ in range(tiles)] for _ in sizes]
    order = [(3 * p + 1) % inputs for p in range(sum(sizes))]
    torch.cuda.synchronize()
    got = g.matmul_acc_grouped(pre, inputs, sizes, pts, step, order=order)
    g.sync()
    assert g.ct_meta(got) == (level, 2, len(order) * tiles, 2)
    out, expert = _view(got), [e for e, n in enumerate(sizes) for _ in range(n)]
    for p, t in np.ndindex(len(order), tiles):
        arr, one = (C.c_void_p * bcount)(*[w.ptr.value for w in pts[expert[p]][t]]), C.c_void_p()
        g._chk(g.dll.hb_matmul_acc_multi(g.ctx, pre.ptr, C.c_int(inputs * bcount), C.c_int(order[p] * bcount), arr, C.c_int(bcount), C.c_int64(step), C.byref(one)))
        g.sync()
        assert torch.equal(out[p * tiles + t], _view(type(pre)(g, one, "ct"))[0]), (p, t)
