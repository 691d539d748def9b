"""Products of a transformer block on ciphertexts beyond one token tile and one weight matrix, as cases that can be timed and compared.

  cross     attention of query tiles to key (or value) tiles of another length: out[j][h][i] = sum_g a[g][h][i] (x) b[g][h][j], the tensor
            products of all pairs of tiles of a head; g runs over the shifted copies of a tile product (and over the key tiles where values are summed)
  grouped   ciphertext x plaintext products grouped by expert: out[p][t] = sum_b sum_k pre[k][order[p]][b] (.) rot_k(w[expert of p][t][b]);
            the experts' groups are ragged, some are empty, an input may be at several experts
  encode    plaintext operands from 4-bit weights with group scales, W = (code - 8) * scale[row // group][column]
  matvec    encrypted vectors x 4-bit weights: out[v][j] = sum_b x[v][b] (.) encode(W block (b, j))

Everything is residues modulo the primes of a context, so outputs are whole numbers and have one right value.  Ciphertexts are
[members][polynomials][limbs][N], plaintexts [limbs][N], both in transform order.
"""
from __future__ import annotations

import ctypes
import importlib
import math
import random

import numpy as np
import torch

own = False

PKG = "encryption-friendly_llm_architecture_b200"
# the benchmark context and the small one of the documentation: (levels, digits of the gadget, Hamming weight of the secret)
RINGS = {16: (12, 4, 192), 12: (8, 3, 64)}
SPECIAL, Q0_BITS, Q_BITS, P_BITS = 3, 60, 42, 60


def _tile(log_n):
    return 1 << ((log_n - 2) // 2)   # two tiles of this side fill the slots


def listed():
    return [
        # one query tile against one key tile in a small ring: the latency of a call
        {"name": "cross_small", "op": "cross", "log_n": 12, "level": 6, "groups": 8, "heads": 1, "queries": 1, "keys": 1},
        # scores of 128 decoder tokens to 512 encoder tokens, twelve heads two per ciphertext, a step of eight shifted copies
        {"name": "cross_scores", "op": "cross", "log_n": 16, "level": 5, "groups": 8, "heads": 6, "queries": 1, "keys": 4},
        # scores x values: 512 queries, the sum over four key tiles and eight copies
        {"name": "cross_values", "op": "cross", "log_n": 16, "level": 5, "groups": 32, "heads": 3, "queries": 4, "keys": 1},
        # 512 queries to 1024 keys
        {"name": "cross_long", "op": "cross", "log_n": 16, "level": 5, "groups": 8, "heads": 6, "queries": 4, "keys": 8},
        # three inputs at four experts, one output tile, small ring
        {"name": "grouped_small", "op": "grouped", "log_n": 12, "level": 5, "inputs": 3, "blocks": 1, "experts": 4, "top": 1, "tiles": 1},
        # five sequences, each at one of four adapters of one 768-wide projection
        {"name": "grouped_adapters", "op": "grouped", "log_n": 16, "level": 5, "inputs": 5, "blocks": 1, "experts": 4, "top": 1, "tiles": 6},
        # four sequences at two of three experts each, 768 inputs in two packed groups, twelve output tiles
        {"name": "grouped_top2", "op": "grouped", "log_n": 16, "level": 5, "inputs": 4, "blocks": 2, "experts": 3, "top": 2, "tiles": 12},
        # an odd matrix with an odd group in a small ring
        {"name": "encode_small", "op": "encode", "log_n": 12, "level": 5, "rows": 100, "cols": 70, "group": 48, "diagonal": True},
        # the weights of the Q, K and V projections
        {"name": "encode_qkv", "op": "encode", "log_n": 16, "level": 5, "rows": 768, "cols": 2304, "group": 128, "diagonal": True},
        # one token through a 768 x 768 head, at the level that one product needs
        {"name": "matvec_head", "op": "matvec", "log_n": 16, "level": 1, "rows": 768, "cols": 768, "group": 64, "vectors": 1},
        # one token through an odd matrix, no size a multiple of anything
        {"name": "matvec_odd", "op": "matvec", "log_n": 16, "level": 3, "rows": 1001, "cols": 333, "group": 48, "vectors": 1},
        # four tokens through a wide matrix, with room for the products that follow
        {"name": "matvec_wide", "op": "matvec", "log_n": 16, "level": 5, "rows": 2048, "cols": 2048, "group": 128, "vectors": 4},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _drawn(rng):
    op, log_n = rng.choice(["cross", "cross", "grouped", "grouped", "encode", "matvec"]), rng.choice([12, 16, 16, 16])
    c = {"op": op, "log_n": log_n, "level": rng.randint(1, 8)}
    if op == "cross":
        return c | {"groups": _log(rng, 1, 64), "heads": rng.randint(1, 6), "queries": _log(rng, 1, 8), "keys": _log(rng, 1, 12)}
    if op == "grouped":
        experts = rng.randint(1, 8)
        return c | {"inputs": rng.randint(1, 6), "blocks": rng.randint(1, 3), "experts": experts, "top": min(experts, rng.randint(1, 3)), "tiles": _log(rng, 1, 12)}
    c |= {"rows": _log(rng, 1, 2048), "cols": _log(rng, 1, 2304), "group": rng.choice([1, 16, 32, 48, 64, 128, 256])}
    return c | ({"diagonal": rng.random() < 0.7} if op == "encode" else {"vectors": rng.randint(1, 5)})


def _cost(c):
    """(bytes held, products): what a pass takes, roughly, on either side."""
    n, N = c["level"] + 1, 1 << c["log_n"]
    if c["op"] == "cross":
        held = c["groups"] * c["heads"] * (c["queries"] + c["keys"]) * 2 + 3 * c["heads"] * c["queries"] * c["keys"]
        return held * n * N * 8, 4 * c["groups"] * c["heads"] * c["queries"] * c["keys"] * n * N
    if c["op"] == "grouped":
        d, pairs = _tile(c["log_n"]), c["inputs"] * c["top"]
        held = d * c["inputs"] * c["blocks"] * 2 + c["experts"] * c["tiles"] * c["blocks"] + pairs * c["tiles"] * 2
        return held * n * N * 8, 2 * d * pairs * c["tiles"] * c["blocks"] * n * N
    kb, nb = _blocks(c)
    return (kb * nb + c.get("vectors", 0) * (kb + nb) * 2) * n * N * 8, kb * nb * (n * N * 8 + N * 8)


def draw(rng):
    most = {}
    for c in listed():
        a, b = _cost(c)
        most[c["op"]] = max(most.get(c["op"], (0, 0)), (a, b), key=lambda v: v[1])
    while True:
        c = _drawn(rng)
        held, products = _cost(c)
        if products <= most[c["op"]][1] and held <= 1.2 * most["grouped"][0] and (c["op"] != "encode" or math.prod(_blocks(c)) <= 48):
            return c


# ---- the arithmetic of a context: primes, scales, roots (the rules of the library, restated) ------------------------
def _is_prime(n):
    d, r = n - 1, 0
    while d % 2 == 0:
        d, r = d // 2, r + 1
    for b in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37):
        x = pow(b, d, n)
        if n % b == 0 or (x != 1 and x != n - 1 and all((x := x * x % n) != n - 1 for _ in range(r - 1))):
            return n == b
    return True


def _below(bits, count, step):
    c, got = (1 << bits) + 1 - step, []
    while len(got) < count:
        if _is_prime(c):
            got.append(c)
        c -= step
    return got


_chains = {}


def _chain(log_n):
    """(primes q_0 .. q_L, scale of each level)"""
    if log_n not in _chains:
        levels, step = RINGS[log_n][0], 2 << log_n
        q = [0] * (levels + 1)
        q[0] = _below(Q0_BITS, 1, step)[0]
        pool, scale = _below(Q_BITS, 4 * levels + 4, step), [0.0] * levels + [2.0 ** Q_BITS]
        for l in range(levels, 0, -1):
            q[l] = min((p for p in pool if p not in q), key=lambda p: abs(float(p) - scale[l] * scale[l] / 2.0 ** Q_BITS))
            scale[l - 1] = scale[l] * scale[l] / float(q[l])
        _chains[log_n] = q, scale
    return _chains[log_n]


def _bitrev(bits):
    i, r = np.arange(1 << bits), np.zeros(1 << bits, np.int64)
    for k in range(bits):
        r |= ((i >> k) & 1) << (bits - 1 - k)
    return r


_tables = {}


def _roots(log_n, limb):
    """psi^bitrev(k), psi the root of the transform modulo prime `limb`"""
    if (log_n, limb) not in _tables:
        q, N = _chain(log_n)[0][limb], 1 << log_n
        psi = next(c for x in range(2, q) if pow(c := pow(x, (q - 1) // (2 * N), q), N, q) == q - 1)
        powers = [1]
        for _ in range(N - 1):
            powers.append(powers[-1] * psi % q)
        _tables[log_n, limb] = torch.from_numpy(np.array(powers, np.int64)[_bitrev(log_n)]).cuda()
    return _tables[log_n, limb]


def _angles(log_n):
    """The twiddles of the encoding transform, distance h and position j at [h + j]: exp(-2 pi i 5^j / 8h)"""
    if log_n not in _tables:
        S, M = 1 << (log_n - 1), 2 << log_n
        re, im, five = [0.0] * S, [0.0] * S, [1]
        for _ in range(S - 1):
            five.append(five[-1] * 5 % M)
        h = 1
        while h < S:
            for j in range(h):
                angle = 2.0 * math.pi * float((8 * h - five[j] % (8 * h)) * (M // (8 * h))) / float(M)
                re[h + j], im[h + j] = math.cos(angle), math.sin(angle)
            h *= 2
        _tables[log_n] = torch.tensor(re, dtype=torch.float64).cuda(), torch.tensor(im, dtype=torch.float64).cuda()
    return _tables[log_n]


def _turn(log_n, steps):
    """Where slot k of a plaintext rotated left by each of `steps` comes from, in transform order: [len(steps)][N]"""
    N, rev = 1 << log_n, _bitrev(log_n)
    odd = 2 * rev + 1
    return torch.from_numpy(np.stack([rev[(pow(5, s % (N // 2), 2 * N) * odd % (2 * N)) >> 1] for s in steps])).cuda()


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _blocks(c):
    """(K-groups of four row tiles, column tiles) of a weight matrix"""
    d = _tile(c["log_n"])
    return -(-c["rows"] // (4 * d)), -(-c["cols"] // d)


def _uniform(c, shape, gen):
    """Residues as ciphertexts have them: uniform below each prime"""
    n, N = c["level"] + 1, 1 << c["log_n"]
    t = torch.empty(*shape, n, N, dtype=torch.int64, device="cuda")
    for l in range(n):
        t[..., l, :].random_(0, _chain(c["log_n"])[0][l], generator=gen)
    return t


def _weights(c, gen):
    """A trained-looking matrix in 4 bits: two rows a byte, the even one in the low half; the largest value of a group is seven steps"""
    rows, cols, group = c["rows"], c["cols"], c["group"]
    w = torch.randn(rows, cols, generator=gen, device="cuda") * 0.02
    groups = -(-rows // group)
    padded = torch.zeros(groups * group, cols, device="cuda")
    padded[:rows] = w
    scales = (padded.view(groups, group, cols).abs().amax(1) / 7.0).contiguous()
    steps = torch.round(w / scales.repeat_interleave(group, 0)[:rows].clamp_min(1e-20)).clamp(-8, 7).to(torch.uint8) + 8
    code = torch.zeros(2 * -(-rows // 2), cols, dtype=torch.uint8, device="cuda")
    code[:rows] = steps & 15
    return code[0::2] | (code[1::2] << 4), scales


def _routes(c, seed):
    """Inputs in the order of their experts, and how many each expert has"""
    rng = random.Random(seed)
    at = [rng.sample(range(c["experts"]), c["top"]) for _ in range(c["inputs"])]
    order = [[i for i in range(c["inputs"]) if e in at[i]] for e in range(c["experts"])]
    return [i for e in order for i in e], [len(e) for e in order]


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "cross":
        s["a"] = _uniform(c, (c["groups"] * c["heads"] * c["queries"], 2), gen)
        s["b"] = _uniform(c, (c["groups"] * c["heads"] * c["keys"], 2), gen)
    elif c["op"] == "grouped":
        s["pre"] = _uniform(c, (_tile(c["log_n"]) * c["inputs"] * c["blocks"], 2), gen)
        s["pts"] = _uniform(c, (c["experts"] * c["tiles"] * c["blocks"],), gen)
        s["order"], s["sizes"] = _routes(c, seed)
    else:
        s["codes"], s["scales"] = _weights(c, gen)
        if c["op"] == "matvec":
            s["x"] = _uniform(c, (c["vectors"] * _blocks(c)[0], 2), gen)
    return s


# ---- what a program of the framework holds -----------------------------------------------------------------------------
_libs = {}


def _lib(log_n):
    if log_n not in _libs:
        pkg = importlib.import_module(PKG)
        levels, digits, weight = RINGS[log_n]
        _libs[log_n] = pkg.open_gpu(pkg.make_params(log_n=log_n, max_level=levels, dnum=digits, hamming_weight=weight))
    return _libs[log_n]


class _Residues:
    """The device memory of a handle, for torch; the handle lives as long as the tensor."""

    def __init__(self, handle):
        lib = handle.lib
        meta = lib.ct_meta(handle) if handle.kind == "ct" else lib.pt_meta(handle)
        shape = (meta[2], meta[1], meta[0] + 1, lib.N) if handle.kind == "ct" else (meta[0] + 1, lib.N)
        address = lib._fn(handle.kind + "_device_ptr")
        address.restype = ctypes.c_void_p
        self.handle = handle
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i8", "data": (address(handle.ptr), False), "version": 3, "strides": None}


def _tensor(handle):
    return torch.as_tensor(_Residues(handle), device="cuda")


def _ct(lib, residues):
    ct = lib.ct_create(residues.shape[2] - 1, 2, residues.shape[0])
    _tensor(ct).copy_(residues)
    return ct


def _pt(lib, residues):
    pt = lib.encode(np.zeros(1), residues.shape[0] - 1)
    _tensor(pt).copy_(residues)
    return pt


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        if case["op"] in ("encode", "matvec"):   # tables that depend on the context alone
            _angles(case["log_n"])
            [_roots(case["log_n"], l) for l in range(case["level"] + 1)]
        return s
    lib = s["lib"] = _lib(case["log_n"])
    if _libs.get("case") != case:   # other work than before: its buffer sizes are of no use to what follows
        lib._chk(lib._fn("release_cached")(lib.ctx))
        _libs["case"] = dict(case)
    if case["op"] in ("encode", "matvec"):
        codes, scales = s.pop("codes").cpu().numpy(), s.pop("scales").cpu().numpy()
        s["w"] = lib.qweight(codes, scales, case["rows"], case["group"])
    for name in ("a", "b", "pre", "x"):
        if name in s:
            s[name] = _ct(lib, s[name])
    if "pts" in s:
        rows = [_pt(lib, p) for p in s["pts"]]
        B, T = case["blocks"], case["tiles"]
        s["pts"] = [[rows[(e * T + t) * B:(e * T + t + 1) * B] for t in range(T)] for e in range(case["experts"])]
    torch.cuda.synchronize()   # the library's stream does not wait for torch's
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        return {"cross": _cross, "grouped": _grouped, "encode": _encode, "matvec": _matvec}[c["op"]](s)
    lib = s["lib"]
    if c["op"] == "cross":
        return _tensor(lib.tensor_acc_cross(s["a"], s["b"], c["groups"], heads=c["heads"]))
    if c["op"] == "grouped":
        return _tensor(lib.matmul_acc_grouped(s["pre"], c["inputs"], s["sizes"], s["pts"], 2 * _tile(c["log_n"]), order=s["order"]))
    if c["op"] == "encode":
        kb, nb = _blocks(c)
        return [_tensor(p) for p in lib.encode_q4(s["w"], _tile(c["log_n"]), 0, kb * nb, c["level"], diagonal=c["diagonal"])]
    return _tensor(lib.matvec_q4(s["x"], s["w"], _tile(c["log_n"])))


# ---- the plain forms: whole numbers, products in pieces of 20 bits -----------------------------------------------------
def _pieces(x):
    return [((x >> s) & 0xFFFFF) for s in (0, 20, 40)]


def _step(r, factor, more, q):
    """(r * factor + more) mod q for r, more's double and the result below 2^60, factor below 2^21: the wrapped sum is exact once its quotient is taken off.
    more = (exact value modulo 2^64, its double)"""
    quotient = ((r.double() * factor + more[1]) / q).long()
    return torch.remainder(r * factor + more[0] - quotient * q, q)


def _times(a, b, q):
    """a * b mod q"""
    r = torch.zeros((), dtype=torch.int64, device=a.device)
    for p in reversed(_pieces(b)):
        r = _step(r, 1 << 20, (a * p, a.double() * p.double()), q)
    return r


def _dots(eq, a, b, q):
    """A sum of products of residues: exact sums of the products of their pieces, put together modulo q"""
    a, b = [p.double() for p in _pieces(a)], [p.double() for p in _pieces(b)]
    r = None
    for weight in (4, 3, 2, 1, 0):
        s = None
        for i in range(max(0, weight - 2), min(2, weight) + 1):
            t = torch.einsum(eq, a[i], b[weight - i])
            s = t if s is None else s.add_(t)
        r = torch.remainder(s.long(), q) if r is None else _step(r, 1 << 20, (s.long(), s), q)
    return r


def _cross(s):
    c = s["case"]
    n, N, q = c["level"] + 1, 1 << c["log_n"], _chain(c["log_n"])[0]
    a = s["a"].view(c["groups"], c["heads"], c["queries"], 2, n, N)
    b = s["b"].view(c["groups"], c["heads"], c["keys"], 2, n, N)
    out = torch.empty(c["keys"], c["heads"], c["queries"], 3, n, N, dtype=torch.int64, device=a.device)
    for l in range(n):
        for h in range(c["heads"]):
            r = _dots("gipn,gjrn->jiprn", a[:, h, :, :, l], b[:, h, :, :, l], q[l])
            out[:, h, :, 0, l], out[:, h, :, 1, l], out[:, h, :, 2, l] = r[:, :, 0, 0], (r[:, :, 0, 1] + r[:, :, 1, 0]) % q[l], r[:, :, 1, 1]
    return out.view(-1, 3, n, N)


def _grouped(s):
    c = s["case"]
    n, N, d, q = c["level"] + 1, 1 << c["log_n"], _tile(c["log_n"]), _chain(c["log_n"])[0]
    pre = s["pre"].view(d, c["inputs"], c["blocks"], 2, n, N)
    pts = s["pts"].view(c["experts"], c["tiles"], c["blocks"], n, N)
    turn = _turn(c["log_n"], [k * 2 * d for k in range(d)])
    out, at = torch.empty(len(s["order"]), c["tiles"], 2, n, N, dtype=torch.int64, device=pre.device), 0
    for e, size in enumerate(s["sizes"]):
        if size:
            which = torch.tensor(s["order"][at:at + size], device=pre.device)
            for l in range(n):
                for p in range(2):
                    out[at:at + size, :, p, l] = _dots("kmbn,tbkn->mtn", pre[:, :, :, p, l][:, which], pts[e, :, :, l][:, :, turn], q[l])
        at += size
    return out.view(-1, 2, n, N)


def _plaintexts(s, diagonal):
    """The operands of all blocks, [column tile][K-group][limbs][N]"""
    c = s["case"]
    rows, cols, d, log_n = c["rows"], c["cols"], _tile(c["log_n"]), c["log_n"]
    (kb, nb), S, n = _blocks(c), 1 << (log_n - 1), c["level"] + 1
    q, scale = _chain(log_n)
    # the values: code - 8 steps of the group's scale, exact in 64 bits; four row tiles as 1/2 (W1 - i W3) | 1/2 (W2 - i W4), column j rolled up by j
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], 1).view(-1, cols)[:rows].double()
    w = torch.zeros(kb * 4 * d, nb * d, dtype=torch.float64, device=code.device)
    w[:rows, :cols] = (code - 8.0) * s["scales"].double().repeat_interleave(c["group"], 0)[:rows]
    w = 0.5 * w.view(kb, 4, d, nb, d).permute(3, 0, 1, 2, 4)
    if diagonal:
        i = torch.arange(d, device=code.device)
        w = w[:, :, :, (i[:, None] + i[None, :]) % d, i[None, :].expand(d, d)]
    re, im = (torch.zeros(nb * kb, S, dtype=torch.float64, device=code.device) for _ in range(2))
    re[:, : 2 * d * d] = torch.cat([w[:, :, 0], w[:, :, 1]], -1).reshape(nb * kb, -1)
    im[:, : 2 * d * d] = -torch.cat([w[:, :, 2], w[:, :, 3]], -1).reshape(nb * kb, -1)
    # slots -> coefficients: additions, subtractions and products rounded one by one, as the bits of a plaintext are defined
    wr, wi = _angles(log_n)
    h = S // 2
    while h:
        re, im = re.view(-1, S // (2 * h), 2, h), im.view(-1, S // (2 * h), 2, h)
        dr, di, tr, ti = re[:, :, 0] - re[:, :, 1], im[:, :, 0] - im[:, :, 1], wr[h:2 * h], wi[h:2 * h]
        re = torch.stack([re[:, :, 0] + re[:, :, 1], dr * tr - di * ti], 2)
        im = torch.stack([im[:, :, 0] + im[:, :, 1], dr * ti + di * tr], 2)
        h //= 2
    back = torch.from_numpy(_bitrev(log_n - 1)).to(code.device)
    coef = torch.cat([re.view(-1, S)[:, back], im.view(-1, S)[:, back]], 1)
    coef = torch.round(coef * (1.0 / S) * scale[c["level"]]).long()
    # residues, and the transform modulo every prime
    out = torch.empty(nb * kb, n, 2 * S, dtype=torch.int64, device=code.device)
    for l in range(n):
        v, roots, m = torch.remainder(coef, q[l]), _roots(log_n, l), 1
        while m < 2 * S:
            v = v.view(-1, m, 2, S // m)
            y = _times(v[:, :, 1], roots[m:2 * m, None], q[l])
            v, m = torch.stack([(v[:, :, 0] + y) % q[l], (v[:, :, 0] - y) % q[l]], 2), 2 * m
        out[:, l] = v.view(-1, 2 * S)
    return out


def _encode(s):
    return list(_plaintexts(s, s["case"]["diagonal"]))


def _matvec(s):
    c = s["case"]
    (kb, nb), n, N, q = _blocks(c), c["level"] + 1, 1 << c["log_n"], _chain(c["log_n"])[0]
    w = _plaintexts(s, False).view(nb, kb, n, N)
    x = s["x"].view(c["vectors"], kb, 2, n, N)
    out = torch.zeros(c["vectors"], nb, 2, n, N, dtype=torch.int64, device=x.device)
    for l in range(n):
        for b in range(kb):
            out[:, :, :, l] = (out[:, :, :, l] + _times(x[:, None, b, :, l], w[None, :, b, None, l], q[l])) % q[l]
    return out.view(-1, 2, n, N)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    """Each input once, each output once; two operations a product, ten a butterfly of the embedding, four one of a transform"""
    c = case
    n, N = c["level"] + 1, 1 << c["log_n"]
    if c["op"] in ("cross", "grouped"):
        held, products = _cost(c)
        return {"bytes": held, "flops": 2 * products}
    (kb, nb), v = _blocks(c), c.get("vectors", 0)
    read = c["rows"] * c["cols"] / 2 + 4 * -(-c["rows"] // c["group"]) * c["cols"]
    moved = v * 2 * (kb + nb) if v else kb * nb
    log_n = c["log_n"]
    transforms = kb * nb * (10 * (N // 4) * (log_n - 1) + 4 * n * (N // 2) * log_n)
    return {"bytes": read + moved * n * N * 8, "flops": transforms + 2 * 2 * v * kb * nb * n * N}


# ---- the right answers, in unbounded whole numbers ---------------------------------------------------------------------
def exact(case, seed):
    """Sums of products of Python's own integers, member by member, for the small cases.  Plaintexts of weights have no value beside the one that the
    rounded transform gives them (a coefficient next to a half goes either way), so what is made of weights has none here."""
    if case["op"] not in ("cross", "grouped") or _cost(case)[1] > 2e7:
        return None
    s, c, q = _inputs(case, seed), case, _chain(case["log_n"])[0]
    n, N = c["level"] + 1, 1 << c["log_n"]
    primes = np.array(q[:n], dtype=object)[:, None]
    host = lambda t: t.cpu().numpy().astype(object)  # noqa: E731
    if c["op"] == "cross":
        a, b = host(s["a"]).reshape(c["groups"], c["heads"], c["queries"], 2, n, N), host(s["b"]).reshape(c["groups"], c["heads"], c["keys"], 2, n, N)
        out = np.zeros((c["keys"], c["heads"], c["queries"], 3, n, N), np.int64)
        for j, h, i in np.ndindex(*out.shape[:3]):
            x, y = a[:, h, i], b[:, h, j]
            for k, terms in enumerate((((0, 0),), ((0, 1), (1, 0)), ((1, 1),))):
                out[j, h, i, k] = (sum((x[:, p] * y[:, r]).sum(0) for p, r in terms) % primes).astype(np.int64)
        return torch.from_numpy(out.reshape(-1, 3, n, N))
    d = _tile(c["log_n"])
    pre, pts = host(s["pre"]).reshape(d, c["inputs"], c["blocks"], 2, n, N), host(s["pts"]).reshape(c["experts"], c["tiles"], c["blocks"], n, N)
    # slot i in transform order is the polynomial's value at psi^(2 bitrev(i) + 1); a rotation takes it from the exponent 5^steps times that
    exponent = {2 * int(r) + 1: i for i, r in enumerate(_bitrev(c["log_n"]))}
    turned = [[exponent[e * pow(5, 2 * d * k, 2 * N) % (2 * N)] for e in exponent] for k in range(d)]
    expert = [e for e, size in enumerate(s["sizes"]) for _ in range(size)]
    out = np.zeros((len(expert), c["tiles"], 2, n, N), np.int64)
    for p, t, poly in np.ndindex(*out.shape[:3]):
        acc = 0
        for k in range(d):
            for b in range(c["blocks"]):
                acc = acc + pre[k, s["order"][p], b, poly] * pts[expert[p], t, b][:, turned[k]]
        out[p, t, poly] = (acc % primes).astype(np.int64)
    return torch.from_numpy(out.reshape(-1, 2, n, N))
