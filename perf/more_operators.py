"""Normalisation of encrypted activations and gradients, as cases that can be timed and compared.

  forward   layer norm of token tiles x[t][b] (t: column tiles, outermost; b: token tiles):
              squares[b] = sum_t (x[t][b] - mean[b]) (x) (x[t][b] - mean[b]) - pad * mean[b] (x) mean[b]   (pad columns of the last tile lie past the width)
              scaled[t][b] = (x[t][b] - mean[b]) (x) rstd[b]
              affine[t][b] = xhat[t][b] (.) gamma[t] + K beta[t],  K the scale of the level as a whole number
  backward  its gradients:
              rows[b] = sum_t g[t][b] (x) xhat[t][b],   rowsum[b] = sum_t g[t][b]
              gamma'[t] = sum_b dy[t][b] (x) xhat[t][b], beta'[t] = sum_b dy[t][b]
              input[t][b] = K (g[t][b] - mean[b]) - xhat[t][b] (x) dot[b]
  norm      the square of the global gradient norm: sum over all tensors and their members of x (x) x
  clip      every tensor times one factor: out_k[i] = x_k[i] (x) f

(x): tensor product of two ciphertexts, three polynomials; (.): product with a plaintext.  What stands between these steps (relinearisation, rescales,
rotations, the polynomial of the inverse root) is not part of a case: its inputs are given.  Everything is residues modulo the primes of a context, so outputs
are whole numbers and have one right value.  Ciphertexts are [members][polynomials][limbs][N], plaintexts [limbs][N], both in transform order.
"""
from __future__ import annotations

import ctypes
import importlib

import numpy as np
import torch

own = False

PKG = "encryption-friendly_llm_architecture_b200"
# the benchmark context and the small one of the documentation: (levels, digits of the gadget, Hamming weight of the secret)
RINGS = {16: (12, 4, 192), 12: (8, 3, 64)}
Q0_BITS, Q_BITS = 60, 42


def _columns(log_n):
    """Columns of a member: two tiles side by side, as many as fill the slots with their rows"""
    return 2 << ((log_n - 2) // 2)


def listed():
    return [
        # one token tile of 768 columns in a small ring: the latency of the calls
        {"name": "forward_small", "op": "forward", "log_n": 12, "level": 6, "tiles": 12, "batch": 1, "pad": 0},
        # four sequences of 128 tokens and 768 columns, at the level where their products live
        {"name": "forward_768", "op": "forward", "log_n": 16, "level": 5, "tiles": 3, "batch": 4, "pad": 0},
        # three sequences of 1001 columns: the last tile is not full
        {"name": "forward_odd", "op": "forward", "log_n": 16, "level": 3, "tiles": 4, "batch": 3, "pad": 23},
        # sixteen sequences of 2048 columns
        {"name": "forward_wide", "op": "forward", "log_n": 16, "level": 5, "tiles": 8, "batch": 16, "pad": 0},
        # the same activations on the way back
        {"name": "backward_small", "op": "backward", "log_n": 12, "level": 6, "tiles": 12, "batch": 1},
        {"name": "backward_768", "op": "backward", "log_n": 16, "level": 5, "tiles": 3, "batch": 4},
        {"name": "backward_wide", "op": "backward", "log_n": 16, "level": 5, "tiles": 8, "batch": 16},
        # the four factors of one LoRA layer in a small ring
        {"name": "norm_small", "op": "norm", "log_n": 12, "level": 6, "single": 4, "wide": 0, "members": 1},
        # the factors of twelve layers, and three full 768 x 768 weights of eighteen members
        {"name": "norm_model", "op": "norm", "log_n": 16, "level": 5, "single": 48, "wide": 3, "members": 18},
        {"name": "clip_small", "op": "clip", "log_n": 12, "level": 6, "single": 4, "wide": 0, "members": 1},
        # the factors of twelve layers with two levels left for the update
        {"name": "clip_lora", "op": "clip", "log_n": 16, "level": 3, "single": 48, "wide": 0, "members": 1},
        {"name": "clip_model", "op": "clip", "log_n": 16, "level": 5, "single": 48, "wide": 3, "members": 18},
    ]


def _members(c):
    """Members of the tensors: `single` ones of one, then `wide` ones of `members`"""
    return [1] * c["single"] + [c["members"]] * c["wide"]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _drawn(rng):
    op, log_n = rng.choice(["forward", "backward", "norm", "clip"]), rng.choice([12, 16, 16, 16])
    c = {"op": op, "log_n": log_n, "level": rng.randint(1, 8)}
    if op in ("norm", "clip"):
        return c | {"single": _log(rng, 1, 96), "wide": rng.choice([0, 1, 2, 5]), "members": rng.randint(2, 20)}
    c |= {"tiles": _log(rng, 1, 12), "batch": _log(rng, 1, 16)}
    return c | ({"pad": rng.choice([0, rng.randrange(_columns(log_n))])} if op == "forward" else {})


def _cost(c):
    """(polynomials read and written, products of residues) of a pass, in units of limbs x N"""
    if c["op"] in ("norm", "clip"):
        m = sum(_members(c))
        return (2 * m + 3, 3 * m) if c["op"] == "norm" else (5 * m + 2, 4 * m)
    T, B = c["tiles"], c["batch"]
    if c["op"] == "forward":   # squares; the product with one factor; the affine part
        return (2 * T * B + 2 * B + 3 * B) + (5 * T * B + 4 * B) + (4 * T * B + 2 * T), 3 * T * B + 4 * T * B + 2 * T * B + T
    return (6 * T * B + 5 * B + 5 * T) + (7 * T * B + 4 * B), 8 * T * B + 6 * T * B


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c)[0] * (c["level"] + 1) << c["log_n"])
    while True:
        c = _drawn(rng)
        if _cost(c)[0] * (c["level"] + 1) << c["log_n"] <= most[c["op"]]:
            return c


# ---- the arithmetic of a context: primes and scales (the rules of the library, restated) -----------------------------
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
    """(primes q_0 .. q_L, scale of each level as the nearest whole number)"""
    if log_n not in _chains:
        levels, step = RINGS[log_n][0], 2 << log_n
        q = [0] * (levels + 1)
        q[0] = _below(Q0_BITS, 1, step)[0]
        pool, scale = _below(Q_BITS, 4 * levels + 4, step), [0.0] * levels + [2.0 ** Q_BITS]
        for l in range(levels, 0, -1):
            q[l] = min((p for p in pool if p not in q), key=lambda p: abs(float(p) - scale[l] * scale[l] / 2.0 ** Q_BITS))
            scale[l - 1] = scale[l] * scale[l] / float(q[l])
        _chains[log_n] = q, [round(s) for s in scale]
    return _chains[log_n]


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _uniform(c, shape, gen):
    """Residues as ciphertexts have them: uniform below each prime"""
    n, N = c["level"] + 1, 1 << c["log_n"]
    t = torch.empty(*shape, n, N, dtype=torch.int64, device="cuda")
    for l in range(n):
        t[..., l, :].random_(0, _chain(c["log_n"])[0][l], generator=gen)
    return t


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] in ("norm", "clip"):
        s = {"xs": [_uniform(c, (m, 2), gen) for m in _members(c)]}
        return s | ({"factor": _uniform(c, (1, 2), gen)} if c["op"] == "clip" else {})
    T, B = c["tiles"], c["batch"]
    wide, narrow = ("x", "xhat"), ("mean", "rstd")
    if c["op"] == "backward":
        wide, narrow = ("dy", "g", "xhat"), ("mean", "dot")
    s = {k: _uniform(c, (T * B, 2), gen) for k in wide} | {k: _uniform(c, (B, 2), gen) for k in narrow}
    if c["op"] == "forward":
        s |= {"gamma": _uniform(c, (T,), gen), "beta": _uniform(c, (T,), gen)}
    return s


# ---- what a program of the framework holds ---------------------------------------------------------------------------
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
    if own:
        lib = _lib(case["log_n"])
        if _libs.get("case") != case:   # other work than before: its buffer sizes are of no use to what follows
            lib._chk(lib._fn("release_cached")(lib.ctx))
            _libs["case"] = dict(case)
        for name in list(s):
            t = s.pop(name)
            s[name] = [_ct(lib, x) for x in t] if name == "xs" else [_pt(lib, p) for p in t] if name in ("gamma", "beta") else _ct(lib, t)
        torch.cuda.synchronize()   # the library's stream does not wait for torch's
        s["lib"] = lib
    return s | {"case": case}


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        return {"forward": _forward, "backward": _backward, "norm": _norm, "clip": _clip}[c["op"]](s)
    lib = s["lib"]
    if c["op"] == "forward":
        T = c["tiles"]
        out = [lib.norm_squares(s["x"], T, mean=s["mean"], pad=c["pad"]), lib.norm_scale(s["x"], s["rstd"], T, mean=s["mean"]),
               lib.norm_affine(s["xhat"], T, gamma=s["gamma"], beta=s["beta"])]
    elif c["op"] == "backward":
        T = c["tiles"]
        out = [*lib.norm_grad_sums(s["dy"], s["xhat"], T, g=s["g"]), lib.norm_grad_input(s["g"], s["mean"], s["xhat"], s["dot"], T)]
    elif c["op"] == "norm":
        out = [lib.square_sum_many(s["xs"])]
    else:
        out = lib.scale_many(s["xs"], s["factor"])
    return [_tensor(h) for h in out]


# ---- the plain forms: whole numbers, products in pieces of 20 bits -----------------------------------------------------
def _step(r, factor, more, q):
    """(r * factor + more) mod q for r, more's double and the result below 2^60, factor below 2^21: the wrapped sum is exact once its quotient is taken off.
    more = (exact value modulo 2^64, its double)"""
    quotient = ((r.double() * factor + more[1]) / q).long()
    return torch.remainder(r * factor + more[0] - quotient * q, q)


def _dot(a, b, q, dim=None):
    """The sum over `dim` of products of residues (None: no sum): exact sums of the products of their pieces, put together modulo q"""
    a, b = ([((x >> s) & 0xFFFFF).double() for s in (0, 20, 40)] for x in (a, b))
    r = None
    for weight in (4, 3, 2, 1, 0):
        s = sum(a[i] * b[weight - i] if dim is None else (a[i] * b[weight - i]).sum(dim) for i in range(max(0, weight - 2), min(2, weight) + 1))
        r = torch.remainder(s.long(), q) if r is None else _step(r, 1 << 20, (s.long(), s), q)
    return r


def _tensored(a, b, q, dim=None):
    """Tensor product of polynomial pairs [..., 2, N] (a sum of them over `dim`): [..., 3, N]"""
    a0, a1, b0, b1 = a[..., 0, :], a[..., 1, :], b[..., 0, :], b[..., 1, :]
    return torch.stack([_dot(a0, b0, q, dim), (_dot(a0, b1, q, dim) + _dot(a1, b0, q, dim)) % q, _dot(a1, b1, q, dim)], -2)


def _limbs(c, shape, polynomials):
    return torch.empty(*shape, polynomials, c["level"] + 1, 1 << c["log_n"], dtype=torch.int64, device="cuda")


def _forward(s):
    c = s["case"]
    T, B = c["tiles"], c["batch"]
    q, scale = _chain(c["log_n"])
    squares, scaled, affine = _limbs(c, (B,), 3), _limbs(c, (T, B), 3), _limbs(c, (T, B), 2)
    for l in range(c["level"] + 1):
        x, xhat = (s[k][:, :, l].view(T, B, 2, -1) for k in ("x", "xhat"))
        mean, rstd, gamma, beta = s["mean"][:, :, l], s["rstd"][:, :, l], s["gamma"][:, None, l], s["beta"][:, None, l]
        centred = torch.remainder(x - mean, q[l])
        past = _dot(_tensored(mean, mean, q[l]), torch.tensor(c["pad"], device="cuda"), q[l])
        squares[:, :, l] = torch.remainder(_tensored(centred, centred, q[l], 0) - past, q[l])
        for t in range(T):
            scaled[t, :, :, l] = _tensored(centred[t], rstd, q[l])
            affine[t, :, :, l] = _dot(xhat[t], gamma[t], q[l])
            affine[t, :, 0, l] = (affine[t, :, 0, l] + _dot(beta[t], torch.tensor(scale[c["level"]] % q[l], device="cuda"), q[l])) % q[l]
    return [squares, scaled.flatten(0, 1), affine.flatten(0, 1)]


def _backward(s):
    c = s["case"]
    T, B = c["tiles"], c["batch"]
    q, scale = _chain(c["log_n"])
    rows, rowsum, cols, colsum, back = _limbs(c, (B,), 3), _limbs(c, (B,), 2), _limbs(c, (T,), 3), _limbs(c, (T,), 2), _limbs(c, (T, B), 3)
    for l in range(c["level"] + 1):
        dy, g, xhat = (s[k][:, :, l].view(T, B, 2, -1) for k in ("dy", "g", "xhat"))
        mean, dot = s["mean"][:, :, l], s["dot"][:, :, l]
        K = torch.tensor(scale[c["level"]] % q[l], device="cuda")
        rows[:, :, l], cols[:, :, l] = _tensored(g, xhat, q[l], 0), _tensored(dy, xhat, q[l], 1)
        one = torch.ones((), dtype=torch.int64, device="cuda")
        rowsum[:, :, l], colsum[:, :, l] = _dot(g, one, q[l], 0), _dot(dy, one, q[l], 1)
        for t in range(T):
            product = _tensored(xhat[t], dot, q[l])
            linear = torch.zeros_like(product)
            linear[:, :2] = _dot(torch.remainder(g[t] - mean, q[l]), K, q[l])
            back[t, :, :, l] = torch.remainder(linear - product, q[l])
    return [rows, rowsum, cols, colsum, back.flatten(0, 1)]


def _norm(s):
    c, q = s["case"], _chain(s["case"]["log_n"])[0]
    out = torch.zeros(1, 3, c["level"] + 1, 1 << c["log_n"], dtype=torch.int64, device="cuda")
    for l in range(c["level"] + 1):
        for x in s["xs"]:
            out[0, :, l] = (out[0, :, l] + _tensored(x[:, :, l], x[:, :, l], q[l], 0)) % q[l]
    return [out]


def _clip(s):
    c, q = s["case"], _chain(s["case"]["log_n"])[0]
    out = [_limbs(c, (m,), 3) for m in _members(c)]
    for l in range(c["level"] + 1):
        for o, x in zip(out, s["xs"]):
            o[:, :, l] = _tensored(x[:, :, l], s["factor"][:, :, l], q[l])
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    """Each input of each step once, each output once; two operations a product.  The inputs that two steps of a pass share (x, mean, g, xhat) count once."""
    c = case
    polynomials, products = _cost(c)
    if c["op"] == "forward":    # x and mean are squared and scaled
        polynomials -= 2 * c["tiles"] * c["batch"] + 2 * c["batch"]
    if c["op"] == "backward":   # g and xhat are summed and turned into the gradient of the input
        polynomials -= 4 * c["tiles"] * c["batch"]
    limb = (c["level"] + 1) << c["log_n"]
    return {"bytes": polynomials * limb * 8, "flops": 2 * products * limb}


# ---- the right answers, in unbounded whole numbers ---------------------------------------------------------------------
def exact(case, seed):
    """Sums of products of Python's own integers, member by member, for the small cases"""
    c = case
    if _cost(c)[1] * (c["level"] + 1) << c["log_n"] > 1.2e7:
        return None
    q, scale = _chain(c["log_n"])
    primes, K = np.array(q[: c["level"] + 1], dtype=object)[:, None], scale[c["level"]]
    s = {k: [x.cpu().numpy().astype(object) for x in v] if isinstance(v, list) else v.cpu().numpy().astype(object) for k, v in _inputs(c, seed).items()}

    def pair(x, y):
        return np.stack([x[0] * y[0], x[0] * y[1] + x[1] * y[0], x[1] * y[1]])

    def back(members):
        return torch.from_numpy(np.stack([m % primes for m in members]).astype(np.int64)).cuda()

    if c["op"] == "norm":
        return [back([sum(pair(m, m) for x in s["xs"] for m in x)])]
    if c["op"] == "clip":
        return [back([pair(m, s["factor"][0]) for m in x]) for x in s["xs"]]
    T, B = c["tiles"], c["batch"]
    at = [(t, b) for t in range(T) for b in range(B)]
    if c["op"] == "forward":
        x, mean, xhat = s["x"], s["mean"], s["xhat"]
        squares = [sum(pair(x[t * B + b] - mean[b], x[t * B + b] - mean[b]) for t in range(T)) - c["pad"] * pair(mean[b], mean[b]) for b in range(B)]
        scaled = [pair(x[t * B + b] - mean[b], s["rstd"][b]) for t, b in at]
        affine = [np.stack([xhat[t * B + b][0] * s["gamma"][t] + K * s["beta"][t], xhat[t * B + b][1] * s["gamma"][t]]) for t, b in at]
        return [back(squares), back(scaled), back(affine)]
    dy, g, xhat, nothing = s["dy"], s["g"], s["xhat"], 0 * s["g"][0][:1]
    rows, rowsum = [sum(pair(g[t * B + b], xhat[t * B + b]) for t in range(T)) for b in range(B)], [sum(g[t * B + b] for t in range(T)) for b in range(B)]
    cols, colsum = [sum(pair(dy[t * B + b], xhat[t * B + b]) for b in range(B)) for t in range(T)], [sum(dy[t * B + b] for b in range(B)) for t in range(T)]
    inner = [np.concatenate([K * (g[t * B + b] - s["mean"][b]), nothing]) - pair(xhat[t * B + b], s["dot"][b]) for t, b in at]
    return [back(rows), back(rowsum), back(cols), back(colsum), back(inner)]
