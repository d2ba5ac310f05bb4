"""64-bit plain implementations of the dropout and 4-bit colour operators,
from their definitions, and the error bounds their tests use.

U is half a step of float32 relative to a value; a bound counts roundings.
"""
from __future__ import annotations

import math

import numpy as np

U = 2.0 ** -24
REST = (0, 3, 8, 15, 24)
BYTES = (8, 16, 24, 32, 48)
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


# ---- dropout

def philox(group, step: int, seed: int) -> np.ndarray:
    """Philox4x32-10 (Salmon et al., SC 2011): [len(group), 4] uint32."""
    u, m, s = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
    g = np.atleast_1d(np.asarray(group, np.uint64))
    c = [g & m, g >> s, np.full_like(g, step & 0xFFFFFFFF), np.full_like(g, step >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> s) ^ c[1] ^ u(k[0]), q & m, (p >> s) ^ c[3] ^ u(k[1]), p & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype(np.uint32)


def draws(index, step: int, seed: int) -> np.ndarray:
    i = np.asarray(index, np.uint64)
    return philox(i >> np.uint64(2), step, seed)[np.arange(i.size), (i & np.uint64(3)).astype(int)]


def keep(index, rate: float, step: int, seed: int):
    """(kept, 1 / the kept share) for the draws `index`."""
    t = int(np.rint(rate * 2.0 ** 32))
    return draws(index, step, seed).astype(np.int64) >= t, 2.0 ** 32 / (2 ** 32 - t)


# ---- records

def encode(dc: np.ndarray, rest: np.ndarray) -> np.ndarray:
    """Records (n, bytes) uint8 of float32 dc (n, 3) and rest (n, B, 3)."""
    n, b = rest.shape[:2]
    rec = np.zeros((n, BYTES[REST.index(b)]), np.uint8)
    with np.errstate(over="ignore"):
        rec[:, :6] = dc.astype(np.float16).view(np.uint8).reshape(n, 6)
    if b == 0:
        return rec
    amax = np.abs(rest.astype(np.float64)).max(1)
    bad = ~np.isfinite(rest).all(1)
    amax[bad] = 0
    # the power of two with amax / 2^e in [3.5, 7), from 2^-127 to 2^125
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.floor(np.log2(np.where(amax > 0, amax, 1))) - 2, -127).astype(int)
    e = np.where(amax >= np.ldexp(7.0, e), e + 1, e)
    e = np.where(amax < np.ldexp(3.5, e), e - 1, e)
    e = np.clip(e, -127, 125)           # above 125 the grid would pass the largest float: saturate
    y = np.ldexp(np.where(bad[:, None], 0.0, rest.astype(np.float64)), -e[:, None])
    dist = np.abs(np.abs(y)[..., None] - LEVELS)
    near = dist.min(-1, keepdims=True)
    tied = dist == near
    even = tied & (np.arange(8) % 2 == 0)
    code = np.where(tied.sum(-1) > 1, even.argmax(-1), tied.argmax(-1))
    code = code + 8 * (np.signbit(y) & ~bad[:, None])
    rec[:, 6:9] = np.where(bad, 255, e + 127)
    nib = np.zeros((n, (3 * b + 1) // 2 * 2), np.uint8)
    nib[:, :3 * b] = code.reshape(n, -1)
    rec[:, 9:9 + nib.shape[1] // 2] = nib[:, 0::2] | nib[:, 1::2] << 4
    return rec


def decode(rec: np.ndarray, degree: int):
    """(dc, rest) in float64."""
    n, b = rec.shape[0], REST[degree]
    dc = np.ascontiguousarray(rec[:, :6]).view(np.float16).astype(np.float64)
    if b == 0:
        return dc, np.zeros((n, 0, 3))
    body = rec[:, 9:9 + (3 * b + 1) // 2]
    nib = np.stack((body & 15, body >> 4), -1).reshape(n, -1)[:, :3 * b].reshape(n, b, 3)
    scale = rec[:, 6:9].astype(int)
    val = np.where(nib & 8, -1.0, 1.0) * LEVELS[nib & 7] * np.ldexp(1.0, scale - 127)[:, None]
    return dc, np.where((scale == 255)[:, None], np.nan, val)


# ---- colours

def _terms():
    """The basis as sums of constant * x^a y^b z^c."""
    s, pi = math.sqrt, math.pi

    def mul(p, q):
        return [(a[0] * b[0], a[1] + b[1], a[2] + b[2], a[3] + b[3]) for a in p for b in q]
    x, y, z = [(1, 1, 0, 0)], [(1, 0, 1, 0)], [(1, 0, 0, 1)]
    xx, yy, zz = mul(x, x), mul(y, y), mul(z, z)

    def k(c, p):
        return [(c * t[0],) + t[1:] for t in p]
    one = [(1, 0, 0, 0)]
    c1, c2, c3 = s(3 / (4 * pi)), s(15 / pi) / 2, s(35 / (2 * pi)) / 4
    d3, e3 = s(21 / (2 * pi)) / 4, s(105 / pi) / 2
    c4, d4, e4, f4 = s(35 / pi) * .75, s(35 / (2 * pi)) * .75, s(5 / pi) * .75, s(5 / (2 * pi)) * .75
    xmy = xx + k(-1, yy)
    three = [k(3, xx) + k(-1, yy), xx + k(-3, yy)]
    return [
        k(s(1 / (4 * pi)), one), k(-c1, y), k(c1, z), k(-c1, x),
        k(c2, mul(x, y)), k(-c2, mul(y, z)), k(s(5 / pi) / 4, k(2, zz) + k(-1, xx) + k(-1, yy)),
        k(-c2, mul(x, z)), k(c2 / 2, xmy),
        k(-c3, mul(y, three[0])), k(e3, mul(mul(x, y), z)),
        k(-d3, mul(y, k(4, zz) + k(-1, xx) + k(-1, yy))),
        k(s(7 / pi) / 4, mul(z, k(2, zz) + k(-3, xx) + k(-3, yy))),
        k(-d3, mul(x, k(4, zz) + k(-1, xx) + k(-1, yy))), k(e3 / 2, mul(z, xmy)),
        k(-c3, mul(x, three[1])),
        k(c4, mul(mul(x, y), xmy)), k(-d4, mul(mul(y, z), three[0])),
        k(e4, mul(mul(x, y), k(7, zz) + k(-1, one))), k(-f4, mul(mul(y, z), k(7, zz) + k(-3, one))),
        k(s(1 / pi) * 3 / 16, mul(zz, k(35, zz) + k(-30, one)) + k(3, one)),
        k(-f4, mul(mul(x, z), k(7, zz) + k(-3, one))), k(e4 / 2, mul(xmy, k(7, zz) + k(-1, one))),
        k(-d4, mul(mul(x, z), three[1])), k(c4 / 4, mul(xx, three[1]) + k(-1, mul(yy, three[0]))),
    ]


TERMS = _terms()


def basis(means: np.ndarray, cam, use: int):
    """(values, sums of the terms' magnitudes), each [n, (use+1)^2], of the
    directions from one camera."""
    d = means.astype(np.float64) - np.asarray(cam, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = d / np.sqrt((d * d).sum(1, keepdims=True))
    val, mag = [], []
    for poly in TERMS[:(use + 1) ** 2]:
        t = [c * d[:, 0] ** i * d[:, 1] ** j * d[:, 2] ** k if i + j + k else np.full(len(d), c)
             for c, i, j, k in poly]
        val.append(sum(t))
        mag.append(sum(np.abs(q) for q in t))
    return np.stack(val, 1), np.stack(mag, 1)


# Roundings of one term of a basis value: the difference from the camera (1),
# the norm's square (3 products and sums) and root (halved, rounded), its
# reciprocal (2 with a Newton step), and the product with the difference:
# 1 + (2 + 3) / 2 + 2 + 1 < 7 per factor of the direction, at most 4 factors;
# the constant's float and the products and sums of the polynomial, at most
# 10.
BASIS_ROUNDINGS = 4 * 7 + 10


def colors(dc, rest, means, cams, use: int):
    """(colours, bounds) [V, n, 3]: a fused multiply-add per coefficient rounds
    the sum at most 24 times, the dc term rounds once and joining it under
    the scale once."""
    coef = np.concatenate((dc[:, None], rest[:, :REST[use]]), 1)
    col, bound = [], []
    for cam in cams:
        b, m = basis(means, cam, use)
        col.append(np.einsum("nk,nkc->nc", b, coef))
        bound.append((BASIS_ROUNDINGS + 26) * U * np.einsum("nk,nkc->nc", m, np.abs(coef)))
    shape = (len(cams), len(means), 3)
    return np.reshape(col, shape), np.reshape(bound, shape)


def colors_backward(v_colors, degree: int, means, cams, use: int, radii=None):
    """(v_dc, v_rest, bound of v_dc, bound of v_rest): a product and a sum
    per view."""
    n = len(means)
    grad, bound = np.zeros((n, 1 + REST[degree], 3)), np.zeros((n, 1 + REST[degree], 3))
    for v, cam in enumerate(cams):
        seen = np.ones(n, bool) if radii is None else radii[v] > 0
        g = np.where(seen[:, None], v_colors[v].astype(np.float64), 0.0)
        b, m = basis(means, cam, use)
        grad[:, :b.shape[1]] += b[:, :, None] * g[:, None]
        bound[:, :b.shape[1]] += m[:, :, None] * np.abs(g)[:, None]
    bound *= (BASIS_ROUNDINGS + 2 + len(cams)) * U
    return grad[:, 0], grad[:, 1:], bound[:, 0], bound[:, 1:]


# ---- inputs

def features(n: int, degree: int, seed: int):
    rng = np.random.default_rng(seed)
    dc = rng.normal(0, 0.3, (n, 3)).astype(np.float32)
    rest = rng.normal(0, 0.05, (n, REST[degree], 3)) * np.exp(rng.normal(0, 1, (n, 1, 1)))
    rest[rng.random(n) < 0.1] = 0
    return dc, rest.astype(np.float32)


def awkward_features(degree: int):
    """Rows at which an encoder can go wrong: ties of the grid, the borders
    of a scale, signed zeros, subnormals, the largest floats, and channels
    that a NaN or an infinity spoils."""
    b = REST[degree]
    tops = [7.0, np.nextafter(np.float32(7), np.float32(0)), 3.5,
            np.nextafter(np.float32(3.5), np.float32(0)), 6.0, 4.0, 2.0 ** -126, 2.0 ** -149,
            7 * 2.0 ** -127, 3.4028234e38, 2.0 ** 127, 1.75 * 2.0 ** 127, 0.0]
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5,
                     -5.0, -0.0, 0.2, -0.2, 1e-30, -1e-30, 0.5, 1, 1.5, 2, 3], np.float64)
    rows = []
    for t in tops:
        row = np.resize(ties, (b, 3)) * (float(t) / 6 if 0 < t < 1e30 else 1)
        row[0] = [t, -t, t]
        rows.append(row)
    rest = np.clip(np.array(rows), -3.4028234e38, 3.4028234e38).astype(np.float32)
    spoiled = np.repeat(rest[:1], 4, 0)
    spoiled[0, 0, 0] = np.nan
    spoiled[1, -1, 1] = np.inf
    spoiled[2, 0, 2] = -np.inf
    spoiled[3, :] = np.nan
    rest = np.concatenate((rest, spoiled))
    dc = np.resize(np.array([0, -0.0, 65504, 65520, -1e9, np.nan, np.inf, 6e-8, 3e-8, 1 + 2 ** -11, 0.3],
                            np.float32), (len(rest), 3))
    return dc, rest
