"""The rasterizer's blend and its derivatives in 64 bits, for the gradient
tests of steps whose opacities pass 1.

What the rasterizer decides -- a pair's alpha, whether it is blended, at the
cap of 0.999 or past the pixel's end -- is replayed in its 32-bit arithmetic
(products and fused operations rounded as the forward rounds them, the
exponential's published steps).  The sums and the derivatives are plain 64-bit
formulas of those alphas.

U is half a step of float32 relative to a value; a bound counts roundings.
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24
CHUNK = 512                       # list entries of a depth chunk
CAP = np.float32(0.999)
F = np.float32


def fma32(a, b, c):
    """a * b + c with one rounding (the product is exact in 64 bits; the sum's
    rounding there moves a tie of 24 bits once in 2^29)."""
    return (np.asarray(a, np.float64) * np.asarray(b, np.float64) + np.asarray(c, np.float64)).astype(F)


def exp32(x):
    """The forward's exp of x in [-80, 0]: Cody-Waite reduction, degree 6."""
    t = fma32(x, F(1.44269502162933349609375), F(12582912.0))
    k = t - F(12582912.0)
    r = fma32(-k, F(0.693145751953125), x)
    r = fma32(-k, F(1.428606765330187045e-06), r)
    p = np.full_like(r, F(0.0013814594130963087))
    for c in (0.0083687193691730499, 0.041668388992547989, 0.1666652113199234, 0.49999994039535522, 1.0, 1.0):
        p = fma32(p, r, F(c))
    return np.ldexp(p, k.astype(np.int32)).astype(F)


def tile_alphas(xy, conic, op, ids, px, py, chunked):
    """(alpha float32 [pairs, pixels], 0 where not blended; final T float32
    [pixels]) of a tile's list `ids`."""
    alpha = np.zeros((len(ids), px.size), F)
    total = np.ones(px.size, F)
    for beg in range(0, max(len(ids), 1), CHUNK if chunked else max(len(ids), 1)):
        T, done = np.ones(px.size, F), np.zeros(px.size, bool)
        for k in range(beg, min(beg + CHUNK, len(ids)) if chunked else len(ids)):
            g = ids[k]
            a, b, c = conic[g]
            dx, dy = xy[g, 0] - px, xy[g, 1] - py
            sigma = fma32(F(0.5), fma32(a, dx * dx, c * dy * dy), b * dx * dy)
            near = (sigma >= 0) & (sigma < F(5.55))
            al = np.minimum(CAP, op[g] * exp32(-np.where(near, sigma, F(1))))
            on = near & (al >= F(1.0) / F(255.0)) & ~done
            nT = T * (F(1) - al)
            done |= on & (nT <= F(1e-4))
            on &= ~done
            T = np.where(on, nT, T)
            alpha[k] = np.where(on, al, F(0))
        total = total * T
    return alpha, total


def tiles(w, h):
    for t in range(-(-h // 16) * -(-w // 16)):
        tx, ty = t % -(-w // 16) * 16, t // -(-w // 16) * 16
        y, x = np.mgrid[ty:min(ty + 16, h), tx:min(tx + 16, w)]
        yield t, x.ravel(), y.ravel()


def backward(xy, conic, op, rgb, offset, ids, w, h, bg, v, chunked):
    """Derivatives of sum(v * image) with respect to each Gaussian's colour
    (raw, clamped at 0 after adding 0.5), conic (the middle one halved, as a
    symmetric matrix's), centre and log opacity: [n, 9], and their bounds.
    Also final T (float32) and counts: pairs at the cap, pairs in front of one."""
    n = len(op)
    grad, mag, err, bins = np.zeros((n, 9)), np.zeros((n, 9)), np.zeros((n, 9)), np.zeros(n)
    final_T, capped, before = np.zeros((h, w), F), 0, 0
    bg = np.asarray(bg, np.float64)
    for t, px, py in tiles(w, h):
        lst = ids[offset[t]:offset[t + 1]]
        assert not chunked or len(lst) <= 2 * CHUNK    # past two, chunks may be cut off
        al32, fT = tile_alphas(xy, conic, op, lst, px.astype(F), py.astype(F), chunked)
        final_T[py, px] = fT
        np.add.at(bins, lst, 1)
        al = al32.astype(np.float64)
        on, cap = al > 0, al32 >= CAP
        capped += int(cap.sum())
        before += int((on & (np.cumsum(cap[::-1], 0)[::-1] - cap > 0)).sum())
        T = np.cumprod(np.concatenate((np.ones((1, px.size)), 1 - al)), 0)
        vo = v[py, px].astype(np.float64)                                       # [pixels, 3]
        col = np.maximum(rgb.astype(np.float64) + 0.5, 0)
        behind, behind_abs = T[-1] * (vo @ bg), T[-1] * (np.abs(vo) @ np.abs(bg))
        # roundings: T's products forward (2 a pair) and back (3 a pair), and the
        # sums of what is behind (1 a pair)
        E = (6 * on.sum(0) + 16) * U
        for k in range(len(lst) - 1, -1, -1):
            g, s = lst[k], on[k]
            if not s.any():
                continue
            a, b, c = conic[g].astype(np.float64)
            dx, dy = np.float64(xy[g, 0]) - px, np.float64(xy[g, 1]) - py
            wgt = al[k] * T[k]
            rv, rv_abs = vo @ col[g], np.abs(vo) @ col[g]
            v_alpha = np.where(s & ~cap[k], T[k] * rv - behind / (1 - al[k]), 0.0)
            va_abs = np.where(s & ~cap[k], T[k] * rv_abs + behind_abs / (1 - al[k]), 0.0)
            d = -al[k] * v_alpha
            d_abs = al[k] * va_abs
            seen = rgb[g] + F(0.5) >= 0
            terms = [wgt * vo[:, j] * seen[j] for j in range(3)]
            terms += [0.5 * d * dx * dx, 0.5 * d * dx * dy, 0.5 * d * dy * dy,
                      d * (a * dx + b * dy), d * (b * dx + c * dy), -d]
            size = [wgt * np.abs(vo[:, j]) * seen[j] for j in range(3)]
            size += [0.5 * d_abs * dx * dx, 0.5 * d_abs * np.abs(dx * dy), 0.5 * d_abs * dy * dy,
                     d_abs * (np.abs(a * dx) + np.abs(b * dy)), d_abs * (np.abs(b * dx) + np.abs(c * dy)), d_abs]
            for j in range(9):
                grad[g, j] += terms[j][s].sum()
                mag[g, j] += size[j][s].sum()
                err[g, j] += (3 * E * size[j])[s].sum()
            behind = behind + np.where(s, wgt * rv, 0.0)
            behind_abs = behind_abs + np.where(s, wgt * rv_abs, 0.0)
    # a warp's sum (two pixels, five halvings, the factor), and a sum of as many
    # warps in any order
    err += mag * (10 + 4 * bins[:, None]) * U
    return grad, err, final_T, capped, before


def blend(xy, conic, op, rgb, offset, ids, w, h, bg):
    """(image, blended pairs, pairs at the cap) of one pass, all in 64 bits:
    what the derivatives are compared with by differences."""
    img, which = np.zeros((h, w, 3)), []
    for t, px, py in tiles(w, h):
        T, col, done = np.ones(px.size), np.zeros((px.size, 3)), np.zeros(px.size, bool)
        for g in ids[offset[t]:offset[t + 1]]:
            dx, dy = xy[g, 0] - px, xy[g, 1] - py
            sigma = 0.5 * (conic[g, 0] * dx * dx + conic[g, 2] * dy * dy) + conic[g, 1] * dx * dy
            al = np.minimum(np.float64(CAP), op[g] * np.exp(-sigma))
            on = (sigma >= 0) & (sigma < 5.55) & (al >= 1 / 255) & ~done
            done |= on & (T * (1 - al) <= 1e-4)
            on &= ~done
            col += np.where(on, al * T, 0.0)[:, None] * np.maximum(rgb[g] + 0.5, 0)
            T = np.where(on, T * (1 - al), T)
            which.append((on, on & (al >= np.float64(CAP))))
        img[py, px] = col + T[:, None] * np.asarray(bg)
    return img, which
