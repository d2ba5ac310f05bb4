"""The 64-bit rasterizer of the gradient tests, on the CPU: its replay of the
forward against the oracle's, its derivatives against differences."""
from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import oracle
from tests import raster_case as rc


def splats(n, w, h, seed, top):
    """Float32 centres, conics, opacities up to `top` and colours of n Gaussians
    on a w x h image, every tile listing all of them."""
    rng = np.random.default_rng(seed)
    f = np.float32
    xy = rng.uniform((0, 0), (w, h), (n, 2)).astype(f)
    m = rng.normal(size=(n, 2, 2)) * 0.25
    m = m @ m.transpose(0, 2, 1) + 0.02 * np.eye(2)
    conic = np.stack((m[:, 0, 0], m[:, 0, 1], m[:, 1, 1]), 1).astype(f)
    tiles = -(-w // 16) * -(-h // 16)
    return (xy, conic, rng.uniform(0.05, top, n).astype(f), rng.normal(0, 0.4, (n, 3)).astype(f),
            np.arange(tiles + 1) * n, np.tile(np.arange(n), tiles))


def test_exp_is_the_forwards():
    x = -np.random.default_rng(0).uniform(0, 6, 4000).astype(np.float32)
    np.testing.assert_array_equal(rc.exp32(x), np.array([oracle.expf(float(v)) for v in x], np.float32))


@pytest.mark.parametrize("top", [0.95, 2.0])
def test_derivatives_against_differences(top):
    """Each derivative against a central difference of the blend, over the
    pixels at which the difference crosses no border."""
    n, w, h, bg = 14, 36, 21, (0.6, 0.1, 0.4)
    xy, conic, op, rgb, offset, ids = splats(n, w, h, 5, top)
    v = np.random.default_rng(6).normal(size=(h, w, 3)).astype(np.float32)
    base = [xy.astype(np.float64), conic.astype(np.float64), op.astype(np.float64), rgb.astype(np.float64)]
    args = offset, ids, w, h, bg
    pixels = list(rc.tiles(w, h))
    seen_cap = 0

    def crossed(a, b):
        bad = np.zeros((h, w), bool)
        for t, px, py in pixels:
            for k in range(n):
                for p, q in zip(a[t * n + k], b[t * n + k]):
                    bad[py, px] |= p != q
        return bad
    for what, g, j, col, factor in (
            [(3, g, c, c, 1.0) for g in range(n) for c in range(3)]
            + [(1, g, 0, 3, 1.0) for g in range(n)] + [(1, g, 1, 4, 0.5) for g in range(n)]
            + [(1, g, 2, 5, 1.0) for g in range(n)] + [(0, g, 0, 6, 1.0) for g in range(n)]
            + [(0, g, 1, 7, 1.0) for g in range(n)] + [(2, g, None, 8, None) for g in range(n)]):
        step, at = 1e-5, (g,) if j is None else (g, j)
        img = []
        for sign in (1, -1):
            p = [a.copy() for a in base]
            p[what][at] += sign * step
            img.append(rc.blend(*p, *args))
        bad = crossed(img[0][1], img[1][1])
        vm = np.where(bad[..., None], 0, v)
        grad, err, _, capped, _ = rc.backward(xy, conic, op, rgb, *args, vm, False)
        seen_cap = max(seen_cap, capped)
        want = (vm * (img[0][0] - img[1][0])).sum() / (2 * step)
        if factor is None:
            factor = base[2][g]                     # d / d log opacity
        # the replay's alphas are rounded (a few U, times 1 / (1 - alpha) up to
        # 1000 in the colour behind), the difference's own error is step^2
        size = np.abs(vm).sum() * (1 + np.abs(base[3]).max())
        assert abs(grad[g, col] - factor * want) <= 1e-6 * size + err[g, col], (what, g, j)
    assert (seen_cap > 50) == (top > 1)


@pytest.mark.parametrize("chunked", [False, True])
def test_two_gaussians_by_hand(chunked):
    """Alpha 0.5 (colour 0.8) before opacity 1.1 (colour 0.3) at one pixel: the
    weights are 0.5, 0.4995 and 0.0005, and the front's alpha moves 0.8 - 0.2997."""
    xy, conic = np.zeros((2, 2), np.float32), np.tile(np.float32([1e-8, 0, 1e-8]), (2, 1))
    op, rgb = np.float32([0.5, 1.1]), np.float32([[0.3] * 3, [-0.2] * 3])
    v = np.zeros((1, 1, 3), np.float32)
    v[0, 0, 0] = 1
    grad, _, final_T, capped, before = rc.backward(xy, conic, op, rgb, np.array([0, 2]), np.array([0, 1]), 1, 1,
                                                   (0, 0, 0), v, chunked)
    assert (capped, before) == (1, 1) and math.isclose(final_T[0, 0], 0.0005, rel_tol=1e-4)
    np.testing.assert_allclose(grad[:, 0], (0.5, 0.4995), rtol=1e-6)
    np.testing.assert_allclose(grad[:, 8], (0.5 * (0.8 - 0.3 * 0.999), 0), rtol=1e-5)
