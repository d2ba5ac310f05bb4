"""Gradients of a training step with dropout whose raised opacities pass 1, so
that the cores of opaque Gaussians are blended at the cap of 0.999: against the
64-bit derivatives of the blend (tests/raster_case.py), in the single-pass and
the depth-chunked raster, with Gaussians before and behind the capped ones."""
from __future__ import annotations

import math

import numpy as np
import pytest

from msplat_b200 import _lib, engine, multigpu, synthetic
from tests import harness
from tests import operators_case as oc
from tests import raster_case as rc

pytestmark = pytest.mark.gpu

SEED, STEP = 0x5EED, 41


@pytest.fixture(autouse=True)
def gpu():
    import torch
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    engine.bind_stream()
    engine.set_step_options()
    yield
    engine.set_step_options()
    _lib.load().cleanup_msplat_cuda()


def run_step(g, cs, gt, rate, mx4=False):
    """One step's gradients (by group) and what its rasterizer had and gave."""
    import torch
    engine.set_step_options(dropout_rate=rate, dropout_seed=SEED, dropout_step=STEP, mx4_colors=mx4)
    model = engine.GaussianModel(g.groups())
    buf = torch.zeros(multigpu.grad_floats(model.n, model.rest_bases), dtype=torch.float32, device="cuda")
    multigpu.EngineOps().grads(model, cs, gt, buf, 0.2, engine.DEFAULT_BG, 1.0, 0.01)
    torch.cuda.synchronize()
    views, vis = multigpu.grad_views(buf, model.n, model.rest_bases)
    e = harness.engine_forward_dump(g.n, cs)
    off, ids, _ = harness.tile_ids_engine(cs, 0)
    return dict(e, acc=engine.debug_buffer("grad_acc", 9 * g.n, np.float32).reshape(g.n, 9).astype(np.float64),
                v=engine.debug_buffer("v_rendered", 3 * cs.width * cs.height, np.float32)
                .reshape(cs.height, cs.width, 3), off=off, ids=ids, vis=vis.cpu().numpy() > 0,
                groups=[t.cpu().numpy() for t in views])


def scene(n, w, h, spread, log_mu, logits, seed):
    g = synthetic.gaussians(n, seed, mean_range=spread, log_scale_mu=math.log(log_mu))
    g.opacities = np.random.default_rng(seed).uniform(*logits, (n, 1)).astype(np.float32)
    return g, harness.setup_cam(synthetic.front_camera(w, h, 3.0))


@pytest.mark.parametrize("rate", [0.2, 0.5])
@pytest.mark.parametrize("n, w, h, spread, log_mu, chunked", [
    (150, 320, 320, 0.7, 0.06, False),         # 400 tiles: single pass
    (151, 1000, 117, 0.4, 0.03, False),        # ragged edges
    (60, 75, 50, 0.7, 0.08, True),             # one depth chunk
    (1500, 32, 16, 0.5, 0.015, True),          # two
])
def test_gradients_at_the_cap(n, w, h, spread, log_mu, chunked, rate):
    import torch
    g, cs = scene(n, w, h, spread, log_mu, (-2.0, 4.6), seed=n)              # sigmoid up to 0.99
    gt = torch.as_tensor(synthetic.target_image(w, h, 1)).cuda()
    r = run_step(g, cs, gt, rate)
    kept, scale = oc.keep(np.arange(n), rate, STEP, SEED)
    np.testing.assert_array_equal(r["vis"] & ~kept, False)
    if n == 1500:
        assert np.diff(r["off"]).max() > rc.CHUNK
    want, bound, final_T, capped, before = rc.backward(
        r["xy"].reshape(n, 2), r["conic"], r["opac"], r["rgb"], r["off"], r["ids"], w, h, engine.DEFAULT_BG,
        r["v"], chunked)
    # the replay is the forward's, and the case is what it is meant to be
    np.testing.assert_array_equal(final_T.ravel(), r["final_T"])
    assert capped >= 20 and before >= 100
    # d log o / d logit = 1 - sigmoid; a few roundings of a sigmoid near 1
    s = 1 / (1 + np.exp(-g.opacities[:, 0].astype(np.float64)))
    bound[:, 8] = bound[:, 8] * (1 - s) + 8 * rc.U * np.abs(want[:, 8])
    want[:, 8] *= 1 - s
    vis = r["vis"]
    assert not any(p[~vis].any() for p in r["groups"])       # the accumulators of these are not written
    off_by = np.abs(r["acc"] - want) / np.maximum(bound, 1e-300)
    for j, name in enumerate(("red", "green", "blue", "a", "b", "c", "x", "y", "logit")):
        bad = vis & (off_by[:, j] > 1)
        assert not bad.any(), (name, int(bad.sum()), float(np.abs(r["acc"] - want)[:, j].max()),
                               float(np.abs(want[:, j]).max()))
    # a colour's gradient reaches dc through the basis' constant
    dc = want[:, :3] * 0.28209479177387814
    assert (np.abs(r["groups"][3][vis] - dc[vis]) <= bound[vis, :3] + 4 * rc.U * np.abs(dc[vis])).all()


@pytest.mark.parametrize("rate", [0.05, 0.15, 0.2, 0.5])
def test_a_saturated_sigmoid_has_no_gradient_of_the_wrong_sign(rate):
    """Logits whose sigmoid rounds to 1: the derivative's factor 1 - s is at most
    a few roundings of 1, and not negative."""
    import torch
    g, cs = scene(150, 320, 320, 0.7, 0.06, (17.5, 30.0), seed=150)
    gt = torch.as_tensor(synthetic.target_image(320, 320, 1)).cuda()
    r = run_step(g, cs, gt, rate)
    want, bound, _, _, _ = rc.backward(
        r["xy"].reshape(150, 2), r["conic"], r["opac"], r["rgb"], r["off"], r["ids"], 320, 320,
        engine.DEFAULT_BG, r["v"], False)
    sure = r["vis"] & (np.abs(want[:, 8]) > bound[:, 8])
    assert sure.sum() >= 20
    ratio = r["acc"][sure, 8] / want[sure, 8]
    assert (ratio >= 0).all() and (ratio <= 4 * rc.U).all()


def test_the_plain_step_skips_what_is_at_the_cap():
    """Without dropout a pair at the cap gives no gradient and does not count
    among what is behind (the reference's step): unlike the derivatives."""
    import torch
    g, cs = scene(150, 320, 320, 0.7, 0.06, (6.0, 9.0), seed=150)     # sigmoid beyond 0.999 for the most part
    gt = torch.as_tensor(synthetic.target_image(320, 320, 1)).cuda()
    r = run_step(g, cs, gt, 0.0)
    want, bound, final_T, capped, _ = rc.backward(
        r["xy"].reshape(150, 2), r["conic"], r["opac"], r["rgb"], r["off"], r["ids"], 320, 320,
        engine.DEFAULT_BG, r["v"], False)
    np.testing.assert_array_equal(final_T.ravel(), r["final_T"])
    assert capped >= 10
    assert (np.abs(r["acc"] - want)[:, :3] > bound[:, :3]).any()
    run = harness.oracle.Run(cs, 150, isect_capacity=64 * 150, adam_steps=[0.0] * 6, adam_bc2=[1.0] * 6)
    params = [x.copy() for x in g.groups()]
    m, v = ([np.zeros_like(x) for x in params] for _ in range(2))
    run.train_step(params, m, v, gt.cpu().numpy(), *[np.zeros(150, np.float32) for _ in range(3)])
    vis = run.radii > 0
    for cols, ref in ((r["acc"][:, :3], run.v_rgb.reshape(-1, 3)), (r["acc"][:, 8:], run.v_opacity.reshape(-1, 1))):
        bad, worst = harness.close(cols[vis], ref[vis], harness.GRAD_RTOL, harness.GRAD_ATOL_FRAC)
        assert bad == 0, worst
