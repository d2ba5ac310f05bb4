"""Dropout of Gaussians and 4-bit colours in the engine's own paths: the
packed renderer, the training step and the trainer.

Forward results are compared bit for bit: with a step (or a render) of the
same scene in which what the option does was done beforehand -- the dropped
Gaussians taken out and the others' opacity raised, or the features replaced
by what their records stand for.  Gradients are held to the parity tests'
bars (harness.GRAD_RTOL, GRAD_ATOL_FRAC: float atomics in another order), and
the opacity gradient to differences of a 64-bit rasterizer.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from msplat_b200 import _lib, engine, multigpu, operators, synthetic
from tests import dataset_case, harness
from tests import operators_case as oc

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def gpu():
    import torch
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    engine.bind_stream()
    engine.set_step_options()
    yield
    engine.set_step_options()
    _lib.load().cleanup_msplat_cuda()


def scene(n, w, h, seed=0, degree=3, use=None, mean_range=1.0, log_mu=math.log(0.02), clusters=0):
    g = synthetic.gaussians(n, seed, mean_range=mean_range, log_scale_mu=log_mu, sh_degree=degree,
                            clusters=clusters)
    cs = harness.setup_cam(synthetic.front_camera(w, h, 3.0), sh_degree=degree,
                           rest_bases=g.features_rest.shape[1])
    if use is not None:
        cs.degrees_to_use = use
    return g, cs


def dump(cs, n):
    p = cs.width * cs.height
    out = {k: engine.debug_buffer(k, c, t) for k, c, t in (
        ("out_img", 3 * p, np.float32), ("final_T", p, np.float32), ("radii", n, np.int32))}
    rgb = engine.debug_buffer("rgb", 4 * n, np.float32).reshape(n, 4)[:, :3]
    op = engine.debug_buffer("conic_op", 4 * n, np.float32).reshape(n, 4)[:, 3]
    vis = out["radii"] > 0
    return dict(out, vis=vis, rgb=rgb[vis], op=op[vis])


def unpacked(g):
    """The scene with the features that its records stand for."""
    import torch
    rec = operators.mx4_pack(torch.as_tensor(g.features_dc).cuda(), torch.as_tensor(g.features_rest).cuda())
    degree = oc.REST.index(g.features_rest.shape[1])
    u = g.copy()
    u.features_dc, u.features_rest = (t.cpu().numpy() for t in operators.mx4_unpack(rec, degree))
    return u


def grads(g, cs, gt, accumulate=None):
    """(gradients by group, visibility) of one step from a fresh model."""
    import torch
    model = engine.GaussianModel(g.groups())
    n = multigpu.grad_floats(model.n, model.rest_bases)
    buf = torch.zeros(n, dtype=torch.float32, device="cuda") if accumulate is None else accumulate
    multigpu.EngineOps().grads(model, cs, gt, buf, 0.2, engine.DEFAULT_BG, 1.0, 0.01,
                               accumulate=accumulate is not None)
    torch.cuda.synchronize()
    views, vis = multigpu.grad_views(buf, model.n, model.rest_bases)
    return [v.cpu().numpy() for v in views], vis.cpu().numpy()


def assert_grads(got, want, label):
    bad, worst = harness.close(got, want, harness.GRAD_RTOL, harness.GRAD_ATOL_FRAC)
    assert bad == 0, f"{label}: {bad} entries out of tolerance (worst {worst:.3g} of max)"


# ---- the packed renderer

@pytest.mark.parametrize("n, w, h, degree, use, kw", [
    (20_000, 200, 160, 3, 3, {}),                                  # depth-chunked raster
    (30_001, 640, 480, 3, 2, {}),                                  # single pass, ragged count
    (10_000, 641, 479, 0, 0, {}), (10_000, 641, 479, 1, 1, {}), (10_000, 641, 479, 2, 2, {}),
    (10_000, 641, 479, 4, 4, {}),
    (60_000, 640, 480, 3, 3, dict(clusters=2, log_mu=math.log(0.03))),   # long lists
    (1, 64, 48, 3, 3, dict(mean_range=0.01)),
])
def test_render_mx4_is_the_render_of_the_unpacked_scene(n, w, h, degree, use, kw):
    g, cs = scene(n, w, h, seed=n % 97, degree=degree, use=use, **kw)
    packed = engine.PackedGaussians.of(engine.GaussianModel(g.groups()))
    plain = engine.GaussianModel(unpacked(g).groups())
    assert packed.nbytes == n * (44 + oc.BYTES[degree])
    for _ in range(2):                       # the second call sees the first one's counters
        engine.render(plain, cs)
        want = dump(cs, n)
        engine.render_mx4(packed, cs)
        got = dump(cs, n)
        for k in want:
            np.testing.assert_array_equal(got[k], want[k], err_msg=k)
    assert want["vis"].any()
    # the colours of the same view as an operator: both within their bound of
    # the exact ones (the renderer's unfused sums round twice as often)
    vis = want["vis"]
    col = packed.colors(np.array([cs.cam_pos]), degrees_to_use=use)[0].cpu().numpy()
    exact, bound = oc.colors(*oc.decode(packed.records.cpu().numpy(), degree), g.means, [cs.cam_pos], use)
    assert (np.abs(col - exact[0]) <= bound[0]).all()
    assert (np.abs(want["rgb"] - exact[0][vis]) <= 2 * bound[0][vis]).all()
    fdc, frest = packed.features()
    np.testing.assert_array_equal(fdc.cpu().numpy(), plain.params[3].cpu().numpy())
    np.testing.assert_array_equal(frest.cpu().numpy(), plain.params[4].cpu().numpy())


def test_render_mx4_leaves_other_renders_alone():
    """Alternating packed and plain renders, unaligned parameters among them."""
    import torch
    g, cs = scene(5_000, 320, 240, seed=5)
    model = engine.GaussianModel(g.groups())
    packed = engine.PackedGaussians.of(model)
    engine.render(model, cs)
    want = dump(cs, g.n)
    engine.render_mx4(packed, cs)
    want4 = dump(cs, g.n)
    assert not np.array_equal(want["out_img"], want4["out_img"])
    room = torch.empty(3 * g.n + 1, device="cuda")
    room[1:] = packed.means.reshape(-1)
    packed.means = room[1:].view(g.n, 3)
    for _ in range(2):
        engine.render(model, cs)
        np.testing.assert_array_equal(dump(cs, g.n)["out_img"], want["out_img"])
        engine.render_mx4(packed, cs)
        np.testing.assert_array_equal(dump(cs, g.n)["out_img"], want4["out_img"])


# ---- training with 4-bit colours

@pytest.mark.parametrize("n, w, h, degree, use", [(8_000, 200, 160, 3, 3), (8_001, 480, 330, 3, 1),
                                                  (5_000, 480, 330, 2, 2), (5_000, 480, 330, 0, 0),
                                                  (5_003, 480, 330, 1, 1), (3_000, 480, 330, 4, 4)])
def test_step_with_mx4_colors(n, w, h, degree, use):
    import torch
    g, cs = scene(n, w, h, seed=7, degree=degree, use=use)
    gt = torch.as_tensor(synthetic.target_image(w, h, 1)).cuda()
    want, wvis = grads(unpacked(g), cs, gt)
    a = dump(cs, n)
    v = engine.debug_buffer("v_rendered", 3 * w * h, np.float32)
    engine.set_step_options(mx4_colors=True)
    got, gvis = grads(g, cs, gt)
    b = dump(cs, n)
    for k in a:
        np.testing.assert_array_equal(b[k], a[k], err_msg=k)
    np.testing.assert_array_equal(engine.debug_buffer("v_rendered", 3 * w * h, np.float32), v)
    np.testing.assert_array_equal(gvis, wvis)
    for p, q, name in zip(got, want, ("means", "scales", "quats", "dc", "rest", "opacities")):
        if q.size:
            assert_grads(p, q, name)


def test_mx4_training_moves_the_float_features():
    """The features themselves stay floats, and the packed scene is what the
    next step's forward showed."""
    import torch
    g, cs = scene(4_000, 320, 240, seed=9)
    gt = torch.as_tensor(synthetic.target_image(cs.width, cs.height, 1)).cuda()
    model = engine.GaussianModel(g.groups())
    engine.set_step_options(mx4_colors=True)
    for _ in range(3):
        before = engine.PackedGaussians.of(model)
        engine.train_step(model, cs, gt)
        shown = dump(cs, g.n)["out_img"]
        engine.render_mx4(before, cs)
        np.testing.assert_array_equal(dump(cs, g.n)["out_img"], shown)
    moved = model.params[4].cpu().numpy()
    assert (moved != g.features_rest).mean() > 0.5
    rec = operators.mx4_pack(model.params[3], model.params[4])
    assert not np.array_equal(operators.mx4_unpack(rec, 3)[1].cpu().numpy(), moved)


# ---- dropout

def exact_pairs(want):
    """Logit pairs (l, L) with 2 sigmoid(l) = sigmoid(L) in the engine's
    float32, so that a rate of 1/2 (factor 2, exact) on l is a plain step on L."""
    n = 200_000
    g, cs = scene(n, 320, 240, seed=2, mean_range=0.4)
    table = []
    for lo, hi in ((-1.8, -0.3), (-0.4, 2.2)):
        g.opacities = np.linspace(lo, hi, n, dtype=np.float32)[:, None]
        engine.render(engine.GaussianModel(g.groups()), cs)
        d = dump(cs, n)
        table.append((d["op"], g.opacities[d["vis"], 0]))
    (s, l), (t, big) = table
    _, i, j = np.intersect1d(2 * s, t, return_indices=True)
    assert i.size >= 200
    k = np.random.default_rng(0).integers(0, i.size, want)
    return l[i[k]], big[j[k]]


@pytest.mark.parametrize("n, w, h", [(6_000, 200, 160), (6_001, 480, 330)])
def test_step_with_dropout(n, w, h):
    """Rate 1/2: the step is that of the kept Gaussians alone at twice the
    opacity; what was dropped is culled."""
    import torch
    seed, step = 0xABCDEF0123456789, 77
    g, cs = scene(n, w, h, seed=3)
    low, high = exact_pairs(n)
    g.opacities = low[:, None].copy()
    kept, scale = oc.keep(np.arange(n), 0.5, step, seed)
    assert scale == 2.0
    sub = synthetic.Gaussians(*[a[kept].copy() for a in g.groups()])
    sub.opacities = high[kept][:, None].copy()
    gt = torch.as_tensor(synthetic.target_image(w, h, 1)).cuda()
    want, wvis = grads(sub, cs, gt)
    a = dump(cs, sub.n)
    v = engine.debug_buffer("v_rendered", 3 * w * h, np.float32)
    engine.set_step_options(dropout_rate=0.5, dropout_seed=seed, dropout_step=step)
    got, gvis = grads(g, cs, gt)
    b = dump(cs, n)
    np.testing.assert_array_equal(b["radii"][kept], a["radii"])
    assert (b["radii"][~kept] == 0).all() and (gvis[~kept] == 0).all()
    np.testing.assert_array_equal(gvis[kept], wvis)
    for k in ("out_img", "final_T", "rgb", "op"):
        np.testing.assert_array_equal(b[k], a[k], err_msg=k)
    np.testing.assert_array_equal(engine.debug_buffer("v_rendered", 3 * w * h, np.float32), v)
    for p, q, name in zip(got[:5], want[:5], ("means", "scales", "quats", "dc", "rest")):
        assert_grads(p[kept], q, name)
        assert not p[~kept].any()
    # with o = 2 s: d o / d l = o (1 - s), where the plain step has o (1 - o)
    s = 1 / (1 + np.exp(-low[kept].astype(np.float64)))
    assert_grads(got[5][kept, 0], want[5][:, 0] * (1 - s) / (1 - 2 * s), "opacities")
    assert not got[5][~kept].any()


def test_dropout_mask_is_the_operators():
    """The step's mask is msplat_dropout's of whole rows, new at each step;
    a rate of 0 is the plain step."""
    import torch
    g, cs = scene(5_003, 320, 240, seed=4)
    gt = torch.as_tensor(synthetic.target_image(cs.width, cs.height, 1)).cuda()
    model = engine.GaussianModel(g.groups())
    engine.render(model, cs)
    plain = dump(cs, g.n)
    seen = []
    for step in (1, 2, 2**33):
        engine.set_step_options(dropout_rate=0.3, dropout_seed=9, dropout_step=step)
        grads(g, cs, gt)
        d = dump(cs, g.n)
        ones = torch.ones(g.n, 1, device="cuda")
        kept = operators.dropout(ones, 0.3, 9, step, whole_rows=True)[:, 0].cpu().numpy() != 0
        np.testing.assert_array_equal(d["vis"], plain["vis"] & kept)
        seen.append(kept)
        engine.render(model, cs)             # renders drop nothing
        np.testing.assert_array_equal(dump(cs, g.n)["out_img"], plain["out_img"])
    assert not np.array_equal(seen[0], seen[1]) and not np.array_equal(seen[1], seen[2])
    engine.set_step_options()
    want, _ = grads(g, cs, gt)
    a = dump(cs, g.n)
    engine.set_step_options(dropout_rate=0.0, dropout_seed=9, dropout_step=1)
    got, _ = grads(g, cs, gt)
    b = dump(cs, g.n)
    for k in a:
        np.testing.assert_array_equal(b[k], a[k])
    for p, q in zip(got, want):
        assert_grads(p, q, "rate 0")


def test_dropped_gaussians_are_culled_ones_to_adam():
    """A dropped Gaussian's features and statistics stay, its other moments
    decay; every kept visible one moves."""
    import torch
    g, cs = scene(3_000, 320, 240, seed=6)
    gt = torch.as_tensor(synthetic.target_image(cs.width, cs.height, 1)).cuda()
    model = engine.GaussianModel(g.groups())
    engine.set_step_options(dropout_rate=0.5, dropout_seed=3, dropout_step=1)
    engine.train_step(model, cs, gt)
    torch.cuda.synchronize()
    kept, _ = oc.keep(np.arange(g.n), 0.5, 1, 3)
    for k in range(6):
        m = model.exp_avg[k].cpu().numpy().reshape(g.n, -1)
        assert not m[~kept].any()
        np.testing.assert_array_equal(model.params[k].cpu().numpy()[~kept], g.groups()[k][~kept])
    assert not model.vis_counts.cpu().numpy()[~kept].any()
    vis = model.vis_counts.cpu().numpy() > 0
    assert vis.any() and (model.params[3].cpu().numpy()[vis] != g.features_dc[vis]).any(1).mean() > 0.9


@pytest.mark.parametrize("w, h", [(200, 160), (480, 330)])
def test_step_in_which_everything_is_dropped(w, h):
    """The background, no gradient, moments that decay from zero: a step like
    any other, and the next one is too."""
    import torch
    g, cs = scene(2_000, w, h, seed=14)
    gt = torch.as_tensor(synthetic.target_image(w, h, 1)).cuda()
    model = engine.GaussianModel(g.groups())
    engine.set_step_options(dropout_rate=1 - 2.0**-31, dropout_seed=1, dropout_step=1, mx4_colors=True)
    got, vis = grads(g, cs, gt)
    assert not vis.any() and not any(p.any() for p in got)
    img = engine.debug_buffer("out_img", 3 * w * h, np.float32).reshape(h, w, 3)
    np.testing.assert_array_equal(img, np.broadcast_to(np.float32(engine.DEFAULT_BG), img.shape))
    engine.train_step(model, cs, gt)
    for k in range(6):
        np.testing.assert_array_equal(model.params[k].cpu().numpy(), g.groups()[k])
    assert _lib.load().msplat_device_errors() == 0
    engine.set_step_options()
    engine.render(engine.GaussianModel(g.groups()), cs)
    want = dump(cs, g.n)
    engine.render(model, cs)
    np.testing.assert_array_equal(dump(cs, g.n)["out_img"], want["out_img"])


def test_views_of_one_step_share_the_mask():
    import torch
    g, _ = scene(2_000, 320, 240, seed=8)
    cams = [harness.setup_cam(c) for c in synthetic.fibonacci_cameras(3, 3.0, 320, 240)]
    gt = torch.as_tensor(synthetic.target_image(320, 240, 1)).cuda()
    engine.set_step_options(dropout_rate=0.4, dropout_seed=1, dropout_step=5, mx4_colors=True)
    buf = torch.zeros(multigpu.grad_floats(g.n, 15), device="cuda")
    grads(g, cams[0], gt, accumulate=buf)
    grads(g, cams[1], gt, accumulate=buf)
    got, vis = grads(g, cams[2], gt, accumulate=buf)
    kept, _ = oc.keep(np.arange(g.n), 0.4, 5, 1)
    assert not vis[~kept].any() and not any(p[~kept].any() for p in got) and vis.max() == 3
    parts = [grads(g, c, gt) for c in cams]
    np.testing.assert_array_equal(sum(p[1] for p in parts), vis)
    for k in range(6):
        assert_grads(got[k], sum(p[0][k].astype(np.float64) for p in parts), str(k))


def raster64(xy, conic, op, rgb, order, w, h, bg):
    """The forward blend in 64 bits (no saturation of the output)."""
    y, x = np.mgrid[0:h, 0:w].astype(np.float64)
    T, img, done = np.ones((h, w)), np.zeros((h, w, 3)), np.zeros((h, w), bool)
    for i in order:
        dx, dy = xy[i, 0] - x, xy[i, 1] - y
        sigma = 0.5 * (conic[i, 0] * dx * dx + conic[i, 2] * dy * dy) + conic[i, 1] * dx * dy
        alpha = np.minimum(0.999, op[i] * np.exp(-sigma))
        on = (sigma >= 0) & (sigma < 5.55) & (alpha >= 1 / 255) & ~done
        done |= on & (T * (1 - alpha) <= 1e-4)
        on &= ~done
        img += np.where(on, alpha * T, 0)[..., None] * np.maximum(rgb[i] + 0.5, 0)
        T = np.where(on, T * (1 - alpha), T)
    return img + T[..., None] * np.asarray(bg)


def test_dropout_opacity_gradient_against_differences():
    """d loss / d logit of a step with dropout against central differences
    of a 64-bit rasterizer under the step's own d loss / d image."""
    import torch
    n, w, h = 24, 48, 32
    g, cs = scene(n, w, h, seed=12, mean_range=0.4, log_mu=math.log(0.15))
    g.opacities = np.linspace(-2.5, -0.6, n, dtype=np.float32)[:, None]    # o = s / 0.7 < 0.51
    gt = torch.as_tensor(synthetic.target_image(w, h, 1)).cuda()
    engine.set_step_options(dropout_rate=0.3, dropout_seed=2, dropout_step=3)
    got, vis = grads(g, cs, gt)
    kept, scale = oc.keep(np.arange(n), 0.3, 3, 2)
    e = harness.engine_forward_dump(n, cs)
    v = engine.debug_buffer("v_rendered", 3 * w * h, np.float32).reshape(h, w, 3).astype(np.float64)
    ids = [i for i in np.argsort(e["depth"], kind="stable") if vis[i]]
    assert 8 <= len(ids) == kept.sum() < n
    logit = g.opacities[:, 0].astype(np.float64)

    def loss(l):
        op = scale / (1 + np.exp(-l))
        return (v * raster64(e["xy"].reshape(n, 2).astype(np.float64), e["conic"].astype(np.float64), op,
                             e["rgb"].astype(np.float64), ids, w, h, engine.DEFAULT_BG)).sum()
    step, want = 1e-6, np.zeros(n)
    for i in ids:
        d = np.zeros(n)
        d[i] = step
        want[i] = (loss(logit + d) - loss(logit - d)) / (2 * step)
    # a pixel at the 1/255 border may fall to either side in 32 and 64 bits;
    # none does in this scene (checked on the image: such a pixel would be
    # off by 1/255 of a colour, rounding moves it by less than 1e-5)
    op = scale / (1 + np.exp(-logit))
    img = raster64(e["xy"].reshape(n, 2).astype(np.float64), e["conic"].astype(np.float64), op,
                   e["rgb"].astype(np.float64), ids, w, h, engine.DEFAULT_BG)
    assert np.abs(np.clip(img, 0, 1) - e["img"].reshape(h, w, 3)).max() < 1e-5
    assert_grads(got[5][:, 0], want, "opacities")


# ---- refusals, and options together in the trainer

def test_packed_scene_refuses_what_does_not_fit():
    """A scene whose arrays disagree would be read out of range."""
    import torch
    g, _ = scene(100, 64, 48, seed=1)
    p = engine.PackedGaussians.of(engine.GaussianModel(g.groups()))
    parts = dict(means=p.means, scales=p.scales, quats=p.quats, opacities=p.opacities, records=p.records,
                 sh_degree=3)
    engine.PackedGaussians(**parts)
    for name, bad in (("means", p.means[:99]), ("scales", p.scales.double()), ("quats", p.quats[:, :3]),
                      ("opacities", p.opacities[:, 0]), ("records", p.records[:99]), ("sh_degree", 2),
                      ("means", p.means.cpu()), ("quats", torch.zeros(4, 100, device="cuda").t())):
        with pytest.raises(ValueError):
            engine.PackedGaussians(**dict(parts, **{name: bad}))


def test_step_refuses_wrong_bases():
    import torch
    g, cs = scene(500, 64, 48, seed=1, degree=2)
    gt = torch.as_tensor(synthetic.target_image(64, 48, 1)).cuda()
    engine.set_step_options(mx4_colors=True)
    cs.degree = 3
    with pytest.raises(_lib.EngineError, match="rest bases"):
        engine.train_step(engine.GaussianModel(g.groups()), cs, gt)
    with pytest.raises(ValueError, match="rate"):
        engine.set_step_options(dropout_rate=1.0)


def test_trainer_with_both_options(tmp_path):
    """A short run with dropout and 4-bit colours: it repeats from a
    checkpoint (the iteration is the draw counter), leaves the process's step
    options alone, and shows and evaluates the packed scene."""
    import msplat_b200 as msplat
    dataset_case.write_colmap(str(tmp_path / "scene"), n_points=400)
    ds = msplat.Dataset(str(tmp_path / "scene"), eval_mode=True, test_every=4)
    cfg = msplat.TrainingConfig(iterations=20, num_downscales=0, sh_degree_interval=2)
    t = msplat.GaussianTrainer(ds, cfg)
    with pytest.raises(ValueError, match="rate"):
        t.set_options(dropout_rate=1.5)
    t.set_options(dropout_rate=0.2, dropout_seed=5, mx4_colors=True)
    for _ in range(6):
        t.step()
    t.save_checkpoint(str(tmp_path / "a.msplat"))
    shown = t.render(0)
    metrics = t.evaluate()
    model, step = engine.GaussianModel.load_checkpoint(str(tmp_path / "a.msplat"))
    assert step == 6
    # the same scene with the unpacked features, rendered the plain way
    packed = engine.PackedGaussians.of(model)
    fdc, frest = packed.features()
    assert not bool((frest == model.params[4]).all())
    model.params[3].copy_(fdc)
    model.params[4].copy_(frest)
    model.save_checkpoint(str(tmp_path / "b.msplat"), step)
    u = msplat.GaussianTrainer(ds, cfg)
    u.load_checkpoint(str(tmp_path / "b.msplat"))
    np.testing.assert_array_equal(u.render(0), shown)
    assert u.evaluate() == metrics
    t.set_options()                          # the reference's training again
    assert not np.array_equal(t.render(0), shown)
    # no option of a trainer stays behind for other steps
    g, cs = scene(2_000, 320, 240, seed=3)
    import torch
    gt = torch.as_tensor(synthetic.target_image(320, 240, 1)).cuda()
    grads(g, cs, gt)
    plain = dump(cs, g.n)
    t.set_options(dropout_rate=0.5, dropout_seed=5, mx4_colors=True)
    t.step()
    grads(g, cs, gt)
    again = dump(cs, g.n)
    for k in plain:
        np.testing.assert_array_equal(again[k], plain[k])
    t.close()
    u.close()
