"""The trainer's own step options: trainers beside each other and beside the
process's options, resumed runs."""
from __future__ import annotations

import threading

import numpy as np
import pytest

import msplat_b200 as msplat
from msplat_b200 import _lib, engine, multigpu, synthetic
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


def trainer(path, **options):
    dataset_case.write_colmap(str(path), n_points=400)
    ds = msplat.Dataset(str(path), eval_mode=True, test_every=4)
    t = msplat.GaussianTrainer(ds, msplat.TrainingConfig(iterations=1000, num_downscales=0, sh_degree_interval=2))
    t.set_options(**options)
    return t


def radii(n):
    return engine.debug_buffer("radii", n, np.int32)


def test_two_trainers_in_two_threads(tmp_path):
    """Each steps with its own options, whatever the other does between, and
    the process's options are what they were."""
    import torch
    a = trainer(tmp_path / "a", dropout_rate=0.5, dropout_seed=5)
    b = trainer(tmp_path / "b", mx4_colors=True)
    a.step()
    b.step()
    g = synthetic.gaussians(2_000, 3)
    cs = harness.setup_cam(synthetic.front_camera(320, 240, 3.0))
    gt = torch.as_tensor(synthetic.target_image(320, 240, 1)).cuda()

    def plain():
        model = engine.GaussianModel(g.groups())
        buf = torch.zeros(multigpu.grad_floats(model.n, 15), device="cuda")
        multigpu.EngineOps().grads(model, cs, gt, buf, 0.2, engine.DEFAULT_BG, 1.0, 0.01)
        return radii(g.n), engine.debug_buffer("out_img", 3 * 320 * 240, np.float32)
    want = plain()
    for _ in range(5):
        threads = [threading.Thread(target=lambda t=t: [t.step() for _ in range(20)]) for t in (a, b)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for p, q in zip(plain(), want):
            np.testing.assert_array_equal(p, q)
    a.close()
    b.close()


def test_a_resumed_run_draws_as_an_uninterrupted_one(tmp_path):
    """The iteration is the draws' step: after a checkpoint of iteration 6 both
    the run and its resumption drop what step 7 drops, and go on so."""
    t = trainer(tmp_path / "scene", dropout_rate=0.4, dropout_seed=5)
    for _ in range(6):
        t.step()
    t.save_checkpoint(str(tmp_path / "a.msplat"))
    u = trainer(tmp_path / "again", dropout_rate=0.4, dropout_seed=5)
    u.load_checkpoint(str(tmp_path / "a.msplat"))
    n = engine.GaussianModel.load_checkpoint(str(tmp_path / "a.msplat"))[0].n
    for step in (7, 8):
        kept, _ = oc.keep(np.arange(n), 0.4, step, 5)
        for run in (t, u):
            stats = run.step()
            assert (stats.iteration, stats.splat_count) == (step, n)
            r = radii(n)
            # were another step's draws taken, each that the view sees would be
            # one of ~kept with probability 0.4: none of 20, 4e-5
            assert not r[~kept].any() and (r[kept] > 0).sum() >= 20
    t.close()
    u.close()


def test_checkpoint_of_an_odd_number_of_bases(tmp_path):
    """Ten rest bases are no whole SH degree, which records hold: a render, an
    evaluation and a step with 4-bit colours say so."""
    t = trainer(tmp_path / "scene")
    t.step()
    t.save_checkpoint(str(tmp_path / "a.msplat"))
    model, step = engine.GaussianModel.load_checkpoint(str(tmp_path / "a.msplat"))
    groups = [p.cpu().numpy() for p in model.params]
    groups[4] = np.ascontiguousarray(groups[4][:, :10])
    engine.GaussianModel(groups).save_checkpoint(str(tmp_path / "b.msplat"), step)
    t.load_checkpoint(str(tmp_path / "b.msplat"))
    t.set_options(mx4_colors=True)
    with pytest.raises(RuntimeError, match="need 15 rest bases, not 10"):
        t.render(0)
    with pytest.raises(RuntimeError, match="rest bases"):
        t.evaluate()
    with pytest.raises(RuntimeError, match="rest bases"):
        t.step()
    t.close()
