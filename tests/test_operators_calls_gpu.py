"""How calls of the dropout and 4-bit colour operators behave beside other
calls: beside an engine call that waits, after a failed one, and with tensors
that autograd follows."""
from __future__ import annotations

import threading

import pytest
import torch

from msplat_b200 import _lib, engine, operators, synthetic
from tests import harness

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def gpu():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    yield
    engine.set_step_options()
    _lib.load().cleanup_msplat_cuda()


def test_operators_do_not_wait_for_an_engine_call():
    """While one thread waits in the engine for about a second's work, another
    thread's operators run to their end on a stream of their own."""
    lib = _lib.load()
    busy, free = torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.randn(1000, 45, device="cuda")
    y, rec = torch.empty_like(x), torch.empty(1000, 32, dtype=torch.uint8, device="cuda")
    dc, rest = torch.randn(1000, 3, device="cuda"), torch.randn(1000, 15, 3, device="cuda")
    out = torch.empty(1, 1000, 3, device="cuda")
    gt = torch.as_tensor(synthetic.target_image(64, 48, 1)).cuda()
    model = engine.GaussianModel(synthetic.gaussians(500, 1).groups())
    cs = harness.setup_cam(synthetic.front_camera(64, 48, 3.0))

    def operate():
        with torch.cuda.stream(free):
            operators.dropout(x, 0.5, 1, 2, out=y)
            operators.mx4_pack(dc, rest, out=rec)
            operators.mx4_colors(rec, 3, dc, [[0.0, 0.0, 9.0]], out=out)
            operators.mx4_unpack(rec, 3, out=(dc, rest))
            operators.mx4_colors_backward(out, 3, dc, [[0.0, 0.0, 9.0]], out=(dc, rest))
        free.synchronize()
    try:
        with torch.cuda.stream(busy):
            engine.bind_stream()
            engine.train_step(model, cs, gt)          # everything allocated and loaded
            lib.msplat_last_loss(1)
            operate()
            torch.cuda.synchronize()
            torch.cuda._sleep(2_000_000_000)          # clock cycles: about a second
            engine.train_step(model, cs, gt)
            waiter = threading.Thread(target=lib.msplat_last_loss, args=(1,))
            waiter.start()
            waiter.join(0.1)
            assert waiter.is_alive()                  # in the engine, waiting
            operate()
            assert waiter.is_alive() and not busy.query()
            waiter.join()
    finally:
        torch.cuda.synchronize()
        engine.bind_stream()
    before = lib.msplat_kernel_launches(1)
    assert before > 0
    operate()
    assert lib.msplat_kernel_launches(0) == 5


def test_an_earlier_calls_failure_is_not_an_operators():
    """An allocation that cannot be met fails by itself; the operators after it
    give their results and no error."""
    lib = _lib.load()
    dc, rest = torch.randn(100, 3, device="cuda"), torch.randn(100, 15, 3, device="cuda")
    g = torch.randn(2, 100, 3, device="cuda")
    cams = [[0.0, 0.0, 9.0], [0.0, 9.0, 0.0]]

    def calls():
        rec = operators.mx4_pack(dc, rest)
        yield from (rec, operators.dropout(rest, 0.5, 1, 2), operators.dropout(rest, 0.5, 1, 2, whole_rows=True),
                    *operators.mx4_unpack(rec, 3), operators.mx4_colors(rec, 3, dc, cams),
                    operators.mx4_colors(rec, 3, dc, cams[:1]),
                    *operators.mx4_colors_backward(g, 3, dc, cams))
    want = list(calls())
    for f in (lambda: operators.mx4_pack(dc, rest), lambda: operators.dropout(rest, 0.5, 1, 2),
              lambda: operators.mx4_colors(want[0], 3, dc, cams), lambda: list(calls())):
        assert not lib.msplat_gpu_alloc(1 << 60, 0)
        assert "failed" in lib.msplat_last_error().decode()
        f()
    assert all(torch.equal(a, b) for a, b in zip(want, calls()))


def test_a_failed_allocation_is_reported_once():
    """It does not come up again as a render's or a step's error."""
    engine.bind_stream()
    lib = _lib.load()
    gt = torch.as_tensor(synthetic.target_image(64, 48, 1)).cuda()
    model = engine.GaussianModel(synthetic.gaussians(500, 1).groups())
    cs = harness.setup_cam(synthetic.front_camera(64, 48, 3.0))
    for alloc in (lib.msplat_gpu_alloc, lib.msplat_shared_alloc):
        for call in (lambda: engine.render(model, cs), lambda: engine.train_step(model, cs, gt)):
            assert not alloc(1 << 60, 0)
            call()
    torch.cuda.synchronize()
