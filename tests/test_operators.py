"""Dropout and 4-bit colour operators, what needs no GPU: the plain
implementations that the GPU tests hold the kernels to, and every refusal of
the C-ABI and of msplat_b200.operators (checked before any CUDA call)."""
from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from msplat_b200 import _lib, build, operators
from tests import operators_case as oc

P = 0x1000  # an aligned address that a refused call must never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


# ---- the plain implementations

@pytest.mark.parametrize("counter, key, want", [
    ((0, 0), 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((2**64 - 1, 2**64 - 1), 2**64 - 1, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x85A308D3243F6A88, 0x0370734413198A2E), 0x299F31D0A4093822,
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, want):
    got = oc.philox(np.array([counter[0]], np.uint64), counter[1], key)[0]
    assert tuple(int(v) for v in got) == want


def test_draws_are_uniform():
    d = oc.draws(np.arange(40_000), step=7, seed=11)
    # 6 standard deviations of a share of 40,000 draws
    for t in (0.1, 0.5, 0.9):
        assert abs((d < t * 2**32).mean() - t) < 6 * np.sqrt(t * (1 - t) / d.size)


@pytest.mark.parametrize("degree", range(5))
def test_record_values_are_nearest(degree):
    dc, rest = oc.features(500, degree, seed=degree)
    rdc, rrest = oc.decode(oc.encode(dc, rest), degree)
    assert (np.abs(rdc - dc) <= 2.0**-11 * np.abs(dc) + 2.0**-25).all()
    if degree:
        # half the widest step of the grid is 2^e, and the largest at least 3.5 2^e
        top = np.abs(rest).max(1, keepdims=True)
        assert (np.abs(rrest - rest) <= top / 3.5).all()
        # what a record stands for packs to itself
        again = oc.encode(rdc.astype(np.float32), rrest.astype(np.float32))
        np.testing.assert_array_equal(again, oc.encode(dc, rest))


def test_record_bytes(lib):
    assert [lib.msplat_mx4_record_bytes(d) for d in range(5)] == list(oc.BYTES)
    assert tuple(operators.RECORD_BYTES) == oc.BYTES and tuple(operators.REST_BASES) == oc.REST


# ---- refusals of the C-ABI

def refused(lib, rc, *words):
    assert rc == -1, rc
    text = lib.msplat_last_error().decode()
    for w in words:
        assert w in text, text


@pytest.mark.parametrize("change, words", [
    (dict(rows=-1), ("invalid shape",)), (dict(cols=0), ("invalid shape",)),
    (dict(xs=3), ("invalid shape",)), (dict(ys=3), ("invalid shape",)),
    (dict(rows=2**61, cols=1, xs=0, ys=0), ("invalid shape",)),
    (dict(rate=-0.1), ("rate",)), (dict(rate=1.0), ("rate",)), (dict(rate=float("nan")), ("rate",)),
    (dict(rate=1 - 2.0**-40), ("rate",)),
    (dict(x=None), ("null",)), (dict(y=None), ("null",)), (dict(y=P, xs=4, ys=5), ("in place",)),
])
def test_dropout_refusals(lib, change, words):
    a = dict(rows=8, cols=4, x=P, xs=4, y=2 * P, ys=4, rate=0.5)
    a.update(change)
    rc = lib.msplat_dropout(a["rows"], a["cols"], a["x"], a["xs"], a["y"], a["ys"], a["rate"], 1, 2,
                            0, None)
    refused(lib, rc, "msplat_dropout", *words)


@pytest.mark.parametrize("n, degree, dc, rest, rec, words", [
    (-1, 3, P, P, P, ("invalid shape",)), (1, -1, P, P, P, ("invalid shape",)),
    (1, 5, P, P, P, ("invalid shape",)), (1, 3, None, P, P, ("null",)), (1, 3, P, None, P, ("null",)),
    (1, 3, P, P, None, ("aligned",)), (1, 3, P, P, P + 8, ("16-byte aligned",)),
    (1, 2, P, P, P + 4, ("8-byte aligned",)),
])
def test_pack_refusals(lib, n, degree, dc, rest, rec, words):
    refused(lib, lib.msplat_mx4_pack(n, degree, dc, rest, rec, None), "msplat_mx4_pack", *words)
    refused(lib, lib.msplat_mx4_unpack(n, degree, rec, dc, rest, None), "msplat_mx4_unpack", *words)


@pytest.mark.parametrize("change, words", [
    (dict(n=-1), ("invalid shape",)), (dict(degree=5), ("invalid shape",)),
    (dict(use=4), ("invalid arguments",)), (dict(use=-1), ("invalid arguments",)),
    (dict(views=65), ("up to 64",)), (dict(views=-1), ("invalid arguments",)),
    (dict(cams=None), ("invalid arguments",)), (dict(means=None), ("null",)), (dict(col=None), ("null",)),
])
def test_colors_refusals(lib, change, words):
    a = dict(n=4, degree=3, use=3, means=P, rec=P, views=2, col=P, dc=P, rest=P,
             cams=np.zeros(200, np.float32).ctypes.data)
    a.update(change)
    refused(lib, lib.msplat_mx4_colors(a["n"], a["degree"], a["use"], a["means"], a["rec"], a["views"],
                                       a["cams"], None, a["col"], None), "msplat_mx4_colors", *words)
    refused(lib, lib.msplat_mx4_colors_backward(a["n"], a["degree"], a["use"], a["means"], a["views"],
                                                a["cams"], None, a["col"], a["dc"], a["rest"], None),
            "msplat_mx4_colors_backward", *words)


def test_colors_refuses_records(lib):
    cams = np.zeros(3, np.float32).ctypes.data
    for rec in (None, P + 8):
        refused(lib, lib.msplat_mx4_colors(1, 3, 3, P, rec, 1, cams, None, P, None), "aligned")
    for out in ((None, P), (P, None)):
        refused(lib, lib.msplat_mx4_colors_backward(1, 3, 3, P, 1, cams, None, P, *out, None), "null")


def test_nothing_to_do_is_no_error(lib):
    """Empty calls succeed without a GPU: nothing is launched."""
    assert lib.msplat_dropout(0, 1, None, 0, None, 0, 0.5, 1, 2, 0, None) == 0
    assert lib.msplat_mx4_pack(0, 3, None, None, None, None) == 0
    assert lib.msplat_mx4_unpack(0, 3, None, None, None, None) == 0
    assert lib.msplat_mx4_colors(0, 3, 3, None, None, 0, None, None, None, None) == 0
    assert lib.msplat_mx4_colors(5, 3, 3, None, None, 0, None, None, None, None) == 0
    assert lib.msplat_mx4_colors_backward(0, 3, 3, None, 0, None, None, None, None, None, None) == 0


# ---- refusals of the Python calls (a CPU tensor is one)

def test_python_refusals():
    x = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="CUDA tensor"):
        operators.dropout(x, 0.5, 1, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        operators.mx4_pack(x, torch.zeros(4, 15, 3))
    with pytest.raises(ValueError, match="bases"):
        operators.mx4_pack(x, torch.zeros(4, 14, 3))
    with pytest.raises(ValueError, match=r"\(N, B, 3\)"):
        operators.mx4_pack(x, x)
    with pytest.raises(ValueError, match="degree"):
        operators.mx4_unpack(torch.zeros(4, 32, dtype=torch.uint8), 7)
    with pytest.raises(ValueError, match="CUDA tensor"):
        operators.mx4_unpack(torch.zeros(4, 32, dtype=torch.uint8), 3)
    with pytest.raises(ValueError, match="CUDA tensor"):
        operators.mx4_colors(torch.zeros(4, 32, dtype=torch.uint8), 3, x, [[0, 0, 0]])
    with pytest.raises(ValueError, match="degree"):
        operators.mx4_colors_backward(torch.zeros(1, 4, 3), 5, x, [[0, 0, 0]])
    with pytest.raises(ValueError, match="degrees_to_use"):
        operators.mx4_colors_backward(torch.zeros(1, 4, 3), 2, x, [[0, 0, 0]], degrees_to_use=3)
    with pytest.raises(ValueError, match="V <= 64"):
        operators.mx4_colors_backward(torch.zeros(65, 4, 3), 2, x, np.zeros((65, 3)))
    with pytest.raises(ValueError, match="host data"):
        operators.mx4_colors_backward(torch.zeros(1, 4, 3), 2, x, torch.zeros(1, 3))


def test_a_negated_view_is_refused():
    """The imaginary part of a conjugate: its memory holds the other sign."""
    x = torch.complex(torch.ones(4, 1), torch.ones(4, 1)).conj().imag
    with pytest.raises(ValueError, match="negated"):
        operators._rows(x, "x")
    assert operators._rows(x.resolve_neg(), "x") == (4, 1, 1)


@pytest.mark.parametrize("use", [-1, 4, 1.5, 2.999, float("nan")])
def test_degrees_to_use_that_are_none(use):
    with pytest.raises(ValueError, match="degrees_to_use"):
        operators._use(use, 3)


def test_camera_positions_as_bytes():
    """C-ordered float32, whatever the array: its type, order and strides."""
    want = np.arange(12, dtype=np.float32).reshape(4, 3)
    wide = np.zeros((8, 6))
    wide[::2, ::2] = want
    for cams in (want, want.astype(np.float64), np.asfortranarray(want), want.tolist(), tuple(map(tuple, want)),
                 wide[::2, ::2], want.astype(int)):
        assert operators._views(cams) == (want.tobytes(), 4)
    assert operators._views(want[:0]) == (b"", 0)


def test_degrees_to_use():
    assert [operators._use(u, 3) for u in (None, 0, 3, np.int64(2), 1.0)] == [3, 0, 3, 2, 1]


def test_counts_past_32_bits_are_refused(monkeypatch):
    """The C-ABI takes columns and Gaussians as ints, which the binding would cut
    down: 2^32 + 64 columns became 64.  Nothing may be called."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    calls = []
    monkeypatch.setattr(operators, "_run", lambda fn, *a: calls.append(fn))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 0)
    with FakeTensorMode():
        def cuda(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device="cuda")
        assert operators.dropout(cuda(2**32 + 64), 0.5, 1, 2).shape == (2**32 + 64,)     # rows are 64-bit
        assert operators.dropout(cuda(1, 2**31 - 1), 0.5, 1, 2).shape == (1, 2**31 - 1)
        assert calls == ["msplat_dropout"] * 2
        calls.clear()
        for n in (2**31, 2**32 + 64):
            rec, means = cuda(n, 8, dtype=torch.uint8), cuda(n, 3)
            for call in (lambda: operators.dropout(cuda(1, n), 0.5, 1, 2),
                         lambda: operators.dropout(cuda(2, n + 3)[:, :n], 0.5, 1, 2, whole_rows=True),
                         lambda: operators.mx4_pack(means, cuda(n, 0, 3)),
                         lambda: operators.mx4_unpack(rec, 0),
                         lambda: operators.mx4_colors(rec, 0, means, [[0, 0, 0]]),
                         lambda: operators.mx4_colors_backward(cuda(1, n, 3), 0, means, [[0, 0, 0]])):
                with pytest.raises(ValueError, match="at most"):
                    call()
    assert not calls


def test_a_torch_without_cuda_can_import_the_module():
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "from msplat_b200 import operators\n"
            "try: operators.dropout(torch.zeros(3), 0.5, 1, 2)\n"
            "except ValueError as e: assert 'CUDA tensor' in str(e)\n"
            "else: raise AssertionError\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300,
                   cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


@pytest.fixture
def fake_cuda(monkeypatch):
    """CUDA tensors without memory, and the calls that would have been made."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    calls = []
    monkeypatch.setattr(operators, "_run", lambda fn, *a: calls.append(fn))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 0)
    with FakeTensorMode():
        yield calls


def operator_calls(grad=(), out=False):
    """Each operator's call with its tensors by name; those in `grad` require a
    gradient."""
    def t(name, *shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda", requires_grad=name in grad)
    rec, means, cams = t("records", 9, 32, dtype=torch.uint8), t("means", 9, 3), [[0, 0, 9]]
    dc, rest = t("dc", 9, 3), t("rest", 9, 15, 3)
    outs = dict(y=t("y", 9, 3), rec=torch.empty(9, 32, dtype=torch.uint8, device="cuda"), pair=(t("out0", 9, 3), t("out1", 9, 15, 3)),
                colors=t("out", 1, 9, 3))

    def kw(name):
        return dict(out=outs[name]) if out else {}
    return outs, {
        "dropout": (("x",), lambda: operators.dropout(t("x", 9, 3), 0.5, 1, 2, **kw("y"))),
        "mx4_pack": (("dc", "rest"), lambda: operators.mx4_pack(dc, rest, **kw("rec"))),
        "mx4_unpack": ((), lambda: operators.mx4_unpack(rec, 3, **kw("pair"))),
        "mx4_colors": (("means",), lambda: operators.mx4_colors(rec, 3, means, cams, **kw("colors"))),
        "mx4_colors_backward": (("v", "means"), lambda: operators.mx4_colors_backward(
            t("v", 1, 9, 3), 3, means, cams, **kw("pair")))}


def test_inputs_that_require_a_gradient_are_refused(fake_cuda):
    """Autograd would not hear of the call: its result would be a constant to
    the graph.  Without gradients the call is made."""
    for name, (inputs, _) in operator_calls()[1].items():
        for i in inputs:
            call = operator_calls(grad=(i,))[1][name][1]
            with pytest.raises(ValueError, match="requires a gradient"):
                call()
            assert not fake_cuda
            with torch.no_grad():
                assert not any(o.requires_grad for o in (call(),) if isinstance(o, torch.Tensor))
            assert fake_cuda == ["msplat_" + name]
            fake_cuda.clear()
    for name, o in (("dropout", "y"), ("mx4_unpack", "out0"), ("mx4_unpack", "out1"), ("mx4_colors", "out"),
                    ("mx4_colors_backward", "out1")):
        with pytest.raises(ValueError, match="requires a gradient"):
            operator_calls(grad=(o,), out=True)[1][name][1]()
    assert not fake_cuda


def test_a_packed_scene_takes_parameters(fake_cuda):
    """A scene to render may hold tensors that require a gradient."""
    from msplat_b200 import engine
    t = [torch.empty(9, w, device="cuda", requires_grad=True) for w in (3, 3, 4, 1)]
    packed = engine.PackedGaussians(*t, torch.empty(9, 32, dtype=torch.uint8, device="cuda"), 3)
    assert packed.n == 9 and packed.means is t[0]


def test_outputs_that_were_handed_in_count_as_modified(fake_cuda):
    """A graph that saved such a tensor must learn that it changed."""
    for name, written in (("dropout", ("y",)), ("mx4_pack", ("rec",)), ("mx4_unpack", ("pair",)),
                          ("mx4_colors", ("colors",)), ("mx4_colors_backward", ("pair",))):
        outs, calls = operator_calls(out=True)

        def versions():
            return {k: [u._version for u in (v if isinstance(v, tuple) else (v,))] for k, v in outs.items()}
        before = versions()
        calls[name][1]()
        after = versions()
        for k in outs:
            assert (after[k] == [v + 1 for v in before[k]]) == (k in written), (name, k)
            assert k in written or after[k] == before[k]


# ---- options of the training step and the packed renderer

def test_packed_scene_refusals():
    from msplat_b200 import engine
    t = torch.zeros
    with pytest.raises(ValueError, match="degree"):
        engine.PackedGaussians(t(4, 3), t(4, 3), t(4, 4), t(4, 1), t(4, 32, dtype=torch.uint8), 7)
    with pytest.raises(ValueError, match="CUDA tensor"):
        engine.PackedGaussians(t(4, 3), t(4, 3), t(4, 4), t(4, 1), t(4, 32, dtype=torch.uint8), 3)


def test_option_refusals(lib):
    for rate in (-0.5, 1.0, float("nan")):
        refused(lib, lib.msplat_set_step_options(C.byref(_lib.MsplatStepOptions(rate, 1, 2, 0))),
                "msplat_set_step_options", "rate")
    assert lib.msplat_set_step_options(C.byref(_lib.MsplatStepOptions(0.5, 1, 2, 1))) == 0
    assert lib.msplat_set_step_options(None) == 0
    refused(lib, lib.msplat_trainer_set_options(None, C.byref(_lib.MsplatTrainerOptions())), "no trainer")


@pytest.mark.parametrize("degree, rec, words", [(5, P, ("degree 5",)), (3, None, ("aligned",)),
                                                (3, P + 8, ("16-byte aligned",))])
def test_render_mx4_refusals(lib, degree, rec, words):
    m = (C.c_float * 16)()
    out = C.c_void_p()
    rc = lib.msplat_render_mx4(4, P, P, 1.0, P, m, m, 1.0, 1.0, 0.0, 0.0, 16, 16, (C.c_int * 3)(1, 1, 1),
                               0.01, degree, min(degree, 3), m, rec, P, m, C.byref(out))
    refused(lib, rc, "msplat_render_mx4", *words)
