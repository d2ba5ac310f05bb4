"""Dropout and 4-bit colour operators on the GPU against plain 64-bit
implementations (tests/operators_case.py), at the sizes, layouts and values
where they can go wrong.  Masks, records and the values they stand for are
exact; the bounds of sums count roundings (tests/operators_case.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from msplat_b200 import operators
from tests import operators_case as oc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    assert torch.cuda.is_available(), "these tests need a CUDA device"


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


# ---- dropout

def want_dropout(x, rate, seed, step, whole):
    rows, cols = x.shape
    idx = np.repeat(np.arange(rows), cols) if whole else np.arange(rows * cols)
    kept, scale = oc.keep(idx, rate, step, seed)
    kept = kept.reshape(x.shape)
    return kept, np.where(kept, x.astype(np.float64) * scale, 0.0)


def check_dropout(got, x, rate, seed, step, whole):
    kept, want = want_dropout(x, rate, seed, step, whole)
    np.testing.assert_array_equal(got != 0, kept & (x != 0))
    # the factor's rounding and the product's
    assert (np.abs(got - want) <= 2.001 * oc.U * np.abs(want)).all()


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("rows, cols", [(1, 1), (2, 1), (3, 1), (5, 1), (1023, 1), (4096, 1), (1, 45),
                                        (127, 45), (128, 45), (129, 45), (1000, 3), (257, 24),
                                        (33, 129), (3, 6001), (1001, 2), (2, 8192), (5, 9001),
                                        (1, 50_000)])
def test_dropout(rows, cols, whole):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = rng.normal(size=(rows, cols)).astype(np.float32)
    seed, step = 0x123456789ABCDEF0 + rows, 2**40 + cols
    got = host(operators.dropout(dev(x), 0.3, seed, step, whole_rows=whole))
    check_dropout(got, x, 0.3, seed, step, whole)


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("off, pad", [(0, 4), (1, 3), (2, 0), (3, 1)])
@pytest.mark.parametrize("rows, cols", [(301, 20), (5000, 1), (3000, 2), (7, 9001)])
def test_dropout_layouts(rows, cols, off, pad, whole):
    """Rows inside a wider array, at any alignment: the result is that of the
    same values side by side, and nothing outside the rows is written."""
    rng = np.random.default_rng(off * 10 + pad)
    base = dev(rng.normal(size=(rows * (cols + pad) + 8,)).astype(np.float32))
    x = base[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    flat = operators.dropout(x.contiguous(), 0.5, 3, 9, whole_rows=whole)
    assert torch.equal(operators.dropout(x, 0.5, 3, 9, whole_rows=whole), flat)
    check_dropout(host(flat), host(x), 0.5, 3, 9, whole)
    room = torch.full_like(base, 7.0)
    out = room[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    operators.dropout(x, 0.5, 3, 9, whole_rows=whole, out=out)
    assert torch.equal(out, flat)
    room2 = room.clone()
    room2[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = 7.0
    assert bool((room2 == 7.0).all())
    keep = base.clone()
    operators.dropout(x, 0.5, 3, 9, whole_rows=whole, out=x)      # in place
    assert torch.equal(x, flat)
    base[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = \
        keep[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    assert torch.equal(base, keep)


def test_dropout_shapes():
    """One dimension: a draw per element; more than two: rows of the last."""
    x = torch.randn(4, 6, 5, device="cuda")
    for whole in (False, True):
        want = operators.dropout(x.reshape(24, 5), 0.4, 1, 2, whole_rows=whole).reshape(4, 6, 5)
        assert torch.equal(operators.dropout(x, 0.4, 1, 2, whole_rows=whole), want)
    y = x.reshape(-1)
    assert torch.equal(operators.dropout(y, 0.4, 1, 2, whole_rows=True), operators.dropout(y, 0.4, 1, 2))
    assert operators.dropout(x[:0], 0.4, 1, 2).shape == (0, 6, 5)
    assert operators.dropout(torch.zeros(3, 0, device="cuda"), 0.4, 1, 2).shape == (3, 0)
    assert operators.dropout(torch.ones((), device="cuda"), 0.0, 1, 2).item() == 1.0
    for bad in (x.transpose(0, 2), x[:, ::2], torch.ones(1, 5, device="cuda").expand(3, 5), x.double(),
                torch.ones(5, 3, device="cuda").t()):
        with pytest.raises(ValueError):
            operators.dropout(bad, 0.4, 1, 2)
    for rate in (1.0, -0.5, float("nan")):
        with pytest.raises(ValueError, match="rate"):
            operators.dropout(x, rate, 1, 2)
    with pytest.raises(ValueError, match="shape"):
        operators.dropout(x, 0.4, 1, 2, out=torch.empty(4, 6, 6, device="cuda"))


@pytest.mark.parametrize("whole", [False, True])
def test_dropout_values(whole):
    """Rate 0 copies; a dropped NaN or infinity is 0 and a kept one stays; a
    gradient takes its forward's mask; seeds and steps differ."""
    x = torch.randn(500, 9, device="cuda")
    assert torch.equal(operators.dropout(x, 0.0, 5, 6, whole_rows=whole), x)
    mask = operators.dropout(torch.ones_like(x), 0.5, 5, 6, whole_rows=whole) != 0
    for bad in (float("nan"), float("inf")):
        y = operators.dropout(torch.full_like(x, bad), 0.5, 5, 6, whole_rows=whole)
        assert bool((y[~mask] == 0).all()) and not bool(torch.isfinite(y[mask]).any())
    assert torch.equal(operators.dropout(x, 0.5, 5, 6, whole_rows=whole), torch.where(mask, x * 2, 0.0))
    for seed, step in ((5, 7), (4, 6), (5 + 2**32, 6), (5, 6 + 2**32)):
        other = operators.dropout(torch.ones_like(x), 0.5, seed, step, whole_rows=whole) != 0
        assert not torch.equal(other, mask)
    same = operators.dropout(x, np.float32(0.5), np.int64(-1), np.uint64(6), whole_rows=np.bool_(whole))
    assert torch.equal(same, operators.dropout(x, 0.5, 2**64 - 1, 6, whole_rows=whole))
    near_one = operators.dropout(x, 1 - 2.0**-31, 5, 6, whole_rows=whole)
    assert bool((near_one == 0).all())


def test_dropout_past_32_bits():
    """Draw indexes past 2^32 (elements), and rows whose offsets pass it."""
    n = 2**32 + 64
    x = torch.ones(n, device="cuda")
    operators.dropout(x, 0.5, 8, 9, out=x)
    tail = host(x[-128:])
    del x
    kept, _ = oc.keep(np.arange(n - 128, n), 0.5, 9, 8)
    np.testing.assert_array_equal(tail, np.where(kept, 2.0, 0.0))
    # the last two: rows so far apart that offsets within a block's share pass it
    for rows, stride, widths in ((70_000, 62_001, (2, 1)), (1100, 2_100_001, (2, 1, 45)),
                                 (3, 1_100_000_001, (9001,))):
        wide = torch.empty(rows * stride, device="cuda").view(rows, stride)
        for cols in widths:
            for whole in (False, True):
                x = wide[:, :cols]
                x.fill_(1)
                out = operators.dropout(x, 0.5, 8, 9, whole_rows=whole)
                check_dropout(host(out), np.ones((rows, cols), np.float32), 0.5, 8, 9, whole)
                assert torch.equal(operators.dropout(x, 0.5, 8, 9, whole_rows=whole, out=x), out)
        del wide, x
    torch.cuda.empty_cache()


# ---- records

@pytest.mark.parametrize("degree", range(5))
@pytest.mark.parametrize("n", [1, 31, 127, 128, 129, 5003])
def test_pack_unpack(n, degree):
    dc, rest = oc.features(n, degree, seed=n + degree)
    rec = operators.mx4_pack(dev(dc), dev(rest))
    np.testing.assert_array_equal(host(rec), oc.encode(dc, rest))
    gdc, grest = operators.mx4_unpack(rec, degree)
    wdc, wrest = oc.decode(host(rec), degree)
    np.testing.assert_array_equal(host(gdc), wdc)
    np.testing.assert_array_equal(host(grest), wrest)


@pytest.mark.parametrize("degree", range(5))
def test_unpack_every_byte(degree):
    """Records of arbitrary bytes: each value of each byte, whether this
    library would write it or not (scales from 2^-127 on; 255 is NaN)."""
    rng = np.random.default_rng(degree)
    rec = rng.integers(0, 256, (6000, oc.BYTES[degree]), dtype=np.uint8)
    rec[:, 1] &= 0xBF                                 # halves that are finite numbers
    rec[:, 3] &= 0xBF
    rec[:, 5] &= 0xBF
    if degree:
        rec[:, 6:9] = rng.integers(0, 253, (6000, 3))
        rec[:7, 6:9] = [[0, 1, 2], [252, 251, 250], [255, 0, 0], [0, 255, 0], [0, 0, 255], [255] * 3, [0] * 3]
    gdc, grest = operators.mx4_unpack(dev(rec), degree)
    wdc, wrest = oc.decode(rec, degree)
    np.testing.assert_array_equal(host(gdc), wdc)
    np.testing.assert_array_equal(host(grest), wrest)


@pytest.mark.parametrize("degree", range(1, 5))
def test_pack_awkward_values(degree):
    dc, rest = oc.awkward_features(degree)
    rec = operators.mx4_pack(dev(dc), dev(rest))
    want = oc.encode(dc, rest)
    # a NaN has many bit patterns
    with np.errstate(over="ignore"):
        nan = np.isnan(dc.astype(np.float16))
    got = host(rec)
    gdc, grest = operators.mx4_unpack(rec, degree)
    np.testing.assert_array_equal(np.isnan(host(gdc)), nan)
    got6, want6 = got[:, :6].copy().view(np.uint16), want[:, :6].copy().view(np.uint16)
    np.testing.assert_array_equal(got6[~nan], want6[~nan])
    np.testing.assert_array_equal(got[:, 6:], want[:, 6:])
    np.testing.assert_array_equal(host(grest), oc.decode(want, degree)[1])


def test_pack_into_slices_and_unaligned_rows():
    """Records in the middle of a record array (aligned as records are), and
    features at any float alignment; neighbours stay as they were."""
    for degree in range(5):
        dc, rest = oc.features(300, degree, seed=40 + degree)
        room = torch.full((310, oc.BYTES[degree]), 0xAB, dtype=torch.uint8, device="cuda")
        fdc, frest = torch.empty(901, device="cuda"), torch.empty(300 * 3 * oc.REST[degree] + 1, device="cuda")
        vdc, vrest = fdc[1:].view(300, 3), frest[1:].view(300, oc.REST[degree], 3)
        vdc.copy_(dev(dc))
        vrest.copy_(dev(rest))
        rec = operators.mx4_pack(vdc, vrest, out=room[5:305])
        np.testing.assert_array_equal(host(rec), oc.encode(dc, rest))
        assert bool((room[:5] == 0xAB).all()) and bool((room[305:] == 0xAB).all())
        odc, orest = torch.full((902,), 7.0, device="cuda"), torch.full((frest.numel() + 1,), 7.0, device="cuda")
        operators.mx4_unpack(rec, degree, out=(odc[1:901].view(300, 3), orest[1:-1].view(vrest.shape)))
        np.testing.assert_array_equal(host(orest[1:-1].view(vrest.shape)), oc.decode(host(rec), degree)[1])
        for t in (odc, orest):
            assert t[0] == 7.0 and t[-1] == 7.0
    with pytest.raises(Exception, match="aligned"):
        room = torch.zeros(65, dtype=torch.uint8, device="cuda")
        operators.mx4_unpack(room[1:33].view(1, 32), 3)


def test_records_past_32_bits():
    """50M Gaussians of degree 3: 2.25e9 rest coefficients."""
    n = 50_000_000
    rest = torch.empty(n, 15, 3, device="cuda").normal_(0, 0.1)
    dc = torch.empty(n, 3, device="cuda").normal_()
    rec = operators.mx4_pack(dc, rest)
    tail = operators.mx4_pack(dc[-1000:].clone(), rest[-1000:].clone())
    assert torch.equal(rec[-1000:], tail)
    np.testing.assert_array_equal(host(tail), oc.encode(host(dc[-1000:]), host(rest[-1000:])))
    operators.mx4_unpack(rec, 3, out=(dc, rest))
    np.testing.assert_array_equal(host(rest[-1000:]), oc.decode(host(tail), 3)[1])
    del rest, dc, rec
    torch.cuda.empty_cache()


# ---- colours

def case(n, degree, views, seed):
    rng = np.random.default_rng(seed)
    dc, rest = oc.features(n, degree, seed)
    means = rng.uniform(-2, 2, (n, 3)).astype(np.float32)
    cams = rng.normal(size=(views, 3))
    cams = (4 * cams / np.linalg.norm(cams, axis=1, keepdims=True)).astype(np.float32)
    radii = (rng.integers(-1, 3, (views, n))).astype(np.int32)
    return oc.encode(dc, rest), means, cams, radii


@pytest.mark.parametrize("degree, use", [(0, 0), (1, 0), (1, 1), (2, 1), (2, 2), (3, 0), (3, 1), (3, 2),
                                         (3, 3), (4, 3), (4, 4)])
@pytest.mark.parametrize("n, views", [(1, 1), (127, 2), (1000, 1), (129, 3), (97, 64)])
def test_colors(n, views, degree, use):
    rec, means, cams, radii = case(n, degree, views, seed=n + 10 * degree + use)
    dc, rest = oc.decode(rec, degree)
    want, bound = oc.colors(dc, rest, means, cams, use)
    got = host(operators.mx4_colors(dev(rec), degree, dev(means), cams, degrees_to_use=use))
    assert got.shape == (views, n, 3)
    assert (np.abs(got - want) <= bound + 1e-44).all()
    # masked: the same bits where seen, untouched elsewhere
    out = torch.full((views, n, 3), 7.0, device="cuda")
    operators.mx4_colors(dev(rec), degree, dev(means), cams, degrees_to_use=use, radii=dev(radii), out=out)
    np.testing.assert_array_equal(host(out), np.where((radii > 0)[..., None], got, np.float32(7)))
    fresh = host(operators.mx4_colors(dev(rec), degree, dev(means), cams, degrees_to_use=use, radii=dev(radii)))
    np.testing.assert_array_equal(fresh, np.where((radii > 0)[..., None], got, np.float32(0)))


def test_colors_special_rows():
    """No view, no Gaussian; NaN channels; a mean at the camera; a mask that
    hides everything, NaN records and means behind it."""
    rec, means, cams, _ = case(50, 3, 2, seed=3)
    assert operators.mx4_colors(dev(rec), 3, dev(means), cams[:0]).shape == (0, 50, 3)
    assert operators.mx4_colors(dev(rec[:0]), 3, dev(means[:0]), cams).shape == (2, 0, 3)
    rec[7, 6] = 255                                   # red of Gaussian 7 is NaN
    means[9] = cams[0]
    got = host(operators.mx4_colors(dev(rec), 3, dev(means), cams))
    nan = np.zeros((2, 50, 3), bool)
    nan[:, 7, 0] = True
    nan[0, 9] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    got = host(operators.mx4_colors(dev(rec), 3, dev(means), cams, degrees_to_use=0))
    assert np.isfinite(got).all()
    rec[:] = 255
    means[:] = np.nan
    out = torch.full((2, 50, 3), 7.0, device="cuda")
    operators.mx4_colors(dev(rec), 3, dev(means), cams, radii=dev(np.zeros((2, 50), np.int32)), out=out)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("n", [1, 33, 128, 300])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_nothing_outside_the_outputs_is_written(n, off):
    """Colours, their gradients and unpacked features into the middle of larger
    arrays, at any alignment: the same values, and the floats around stay."""
    for degree, views in ((0, 1), (1, 2), (2, 1), (3, 1), (3, 3), (4, 1)):
        rec, means, cams, radii = case(n, degree, views, seed=off + n)
        g = torch.randn(views, n, 3, device="cuda")

        def room(*shape):
            size = int(np.prod(shape))
            t = torch.full((size + 12,), 7.0, device="cuda")
            return t, t[off + 4:off + 4 + size].view(shape)

        def around(t, view):
            t = t.clone()
            t[off + 4:off + 4 + view.numel()] = 7.0
            assert bool((t == 7.0).all())
        for r in (None, dev(radii)):
            whole, out = room(views, n, 3)
            out.zero_()
            operators.mx4_colors(dev(rec), degree, dev(means), cams, radii=r, out=out)
            assert torch.equal(out, operators.mx4_colors(dev(rec), degree, dev(means), cams, radii=r))
            around(whole, out)
            (w0, o0), (w1, o1) = room(n, 3), room(n, oc.REST[degree], 3)
            operators.mx4_colors_backward(g, degree, dev(means), cams, radii=r, out=(o0, o1))
            want = operators.mx4_colors_backward(g, degree, dev(means), cams, radii=r)
            assert torch.equal(o0, want[0]) and torch.equal(o1, want[1])
            around(w0, o0)
            around(w1, o1)
        operators.mx4_unpack(dev(rec), degree, out=(o0, o1))
        want = operators.mx4_unpack(dev(rec), degree)
        assert torch.equal(o0, want[0]) and torch.equal(o1, want[1])
        around(w0, o0)
        around(w1, o1)


def test_one_view_is_a_row_of_several():
    """The variants for one view and for several give the same bits."""
    rec, means, cams, radii = case(5000, 3, 4, seed=77)
    many = operators.mx4_colors(dev(rec), 3, dev(means), cams)
    for v in range(4):
        one = operators.mx4_colors(dev(rec), 3, dev(means), cams[v:v + 1])
        assert torch.equal(one[0], many[v])


def test_colors_past_32_bits():
    """64 views of 12M Gaussians: 2.3e9 colours."""
    n, views = 12_000_000, 64
    rec, means, cams, _ = case(1000, 1, views, seed=5)
    big = torch.zeros(n, 16, dtype=torch.uint8, device="cuda")
    big[-1000:] = dev(rec)
    pos = torch.ones(n, 3, device="cuda")
    pos[-1000:] = dev(means)
    out = operators.mx4_colors(big, 1, pos, cams)
    assert torch.equal(out[:, -1000:], operators.mx4_colors(dev(rec), 1, dev(means), cams))
    del big, pos, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("degree, use", [(0, 0), (1, 0), (1, 1), (2, 2), (3, 2), (3, 3), (4, 3), (4, 4)])
@pytest.mark.parametrize("n, views", [(1, 1), (127, 2), (1000, 1), (129, 3), (97, 64)])
@pytest.mark.parametrize("masked", [False, True])
def test_colors_backward(n, views, degree, use, masked):
    _, means, cams, radii = case(n, degree, views, seed=n + 10 * degree + use)
    radii = radii if masked else None
    g = np.random.default_rng(n).normal(size=(views, n, 3)).astype(np.float32)
    want = oc.colors_backward(g, degree, means, cams, use, radii)
    if masked:
        g[radii <= 0] = np.nan                        # must not be read as numbers
    got = operators.mx4_colors_backward(dev(g), degree, dev(means), cams, degrees_to_use=use,
                                        radii=None if radii is None else dev(radii))
    for a, w, bound in zip(got, want[:2], want[2:]):
        assert a.shape == w.shape
        assert (np.abs(host(a) - w) <= bound).all()
    assert bool((got[1][:, oc.REST[use]:] == 0).all())


def test_colors_backward_no_view_and_differences():
    """No view: zeros over whatever was there.  And the gradient against
    differences of the colours, which are linear in coefficients that records
    hold exactly."""
    n, degree = 200, 3
    _, means, cams, _ = case(n, degree, 3, seed=21)
    out = (torch.full((n, 3), 7.0, device="cuda"), torch.full((n, 15, 3), 7.0, device="cuda"))
    operators.mx4_colors_backward(torch.empty(0, n, 3, device="cuda"), degree, dev(means), cams[:0], out=out)
    assert all(bool((t == 0).all()) for t in out)
    rng = np.random.default_rng(22)
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4], np.float32)
    two = [(grid[rng.integers(0, 7, (n, 15, 3))] * rng.choice([-1, 1], (n, 15, 3))).astype(np.float32)
           for _ in range(2)]
    for t in two:
        t[:, 0] = 6                                   # the same scale in both
    dcs = [(rng.integers(-8, 9, (n, 3)) / 8).astype(np.float32) for _ in range(2)]
    cols = [host(operators.mx4_colors(operators.mx4_pack(dev(d), dev(t)), degree, dev(means), cams))
            .astype(np.float64) for d, t in zip(dcs, two)]
    v = rng.normal(size=cols[0].shape).astype(np.float32)
    gdc, grest = (host(t).astype(np.float64) for t in
                  operators.mx4_colors_backward(dev(v), degree, dev(means), cams))
    by_grad = (gdc * (dcs[1] - dcs[0])).sum() + (grest * (two[1] - two[0])).sum()
    by_diff = (v * (cols[1] - cols[0])).sum()
    bounds = [oc.colors(d.astype(np.float64), t.astype(np.float64), means, cams, degree)[1]
              for d, t in zip(dcs, two)]
    _, _, bdc, brest = oc.colors_backward(v, degree, means, cams, degree)
    tol = ((np.abs(v) * (bounds[0] + bounds[1])).sum() + (bdc * np.abs(dcs[1] - dcs[0])).sum()
           + (brest * np.abs(two[1] - two[0])).sum())
    assert abs(by_grad - by_diff) <= tol


# ---- streams, graphs, refusals that need a GPU

def chain(x, dc, rest, means, cams, g):
    y = operators.dropout(x, 0.4, 5, 6, whole_rows=True)
    rec = operators.mx4_pack(dc, rest)
    col = operators.mx4_colors(rec, 3, means, cams)
    back = operators.mx4_unpack(rec, 3)
    grad = operators.mx4_colors_backward(g, 3, means, cams)
    return [y, rec, col, *back, *grad]


def test_another_stream_and_a_captured_graph():
    def inputs(seed):
        dc, rest = oc.features(3000, 3, seed)
        _, means, cams, _ = case(3000, 3, 2, seed)
        rng = np.random.default_rng(seed)
        return [dev(rng.normal(size=(3000, 45)).astype(np.float32)), dev(dc), dev(rest), dev(means)], cams, \
            dev(rng.normal(size=(2, 3000, 3)).astype(np.float32))
    (a, cams, g), (b, _, g2) = inputs(1), inputs(2)
    want_a, want_b = chain(*a, cams, g), chain(*b, cams, g2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = chain(*a, cams, g)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want_a))
    held = [t.clone() for t in a]
    gh = g.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = chain(*held, cams, gh)
    cams_then = cams.copy()
    cams[:] = 0                                       # a capture keeps its own cameras
    for src, gs, want in ((a, g, want_a), (b, g2, want_b), (a, g, want_a)):
        for t, s in zip(held, src):
            t.copy_(s)
        gh.copy_(gs)
        graph.replay()
        torch.cuda.synchronize()
        if want is want_b:
            want = chain(*b, cams_then, g2)
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_calls_at_once():
    """Threads with streams of their own: each call's result is that of the
    call alone (nothing is shared between calls)."""
    from concurrent.futures import ThreadPoolExecutor

    def work(seed):
        dc, rest = oc.features(20_000 + seed, 3, seed)
        _, means, cams, _ = case(20_000 + seed, 3, 2, seed)
        x, g = dev(rest.reshape(len(rest), 45)), torch.ones(2, len(rest), 3, device="cuda")
        return [x, dev(dc), dev(rest), dev(means)], cams, g
    inputs = [work(s) for s in range(4)]
    want = [chain(*a, cams, g) for a, cams, g in inputs]
    torch.cuda.synchronize()

    def run(k):
        a, cams, g = inputs[k]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                out = chain(*a, cams, g)
        stream.synchronize()
        return out
    with ThreadPoolExecutor(4) as pool:
        for got, w in zip(pool.map(run, range(4)), want):
            assert all(torch.equal(p, q) for p, q in zip(got, w))


def test_python_refusals_on_tensors():
    rec = torch.zeros(4, 32, dtype=torch.uint8, device="cuda")
    means, cams = torch.zeros(4, 3, device="cuda"), [[0.0, 0.0, 4.0]]
    bad = [
        lambda: operators.mx4_colors(rec, 2, means, cams), lambda: operators.mx4_colors(rec, 3, means[:3], cams),
        lambda: operators.mx4_colors(rec, 3, means.double(), cams),
        lambda: operators.mx4_colors(rec, 3, means.cpu(), cams),
        lambda: operators.mx4_colors(rec, 3, means, [0.0, 0.0, 4.0]),
        lambda: operators.mx4_colors(rec, 3, means, torch.zeros(1, 3, device="cuda")),
        lambda: operators.mx4_colors(rec, 3, means, cams, radii=torch.ones(1, 4, device="cuda")),
        lambda: operators.mx4_colors(rec, 3, means, cams, radii=torch.ones(4, dtype=torch.int32, device="cuda")),
        lambda: operators.mx4_colors(rec, 3, means, cams, out=torch.ones(4, 3, device="cuda")),
        lambda: operators.mx4_colors(rec.float(), 3, means, cams),
        lambda: operators.mx4_colors(rec.t().contiguous().t(), 3, means, cams),
        lambda: operators.mx4_unpack(rec, 3, out=(means,)),
        lambda: operators.mx4_pack(means, torch.zeros(5, 15, 3, device="cuda")),
        lambda: operators.mx4_colors_backward(means, 3, means, cams),
        lambda: operators.mx4_colors_backward(means[None], 3, means, cams, out=(means, means)),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {k} was not refused")
