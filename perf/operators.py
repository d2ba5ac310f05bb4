"""Timed cases of the engine's dropout and 4-bit colour operators.

Each case is one pass through an operator, either in its plain form
(elementary torch operations in 32 bits) or, with `own` set, through
msplat_b200.operators, the calls a user makes.  `exact` is the same from
the operators' definitions in 64 bits.

  dropout    y = x * s where kept, 0 where dropped, and the same map on the
             gradient of y (its backward pass); the mask is a function of
             (seed, step, index) and is never stored
  pack       spherical-harmonics colours into 4-bit records and back to the
             values that the records stand for
  colors     view-dependent colours of all Gaussians for V cameras from the
             records
  backward   the gradient of the colour coefficients from that of the colours
"""
import math

import numpy as np
import torch

own = False

REST = (0, 3, 8, 15, 24)            # SH coefficients beside dc, per channel, by degree
RECORD = (8, 16, 24, 32, 48)        # bytes of a Gaussian's record, by degree


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one opacity per Gaussian of the smallest benchmark scene: latency
        dict(name="dropout_opacity_65k", op="dropout", rows=65_536, cols=1, pad=0, rate=0.1, whole_rows=True),
        # whole Gaussians' colour rows of the 1M scene
        dict(name="dropout_rows_1m", op="dropout", rows=1_000_000, cols=45, pad=0, rate=0.2, whole_rows=True),
        # single coefficients, odd sizes, rows inside a wider array
        dict(name="dropout_elements_odd", op="dropout", rows=333_337, cols=23, pad=4, rate=0.35, whole_rows=False),
        # the smallest benchmark scene
        dict(name="pack_65k", op="pack", n=65_536, degree=3),
        # a scene trained at degree 2, odd count
        dict(name="pack_odd_deg2", op="pack", n=333_337, degree=2),
        # the largest benchmark scene
        dict(name="pack_6m", op="pack", n=6_000_000, degree=3),
        # one frame of the smallest scene: latency
        dict(name="colors_65k", op="colors", n=65_536, degree=3, use=3, views=1, visible=1.0),
        # one frame of the 1M scene, two Gaussians of five culled
        dict(name="colors_1m_culled", op="colors", n=1_000_000, degree=3, use=3, views=1, visible=0.6),
        # eight cameras of the largest scene
        dict(name="colors_6m_8views", op="colors", n=6_000_000, degree=3, use=3, views=8, visible=1.0),
        # degree 4, odd sizes, a mask for each of three cameras
        dict(name="colors_odd_deg4", op="colors", n=250_007, degree=4, use=4, views=3, visible=0.5),
        # one view's gradients of the 1M scene
        dict(name="backward_1m", op="backward", n=1_000_000, degree=3, use=3, views=1, visible=0.6),
        # a batch of eight views, early in training (degree 2 of 3 in use)
        dict(name="backward_200k_8views", op="backward", n=200_003, degree=3, use=2, views=8, visible=0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dropout", "pack", "colors", "backward"))
    if op == "dropout":
        cols = rng.choice((1, 1, 3, 4, 9, 24, 45, rng.randint(2, 72)))
        rows = _log(rng, 1, 40_000_000 // cols)
        return dict(op=op, rows=rows, cols=cols, pad=rng.choice((0, 0, 1, 3, 4)), rate=round(rng.uniform(0.0, 0.9), 3),
                    whole_rows=rng.random() < 0.5)
    degree = rng.randint(0, 4)
    if op == "pack":
        return dict(op=op, n=_log(rng, 1, 4_000_000), degree=degree)
    views = rng.choice((1, 1, 2, 3, 5, 8, 16, 64))
    n = _log(rng, 1, 4_000_000 // views)
    return dict(op=op, n=n, degree=degree, use=rng.randint(0, degree), views=views,
                visible=rng.choice((1.0, 1.0, 0.6, 0.1)))


# ---------------------------------------------------------------- inputs

def _features(n, degree, g):
    """Colours as a trained scene has them: dc N(0, 0.3); rest N(0, 0.05)
    times a factor of its own for each Gaussian; Gaussians that no view has
    moved yet keep zeros."""
    dc = torch.randn(n, 3, generator=g, device="cuda") * 0.3
    rest = torch.randn(n, REST[degree], 3, generator=g, device="cuda") * 0.05
    rest *= torch.exp(torch.randn(n, 1, 1, generator=g, device="cuda"))
    rest *= (torch.rand(n, 1, 1, generator=g, device="cuda") > 0.08).float()
    return dc, rest


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case, seed=seed * 0x9E3779B97F4A7C15 % 2**64, step=seed % 30_000)
    if case["op"] == "dropout":
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        s["x"] = torch.randn(rows, cols + pad, generator=g, device="cuda")[:, :cols]
        s["v_y"] = torch.randn(rows, cols + pad, generator=g, device="cuda")[:, :cols]
        return s
    n, degree = case["n"], case["degree"]
    if case["op"] == "pack":
        s["dc"], s["rest"] = _features(n, degree, g)
        return s
    views = case["views"]
    s["means"] = torch.rand(n, 3, generator=g, device="cuda") * 4 - 2
    cam = np.random.RandomState(seed % 2**32).randn(views, 3)
    s["cams"] = (4 * cam / np.linalg.norm(cam, axis=1, keepdims=True)).astype(np.float32)
    s["radii"] = None
    if case["visible"] < 1:
        hit = torch.rand(views, n, generator=g, device="cuda") < case["visible"]
        s["radii"] = (hit * torch.randint(1, 60, (views, n), generator=g, device="cuda")).int()
    if case["op"] == "colors":
        dc, rest = _features(n, degree, g)
        s["records"] = _pack(dc, rest, degree)
        s["out"] = torch.zeros(views, n, 3, device="cuda")
    else:
        s["v_colors"] = torch.randn(views, n, 3, generator=g, device="cuda") * 1e-3
    return s


# ---------------------------------------------------------------- plain forms

def _philox(counter, step, seed):
    """Philox4x32-10 (Salmon et al., SC 2011) in 64-bit integers: four draws
    for each counter value."""
    m32 = 0xFFFFFFFF
    c = [counter & m32, counter >> 32 & m32, torch.full_like(counter, step & m32),
         torch.full_like(counter, step >> 32 & m32)]
    k0, k1 = seed & m32, seed >> 32 & m32
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [q >> 32 & m32 ^ c[1] ^ k0, q & m32, p >> 32 & m32 ^ c[3] ^ k1, p & m32]
        k0, k1 = k0 + 0x9E3779B9 & m32, k1 + 0xBB67AE85 & m32
    return torch.stack(c, -1)


def _dropout(x, v_y, rate, seed, step, whole_rows):
    rows, cols = x.shape
    count = rows if whole_rows else rows * cols
    draws = _philox(torch.arange((count + 3) // 4, device=x.device), step, seed).reshape(-1)[:count]
    threshold = round(rate * 2**32)
    kept = (draws >= threshold).reshape(rows, 1 if whole_rows else cols)
    scale = 2**32 / (2**32 - threshold)
    return torch.where(kept, x * scale, 0.0), torch.where(kept, v_y * scale, 0.0)


def _quantise(rest):
    """The e8m0 byte of each channel and the signed e2m1 codes."""
    amax = rest.abs().amax(1) if rest.shape[1] else rest.new_zeros(rest.shape[0], 3)
    byte = ((amax.view(torch.int32) + 0x200000 >> 23) - 2).clamp(min=0)
    y = rest * (254 - byte << 23).view(torch.float32)[:, None]      # times 2^(127 - byte), exact
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    return byte, code + 8 * torch.signbit(y)


def _pack(dc, rest, degree):
    n = dc.shape[0]
    records = torch.zeros(n, RECORD[degree], dtype=torch.uint8, device=dc.device)
    records[:, :6] = dc.half().view(torch.uint8).reshape(n, 6)
    if degree:
        byte, code = _quantise(rest)
        records[:, 6:9] = byte.to(torch.uint8)
        code = torch.nn.functional.pad(code.reshape(n, -1), (0, REST[degree] * 3 % 2)).reshape(n, -1, 2)
        records[:, 9:9 + code.shape[1]] = (code[:, :, 0] + 16 * code[:, :, 1]).to(torch.uint8)
    return records


def _unpack(records, degree):
    n = records.shape[0]
    dc = records[:, :6].contiguous().view(torch.float16).float()
    count = REST[degree] * 3
    codes = records[:, 9:9 + (count + 1) // 2].int()
    codes = torch.stack((codes & 15, codes >> 4), -1).reshape(n, -1)[:, :count].reshape(n, REST[degree], 3)
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=records.device)
    levels = torch.cat((levels, -levels))
    byte = records[:, 6:9].int()
    scale = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)      # 2^(byte - 127)
    return dc, levels[codes.long()] * scale[:, None] if count else levels.new_zeros(n, 0, 3)


def _basis(means, cams, use):
    """[V, n, bases in use] SH basis of the direction from each camera to each mean."""
    d = means[None] - cams[:, None]
    x, y, z = (d / (d * d).sum(-1, keepdim=True).sqrt()).unbind(-1)
    b = [torch.full_like(x, 0.28209479177387814)]
    if use >= 1:
        b += [-0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x]
    if use >= 2:
        xx, yy, zz = x * x, y * y, z * z
        b += [1.0925484305920792 * x * y, -1.0925484305920792 * y * z, 0.31539156525252005 * (2 * zz - xx - yy),
              -1.0925484305920792 * x * z, 0.5462742152960396 * (xx - yy)]
    if use >= 3:
        b += [-0.5900435899266435 * y * (3 * xx - yy), 2.890611442640554 * x * y * z,
              -0.4570457994644658 * y * (4 * zz - xx - yy), 0.3731763325901154 * z * (2 * zz - 3 * xx - 3 * yy),
              -0.4570457994644658 * x * (4 * zz - xx - yy), 1.445305721320277 * z * (xx - yy),
              -0.5900435899266435 * x * (xx - 3 * yy)]
    if use >= 4:
        b += [2.5033429417967046 * x * y * (xx - yy), -1.7701307697799304 * y * z * (3 * xx - yy),
              0.9461746957575601 * x * y * (7 * zz - 1), -0.6690465435572892 * y * z * (7 * zz - 3),
              0.10578554691520431 * (zz * (35 * zz - 30) + 3), -0.6690465435572892 * x * z * (7 * zz - 3),
              0.47308734787878004 * (xx - yy) * (7 * zz - 1), -1.7701307697799304 * x * z * (xx - 3 * yy),
              0.6258357354491761 * (xx * (xx - 3 * yy) - yy * (3 * xx - yy))]
    return torch.stack(b, -1)


def _colors(s):
    dc, rest = _unpack(s["records"], s["degree"])
    basis = _basis(s["means"], torch.from_numpy(s["cams"]).cuda(), s["use"])
    coef = torch.cat((dc[:, None], rest[:, :REST[s["use"]]]), 1)
    col = (basis[..., None] * coef).sum(2)
    return col if s["radii"] is None else torch.where(s["radii"][..., None] > 0, col, 0.0)


def _backward(s):
    v = s["v_colors"] if s["radii"] is None else torch.where(s["radii"][..., None] > 0, s["v_colors"], 0.0)
    basis = _basis(s["means"], torch.from_numpy(s["cams"]).cuda(), s["use"])
    grad = (basis[..., None] * v[:, :, None]).sum(0)
    rest = torch.zeros(s["n"], REST[s["degree"]], 3, device="cuda")
    rest[:, :REST[s["use"]]] = grad[:, 1:]
    return grad[:, 0].contiguous(), rest


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "dropout":
        y, v_x = _dropout(s["x"], s["v_y"], s["rate"], s["seed"], s["step"], s["whole_rows"])
        return {"y": y, "v_x": v_x}
    if s["op"] == "pack":
        dc, rest = _unpack(_pack(s["dc"], s["rest"], s["degree"]), s["degree"])
        return {"dc": dc, "rest": rest}
    if s["op"] == "colors":
        return {"colors": _colors(s)}
    v_dc, v_rest = _backward(s)
    return {"v_dc": v_dc, "v_rest": v_rest}


def _run_own(s):
    from msplat_b200 import operators as ops
    if s["op"] == "dropout":
        return {"y": ops.dropout(s["x"], s["rate"], s["seed"], s["step"], whole_rows=s["whole_rows"]),
                "v_x": ops.dropout(s["v_y"], s["rate"], s["seed"], s["step"], whole_rows=s["whole_rows"])}
    if s["op"] == "pack":
        dc, rest = ops.mx4_unpack(ops.mx4_pack(s["dc"], s["rest"]), s["degree"])
        return {"dc": dc, "rest": rest}
    if s["op"] == "colors":
        return {"colors": ops.mx4_colors(s["records"], s["degree"], s["means"], s["cams"], degrees_to_use=s["use"],
                                         radii=s["radii"], out=s["out"])}
    v_dc, v_rest = ops.mx4_colors_backward(s["v_colors"], s["degree"], s["means"], s["cams"], degrees_to_use=s["use"],
                                           radii=s["radii"])
    return {"v_dc": v_dc, "v_rest": v_rest}


def work(case):
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 16 * n, "flops": 2 * n}
    n, coefs = case["n"], 3 + 3 * REST[case["degree"]]
    if case["op"] == "pack":
        return {"bytes": 8 * n * coefs, "flops": 2 * n * coefs}
    views = case["views"]
    mask = 4 * views * n if case["visible"] < 1 else 0
    seen = views * n * case["visible"]                          # colours of a view
    some = n * (1 - (1 - case["visible"]) ** views)             # Gaussians that at least one view sees
    rows = some * RECORD[case["degree"]] if case["op"] == "colors" else n * 4 * coefs
    return {"bytes": 12 * some + rows + 12 * seen + mask, "flops": 2 * seen * (3 + 3 * REST[case["use"]])}


# ---------------------------------------------------------------- 64 bits

def _exact_draws(count, seed, step):
    u = np.uint64
    m32, s32 = u(0xFFFFFFFF), u(32)
    i = np.arange((count + 3) // 4, dtype=np.uint64)
    c0, c1, c2, c3 = i & m32, i >> s32, np.full_like(i, step & 0xFFFFFFFF), np.full_like(i, step >> 32)
    for r in range(10):
        k0 = u((seed + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c0 * u(0xD2511F53), c2 * u(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> s32) ^ c1 ^ k0, b & m32, (a >> s32) ^ c3 ^ k1, a & m32
    out = np.empty((i.size, 4), np.uint32)
    out[:, 0], out[:, 1], out[:, 2], out[:, 3] = c0, c1, c2, c3
    return out.reshape(-1)[:count]


def _exact_basis(means, cam, use):
    """Real spherical harmonics of one camera's directions, from their closed
    forms; the sign of odd orders as in the colour convention of the scenes."""
    d = means.double() - torch.tensor([float(v) for v in cam], dtype=torch.float64, device=means.device)
    d = d / torch.linalg.norm(d, dim=1, keepdim=True)
    x, y, z = d[:, 0], d[:, 1], d[:, 2]
    pi, r2 = math.pi, 2.0
    b = [torch.ones_like(x) * math.sqrt(1 / (4 * pi))]
    if use > 0:
        k = math.sqrt(3 / (4 * pi))
        b += [-k * y, k * z, -k * x]
    if use > 1:
        k = math.sqrt(15 / pi) / 2
        b += [k * x * y, -k * y * z, math.sqrt(5 / pi) / 4 * (3 * z**2 - 1), -k * x * z, k / 2 * (x**2 - y**2)]
    if use > 2:
        k, m = math.sqrt(35 / (r2 * pi)) / 4, math.sqrt(21 / (r2 * pi)) / 4
        n = math.sqrt(105 / pi) / 2
        b += [-k * y * (3 * x**2 - y**2), n * x * y * z, -m * y * (5 * z**2 - 1),
              math.sqrt(7 / pi) / 4 * (5 * z**3 - 3 * z), -m * x * (5 * z**2 - 1), n / 2 * z * (x**2 - y**2),
              -k * x * (x**2 - 3 * y**2)]
    if use > 3:
        k, m = math.sqrt(35 / pi) * 3 / 4, math.sqrt(35 / (r2 * pi)) * 3 / 4
        n, o = math.sqrt(5 / pi) * 3 / 4, math.sqrt(5 / (r2 * pi)) * 3 / 4
        b += [k * x * y * (x**2 - y**2), -m * y * z * (3 * x**2 - y**2), n * x * y * (7 * z**2 - 1),
              -o * y * z * (7 * z**2 - 3), math.sqrt(1 / pi) * 3 / 16 * (35 * z**4 - 30 * z**2 + 3),
              -o * x * z * (7 * z**2 - 3), n / 2 * (x**2 - y**2) * (7 * z**2 - 1), -m * x * z * (x**2 - 3 * y**2),
              k / 4 * (x**4 - 6 * x**2 * y**2 + y**4)]
    return torch.stack(b, 1)


def _two_to(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_round(dc, rest):
    """The values that 4-bit records stand for: dc to half precision; each
    channel of a Gaussian's rest to the e2m1 grid of the power of two that
    puts its largest magnitude in [3.5, 7)."""
    half = torch.from_numpy(dc.cpu().numpy().astype(np.float16).astype(np.float64)).to(dc.device)
    r = rest.double()
    if not r.shape[1]:
        return half, r
    top = r.abs().amax(1, keepdim=True)
    _, e = torch.frexp(top / 7)                   # top / 7 = m 2^e with m in [0.5, 1)
    e = torch.where(top / 7 == _two_to(e - 1), e - 1, e).clamp(min=-127)
    e = torch.where(top >= 7 * _two_to(e), e + 1, e)
    step = _two_to(e)
    a = r / step
    # the spacing of the grid is 0.5 below 2, 1 below 4, 2 above; round half to even
    space = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return half, torch.round(a / space) * space * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        count = rows if case["whole_rows"] else rows * cols
        threshold = int(np.rint(case["rate"] * 2.0**32))
        kept = _exact_draws(count, s["seed"], s["step"]).astype(np.int64) >= threshold
        kept = torch.from_numpy(kept).cuda().reshape(rows, -1)
        keep_rate = 1 - threshold / 2**32
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        return {"y": torch.where(kept, s["x"].double() / keep_rate, zero),
                "v_x": torch.where(kept, s["v_y"].double() / keep_rate, zero)}
    degree = case["degree"]
    if case["op"] == "pack":
        dc, rest = _exact_round(s["dc"], s["rest"])
        return {"dc": dc, "rest": rest}
    use, views = case["use"], case["views"]
    hit = [None if s["radii"] is None else (s["radii"][v] > 0).double()[:, None] for v in range(views)]
    if case["op"] == "colors":
        raw = s["records"].cpu().numpy()
        n, count = case["n"], 3 * REST[degree]
        dc = np.ascontiguousarray(raw[:, :6]).view(np.float16).astype(np.float64)
        coef = torch.from_numpy(dc).cuda()[:, None]
        if use:
            nibbles = np.empty((n, 2 * (raw.shape[1] - 9)), np.uint8)
            nibbles[:, 0::2], nibbles[:, 1::2] = raw[:, 9:] & 15, raw[:, 9:] >> 4
            table = np.array([(-1) ** (q >> 3) * ((q & 1) / 2 if (q & 7) < 2 else (1 + (q & 1) / 2) * 2.0 ** ((q >> 1 & 3) - 1))
                              for q in range(16)])
            codes = torch.from_numpy(nibbles[:, :count]).cuda().long()
            rest = torch.from_numpy(table).cuda()[codes].reshape(n, -1, 3)
            scale = torch.from_numpy(np.ldexp(1.0, raw[:, 6:9].astype(np.int32) - 127)).cuda()
            coef = torch.cat((coef, (rest * scale[:, None])[:, :REST[use]]), 1)
        out = torch.empty(views, n, 3, dtype=torch.float64, device="cuda")
        for v in range(views):
            basis = _exact_basis(s["means"], s["cams"][v], use)
            for c in range(3):
                out[v, :, c] = (basis * coef[:, :, c]).sum(1)
            if hit[v] is not None:
                out[v] *= hit[v]
        return {"colors": out}
    grad = torch.zeros(case["n"], 1 + REST[degree], 3, dtype=torch.float64, device="cuda")
    for v in range(views):
        basis = _exact_basis(s["means"], s["cams"][v], use)
        g = s["v_colors"][v].double() * (1 if hit[v] is None else hit[v])
        grad[:, :basis.shape[1]] += basis[:, :, None] * g[:, None]
    return {"v_dc": grad[:, 0].contiguous(), "v_rest": grad[:, 1:].contiguous()}
