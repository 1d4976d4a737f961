"""The layer operators (linear with its fused epilogue, its gradient, dropout)
against a 64-bit restatement.

Tolerances, per element, from the arithmetic:

* a product's sum of K terms in f32: at most (K + 16) additions, each off by at
  most 2^-23 of the running magnitude (the tensor cores truncate), so
  (K + 16) 2^-23 sum |a||b|; three-way bf16 splits of f32 operands drop terms
  of 2^-23 |a||b| a product at most, within the same bound;
* an activation changes its argument's error by a factor of at most 1.13 (the
  largest slope, GELU's) and adds 2^-18 of |z|;
* the output's rounding to 8 (bf16) or 11 (f16) significant bits: 2^-8 or
  2^-11 of the result at most (f16: 2^-24 absolute among subnormals); f32:
  2^-23;
* the gradients' products of 16-bit types read dz rounded to that type: one
  rounding of each term.
"""
import math

import numpy as np
import pytest
import torch

from ferrograd_b200 import kernels
from layer_ref import ACTS, drop as ref_drop, keep_mask, linear as ref_linear, \
    linear_grad as ref_grad, philox4x32, slope as ref_slope

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUND = {"f32": 2.0 ** -23, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -24}
STEP = 2.0 ** -23
CURVE = 2.0 ** -18


def randn(rng, rows, cols, dt, scale=1.0):
    a = rng.standard_normal((rows, cols)) * scale
    return torch.from_numpy(a).to(dt).cuda()


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def check(got, ref, tol, what):
    got = f64(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4], tol[bad][:4])


def layouts(t, kind, rng):
    """The same values in another layout."""
    if kind == "pitched":
        wide = torch.zeros((t.shape[0], t.shape[1] + 11), dtype=t.dtype, device=t.device)
        wide[:, 3:3 + t.shape[1]] = t
        return wide[:, 3:3 + t.shape[1]]
    if kind == "aligned_pitch":
        wide = torch.zeros((t.shape[0], (t.shape[1] + 15) // 8 * 8 + 16), dtype=t.dtype,
                           device=t.device)
        wide[:, 8:8 + t.shape[1]] = t
        return wide[:, 8:8 + t.shape[1]]
    if kind == "transposed":
        return t.t().contiguous().t()
    if kind == "strided":
        wide = torch.zeros((t.shape[0] * 2, t.shape[1] * 3), dtype=t.dtype, device=t.device)
        wide[::2, ::3] = t
        return wide[::2, ::3]
    return t


def forward_case(dtype, m, n, k, act, spec, residual, bias, pre, seed, xl="plain", wl="plain"):
    rng = np.random.default_rng(seed)
    dt = TYPES[dtype]
    x = layouts(randn(rng, m, k, dt), xl, rng)
    w = layouts(randn(rng, n, k, dt, 1 / math.sqrt(max(k, 1))), wl, rng)
    b = randn(rng, 1, n, dt, 0.5)[0] if bias else None
    r = randn(rng, m, n, dt) if residual else None
    got = kernels.linear(x, w, b, act=act, residual=r,
                         drop=kernels.Dropout(*spec) if spec else None, save_pre=pre)
    out, z = got if pre else (got, None)
    ref, refz = ref_linear(f64(x), f64(w), f64(b), act, spec, f64(r))
    size = np.abs(f64(x)) @ np.abs(f64(w)).T + (np.abs(f64(b)) if bias else 0.0)
    tz = (k + 16) * STEP * size
    u, tiny = ROUND[dtype], TINY[dtype]
    if pre:
        check(z, refz, tz + u * np.abs(refz) + tiny, "pre")
    scale = 65536.0 / (65536 - math.floor(spec[0] * 65536 + 0.5)) if spec and spec[0] < 1 else 1.0
    tol = scale * (1.13 * tz + (CURVE * np.abs(refz) if act != "none" else 0.0))
    tol = tol + u * np.abs(ref) + tiny + 2 * STEP * (np.abs(f64(r)) if residual else 0.0)
    check(out, ref, tol, "out")
    return x, w, b, r, out


SIZES = [(1, 1, 1), (1, 10, 7), (2, 16, 8), (3, 8, 64), (7, 257, 33), (16, 16, 16), (17, 129, 65),
         (64, 64, 64), (128, 256, 64), (130, 258, 96), (127, 255, 129), (256, 128, 784),
         (300, 512, 1000), (513, 515, 517), (1, 4096, 1024), (8, 1000, 2048), (9, 1024, 4096),
         (33, 2048, 512), (520, 1040, 72), (1100, 2064, 264)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(dtype, m, n, k):
    i = SIZES.index((m, n, k))
    act = ACTS[i % 5]
    spec = (0.25, 0x123456789ABCDEF0 + i, (7 << 40) + i) if i % 3 else None
    forward_case(dtype, m, n, k, act, spec, i % 2 == 0, i % 4 != 3, i % 3 == 1, i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(5, 72, 40), (200, 264, 136)])
def test_linear_activations(dtype, act, m, n, k):
    forward_case(dtype, m, n, k, act, (0.1, 5, 6), True, True, True, 77)


LAYOUTS = ["plain", "pitched", "aligned_pitch", "transposed", "strided"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("xl", LAYOUTS)
@pytest.mark.parametrize("wl", LAYOUTS)
@pytest.mark.parametrize("m,n,k", [(4, 80, 48), (150, 136, 200)])
def test_linear_layouts(dtype, xl, wl, m, n, k):
    forward_case(dtype, m, n, k, "gelu", (0.5, 1, 2), False, True, False, 3, xl, wl)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(0, 5, 4), (5, 0, 3), (4, 12, 0), (0, 0, 0), (200, 300, 0)])
def test_empty_sizes(dtype, m, n, k):
    forward_case(dtype, m, n, k, "silu", (0.3, 1, 2), True, True, True, 1)
    grad_case(dtype, m, n, k, "silu", (0.3, 1, 2), 1)


def grad_case(dtype, m, n, k, act, spec, seed, xl="plain", wl="plain", yl="plain", need=(1, 1, 1)):
    rng = np.random.default_rng(seed)
    dt = TYPES[dtype]
    x = layouts(randn(rng, m, k, dt), xl, rng)
    w = layouts(randn(rng, n, k, dt, 1 / math.sqrt(max(k, 1))), wl, rng)
    dy = layouts(randn(rng, m, n, dt), yl, rng)
    pre = randn(rng, m, n, dt, 1.5) if act != "none" else None
    got = kernels.linear_grad(dy, x, w, pre=pre, act=act,
                              drop=kernels.Dropout(*spec) if spec else None,
                              need_dx=bool(need[0]), need_dw=bool(need[1]), need_db=bool(need[2]))
    dx, dw, db, dz = ref_grad(f64(dy), f64(x), f64(w), f64(pre), act, spec)
    u, tiny = ROUND[dtype], TINY[dtype]
    # dz: the slope's error (absolute, of a slope of size one), then the
    # rounding of 16-bit types
    scale = 65536.0 / (65536 - math.floor(spec[0] * 65536 + 0.5)) if spec and spec[0] < 1 else 1.0
    tdz = (CURVE * scale * np.abs(f64(dy)) if act not in ("none", "relu") else 0.0) \
        + 2 * STEP * np.abs(dz)
    rounded = tdz + (u * np.abs(dz) + tiny if dtype != "f32" else 0.0)
    for name, g, ref, left, right, terms in (("dx", got[0], dx, np.abs(dz), np.abs(f64(w)), n),
                                             ("dw", got[1], dw, np.abs(dz).T, np.abs(f64(x)), m)):
        if not need[0 if name == "dx" else 1]:
            assert g is None
            continue
        r = rounded if name == "dx" else np.broadcast_to(rounded, dz.shape).T
        tol = (terms + 16) * STEP * (left @ right) + r @ right + u * np.abs(ref) + tiny
        check(g, ref, tol, name)
    if need[2]:
        tol = ((m + 16) * STEP * np.abs(dz) + tdz).sum(0) + u * np.abs(db) + tiny
        check(got[2], db, tol, "db")
    else:
        assert got[2] is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_grad(dtype, m, n, k):
    i = SIZES.index((m, n, k))
    spec = (0.25, 0xFEDCBA9876543210 - i, (3 << 33) + i) if i % 3 != 1 else None
    grad_case(dtype, m, n, k, ACTS[(i + 2) % 5], spec, i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_grad_activations(dtype, act):
    grad_case(dtype, 90, 72, 56, act, (0.1, 5, 6), 12)
    grad_case(dtype, 90, 72, 56, act, None, 13)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("yl", LAYOUTS)
@pytest.mark.parametrize("xl,wl", [("plain", "transposed"), ("pitched", "plain"),
                                   ("transposed", "pitched"), ("aligned_pitch", "strided"),
                                   ("strided", "aligned_pitch")])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_grad_layouts(dtype, yl, xl, wl, act):
    grad_case(dtype, 136, 152, 72, act, (0.5, 1, 2) if act == "gelu" else None, 3, xl, wl, yl)


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (0, 0, 0)])
def test_linear_grad_of_what_is_wanted(need):
    grad_case("bf16", 70, 40, 24, "silu", (0.2, 1, 9), 2, need=need)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 24), (200, 136, 264), (130, 77, 51), (6, 0, 9)])
def test_gradient_that_went_round(dtype, m, n, k):
    """dx_residual is added before dx is rounded."""
    rng = np.random.default_rng(m)
    dt = TYPES[dtype]
    x, w, dy = randn(rng, m, k, dt), randn(rng, n, k, dt, 0.2), randn(rng, m, n, dt)
    r = layouts(randn(rng, m, k, dt), "pitched", rng)
    got = kernels.linear_grad(dy, x, w, dx_residual=r)
    product = f64(dy) @ f64(w)
    ref = f64(r) + product
    tol = (n + 16) * STEP * (np.abs(f64(dy)) @ np.abs(f64(w))) + 2 * STEP * np.abs(f64(r))
    check(got[0], ref, tol + ROUND[dtype] * np.abs(ref) + TINY[dtype], "dx")
    plain = kernels.linear_grad(dy, x, w)
    assert torch.equal(got[1], plain[1]) and torch.equal(got[2], plain[2])
    with pytest.raises(ValueError):
        kernels.linear_grad(dy, x, w, need_dx=False, dx_residual=r)
    with pytest.raises(ValueError):
        kernels.linear_grad(dy, x, w, dx_residual=r[:, 1:])


def test_broadcast_gradient():
    """The gradient of a sum arrives as one value expanded (strides 0)."""
    rng = np.random.default_rng(0)
    for dtype, dt in TYPES.items():
        x, w = randn(rng, 40, 24, dt), randn(rng, 56, 24, dt, 0.2)
        pre = randn(rng, 40, 56, dt)
        one = torch.full((1, 1), 0.5, dtype=dt, device="cuda")
        wide = kernels.linear_grad(one.expand(40, 56), x, w, pre=pre, act="gelu_tanh")
        full = kernels.linear_grad(one.expand(40, 56).contiguous(), x, w, pre=pre, act="gelu_tanh")
        for a, b in zip(wide, full):
            assert torch.equal(a, b)
        wide = kernels.linear_grad(one.expand(40, 56), x, w)
        full = kernels.linear_grad(one.expand(40, 56).contiguous(), x, w)
        for a, b in zip(wide, full):
            assert torch.equal(a, b)


@pytest.mark.parametrize("act", ACTS[1:])
def test_gradient_against_differences(act):
    """d/dx, d/dw and d/dbias of sum(c * linear(x, w, bias)) by central
    differences of the 64-bit forward pass with the same mask.  A step h leaves
    h^2 |f'''| / 6 (third derivatives below 4 in these sums' units) and
    2^-52 / h of rounding; the f32 gradient is off by 2^-18 of its terms."""
    rng = np.random.default_rng(4)
    m, n, k, h = 6, 9, 5, 1e-4
    x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    b, c = rng.standard_normal(n), rng.standard_normal((m, n))
    x, w, b, c = (a.astype(np.float32).astype(np.float64) for a in (x, w, b, c))
    spec = (0.3, 11, 22)
    t = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    drop = kernels.Dropout(*spec)
    _, pre = kernels.linear(t(x), t(w), t(b), act=act, drop=drop, save_pre=True)
    dx, dw, db = kernels.linear_grad(t(c), t(x), t(w), pre=pre, act=act, drop=drop)
    z = x @ w.T + b
    assert np.abs(z).min() > 10 * h  # no step crosses ReLU's corner

    def loss(x, w, b):
        return float((c * ref_linear(x, w, b, act, spec, None)[0]).sum())

    for got, which in ((dx, 0), (dw, 1), (db, 2)):
        args = [x, w, b]
        base = args[which]
        num = np.zeros_like(base)
        for i in np.ndindex(base.shape):
            up, down = base.copy(), base.copy()
            up[i] += h
            down[i] -= h
            num[i] = (loss(*args[:which], up, *args[which + 1:])
                      - loss(*args[:which], down, *args[which + 1:])) / (2 * h)
        scale = np.abs(c).sum() * max(np.abs(x).max(), np.abs(w).max(), 1.0)
        assert np.abs(f64(got) - num).max() <= (CURVE + 4 * h * h) * scale


# ---- dropout ----------------------------------------------------------------------


def test_philox_known_answer():
    """The generator's published test vector (pi's digits as counter and key)."""
    got = philox4x32((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0))
    assert [int(w) for w in got] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 1001), (64, 64), (1000, 136),
                                       (2, 70000)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(dtype, rows, cols, residual):
    rng = np.random.default_rng(rows + cols)
    dt = TYPES[dtype]
    x = randn(rng, rows, cols, dt)
    r = randn(rng, rows, cols, dt) if residual else None
    spec = (0.4, 0xABCDEF0123456789, (1 << 60) + 17)
    got = kernels.dropout(x, kernels.Dropout(*spec), residual=r)
    d = ref_drop(f64(x), spec)
    ref = d if r is None else d + f64(r)
    tol = ROUND[dtype] * np.abs(ref) + 2 * STEP * np.abs(d) + TINY[dtype]
    check(got, ref, tol, "dropout")
    if not residual:  # what is dropped is exactly 0, and the gradient has the same mask
        kept = keep_mask(rows, cols, *spec)
        assert np.all(f64(got)[~kept] == 0.0)
        ones = torch.ones_like(x)
        assert np.array_equal(f64(kernels.dropout_grad(ones, kernels.Dropout(*spec))) != 0, kept)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_layouts_and_shapes(dtype):
    rng = np.random.default_rng(9)
    drop = kernels.Dropout(0.3, 4, 5)
    base = randn(rng, 33, 95, TYPES[dtype])
    want = kernels.dropout(base, drop)
    for kind in ("pitched", "aligned_pitch"):
        assert torch.equal(kernels.dropout(layouts(base, kind, rng), drop), want)
    cube = randn(rng, 6 * 5, 32, TYPES[dtype])
    assert torch.equal(kernels.dropout(cube.view(6, 5, 32), drop).view(30, 32),
                       kernels.dropout(cube, drop))
    line = randn(rng, 1, 1000, TYPES[dtype])
    assert torch.equal(kernels.dropout(line[0], drop), kernels.dropout(line, drop)[0])
    for shape in ((0, 8), (8, 0), (0,)):
        assert kernels.dropout(torch.empty(shape, dtype=TYPES[dtype], device="cuda"),
                               drop).shape == shape


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(20, 41), (40, 64)])
def test_dropout_extremes(dtype, rows, cols):
    """p = 0 and p below 2^-17 keep everything, p = 1 nothing (whole rows and
    columns empty); what is dropped is 0 even if it was NaN or infinite."""
    rng = np.random.default_rng(1)
    x = randn(rng, rows, cols, TYPES[dtype])
    assert torch.equal(kernels.dropout(x, kernels.Dropout(0.0, 1)), x)
    assert torch.equal(kernels.dropout(x, kernels.Dropout(1e-6, 1)), x)
    assert torch.equal(kernels.dropout(x, None), x)
    bad = x.clone()
    bad[::3] = float("nan")
    bad[1::3] = float("inf")
    assert not kernels.dropout(bad, kernels.Dropout(1.0, 1)).any()
    assert torch.equal(kernels.dropout(bad, kernels.Dropout(1.0, 1), residual=x), x)
    half = kernels.Dropout(0.5, 3)
    kept = torch.from_numpy(keep_mask(rows, cols, 0.5, 3, 0)).cuda()
    got = kernels.dropout(bad, half)
    assert not got[~kept].any()
    assert torch.equal(got[kept].isnan(), bad[kept].isnan())
    w = randn(rng, cols, 24, TYPES[dtype])
    y = randn(rng, rows, 24, TYPES[dtype])
    assert torch.equal(kernels.linear(y, w, act="gelu", drop=kernels.Dropout(1.0, 1), residual=x), x)
    for g in kernels.linear_grad(bad, y, w, pre=x, act="gelu", drop=kernels.Dropout(1.0, 1)):
        assert not g.any()


def test_mask_is_fair():
    """Over 2^20 elements the kept share is within 5 standard deviations, in
    every one of the eight positions of a block and over the two halves."""
    p, n = 0.1, 1 << 20
    x = torch.ones((1024, 1024), device="cuda")
    kept = (kernels.dropout(x, kernels.Dropout(p, 99, 1)) != 0)
    for part in [kept] + [kept[:, i::8] for i in range(8)] + [kept[:512], kept[512:]]:
        dev = math.sqrt(p * (1 - p) * part.numel())
        assert abs(float(part.sum()) - (1 - p) * part.numel()) <= 5 * dev + 1
    other = (kernels.dropout(x, kernels.Dropout(p, 99, 2)) != 0)
    same = float((kept == other).sum())
    q = p * p + (1 - p) * (1 - p)
    assert abs(same - q * n) <= 5 * math.sqrt(q * (1 - q) * n)


# ---- values at the ends of the range -------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_far_values(dtype, act):
    """Through w = 1: large z gives z (or, to the left, 0) and slopes 1 (0);
    an infinity the same; NaN stays NaN, but for ReLU's (0 < z) ? z : 0."""
    big = 3e4 if dtype == "f16" else 1e30
    z = torch.tensor([[50.0, -50.0, big, -big, float("nan")]], dtype=TYPES[dtype], device="cuda").t()
    one = torch.ones((1, 1), dtype=TYPES[dtype], device="cuda")
    got = f64(kernels.linear(z, one, act=act))[:, 0]
    dx = f64(kernels.linear_grad(torch.ones_like(z), z, one, pre=z.contiguous(), act=act)[0])[:, 0]
    zz = f64(z)[:, 0]
    if act == "none":
        assert np.array_equal(got[:4], zz[:4]) and np.all(dx[:4] == 1)
    else:
        assert np.allclose(got[[0, 2]], zz[[0, 2]], rtol=ROUND[dtype])
        assert np.all(np.abs(got[[1, 3]]) <= 1e-12)
        assert np.allclose(dx[:4], [1, 0, 1, 0], atol=1e-12)
    if act == "relu":
        assert got[4] == 0 and dx[4] == 0
    else:
        assert np.isnan(got[4])
        assert act == "none" or np.isnan(dx[4])
    pre = torch.tensor([[float("inf"), -float("inf")]], dtype=TYPES[dtype], device="cuda").t()
    dx = f64(kernels.linear_grad(torch.ones_like(pre), pre, one, pre=pre.contiguous(), act=act,
                                 need_dw=False)[0])[:, 0]
    assert np.array_equal(dx, [1, 1] if act == "none" else [1, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(6, 40, 72), (140, 200, 264)])
def test_nan_stays_in_its_row(dtype, m, n, k):
    rng = np.random.default_rng(5)
    x, w = randn(rng, m, k, TYPES[dtype]), randn(rng, n, k, TYPES[dtype])
    clean = kernels.linear(x, w)
    x[3, 5] = float("nan")
    w[7, 2] = float("inf")
    got = kernels.linear(x, w)
    rows = [i for i in range(m) if i != 3]
    cols = [i for i in range(n) if i != 7]
    assert got[3].isnan().all()
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    assert not got[rows][:, 7].isfinite().any()


# ---- streams, graphs, aliasing, repeatability -----------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(4, 256, 512), (256, 512, 320), (700, 1030, 250)])
def test_repeatable_in_place_and_on_another_stream(dtype, m, n, k):
    rng = np.random.default_rng(8)
    dt = TYPES[dtype]
    x, w, r = randn(rng, m, k, dt), randn(rng, n, k, dt, 0.05), randn(rng, m, n, dt)
    drop = kernels.Dropout(0.1, 3, 4)
    first = kernels.linear(x, w, act="silu", residual=r, drop=drop)
    assert torch.equal(kernels.linear(x, w, act="silu", residual=r, drop=drop), first)
    own = r.clone()
    assert kernels.linear(x, w, act="silu", residual=own, drop=drop, out=own) is own
    assert torch.equal(own, first)
    _, pre = kernels.linear(x, w, save_pre=True)
    grads = kernels.linear_grad(r, x, w, pre=pre, act="silu", drop=drop)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = kernels.linear(x, w, act="silu", residual=r, drop=drop)
        again = kernels.linear_grad(r, x, w, pre=pre, act="silu", drop=drop)
    raw = kernels.linear(x, w, act="silu", residual=r, drop=drop, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(other, first) and torch.equal(raw, first)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)
    same = x.clone()
    if k == n:
        kernels.dropout(same, drop, out=same)
    y = r.clone()
    assert torch.equal(kernels.dropout(y, drop, out=y), kernels.dropout(r, drop))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(2, 512, 640), (384, 640, 512)])
def test_graph_capture(dtype, m, n, k):
    rng = np.random.default_rng(8)
    dt = TYPES[dtype]
    x, w, dy = randn(rng, m, k, dt), randn(rng, n, k, dt, 0.05), randn(rng, m, n, dt)
    drop = kernels.Dropout(0.1, 3, 4)

    def step():
        out, pre = kernels.linear(x, w, act="gelu", drop=drop, save_pre=True)
        return (out, pre) + kernels.linear_grad(dy, x, w, pre=pre, act="gelu", drop=drop)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for g in got:
            g.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_f32_keeps_f32_accuracy():
    """Relative 2-norm errors of long f32 sums, random and of one sign.  A
    tensor-core chain of few truncating additions, joined by rounded ones,
    stays within 2^-19 (K = 4096 roundings at random give about 2^-20)."""
    rng = np.random.default_rng(6)
    for shift in (0.0, 1.0):
        x = torch.from_numpy(rng.standard_normal((512, 4096)) + shift).float().cuda()
        w = torch.from_numpy(rng.standard_normal((384, 4096)) * 0.02 + shift * 0.02).float().cuda()
        got = kernels.linear(x, w)
        ref = x.double() @ w.double().t()
        assert float((got - ref).norm() / ref.norm()) <= 2.0 ** -19
        dx, dw, _ = kernels.linear_grad(got, x, w)
        for g, r in ((dx, got.double() @ w.double()), (dw, got.double().t() @ x.double())):
            assert float((g - r).norm() / r.norm()) <= 2.0 ** -19


# ---- refusals --------------------------------------------------------------------------


def test_refusals():
    x, w = torch.zeros((4, 6), device="cuda"), torch.zeros((5, 6), device="cuda")
    out = torch.zeros((4, 5), device="cuda")
    bad = [
        lambda: kernels.linear(x.cpu(), w),
        lambda: kernels.linear(x.double(), w.double()),
        lambda: kernels.linear(x, w.half()),
        lambda: kernels.linear(x, w[:, :5]),
        lambda: kernels.linear(x[0], w),
        lambda: kernels.linear(x, w, torch.zeros(4, device="cuda")),
        lambda: kernels.linear(x, w, torch.zeros(10, device="cuda")[::2]),
        lambda: kernels.linear(x, w, act="tanh"),
        lambda: kernels.linear(x, w, residual=torch.zeros((5, 4), device="cuda")),
        lambda: kernels.linear(x, w, residual=torch.zeros((5, 4), device="cuda").t()),
        lambda: kernels.linear(x, w, out=torch.zeros((4, 5), device="cuda", dtype=torch.half)),
        lambda: kernels.linear(x, w, drop=kernels.Dropout(1.5, 0)),
        lambda: kernels.linear(x, w, drop=kernels.Dropout(-0.1, 0)),
        lambda: kernels.linear(x, w, drop=kernels.Dropout(float("nan"), 0)),
        lambda: kernels.linear_grad(out, x, w, act="gelu"),
        lambda: kernels.linear_grad(out.t(), x, w),
        lambda: kernels.linear_grad(out, x, w, pre=out[:, :4], act="gelu"),
        lambda: kernels.dropout(x.t(), kernels.Dropout(0.5, 0)),
        lambda: kernels.dropout(x.int(), kernels.Dropout(0.5, 0)),
        lambda: kernels.dropout(x, kernels.Dropout(2.0, 0)),
        lambda: kernels.dropout(x, kernels.Dropout(0.5, 0), out=out),
        # outputs over inputs
        lambda: kernels.linear(x, x[:, :6], out=x[:, :4]),
        lambda: kernels.linear(x, w, residual=torch.zeros(30, device="cuda")[:20].view(4, 5),
                               out=w.view(-1)[:20].view(4, 5)),
    ]
    buf = torch.zeros((8, 5), device="cuda")
    bad.append(lambda: kernels.linear(x, w, residual=buf[:4], out=buf[1:5]))
    bad.append(lambda: kernels.dropout(buf[:4], kernels.Dropout(0.5, 0), out=buf[1:5]))
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, kernels._lib.FerroError)):
            f()
            pytest.fail(f"refusal {i} was accepted")
    # columns of one buffer side by side are not an overlap
    both = torch.zeros((4, 12), device="cuda")
    both[:, :6] = 1
    kernels.linear(both[:, :6], torch.ones((5, 6), device="cuda"), out=both[:, 6:11])
    assert torch.equal(both[:, 6:11], torch.full((4, 5), 6.0, device="cuda"))
    assert torch.equal(both[:, :6], torch.ones((4, 6), device="cuda"))


# ---- large sizes, against 64 bits on the device ----------------------------------------


def device_check(got, ref, tol, what):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4])


def device_act(z, act):
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z.clamp(min=0.0) if act == "relu" else z


LARGE = [(2560, 2304, 320), (2501, 2311, 333), (2050, 4100, 1031), (4097, 1280, 4104),
         (1024, 1024, 20480), (2048, 2304, 17000), (96, 72, 40000), (130, 77, 33001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", LARGE)
def test_linear_large(dtype, m, n, k):
    """The same bounds as above; every form of the product, chains of 16384 and
    longer among them."""
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    dt = TYPES[dtype]
    new = lambda r, c, s: torch.empty((r, c), dtype=dt, device="cuda").normal_(  # noqa: E731
        0, s, generator=gen)
    x, w, b, r = new(m, k, 1), new(n, k, 1 / math.sqrt(k)), new(1, n, 1)[0], new(m, n, 1)
    act = "gelu" if k % 2 else "relu"
    spec = (0.2, 31, 1 << 35)
    out, pre = kernels.linear(x, w, b, act=act, residual=r, drop=kernels.Dropout(*spec),
                              save_pre=True)
    z = x.double() @ w.double().t() + b.double()
    size = x.double().abs() @ w.double().abs().t() + b.double().abs()
    tz = (k + 16) * STEP * size
    u, tiny = ROUND[dtype], TINY[dtype]
    device_check(pre, z, tz + u * z.abs() + tiny, "pre")
    keep = torch.from_numpy(keep_mask(m, n, *spec)).cuda()
    scale = 65536.0 / (65536 - math.floor(spec[0] * 65536 + 0.5))
    ref = torch.where(keep, device_act(z, act) * scale, 0.0) + r.double()
    tol = scale * (1.13 * tz + CURVE * z.abs()) + u * ref.abs() + tiny + 2 * STEP * r.double().abs()
    device_check(out, ref, tol, "out")
    # without the worst case's slack: random errors are far smaller than the bound
    limit = {"f32": 2.0 ** -19, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    assert float((pre.double() - z).norm() / z.norm()) <= limit


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(2560, 2304, 1320), (2501, 2311, 1333), (20000, 264, 520),
                                   (260, 20008, 136)])
def test_grad_large(dtype, m, n, k):
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    dt = TYPES[dtype]
    new = lambda r, c, s: torch.empty((r, c), dtype=dt, device="cuda").normal_(  # noqa: E731
        0, s, generator=gen)
    dy, x, w = new(m, n, 0.1), new(m, k, 1), new(n, k, 1 / math.sqrt(k))
    pre = new(m, n, 1.5)
    dx, dw, db = kernels.linear_grad(dy, x, w, pre=pre, act="relu")
    dz = torch.where(pre > 0, dy, 0.0).double()  # exact in every type
    u, tiny = ROUND[dtype], TINY[dtype]
    for got, a, b, terms, name in ((dx, dz, w.double(), n, "dx"), (dw, dz.t(), x.double(), m, "dw")):
        ref = a @ b
        tol = (terms + 16) * STEP * (a.abs() @ b.abs()) + u * ref.abs() + tiny
        device_check(got, ref, tol, name)
        limit = {"f32": 2.0 ** -19, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
        assert float((got.double() - ref).norm() / ref.norm()) <= limit, name
    ref = dz.sum(0)
    device_check(db, ref, (m + 16) * STEP * dz.abs().sum(0) + u * ref.abs() + tiny, "db")


def test_offsets_beyond_32_bits():
    """Outputs of more than 2^32 elements: the last rows are what they are by
    themselves (the mask goes by the row's number, so dropout is shifted by hand)."""
    rows, cols = 70000, 66008
    x = torch.empty((rows, 16), dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.empty((cols, 16), dtype=torch.bfloat16, device="cuda").normal_()
    out = kernels.linear(x, w, act="silu")
    assert out.numel() > 1 << 32
    for part in (slice(0, 100), slice(rows // 2, rows // 2 + 100), slice(rows - 100, rows)):
        assert torch.equal(out[part], kernels.linear(x[part], w, act="silu"))
    drop = kernels.Dropout(0.5, 3, 4)
    kernels.dropout(out, drop, out=out)
    tail = kernels.linear(x[-7:], w, act="silu")
    # the last rows' mask from the definition
    blocks = cols // 8
    col, row = np.meshgrid(np.arange(blocks), np.arange(rows - 7, rows))
    words = philox4x32((col, row, np.full_like(col, 4), np.full_like(col, 0)), (3, 0))
    r16 = np.stack([h for v in words for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], axis=2)
    keep = torch.from_numpy(r16.reshape(7, cols) >= 32768).cuda()
    assert torch.equal(out[-7:], torch.where(keep, tail * 2, torch.zeros_like(tail)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(2, 264, 320), (40, 264, 320), (2560, 2304, 320)])
def test_repeated_and_overlapping_rows(dtype, m, n, k):
    """A residual expanded over the rows and an x whose rows overlap (stride 8)
    give what their copies give."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    new = lambda *s: torch.empty(s, dtype=TYPES[dtype], device="cuda").normal_(  # noqa: E731
        generator=gen)
    w, r = new(n, k), new(1, n).expand(m, n)
    x = new(8 * m + k).as_strided((m, k), (8, 1))
    drop = kernels.Dropout(0.3, 1, 2)
    got = kernels.linear(x, w, act="relu", residual=r, drop=drop)
    want = kernels.linear(x.contiguous(), w, act="relu", residual=r.contiguous(), drop=drop)
    assert torch.equal(got, want)
    dy, base = new(m, n), new(1, k).expand(m, k)
    got = kernels.linear_grad(dy, x, w, dx_residual=base)
    want = kernels.linear_grad(dy, x.contiguous(), w, dx_residual=base.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
