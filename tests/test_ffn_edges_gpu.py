"""The feed-forward operators at the ends of their ranges: waits that run out,
values near the limits of the types, special values, and variants that ordinary
shapes seldom take. Tolerances as in test_ffn_gpu.py (u(t) is half a step of the
type t relative to the value), unless a test states its own."""
import math

import pytest
import torch

from test_ffn_gpu import EPS, T, TINY, U, Mat, act64, gen, lib, norm64, normwise, product64, product_inputs, ptr, rand, scratch, within  # noqa: F401,E501

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------ waits
@pytest.mark.parametrize("dtype,cols", [("bf16", 5120), ("f32", 2048), ("bf16", 16384)])
@pytest.mark.parametrize("with_dhidden", [False, True])
def test_norm_gradient_wait_expiry_is_reported_and_the_context_stays_usable(lib, monkeypatch, dtype, cols, with_dhidden):
    """The gradients of long rows, which bulk copies bring in, with those left out
    (TTC_TEST_STALL=norm: nothing is ever in flight) and more rows a block than the
    ring holds: the wait runs out after about a millisecond, nothing more is sent
    for, the next synchronisation reports it, and the same call then repeats its
    earlier result."""
    rows = 2500
    g = gen(cols)
    hid, dy, dh = (Mat(rows, cols, dtype, fill=rand(g, rows, cols)) for _ in range(3))
    w = Mat(1, cols, dtype, fill=1 + rand(g, 1, cols, 0.1))

    def call():
        dx, dw = Mat(rows, cols, dtype), Mat(1, cols, dtype)
        d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, cols, hid.ptr, cols, w.ptr, dx.ptr, cols, dw.ptr,
                                       lib.DTYPES[dtype], dhidden=dh.ptr if with_dhidden else None, lddh=cols)
        ws = scratch(lib, d)
        lib.rms_norm_backward(d, ws)
        return dx, dw, ws

    first = call()
    lib.synchronize()
    monkeypatch.setenv("TTC_TEST_STALL", "norm")
    stalled = call()  # noqa: F841 -- its buffers stay until the kernels have ended
    with pytest.raises(lib.TTCError) as e:
        lib.synchronize()
    assert e.value.code == lib.ERR_TIMEOUT and "bounded wait expired" in str(e.value)
    monkeypatch.delenv("TTC_TEST_STALL")
    lib.synchronize()
    again = call()
    lib.synchronize()
    for a, b in zip(first[:2], again[:2]):
        assert torch.isfinite(a.t).all() and torch.equal(a.t, b.t)


# ------------------------------------------------------------------------------------------------ activations
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def factor64(act, z):
    """(s, s') of act(z) = z s(z): the factor of each activation and its derivative."""
    if act == "silu":
        s = torch.sigmoid(z)
        return s, s * torch.sigmoid(-z)
    if act == "gelu":
        # by erfc: torch.special.ndtr is (1 + erf) / 2, which keeps nothing of the tail
        return torch.special.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(8 / math.pi)
        t = a * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(t)
        return s, s * torch.sigmoid(-t) * a * (1 + 0.134145 * z * z)
    s = (z > 0).double() if act == "relu" else torch.ones_like(z)
    return s, torch.zeros_like(z)


def tail(dtype, n):
    """n values over [-10, 0] and a few positive ones, in the type."""
    z = torch.linspace(-10, 0, n - 40, dtype=torch.float64, device="cuda")
    return torch.cat([z, torch.linspace(0, 10, 40, dtype=torch.float64, device="cuda")]).to(T[dtype])


def relative(act, z):
    """How far an activation's factor may be off: 2^-21 (1 + |ln s|) of itself. The argument of its exponential is
    |ln s| large and goes through at most five roundings (2^-24 of it each), 2^x and 1 / x are good to 2^-22, and the
    fitted factor of the normal distribution to 2^-23."""
    s = factor64(act, z)[0]
    return 2.0 ** -21 * (1 - torch.log(s.clamp_min(1e-300)))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("M,N,odd", [(300, 72, False), (300, 67, True), (2560, 2048, False), (2560, 2050, True)])
def test_activation_tails_keep_their_relative_accuracy(lib, act, dtype, out, M, N, odd):
    """act(z) itself: one term a product (exact in fp32), w = 1. On each kernel, and where results leave by
    elements. The gated product with up = 1 likewise."""
    K = 8
    z = tail(dtype, M)
    x, w, wu = Mat(M, K, dtype, fill=0), Mat(N, K, dtype, fill=0), Mat(N, K, dtype, fill=0)
    x.t[:, 0] = z
    x.t[:, 1] = 1
    w.t[:, 0] = 1
    wu.t[:, 1] = 1
    zz = z.double()
    want = (zz * factor64(act, zz)[0]).view(M, 1).expand(M, N)
    tol = (U[out] + relative(act, zz).view(M, 1)) * want.abs() + TINY[out] + 2.0 ** -119
    pad = 3 if odd else 0
    for gated in (False, True):
        y = Mat(M, N, out, pad)
        common = dict(dtype=lib.DTYPES[dtype], y_dtype=lib.DTYPES[out], trans_w=True, act=lib.ACTIVATIONS[act])
        if gated:
            d = lib.gated_linear_desc(M, N, K, x.ptr, K, w.ptr, wu.ptr, K, y.ptr, y.ld, **common)
            lib.gated_linear(d, scratch(lib, d))
        else:
            d = lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, y.ld, **common)
            lib.linear(d, scratch(lib, d))
        within(y.t, want, tol, f"{act} gated {gated}")
        assert y.untouched_outside()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
def test_activation_gradients_in_the_tails(lib, act, dtype, pad):
    """dz, dg and du themselves: dx with w = 1 in one row and dy = 1 (up = 1). dz = s + z s' is off by what s is, and
    s' (a product of s, 1 - s or the same exponential, at most three factors) by three times that."""
    M, K = 300, 8
    z = tail(dtype, M)
    zz = z.double()
    s, ds = factor64(act, zz)
    slope = s + zz * ds
    rel = relative(act, zz)
    tol_slope = U[dtype] * slope.abs() + rel * s + 3 * rel * (zz * ds).abs() + TINY[dtype] + 2.0 ** -119
    tol_value = (U[dtype] + rel) * (zz * s).abs() + TINY[dtype] + 2.0 ** -119
    pre, one = Mat(M, 1, dtype, pad, fill=z.view(M, 1)), Mat(M, 1, dtype, pad, fill=1)
    x = Mat(M, K, dtype, fill=1)
    w1, w0 = Mat(1, K, dtype, fill=1), Mat(1, K, dtype, fill=0)
    dx = Mat(M, K, dtype)
    d = lib.linear_backward_desc(M, 1, K, one.ptr, one.ld, x.ptr, K, w1.ptr, K, lib.DTYPES[dtype], trans_w=True,
                                 act=lib.ACTIVATIONS[act], pre=pre.ptr, ldp=pre.ld, dx=dx.ptr, lddx=K)
    lib.linear_backward(d, scratch(lib, d))
    within(dx.t, slope.view(M, 1).expand(M, K), tol_slope.view(M, 1), "dz")
    for wg, wu, want, tol, name in ((w1, w0, slope, tol_slope, "dg"), (w0, w1, zz * s, tol_value, "du")):
        d = lib.gated_linear_backward_desc(M, 1, K, one.ptr, one.ld, x.ptr, K, wg.ptr, wu.ptr, K, pre.ptr, one.ptr, pre.ld,
                                           lib.DTYPES[dtype], trans_w=True, act=lib.ACTIVATIONS[act], dx=dx.ptr, lddx=K)
        lib.gated_linear_backward(d, scratch(lib, d))
        within(dx.t, want.view(M, 1).expand(M, K), tol.view(M, 1), name)


# ----------------------------------------------------------------------------------------------- rows of the norm
# One row length for each of the norm's kernels: a warp a row (one, two, four chunks), a block, a cluster, two passes.
ROW_LENGTHS = [64, 300, 1000, 2000, 6000, 40000]


def run_norm(lib, x, w, dtype, out, pad=0, eps=EPS, residual=None):
    """(y, scales, hidden) of the rows of x, the two last ones where they exist."""
    rows, cols = x.shape
    X, W = Mat(rows, cols, dtype, pad, fill=x), Mat(1, cols, dtype, fill=w)
    res, hid = (Mat(rows, cols, dtype, pad, fill=residual), Mat(rows, cols, dtype, pad)) if residual is not None else (None, None)
    y, sc = Mat(rows, cols, out, pad), Mat(1, rows, "f32") if out == "e4m3" else None
    lib.rms_norm(lib.rms_norm_desc(rows, cols, X.ptr, X.ld, W.ptr, y.ptr, y.ld, lib.DTYPES[dtype], y_dtype=lib.DTYPES[out],
                                   eps=eps, scales=ptr(sc), residual=ptr(res), ldr=X.ld, hidden=ptr(hid), ldh=X.ld))
    assert y.untouched_outside()
    return y.t, None if sc is None else sc.t[0], None if hid is None else hid.t


@pytest.mark.parametrize("cols", ROW_LENGTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
def test_e4m3_scales_show_rows_with_nan_and_infinities(lib, cols, dtype, pad):
    """Such a row has the scale NaN and NaN throughout, wherever in the row it is; a row of zeros has the smallest
    scale; the rows beside them are what they are without it."""
    g = gen(cols)
    x, w = rand(g, 9, cols), 1 + rand(g, 1, cols, 0.1)
    clean = run_norm(lib, x, w, dtype, "e4m3", pad)
    bad = {1: (0, "nan"), 3: (cols - 1, "nan"), 5: (cols // 2, "inf"), 7: (cols - 1, "-inf")}
    for r, (c, v) in bad.items():
        x[r, c] = float(v)
    x[4] = 0
    y, sc, _ = run_norm(lib, x, w, dtype, "e4m3", pad)
    for r in range(9):
        if r in bad:
            assert torch.isnan(sc[r]) and torch.isnan(y[r].double()).all(), r
        elif r == 4:
            assert sc[r] == 2.0 ** -126 and (y[r].double() == 0).all()
        else:
            assert sc[r] == clean[1][r] and torch.equal(y[r].double(), clean[0][r].double()), r


def far_rows(g, rows, cols):
    """Rows of ordinary size, of 1e25, close to the largest value, of 1e-25 and of 1e-30, in turn."""
    x = rand(g, rows, cols)
    size = torch.tensor([1.0, 1e25, 1.0, 1e-25, 1e-30], device="cuda", dtype=torch.float64).repeat(rows // 5 + 1)[:rows]
    x = x * size.view(rows, 1)
    x[2::5] *= 1.5e38 / x[2::5].abs().amax(dim=1, keepdim=True)
    return x


FAR = [(2500, 64), (2500, 300), (2500, 1000), (2500, 2000), (700, 6000), (330, 40000)]


@pytest.mark.parametrize("rows,cols", FAR)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["plain", "residual odd", "e4m3", "e4m3 residual odd"])
@pytest.mark.parametrize("eps", [EPS, 0.0])
def test_norm_of_rows_whose_squares_leave_fp32(lib, rows, cols, dtype, form, eps):
    """Finite rows have their formula's value whatever their size, beside ordinary rows; scaling by a power of two
    is exact, so the bounds are those of ordinary rows."""
    g = gen(rows + cols)
    pad = 3 if "odd" in form else 0
    x = Mat(rows, cols, dtype, fill=far_rows(g, rows, cols)).f64()
    res = Mat(rows, cols, dtype, fill=far_rows(g, rows, cols)).f64() if "residual" in form else None
    w = Mat(1, cols, dtype, fill=1 + rand(g, 1, cols, 0.1)).f64()
    out = "e4m3" if "e4m3" in form else dtype
    y, sc, hid = run_norm(lib, x, w, dtype, out, pad, eps, res)
    h = x if res is None else x + res
    want = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps) * w
    rel = ((cols / 32 + 16) / 2 + 10) * 2.0 ** -24
    if out != "e4m3":
        within(y, want, (U[out] + rel) * want.abs() + TINY[out], "y")
    else:
        scale = (want.abs().amax(dim=1) / 448).clamp_min(2.0 ** -126)
        within(sc, scale, (rel + 2.0 ** -22) * scale, "scales")
        q = want / scale[:, None]
        within(y, q, (U["e4m3"] + 2 * rel + 2.0 ** -22) * q.abs() + TINY["e4m3"], "q")
    if hid is not None:
        within(hid, h, (U[dtype] + 2.0 ** -24) * h.abs() + TINY[dtype], "hidden")


@pytest.mark.parametrize("rows,cols", FAR)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_of_far_rows_in_place(lib, rows, cols, dtype):
    g = gen(rows)
    x, res = (Mat(rows, cols, dtype, fill=far_rows(g, rows, cols)) for _ in range(2))
    w = Mat(1, cols, dtype, fill=1 + rand(g, 1, cols, 0.1))
    want, _, want_h = run_norm(lib, x.f64(), w.f64(), dtype, dtype, eps=0.0, residual=res.f64())
    lib.rms_norm(lib.rms_norm_desc(rows, cols, x.ptr, cols, w.ptr, x.ptr, cols, lib.DTYPES[dtype], eps=0.0,
                                   residual=res.ptr, ldr=cols, hidden=res.ptr, ldh=cols))
    assert torch.equal(x.t, want) and torch.equal(res.t, want_h)
    # the other way round: hidden over x, y over the residual
    x, res = (Mat(rows, cols, dtype, fill=far_rows(g, rows, cols)) for _ in range(2))
    want, _, want_h = run_norm(lib, x.f64(), w.f64(), dtype, dtype, eps=0.0, residual=res.f64())
    lib.rms_norm(lib.rms_norm_desc(rows, cols, x.ptr, cols, w.ptr, res.ptr, cols, lib.DTYPES[dtype], eps=0.0,
                                   residual=res.ptr, ldr=cols, hidden=x.ptr, ldh=cols))
    assert torch.equal(res.t, want) and torch.equal(x.t, want_h)


@pytest.mark.parametrize("rows,cols", FAR)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["plain", "dhidden", "odd"])
@pytest.mark.parametrize("eps", [EPS, 0.0])
def test_norm_gradients_of_rows_whose_squares_leave_fp32(lib, rows, cols, dtype, form, eps):
    """As above, for the gradients; dx over dy gives the same, and so does a call without dweight."""
    g = gen(rows + 3 * cols)
    pad = 3 if form == "odd" else 0
    hid = Mat(rows, cols, dtype, pad, fill=far_rows(g, rows, cols))
    dy = Mat(rows, cols, dtype, pad, fill=rand(g, rows, cols))
    dh = Mat(rows, cols, dtype, pad, fill=rand(g, rows, cols)) if form == "dhidden" else None
    wt = "f32" if form == "dhidden" else dtype
    w = Mat(1, cols, wt, fill=1 + rand(g, 1, cols, 0.1))
    dx, dw = Mat(rows, cols, dtype, pad), Mat(1, cols, wt)

    def call(dx, dw):
        d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, dy.ld, hid.ptr, hid.ld, w.ptr, dx.ptr, dx.ld, ptr(dw),
                                       lib.DTYPES[dtype], weight_dtype=lib.DTYPES[wt], eps=eps, dhidden=ptr(dh), lddh=cols)
        lib.rms_norm_backward(d, scratch(lib, d))

    call(dx, dw)
    h, e, ww = hid.f64(), dy.f64(), w.f64()
    r = 1 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    first = r * e * ww
    unit = h * r
    second = r * unit * (e * ww * unit).sum(1, keepdim=True) / cols
    spread = r * unit.abs() * (e * ww * unit).abs().sum(1, keepdim=True) / cols
    want = first - second + (dh.f64() if dh else 0)
    rel = (1.5 * (cols / 32 + 16) + 20) * 2.0 ** -24
    within(dx.t, want, U[dtype] * want.abs() + rel * (first.abs() + spread) + 2.0 ** -23 * want.abs() + TINY[dtype], "dx")
    terms = e * unit
    relw = rel + (min(rows, rows / 148 + 2) + 700) * 2.0 ** -24
    within(dw.t[0], terms.sum(0), U[wt] * terms.sum(0).abs() + relw * terms.abs().sum(0) + TINY[wt], "dweight")
    assert dx.untouched_outside() and dw.untouched_outside()
    without = Mat(rows, cols, dtype, pad)
    call(without, None)
    assert torch.equal(without.t, dx.t)
    if dh is not None:
        kept = dh.t.clone()
        call(dh, None)
        assert torch.equal(dh.t, dx.t)
        dh.t.copy_(kept)
    call(dy, None)
    assert torch.equal(dy.t, dx.t)


# ----------------------------------------------------------------------------------------------- e4m3 scales
@pytest.mark.parametrize("M,N,pad", [(3, 256, 0), (3, 256, 3), (300, 256, 0), (2560, 2048, 0), (2560, 2050, 0)])
@pytest.mark.parametrize("xs,ws", [(2.0 ** 110, 2.0 ** -100), (2.0 ** -120, 2.0 ** 110), (2.0 ** -60, 2.0 ** -60), (1.0, 0.75)])
def test_scales_are_multiplied_with_one_another_first(lib, M, N, pad, xs, ws):
    """On every kernel and path the same: the values here are whole numbers times a power of two, exact in fp32, and
    only the product of the scales keeps them in range."""
    K = 64
    g = gen(M)
    x, w = Mat(M, K, "e4m3", fill=448), Mat(N, K, "e4m3", fill=448)
    x.t[1:].copy_(torch.randint(-8, 9, (M - 1, K), generator=g, device="cuda").float())
    w.t[1:].copy_(torch.randint(-8, 9, (N - 1, K), generator=g, device="cuda").float())
    XS, WS = Mat(1, M, "f32", fill=xs), Mat(1, N, "f32", fill=ws)
    want = (x.f64() @ w.f64().t()) * (xs * ws)
    y = Mat(M, N, "f32", pad)
    lib.linear(lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, y.ld, lib.E4M3, y_dtype=lib.F32, trans_w=True,
                               x_scales=XS.ptr, w_scales=WS.ptr))
    assert torch.equal(y.f64(), want)
    gate, up = Mat(M, N, "f32", pad), Mat(M, N, "f32", pad)
    lib.gated_linear(lib.gated_linear_desc(M, N, K, x.ptr, K, w.ptr, w.ptr, K, y.ptr, y.ld, lib.E4M3, y_dtype=lib.F32,
                                           trans_w=True, gate=gate.ptr, up=up.ptr, ldp=up.ld, x_scales=XS.ptr,
                                           wg_scales=WS.ptr, wu_scales=WS.ptr))
    assert torch.equal(gate.f64(), want) and torch.equal(up.f64(), want)


# ------------------------------------------------------------------------------------------------ seldom taken
def pre_values(g, M, N, dtype):
    """What the gradients' activations see: ordinary values, zeros of both signs and the negative tail."""
    z = rand(g, M, N, 2.0)
    pick = torch.rand(M, N, generator=g, device="cuda")
    z = torch.where(pick < 0.1, torch.zeros_like(z), z)
    z = torch.where(pick < 0.05, -torch.zeros_like(z), z)
    z = torch.where(pick > 0.8, -2.0 - 8.0 * torch.rand(M, N, generator=g, device="cuda", dtype=torch.float64), z)
    return z.to(T[dtype])


# the tile kernel with both products in one launch, its column path, the pair kernel, its element path
GRADIENT_SHAPES = [(40, 200, 72, 0), (67, 129, 257, 3), (2304, 2080, 136, 0), (2560, 2050, 72, 3)]


@pytest.mark.parametrize("M,N,K,pad", GRADIENT_SHAPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", True), ("f16", True), ("bf16", False)])
def test_linear_gradients_of_every_activation(lib, M, N, K, pad, act, dtype, trans_w):
    """Bounds as in test_ffn_gpu.test_linear_backward, and the norm-wise one for f16 too."""
    g = gen(M + N + K)
    x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, dtype, trans_w, pad, 0)
    dy, pre = Mat(M, N, dtype, pad, fill=rand(g, M, N)), Mat(M, N, dtype, pad, fill=pre_values(g, M, N, dtype))
    dx, db = Mat(M, K, dtype, pad), Mat(1, N, dtype)
    dw = Mat(N, K, dtype, pad) if trans_w else Mat(K, N, dtype, pad)
    d = lib.linear_backward_desc(M, N, K, dy.ptr, dy.ld, x.ptr, x.ld, w.ptr, w.ld, lib.DTYPES[dtype], trans_w=trans_w,
                                 act=lib.ACTIVATIONS[act], pre=pre.ptr, ldp=pre.ld, dx=dx.ptr, lddx=dx.ld, dw=dw.ptr,
                                 lddw=dw.ld, dbias=db.ptr)
    lib.linear_backward(d, scratch(lib, d))
    dz = dy.f64() * act64(act, pre.f64())[1]
    ddz = (U[dtype] + 2.0 ** -20) * dz.abs() + 2.0 ** -20 * dy.f64().abs() + TINY[dtype]
    for got, a, da, b, name in ((dx.t, dz, ddz, wv.t(), "dx"), (dw.t if trans_w else dw.t.t(), dz.t(), ddz.t(), xv, "dw")):
        want, acc = product64(a, b)
        within(got, want, U[dtype] * want.abs() + da @ b.abs() + acc + TINY[dtype], name)
        normwise(got, want, dtype, name, (a, b))
    tol = U[dtype] * dz.sum(0).abs() + (M / 64 + 300) * 2.0 ** -24 * dz.abs().sum(0) + 2.0 ** -20 * dy.f64().abs().sum(0)
    within(db.t[0], dz.sum(0), tol + TINY[dtype], "dbias")
    assert dx.untouched_outside() and dw.untouched_outside() and db.untouched_outside()


@pytest.mark.parametrize("M,N,K,pad", GRADIENT_SHAPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", True), ("f16", True), ("bf16", False)])
def test_gated_gradients_of_every_activation(lib, M, N, K, pad, act, dtype, trans_w):
    """Bounds as in test_ffn_gpu.test_gated_linear_backward, and the norm-wise one for f16 too."""
    g = gen(M + N + 3 * K)
    x, (wg, wu), xv, (gv, uv), _, _ = product_inputs(g, M, N, K, dtype, trans_w, pad, 0, ("wg", "wu"))
    dy, up = (Mat(M, N, dtype, pad, fill=rand(g, M, N)) for _ in range(2))
    gate = Mat(M, N, dtype, pad, fill=pre_values(g, M, N, dtype))
    dx = Mat(M, K, dtype, pad)
    dwg, dwu = (Mat(N, K, dtype, pad) if trans_w else Mat(K, N, dtype, pad) for _ in range(2))
    d = lib.gated_linear_backward_desc(M, N, K, dy.ptr, dy.ld, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, gate.ptr, up.ptr,
                                       gate.ld, lib.DTYPES[dtype], trans_w=trans_w, act=lib.ACTIVATIONS[act], dx=dx.ptr,
                                       lddx=dx.ld, dwg=dwg.ptr, dwu=dwu.ptr, lddw=dwg.ld)
    lib.gated_linear_backward(d, scratch(lib, d))
    a, s = act64(act, gate.f64())
    e, u = dy.f64(), up.f64()
    dg, du = e * u * s, e * a
    ddg = (U[dtype] + 2.0 ** -20) * dg.abs() + 2.0 ** -20 * (e * u).abs() + TINY[dtype]
    ddu = (U[dtype] + 2.0 ** -20) * du.abs() + 2.0 ** -20 * e.abs() + TINY[dtype]
    zg, ag = product64(dg, gv.t())
    zu, au = product64(du, uv.t())
    want = zg + zu
    within(dx.t, want, U[dtype] * want.abs() + ddg @ gv.t().abs() + ddu @ uv.t().abs() + 2 * (ag + au) + TINY[dtype], "dx")
    normwise(dx.t, want, dtype, "dx", (dg, gv.t()), (du, uv.t()))
    for got, v, dv, name in ((dwg, dg, ddg, "dwg"), (dwu, du, ddu, "dwu")):
        want, acc = product64(v.t(), xv)
        stored = got.t if trans_w else got.t.t()
        within(stored, want, U[dtype] * want.abs() + dv.t() @ xv.abs() + acc + TINY[dtype], name)
        normwise(stored, want, dtype, name, (v.t(), xv))
        assert got.untouched_outside()
    assert dx.untouched_outside()


@pytest.mark.parametrize("N", [2688, 2944, 3200, 4736, 6272])  # 7, 6, 5, 4 and 3 shares of the sum on 148 SMs
@pytest.mark.parametrize("M,K", [(100, 2560), (93, 2568), (200, 2600)])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_every_number_of_shares(lib, N, M, K, dtype):
    """Sums split over clusters whose size is no power of two, in even and uneven shares."""
    g = gen(N + M)
    pad = -K % 16
    x, (w,), xv, (wv,), xs, (ws,) = product_inputs(g, M, N, K, dtype, True, pad, 0)
    y = Mat(M, N, "bf16")
    lib.linear(lib.linear_desc(M, N, K, x.ptr, x.ld, w.ptr, w.ld, y.ptr, N, lib.DTYPES[dtype], y_dtype=lib.BF16, trans_w=True,
                               x_scales=ptr(xs), w_scales=ptr(ws)))
    z, dz = product64(xv, wv)
    within(y.t, z, (U["bf16"] + 2.0 ** -23) * z.abs() + dz + TINY["bf16"], "linear")
    assert y.untouched_outside()
    half = N // 2  # the gated kernel's tiles are half as wide
    x, (wg, wu), xv, (gv, uv), xs, (gs, us) = product_inputs(g, M, half, K, dtype, True, pad, 0, ("wg", "wu"))
    y = Mat(M, half, "bf16")
    lib.gated_linear(lib.gated_linear_desc(M, half, K, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, y.ptr, half, lib.DTYPES[dtype],
                                           y_dtype=lib.BF16, trans_w=True, act=lib.ACT_NONE, x_scales=ptr(xs),
                                           wg_scales=ptr(gs), wu_scales=ptr(us)))
    a, da = product64(xv, gv)
    u, du = product64(xv, uv)
    want = a * u
    within(y.t, want, (U["bf16"] + 2.0 ** -23) * want.abs() + da * u.abs() + a.abs() * du + da * du + TINY["bf16"], "gated")
    assert y.untouched_outside()


@pytest.mark.parametrize("cols", ROW_LENGTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
def test_nan_and_infinities_stay_in_their_rows_of_the_norm(lib, cols, dtype, pad):
    """A NaN makes its row NaN, an infinity is NaN in its place and the rest of its row 0 (h rsqrt(inf)), in the
    gradients both make the row of dx NaN; the rows beside them are what they are without."""
    rows = 700
    g = gen(cols)
    x, w, dy = rand(g, rows, cols), 1 + rand(g, 1, cols, 0.1), rand(g, rows, cols)

    def gradients(x):
        X, DY, W, dx = (Mat(t.shape[0], cols, dtype, p, fill=t) for t, p in ((x, pad), (dy, pad), (w, 0), (x, pad)))
        d = lib.rms_norm_backward_desc(rows, cols, DY.ptr, DY.ld, X.ptr, X.ld, W.ptr, dx.ptr, dx.ld, None, lib.DTYPES[dtype])
        lib.rms_norm_backward(d)
        return dx.t

    clean, clean_dx = run_norm(lib, x, w, dtype, dtype, pad)[0], gradients(x)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for r, c, v in ((1, 0, "nan"), (300, cols - 1, "nan"), (2, cols // 2, "inf"), (699, cols - 1, "-inf")):
        x[r, c] = float(v)
        bad[r] = True
    y, dx = run_norm(lib, x, w, dtype, dtype, pad)[0], gradients(x)
    assert torch.equal(y[~bad], clean[~bad]) and torch.equal(dx[~bad], clean_dx[~bad])
    assert torch.isnan(y[[1, 300]]).all() and torch.isnan(dx[bad]).all()
    for r, c in ((2, cols // 2), (699, cols - 1)):
        assert torch.isnan(y[r, c]) and int((y[r] == 0).sum()) == cols - 1


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_wait_expiry_with_residual_copies_on_their_way(lib, monkeypatch, out):
    """The large products' loads left out, the residual's not: the kernel waits for those before it leaves."""
    M, N, K = 2048, 2560, 256
    g = gen(9)
    x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0)
    y, res = Mat(M, N, out), Mat(M, N, out, fill=rand(g, M, N))
    d = lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.BF16, y_dtype=lib.DTYPES[out], trans_w=True,
                        residual=res.ptr, ldr=N)
    torch.cuda.synchronize()
    monkeypatch.setenv("TTC_TEST_STALL", "linear")
    lib.linear(d)
    with pytest.raises(lib.TTCError) as e:
        lib.synchronize()
    assert e.value.code == lib.ERR_TIMEOUT
    monkeypatch.delenv("TTC_TEST_STALL")
    lib.linear(d)
    lib.synchronize()
    z, dz = product64(xv, wv)
    want = z + res.f64()
    within(y.t, want, (U[out] + 2.0 ** -22) * (want.abs() + res.f64().abs()) + dz + TINY[out], "y")


@pytest.mark.parametrize("rows,cols", FAR)
@pytest.mark.parametrize("pad", [0, 3])
def test_norm_rows_at_the_borders_of_the_range(lib, rows, cols, pad):
    """fp32 rows whose sums of squares lie within a few roundings of the largest value and of 2^-90, on both sides:
    each row is taken one way or the other, once, also where y and dx replace their inputs."""
    g = gen(rows + 7 * cols)
    # every element the same size, so that the sum is cols v^2; 41 steps of 2^-22 around each border
    near = 1 + (torch.arange(rows, device="cuda", dtype=torch.float64) % 41 - 20) * 2.0 ** -22
    border = torch.tensor([2.0 ** 128, 2.0 ** -90], device="cuda", dtype=torch.float64).repeat(rows // 2 + 1)[:rows]
    sign = (torch.rand(rows, cols, generator=g, device="cuda") < 0.5).double() * 2 - 1
    x = sign * (torch.sqrt(border / cols) * near).view(rows, 1)
    X, Y = Mat(rows, cols, "f32", pad, fill=x), Mat(rows, cols, "f32", pad)
    w = Mat(1, cols, "f32", fill=1 + rand(g, 1, cols, 0.1))
    dy, dx, dw = Mat(rows, cols, "f32", pad, fill=rand(g, rows, cols)), Mat(rows, cols, "f32", pad), Mat(1, cols, "f32")
    h, e, ww = X.f64(), dy.f64(), w.f64()
    r = 1 / torch.sqrt((h * h).mean(dim=1, keepdim=True))
    unit = h * r
    want = unit * ww
    rel = ((cols / 32 + 16) / 2 + 10) * 2.0 ** -24

    def back(dx, dw):
        d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, dy.ld, X.ptr, X.ld, w.ptr, dx.ptr, dx.ld, ptr(dw), lib.F32, eps=0.0)
        lib.rms_norm_backward(d, scratch(lib, d))

    back(dx, dw)
    first, spread = r * e * ww, r * unit.abs() * (e * ww * unit).abs().sum(1, keepdim=True) / cols
    rel_dx = (1.5 * (cols / 32 + 16) + 20) * 2.0 ** -24
    want_dx = first - r * unit * (e * ww * unit).sum(1, keepdim=True) / cols
    within(dx.t, want_dx, U["f32"] * want_dx.abs() + rel_dx * (first.abs() + spread) + 2.0 ** -23 * want_dx.abs() + TINY["f32"], "dx")
    relw = rel_dx + (min(rows, rows / 148 + 2) + 700) * 2.0 ** -24
    terms = e * unit
    within(dw.t[0], terms.sum(0), U["f32"] * terms.sum(0).abs() + relw * terms.abs().sum(0) + TINY["f32"], "dweight")
    back(dy, None)
    assert torch.equal(dy.t, dx.t)

    def forward(y):
        lib.rms_norm(lib.rms_norm_desc(rows, cols, X.ptr, X.ld, w.ptr, y.ptr, y.ld, lib.F32, eps=0.0))

    forward(Y)
    within(Y.t, want, (U["f32"] + rel) * want.abs() + TINY["f32"], "y")
    forward(X)
    assert torch.equal(X.t, Y.t)
