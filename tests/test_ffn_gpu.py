"""The feed-forward operators (ttc_rms_norm, ttc_linear, ttc_gated_linear and
their gradients) against their definitions in 64 bits, at the sizes, strides
and values where they can go wrong.

Tolerances, derived once for all cases. u(t) is half a step of the type t
relative to the value (bf16 2^-8, fp16 2^-11, fp32 2^-24, e4m3 2^-4), tiny(t)
half its smallest step. S is the sum of |x||w| of a product.
* A sum of L fp32 terms taken one after the other is off by at most
  L 2^-24 of the sum of their absolute values. The norm's longest run of adds
  is cols / 32 + 16, and the square root halves it.
* A product accumulates 16 (8-bit types: 32) deep steps into an fp32
  accumulator; a step is one rounding, at worst a truncation (2^-23), with as
  much again for the sum inside the step: (K / 16 + 16) 2^-22 S.
* Activations have slopes within +-1.13 and are computed to 2^-20.
* A stored value is off by u of itself more.
* Gradients round dz (dg, du) to the type for the products: u of each term at
  worst; as the roundings are independent, over the whole matrix the error is
  sqrt(2) u / sqrt(3) < 0.82 u of its norm with the output's own rounding, and
  1.2 u bounds it with room for the accumulation. Of its norm or of E, the root
  of the summed squares of all terms, where that is larger: u / sqrt(3) is each
  term's own rms error, so a sum that cancels (300 terms that add up to a value
  a fifth of E) carries u E / sqrt(3) whatever is left of it. It is a statement
  about many values; matrices below 64 values have the bound by value alone.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134, "e4m3": 2.0 ** -10}
EPS = 1e-6
SENTINEL = 3.0


@pytest.fixture(scope="module")
def lib(ttc):
    """The library on torch's stream for this module's tests."""
    torch.cuda.init()
    ttc.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ttc
    torch.cuda.synchronize()
    ttc.set_stream(None)


class Mat:
    """A matrix inside a larger buffer: `pad` extra elements a row, `shift`
    elements in front; everything outside the matrix holds a sentinel."""

    def __init__(self, rows, cols, dtype, pad=0, shift=0, fill=None):
        self.ld = cols + pad
        self.buf = torch.full((shift + rows * self.ld + 64,), SENTINEL, device="cuda").to(T[dtype])
        self.t = self.buf[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols]
        if fill is not None:
            self.t.copy_(fill)
        self.outside = torch.ones(self.buf.numel(), dtype=torch.bool, device="cuda")
        self.outside[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols] = False

    @property
    def ptr(self):
        return self.t.data_ptr() if self.t.numel() else self.buf.data_ptr()

    def f64(self):
        return self.t.double()

    def untouched_outside(self):
        return bool((self.buf[self.outside].double() == SENTINEL).all())


def rand(gen, rows, cols, scale=1.0):
    return torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.float64) * scale


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def within(got, want, tol, what=""):
    """Everywhere |got - want| <= tol, infinities and NaN in the same places."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    off = (got - want).abs()[fine]
    lim = tol.expand_as(want)[fine]
    bad = off > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / lim).max()):.3g} x its bound"


def normwise(got, want, dtype, what, *terms):
    """`terms`: the pairs of factors whose products, summed, are `want`."""
    n = max(want.norm(), sum((a.square() @ b.square()).sum() for a, b in terms).sqrt())
    if want.numel() >= 64 and n > 0:
        err = float((got.double() - want).norm() / n)
        assert err <= 1.2 * U[dtype], f"{what}: norm-wise {err:.3g}"


def act64(act, z):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(8 / math.pi)
        p = torch.sigmoid(a * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * a * (1 + 0.134145 * z * z)
    return z, torch.ones_like(z)


def ptr(m):
    return None if m is None else m.ptr


def ld(m):
    return 0 if m is None else m.ld


def scratch(lib, desc):
    n = lib.workspace_size(desc)
    # filled with ones' bits (NaN in every type): nothing may depend on what a workspace holds
    return torch.full((n,), 255, dtype=torch.uint8, device="cuda") if n else None


# ------------------------------------------------------------------------------------------------------- norm
NORM_SHAPES = [(1, 1), (1, 8), (1, 4096), (3, 7), (5, 100), (2, 1000), (130, 257), (4, 1024), (7, 2048), (33, 4104),
               (2, 16384), (3, 16392), (2, 40000), (1, 131), (700, 64)]


def norm64(x, res, w):
    h = x + res if res is not None else x
    return h, h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS) * w


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["plain", "residual", "odd", "e4m3", "e4m3 residual odd"])
def test_rms_norm(lib, rows, cols, dtype, form):
    g = gen(rows * 7 + cols)
    pad, shift = (3, 1) if "odd" in form else (8, 8)
    x = Mat(rows, cols, dtype, pad, shift, rand(g, rows, cols) * torch.exp(rand(g, 1, cols)))
    res = Mat(rows, cols, dtype, pad + 2, 2 * shift, rand(g, rows, cols, 2.0)) if "residual" in form else None
    wt = "f32" if "odd" in form else dtype
    w = Mat(1, cols, wt, 0, shift, 1 + rand(g, 1, cols, 0.1))
    yt = "e4m3" if "e4m3" in form else dtype
    y = Mat(rows, cols, yt, pad, shift)
    hid = Mat(rows, cols, dtype, pad, shift) if "residual" in form else None
    sc = Mat(1, rows, "f32") if yt == "e4m3" else None
    lib.rms_norm(lib.rms_norm_desc(rows, cols, x.ptr, x.ld, w.ptr, y.ptr, y.ld, lib.DTYPES[dtype],
                                   y_dtype=lib.DTYPES[yt], weight_dtype=lib.DTYPES[wt], eps=EPS, residual=ptr(res),
                                   ldr=ld(res), hidden=ptr(hid), ldh=ld(hid), scales=ptr(sc)))
    h, want = norm64(x.f64(), res.f64() if res else None, w.f64())
    rel = ((cols / 32 + 16) / 2 + 10) * 2.0 ** -24
    if yt != "e4m3":
        within(y.t, want, (U[yt] + rel) * want.abs() + TINY[yt], "y")
    else:
        scale = (want.abs().amax(dim=1) / 448).clamp_min(2.0 ** -126)
        within(sc.t[0], scale, (rel + 2.0 ** -22) * scale, "scales")
        q = want / scale[:, None]
        # half a step of the e4m3 value (2^-10 below 2^-6), or one step where the fp32 value sits at a border
        within(y.t, q, (U["e4m3"] + 2 * rel + 2.0 ** -22) * q.abs() + TINY["e4m3"], "q")
    for m in (y, hid, sc):
        assert m is None or m.untouched_outside()
    if hid:
        within(hid.t, h, (U[dtype] + 2.0 ** -24) * h.abs() + TINY[dtype], "hidden")


def test_rms_norm_in_place(lib):
    """hidden over the residual and y over x: what a decoding loop does."""
    rows, cols = 9, 3000
    g = gen(1)
    for dtype in ("bf16", "f32"):
        for cols in (520, 3000, 20000):
            x, res = (Mat(rows, cols, dtype, fill=rand(g, rows, cols)) for _ in range(2))
            w = Mat(1, cols, dtype, fill=1 + rand(g, 1, cols, 0.1))
            h, want = norm64(x.f64(), res.f64(), w.f64())
            lib.rms_norm(lib.rms_norm_desc(rows, cols, x.ptr, x.ld, w.ptr, x.ptr, x.ld, lib.DTYPES[dtype], eps=EPS,
                                           residual=res.ptr, ldr=res.ld, hidden=res.ptr, ldh=res.ld))
            rel = ((cols / 32 + 16) / 2 + 10) * 2.0 ** -24
            within(x.t, want, (U[dtype] + rel) * want.abs() + TINY[dtype], "y")
            within(res.t, h, (U[dtype] + 2.0 ** -24) * h.abs() + TINY[dtype], "hidden")


@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_rms_norm_special_rows(lib, out):
    """A row of zeros, of the smallest and of the largest values, and rows with
    an infinity or a NaN: each stays in its own row."""
    cols = 1536
    x = torch.randn(6, cols, device="cuda").bfloat16()
    x[1] = 0
    x[2] = 1e-30
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    w = torch.ones(cols, device="cuda").bfloat16()
    y = torch.empty(6, cols, device="cuda", dtype=T[out])
    sc = torch.empty(6, device="cuda") if out == "e4m3" else None
    lib.rms_norm(lib.rms_norm_desc(6, cols, x.data_ptr(), cols, w.data_ptr(), y.data_ptr(), cols, lib.BF16,
                                   y_dtype=lib.DTYPES[out], eps=EPS, scales=None if sc is None else sc.data_ptr()))
    v = y.double()
    assert torch.isfinite(v[[0, 1, 2, 5]]).all() and (v[1] == 0).all()
    if sc is None:
        within(v[2], x[2].double() / math.sqrt(EPS), 2 * U["bf16"] * (x[2].double() / math.sqrt(EPS)).abs())
        assert torch.isnan(v[3]).all()
    else:
        assert sc[1] == 2.0 ** -126 and torch.isfinite(sc[[0, 1, 2, 5]]).all()
        assert v[2].abs().max() > 200  # a row of tiny equal values still uses the range
        assert torch.isnan(v[3]).all()
    assert torch.isnan(v[4, 7])


@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(2500, 520)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["plain", "dhidden", "odd"])
def test_rms_norm_backward(lib, rows, cols, dtype, form):
    g = gen(rows * 5 + cols)
    pad, shift = (5, 1) if form == "odd" else (8, 8)
    hid = Mat(rows, cols, dtype, pad, shift, rand(g, rows, cols) * torch.exp(rand(g, 1, cols, 0.5)))
    dy = Mat(rows, cols, dtype, pad, shift, rand(g, rows, cols))
    dh = Mat(rows, cols, dtype, pad, shift, rand(g, rows, cols)) if form != "plain" else None
    wt = "f32" if form == "odd" else dtype
    w = Mat(1, cols, wt, 0, shift, 1 + rand(g, 1, cols, 0.1))
    dx, dw = Mat(rows, cols, dtype, pad, shift), Mat(1, cols, wt, 0, shift)
    d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, dy.ld, hid.ptr, hid.ld, w.ptr, dx.ptr, dx.ld, dw.ptr,
                                   lib.DTYPES[dtype], weight_dtype=lib.DTYPES[wt], eps=EPS, dhidden=ptr(dh), lddh=ld(dh))
    lib.rms_norm_backward(d, scratch(lib, d))
    h, e, ww = hid.f64(), dy.f64(), w.f64()
    r = 1 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    first = r * e * ww
    second = r ** 3 * h * (e * ww * h).sum(1, keepdim=True) / cols
    spread = r ** 3 * h.abs() * (e * ww * h).abs().sum(1, keepdim=True) / cols
    want = first - second + (dh.f64() if dh else 0)
    rel = (1.5 * (cols / 32 + 16) + 20) * 2.0 ** -24
    within(dx.t, want, U[dtype] * want.abs() + rel * (first.abs() + spread) + 2.0 ** -23 * want.abs() + TINY[dtype], "dx")
    terms = e * h * r
    # a column is added over at most rows / 148 + 2 rows of a block and then over the blocks
    relw = rel + (min(rows, rows / 148 + 2) + 700) * 2.0 ** -24
    within(dw.t[0], terms.sum(0), U[wt] * terms.sum(0).abs() + relw * terms.abs().sum(0) + TINY[wt], "dweight")
    assert dx.untouched_outside() and dw.untouched_outside()


def test_rms_norm_backward_without_weight_gradient_and_in_place(lib):
    rows, cols = 37, 1000
    g = gen(3)
    hid, dy, dh = (Mat(rows, cols, "bf16", fill=rand(g, rows, cols)) for _ in range(3))
    w = Mat(1, cols, "bf16", fill=1 + rand(g, 1, cols, 0.1))
    one, two = Mat(rows, cols, "bf16"), Mat(1, cols, "bf16")
    d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, cols, hid.ptr, cols, w.ptr, one.ptr, cols, two.ptr, lib.BF16,
                                   dhidden=dh.ptr, lddh=cols)
    lib.rms_norm_backward(d, scratch(lib, d))
    for target in (dy, dh):
        saved = target.t.clone()
        d = lib.rms_norm_backward_desc(rows, cols, dy.ptr, cols, hid.ptr, cols, w.ptr, target.ptr, cols, None, lib.BF16,
                                       dhidden=dh.ptr, lddh=cols)
        assert lib.workspace_size(d) == 0
        lib.rms_norm_backward(d)
        assert torch.equal(target.t, one.t)
        target.t.copy_(saved)


def test_rms_norm_gradient_against_differences(lib):
    """The fp32 gradients along random directions against central differences of
    the definition in 64 bits."""
    rows, cols = 6, 777
    g = gen(9)
    x, w, dy = (rand(g, r, cols).float().double() for r in (rows, 1, rows))
    X, W, DY = (Mat(t.shape[0], cols, "f32", fill=t) for t in (x, w, dy))
    dx, dw = Mat(rows, cols, "f32"), Mat(1, cols, "f32")
    d = lib.rms_norm_backward_desc(rows, cols, DY.ptr, cols, X.ptr, cols, W.ptr, dx.ptr, cols, dw.ptr, lib.F32, eps=EPS)
    lib.rms_norm_backward(d, scratch(lib, d))
    step = 1e-5
    for _ in range(4):
        a, b = rand(g, rows, cols), rand(g, 1, cols)
        up = (norm64(x + step * a, None, w + step * b)[1] * dy).sum()
        down = (norm64(x - step * a, None, w - step * b)[1] * dy).sum()
        diff = (up - down) / (2 * step)
        got = (dx.f64() * a).sum() + (dw.f64() * b).sum()
        # the differences' own error is of step^2 = 1e-10; the kernel's of 2^-24 of the terms, added over 4662 + 777
        size = (dx.f64() * a).abs().sum() + (dw.f64() * b).abs().sum()
        assert abs(got - diff) <= 1e-5 * size


# --------------------------------------------------------------------------------------------------- products
SHAPES = [(1, 64, 64), (1, 1024, 512), (3, 8, 8), (2, 136, 1000), (16, 256, 320), (17, 200, 72), (33, 129, 257),
          (64, 512, 128), (77, 1000, 264), (130, 384, 520), (256, 1024, 512), (300, 1, 1), (1, 1, 4096), (513, 264, 136),
          (1000, 776, 200), (1300, 4104, 136), (2304, 2080, 72), (2560, 2050, 64)]


def product_inputs(g, M, N, K, dtype, trans_w, pad, shift, weights=("w",), scale=None):
    """x, the weights as stored, their values as [K, N], and the scale vectors."""
    x = Mat(M, K, dtype, pad, shift, rand(g, M, K))
    scale = K ** -0.5 if scale is None else scale
    ws, vals = [], []
    for _ in weights:
        w = rand(g, K, N, scale if dtype != "e4m3" else 1.0)
        m = Mat(N, K, dtype, pad, shift, w.t()) if trans_w else Mat(K, N, dtype, pad, shift, w)
        ws.append(m)
        vals.append(m.f64().t() if trans_w else m.f64())
    xv, xs, wss = x.f64(), None, [None] * len(ws)
    if dtype == "e4m3":
        xs = Mat(1, M, "f32", fill=torch.exp(rand(g, 1, M, 0.3)))
        wss = [Mat(1, N, "f32", fill=torch.exp(rand(g, 1, N, 0.3)) * scale) for _ in ws]
        xv = xv * xs.f64().t()
        vals = [v * s.f64() for v, s in zip(vals, wss)]
    return x, ws, xv, vals, xs, wss


def product64(xv, wv):
    """The product and its error bound before the output's rounding."""
    K = xv.shape[1]
    return xv @ wv, (K / 16 + 16) * 2.0 ** -22 * (xv.abs() @ wv.abs())


def act_bound(act, z, dz):
    a = act64(act, z)[0]
    return a, 1.13 * dz + 2.0 ** -20 * z.abs()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", False), ("bf16", True), ("f16", False), ("f16", True), ("e4m3", True)])
@pytest.mark.parametrize("form", ["plain", "all", "odd", "f32", "residual"])
def test_linear(lib, M, N, K, dtype, trans_w, form):
    g = gen(M + 3 * N + 5 * K)
    pad, shift = {"plain": (-K % 16 if trans_w else 0, 0), "odd": (3, 1)}.get(form, (16, 16))
    out = "bf16" if dtype == "e4m3" else dtype
    if form in ("odd", "f32"):
        out = "f32"
    act = {"plain": "none", "all": "gelu_tanh", "odd": "silu", "f32": "gelu", "residual": "relu"}[form]
    x, (w,), xv, (wv,), xs, (ws,) = product_inputs(g, M, N, K, dtype, trans_w, pad, shift)
    y = Mat(M, N, out, pad, shift)
    bias = Mat(1, N, out, 0, shift, rand(g, 1, N)) if form not in ("plain", "residual") else None
    res = Mat(M, N, out, pad, shift, rand(g, M, N)) if form != "plain" else None
    pre = Mat(M, N, out, pad, shift) if form in ("all", "f32") else None
    d = lib.linear_desc(M, N, K, x.ptr, x.ld, w.ptr, w.ld, y.ptr, y.ld, lib.DTYPES[dtype], y_dtype=lib.DTYPES[out],
                        trans_w=trans_w, act=lib.ACTIVATIONS[act], bias=ptr(bias), residual=ptr(res), ldr=ld(res),
                        pre=ptr(pre), ldp=ld(pre), x_scales=ptr(xs), w_scales=ptr(ws))
    lib.linear(d, scratch(lib, d))
    z, dz = product64(xv, wv)
    if bias:
        z = z + bias.f64()
        dz = dz + 2.0 ** -23 * z.abs()
    a, da = act_bound(act, z, dz)
    want = a + (res.f64() if res else 0)
    within(y.t, want, (U[out] + 2.0 ** -23) * want.abs() + da + TINY[out], "y")
    if pre:
        within(pre.t, z, U[out] * z.abs() + dz + TINY[out], "pre")
    assert y.untouched_outside() and (pre is None or pre.untouched_outside())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M", [1, 40, 700])
def test_linear_activations_and_far_values(lib, act, M):
    """Every activation over a range in which its exponentials overflow."""
    N, K = 320, 64
    g = gen(M)
    x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0, scale=16.0)
    y = Mat(M, N, "bf16")
    d = lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True, act=lib.ACTIVATIONS[act])
    lib.linear(d)
    z, dz = product64(xv, wv)
    a, da = act_bound(act, z, dz)
    within(y.t, a, U["bf16"] * a.abs() + da + TINY["bf16"], act)


def test_linear_residual_in_place(lib):
    M, N, K = 70, 520, 256
    g = gen(4)
    for M in (1, 70, 600):
        x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0)
        y = Mat(M, N, "bf16", fill=rand(g, M, N))
        r = y.f64().clone()
        lib.linear(lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True, residual=y.ptr, ldr=N))
        z, dz = product64(xv, wv)
        within(y.t, z + r, (U["bf16"] + 2.0 ** -23) * (z + r).abs() + dz, "y")


@pytest.mark.parametrize("M", [1, 20, 300, 1100])
def test_products_keep_infinities_and_nan_in_their_rows(lib, M):
    """A NaN or an infinity in one token's row reaches that row alone, whatever
    shares its tile; nothing behind the last row or column is read as a value."""
    N, K = 264, 200
    g = gen(M)
    x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0)
    r = M // 2
    x.t[r, K - 1] = float("nan")
    y = Mat(M, N, "bf16")
    lib.linear(lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True))
    bad = torch.isnan(y.t).any(dim=1)
    assert torch.isnan(y.t[r]).all() and int(bad.sum()) == 1
    x.t[r, K - 1] = float("inf")
    lib.linear(lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True))
    bad = ~torch.isfinite(y.t).all(dim=1)
    assert torch.isinf(y.t[r]).all() and int(bad.sum()) == 1


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", False), ("bf16", True), ("f16", True), ("e4m3", True)])
@pytest.mark.parametrize("form", ["plain", "saved", "odd", "f32"])
def test_gated_linear(lib, M, N, K, dtype, trans_w, form):
    g = gen(M + 2 * N + 7 * K)
    pad, shift = {"plain": (0, 0), "saved": (16, 16), "odd": (3, 1), "f32": (16, 16)}[form]
    out = "bf16" if dtype == "e4m3" else dtype
    if form in ("odd", "f32"):
        out = "f32"
    act = {"plain": "silu", "saved": "gelu", "odd": "gelu_tanh", "f32": "relu"}[form]
    x, (wg, wu), xv, (gv, uv), xs, (gs, us) = product_inputs(g, M, N, K, dtype, trans_w, pad, shift, ("wg", "wu"))
    y = Mat(M, N, out, pad, shift)
    gate, up = (Mat(M, N, out, pad, shift) if form in ("saved", "f32") else None for _ in range(2))
    d = lib.gated_linear_desc(M, N, K, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, y.ptr, y.ld, lib.DTYPES[dtype],
                              y_dtype=lib.DTYPES[out], trans_w=trans_w, act=lib.ACTIVATIONS[act], gate=ptr(gate),
                              up=ptr(up), ldp=ld(gate), x_scales=ptr(xs), wg_scales=ptr(gs), wu_scales=ptr(us))
    lib.gated_linear(d, scratch(lib, d))
    zg, dg = product64(xv, gv)
    zu, du = product64(xv, uv)
    a, da = act_bound(act, zg, dg)
    want = a * zu
    within(y.t, want, (U[out] + 2.0 ** -23) * want.abs() + da * zu.abs() + a.abs() * du + da * du + TINY[out], "y")
    if gate:
        within(gate.t, zg, U[out] * zg.abs() + dg + TINY[out], "gate")
        within(up.t, zu, U[out] * zu.abs() + du + TINY[out], "up")
        assert gate.untouched_outside() and up.untouched_outside()
    assert y.untouched_outside()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("form", ["plain", "act", "odd"])
def test_linear_backward(lib, M, N, K, dtype, trans_w, form):
    g = gen(M + 11 * N + K)
    pad, shift = (3, 1) if form == "odd" else (8, 8)
    act = {"plain": "none", "act": "gelu", "odd": "gelu_tanh"}[form]
    x, (w,), xv, (wv,), _, _ = product_inputs(g, M, N, K, dtype, trans_w, pad, shift)
    dy = Mat(M, N, dtype, pad, shift, rand(g, M, N))
    pre = Mat(M, N, dtype, pad, shift, rand(g, M, N, 2.0)) if act != "none" else None
    dx = Mat(M, K, dtype, pad, shift)
    dw = Mat(N, K, dtype, pad, shift) if trans_w else Mat(K, N, dtype, pad, shift)
    db = Mat(1, N, dtype, 0, shift)
    d = lib.linear_backward_desc(M, N, K, dy.ptr, dy.ld, x.ptr, x.ld, w.ptr, w.ld, lib.DTYPES[dtype], trans_w=trans_w,
                                 act=lib.ACTIVATIONS[act], pre=ptr(pre), ldp=ld(pre), dx=dx.ptr, lddx=dx.ld, dw=dw.ptr,
                                 lddw=dw.ld, dbias=db.ptr)
    lib.linear_backward(d, scratch(lib, d))
    dz = dy.f64()
    ddz = torch.zeros_like(dz)
    if pre:
        dz = dz * act64(act, pre.f64())[1]
        ddz = (U[dtype] + 2.0 ** -20) * dz.abs() + 2.0 ** -20 * dy.f64().abs() + TINY[dtype]
    for got, (a, da, b), name in ((dx.t, (dz, ddz, wv.t()), "dx"),
                                  (dw.t.t() if trans_w else dw.t, (dz.t(), ddz.t(), xv), "dw")):
        want, acc = product64(a, b)
        tol = U[dtype] * want.abs() + da @ b.abs() + acc + TINY[dtype]
        if name == "dw":
            want, tol = want.t(), tol.t()
        within(got, want, tol, name)
        if dtype == "bf16":
            normwise(got, want, dtype, name, (a, b))
    tol = U[dtype] * dz.sum(0).abs() + (M / 64 + 300) * 2.0 ** -24 * dz.abs().sum(0) + 2.0 ** -20 * dy.f64().abs().sum(0)
    within(db.t[0], dz.sum(0), tol + TINY[dtype], "dbias")
    assert dx.untouched_outside() and dw.untouched_outside() and db.untouched_outside()


@pytest.mark.parametrize("wanted", ["dx", "dw", "dbias", "none"])
def test_linear_backward_parts(lib, wanted):
    """Each gradient alone equals the same gradient of the whole call."""
    M, N, K = 90, 264, 136
    g = gen(5)
    x, (w,), _, _, _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0)
    dy, pre = Mat(M, N, "bf16", fill=rand(g, M, N)), Mat(M, N, "bf16", fill=rand(g, M, N))

    def call(**kw):
        d = lib.linear_backward_desc(M, N, K, dy.ptr, N, x.ptr, K, w.ptr, K, lib.BF16, trans_w=True, act=lib.ACT_SILU,
                                     pre=pre.ptr, ldp=N, **kw)
        lib.linear_backward(d, scratch(lib, d))

    whole = {"dx": Mat(M, K, "bf16"), "dw": Mat(N, K, "bf16"), "dbias": Mat(1, N, "bf16")}
    part = {k: Mat(v.t.shape[0], v.t.shape[1], "bf16", fill=torch.full_like(v.t, 9.0)) for k, v in whole.items()}
    lds = {"dx": dict(lddx=K), "dw": dict(lddw=K), "dbias": {}}
    call(dx=whole["dx"].ptr, lddx=K, dw=whole["dw"].ptr, lddw=K, dbias=whole["dbias"].ptr)
    call(**({wanted: part[wanted].ptr, **lds[wanted]} if wanted != "none" else {}))
    for k in whole:
        assert torch.equal(part[k].t, whole[k].t if k == wanted else torch.full_like(part[k].t, 9.0)), k


@pytest.mark.parametrize("M,N,K,trans_w", [(512, 1024, 128, True), (300, 1032, 200, False), (33, 4096, 520, True),
                                           (700, 129, 1001, False), (16, 72, 2056, True)])
@pytest.mark.parametrize("gated", [False, True])
def test_gradients_alone_equal_those_of_the_whole_call(lib, M, N, K, trans_w, gated):
    """Whichever products share a launch, a gradient's sums are the same."""
    g = gen(M + N + K)
    x, ws, _, _, _, _ = product_inputs(g, M, N, K, "bf16", trans_w, 0, 0, ("wg", "wu") if gated else ("w",))
    dy, gate, up = (Mat(M, N, "bf16", fill=rand(g, M, N)) for _ in range(3))
    shape = (N, K) if trans_w else (K, N)

    def call(want_dx, want_dw):
        dx = Mat(M, K, "bf16") if want_dx else None
        dws = [Mat(*shape, "bf16") for _ in ws] if want_dw else [None for _ in ws]
        kw = dict(dx=ptr(dx), lddx=K, lddw=shape[1])
        if gated:
            d = lib.gated_linear_backward_desc(M, N, K, dy.ptr, N, x.ptr, K, ws[0].ptr, ws[1].ptr, shape[1], gate.ptr,
                                               up.ptr, N, lib.BF16, trans_w=trans_w, act=lib.ACT_SILU,
                                               dwg=ptr(dws[0]), dwu=ptr(dws[1]), **kw)
            lib.gated_linear_backward(d, scratch(lib, d))
        else:
            d = lib.linear_backward_desc(M, N, K, dy.ptr, N, x.ptr, K, ws[0].ptr, shape[1], lib.BF16, trans_w=trans_w,
                                         act=lib.ACT_NONE, dw=ptr(dws[0]), **kw)
            lib.linear_backward(d, scratch(lib, d))
        return dx, dws

    dx, dws = call(True, True)
    alone, _ = call(True, False)
    assert torch.equal(dx.t, alone.t)
    _, alone = call(False, True)
    for a, b in zip(dws, alone):
        assert torch.equal(a.t, b.t)


@pytest.mark.parametrize("M", [1, 7, 8, 9, 64, 65, 130, 255, 256, 257, 449, 512, 513, 1000, 16385])
@pytest.mark.parametrize("N,act", [(1, "none"), (259, "gelu"), (2048, "relu")])
def test_bias_gradient_over_bands_of_rows(lib, M, N, act):
    """Row counts around those where the column sums change hands: whole numbers, so exact in any order."""
    g = gen(M + N)
    vals = torch.randint(-3, 4, (M, N), generator=g, device=g.device).to(torch.float32)
    dy = Mat(M, N, "f16", fill=vals)
    pre = Mat(M, N, "f16", fill=torch.where(torch.rand(M, N, generator=g, device=g.device) < 0.5, 100.0, -100.0))
    db = Mat(1, N, "f16")
    d = lib.linear_backward_desc(M, N, 8, dy.ptr, N, None, 8, None, 8, lib.F16, trans_w=True,
                                 act=lib.ACTIVATIONS[act], pre=pre.ptr if act != "none" else None, ldp=N, dbias=db.ptr)
    lib.linear_backward(d, scratch(lib, d))
    on = torch.ones_like(vals) if act == "none" else (pre.t > 0).float()  # the slope at +-100 is 1 or 0
    assert torch.equal(db.t[0], (vals * on).sum(0).to(torch.float16))
    assert db.untouched_outside()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,trans_w", [("bf16", False), ("bf16", True), ("f16", False)])
@pytest.mark.parametrize("form", ["plain", "odd"])
def test_gated_linear_backward(lib, M, N, K, dtype, trans_w, form):
    g = gen(M + 13 * N + K)
    pad, shift = (3, 1) if form == "odd" else (8, 8)
    act = "silu" if form == "plain" else "gelu_tanh"
    x, (wg, wu), xv, (gv, uv), _, _ = product_inputs(g, M, N, K, dtype, trans_w, pad, shift, ("wg", "wu"))
    dy, gate, up = (Mat(M, N, dtype, pad, shift, rand(g, M, N, s)) for s in (1.0, 2.0, 1.0))
    dx = Mat(M, K, dtype, pad, shift)
    dwg, dwu = (Mat(N, K, dtype, pad, shift) if trans_w else Mat(K, N, dtype, pad, shift) for _ in range(2))
    d = lib.gated_linear_backward_desc(M, N, K, dy.ptr, dy.ld, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, gate.ptr, up.ptr,
                                       gate.ld, lib.DTYPES[dtype], trans_w=trans_w, act=lib.ACTIVATIONS[act], dx=dx.ptr,
                                       lddx=dx.ld, dwg=dwg.ptr, dwu=dwu.ptr, lddw=dwg.ld)
    lib.gated_linear_backward(d, scratch(lib, d))
    a, s = act64(act, gate.f64())
    e = dy.f64()
    dg, du = e * up.f64() * s, e * a
    ddg = (U[dtype] + 2.0 ** -20) * dg.abs() + 2.0 ** -20 * (e * up.f64()).abs() + TINY[dtype]
    ddu = (U[dtype] + 2.0 ** -20) * du.abs() + 2.0 ** -20 * e.abs() + TINY[dtype]
    zg, ag = product64(dg, gv.t())
    zu, au = product64(du, uv.t())
    want = zg + zu
    within(dx.t, want, U[dtype] * want.abs() + ddg @ gv.t().abs() + ddu @ uv.t().abs() + 2 * (ag + au) + TINY[dtype], "dx")
    if dtype == "bf16":
        normwise(dx.t, want, dtype, "dx", (dg, gv.t()), (du, uv.t()))
    for got, v, dv, name in ((dwg, dg, ddg, "dwg"), (dwu, du, ddu, "dwu")):
        want, acc = product64(v.t(), xv)
        tol = U[dtype] * want.abs() + dv.t() @ xv.abs() + acc + TINY[dtype]
        stored = got.t if trans_w else got.t.t()
        within(stored, want, tol, name)
        if dtype == "bf16":
            normwise(stored, want, dtype, name, (v.t(), xv))
        assert got.untouched_outside()
    assert dx.untouched_outside()


@pytest.mark.parametrize("M,N,K", [(5, 132, 72), (40, 129, 200), (33, 1001, 136), (600, 132, 4104), (2048, 2052, 2056), (700, 2049, 3000)])
@pytest.mark.parametrize("trans_w", [False, True])
def test_widths_that_end_inside_an_aligned_row(lib, M, N, K, trans_w):
    """Rows padded to 16 bytes around widths that are no multiple of 8: everything
    is aligned, and still nothing past the last column may be written, nor
    anything of one weight's gradient into the other's."""
    g = gen(N)
    pad = lambda n: -n % 8 + 8  # noqa: E731
    x = Mat(M, K, "bf16", pad(K), 8, rand(g, M, K))
    shape = (N, K) if trans_w else (K, N)
    wg, wu = (Mat(*shape, "bf16", pad(shape[1]), 8, rand(g, *shape, K ** -0.5)) for _ in range(2))
    gate, up, y, dy, bias, res = (Mat(M if i < 4 or i == 5 else 1, N, "bf16", pad(N), 8, rand(g, M if i < 4 or i == 5 else 1, N))
                                  for i in range(6))
    dx = Mat(M, K, "bf16", pad(K), 8)
    dwg, dwu = (Mat(*shape, "bf16", pad(shape[1]), 8) for _ in range(2))
    z = Mat(M, N, "bf16", pad(N), 8)
    d = lib.linear_desc(M, N, K, x.ptr, x.ld, wg.ptr, wg.ld, z.ptr, z.ld, lib.BF16, trans_w=trans_w, bias=bias.ptr,
                        residual=res.ptr, ldr=res.ld)
    lib.linear(d, scratch(lib, d))
    wgv, wuv = (w.f64().t() if trans_w else w.f64() for w in (wg, wu))
    want, acc = product64(x.f64(), wgv)
    want = want + bias.f64() + res.f64()
    within(z.t, want, (U["bf16"] + 2.0 ** -22) * (want.abs() + bias.f64().abs() + res.f64().abs()) + acc, "linear")
    d = lib.gated_linear_desc(M, N, K, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, y.ptr, y.ld, lib.BF16, trans_w=trans_w,
                              gate=gate.ptr, up=up.ptr, ldp=gate.ld)
    lib.gated_linear(d, scratch(lib, d))
    zg, ag = product64(x.f64(), wgv)
    zu, au = product64(x.f64(), wuv)
    within(gate.t, zg, U["bf16"] * zg.abs() + ag, "gate")
    within(up.t, zu, U["bf16"] * zu.abs() + au, "up")
    d = lib.gated_linear_backward_desc(M, N, K, dy.ptr, dy.ld, x.ptr, x.ld, wg.ptr, wu.ptr, wg.ld, gate.ptr, up.ptr,
                                       gate.ld, lib.BF16, trans_w=trans_w, dx=dx.ptr, lddx=dx.ld, dwg=dwg.ptr,
                                       dwu=dwu.ptr, lddw=dwg.ld)
    lib.gated_linear_backward(d, scratch(lib, d))
    a, s = act64("silu", gate.f64())
    dg, du = dy.f64() * up.f64() * s, dy.f64() * a
    normwise(dx.t, dg @ wgv.t() + du @ wuv.t(), "bf16", "dx", (dg, wgv.t()), (du, wuv.t()))
    for got, v in ((dwg, dg), (dwu, du)):
        normwise(got.t if trans_w else got.t.t(), v.t() @ x.f64(), "bf16", "dw", (v.t(), x.f64()))
    for m in (z, y, gate, up, dx, dwg, dwu):
        assert m.untouched_outside()


def test_activation_slopes_at_far_values(lib):
    """dz = dy act'(pre) where exponentials overflow and z^2 exceeds fp32: with
    one output column and w = 1, dx is dz itself."""
    zs = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 30.0, -30.0, 88.0, -88.0, 1e4, -1e4, 1e20, -1e20, 3e38, -3e38],
                      device="cuda").bfloat16()
    M = zs.numel()
    pre = zs.view(M, 1).contiguous()
    one = torch.ones(M, 1, device="cuda").bfloat16()
    w = torch.ones(1, 1, device="cuda").bfloat16()
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        dx = torch.empty(M, 1, device="cuda").bfloat16()
        d = lib.linear_backward_desc(M, 1, 1, one.data_ptr(), 1, one.data_ptr(), 1, w.data_ptr(), 1, lib.BF16,
                                     trans_w=True, act=lib.ACTIVATIONS[act], pre=pre.data_ptr(), ldp=1,
                                     dx=dx.data_ptr(), lddx=1)
        lib.linear_backward(d, scratch(lib, d))
        z = zs.double()
        want = act64(act, z.clamp(-1e6, 1e6))[1]
        within(dx.view(-1), want, 2 * U["bf16"] * want.abs() + 2.0 ** -20, act)


def test_gated_gradient_against_differences(lib):
    """The gradients along random directions against central differences of the
    whole definition in 64 bits, from gate and up saved by the forward call."""
    M, N, K = 24, 40, 56
    g = gen(8)
    x, (wg, wu), xv, (gv, uv), _, _ = product_inputs(g, M, N, K, "bf16", True, 0, 0, ("wg", "wu"))
    dy, y, gate, up = (Mat(M, N, "bf16", fill=rand(g, M, N)) for _ in range(4))
    lib.gated_linear(lib.gated_linear_desc(M, N, K, x.ptr, K, wg.ptr, wu.ptr, K, y.ptr, N, lib.BF16, trans_w=True,
                                           gate=gate.ptr, up=up.ptr, ldp=N))
    dx, dwg, dwu = Mat(M, K, "bf16"), Mat(N, K, "bf16"), Mat(N, K, "bf16")
    d = lib.gated_linear_backward_desc(M, N, K, dy.ptr, N, x.ptr, K, wg.ptr, wu.ptr, K, gate.ptr, up.ptr, N, lib.BF16,
                                       trans_w=True, dx=dx.ptr, lddx=K, dwg=dwg.ptr, dwu=dwu.ptr, lddw=K)
    lib.gated_linear_backward(d, scratch(lib, d))

    def loss(x, a, b):
        return (act64("silu", x @ a)[0] * (x @ b) * dy.f64()).sum()

    step = 1e-4
    for _ in range(4):
        ex, eg, eu = rand(g, M, K), rand(g, K, N), rand(g, K, N)
        diff = (loss(xv + step * ex, gv + step * eg, uv + step * eu) - loss(xv - step * ex, gv - step * eg, uv - step * eu)) / (2 * step)
        parts = [dx.f64() * ex, dwg.f64().t() * eg, dwu.f64().t() * eu]
        got = sum(p.sum() for p in parts)
        # each gradient is off by at most 1.2 u of its norm from its own roundings and by about as much from
        # those of gate and up: 2.4 u of the norms, which the direction carries over with its own length
        room = sum(2.4 * U["bf16"] * p.norm() * math.sqrt(3.0) for p in parts)
        assert abs(got - diff) <= 3 * room


# ------------------------------------------------------------------------------------------- calls and streams
def test_no_rows(lib):
    """M = 0: gradients of the weights are zeros, everything else stays."""
    N, K = 72, 40
    y = Mat(4, N, "bf16", fill=torch.full((4, N), 5.0, device="cuda"))
    w = Mat(N, K, "bf16", fill=torch.ones(N, K, device="cuda"))
    lib.linear(lib.linear_desc(0, N, K, None, K, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True))
    lib.gated_linear(lib.gated_linear_desc(0, N, K, None, K, w.ptr, w.ptr, K, y.ptr, N, lib.BF16, trans_w=True))
    lib.rms_norm(lib.rms_norm_desc(0, N, None, N, w.ptr, y.ptr, N, lib.BF16))
    assert (y.t == 5).all()
    for trans in (True, False):
        shape = (N, K) if trans else (K, N)
        a, b, c = (Mat(*shape, "bf16", 3) for _ in range(3))
        db = Mat(1, N, "bf16")
        lib.linear_backward(lib.linear_backward_desc(0, N, K, None, N, None, K, w.ptr, a.ld, lib.BF16, trans_w=trans,
                                                     dw=a.ptr, lddw=a.ld, dbias=db.ptr))
        lib.gated_linear_backward(lib.gated_linear_backward_desc(
            0, N, K, None, N, None, K, w.ptr, w.ptr, b.ld, None, None, N, lib.BF16, trans_w=trans, dwg=b.ptr, dwu=c.ptr,
            lddw=b.ld))
        for m in (a, b, c, db):
            assert (m.t == 0).all() and m.untouched_outside()
    dw = Mat(1, N, "bf16")
    lib.rms_norm_backward(lib.rms_norm_backward_desc(0, N, None, N, None, N, w.ptr, None, N, dw.ptr, lib.BF16))
    assert (dw.t == 0).all()


def block_inputs(seed, M, D, H):
    g = gen(seed)
    t = {"x": rand(g, M, D), "res": rand(g, M, D, 2.0), "wn": 1 + rand(g, 1, D, 0.1), "wg": rand(g, H, D, D ** -0.5),
         "wu": rand(g, H, D, D ** -0.5), "wd": rand(g, D, H, H ** -0.5), "dout": rand(g, M, D)}
    return {k: v.bfloat16().contiguous() for k, v in t.items()}


def run_block(lib, t, M, D, H, keep):
    """Forward and backward of a pre-norm gated block through the library; `keep` holds every buffer."""
    def new(name, *shape):
        if name not in keep:
            keep[name] = torch.full(shape, float("nan"), device="cuda", dtype=torch.bfloat16)
        return keep[name].data_ptr()

    def call(fn, name, desc):
        if name not in keep:
            keep[name] = scratch(lib, desc)
        fn(desc, keep[name])

    p = {k: v.data_ptr() for k, v in t.items()}
    lib.rms_norm(lib.rms_norm_desc(M, D, p["x"], D, p["wn"], new("y", M, D), D, lib.BF16, residual=p["res"], ldr=D,
                                   hidden=new("h", M, D), ldh=D))
    call(lib.gated_linear, "ws0", lib.gated_linear_desc(
        M, H, D, new("y", M, D), D, p["wg"], p["wu"], D, new("a", M, H), H, lib.BF16, trans_w=True,
        gate=new("gate", M, H), up=new("up", M, H), ldp=H))
    call(lib.linear, "ws1", lib.linear_desc(M, D, H, new("a", M, H), H, p["wd"], H, new("out", M, D), D, lib.BF16,
                                            trans_w=True, residual=new("h", M, D), ldr=D))
    call(lib.linear_backward, "ws2", lib.linear_backward_desc(
        M, D, H, p["dout"], D, new("a", M, H), H, p["wd"], H, lib.BF16, trans_w=True, dx=new("da", M, H), lddx=H,
        dw=new("dwd", D, H), lddw=H))
    call(lib.gated_linear_backward, "ws3", lib.gated_linear_backward_desc(
        M, H, D, new("da", M, H), H, new("y", M, D), D, p["wg"], p["wu"], D, new("gate", M, H), new("up", M, H), H,
        lib.BF16, trans_w=True, dx=new("dyn", M, D), lddx=D, dwg=new("dwg", H, D), dwu=new("dwu", H, D), lddw=D))
    call(lib.rms_norm_backward, "ws4", lib.rms_norm_backward_desc(
        M, D, new("dyn", M, D), D, new("h", M, D), D, p["wn"], new("dx", M, D), D, new("dwn", 1, D), lib.BF16,
        dhidden=p["dout"], lddh=D))
    return keep


def block64(t):
    v = {k: x.double().requires_grad_(k != "dout") for k, x in t.items()}
    h = v["x"] + v["res"]
    y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS) * v["wn"]
    g, u = y @ v["wg"].t(), y @ v["wu"].t()
    out = (g / (1 + torch.exp(-g)) * u) @ v["wd"].t() + h
    out.backward(v["dout"])
    return {"out": out.detach(), "dx": v["x"].grad, "dwn": v["wn"].grad, "dwg": v["wg"].grad, "dwu": v["wu"].grad,
            "dwd": v["wd"].grad}


@pytest.mark.parametrize("M,D,H", [(1, 256, 512), (50, 264, 520), (600, 512, 1024)])
def test_a_whole_block_forward_and_backward(lib, M, D, H):
    """Norm, gated pair, projection back with the residual, and all gradients, in
    a row as a training step runs them, against autograd on the definition in
    64 bits. Each intermediate is stored once in bf16: at most 9 roundings lie
    on the way to any output, each of at most u (over a matrix u / sqrt(3)), so
    norm-wise an output is off by sqrt(9) u / sqrt(3) < 1.8 u; 3 u bounds it."""
    t = block_inputs(M, M, D, H)
    keep = run_block(lib, t, M, D, H, {})
    for k, want in block64(t).items():
        err = float((keep[k].double() - want).norm() / want.norm())
        assert err <= 3 * U["bf16"], (k, err)


def test_block_in_eight_bits(lib):
    """The serving form: the norm writes e4m3 with row scales, the gated pair and
    the projection read e4m3 weights with column scales. Against the definition
    in 64 bits on the same quantised weights; the activations' two roundings to
    e4m3 (u = 2^-4, over a matrix u / sqrt(3)) bound the result norm-wise by
    2 u: sqrt(2 + 1) u / sqrt(3) with the gate's own slope."""
    M, D, H = 7, 512, 1024
    t = block_inputs(2, M, D, H)

    def quantised(w):
        s = w.double().abs().amax(dim=1) / 448
        return (w.double() / s[:, None]).float().to(T["e4m3"]), s.float()

    q = {k: quantised(t[k]) for k in ("wg", "wu", "wd")}
    y8, s8 = torch.empty(M, D, device="cuda", dtype=T["e4m3"]), torch.empty(M, device="cuda")
    h, a, out = (torch.empty(M, n, device="cuda", dtype=torch.bfloat16) for n in (D, H, D))
    a8, sa = torch.empty(M, H, device="cuda", dtype=T["e4m3"]), torch.empty(M, device="cuda")
    lib.rms_norm(lib.rms_norm_desc(M, D, t["x"].data_ptr(), D, t["wn"].data_ptr(), y8.data_ptr(), D, lib.BF16,
                                   y_dtype=lib.E4M3, residual=t["res"].data_ptr(), ldr=D, hidden=h.data_ptr(), ldh=D,
                                   scales=s8.data_ptr()))
    lib.gated_linear(lib.gated_linear_desc(M, H, D, y8.data_ptr(), D, q["wg"][0].data_ptr(), q["wu"][0].data_ptr(), D,
                                           a.data_ptr(), H, lib.E4M3, y_dtype=lib.BF16, trans_w=True,
                                           x_scales=s8.data_ptr(), wg_scales=q["wg"][1].data_ptr(),
                                           wu_scales=q["wu"][1].data_ptr()))
    sa.copy_((a.float().abs().amax(dim=1) / 448).clamp_min(2.0 ** -126))
    a8.copy_(a.float() / sa[:, None])
    lib.linear(lib.linear_desc(M, D, H, a8.data_ptr(), H, q["wd"][0].data_ptr(), H, out.data_ptr(), D, lib.E4M3,
                               y_dtype=lib.BF16, trans_w=True, residual=h.data_ptr(), ldr=D, x_scales=sa.data_ptr(),
                               w_scales=q["wd"][1].data_ptr()))
    w = {k: v.double() * s.double()[:, None] for k, (v, s) in q.items()}
    hh, y = norm64(t["x"].double(), t["res"].double(), t["wn"].double())
    g, u = y @ w["wg"].t(), y @ w["wu"].t()
    add = (g * torch.sigmoid(g) * u) @ w["wd"].t()
    err = float((out.double() - hh - add).norm() / add.norm())
    assert err <= 2 * U["e4m3"], err


def test_capture_and_replay_with_new_inputs(lib):
    """The whole block recorded into a CUDA graph and replayed on other inputs
    and after the workspace was overwritten: the same bits as direct calls."""
    M, D, H = 130, 256, 512
    t = block_inputs(1, M, D, H)
    keep = run_block(lib, t, M, D, H, {})
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        try:
            with torch.cuda.graph(graph, stream=side):
                lib.set_stream(side.cuda_stream)
                run_block(lib, t, M, D, H, keep)
        finally:
            lib.set_stream(torch.cuda.default_stream().cuda_stream)
    other = block_inputs(2, M, D, H)
    want = {k: v.clone() for k, v in run_block(lib, other, M, D, H, {}).items() if v is not None and not k.startswith("ws")}
    for k in t:
        t[k].copy_(other[k])
    for k, v in keep.items():
        if v is not None:
            v.fill_(255 if k.startswith("ws") else float("nan"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for k, v in want.items():
        assert torch.equal(keep[k], v), k


_FIRST_IN_A_CAPTURE = r"""
import sys, torch
sys.path.insert(0, %r)
sys.path.insert(0, %r)
import test_ffn_gpu as t
from tt_lazy_b200 import capi as lib
lib.init(0)
M, D, H = 300, 256, 2560
x = t.block_inputs(1, M, D, H)
keep = {}
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.stream(side):
    with torch.cuda.graph(graph, stream=side):
        lib.set_stream(side.cuda_stream)
        t.run_block(lib, x, M, D, H, keep)
lib.set_stream(torch.cuda.default_stream().cuda_stream)
graph.replay()
torch.cuda.synchronize()
got = {k: v.clone() for k, v in keep.items() if v is not None and not k.startswith("ws")}
want = t.run_block(lib, x, M, D, H, {})
lib.synchronize()
assert all(torch.equal(v, want[k]) for k, v in got.items())
print("equal", len(got))
"""


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing that a first call sets up is refused while a stream is being captured."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", _FIRST_IN_A_CAPTURE % (os.path.dirname(here), here)], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_offsets_past_32_bits(lib):
    """Tensors of more than 2^31 elements: rows from their far end against the same
    rows computed in a small call."""
    torch.cuda.empty_cache()
    rows, cols = 270_000, 8192
    x = torch.randn(1000, cols, device="cuda").bfloat16().repeat(rows // 1000, 1)
    y, hidden = torch.empty_like(x), torch.empty_like(x)
    w = torch.randn(cols, device="cuda").bfloat16()
    assert x.numel() > 2 ** 31

    def norm(x, y, h):
        lib.rms_norm(lib.rms_norm_desc(x.shape[0], cols, x.data_ptr(), cols, w.data_ptr(), y.data_ptr(), cols, lib.BF16,
                                       residual=x.data_ptr(), ldr=cols, hidden=h.data_ptr(), ldh=cols))

    norm(x, y, hidden)
    small_y, small_h = torch.empty_like(x[:1000]), torch.empty_like(x[:1000])
    norm(x[:1000], small_y, small_h)
    for k in (0, rows // 1000 - 1):
        assert torch.equal(y[k * 1000:(k + 1) * 1000], small_y) and torch.equal(hidden[k * 1000:(k + 1) * 1000], small_h)
    dx, small_dx = y, small_y

    def back(x, dx):
        d = lib.rms_norm_backward_desc(x.shape[0], cols, x.data_ptr(), cols, x.data_ptr(), cols, w.data_ptr(),
                                       dx.data_ptr(), cols, None, lib.BF16, dhidden=x.data_ptr(), lddh=cols)
        lib.rms_norm_backward(d)

    back(x, dx)
    back(x[:1000], small_dx)
    assert torch.equal(dx[-1000:], small_dx)
    # a product with a far x, and one with a far y
    N = 72
    wn = (torch.randn(N, cols, device="cuda") / 90).bfloat16()
    out = torch.empty(rows, N, device="cuda", dtype=torch.bfloat16)
    lib.linear(lib.linear_desc(rows, N, cols, x.data_ptr(), cols, wn.data_ptr(), cols, out.data_ptr(), N, lib.BF16,
                               trans_w=True))
    want = x[:1000].double() @ wn.double().t()
    bound = U["bf16"] * want.abs() + (cols / 16 + 16) * 2.0 ** -22 * (x[:1000].double().abs() @ wn.double().abs().t())
    within(out[-1000:], want, bound, "far x")
    del hidden, out
    K = 64
    a = torch.randn(1000, K, device="cuda").bfloat16().repeat(rows // 1000, 1)
    wk = torch.randn(cols, K, device="cuda").bfloat16()
    bias = torch.randn(cols, device="cuda").bfloat16()
    for residual in (None, x):
        lib.linear(lib.linear_desc(rows, cols, K, a.data_ptr(), K, wk.data_ptr(), K, y.data_ptr(), cols, lib.BF16,
                                   trans_w=True, bias=bias.data_ptr(),
                                   residual=None if residual is None else residual.data_ptr(), ldr=cols))
        want = a[:1000].double() @ wk.double().t() + bias.double()
        acc = (K / 16 + 16) * 2.0 ** -22 * (a[:1000].double().abs() @ wk.double().abs().t()) + 2.0 ** -22 * want.abs()
        want = want + (0 if residual is None else x[:1000].double())
        within(y[-1000:], want, (U["bf16"] + 2.0 ** -23) * want.abs() + acc, "far y")
    del x, y, a, dx
    torch.cuda.empty_cache()


def test_two_streams_at_once(lib):
    """Calls queued on two streams with their own buffers do not disturb each other."""
    M, D, H = 40, 512, 1024
    sets = [(block_inputs(i, M, D, H), {}, torch.cuda.Stream()) for i in (10, 11)]
    want = [{k: v.clone() for k, v in run_block(lib, t, M, D, H, {}).items() if v is not None and not k.startswith("ws")}
            for t, _, _ in sets]
    for t, keep, _ in sets:
        run_block(lib, t, M, D, H, keep)
    torch.cuda.synchronize()
    try:
        for _ in range(20):
            for t, keep, stream in sets:
                lib.set_stream(stream.cuda_stream)
                run_block(lib, t, M, D, H, keep)
    finally:
        lib.set_stream(torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    for w, (_, keep, _) in zip(want, sets):
        for k, v in w.items():
            assert torch.equal(keep[k], v), k


def test_results_do_not_change_from_call_to_call(lib):
    M, D, H = 333, 520, 776
    t = block_inputs(3, M, D, H)
    first = {k: v.clone() for k, v in run_block(lib, t, M, D, H, {}).items() if v is not None and not k.startswith("ws")}
    for _ in range(5):
        again = run_block(lib, t, M, D, H, {})
        for k, v in first.items():
            assert torch.equal(again[k], v), k


@pytest.mark.parametrize("M,N,K", [(4, 256, 512), (2048, 2560, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_wait_expiry_is_reported_and_the_context_stays_usable(lib, monkeypatch, M, N, K, dtype):
    """Both product kernels with their loads left out (TTC_TEST_STALL=linear: nothing
    is ever in flight): the bounded waits run out after about a millisecond, the
    next synchronisation reports it, and the same call then runs."""
    g = gen(6)
    x, (w,), xv, (wv,), xs, (ws,) = product_inputs(g, M, N, K, dtype, True, 0, 0)
    y = Mat(M, N, "bf16")
    d = lib.linear_desc(M, N, K, x.ptr, K, w.ptr, K, y.ptr, N, lib.DTYPES[dtype], y_dtype=lib.BF16, trans_w=True,
                        x_scales=ptr(xs), w_scales=ptr(ws))
    torch.cuda.synchronize()
    monkeypatch.setenv("TTC_TEST_STALL", "linear")
    lib.linear(d)
    with pytest.raises(lib.TTCError) as e:
        lib.synchronize()
    assert e.value.code == lib.ERR_TIMEOUT and "bounded wait expired" in str(e.value)
    monkeypatch.delenv("TTC_TEST_STALL")
    lib.synchronize()
    lib.linear(d)
    z, dz = product64(xv, wv)
    within(y.t, z, (U["bf16"] + 2.0 ** -23) * z.abs() + dz + TINY["bf16"], "y")


def test_library_buffers_in_sixteen_bits(ttc):
    """DeviceArray with 16-bit elements, on the library's own stream, without torch."""
    ttc.set_stream(None)
    rng = np.random.default_rng(0)
    M, N, K = 5, 64, 96
    x, w = rng.standard_normal((M, K)).astype(np.float16), (rng.standard_normal((K, N)) / 10).astype(np.float16)
    X, W = ttc.DeviceArray.from_numpy(x, np.float16), ttc.DeviceArray.from_numpy(w, np.float16)
    Y = ttc.DeviceArray.zeros((M, N), np.float16)
    ttc.linear(ttc.linear_desc(M, N, K, X.ptr, K, W.ptr, N, Y.ptr, N, ttc.F16))
    want = x.astype(np.float64) @ w.astype(np.float64)
    tol = U["f16"] * np.abs(want) + (K / 16 + 16) * 2.0 ** -22 * (np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64)))
    assert np.all(np.abs(Y.numpy().astype(np.float64) - want) <= tol + TINY["f16"])
    assert C.sizeof(ttc.LinearDesc) > 0
