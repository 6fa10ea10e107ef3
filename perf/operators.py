"""The feed-forward block's operators in 16 and 8 bits, as cases to time and to compare.

Three operators, each in the directions that a program calls it in:

* ``norm``           root-mean-square norm of ``x + residual``, with a 16/32-bit output or an e4m3 output and a scale per row
* ``norm_backward``  its gradients: of the input (with the residual stream's own gradient added) and of the weight
* ``linear``         act(x W + b) + residual, from 16-bit operands or e4m3 operands with row and column scales
* ``linear_backward``  its gradients: dx, dW, db, from the saved pre-activation
* ``gated``          act(x Wg) * (x Wu), from the same kinds of operands
* ``gated_backward``   its gradients: dx, dWg, dWu, from the saved gate and up products

With ``own`` false, ``run`` computes them with elementary torch operations in 32 bits; with ``own`` true it calls
``tt_lazy_b200.capi``. ``exact`` computes them again from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
EPS = 1e-6
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # serving, one token: the residual stream's norm that feeds an 8-bit projection; latency alone counts
        dict(name="norm one token e4m3", op="norm", rows=1, cols=4096, dtype="bf16", out="e4m3", residual=True),
        # a prompt, or a training batch: memory bandwidth
        dict(name="norm prompt", op="norm", rows=8192, cols=4096, dtype="bf16", out="bf16", residual=True),
        # training: both gradients, the residual stream's own gradient added
        dict(name="norm backward training", op="norm_backward", rows=16384, cols=4096, dtype="bf16", residual=True),
        # the framework's own type, a ragged batch with rows that end inside a vector block
        dict(name="norm backward f32 ragged", op="norm_backward", rows=4099, cols=1000, dtype="f32", residual=False),
        # serving, one token: the projection back to the model's width, with the residual; reads the weights once
        dict(name="linear one token", op="linear", m=1, n=4096, k=16384, dtype="bf16", out="bf16", act="none", bias=False,
             residual=True, trans_w=True),
        # the small network of the benchmark's own set, weights stored [in, out]
        dict(name="linear small network", op="linear", m=256, n=1024, k=512, dtype="f16", out="f16", act="gelu_tanh", bias=True,
             residual=False, trans_w=False),
        # a prompt through 8-bit weights and activations
        dict(name="linear prompt e4m3", op="linear", m=4096, n=4096, k=16384, dtype="e4m3", out="bf16", act="none", bias=False,
             residual=True, trans_w=True),
        # training: three gradients of a projection with bias and activation
        dict(name="linear backward training", op="linear_backward", m=8192, n=16384, k=4096, dtype="bf16", act="gelu",
             bias=True, trans_w=True),
        # serving, a few sequences' single tokens
        dict(name="gated four tokens", op="gated", m=4, n=16384, k=4096, dtype="bf16", out="bf16", act="silu", trans_w=True),
        # serving, a ragged batch of tokens in 8 bits
        dict(name="gated ragged batch e4m3", op="gated", m=77, n=16384, k=4096, dtype="e4m3", out="bf16", act="silu",
             trans_w=True),
        # a long prompt, or the forward pass of training, weights stored [in, out]
        dict(name="gated prompt", op="gated", m=8191, n=16384, k=4096, dtype="bf16", out="bf16", act="silu", trans_w=False),
        # training: three gradients of the gated pair
        dict(name="gated backward training", op="gated_backward", m=4096, n=16384, k=4096, dtype="bf16", act="silu",
             trans_w=True),
    ]


def _size(rng, low, high, odd=0.25):
    """A size whose logarithm is uniform over [low, high]: a multiple of 8, or (one time in four) any number."""
    s = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return s if rng.random() < odd else min(high, max(8, 8 * round(s / 8)))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "linear", "linear_backward", "gated", "gated_backward"])
    if op in ("norm", "norm_backward"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        cols = _size(rng, 256, 16384)
        rows = _size(rng, 1, min(16384, 16384 * 4096 // cols), odd=0.75)
        if op == "norm":
            return dict(op=op, rows=rows, cols=cols, dtype=dtype, out=rng.choice([dtype, dtype, "e4m3"]), residual=rng.random() < 0.7)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7)
    n, k = _size(rng, 256, 16384), _size(rng, 256, 16384)
    pair = 2 if op.startswith("gated") else 1
    # 2 m n k operations a product; a backward pass makes two products of each forward one
    most = int(8191 * 16384 * 4096 * 2 // (n * k * pair * (2 if op.endswith("backward") else 1)))
    m = _size(rng, 1, max(1, min(8192, most)), odd=0.75)
    dtype = rng.choice(["bf16", "bf16", "f16"] + ([] if op.endswith("backward") else ["e4m3"]))
    case = dict(op=op, m=m, n=n, k=k, dtype=dtype, trans_w=True if dtype == "e4m3" else rng.random() < 0.5)
    if op == "linear":
        return dict(case, out="bf16" if dtype == "e4m3" else dtype, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    if op == "linear_backward":
        return dict(case, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.5)
    case["act"] = rng.choice(["silu", "silu", "gelu_tanh", "gelu", "relu"])
    return dict(case, out="bf16" if dtype == "e4m3" else dtype) if op == "gated" else case


# --------------------------------------------------------------------------------------------------- inputs
def _quantised(t):
    """t in e4m3 with one scale per row (an activation) or per output column (a weight stored [out, in]): both are rows here."""
    s = (t.abs().amax(dim=1) / E4M3_MAX).clamp_min(MIN_SCALE)
    return (t / s[:, None]).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = "cuda"

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype or t)

    s = {"case": dict(case)}
    t = DTYPES[case["dtype"]]
    if case["op"] in ("norm", "norm_backward"):
        rows, cols = case["rows"], case["cols"]
        spread = torch.exp(0.5 * torch.randn(cols, generator=g, device=dev))  # channels differ in size, as hidden states do
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device=dev)).to(t)
        x = (torch.randn(rows, cols, generator=g, device=dev) * spread).to(t)
        if case["op"] == "norm":
            s["x"] = x
            s["residual"] = normal(rows, cols, scale=2.0) if case["residual"] else None
            s["y"] = torch.empty(rows, cols, dtype=DTYPES[case["out"]], device=dev)
            s["hidden"] = torch.empty_like(x) if case["residual"] else None
            s["scales"] = torch.empty(rows, dtype=torch.float32, device=dev) if case["out"] == "e4m3" else None
        else:
            s["hidden"] = x
            s["dy"] = normal(rows, cols, scale=0.01)
            s["dhidden"] = normal(rows, cols, scale=0.01) if case["residual"] else None
            s["dx"] = torch.empty_like(x)
            s["dweight"] = torch.empty_like(s["weight"])
        return s
    m, n, k = case["m"], case["n"], case["k"]
    out = DTYPES[case.get("out", case["dtype"])]

    def weight(name):
        w = torch.randn(n, k, generator=g, device=dev) * k ** -0.5
        if case["dtype"] == "e4m3":
            s[name], s[name + "_scales"] = _quantised(w)
        else:
            s[name] = (w if case["trans_w"] else w.t().contiguous()).to(t)

    if case["dtype"] == "e4m3":
        s["x"], s["x_scales"] = _quantised(torch.randn(m, k, generator=g, device=dev))
    else:
        s["x"] = normal(m, k)
    if case["op"] == "linear":
        weight("w")
        s["bias"] = normal(n, scale=0.1, dtype=out) if case["bias"] else None
        s["residual"] = normal(m, n, dtype=out) if case["residual"] else None
        s["y"] = torch.empty(m, n, dtype=out, device=dev)
    elif case["op"] == "linear_backward":
        weight("w")
        s["pre"] = normal(m, n) if case["act"] != "none" else None
        s["dy"] = normal(m, n, scale=0.01)
        s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
        s["dbias"] = torch.empty(n, dtype=t, device=dev) if case["bias"] else None
    else:
        weight("wg")
        weight("wu")
        if case["op"] == "gated":
            s["y"] = torch.empty(m, n, dtype=out, device=dev)
        else:
            s["gate"], s["up"] = normal(m, n), normal(m, n)
            s["dy"] = normal(m, n, scale=0.01)
            s["dx"], s["dwg"], s["dwu"] = torch.empty_like(s["x"]), torch.empty_like(s["wg"]), torch.empty_like(s["wu"])
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _act(act, z):
    if act == "relu":
        return torch.clamp_min(z, 0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        h = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _norm_plain(s, case):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    hidden = h.to(s["x"].dtype) if s["residual"] is not None else None
    if s["scales"] is None:
        return {"y": y.to(s["y"].dtype), "hidden": hidden}
    scales = (y.abs().amax(dim=1) / E4M3_MAX).clamp_min(MIN_SCALE)
    return {"y": (y * (1 / scales)[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(s["y"].dtype), "hidden": hidden, "scales": scales}


def _norm_backward_plain(s, case):
    h, dy = s["hidden"].float(), s["dy"].float()
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    xhat = h * rstd
    dxhat = dy * s["weight"].float()
    dx = rstd * (dxhat - xhat * (dxhat * xhat).mean(dim=1, keepdim=True))
    if s["dhidden"] is not None:
        dx = dx + s["dhidden"].float()
    return {"dx": dx.to(s["dx"].dtype), "dweight": (dy * xhat).sum(dim=0).to(s["dweight"].dtype)}


def _product(s, case, name):
    w = s[name].float()
    z = s["x"].float() @ (w.t() if case["trans_w"] else w)
    return z * s["x_scales"][:, None] * s[name + "_scales"] if case["dtype"] == "e4m3" else z


def _linear_plain(s, case):
    z = _product(s, case, "w")
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(case["act"], z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(s["y"].dtype)}


def _linear_backward_plain(s, case):
    dz, x, w = s["dy"].float(), s["x"].float(), s["w"].float()
    if s["pre"] is not None:
        dz = dz * _act_slope(case["act"], s["pre"].float())
    dx = dz @ (w if case["trans_w"] else w.t())
    dw = dz.t() @ x if case["trans_w"] else x.t() @ dz
    dbias = dz.sum(dim=0).to(s["dbias"].dtype) if s["dbias"] is not None else None
    return {"dx": dx.to(s["dx"].dtype), "dw": dw.to(s["dw"].dtype), "dbias": dbias}


def _gated_plain(s, case):
    return {"y": (_act(case["act"], _product(s, case, "wg")) * _product(s, case, "wu")).to(s["y"].dtype)}


def _gated_backward_plain(s, case):
    dy, g, u, x = s["dy"].float(), s["gate"].float(), s["up"].float(), s["x"].float()
    dg, du = dy * u * _act_slope(case["act"], g), dy * _act(case["act"], g)
    wg, wu = s["wg"].float(), s["wu"].float()
    if case["trans_w"]:
        dx, dwg, dwu = dg @ wg + du @ wu, dg.t() @ x, du.t() @ x
    else:
        dx, dwg, dwu = dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du
    return {"dx": dx.to(s["dx"].dtype), "dwg": dwg.to(s["dwg"].dtype), "dwu": dwu.to(s["dwu"].dtype)}


# ------------------------------------------------------------------------------------- the framework's calls
_capi = None


def _library():
    """tt_lazy_b200.capi, initialised once on torch's device and set to torch's stream, as a program does at its start."""
    global _capi
    if _capi is None:
        from tt_lazy_b200 import capi

        capi.init(torch.cuda.current_device())
        capi.set_stream(torch.cuda.current_stream().cuda_stream)
        _capi = capi
    return _capi


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(capi, desc):
    size = capi.workspace_size(desc)
    return torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


def _norm_own(s, case):
    c, rows, cols = _library(), case["rows"], case["cols"]
    c.rms_norm(c.rms_norm_desc(
        rows, cols, _ptr(s["x"]), cols, _ptr(s["weight"]), _ptr(s["y"]), cols, dtype=c.DTYPES[case["dtype"]], y_dtype=c.DTYPES[case["out"]],
        eps=EPS, residual=_ptr(s["residual"]), ldr=cols, hidden=_ptr(s["hidden"]), ldh=cols, scales=_ptr(s["scales"])))
    out = {"y": s["y"], "hidden": s["hidden"]}
    return dict(out, scales=s["scales"]) if s["scales"] is not None else out


def _norm_backward_own(s, case):
    c, rows, cols = _library(), case["rows"], case["cols"]
    d = c.rms_norm_backward_desc(
        rows, cols, _ptr(s["dy"]), cols, _ptr(s["hidden"]), cols, _ptr(s["weight"]), _ptr(s["dx"]), cols, _ptr(s["dweight"]),
        dtype=c.DTYPES[case["dtype"]], eps=EPS, dhidden=_ptr(s["dhidden"]), lddh=cols)
    c.rms_norm_backward(d, _workspace(c, d))
    return {"dx": s["dx"], "dweight": s["dweight"]}


def _linear_own(s, case):
    c, m, n, k = _library(), case["m"], case["n"], case["k"]
    d = c.linear_desc(
        m, n, k, _ptr(s["x"]), k, _ptr(s["w"]), k if case["trans_w"] else n, _ptr(s["y"]), n, dtype=c.DTYPES[case["dtype"]],
        y_dtype=c.DTYPES[case["out"]], trans_w=case["trans_w"], act=c.ACTIVATIONS[case["act"]], bias=_ptr(s["bias"]),
        residual=_ptr(s["residual"]), ldr=n, x_scales=_ptr(s.get("x_scales")), w_scales=_ptr(s.get("w_scales")))
    c.linear(d, _workspace(c, d))
    return {"y": s["y"]}


def _linear_backward_own(s, case):
    c, m, n, k = _library(), case["m"], case["n"], case["k"]
    ldw = k if case["trans_w"] else n
    d = c.linear_backward_desc(
        m, n, k, _ptr(s["dy"]), n, _ptr(s["x"]), k, _ptr(s["w"]), ldw, dtype=c.DTYPES[case["dtype"]], trans_w=case["trans_w"],
        act=c.ACTIVATIONS[case["act"]], pre=_ptr(s["pre"]), ldp=n, dx=_ptr(s["dx"]), lddx=k, dw=_ptr(s["dw"]), lddw=ldw,
        dbias=_ptr(s["dbias"]))
    c.linear_backward(d, _workspace(c, d))
    return {"dx": s["dx"], "dw": s["dw"], "dbias": s["dbias"]}


def _gated_own(s, case):
    c, m, n, k = _library(), case["m"], case["n"], case["k"]
    d = c.gated_linear_desc(
        m, n, k, _ptr(s["x"]), k, _ptr(s["wg"]), _ptr(s["wu"]), k if case["trans_w"] else n, _ptr(s["y"]), n,
        dtype=c.DTYPES[case["dtype"]], y_dtype=c.DTYPES[case["out"]], trans_w=case["trans_w"], act=c.ACTIVATIONS[case["act"]],
        x_scales=_ptr(s.get("x_scales")), wg_scales=_ptr(s.get("wg_scales")), wu_scales=_ptr(s.get("wu_scales")))
    c.gated_linear(d, _workspace(c, d))
    return {"y": s["y"]}


def _gated_backward_own(s, case):
    c, m, n, k = _library(), case["m"], case["n"], case["k"]
    ldw = k if case["trans_w"] else n
    d = c.gated_linear_backward_desc(
        m, n, k, _ptr(s["dy"]), n, _ptr(s["x"]), k, _ptr(s["wg"]), _ptr(s["wu"]), ldw, _ptr(s["gate"]), _ptr(s["up"]), n,
        dtype=c.DTYPES[case["dtype"]], trans_w=case["trans_w"], act=c.ACTIVATIONS[case["act"]], dx=_ptr(s["dx"]), lddx=k,
        dwg=_ptr(s["dwg"]), dwu=_ptr(s["dwu"]), lddw=ldw)
    c.gated_linear_backward(d, _workspace(c, d))
    return {"dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"]}


PLAIN = {"norm": _norm_plain, "norm_backward": _norm_backward_plain, "linear": _linear_plain, "linear_backward": _linear_backward_plain,
         "gated": _gated_plain, "gated_backward": _gated_backward_plain}
OWN = {"norm": _norm_own, "norm_backward": _norm_backward_own, "linear": _linear_own, "linear_backward": _linear_backward_own,
       "gated": _gated_own, "gated_backward": _gated_backward_own}


def run(state):
    case = state["case"]
    return (OWN if own else PLAIN)[case["op"]](state, case)


# ------------------------------------------------------------------------------------------------------ work
def work(case):
    op, e = case["op"], SIZES[case["dtype"]]
    if op == "norm":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * (e * (3 if case["residual"] else 1) + SIZES[case["out"]]) + c * e + (4 * r if case["out"] == "e4m3" else 0),
                "flops": r * c * 5}
    if op == "norm_backward":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * e * (4 if case["residual"] else 3) + 2 * c * e, "flops": r * c * 12}
    m, n, k, o = case["m"], case["n"], case["k"], SIZES[case.get("out", case["dtype"])]
    if op == "linear":
        scales = 4 * (m + n) if case["dtype"] == "e4m3" else 0
        return {"bytes": e * (m * k + k * n) + o * (m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)) + scales,
                "flops": 2 * m * n * k}
    if op == "linear_backward":
        return {"bytes": e * (m * n * (1 if case["act"] == "none" else 2) + 2 * m * k + 2 * n * k + (n if case["bias"] else 0)),
                "flops": 4 * m * n * k}
    if op == "gated":
        scales = 4 * (m + 2 * n) if case["dtype"] == "e4m3" else 0
        return {"bytes": e * (m * k + 2 * k * n) + o * m * n + scales, "flops": 4 * m * n * k}
    return {"bytes": e * (3 * m * n + 2 * m * k + 4 * n * k), "flops": 8 * m * n * k}


# ----------------------------------------------------------------------------------- the definitions, 64 bits
def _phi(z):
    """The normal distribution's density and distribution at z."""
    return torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi), torch.special.ndtr(z)


def _act64(act, z):
    """(the activation, its derivative) of z."""
    if act == "relu":
        on = z > 0
        return torch.where(on, z, 0.0), on.double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        density, dist = _phi(z)
        return z * dist, dist + z * density
    if act == "gelu_tanh":  # 0.5 (1 + tanh t) = sigmoid(2 t)
        a = math.sqrt(8 / math.pi)
        p = torch.sigmoid(a * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * a * (1 + 0.134145 * z ** 2)
    return z, torch.ones_like(z)


def _values(s, name, case):
    """A stored operand as the values it stands for, weights as [out, in]."""
    v = s[name].double()
    if name == "x" or case["trans_w"]:
        return v * s[name + "_scales"].double().unsqueeze(1) if case["dtype"] == "e4m3" else v
    return v.T


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0)
        y = s["weight"].double() * (h / torch.sqrt(h.square().sum(1, keepdim=True) / case["cols"] + EPS))
        hidden = h if case["residual"] else None
        if case["out"] != "e4m3":
            return {"y": y, "hidden": hidden}
        scales = torch.clamp(y.abs().max(1).values / E4M3_MAX, min=MIN_SCALE)
        return {"y": (y / scales.unsqueeze(1)).float().to(torch.float8_e4m3fn).double(), "hidden": hidden, "scales": scales}
    if op == "norm_backward":
        h, dy, w = s["hidden"].double(), s["dy"].double(), s["weight"].double()
        n = case["cols"]
        r = 1 / torch.sqrt(h.square().sum(1, keepdim=True) / n + EPS)
        dx = r * dy * w - r ** 3 / n * h * (dy * w * h).sum(1, keepdim=True)
        return {"dx": dx + s["dhidden"].double() if case["residual"] else dx, "dweight": (dy * h * r).sum(0)}
    x = _values(s, "x", case)
    if op == "linear":
        z = torch.einsum("mk,nk->mn", x, _values(s, "w", case))
        if case["bias"]:
            z = z + s["bias"].double()
        y = _act64(case["act"], z)[0]
        return {"y": y + s["residual"].double() if case["residual"] else y}
    if op == "linear_backward":
        dz, w = s["dy"].double(), _values(s, "w", case)
        if case["act"] != "none":
            dz = dz * _act64(case["act"], s["pre"].double())[1]
        dw = torch.einsum("mn,mk->nk", dz, x)
        return {"dx": torch.einsum("mn,nk->mk", dz, w), "dw": (dw if case["trans_w"] else dw.T).contiguous(),
                "dbias": dz.sum(0) if case["bias"] else None}
    wg, wu = _values(s, "wg", case), _values(s, "wu", case)
    if op == "gated":
        return {"y": _act64(case["act"], torch.einsum("mk,nk->mn", x, wg))[0] * torch.einsum("mk,nk->mn", x, wu)}
    a, da = _act64(case["act"], s["gate"].double())
    dy = s["dy"].double()
    dg, du = dy * s["up"].double() * da, dy * a
    dx = torch.einsum("mn,nk->mk", dg, wg) + torch.einsum("mn,nk->mk", du, wu)
    dwg, dwu = torch.einsum("mn,mk->nk", dg, x), torch.einsum("mn,mk->nk", du, x)
    return {"dx": dx, "dwg": (dwg if case["trans_w"] else dwg.T).contiguous(), "dwu": (dwu if case["trans_w"] else dwu.T).contiguous()}
