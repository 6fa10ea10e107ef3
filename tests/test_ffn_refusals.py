"""The feed-forward operators refuse what they do not take, with a status and
a message, before anything reaches a device: descriptors are checked first, so
these run without a GPU (calls with a good descriptor then answer that the
library is not initialised)."""
import ctypes as C

import pytest

from tt_lazy_b200 import capi

P = 0x10000  # an address that is never dereferenced: every call here ends before a launch


def norm(**kw):
    a = dict(rows=4, cols=64, x=P, ldx=64, weight=P, y=P, ldy=64, dtype=capi.BF16)
    a.update(kw)
    return capi.rms_norm_desc(**a)


def norm_backward(**kw):
    a = dict(rows=4, cols=64, dy=P, lddy=64, hidden=P, ldh=64, weight=P, dx=P, lddx=64, dweight=P, dtype=capi.BF16)
    a.update(kw)
    return capi.rms_norm_backward_desc(**a)


def linear(**kw):
    a = dict(M=4, N=64, K=32, x=P, ldx=32, w=P, ldw=64, y=P, ldy=64, dtype=capi.BF16)
    a.update(kw)
    return capi.linear_desc(**a)


def linear_backward(**kw):
    a = dict(M=4, N=64, K=32, dy=P, lddy=64, x=P, ldx=32, w=P, ldw=64, dtype=capi.BF16, dx=P, lddx=32, dw=P, lddw=64,
             dbias=P)
    a.update(kw)
    return capi.linear_backward_desc(**a)


def gated(**kw):
    a = dict(M=4, N=64, K=32, x=P, ldx=32, wg=P, wu=P, ldw=64, y=P, ldy=64, dtype=capi.BF16)
    a.update(kw)
    return capi.gated_linear_desc(**a)


def gated_backward(**kw):
    a = dict(M=4, N=64, K=32, dy=P, lddy=64, x=P, ldx=32, wg=P, wu=P, ldw=64, gate=P, up=P, ldp=64, dtype=capi.BF16,
             dx=P, lddx=32, dwg=P, dwu=P, lddw=64)
    a.update(kw)
    return capi.gated_linear_backward_desc(**a)


CALLS = {capi.RmsNormDesc: "ttc_rms_norm", capi.RmsNormBackwardDesc: "ttc_rms_norm_backward",
         capi.LinearDesc: "ttc_linear", capi.LinearBackwardDesc: "ttc_linear_backward",
         capi.GatedLinearDesc: "ttc_gated_linear", capi.GatedLinearBackwardDesc: "ttc_gated_linear_backward"}
INVALID, UNSUPPORTED = capi.ERR_INVALID, capi.ERR_UNSUPPORTED
E8 = dict(dtype=capi.E4M3, y_dtype=capi.BF16, trans_w=True, ldw=32, x_scales=P)

REFUSED = [
    # shapes
    (norm(rows=-1), INVALID, "shape"), (norm(cols=0), INVALID, "shape"), (norm(rows=1 << 31), UNSUPPORTED, "rows"),
    (norm_backward(cols=0), INVALID, "shape"), (linear(M=-1), INVALID, "shape"), (linear(N=0), INVALID, "shape"),
    (linear(K=0), INVALID, "shape"), (linear(N=(1 << 24) + 1, ldw=1 << 25, ldy=1 << 25), UNSUPPORTED, "exceed"),
    (linear(M=(1 << 30) + 1), UNSUPPORTED, "exceed"), (linear_backward(K=0), INVALID, "shape"),
    (gated(N=-5), INVALID, "shape"), (gated_backward(K=0), INVALID, "shape"),
    # types
    (norm(dtype=capi.E4M3), INVALID, "dtype"), (norm(dtype=9), INVALID, "dtype"),
    (norm(dtype=capi.F16, weight_dtype=capi.BF16), INVALID, "weight_dtype"),
    (norm(dtype=capi.BF16, y_dtype=capi.F16), INVALID, "y_dtype"),
    (norm(dtype=capi.BF16, y_dtype=capi.F32), INVALID, "y_dtype"),
    (norm_backward(weight_dtype=capi.F16), INVALID, "weight_dtype"),
    (linear(dtype=capi.F32), UNSUPPORTED, "ttc_gemm"), (linear(dtype=17), INVALID, "dtype"),
    (linear(y_dtype=capi.F16), INVALID, "y_dtype"), (linear(y_dtype=capi.E4M3), INVALID, "y_dtype"),
    (linear(**{**E8, "y_dtype": capi.E4M3, "w_scales": P}), INVALID, "y_dtype"),
    (linear_backward(dtype=capi.E4M3), INVALID, "dtype"), (linear_backward(dtype=capi.F32), UNSUPPORTED, "ttc_gemm"),
    (gated(dtype=capi.F32), UNSUPPORTED, "ttc_gemm"), (gated_backward(dtype=capi.E4M3), INVALID, "dtype"),
    (linear(dtype=capi.E4M3, y_dtype=capi.BF16, x_scales=P, w_scales=P), UNSUPPORTED, "trans_w"),
    # options
    (norm(eps=-1.0), INVALID, "eps"), (norm(eps=float("nan")), INVALID, "eps"), (linear(act=5), INVALID, "activation"),
    (linear(act=-1), INVALID, "activation"), (linear(trans_w=2, ldw=64), INVALID, "trans_w"),
    (gated(act=77), INVALID, "activation"), (gated_backward(act=77), INVALID, "activation"),
    # missing tensors
    (norm(x=None), INVALID, "x is NULL"), (norm(weight=None), INVALID, "weight is NULL"),
    (norm(y=None), INVALID, "y is NULL"), (norm(y_dtype=capi.E4M3), INVALID, "scales is NULL"),
    (norm(scales=P), INVALID, "scales"), (norm_backward(dx=None), INVALID, "dx is NULL"),
    (linear(w=None), INVALID, "w is NULL"), (linear(**E8), INVALID, "w_scales is NULL"),
    (linear(x_scales=P), INVALID, "x_scales"), (linear(w_scales=P), INVALID, "w_scales"),
    (linear_backward(act=capi.ACT_SILU), INVALID, "pre is NULL"), (linear_backward(x=None), INVALID, "x is NULL"),
    (linear_backward(w=None), INVALID, "w is NULL"), (gated(wu=None), INVALID, "wu is NULL"),
    (gated(gate=P, ldp=64), INVALID, "both or neither"), (gated(up=P, ldp=64), INVALID, "both or neither"),
    (gated(**E8, wg_scales=P), INVALID, "wu_scales is NULL"), (gated_backward(gate=None), INVALID, "gate is NULL"),
    (gated_backward(dwu=None), INVALID, "both or neither"),
    # leading dimensions below the width
    (norm(ldx=63), INVALID, "leading dimension"), (norm(residual=P, ldr=0), INVALID, "leading dimension"),
    (norm(hidden=P, ldh=63), INVALID, "leading dimension"), (norm_backward(dhidden=P), INVALID, "leading dimension"),
    (linear(ldx=31), INVALID, "leading dimension"), (linear(ldw=63), INVALID, "leading dimension"),
    (linear(trans_w=True, ldw=31), INVALID, "leading dimension"), (linear(pre=P, ldp=3), INVALID, "leading dimension"),
    (linear(residual=P, ldr=-64), INVALID, "leading dimension"), (linear_backward(lddw=63), INVALID, "leading"),
    (gated(ldy=1), INVALID, "leading dimension"), (gated_backward(ldp=63), INVALID, "leading dimension"),
    # addresses that are not aligned to their elements
    (norm(x=P + 1), INVALID, "aligned"), (norm(dtype=capi.F32, y=P + 2), INVALID, "aligned"),
    (linear(w=P + 1), INVALID, "aligned"), (linear(bias=P + 1), INVALID, "aligned"),
    (linear(**E8, w_scales=P + 2), INVALID, "aligned"), (gated(y=P + 1), INVALID, "aligned"),
    (gated_backward(dwg=P + 1), INVALID, "aligned"),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused_with_status_and_message(i):
    desc, code, text = REFUSED[i]
    L = capi.lib()
    name = CALLS[type(desc)]
    names = [name] + ([name + "_workspace"] if type(desc) in capi._WITH_WORKSPACE else [])
    for fn in names:
        n = C.c_size_t(77)
        args = (C.byref(desc), C.byref(n)) if fn.endswith("_workspace") else (C.byref(desc),)
        rc = getattr(L, fn)(*args)
        message = L.ttc_last_error().decode()
        assert rc == code and text in message, (fn, rc, message)
        if fn.endswith("_workspace"):
            assert n.value == 0


@pytest.mark.parametrize("desc", [norm_backward(), linear_backward(act=capi.ACT_SILU, pre=P, ldp=64), gated_backward(),
                                  linear_backward(dw=None, dx=None, x=None, w=None)])
def test_workspace_that_is_missing_short_or_misaligned_is_refused(desc):
    L = capi.lib()
    fn = getattr(L, CALLS[type(desc)])
    need = capi.workspace_size(desc)
    assert need > 0 and need % 256 == 0
    for address, size in ((None, need), (P, need - 1), (P + 128, need), (P, 0)):
        desc.workspace, desc.workspace_bytes = address, size
        assert fn(C.byref(desc)) == INVALID
        assert b"workspace" in L.ttc_last_error()


def test_norm_rows_whose_column_index_could_pass_32_bits_are_refused():
    L, n, widest = capi.lib(), C.c_size_t(), 1 << 30
    for cols in (widest + 1, (1 << 31) - 1):
        desc = norm(cols=cols, ldx=cols, ldy=cols)
        assert L.ttc_rms_norm(C.byref(desc)) == UNSUPPORTED
        assert b"columns" in L.ttc_last_error()
        desc = norm_backward(cols=cols, lddy=cols, ldh=cols, lddx=cols)
        for rc in (L.ttc_rms_norm_backward(C.byref(desc)), L.ttc_rms_norm_backward_workspace(C.byref(desc), C.byref(n))):
            assert rc == UNSUPPORTED and b"columns" in L.ttc_last_error()
    assert capi.workspace_size(norm_backward(cols=widest, lddy=widest, ldh=widest, lddx=widest)) >= 4 * widest


def test_null_descriptors_are_refused():
    L = capi.lib()
    n = C.c_size_t()
    for fn in CALLS.values():
        assert getattr(L, fn)(None) == INVALID
    for desc, fn in capi._WITH_WORKSPACE.items():
        assert getattr(L, fn + "_workspace")(None, C.byref(n)) == INVALID
        assert getattr(L, fn + "_workspace")(C.byref(desc()), None) == INVALID


def test_aligned_forward_products_need_no_workspace():
    assert capi.workspace_size(linear()) == 0
    assert capi.workspace_size(linear(M=8192)) == 0
    assert capi.workspace_size(gated(trans_w=True, ldw=32)) == 0


def test_no_rows_needs_no_tensors_and_no_workspace():
    """Zero rows is a valid call: nothing is read, so nothing has to be set."""
    for desc in (linear_backward(M=0, dy=None, x=None, w=None), gated_backward(M=0, dy=None, x=None, wg=None, wu=None)):
        assert capi.workspace_size(desc) == 0


def test_structures_match_the_header(tmp_path):
    """The ctypes structures have the layout that a C compiler gives the header's."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"ttc_rms_norm_desc": capi.RmsNormDesc, "ttc_rms_norm_backward_desc": capi.RmsNormBackwardDesc,
             "ttc_linear_desc": capi.LinearDesc, "ttc_linear_backward_desc": capi.LinearBackwardDesc,
             "ttc_gated_linear_desc": capi.GatedLinearDesc,
             "ttc_gated_linear_backward_desc": capi.GatedLinearBackwardDesc}
    lines = ['#include <stdio.h>', '#include "tt_cuda.h"', "int main(void) {"]
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "layout")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe])
    got = dict(line.split() for line in subprocess.check_output([exe], text=True).splitlines())
    for c, py in names.items():
        assert int(got[c]) == C.sizeof(py), c
        for f in py._fields_:
            assert int(got[f"{c}.{f[0]}"]) == getattr(py, f[0]).offset, (c, f[0])
