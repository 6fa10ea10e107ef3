"""The feed-forward operators at the ends of their ranges: waits that run out,
values near the limits of the types, special values, and variants that ordinary
shapes seldom take. Tolerances as in test_ffn_gpu.py (u(t) is half a step of the
type t relative to the value), unless a test states its own."""
import math  # noqa: F401

import pytest
import torch

from test_ffn_gpu import EPS, TINY, U, Mat, act64, gen, lib, norm64, normwise, product64, product_inputs, ptr, rand, scratch, within  # noqa: F401,E501

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
