"""Matrices of more than 2^31 elements: inputs and their gradient, results and pre-activations, and
4-bit matrices, checked on rows and columns at both ends and around element 2^31."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from test_mxfp4_gpu import reference, unpacked  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

KIND = torch.bfloat16
M, WIDE = 66000, 32768  # 2.16e9 elements; row 65536 starts at element 2^31
ROWS = [0, 1, 65535, 65536, 65537, M - 1]
COLS = [0, 77, WIDE - 1]
assert M * WIDE > 1 << 31

if torch.cuda.get_device_properties(0).total_memory < 100e9:  # pragma: no cover
    pytest.skip("needs 100 GB of device memory", allow_module_level=True)


def big(seed):
    """(M, WIDE) normal values, in parts so that no float32 copy of them all exists."""
    out = torch.empty((M, WIDE), dtype=KIND, device="cuda")
    for i in range(0, M, 8192):
        part = out[i:i + 8192]
        part.copy_(fu.normal(part.shape, KIND, seed + i))
    return out


def at(t, rows):
    return t[torch.tensor(rows, device=t.device)]


def test_wide_input_and_its_gradient():
    h = 40
    x = big(1)
    wg, wu = (fu.normal((h, WIDE), KIND, s, WIDE ** -0.5) for s in (2, 3))
    dh = fu.normal((M, h), KIND, 4)
    out, saved = tb.gated_linear_forward(x, wg, wu)
    dx, dwg, dwu, _, _ = tb.gated_linear_backward(dh, saved, (True, True, True, False, False))
    ref = fu.Gated(at(x, ROWS), wg, wu, None, None, "silu", KIND)
    fu.within(at(out, ROWS), ref.h, ref.h_tol, "h")
    fu.within(at(dx, ROWS), *ref.backward(at(dh, ROWS))["dx"], "dx")
    # Some columns of the weights' gradients, from the kept pre-activations: sums over all rows.
    pre = saved.tensors[-1][:, :, :h].double()
    a, s = fu.act_and_slope(pre[0], "silu")
    v = dh.double()
    cols = x[:, COLS].double()
    for got, d in ((dwg, v * pre[1] * s), (dwu, v * a)):
        want = d.t() @ cols
        # dg and du within 2^-17 and rounded once; their sum; the result.
        tol = (2.0 ** -17 + fu.HALF[KIND] + fu.acc(M)) * (d.abs().t() @ cols.abs())
        fu.within(got[:, COLS], want, tol + fu.HALF[KIND] * want.abs(), "dW")
    assert xd.kernel_status() == 0


def test_wide_result():
    k = 64
    x = fu.normal((M, k), KIND, 1)
    wg, wu = (fu.normal((WIDE, k), KIND, s, k ** -0.5) for s in (2, 3))
    out, saved = tb.gated_linear_forward(x, wg, wu, activation="sigmoid")
    ref = fu.Gated(at(x, ROWS), wg, wu, None, None, "sigmoid", KIND)
    fu.within(at(out, ROWS), ref.h, ref.h_tol, "h")
    assert torch.equal(at(tb.gated_linear(x, wg, wu, activation="sigmoid"), ROWS), at(out, ROWS))
    del out
    dh = big(7)
    dx, dwg, dwu, dbg, dbu = tb.gated_linear_backward(dh, saved)
    fu.within(at(dx, ROWS), *ref.backward(at(dh, ROWS))["dx"], "dx")
    part = fu.Gated(x, wg[COLS], wu[COLS], None, None, "sigmoid", KIND)
    want = part.backward(dh[:, COLS])
    for n, t in (("dw_gate", dwg), ("dw_up", dwu), ("db_gate", dbg), ("db_up", dbu)):
        fu.within(t[COLS], *want[n], n)
    assert xd.kernel_status() == 0


def test_4_bit_matrices():
    n = 40
    x = big(1)
    q = tb.quantize_mxfp4(x)
    back = tb.dequantize_mxfp4(q, KIND)
    values = reference(at(x, ROWS))[0]
    assert torch.equal(at(back, ROWS).double(), values.to(KIND).double())
    del back
    w = tb.quantize_mxfp4(fu.normal((n, WIDE), torch.float32, 2, WIDE ** -0.5))
    wv = unpacked(w)[0][:, :WIDE]
    y = values @ wv.t()
    tol = fu.acc(WIDE) * (values.abs() @ wv.abs().t()) + fu.HALF[KIND] * y.abs()
    fu.within(at(tb.linear_mxfp4(x, w), ROWS), y, tol, "wide input")
    fu.within(at(tb.linear_mxfp4(q, w, dtype=KIND), ROWS), y, tol, "wide 4-bit input")
    # As a weight: features at both ends and around 2^31, one row and more than 128.
    few = fu.normal((200, WIDE), KIND, 3)
    fv = reference(few)[0]
    for rows in (1, 200):
        y = fv[:rows] @ values.t()
        tol = fu.acc(WIDE) * (fv[:rows].abs() @ values.abs().t()) + fu.HALF[KIND] * y.abs()
        got = tb.linear_mxfp4(few[:rows], q)
        fu.within(got[:, torch.tensor(ROWS, device="cuda")], y, tol, "wide weight")
    del q, x
    narrow = fu.normal((M, 64), KIND, 4)
    w = tb.quantize_mxfp4(fu.normal((WIDE, 64), torch.float32, 5, 0.125))
    wv, xv = unpacked(w)[0][:, :64], reference(at(narrow, ROWS))[0]
    y = xv @ wv.t()
    tol = fu.acc(64) * (xv.abs() @ wv.abs().t()) + fu.HALF[KIND] * y.abs() + fu.TINY[KIND]
    fu.within(at(tb.linear_mxfp4(narrow, w), ROWS), y, tol, "wide result")
    assert xd.kernel_status() == 0
