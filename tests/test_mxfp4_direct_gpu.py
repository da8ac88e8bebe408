"""Few rows of an MXFP4 product, quantised inside it or by a pass in front: the same results, up to
the bounds on rows and values, through the C entries with and without memory for the codes."""
from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402
from xvram_b200._native import Mxfp4Product, lib  # noqa: E402

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


@pytest.mark.parametrize("shape", [(1, 70, 65536), (2, 260, 32768), (4, 300, 16384), (8, 1100, 8192),
                                   (16, 2300, 4096), (16, 20000, 2048), (15, 130, 4353), (3, 24, 31),
                                   (16, 40, 1), (5, 2400, 6553)])
@pytest.mark.parametrize("kind", TYPES)
def test_with_and_without_memory_for_the_codes(kind, shape):
    m, n, k = shape
    assert m <= 16 and m * k <= 65536
    x = fu.normal((m, k), kind, 1)
    ws = [tb.quantize_mxfp4(fu.normal((n, k), torch.float32, s, k ** -0.5)) for s in (2, 3)]
    size = m * ((k + 31) // 32) * 16
    guard = torch.full((size + (k + 127) // 128 * 512 + 64,), 77, dtype=torch.uint8, device="cuda")
    xq = tb.quantize_mxfp4(x)
    for call, count, whole in ((lib.xvram_b200_mxfp4_linear, 1, lambda a: tb.linear_mxfp4(a, ws[0])),
                               (lib.xvram_b200_mxfp4_gated, 2, lambda a: tb.gated_linear_mxfp4(a, *ws))):
        got = []
        for codes in (0, guard.data_ptr()):
            out = torch.full((m, n), 7.0, dtype=kind, device="cuda")
            d = Mxfp4Product(C.sizeof(Mxfp4Product), TYPES[kind], TYPES[kind], 0, m, n, k, x.data_ptr(), k,
                             codes, codes and codes + size, ws[0].codes.data_ptr(),
                             ws[1].codes.data_ptr(), ws[0].scales.data_ptr(), ws[1].scales.data_ptr())
            d.out, d.ld_out, d.stream = out.data_ptr(), n, torch.cuda.current_stream().cuda_stream
            assert call(C.byref(d)) == 0
            got.append(out)
        v = [tb.dequantize_mxfp4(w).double() for w in ws]
        xv = tb.dequantize_mxfp4(xq).double()
        if count == 1:
            y = xv @ v[0].t()
            tol = fu.acc(k) * (xv.abs() @ v[0].abs().t()) + fu.HALF[kind] * y.abs() + fu.TINY[kind]
        else:
            ref = fu.Gated(xv, *v, None, None, "silu", kind)
            y, tol = ref.h, ref.h_tol
        for t in (*got, whole(x)):
            fu.within(t, y, tol, call.__name__)
    assert bool((guard[-64:] == 77).all())
    assert xd.kernel_status() == 0
