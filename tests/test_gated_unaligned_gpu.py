"""16-bit rows from any element on, on the gated block's few-rows kernel: through the C entry and
through the bridge."""
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
from xvram_b200._native import Gated, lib  # noqa: E402

TYPES = {torch.float16: 0, torch.bfloat16: 1}


def placed(r, c, ld, start, kind, seed, scale=1.0):
    """A (r, c) matrix of leading dimension ld that begins `start` elements into its storage and
    ends with it."""
    buffer = torch.empty(start + (r - 1) * ld + c, dtype=kind, device="cuda")
    t = buffer.as_strided((r, c), (ld, 1), start)
    t.copy_(fu.normal((r, c), kind, seed, scale))
    return t


@pytest.mark.parametrize("h,k", [(40, 1), (41, 33), (2401, 264), (2400, 515), (130, 4097)])
@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("kind", TYPES)
def test_c_entry(kind, m, h, k):
    for start, ld in ((0, k), (1, k), (3, k + 2), (1, (k + 8) // 8 * 8)):
        x = placed(m, k, ld, start, kind, 1)
        wg, wu = (placed(h, k, ld, start, kind, s, k ** -0.5) for s in (2, 3))
        bg, bu = (placed(1, h, h, 1, kind, s, 0.5)[0] for s in (4, 5))
        out = torch.full((m + 1, h + 1), 7.0, dtype=kind, device="cuda")
        pre = torch.full((2, m, (h + 3) // 4 * 4), 7.0, device="cuda")
        d = Gated(C.sizeof(Gated), TYPES[kind], 0, 0, 0, 0, m, h, k, x.data_ptr(), wg.data_ptr(),
                  wu.data_ptr(), ld, ld, ld, bg.data_ptr(), bu.data_ptr(), pre[0].data_ptr(),
                  pre[1].data_ptr(), pre.shape[2])
        d.stream = torch.cuda.current_stream().cuda_stream
        assert lib.xvram_b200_gated_forward(C.byref(d), out.data_ptr(), h + 1) == 0
        ref = fu.Gated(x, wg, wu, bg, bu, "silu", kind)
        fu.within(out[:m, :h], ref.h, ref.h_tol, "h")
        for p, want, tol in ((pre[0], ref.g, ref.eg), (pre[1], ref.u, ref.eu)):
            fu.within(p[:, :h], want, tol, "kept")
            assert bool((p[:, h:] == 7).all())
        assert bool((out[m:] == 7).all()) and bool((out[:, h:] == 7).all())
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("m", [1, 2, 4, 5])
@pytest.mark.parametrize("kind", TYPES)
def test_bridge(kind, m):
    """On both sides of the rule's bounds: 2 x 2^22 values, and one column more."""
    for h, k in ((20, 37), (4096, 2048 - 1), (4097, 2047), (4099, 2047), (1 << 13, 1025)):
        x = fu.normal((m, k), kind, 1)
        wg, wu = (fu.normal((h, k), kind, s, k ** -0.5) for s in (2, 3))
        ref = fu.Gated(x, wg, wu, None, None, "gelu", kind)
        fu.within(tb.gated_linear(x, wg, wu, activation="gelu"), ref.h, ref.h_tol, "h")
    wide = torch.nn.functional.pad(wg, (0, 7))[:, :1025]
    fu.within(tb.gated_linear(x, wide, wu, activation="gelu"), ref.h, ref.h_tol, "one weight")
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_rule_meets_the_bridge(kind):
    """The entry takes unaligned rows exactly where the bridge leaves them."""
    out = torch.empty((5, 1 << 13), dtype=kind, device="cuda")
    w = torch.zeros(((1 << 13) * 1025 + 8,), dtype=kind, device="cuda")
    x = torch.zeros((5 * 1025,), dtype=kind, device="cuda")
    for m, h, k, ok in ((1, 1 << 13, 1025, True), (4, 1 << 13, 1024, True), (4, 1 << 13, 1025, False),
                        (5, 8, 8, False)):
        d = Gated(C.sizeof(Gated), TYPES[kind], 0, 0, 0, 0, m, h, k, x.data_ptr(), w.data_ptr() + 2,
                  w.data_ptr() + 2, k, k, k)
        d.stream = torch.cuda.current_stream().cuda_stream
        assert lib.xvram_b200_gated_forward(C.byref(d), out.data_ptr(), 1 << 13) == (0 if ok else 1)
        few = m == 1 or (m <= tb._FEW_ROWS and h * k <= tb._FEW_VALUES)
        assert few == ok
