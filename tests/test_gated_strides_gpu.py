"""The gated block on operands whose strides torch leaves as they are: empty ones and sizes of
one."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 4, 1), (200, 1, 1), (40, 9, 1), (1, 1, 6),
                                   (0, 3, 8), (2, 0, 8)])
@pytest.mark.parametrize("kind", TYPES)
def test_strides_of_small_and_empty_operands(kind, shape):
    m, h, k = shape
    ops = []
    for i, (r, c) in enumerate(((m, k), (h, k), (h, k))):
        base = fu.normal((3 * r + 2, 5 * c + 4), kind, i)
        ops.append([base[:3 * r:3, :5 * c:5], base.t().contiguous().t()[1:r + 1, 1:c + 1]])
    dh = fu.normal((m, h), kind, 9)
    for x in ops[0]:
        for g in ops[1]:
            for u in ops[2]:
                leaves = [t.detach().requires_grad_() for t in (x, g, u)]
                ref = fu.Gated(x, g, u, None, None, "silu", kind)
                y = tb.gated_linear(*leaves)
                fu.within(y.detach(), ref.h, ref.h_tol, "h")
                got = torch.autograd.grad(y, leaves, dh)
                want = ref.backward(dh)
                for n, t in zip(("dx", "dw_gate", "dw_up"), got):
                    fu.within(t, *want[n], n)
    assert xd.kernel_status() == 0
