"""The gated block's gradients when autograd's saved-tensor hooks move its saved tensors: to the
host and back, to other strides, and through checkpointing."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_host as fh  # noqa: E402
import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402
from torch.utils.checkpoint import checkpoint  # noqa: E402

TYPES = [torch.float16, torch.bfloat16, torch.float32]
HOOKS = {"host": lambda: torch.autograd.graph.save_on_cpu(),
         "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
         "columns": lambda: torch.autograd.graph.saved_tensors_hooks(
             lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone())}


def gradients(args, dh, hooks=None, call=tb.gated_linear):
    leaves = [t.detach().requires_grad_() for t in args]
    if hooks is None:
        h = call(*leaves)
    else:
        with hooks():
            h = call(*leaves)
    return torch.autograd.grad(h, leaves, dh)


@pytest.mark.parametrize("shape", [(3, 40, 56), (200, 72, 64), (1, 9, 5)])
@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("kind", TYPES)
def test_hooks_may_change_the_layout(kind, hooks, shape):
    m, h, k = shape
    x = fu.normal((m, k), kind, 1)
    wg, wu = (fu.normal((h, k), kind, s, k ** -0.5) for s in (2, 3))
    bg, bu = (fu.normal((h,), kind, s, 0.5) for s in (4, 5))
    dh = fu.normal((m, h), kind, 6)
    want = fu.Gated(x, wg, wu, bg, bu, "silu", kind).backward(dh)
    names = ("dx", "dw_gate", "dw_up", "db_gate", "db_up")
    cases = [(xv, wg, wu) for xv in fh.layouts(x)]
    cases += [(x, g, u) for g, u in zip(fh.layouts(wg), fh.layouts(wu))]
    for ops in cases:
        for n, t in zip(names, gradients((*ops, bg, bu), dh, HOOKS[hooks])):
            fu.within(t, *want[n], n)
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed(reentrant):
    kind = torch.bfloat16
    args = [fu.normal((50, 72), kind, 1), *(fu.normal((33, 72), kind, s, 72 ** -0.5) for s in (2, 3))]
    dh = fu.normal((50, 33), kind, 4)

    def call(*leaves):
        return checkpoint(tb.gated_linear, *leaves, use_reentrant=reentrant)
    if reentrant:  # it has no autograd.grad
        leaves = [t.detach().requires_grad_() for t in args]
        call(*leaves).backward(dh)
        got = [t.grad for t in leaves]
    else:
        got = gradients(args, dh, call=call)
    for a, b in zip(got, gradients(args, dh)):
        assert torch.equal(a, b)
