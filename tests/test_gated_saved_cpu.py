"""The gated block's saved tensors under torch's saved-tensor hooks, which may return the same
values with other strides (`torch.autograd.graph.save_on_cpu` does): what the backward pass hands
to the library, on a stand-in for it in host memory."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import feed_host as fh  # noqa: E402
import feed_util as fu  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

TYPES = [torch.float16, torch.float32]


def as_columns(t):
    return t.t().contiguous().t() if t.dim() == 2 else t.clone()


def misplaced(t):
    """At an address that is not a multiple of 16 bytes."""
    buffer = t.new_empty(t.numel() + 1)
    buffer[1:] = t.flatten()
    return buffer[1:].view(t.shape)


HOOKS = {"same": lambda t: t, "contiguous": lambda t: t.clone(memory_format=torch.contiguous_format),
         "columns": as_columns, "misplaced": misplaced,
         "wide": lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]]}


@pytest.fixture
def host(monkeypatch):
    with fh.installed(monkeypatch, tb) as library:
        yield library


def check(args, dh, hook):
    kind = args[0].dtype
    ref = fu.Gated(*args, "silu", kind)
    leaves = [t.detach().requires_grad_() for t in args]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        h = tb.gated_linear(*leaves)
    h.backward(dh)
    fu.within(h.detach(), ref.h, ref.h_tol, "h")
    want = ref.backward(dh)
    for n, t in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), leaves):
        fu.within(t.grad, *want[n], n)


@pytest.mark.parametrize("shape", [(6, 9, 16), (5, 8, 7), (1, 3, 5), (9, 1, 8), (4, 16, 1)])
@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("kind", TYPES)
def test_hooks_may_change_the_layout(host, kind, hook, shape):
    m, h, k = shape
    x = fu.normal((m, k), kind, 1, device="cpu")
    wg, wu = (fu.normal((h, k), kind, s, k ** -0.5, "cpu") for s in (2, 3))
    bias = [fu.normal((h,), kind, s, 0.5, "cpu") for s in (4, 5)]
    dh = fu.normal((m, h), kind, 6, device="cpu")
    for xv in fh.layouts(x):
        check((xv, wg, wu, *bias), dh, HOOKS[hook])
    for g, u in zip(fh.layouts(wg), fh.layouts(wu)):
        check((x, g, u, *bias), dh, HOOKS[hook])
    check((x, fh.layouts(wg)[1], wu, *bias), dh, HOOKS[hook])
    assert host.calls.count("backward") == 11


@pytest.mark.parametrize("hook", [lambda t: t.double(), lambda t: t[:1], lambda t: t.flatten(),
                                  lambda t: t.to("meta")])
def test_other_tensors_are_refused(host, hook):
    x, wg, wu = (torch.ones(s, requires_grad=True) for s in ((4, 8), (3, 8), (3, 8)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        h = tb.gated_linear(x, wg, wu)
    with pytest.raises(RuntimeError, match="saved tensor"):
        h.sum().backward()
    assert "backward" not in host.calls


def test_explicit_backward_of_every_layout(host):
    m, h, k = 5, 6, 9
    for kind in TYPES:
        x = fu.normal((m, k), kind, 1, device="cpu")
        wg, wu = (fu.normal((h, k), kind, s, k ** -0.5, "cpu") for s in (2, 3))
        dh = fu.normal((m, h), kind, 4, device="cpu")
        want = fu.Gated(x, wg, wu, None, None, "gelu", kind).backward(dh)
        for xv in fh.layouts(x):
            for g, u in zip(fh.layouts(wg), fh.layouts(wu)):
                _, saved = tb.gated_linear_forward(xv, g, u, activation="gelu")
                for n, t in zip(("dx", "dw_gate", "dw_up"), tb.gated_linear_backward(dh, saved)):
                    fu.within(t, *want[n], n)
