"""Forward-mode derivatives: the feed-forward operators have none, so a tensor with a tangent is
refused instead of being answered without one (which torch reads as a zero derivative)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import feed_host as fh  # noqa: E402
from torch.autograd import forward_ad  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

SHAPES = {"x": (4, 32), "w_gate": (3, 32), "w_up": (3, 32), "bias_gate": (3,), "bias_up": (3,)}


@pytest.fixture
def host(monkeypatch):
    with fh.installed(monkeypatch, tb) as library:
        yield library


def arguments(dual=None, requires_grad=False):
    args = {n: torch.ones(s, requires_grad=requires_grad) for n, s in SHAPES.items()}
    if dual:
        args[dual] = forward_ad.make_dual(args[dual], torch.ones(SHAPES[dual]))
    return args


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", SHAPES)
def test_gated_linear(host, name, requires_grad):
    with forward_ad.dual_level():
        args = arguments(name, requires_grad)
        with pytest.raises(RuntimeError, match="forward-mode"):
            tb.gated_linear(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            tb.gated_linear(**args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            tb.gated_linear_forward(**args)
        assert not host.calls
        tb.gated_linear(**arguments())  # no tangent: nothing to refuse
    assert host.calls == ["forward"]


def test_gradient_of_the_result_with_a_tangent(host):
    with forward_ad.dual_level():
        dh = forward_ad.make_dual(torch.ones(4, 3), torch.ones(4, 3))
        _, saved = tb.gated_linear_forward(**arguments())
        with pytest.raises(RuntimeError, match="forward-mode"):
            tb.gated_linear_backward(dh, saved)
        args = arguments(requires_grad=True)
        h = tb.gated_linear(**args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(h, args["x"], dh)
    assert "backward" not in host.calls


def test_mxfp4():
    w = tb.Mxfp4Matrix(torch.zeros(3 * 16, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8),
                       (3, 32))
    with forward_ad.dual_level():
        x, b = (forward_ad.make_dual(torch.ones(s), torch.ones(s)) for s in ((4, 32), (3,)))
        plain = torch.ones(4, 32)
        for call in (lambda: tb.quantize_mxfp4(x), lambda: tb.linear_mxfp4(x, w),
                     lambda: tb.linear_mxfp4(plain, w, b), lambda: tb.gated_linear_mxfp4(x, w, w),
                     lambda: tb.gated_linear_mxfp4(plain, w, w, b),
                     lambda: tb.gated_linear_mxfp4(plain, w, w, None, b),
                     lambda: tb.linear_mxfp4(w, w, b)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
