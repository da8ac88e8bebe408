"""Which operands of the gated block are copied to padded rows, on a stand-in for the library in
host memory: 16-bit ones, unless the few rows of x run on the kernel that reads any row."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import feed_host as fh  # noqa: E402
import feed_util as fu  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402


@pytest.fixture
def host(monkeypatch):
    with fh.installed(monkeypatch, tb) as library:
        yield library


def check(host, x, wg, wu, calls):
    host.calls.clear()
    ref = fu.Gated(x, wg, wu, None, None, "silu", x.dtype)
    fu.within(tb.gated_linear(x, wg, wu), ref.h, ref.h_tol, "h")
    assert host.calls == calls


@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
@pytest.mark.parametrize("m", [1, 2, 4])
def test_few_rows_read_unaligned_weights_in_place(host, kind, m):
    x = fu.normal((m, 37), kind, 1, device="cpu")
    wg, wu = (fu.normal((20, 37), kind, s, 1 / 6, "cpu") for s in (2, 3))
    check(host, x, wg, wu, ["forward"])
    check(host, x, *(t[:, 1:] for t in (fu.normal((20, 38), kind, s, 1 / 6, "cpu") for s in (2, 3))),
          ["forward"])


def test_what_is_still_padded(host):
    kind = torch.float16
    x = fu.normal((2, 37), kind, 1, device="cpu")
    wg, wu = (fu.normal((20, 37), kind, s, 1 / 6, "cpu") for s in (2, 3))
    wide = [torch.nn.functional.pad(t, (0, 3))[:, :37] for t in (wg, wu)]
    check(host, x, *wide, ["pack", "forward"])      # x alone: aligned weights are read faster
    check(host, fu.normal((5, 37), kind, 1, device="cpu"), wg, wu, ["pack", "forward"])
    columns = [t.t().contiguous().t()[1:] for t in (wg, wu)]
    check(host, x, *columns, ["pack", "forward"])   # stored along the other axis
    # Weights above the few-rows kernel's share: one row alone is read in place.
    big = [torch.zeros((1 << 13, 1025), dtype=kind) for _ in range(2)]
    for m, calls in ((1, ["forward"]), (2, ["pack", "forward"])):
        host.calls.clear()
        tb.gated_linear(torch.zeros((m, 1025), dtype=kind), *big)
        assert host.calls == calls
    # The backward's kernels want them aligned.
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    host.calls.clear()
    tb.gated_linear(*leaves).sum().backward()
    assert host.calls == ["pack", "forward", "backward"]
