"""Strides that torch calls contiguous whatever they are: those of empty tensors and of sizes of
one.  The gated block takes them, on a stand-in for the library in host memory."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import feed_host as fh  # noqa: E402
import feed_util as fu  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

TYPES = [torch.float16, torch.float32]


@pytest.fixture
def host(monkeypatch):
    with fh.installed(monkeypatch, tb) as library:
        yield library


def odd_views(r, c, kind, seed):
    """(r, c) matrices with strides that no kernel would read, at odd places."""
    base = fu.normal((3 * r + 2, 5 * c + 4), kind, seed, device="cpu")
    return [base[:3 * r:3, :5 * c:5], base[1:3 * r + 1:3, 2:5 * c + 2:5],
            base.t().contiguous().t()[1:3 * r + 1:3, 3:5 * c + 3:5],
            base.t().contiguous().t()[1:r + 1, 1:c + 1]]


def check(args, seed):
    x, wg = args[:2]
    kind, m, h = x.dtype, x.shape[0], wg.shape[0]
    dh = fu.normal((m, h), kind, seed, device="cpu")
    ref = fu.Gated(*args, None, None, "silu", kind)
    fu.within(tb.gated_linear(*args), ref.h, ref.h_tol, "h")
    leaves = [t.detach().requires_grad_() for t in args]
    got = torch.autograd.grad(tb.gated_linear(*leaves), leaves, dh)
    want = ref.backward(dh)
    for n, t in zip(("dx", "dw_gate", "dw_up"), got):
        if t.numel() and m and h:
            fu.within(t, *want[n], n)


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 4, 1), (4, 1, 1), (1, 1, 6), (0, 3, 8), (0, 1, 1),
                                   (2, 0, 8), (2, 0, 1), (0, 0, 3), (33, 1, 1), (3, 5, 4)])
@pytest.mark.parametrize("kind", TYPES)
def test_strides_of_small_and_empty_operands(host, kind, shape):
    m, h, k = shape
    plain = [fu.normal(s, kind, i, device="cpu") for i, s in enumerate(((m, k), (h, k), (h, k)))]
    check(plain, 9)
    views = [odd_views(*t.shape, kind, 3 + i) for i, t in enumerate(plain)]
    for i in range(3):
        for v in views[i]:
            check([v if j == i else t for j, t in enumerate(plain)], 10)
    for g in views[1]:
        for u in views[2]:
            check([plain[0], g, u], 12)
    for together in zip(*views):
        check(list(together), 11)


@pytest.mark.parametrize("kind", TYPES)
def test_an_empty_batch_of_every_second_column(host, kind):
    w = torch.ones((3, 8), dtype=kind)
    assert tb.gated_linear(torch.empty((4, 16), dtype=kind)[0:0, ::2], w, w).shape == (0, 3)
    none = torch.empty((4, 16), dtype=kind)[0:0, ::2]
    assert tb.gated_linear(torch.ones((2, 8), dtype=kind), none, none).shape == (2, 0)
