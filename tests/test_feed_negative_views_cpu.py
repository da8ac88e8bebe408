"""Views that stand for their memory's negative (the imaginary part of a conjugate) give what their
values give.  Their elements are two apart, so only rows and biases of one element are ever read in
place."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from feed_host import installed  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

KINDS = [torch.float32, torch.float16]


def negative(t):
    """t as the imaginary part of a conjugate."""
    z = torch.complex(torch.zeros_like(t, dtype=torch.float32), -t.float()).to(
        torch.complex32 if t.dtype == torch.float16 else torch.complex64).conj().imag
    assert z.is_neg() and z.dtype == t.dtype and torch.equal(z, t)
    return z


def values(shape, kind, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(3, 5, 8), (3, 5, 1), (3, 1, 4), (1, 1, 1), (40, 16, 7)])
def test_gated(monkeypatch, kind, shape):
    m, h, k = shape
    with installed(monkeypatch, tb):
        args = [values(s, kind, i) for i, s in enumerate([(m, k), (h, k), (h, k), (h,), (h,)])]
        dh = values((m, h), kind, 9)
        want, saved = tb.gated_linear_forward(*args)
        grads = tb.gated_linear_backward(dh, saved)
        for i in range(5):
            changed = list(args)
            changed[i] = negative(args[i])
            assert torch.equal(tb.gated_linear(*changed), want)
            leaves = [t.detach().requires_grad_() for t in changed]
            got = torch.autograd.grad(tb.gated_linear(*leaves), leaves, negative(dh))
            assert all(torch.equal(a, b) for a, b in zip(got, grads))
        assert all(torch.equal(a, b) for a, b in
                   zip(tb.gated_linear_backward(negative(dh), saved), grads))


@pytest.mark.parametrize("shape", [(3, 4), (3, 1), (1, 1)])
def test_rows_and_biases_are_resolved(shape):
    """What the 4-bit operators read their input and biases by."""
    x = values(shape, torch.float32, 1)
    rows, ld = tb._rows(negative(x))
    assert not rows.is_neg() and torch.equal(rows, x) and ld >= shape[1]
    b = tb._check_bias(negative(x[0]), shape[1], torch.float32, x.device, "bias")
    assert not b.is_neg() and torch.equal(b, x[0])
