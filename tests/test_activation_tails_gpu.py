"""The gated block's activations and slopes over their whole range: near zero, in both tails, and
where the exponential under- or overflows.

The weights are zeros, so that g = bias_gate and u = bias_up = 1 exactly, and dh is 1 in row 0 and
0 elsewhere: then h = act(g), dw_up = act(g) and dw_gate = act'(g), with x = 1, and only the
activation's arithmetic and the result's rounding are off.

Bounds, in units of 2^-23 (E) relative to the magnitudes that are added:
  * e = exp(-|z|): FP32 within 2 (the documented bound of expf is 2 units in the last place at
    most); the fast form for 16-bit results within 2 + 1.173 |z| (the documented bound of
    __expf).  r = 1 / (1 + e) adds at most half a unit for the sum, 2 for the division (2 units
    for __fdividef, half a unit in FP32) and e's own error once: q and 1 - q, r or e r, are within
    2 (2 + 1.173 |z|) + 2.5 + 0.5, which (8 + 3 |z|) covers, and FP32 within 8;
  * sigmoid' = q (1 - q): twice that.  act' = q + v q (1 - q) of SiLU: the terms are added with
    their own errors, so the bound is (16 + 6 |z|) E (q + |v| q (1 - q));
  * tanh-GELU: z = 2 c (v + k v^3) carries six roundings, 3 |z| E as an absolute error, which is the
    relative error of e: 3 |z| more, twice for the slope, and its polynomial 3 more;
  * GELU: erfc(-v / sqrt 2) has the relative condition v^2 for v < 0 (its logarithm's slope), so the
    argument's two roundings give v^2 E, the function itself 4 (documented); the fast form's fit
    is within 8e-7 = 7 E, its exponential within 2 + 1.173 v^2 / 2 with its argument's rounding
    v^2 / 4, its division 2: (16 + 2 v^2) E covers both;
  * half a step of the result's type, and its smallest value's half.  Below FP32's normal range
    (2^-126) e is held in steps of 2^-149: |v| 2^-149 covers what that leaves in v e;
  * the 16-bit forward divides by 1 + exp(-z) as __fdividef does: zero from 2^126 on (documented),
    where q < 2^-126.  That is z < -87.3; q |v| falls from there on, so v q is off by less than
    87.4 x 2^-126 for SiLU (z = v), and by less for the tanh form, whose z is larger than v there.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

TYPES = [torch.float16, torch.bfloat16, torch.float32]
E = 2.0 ** -23


def points(kind):
    near = torch.linspace(-6, 6, 97)
    far = torch.tensor([6.5, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 20, 25, 30, 40, 60, 80, 86, 87, 87.5,
                        88, 88.5, 89, 90, 95, 100, 103, 104, 110, 1e3, 1e4])
    more = torch.tensor([] if kind == torch.float16 else [1e12, 1e13, 1e20, 1e30])
    return torch.cat([near, far, -far, more, -more, torch.tensor([0.0, -0.0])]).to(kind).cuda()


def logistic(z):
    """(sigmoid(z), 1 - sigmoid(z)) in 64 bits, neither from the other."""
    e = torch.exp(-z.abs())
    big, small = 1 / (1 + e), e / (1 + e)
    return torch.where(z >= 0, big, small), torch.where(z >= 0, small, big)


def reference(v, act, fast):
    """act, its bound, act' and its bound (without the result's rounding)."""
    v = v.double()
    if act == "relu":
        zero = torch.zeros_like(v)
        return v.clamp(min=0), zero, (v > 0).double(), zero
    if act == "gelu":
        q = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        t = torch.nan_to_num(v * torch.exp(-0.5 * v * v)) / math.sqrt(2 * math.pi)
        rel = (16 + 2 * torch.minimum(v * v, torch.tensor(4e4, device=v.device))) * E
        return v * q, rel * (v * q).abs(), q + t, rel * (q + t.abs())
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        z = 2 * c * (v + 0.044715 * v ** 3)
        slope = 2 * c * (1 + 3 * 0.044715 * v * v)
    else:
        z, slope = v, torch.ones_like(v)
    q, p = logistic(z)
    a = z.abs().clamp(max=200)  # beyond it e is 0
    rel = (8 + (3 * a if fast else 0) + (3 * a if act == "gelu_tanh" else 0)) * E
    if act == "sigmoid":
        return q, rel * q, q * p, 2 * rel * q * p
    t = torch.nan_to_num(v * q * p * slope)
    return v * q, (rel + E) * (v * q).abs(), q + t, (2 * rel + 3 * E) * (q + t.abs())


@pytest.mark.parametrize("m", [1, 20, 200])
@pytest.mark.parametrize("act", fu.ACTS)
@pytest.mark.parametrize("kind", TYPES)
def test_whole_range(kind, act, m):
    g = points(kind)
    h = g.numel()
    x = torch.ones((m, 1), dtype=kind, device="cuda")
    zeros = torch.zeros((h, 1), dtype=kind, device="cuda")
    dh = torch.zeros((m, h), dtype=kind, device="cuda")
    dh[0] = 1
    leaves = [t.requires_grad_() for t in (zeros, zeros.clone())]
    y = tb.gated_linear(x, *leaves, g, torch.ones_like(g), activation=act)
    d_gate, d_up = torch.autograd.grad(y, leaves, dh)
    fast = kind != torch.float32
    a, a_tol, s, s_tol = reference(g, act, fast)
    least = fu.TINY[kind] + g.double().abs().clamp(max=200) * 2.0 ** -149
    r = fu.HALF[kind]
    # The tensor cores may take FP32 values below the normal range for zero in a sum.
    product = 2.0 ** -126 if fast else 0.0
    tail = 88 * 2.0 ** -126 if fast else 0.0
    for got in (y.detach()[0], y.detach()[-1]):
        fu.within(got, a, a_tol + r * (a.abs() + a_tol) + least + tail, "act")
    fu.within(d_up[:, 0], a, a_tol + 2 * r * (a.abs() + a_tol) + 2 * least + product, "act in dW")
    fu.within(d_gate[:, 0], s, s_tol + 2 * r * (s.abs() + s_tol) + 2 * least + product, "slope")
    assert xd.kernel_status() == 0
