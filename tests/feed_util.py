"""64-bit references and error bounds for the feed-forward operators.

Bounds, with r = eps / 2 of the result's type and t its smallest subnormal's half:
  * a product summed in FP32 is off by at most ACC(k) sum |x||w|: the tensor core adds k / 16 (or
    fewer) partial sums that it does not round to nearest, each within 2^-22 of the sum of
    magnitudes; an FFMA chain rounds k times by 2^-24.  ACC(k) = (k / 16 + 4) 2^-22 covers
    the first, and (k + 4) 2^-24 the second, which is the larger for k > 16 by at most 4 x; both
    use ACC(k) = (k + 16) 2^-24;
  * every activation here has |act'| <= 1.13 and |act''| <= 1, and is evaluated within 2^-19
    relative (the fast exponential and division), so h = act(g) u is off by at most
    (1.13 dg)(|u| + du) + |act(g)| du + 2^-19 |h|, then r |h| + t;
  * dg = dh u act'(g) is off by |dh| (|u| dg + 1.13 du + 2 dg du + 2^-18 (|u| + du)), du's by
    |dh| (1.13 dg + 2^-19 |act(g)|); 16-bit types round both once more (r |.| + t);
  * a sum of products of those is off by the sum of the factors' errors plus ACC.
"""
from __future__ import annotations

import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def acc(k: int) -> float:
    return (k + 16) * 2.0 ** -24


def act_and_slope(v: torch.Tensor, name: str):
    """(act(v), act'(v)) in 64 bits, from the formulas."""
    v = v.double()
    if name == "silu":
        q = 1 / (1 + torch.exp(-v))
        return v * q, q + v * q * (1 - q)
    if name == "gelu":
        q = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return v * q, q + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        q = 1 / (1 + torch.exp(-2 * c * (v + 0.044715 * v ** 3)))
        return v * q, q + v * q * (1 - q) * 2 * c * (1 + 3 * 0.044715 * v * v)
    if name == "relu":
        return torch.where(v > 0, v, 0 * v), (v > 0).double()
    q = 1 / (1 + torch.exp(-v))
    return q, q * (1 - q)


class Gated:
    """The block's values, gradients and their bounds in 64 bits."""

    def __init__(self, x, w_gate, w_up, bias_gate, bias_up, name, kind):
        d = lambda t: None if t is None else t.detach().double()
        self.x, self.wg, self.wu = d(x), d(w_gate), d(w_up)
        self.kind, k = kind, x.shape[1]
        self.g, self.u = self.x @ self.wg.t(), self.x @ self.wu.t()
        self.eg = acc(k) * (self.x.abs() @ self.wg.abs().t())
        self.eu = acc(k) * (self.x.abs() @ self.wu.abs().t())
        if bias_gate is not None:
            self.g = self.g + d(bias_gate)
            self.eg = self.eg + 2.0 ** -24 * self.g.abs()
        if bias_up is not None:
            self.u = self.u + d(bias_up)
            self.eu = self.eu + 2.0 ** -24 * self.u.abs()
        self.a, self.s = act_and_slope(self.g, name)
        self.h = self.a * self.u
        self.h_tol = (1.13 * self.eg * (self.u.abs() + self.eu) + self.a.abs() * self.eu +
                      (2.0 ** -19 + HALF[kind]) * self.h.abs() + TINY[kind])

    def backward(self, dh):
        """{name: (gradient, bound)}"""
        dh = dh.double()
        r, t = HALF[self.kind], TINY[self.kind]
        dg, du = dh * self.u * self.s, dh * self.a
        eg = dh.abs() * (self.u.abs() * self.eg + 1.13 * self.eu + 2 * self.eg * self.eu +
                         2.0 ** -18 * (self.u.abs() + self.eu))
        eu = dh.abs() * (1.13 * self.eg + 2.0 ** -19 * self.a.abs())
        m, h = dh.shape
        out = {}
        for n, v, e in (("db_gate", dg, eg), ("db_up", du, eu)):
            total = v.sum(0)
            out[n] = (total, (e + acc(m) * v.abs()).sum(0) + r * total.abs() + t)
        if self.kind != torch.float32:
            eg, eu = eg + r * dg.abs() + t, eu + r * du.abs() + t
        for n, v, e in (("dw_gate", dg, eg), ("dw_up", du, eu)):
            w = v.t() @ self.x
            out[n] = (w, (e + acc(m) * (v.abs() + e)).t() @ self.x.abs() + r * w.abs() + t)
        dx = dg @ self.wg + du @ self.wu
        ex = ((eg + acc(2 * h) * (dg.abs() + eg)) @ self.wg.abs() +
              (eu + acc(2 * h) * (du.abs() + eu)) @ self.wu.abs())
        out["dx"] = (dx, ex + r * dx.abs() + t)
        return out


def within(got, want, tol, name=""):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), (name, int(bad.sum()), float(d[bad].max()), float(tol[bad].min()))


def normal(shape, dtype, seed, scale=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)
