"""The gated block's FP16 gradients where dg and du, the operands of their products, lie outside
FP16's range: the gradients are right wherever they themselves fit.

Bounds are feed_util's, with one change: the products' operands are held times a power of two that
brings the largest of them into [2^14, 2^15) (or as they are, when that lies in [2^-8, 2^16)), so
what is lost below FP16's smallest step is at most 2^-25 times the inverse: 2^-39 of the largest
when scaled, and 2^-25 <= 2^-17 of it when not."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402

KIND = torch.float16
NAMES = ("dx", "dw_gate", "dw_up", "db_gate", "db_up")
# Few rows and few tiles run with K split, more on CTA pairs; an odd size and a whole one.
SHAPES = [(1, 40, 24), (70, 151, 88), (300, 264, 200), (1500, 1304, 2600)]


def bounds(ref, dh):
    """ref.backward's bounds with the elementwise operands' smallest step as held (KIND's)."""
    v = dh.double()
    finite = [t[t.isfinite()].abs().max() for t in (v * ref.u * ref.s, v * ref.a)]
    most = float(torch.stack(finite).max())
    tiny = fu.TINY[KIND]
    lost = tiny if 2.0 ** -8 <= most <= 65504 else most * 2.0 ** -39
    out = {}
    r = fu.HALF[KIND]
    ref.kind = torch.float32  # the operands' unrounded bounds and the biases'
    plain = ref.backward(dh)
    ref.kind = KIND
    dg, du = v * ref.u * ref.s, v * ref.a
    eg = v.abs() * (ref.u.abs() * ref.eg + 1.13 * ref.eu + 2 * ref.eg * ref.eu +
                    2.0 ** -18 * (ref.u.abs() + ref.eu))
    eu = v.abs() * (1.13 * ref.eg + 2.0 ** -19 * ref.a.abs())
    m, h = dh.shape
    for n in ("db_gate", "db_up"):
        total, e = plain[n]
        out[n] = (total, e + r * total.abs() + tiny)
    eg, eu = eg + r * dg.abs() + lost, eu + r * du.abs() + lost
    for n, w, e in (("dw_gate", dg, eg), ("dw_up", du, eu)):
        total = w.t() @ ref.x
        out[n] = (total, (e + fu.acc(m) * (w.abs() + e)).t() @ ref.x.abs() + r * total.abs() + tiny)
    total = dg @ ref.wg + du @ ref.wu
    ex = ((eg + fu.acc(2 * h) * (dg.abs() + eg)) @ ref.wg.abs() +
          (eu + fu.acc(2 * h) * (du.abs() + eu)) @ ref.wu.abs())
    out["dx"] = (total, ex + r * total.abs() + tiny)
    return out


def problem(shape, x_scale, w_scale, up_bias):
    m, h, k = shape
    x = fu.normal((m, k), KIND, 1, x_scale)
    wg, wu = (fu.normal((h, k), KIND, s, w_scale * k ** -0.5) for s in (2, 3))
    bg = fu.normal((h,), KIND, 4, 0.5)
    bu = (fu.normal((h,), KIND, 5) * up_bias).to(KIND)
    return x, wg, wu, bg, bu


def gradients(args, dh):
    _, saved = tb.gated_linear_forward(*args)
    return dict(zip(NAMES, tb.gated_linear_backward(dh, saved)))


# x, weights, the up projection's bias, dh: the operands reach 1e6 with small weights and inputs;
# they are about 2^-24 with large weights (dx fits), and with large inputs (dW fits).
CASES = {"above": (2.0 ** -9, 2.0 ** -9, 1.2e4, 16.0), "below, dx": (2.0 ** -10, 2.0 ** 6, 0.0, 2.0 ** -18),
         "below, dW": (2.0 ** 6, 2.0 ** -10, 0.0, 2.0 ** -18)}


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("shape", SHAPES)
def test_operands_outside_the_range(shape, case):
    *scales, dh_scale = CASES[case]
    args = problem(shape, *scales)
    dh = fu.normal(shape[:2], KIND, 6, dh_scale)
    ref = fu.Gated(*args, "silu", KIND)
    most = float((dh.double() * ref.u * ref.s).abs().max())
    assert most > 65520 if case == "above" else most < 2.0 ** -8  # the case is what it says
    want, got = bounds(ref, dh), gradients(args, dh)
    for n in NAMES:
        total, tol = want[n]
        fits = total.abs() + tol < 65504
        assert bool(fits.any())
        fu.within(got[n][fits], total[fits], tol[fits], n)
    again = gradients(args, dh)
    assert all(torch.equal(got[n], again[n]) for n in NAMES)
    assert xd.kernel_status() == 0


def test_special_values_do_not_set_the_scale():
    """Rows of dh with an infinity or a NaN leave the other rows' input gradients within their
    bounds, under operands above the range, inside it and below it."""
    for case in (*CASES.values(), (1.0, 1.0, 1.0, 1.0)):
        *scales, dh_scale = case
        args = problem((200, 72, 64), *scales)
        dh = fu.normal((200, 72), KIND, 6, dh_scale)
        ref = fu.Gated(*args, "silu", KIND)
        total, tol = bounds(ref, dh)["dx"]
        bad = dh.clone()
        bad[3, 5], bad[150, 0] = float("inf"), float("nan")
        rest = [r for r in range(200) if r not in (3, 150)]
        dx = gradients(args, bad)["dx"]
        fu.within(dx[rest], total[rest], tol[rest], "dx")
        assert not bool(dx[3].isfinite().any()) and bool(dx[150].isnan().all())


def test_captured_pass_chooses_its_scale_at_each_replay():
    args = problem((150, 104, 88), 2.0 ** -9, 2.0 ** -9, 1.2e4)
    dhs = [fu.normal((150, 104), KIND, 6, s) for s in (16.0, 2.0 ** -4, 2.0 ** -20)]
    _, saved = tb.gated_linear_forward(*args)
    want = [tb.gated_linear_backward(d, saved) for d in dhs]
    static = dhs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.gated_linear_backward(static, saved)
    for i in (1, 0, 2, 0):
        static.copy_(dhs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
