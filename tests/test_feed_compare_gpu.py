"""Comparisons over the forms of the feed-forward operators: every activation on every kernel, NaN
scales in 4-bit weights, and the block's gradients against differences with bounds of their own.
Bounds are feed_util's unless a test derives others."""
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
# Few rows, up to 128 rows, more rows; sizes that end inside tiles, blocks and 16 bytes.
ROWS = [1, 16, 90, 300]


def operands(kind, m, h, k, seed):
    x = fu.normal((m, k), kind, seed, 2.0)
    ws = [fu.normal((h, k), kind, seed + i, k ** -0.5) for i in (1, 2)]
    return x, *ws, *(fu.normal((h,), kind, seed + i, 0.5) for i in (3, 4))


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("act", fu.ACTS)
@pytest.mark.parametrize("kind", TYPES)
def test_each_activation_of_the_block(kind, act, m):
    for h, k in ((136, 200), (77, 65)):
        args = operands(kind, m, h, k, 10)
        for bias in (args[3:], (None, None)):
            ref = fu.Gated(*args[:3], *bias, act, kind)
            fu.within(tb.gated_linear(*args[:3], *bias, activation=act), ref.h, ref.h_tol, act)
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("act", fu.ACTS)
@pytest.mark.parametrize("kind", TYPES)
def test_each_activation_of_the_4_bit_block(kind, act, m):
    for h, k in ((136, 320), (261, 1001)):
        x, wg, wu, *bias = operands(kind, m, h, k, 20)
        q = [tb.quantize_mxfp4(w) for w in (wg, wu)]
        xv, *wv = (tb.dequantize_mxfp4(t) for t in (tb.quantize_mxfp4(x), *q))
        for b in (bias, (None, None)):
            ref = fu.Gated(xv, *wv, *b, act, kind)
            fu.within(tb.gated_linear_mxfp4(x, *q, *b, activation=act), ref.h, ref.h_tol, act)
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("kind", TYPES)
def test_nan_scales_in_weights(kind, m):
    """A weight block whose scale byte is 255 is NaN: its feature is NaN in every row, also where x is
    zero in that block, and every other feature has the bits that it has without."""
    h, k = 150, 200
    x, wg, wu, *_ = operands(kind, m, h, k, 30)
    x[:, 64:96] = 0
    clean = [tb.quantize_mxfp4(w) for w in (wg, wu)]
    for row, value in ((3, float("nan")), (149, float("inf"))):
        w = wg.clone()
        w[row, 70] = value
        q = tb.quantize_mxfp4(w)
        assert int((q.scales == 255).sum()) == 1
        others = [r for r in range(h) if r != row]
        for got, want in ((tb.linear_mxfp4(x, q), tb.linear_mxfp4(x, clean[0])),
                          (tb.linear_mxfp4(x, q, relu=True), tb.linear_mxfp4(x, clean[0], relu=True)),
                          (tb.gated_linear_mxfp4(x, q, clean[1]), tb.gated_linear_mxfp4(x, *clean)),
                          (tb.gated_linear_mxfp4(x, clean[1], q),
                           tb.gated_linear_mxfp4(x, clean[1], clean[0]))):
            assert bool(got[:, row].isnan().all())
            assert torch.equal(got[:, others], want[:, others])
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("act", fu.ACTS)
def test_gradients_against_close_differences(act):
    """Central differences of f = sum(h dh) along each gradient's own direction, so that the
    derivative is its norm n.  The difference quotient over 2 e is off by
      * the block's error in the two values: (B+ + B-) / 2 e with B = sum |dh| h_tol;
      * the moved leaf's rounding to FP32, half a step of each element: n 2^-24 |leaf| / e;
      * the curve: from 64-bit differences over e and e / 2, whose gap is 3/4 of the first's e^2 term:
        2 gaps;
      * n's own error: the norm of the gradient's bounds.
    Together they stay below 2% of n, so a gradient that is 2% too large or too small is seen."""
    kind, m, h, k, e = torch.float32, 20, 30, 24, 2.0 ** -3
    leaves = [fu.normal((m, k), kind, 1)]
    leaves += [fu.normal((h, k), kind, s, k ** -0.5) for s in (2, 3)]
    leaves += [fu.normal((h,), kind, s) for s in (5, 6)]
    if act == "relu":  # the kink out of reach
        leaves[3] = leaves[3] + 8.0
    dh = fu.normal((m, h), kind, 7)
    ls = [t.clone().requires_grad_() for t in leaves]
    grads = torch.autograd.grad(tb.gated_linear(*ls, activation=act), ls, dh)
    limits = fu.Gated(*leaves, act, kind).backward(dh)
    for i, (name, g) in enumerate(zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), grads)):
        n = float(g.double().norm())
        direction = g.double() / n

        def exact(step):
            moved = [t.double() for t in leaves]
            moved[i] = moved[i] + step * direction
            ref = fu.Gated(*moved, act, kind)
            if act == "relu":
                assert float(ref.g.min()) > 0
            return float((ref.h * dh.double()).sum())
        value, error = [], n * 2.0 ** -24 * float(leaves[i].double().norm() + e) / e
        for sign in (1, -1):
            moved = list(leaves)
            moved[i] = (leaves[i].double() + sign * e * direction).float()
            ref = fu.Gated(*moved, act, kind)
            value.append(float((tb.gated_linear(*moved, activation=act).double() * dh.double()).sum()))
            error += float((ref.h_tol * dh.double().abs()).sum()) / (2 * e)
        wide, close = ((exact(s) - exact(-s)) / (2 * s) for s in (e, e / 2))
        error += 2 * abs(wide - close) + float(limits[name][1].norm())
        assert error <= 0.02 * n, (act, name, error, n)
        assert abs((value[0] - value[1]) / (2 * e) - n) <= error, (act, name, value, n, error)
