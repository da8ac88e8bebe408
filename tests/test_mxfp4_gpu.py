"""MXFP4 quantisation, its inverse and the linear and gated products of MXFP4 operands
(xvram_b200.torch_bridge) against 64-bit references.

Quantisation and its inverse in float32 are exact, so they are compared for equality.  A product
of two E2M1 values and two power-of-two scales is exact in FP32, so the products' error is that
of the FP32 sums (feed_util.acc) and of the result's rounding."""
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
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def blocks_of(x):
    """x in 64 bits as (rows, blocks, 32), the last block padded with zeros."""
    x = x.double()
    rows, cols = x.shape
    pad = -cols % 32
    return torch.cat([x, x.new_zeros(rows, pad)], 1).view(rows, -1, 32)


def reference(x):
    """(values, scale bytes) of x's quantisation, in 64 bits."""
    rows, cols = x.shape
    b = blocks_of(x)
    top = b.abs().amax(2)
    # The exponent field of a double is floor(log2) + 1023 (0 for zero).
    e = torch.clamp((top.view(torch.int64) >> 52) - 1023 - 2, -127, 127)
    scale = ((e + 1023) << 52).view(torch.float64)[..., None]
    a = b.abs() / scale
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    near = (a[..., None] - table).abs()
    # Distances in an order where the even code of two that are as near comes first.
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)
    value = table[order[near[..., order].argmin(-1)]]
    value = torch.where(b < 0, -value, value) * scale
    bad = ~torch.isfinite(b).all(2)
    value[bad] = float("nan")
    s = torch.where(bad, 255, e + 127)
    return value.flatten(1)[:, :cols], s


def unpacked(q):
    """(values, scale bytes) that q's bytes stand for, by the storage rule."""
    rows, cols = q.shape
    blocks = (cols + 31) // 32
    codes = q.codes.view(rows, blocks * 16).int()
    c = torch.stack([codes & 15, codes >> 4], 2).flatten(1)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64,
                         device=codes.device)
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(blocks, device=codes.device)[None]
    tiles = q.scales.view((rows + 127) // 128, (cols + 127) // 128, 512)
    s = tiles[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].long()
    scale = torch.where(s == 255, float("nan"), torch.ldexp(torch.ones_like(s, dtype=torch.float64),
                                                            s - 127))
    v = table[c.long()].view(rows, blocks, 32) * scale[..., None]
    return v.flatten(1), s


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


QUANTISED = [(1, 1), (1, 32), (2, 33), (5, 31), (128, 128), (129, 1000), (300, 96), (1, 4097)]


@pytest.mark.parametrize("shape", QUANTISED)
@pytest.mark.parametrize("kind", TYPES)
def test_quantisation_is_exact(kind, shape):
    x = fu.normal(shape, kind, 1) * torch.exp2(torch.randint(-8, 9, (shape[0], 1), device="cuda"))
    x = x.to(kind)
    q = tb.quantize_mxfp4(x)
    want, s = reference(x)
    got, scales = unpacked(q)
    assert torch.equal(scales, s)
    assert same(got[:, :shape[1]], want)
    assert not bool(got[:, shape[1]:].any())  # padding codes are zero
    for dtype in TYPES:
        back = tb.dequantize_mxfp4(q, dtype)
        assert back.dtype == dtype and back.shape == shape
        assert same(back, want.to(dtype))
    pad = q.scales.clone()
    r, b = (t.flatten() for t in torch.meshgrid(torch.arange(pad.shape[0] * 128, device="cuda"),
                                                torch.arange(pad.shape[1] * 4, device="cuda"),
                                                indexing="ij"))
    outside = (r >= shape[0]) | (b >= s.shape[1])
    v = pad[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]
    assert bool((v[outside] == 127).all())


def test_quantisation_of_special_values():
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(torch.float32).max
    rows = [[0.0] * 32,                                    # zeros: the smallest scale
            [-0.0] * 32,
            [1.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [4.0] * 23,  # ties and saturation
            [top] * 32, [-top] + [1.0] * 31,
            [2.0 ** -126] * 32, [2.0 ** -149] * 32,        # the scale's lowest value
            [2.0 ** -130, -2.0 ** -131] * 16,
            [inf] + [1.0] * 31, [nan] + [1.0] * 31, [1.0] * 31 + [-inf]]
    x = torch.tensor(rows, device="cuda")
    q = tb.quantize_mxfp4(x)
    want, s = reference(x)
    got, scales = unpacked(q)
    assert torch.equal(scales, s)
    assert same(got, want)
    assert same(tb.dequantize_mxfp4(q), want.float())


def test_quantisation_of_strided_rows():
    base = fu.normal((40, 200), torch.bfloat16, 2)
    for x in (base[:, 1:140], base[::2, :64], base.t(), base[3:4].expand(5, 200)):
        assert same(unpacked(tb.quantize_mxfp4(x))[0][:, :x.shape[1]], reference(x)[0])


SHAPES = [(1, 1, 1), (1, 8, 32), (3, 5, 7), (16, 128, 64), (128, 256, 256), (129, 257, 300),
          (130, 130, 96), (40, 700, 1000), (257, 384, 2080),
          # Up to 16 rows and 65536 values are quantised inside the product: the most rows, one row
          # and one value more, the longest rows.
          (16, 3000, 4096), (16, 300, 4097), (17, 260, 2100), (1, 130, 65536), (1, 64, 65568),
          (8, 130, 8192)]


def operands(kind, m, n, k, seed, count):
    x = fu.normal((m, k), kind, seed)
    ws = [tb.quantize_mxfp4(fu.normal((n, k), torch.float32, seed + 1 + i, k ** -0.5))
          for i in range(count)]
    return x, ws


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_linear(kind, shape):
    m, n, k = shape
    x, (w,) = operands(kind, m, n, k, 3, 1)
    bias = fu.normal((n,), kind, 9)
    xv, wv = reference(x)[0], unpacked(w)[0][:, :k]
    y = xv @ wv.t()
    e = fu.acc(k) * (xv.abs() @ wv.abs().t())
    got = tb.linear_mxfp4(x, w)
    assert got.dtype == kind and got.is_contiguous()
    fu.within(got, y, e + fu.HALF[kind] * y.abs() + fu.TINY[kind], "y")
    z = torch.relu(y + bias.double())
    got = tb.linear_mxfp4(x, w, bias, relu=True)
    fu.within(got, z, e + (2.0 ** -24 + fu.HALF[kind]) * (y + bias.double()).abs() +
              fu.TINY[kind], "relu")
    assert torch.equal(tb.linear_mxfp4(tb.quantize_mxfp4(x), w, dtype=kind), tb.linear_mxfp4(x, w))
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_gated(kind, shape):
    m, h, k = shape
    x, (wg, wu) = operands(kind, m, h, k, 4, 2)
    bg, bu = (fu.normal((h,), kind, s, 0.5) for s in (10, 11))
    xv = reference(x)[0]
    for bias in ((None, None), (bg, bu)):
        ref = fu.Gated(xv, unpacked(wg)[0][:, :k], unpacked(wu)[0][:, :k], *bias, "silu", kind)
        got = tb.gated_linear_mxfp4(x, wg, wu, *bias)
        assert got.dtype == kind
        fu.within(got, ref.h, ref.h_tol, "h")
    assert xd.kernel_status() == 0
