"""The gated feed-forward block (xvram_b200.torch_bridge.gated_linear) and its gradients
against 64-bit references, with the bounds that feed_util derives."""
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
# (batch, out, in): one element, fewer than a tile, whole tiles, one past them, long sums.
SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (128, 128, 64), (129, 257, 65), (5, 300, 1000),
          (257, 136, 520)]


def problem(kind, m, h, k, seed=0, bias=True):
    x = fu.normal((m, k), kind, seed)
    wg, wu = (fu.normal((h, k), kind, seed + i, k ** -0.5) for i in (1, 2))
    bg, bu = (fu.normal((h,), kind, seed + i, 0.5) if bias else None for i in (3, 4))
    return x, wg, wu, bg, bu


def check_forward(args, act):
    ref = fu.Gated(*args, act, args[0].dtype)
    got = tb.gated_linear(*args, activation=act)
    assert got.dtype == args[0].dtype and got.is_contiguous()
    fu.within(got, ref.h, ref.h_tol, "h")
    assert xd.kernel_status() == 0
    return got


def check_gradients(args, act, dh):
    ref = fu.Gated(*args, act, args[0].dtype)
    leaves = [None if t is None else t.detach().requires_grad_() for t in args]
    h = tb.gated_linear(*leaves, activation=act)
    fu.within(h.detach(), ref.h, ref.h_tol, "h")
    h.backward(dh)
    want = ref.backward(dh)
    for n, t in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), leaves):
        if t is not None:
            fu.within(t.grad, *want[n], n)
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_forward(kind, shape):
    check_forward(problem(kind, *shape), "silu")


@pytest.mark.parametrize("act", fu.ACTS)
@pytest.mark.parametrize("kind", TYPES)
def test_forward_activations_without_bias(kind, act):
    check_forward(problem(kind, 33, 72, 96, 5, bias=False), act)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_gradients(kind, shape):
    m, h, k = shape
    check_gradients(problem(kind, m, h, k, 10), "silu", fu.normal((m, h), kind, 20))


@pytest.mark.parametrize("act", fu.ACTS)
@pytest.mark.parametrize("kind", TYPES)
def test_gradients_of_each_activation(kind, act):
    check_gradients(problem(kind, 70, 144, 40, 30), act, fu.normal((70, 144), kind, 31))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_more_tiles_than_the_gpu_holds(kind):
    """Each resident CTA pair walks several tiles, in the forward and in both gradient products."""
    m, h, k = 2200, 1500, 2050
    check_gradients(problem(kind, m, h, k, 40), "gelu_tanh", fu.normal((m, h), kind, 41))


def layouts(t):
    """The same matrix as rows, as columns, inside a larger one at an odd place, and with no
    contiguous axis."""
    r, c = t.shape
    big = t.new_zeros((r + 2, c + 3))
    big[1:r + 1, 1:c + 1] = t
    tall = t.new_zeros((c + 1, r + 5))
    tall[1:, 3:r + 3] = t.t()
    wide = t.new_zeros((r, 2 * c))
    wide[:, ::2] = t
    return [t, t.t().contiguous().t(), big[1:r + 1, 1:c + 1], tall[1:, 3:r + 3].t(), wide[:, ::2]]


@pytest.mark.parametrize("shape", [(3, 40, 56), (200, 72, 64), (1, 9, 5), (70, 1, 33), (40, 8, 1)])
@pytest.mark.parametrize("kind", TYPES)
def test_every_operand_layout(kind, shape):
    m, h, k = shape
    x, wg, wu, bg, bu = problem(kind, m, h, k, 50)
    dh = fu.normal((m, h), kind, 51)
    for xv in layouts(x):
        check_gradients((xv, wg, wu, bg, bu), "silu", dh)
    for g, u in zip(layouts(wg), layouts(wu)):
        check_forward((x, g, u, bg, bu), "silu")
        check_gradients((x, g, u, bg, bu), "silu", dh)
    check_gradients((x, wg, layouts(wu)[1], bg, bu), "silu", dh)  # stored in different ways
    for dhv in layouts(dh)[1:] + [dh[:1].expand(m, h)]:
        check_gradients((x, wg, wu, bg, bu), "silu", dhv)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 6, 7, 8, 9, 17])
@pytest.mark.parametrize("kind", TYPES)
def test_each_number_of_few_rows(kind, m):
    """One or two features per warp, rows of whole 16 bytes, with a rest, and unaligned."""
    for h, k in ((40, 512), (40, 516), (2400, 515), (2401, 264)):
        check_forward(problem(kind, m, h, k, 60 + m), "silu")


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(140, 4000, 300), (300, 2100, 520), (1021, 2730, 77)])
def test_gradients_with_few_tiles_and_a_long_sum(kind, shape):
    """dx has few tiles and K = 2 out: it runs over several row tiles with K split."""
    m, h, k = shape
    check_gradients(problem(kind, m, h, k, 70), "sigmoid", fu.normal((m, h), kind, 71))
