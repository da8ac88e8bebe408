"""The feed-forward operators as a program uses them: empty batches, streams, captured graphs,
special values, strided results, a run of several together, and gradients against differences."""
from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import feed_util as fu  # noqa: E402
from xvram_b200 import device as xd  # noqa: E402
from xvram_b200 import torch_bridge as tb  # noqa: E402
from xvram_b200._native import Gated, lib  # noqa: E402

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def weights(kind, h, k, seed):
    return [fu.normal((h, k), kind, seed + i, k ** -0.5) for i in range(2)]


@pytest.mark.parametrize("kind", TYPES)
def test_empty_batches_and_outputs(kind):
    wg, wu = (w.requires_grad_() for w in weights(kind, 24, 16, 1))
    x = torch.empty((0, 16), dtype=kind, device="cuda", requires_grad=True)
    b = torch.ones(24, dtype=kind, device="cuda", requires_grad=True)
    h = tb.gated_linear(x, wg, wu, b)
    assert h.shape == (0, 24)
    h.sum().backward()
    assert x.grad.shape == (0, 16)
    assert not bool(wg.grad.any()) and not bool(wu.grad.any()) and not bool(b.grad.any())
    none = torch.empty((0, 16), dtype=kind, device="cuda", requires_grad=True)
    y = fu.normal((3, 16), kind, 2).requires_grad_()
    tb.gated_linear(y, none, none).sum().backward()
    assert not bool(y.grad.any()) and none.grad.shape == (0, 16)
    q = tb.quantize_mxfp4(wg.detach())
    e = tb.quantize_mxfp4(x.detach())
    assert tb.linear_mxfp4(x.detach(), q).shape == (0, 24)
    assert tb.gated_linear_mxfp4(e, q, q).shape == (0, 24)
    assert tb.linear_mxfp4(y.detach(), e).shape == (3, 0)
    assert tb.dequantize_mxfp4(e).shape == (0, 16)


def test_refusals_on_the_gpu():
    x, (wg, wu) = fu.normal((2, 16), torch.bfloat16, 1), weights(torch.bfloat16, 8, 16, 2)
    with pytest.raises(ValueError, match="device"):
        tb.gated_linear(x, wg, wu.cpu())
    for bias in (torch.ones(7, device="cuda", dtype=x.dtype), torch.ones(8, device="cuda"),
                 torch.ones((8, 1), device="cuda", dtype=x.dtype)):
        with pytest.raises(ValueError, match="bias"):
            tb.gated_linear(x, wg, wu, bias)
        with pytest.raises(ValueError, match="bias"):
            tb.linear_mxfp4(x, tb.quantize_mxfp4(wg), bias)
    with pytest.raises(RuntimeError, match="no gradient"):
        tb.quantize_mxfp4(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        tb.linear_mxfp4(x.clone().requires_grad_(), tb.quantize_mxfp4(wg))
    h, saved = tb.gated_linear_forward(x, wg, wu)
    for dh in (h[:1], h.float(), h.cpu()):
        with pytest.raises(ValueError, match="dh"):
            tb.gated_linear_backward(dh, saved)
    # 16-bit operands of the C entry must be aligned for the tensor cores (more than a few rows).
    d = Gated(C.sizeof(Gated), 1, 0, 0, 0, 0, 200, 8, 16)
    big = torch.zeros(200 * 17 + 8, dtype=x.dtype, device="cuda")
    out = torch.empty((200, 8), dtype=x.dtype, device="cuda")
    d.x, d.w_gate, d.w_up = big.data_ptr(), wg.data_ptr(), wu.data_ptr()
    d.ldx, d.ld_gate, d.ld_up = 17, 16, 16
    assert lib.xvram_b200_gated_forward(C.byref(d), out.data_ptr(), 8) == 1
    d.x, d.ldx = big.data_ptr() + 2, 16
    assert lib.xvram_b200_gated_forward(C.byref(d), out.data_ptr(), 8) == 1
    d.x, d.data_type = big.data_ptr(), 2
    d.pre_gate = d.pre_up = out.data_ptr()
    d.ld_pre = 8
    assert lib.xvram_b200_gated_backward(C.byref(d), out.data_ptr(), 8, 0, 0, 0, 0, 0, 0, 0) == 1


def test_second_derivative_refused():
    x, (wg, wu) = fu.normal((2, 16), torch.float32, 1), weights(torch.float32, 8, 16, 2)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(tb.gated_linear(x, wg, wu).sum(), x, create_graph=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_streams_and_graphs(kind, m):
    """Work on a side stream, and a captured training step and MXFP4 layer replayed on new
    inputs, equal the eager results bit for bit."""
    k, h = 96, 136
    x, (wg, wu) = fu.normal((m, k), kind, 3), weights(kind, h, k, 4)
    b = fu.normal((h,), kind, 6)
    dh = fu.normal((m, h), kind, 7)
    q = [tb.quantize_mxfp4(w) for w in (wg, wu)]

    def step(x):
        y, saved = tb.gated_linear_forward(x, wg, wu, b, b, "gelu")
        return (y, *tb.gated_linear_backward(dh, saved), tb.gated_linear_mxfp4(x, *q),
                tb.linear_mxfp4(x, q[0], b, relu=True))
    new = fu.normal((m, k), kind, 8)
    want, want_new = step(x), step(new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
        got_again = step(x)
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = step(static)
    static.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    for a, b_, c, d, e in zip(want, got, got_again, want_new, out):
        assert torch.equal(a, b_) and torch.equal(a, c) and torch.equal(d, e)
    assert xd.kernel_status() == 0


def test_two_graphs_share_no_workspace():
    """Two captured steps of different inputs, replayed in turn and again, keep their results."""
    kind, m, k, h = torch.float16, 200, 72, 88
    (wg, wu) = weights(kind, h, k, 1)
    xs = [fu.normal((m, k), kind, s) for s in (2, 3)]
    dh = fu.normal((m, h), kind, 4)

    def step(x):
        y, saved = tb.gated_linear_forward(x, wg, wu)
        return (y, *tb.gated_linear_backward(dh, saved)[:3])
    want = [step(x) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i].replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [3, 20, 200])
def test_special_values_stay_in_their_rows(kind, m):
    """A NaN or an infinity in a row of x reaches that row's results and no other, and the
    results of the other rows are the same bits as without it."""
    k, h = 64, 72
    x, (wg, wu) = fu.normal((m, k), kind, 1), weights(kind, h, k, 2)
    bad = x.clone()
    bad[1, 5], bad[m - 1, 0] = float("nan"), float("inf")
    rest = [r for r in range(m) if r not in (1, m - 1)]
    q = [tb.quantize_mxfp4(w) for w in (wg, wu)]
    for f in (lambda v: tb.gated_linear(v, wg, wu), lambda v: tb.gated_linear_mxfp4(v, *q),
              lambda v: tb.linear_mxfp4(v, q[0])):
        clean, got = f(x), f(bad)
        assert torch.equal(clean[rest], got[rest])
        assert bool(got[1].isnan().all())
        assert not bool(got[m - 1].isfinite().all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [1, 9, 130])
def test_nothing_outside_the_result_is_written(kind, m):
    """Rows of a wider result, and rows behind the last, keep what they held."""
    k, h = 40, 50
    x, (wg, wu) = fu.normal((m, k), kind, 1), weights(kind, h, k, 2)
    want = tb.gated_linear(x, wg, wu)
    for ld in (h, h + 1, h + 6):
        out = torch.full((m + 3, ld), 7.0, dtype=kind, device="cuda")
        size = x.element_size()
        ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
        d = Gated(C.sizeof(Gated), {2: 0, 4: 2}[size] if kind != torch.bfloat16 else 1, 0, 0, 0, 0, m,
                  h, k, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), k, k, k)
        d.workspace, d.workspace_bytes = (ws.data_ptr() + 255) // 256 * 256, (1 << 22) - 256
        d.stream = torch.cuda.current_stream().cuda_stream
        assert lib.xvram_b200_gated_forward(C.byref(d), out.data_ptr(), ld) == 0
        assert torch.equal(out[:m, :h], want)
        assert bool((out[:m, h:] == 7).all()) and bool((out[m:] == 7).all())


def test_same_weight_twice_and_saved_tensor_change():
    kind = torch.float32
    x, (w, _) = fu.normal((5, 24), kind, 1), weights(kind, 16, 24, 2)
    w.requires_grad_()
    tb.gated_linear(x, w, w).sum().backward()
    d = w.detach().double()
    g = x.double() @ d.t()
    a, s = fu.act_and_slope(g, "silu")
    want = (g * s + a).t() @ x.double()
    assert float((w.grad.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    h = tb.gated_linear(x, w, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


@pytest.mark.parametrize("act", fu.ACTS)
def test_gradients_against_differences(act):
    """Central differences of sum(h dh) in FP32 along a random direction.  With e = 2^-7 a
    difference of the block's FP32 values (each within 2^-20 of sums of at most 40) is off by at
    most 600 2^-20 40 / 2 e < 2; divided by the largest gradient's scale that is under 2%, the third
    derivative's e^2 share under 0.1%.  The direction is the gradient itself, so the derivative is
    its squared norm."""
    kind, m, h, k = torch.float32, 20, 30, 24
    leaves = [fu.normal((m, k), kind, 1), *weights(kind, h, k, 2)]
    leaves += [fu.normal((h,), kind, 5), fu.normal((h,), kind, 6)]
    # A ReLU's kink is kept away: no pre-activation of the gate within the step.
    if act == "relu":
        leaves[3] = leaves[3] + 6.0
    dh = fu.normal((m, h), kind, 7)
    ls = [t.clone().requires_grad_() for t in leaves]
    grads = torch.autograd.grad(tb.gated_linear(*ls, activation=act), ls, dh)
    for i, g in enumerate(grads):
        n = float(g.double().norm())
        e = 2.0 ** -7
        value = []
        for sign in (1, -1):
            moved = list(leaves)
            moved[i] = leaves[i] + sign * e * g / n
            value.append(float((tb.gated_linear(*moved, activation=act).double() *
                                dh.double()).sum()))
        slope = (value[0] - value[1]) / (2 * e)
        assert abs(slope - n) <= 0.02 * n + 2.0, (act, i, slope, n)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
def test_a_run_of_layers(kind):
    """A feed-forward layer as it is trained and then served: the gated block and its gradients,
    the linear layer behind it, its weights brought to 4 bits, and both served from them."""
    m, k, h = 24, 128, 192
    x = fu.normal((m, k), kind, 1)
    wg, wu = (w.requires_grad_() for w in weights(kind, h, k, 2))
    down = fu.normal((k, h), kind, 4, h ** -0.5)
    hid = tb.gated_linear(x, wg, wu)
    y = tb.linear(hid.detach(), down)
    want = fu.Gated(x, wg, wu, None, None, "silu", kind)
    fu.within(hid.detach(), want.h, want.h_tol, "hidden")
    r = hid.detach().double() @ down.double().t()
    fu.within(y, r, 1e-6 * h * float(hid.detach().abs().max()) * float(down.abs().max()) +
              fu.HALF[kind] * r.abs(), "down")
    dh = fu.normal((m, h), kind, 5)
    hid.backward(dh)
    for n, t in (("dw_gate", wg), ("dw_up", wu)):
        fu.within(t.grad, *want.backward(dh)[n], n)
    with torch.no_grad():
        for w in (wg, wu):
            w -= 0.01 * w.grad
    q = [tb.quantize_mxfp4(w.detach()) for w in (wg, wu, down)]
    v = [tb.dequantize_mxfp4(t).double() for t in q]
    hq = tb.gated_linear_mxfp4(x, q[0], q[1])
    xv = tb.dequantize_mxfp4(tb.quantize_mxfp4(x)).double()
    ref = fu.Gated(xv, v[0], v[1], None, None, "silu", kind)
    fu.within(hq, ref.h, ref.h_tol, "4-bit hidden")
    hv = tb.dequantize_mxfp4(tb.quantize_mxfp4(hq)).double()
    yq = tb.linear_mxfp4(hq, q[2])
    ref = hv @ v[2].t()
    fu.within(yq, ref, fu.acc(h) * (hv.abs() @ v[2].abs().t()) + fu.HALF[kind] * ref.abs() +
              fu.TINY[kind], "4-bit down")
    assert xd.kernel_status() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_only_the_wanted_gradients(kind):
    """Each subset of the gradients has the bits that all of them together have."""
    x, (wg, wu) = fu.normal((150, 88), kind, 1), weights(kind, 104, 88, 2)
    b = fu.normal((104,), kind, 4)
    dh = fu.normal((150, 104), kind, 5)
    _, saved = tb.gated_linear_forward(x, wg, wu, b, b, "gelu_tanh")
    want = tb.gated_linear_backward(dh, saved)
    for bits in range(32):
        needs = tuple(bool(bits >> i & 1) for i in range(5))
        got = tb.gated_linear_backward(dh, saved, needs)
        for n, g, w in zip(needs, got, want):
            assert (g is None) if not n else torch.equal(g, w)
    frozen = wg.clone().requires_grad_()  # autograd asks for one weight's gradient alone
    tb.gated_linear(x, frozen, wu, b, b, "gelu_tanh").backward(dh)
    assert torch.equal(frozen.grad, want[1])


@pytest.mark.parametrize("kind", TYPES)
def test_empty_batches_of_odd_sizes(kind):
    x = torch.empty((0, 9), dtype=kind, device="cuda", requires_grad=True)
    wg, wu = (w.requires_grad_() for w in weights(kind, 7, 9, 1))
    tb.gated_linear(x, wg, wu).sum().backward()
    assert x.grad.shape == (0, 9) and not bool(wg.grad.any()) and not bool(wu.grad.any())
    q = tb.quantize_mxfp4(wg.detach())
    assert tb.gated_linear_mxfp4(x.detach(), q, q).shape == (0, 7)


def test_two_threads_at_once():
    """Calls from two host threads on streams of their own give what they give alone."""
    import threading
    kind = torch.bfloat16
    x, (wg, wu) = fu.normal((60, 136), kind, 1), weights(kind, 264, 136, 2)
    q = [tb.quantize_mxfp4(w) for w in (wg, wu)]
    want = (tb.gated_linear(x, wg, wu), tb.gated_linear_mxfp4(x, *q), tb.linear_mxfp4(x[:3], q[0]))
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                got = (tb.gated_linear(x, wg, wu), tb.gated_linear_mxfp4(x, *q),
                       tb.linear_mxfp4(x[:3], q[0]))
                s.synchronize()
                wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and xd.kernel_status() == 0
