"""PyTorch tiled-GEMM bridge: `mm` and `linear` on this library's kernels.

The reference routes bias-free `mm` / `linear` of torch graphs whose working set exceeds
the device budget through its native tiled GEMM (reference
python/xvram/torch_native.py:1876-1935, `_submit_tiled_gemm` / `_make_gemm_problem`).
This bridge serves the same two operations, B200-side:

* CUDA tensors run in HBM through `xvram_b200_sgemm_device` (float32) or
  `xvram_b200_gemm_device_typed` (the other types) on torch's current stream.
  Row-major (C-contiguous) and column-major (transposed) views are passed as the matching
  column-major operand and operation, so no copy is made for either.
* Host tensors run out of core through an SDK session (`xvram_get_api`): the operands
  live in page-locked host memory and stream through the session's device budget, as in
  the reference's oversized path.
* `linear` takes a bias and a ReLU (the reference's route refuses biased linear layers,
  torch_native.py:1913-1921); on the GPU they are one pass of `xvram_b200_bias_activation`
  over the output.

Element types are the reference route's (python/xvram/torch_native.py:95-100): float32,
and float16 / bfloat16 / float64 matrices of one type, with the result in that type --
FP16 / BF16 under strict FP32 arithmetic (the products are exact in FP32, the result is
rounded to the type once), FP64 in FP64.  `tensor_cores=True` selects the three-term TF32
kernel for float32 (FP32-accurate within max|err| / (K max|a| max|b|) <= 1e-6); the
default is strict FP32 FFMA.  Bias and ReLU are float32 only (the reference route takes
neither).  There is no CPU fallback: without a GPU every call raises.

Beside `linear` stand the feed-forward operators (the reference has none of them), for CUDA
tensors:

* `gated_linear`, the gated block act(x Wg^T + bg) * (x Wu^T + bu), differentiable, and its
  explicit forms `gated_linear_forward` / `gated_linear_backward`;
* `quantize_mxfp4` / `dequantize_mxfp4` and `Mxfp4Matrix`, microscaled 4-bit matrices, with
  `linear_mxfp4` and `gated_linear_mxfp4`, the same layers over 4-bit operands.
"""
from __future__ import annotations

import atexit
import contextlib
import ctypes
import threading

import torch
from torch.autograd import forward_ad

from . import device as xd
from . import sdk
from ._native import Gated, Mxfp4Product, Pack, lib

_TF32X3 = 3
_TYPES = {torch.float16: sdk.FP16, torch.bfloat16: sdk.BF16, torch.float32: sdk.FP32,
          torch.float64: sdk.FP64}


def _dtype_of(a: torch.Tensor, b: torch.Tensor) -> torch.dtype:
    if a.dtype != b.dtype or a.dtype not in _TYPES:
        raise TypeError("mm supports float16, bfloat16, float32 and float64 matrices of one "
                        f"type (got {a.dtype} and {b.dtype})")
    return a.dtype


def _colmajor(x: torch.Tensor):
    """(storage is op(S) of a column-major S, ld, op): a row-major (r, c) tensor is the
    column-major (c, r) matrix transposed."""
    if x.dim() != 2:
        raise ValueError("expected a 2-D tensor")
    r, c = x.shape
    s0, s1 = x.stride()
    if s1 == 1 and s0 >= max(c, 1):
        return x, s0, 1          # row-major: column-major X^T, ld = row stride, op T
    if s0 == 1 and s1 >= max(r, 1):
        return x, s1, 0          # column-major: X itself, op N
    x = x.contiguous()
    return x, max(c, 1), 1


def _check(st: int, what: str) -> None:
    if st != 0:
        raise RuntimeError(f"{what} failed with xvram_status {st}")


def mm(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None,
       tensor_cores: bool = False) -> torch.Tensor:
    """a @ b for (m x k) @ (k x n) matrices of one floating type, on the device the
    tensors are on; the result has that type."""
    dtype = _dtype_of(a, b)
    if tensor_cores and dtype != torch.float32:
        raise TypeError("tensor_cores applies to float32 matrices")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"shapes {tuple(a.shape)} and {tuple(b.shape)} do not multiply")
    if a.device != b.device:
        raise ValueError("a and b must be on the same device")
    if a.device.type != "cuda":
        return _host_session().mm(a, b, out, tensor_cores)
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=a.device)
    elif out.shape != (m, n) or not out.is_contiguous() or out.dtype != dtype:
        raise ValueError(f"out must be a contiguous {dtype} (m, n) tensor")
    if m == 0 or n == 0:
        return out
    if k == 0:
        return out.zero_()
    # Row-major C (m x n) is column-major C^T (n x m) = op(B)^T op(A)^T.
    bs, ldb, ob = _colmajor(b)       # b as op_b(S_b): b = S_b^T when ob == 1
    as_, lda, oa = _colmajor(a)
    # C^T = b^T a^T: the first operand is b^T = op(S_b) with the operation flipped, etc.
    if dtype == torch.float32:
        st = xd.sgemm(1 - ob, 1 - oa, n, m, k, 1.0, bs, ldb, as_, lda, 0.0, out, n,
                      path=_TF32X3 if tensor_cores else 0)
        _check(st, "xvram_b200_sgemm_device")
    else:
        st = xd.gemm_typed(1 - ob, 1 - oa, n, m, k, 1.0, bs, ldb, as_, lda, 0.0, out, n)
        _check(st, "xvram_b200_gemm_device_typed")
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           relu: bool = False, tensor_cores: bool = False) -> torch.Tensor:
    """x @ weight^T (+ bias) (then ReLU), x: (batch, in), weight: (out, in)."""
    if (bias is not None or relu) and x.dtype != torch.float32:
        raise TypeError("bias and ReLU apply to float32 matrices")
    if x.device.type != "cuda":
        return _host_session().linear(x, weight, bias, relu, tensor_cores)
    y = mm(x, weight.t(), tensor_cores=tensor_cores)
    if bias is not None or relu:
        if bias is not None and (bias.dtype != torch.float32 or bias.numel() != y.shape[1]):
            raise ValueError("bias must be float32 with one value per output feature")
        b = bias.contiguous() if bias is not None else None
        # y is row-major (batch, out) = column-major (out, batch): bias runs along rows.
        st = xd.bias_activation(y, y.shape[1], y.shape[1], y.shape[0], b, relu)
        _check(st, "xvram_b200_bias_activation")
    return y


# ---------------------------------------------------------------- feed-forward operators
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}
_HERE = contextlib.nullcontext()
_FEED_TYPES = {torch.float16: sdk.FP16, torch.bfloat16: sdk.BF16, torch.float32: sdk.FP32}


def _activation(name: str) -> int:
    act = ACTIVATIONS.get(name)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)} (got {name!r})")
    return act


def _on_device(index: int):
    """Makes device `index` current for the library's calls, which use the current device."""
    return _HERE if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


# The stream handle itself: building torch's Stream object costs 2 us of a call of 10.
_stream = torch._C._cuda_getCurrentRawStream if hasattr(
    torch._C, "_cuda_getCurrentRawStream") else (
        lambda index: torch.cuda.current_stream(index).cuda_stream)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _dual_level() -> bool:
    """Whether a forward-mode level is open.  Outside one no tensor has a tangent."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def _refuse_tangents(what: str, *tensors) -> None:
    """Forward-mode derivatives are not implemented, and a result without a tangent would read
    as a zero derivative."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None
           for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _operand(x: torch.Tensor, r: int, c: int, per: int, aligned: bool):
    """(leading dimension, transposed, padded) of x as the kernels read it.  padded: x must be
    copied with rows (or, transposed, columns) of whole 16 bytes first.  `per`: elements in 16
    bytes; `aligned`: rows must be multiples of them.  (None, ...): neither rows nor columns are
    contiguous, which a contiguous x never answers."""
    s0, s1 = x.stride()
    # Strides of empty tensors and of sizes of one are never used, and torch leaves them as they
    # are, in what it calls contiguous too.
    if r == 0:
        return (c + per - 1) // per * per, 0, False
    if c == 1:
        s1 = 1
    if s1 == 1 and (s0 >= c or r == 1):
        if r == 1:
            s0 = (c + per - 1) // per * per
        if not aligned or (s0 % per == 0 and x.data_ptr() % 16 == 0):
            return s0, 0, False
        return (c + per - 1) // per * per, 0, True
    if s0 == 1 and s1 >= r:
        if not aligned or (s1 % per == 0 and x.data_ptr() % 16 == 0):
            return s1, 1, False
        return (r + per - 1) // per * per, 1, True
    return None, 0, False


def _pack(padded: list, like: torch.Tensor, per: int, kind: int, index: int):
    """Copies (tensor, rows, leading dimension, transposed) with padded rows into one buffer, in
    one launch: (buffer, each copy's element offset)."""
    offsets, end = [], 0
    for _, rows, ld, _ in padded:
        offsets.append(end)
        end += rows * ld
    buffer = like.new_empty(end)
    base, size = buffer.data_ptr(), 16 // per
    items = (Pack * len(padded))()
    for item, (x, rows, ld, transposed), off in zip(items, padded, offsets):
        s0, s1 = x.stride()
        r, c = x.shape
        item.src, item.dst, item.ld_dst = x.data_ptr(), base + off * size, ld
        item.ld_src, item.rows, item.cols = (s1, c, r) if transposed else (s0, r, c)
    _check(lib.xvram_b200_pack_rows(kind, items, len(padded), _stream(index)),
           "xvram_b200_pack_rows")
    return buffer, offsets


_GATED_SIZE = ctypes.sizeof(Gated)
# Up to 16 rows of 65536 values together (XVRAM_B200_MXFP4_DIRECT_*) may be quantised inside the
# product; up to half of these values that is taken as it is, and above the library chooses, for
# which it needs memory for the codes.
_DIRECT_ROWS, _DIRECT_VALUES = 16, 32768
_PRODUCT_SIZE = ctypes.sizeof(Mxfp4Product)


def _check_bias(b: torch.Tensor, h: int, dtype: torch.dtype, device: torch.device, name: str):
    if b.dtype != dtype or b.device != device or b.dim() != 1 or b.numel() != h:
        raise ValueError(f"{name} must hold {h} values of the result's type on its device")
    return (b.resolve_neg() if h == 1 else b).contiguous()


def _check_gated(x, w_gate, w_up, dtype: torch.dtype, device: torch.device) -> None:
    if dtype not in _FEED_TYPES or w_gate.dtype != dtype or w_up.dtype != dtype:
        raise TypeError("gated_linear supports float16, bfloat16 and float32 matrices of one type "
                        f"(got {dtype}, {w_gate.dtype} and {w_up.dtype})")
    xs, gs = x.shape, w_gate.shape
    if len(xs) != 2 or len(gs) != 2 or gs != w_up.shape or xs[1] != gs[1]:
        raise ValueError(f"x (batch, in) and two (out, in) weights expected (got {tuple(xs)}, "
                         f"{tuple(gs)} and {tuple(w_up.shape)})")
    if xs[1] == 0:
        raise ValueError("gated_linear needs at least one input feature")
    if device.type != "cuda":
        raise RuntimeError("gated_linear needs CUDA tensors (there is no CPU path)")
    if w_gate.device != device or w_up.device != device:
        raise ValueError("x and the weights must be on the same device")


class GatedSaved:
    """What `gated_linear_backward` needs of a forward pass: x, w_gate and w_up (or copies that
    the kernels read without another one; the caller's own must not be changed in between) and the
    FP32 pre-activations (2, batch, out padded to whole 16 bytes), the problem (element type,
    activation, batch, out, in, torch type, device), and where the three are padded copies in one
    buffer, its size and their places."""
    __slots__ = ("tensors", "problem", "places")

    def __init__(self, tensors, problem, places):
        self.tensors, self.problem, self.places = tensors, problem, places


# Up to _FEW_ROWS rows of 16-bit values run on the forward's few-rows kernel, which reads rows from
# any element on, while a weight has at most _FEW_VALUES values; one row always does.
_FEW_ROWS, _FEW_VALUES = 4, 1 << 23


def _operands(x, w_gate, w_up, per: int, aligned: bool, kind: int, index: int, few: bool = False):
    """x and the weights as the kernels read them, and their places: each one's element offset
    and leading dimension, and whether x and the weights are transposed; then which of the
    three are padded copies in one buffer, those being the buffer.  Not padded: the tensor itself
    or a contiguous copy.  `few`: the few-rows kernel may take the operands."""
    (m, k), h = x.shape, w_gate.shape[0]
    if k == 1:
        # The imaginary part of a conjugate stands for its memory's negative.  Its elements are
        # never neighbours, so that it is copied below unless the stride does not count.
        x, w_gate, w_up = x.resolve_neg(), w_gate.resolve_neg(), w_up.resolve_neg()
    ldx, xt, px = _operand(x, m, k, per, aligned)
    ldg, gt, pg = _operand(w_gate, h, k, per, aligned)
    ldu, ut, pu = _operand(w_up, h, k, per, aligned)
    if ldx is None or ldg is None or ldu is None or gt != ut:
        # Neither rows nor columns contiguous, or weights stored in different ways.
        x, w_gate, w_up = x.contiguous(), w_gate.contiguous(), w_up.contiguous()
        ldx, xt, px = _operand(x, m, k, per, aligned)
        ldg, gt, pg = _operand(w_gate, h, k, per, aligned)
        ldu, ut, pu = _operand(w_up, h, k, per, aligned)
    if few and (pg or pu) and not xt and not gt:
        # Copying the weights costs more than reading them by elements (BF16, 1 x 2047 x 4099: 22.1
        # us against 13.7, 1 x 4095 x 8192 76 against 36, 4 x 1001 x 2730 13.6 against 8.6); copying x
        # alone does not.
        (ldx, _, px), (ldg, _, pg), (ldu, _, pu) = (
            _operand(t, t.shape[0], k, per, False) for t in (x, w_gate, w_up))
    ox = og = ou = 0
    if px or pg or pu:
        padded = [t for p, t in ((px, (x, k if xt else m, ldx, xt)),
                                 (pg, (w_gate, k if gt else h, ldg, gt)),
                                 (pu, (w_up, k if gt else h, ldu, gt))) if p]
        buffer, offsets = _pack(padded, x, per, kind, index)
        if px:
            x, ox = buffer, offsets.pop(0)
        if pg:
            w_gate, og = buffer, offsets.pop(0)
        if pu:
            w_up, ou = buffer, offsets.pop(0)
    return x, w_gate, w_up, (ox, ldx, og, ldg, ou, ldu, xt, gt), (px, pg, pu)


def _gated_forward(x, w_gate, w_up, bias_gate, bias_up, activation: str, keep: bool):
    act = _activation(activation)
    dtype, device = x.dtype, x.device
    _check_gated(x, w_gate, w_up, dtype, device)
    kind, index = _FEED_TYPES[dtype], device.index
    (m, k), h = x.shape, w_gate.shape[0]
    if bias_gate is not None:
        bias_gate = _check_bias(bias_gate, h, dtype, device, "bias_gate")
    if bias_up is not None:
        bias_up = _check_bias(bias_up, h, dtype, device, "bias_up")
    per = 4 if kind == sdk.FP32 else 8
    # The float32 GEMM reads any operand, but unaligned ones several times slower than it takes to
    # copy them; its few-rows kernel reads them at full speed.  The backward needs them aligned.
    aligned = kind != sdk.FP32 or keep or m > 32
    few = kind != sdk.FP32 and not keep and (m == 1 or (m <= _FEW_ROWS and h * k <= _FEW_VALUES))
    with _on_device(index):
        x, w_gate, w_up, places, padded = _operands(x, w_gate, w_up, per, aligned, kind, index, few)
        ox, ldx, og, ldg, ou, ldu, xt, wt = places
        out = x.new_empty((m, h))
        pre, pg0, pu0, ldp = None, 0, 0, 0
        if keep:
            ldp = (h + 3) // 4 * 4
            pre = x.new_empty((2, m, ldp), dtype=torch.float32)
            pg0 = pre.data_ptr()
            pu0 = pg0 + m * ldp * 4
        size = 16 // per
        d = Gated(_GATED_SIZE, kind, act, xt, wt, 0, m, h, k, x.data_ptr() + ox * size,
                  w_gate.data_ptr() + og * size, w_up.data_ptr() + ou * size, ldx, ldg, ldu,
                  0 if bias_gate is None else bias_gate.data_ptr(),
                  0 if bias_up is None else bias_up.data_ptr(), pg0, pu0, ldp, 0, 0,
                  _stream(index))
        ws = _gated_workspace(d, 0, x) if kind == sdk.FP32 else None  # noqa: F841  (alive here)
        st = lib.xvram_b200_gated_forward(ctypes.byref(d), out.data_ptr(), h)
        if st:
            _check(st, "xvram_b200_gated_forward")
    if not keep:
        return out, None
    problem = (kind, act, m, h, k, dtype, device)
    if all(padded):
        return out, GatedSaved((x, pre), problem, (x.numel(), places))
    saved = [t.as_strided((r, k), (1, ld) if tr else (ld, 1), o) if p else t
             for t, r, o, ld, tr, p in ((x, m, ox, ldx, xt, padded[0]),
                                        (w_gate, h, og, ldg, wt, padded[1]),
                                        (w_up, h, ou, ldu, wt, padded[2]))]
    return out, GatedSaved((*saved, pre), problem, None)


def _gated_workspace(d, backward: int, like: torch.Tensor):
    need = lib.xvram_b200_gated_workspace_bytes(ctypes.byref(d), backward)
    if not need:
        return None
    ws = like.new_empty((need + 256,), dtype=torch.uint8)
    d.workspace = (ws.data_ptr() + 255) // 256 * 256
    d.workspace_bytes = need
    return ws


def gated_linear_forward(x, w_gate, w_up, bias_gate=None, bias_up=None, activation="silu"):
    """(h, saved): the gated block's result and what `gated_linear_backward` needs.  For callers
    that drive the backward pass themselves; autograd is not involved."""
    if _dual_level():
        _refuse_tangents("gated_linear", x, w_gate, w_up, bias_gate, bias_up)
    with torch.no_grad():
        return _gated_forward(x, w_gate, w_up, bias_gate, bias_up, activation, True)


def gated_linear_backward(dh: torch.Tensor, saved: GatedSaved,
                          needs=(True, True, True, True, True)):
    """Gradients (dx, dw_gate, dw_up, db_gate, db_up) of the block from dh = dL/dh; those that
    `needs` does not ask for are None.  Sums are FP32; for float16 / bfloat16 the gradients of the
    pre-activations are rounded to the type once, as the tensor cores' operands (float16: times a
    power of two where its range would lose them, so that gradients which fit are right)."""
    if _dual_level():
        _refuse_tangents("gated_linear's backward", dh)
    kind, act, m, h, k, dtype, device = saved.problem
    *operands, pre = saved.tensors
    places = saved.places
    # Strides are read from the tensors: autograd's saved-tensor hooks may have changed them.
    ldp = (h + 3) // 4 * 4
    shapes = ((m, k), (h, k), (h, k)) if places is None else ((places[0],),)
    for t, shape, of in (*zip(operands, shapes, (dtype, dtype, dtype)),
                         (pre, (2, m, ldp), torch.float32)):
        if t.shape != shape or t.dtype != of or t.device != device:
            raise RuntimeError(f"a saved tensor of gated_linear must be {shape} {of} on {device} "
                               f"(got {tuple(t.shape)} {t.dtype} on {t.device})")
    if dh.shape != (m, h) or dh.dtype != dtype or dh.device != device:
        raise ValueError(f"dh must be a ({m}, {h}) {dtype} tensor on {device}")
    index, size = device.index, 4 if kind == sdk.FP32 else 2
    with _on_device(index):
        if not pre.is_contiguous() or pre.data_ptr() % 16:
            pre = pre.clone(memory_format=torch.contiguous_format)
        if places is None:
            x, w_gate, w_up, place, _ = _operands(*operands, 16 // size, True, kind, index)
        else:
            x, place = operands[0], places[1]
            if not x.is_contiguous() or x.data_ptr() % 16:
                x = x.clone(memory_format=torch.contiguous_format)
            w_gate = w_up = x
        ox, ldx, og, ldg, ou, ldu, xt, wt = place
        dh, lddh = _rows(dh.detach() if dh.requires_grad else dh)
        dx = dh.new_empty((m, k)) if needs[0] else None
        dwg = dh.new_empty((h, k)) if needs[1] else None
        dwu = dh.new_empty((h, k)) if needs[2] else None
        dbg = dh.new_empty((h,)) if needs[3] else None
        dbu = dh.new_empty((h,)) if needs[4] else None
        pg0 = pre.data_ptr()
        d = Gated(_GATED_SIZE, kind, act, xt, wt, 0, m, h, k, x.data_ptr() + ox * size,
                  w_gate.data_ptr() + og * size, w_up.data_ptr() + ou * size, ldx, ldg, ldu, 0, 0,
                  pg0, pg0 + m * ldp * 4, ldp, 0, 0, _stream(index))
        ws = _gated_workspace(d, 1, dh)  # noqa: F841  (alive until the launches)
        _check(lib.xvram_b200_gated_backward(ctypes.byref(d), dh.data_ptr(), lddh, _ptr(dx), k,
                                             _ptr(dwg), _ptr(dwu), k, _ptr(dbg), _ptr(dbu)),
               "xvram_b200_gated_backward")
    return dx, dwg, dwu, dbg, dbu


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, bias_gate, bias_up, activation):
        out, saved = _gated_forward(x, w_gate, w_up, bias_gate, bias_up, activation, True)
        ctx.save_for_backward(*saved.tensors)
        ctx.problem, ctx.places = saved.problem, saved.places
        return out

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("gated_linear has no second derivative")
        saved = GatedSaved(ctx.saved_tensors, ctx.problem, ctx.places)
        return (*gated_linear_backward(dh, saved, ctx.needs_input_grad), None)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 bias_gate: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
                 activation: str = "silu") -> torch.Tensor:
    """act(x @ w_gate^T + bias_gate) * (x @ w_up^T + bias_up), x: (batch, in), weights:
    (out, in), on CUDA tensors of one type (float16, bfloat16 or float32); activation: silu,
    gelu, gelu_tanh, relu or sigmoid.  float16 / bfloat16 run as one tensor-core kernel with FP32
    accumulation and one rounding, float32 in strict FP32.  Row-major and transposed operands
    are read in place (16-bit ones where their base and leading dimension are multiples of 16
    bytes; others are copied first, unless the call runs on the few-rows kernel: one row, or up to
    four with weights of up to 2^23 values).  Differentiable once in every tensor argument, in
    reverse mode; tensors with a forward-mode tangent are refused."""
    if _dual_level():
        _refuse_tangents("gated_linear", x, w_gate, w_up, bias_gate, bias_up)
    if torch.is_grad_enabled() and (
            x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
            (bias_gate is not None and bias_gate.requires_grad) or
            (bias_up is not None and bias_up.requires_grad)):
        return _GatedLinear.apply(x, w_gate, w_up, bias_gate, bias_up, activation)
    return _gated_forward(x, w_gate, w_up, bias_gate, bias_up, activation, False)[0]


class Mxfp4Matrix:
    """A (rows, cols) matrix in microscaled 4-bit floating point, stored as
    include/xvram_b200.h lays it out: `codes` rows x ceil(cols / 32) x 16 bytes, `scales`
    ceil(rows / 128) x ceil(cols / 128) tiles of 512 bytes, both contiguous uint8 CUDA tensors of
    any shape.  Codes past the last column must be 0 and scales past the end not 255."""
    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int]):
        rows, cols = shape
        if rows < 0 or cols < 0:
            raise ValueError("negative size")
        need = rows * ((cols + 31) // 32) * 16
        if codes.dtype is not torch.uint8 or codes.numel() != need or \
                not codes.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError(f"codes of a ({rows}, {cols}) MXFP4 matrix must be {need} "
                             "contiguous bytes (uint8), 16-byte aligned")
        need = ((rows + 127) // 128) * ((cols + 127) // 128) * 512
        if scales.dtype is not torch.uint8 or scales.numel() != need or \
                not scales.is_contiguous() or scales.data_ptr() % 16:
            raise ValueError(f"scales of a ({rows}, {cols}) MXFP4 matrix must be {need} "
                             "contiguous bytes (uint8), 16-byte aligned")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        self.codes, self.scales, self.shape = codes, scales, (rows, cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device


def _rows(x: torch.Tensor):
    """(x with contiguous rows, its leading dimension)"""
    cols = x.shape[1]
    if cols == 1:
        x = x.resolve_neg()
    s0, s1 = x.stride()
    if s1 != 1 or s0 < cols:
        x = x.contiguous()
        s0 = cols
    return x, s0


def quantize_mxfp4(x: torch.Tensor) -> Mxfp4Matrix:
    """x (rows, cols; float16, bfloat16 or float32, CUDA) in MXFP4: blocks of 32 along each row
    share the scale 2^(floor(log2 max|v|) - 2); elements are rounded to the nearest E2M1 value,
    ties to even, saturating at 6 scales.  A block with a NaN or an infinity reads back as NaN."""
    if x.dtype not in _FEED_TYPES:
        raise TypeError(f"quantize_mxfp4 takes float16, bfloat16 or float32 (got {x.dtype})")
    if x.dim() != 2:
        raise ValueError("expected a 2-D tensor")
    if _dual_level():
        _refuse_tangents("quantize_mxfp4", x)
    if x.device.type != "cuda":
        raise RuntimeError("quantize_mxfp4 needs a CUDA tensor (there is no CPU path)")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("quantize_mxfp4 has no gradient: detach its input")
    rows, cols = x.shape
    with _on_device(x.device.index):
        x, ldx = _rows(x)
        codes = x.new_empty((rows, (cols + 31) // 32 * 16), dtype=torch.uint8)
        scales = x.new_empty(((rows + 127) // 128, (cols + 127) // 128, 512), dtype=torch.uint8)
        _check(lib.xvram_b200_mxfp4_quantize(_FEED_TYPES[x.dtype], rows, cols, x.data_ptr(), ldx,
                                             codes.data_ptr(), scales.data_ptr(),
                                             _stream(x.device.index)),
               "xvram_b200_mxfp4_quantize")
    q = Mxfp4Matrix.__new__(Mxfp4Matrix)  # its invariants hold: no checks
    q.codes, q.scales, q.shape = codes, scales, (rows, cols)
    return q


def dequantize_mxfp4(q: Mxfp4Matrix, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of q as a (rows, cols) tensor (exact in float32, rounded once in float16 and
    bfloat16)."""
    if dtype not in _FEED_TYPES:
        raise TypeError(f"dequantize_mxfp4 gives float16, bfloat16 or float32 (got {dtype})")
    if q.device.type != "cuda":
        raise RuntimeError("dequantize_mxfp4 needs a CUDA matrix (there is no CPU path)")
    rows, cols = q.shape
    with _on_device(q.device.index):
        out = q.codes.new_empty((rows, cols), dtype=dtype)
        _check(lib.xvram_b200_mxfp4_dequantize(_FEED_TYPES[dtype], rows, cols, q.codes.data_ptr(),
                                               q.scales.data_ptr(), out.data_ptr(), cols,
                                               _stream(q.device.index)),
               "xvram_b200_mxfp4_dequantize")
    return out


def _mxfp4_product(x, first, last, bias0, bias1, activation: int, dtype, what: str,
                   call) -> torch.Tensor:
    """The product `call` of x and one (first is last) or two MXFP4 weights, its arguments
    checked."""
    quantised = isinstance(x, Mxfp4Matrix)
    given = torch.float32 if quantised else x.dtype
    dtype = given if dtype is None else dtype
    if dtype not in _FEED_TYPES or given not in _FEED_TYPES:
        raise TypeError(f"{what} supports float16, bfloat16 and float32 (got {given} to {dtype})")
    shape, device = x.shape, x.device
    if not isinstance(first, Mxfp4Matrix) or not isinstance(last, Mxfp4Matrix) or \
            len(shape) != 2 or first.shape[1] != shape[1] or last.shape != first.shape:
        raise ValueError(f"{what} takes x (batch, in) and MXFP4 weights (out, in)")
    m, k = shape
    n = first.shape[0]
    if k == 0:
        raise ValueError(f"{what} needs at least one input feature")
    if _dual_level():
        _refuse_tangents(what, x, bias0, bias1)
    if device.type != "cuda" or first.codes.device != device or last.codes.device != device:
        raise RuntimeError(f"{what} needs its operands on one CUDA device (there is no CPU path)")
    if torch.is_grad_enabled() and (
            (not quantised and x.requires_grad) or
            (bias0 is not None and bias0.requires_grad) or
            (bias1 is not None and bias1.requires_grad)):
        raise RuntimeError(f"{what} has no gradient: detach its input and biases")
    index = device.index
    with _on_device(index):
        if quantised:
            src, ldx, codes, scales, like = 0, 0, x.codes.data_ptr(), x.scales.data_ptr(), x.codes
        else:
            like, ldx = _rows(x)
            src, codes, scales = like.data_ptr(), 0, 0
        if not quantised and (m > _DIRECT_ROWS or m * k > _DIRECT_VALUES):
            size = m * ((k + 31) // 32) * 16
            buffer = like.new_empty((size + (m + 127) // 128 * ((k + 127) // 128) * 512,),
                                    dtype=torch.uint8)
            codes = buffer.data_ptr()
            scales = codes + size
        out = like.new_empty((m, n), dtype=dtype)
        b0 = b1 = 0
        if bias0 is not None:
            bias0 = _check_bias(bias0, n, dtype, device, "bias")
            b0 = bias0.data_ptr()
        if bias1 is not None:
            bias1 = _check_bias(bias1, n, dtype, device, "bias")
            b1 = bias1.data_ptr()
        d = Mxfp4Product(_PRODUCT_SIZE, _FEED_TYPES[given], _FEED_TYPES[dtype], activation, m, n, k,
                         src, ldx, codes, scales, first.codes.data_ptr(), last.codes.data_ptr(),
                         first.scales.data_ptr(), last.scales.data_ptr(), b0, b1,
                         out.data_ptr(), n, _stream(index))
        st = call(ctypes.byref(d))
        if st:
            _check(st, what)
    return out


def linear_mxfp4(x, weight: Mxfp4Matrix, bias: torch.Tensor | None = None, relu: bool = False,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
    """Q(x) @ weight^T (+ bias) (then ReLU) on the block-scaled tensor-core product of two MXFP4
    operands, FP32 accumulation, rounded once.  x: (batch, in), a float tensor that is quantised
    here or an Mxfp4Matrix; weight: (out, in).  The result (and the bias) has `dtype`: x's type by
    default, float32 for an Mxfp4Matrix.  Inference only: no gradient."""
    return _mxfp4_product(x, weight, weight, bias, None, 1 if relu else 0, dtype, "linear_mxfp4",
                          lib.xvram_b200_mxfp4_linear)


def gated_linear_mxfp4(x, w_gate: Mxfp4Matrix, w_up: Mxfp4Matrix,
                       bias_gate: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
                       activation: str = "silu", dtype: torch.dtype | None = None) -> torch.Tensor:
    """`gated_linear` over MXFP4 operands, with `linear_mxfp4`'s input and types: both products,
    the biases, the activation and the product of the two in one kernel.  No gradient."""
    return _mxfp4_product(x, w_gate, w_up, bias_gate, bias_up, _activation(activation), dtype,
                          "gated_linear_mxfp4", lib.xvram_b200_mxfp4_gated)


class HostGemm:
    """Out-of-core mm / linear for host tensors through one SDK session.

    Every call uploads its operands into session allocations (page-locked host backing
    when they do not fit the budget), runs one GEMM plan (and, for linear, one bias/ReLU
    transaction) and reads the result back.  `budget_bytes` caps the session's device
    memory (0 = free memory minus headroom)."""

    def __init__(self, budget_bytes: int = 0, device_ordinal: int | None = None):
        ordinal = torch.cuda.current_device() if device_ordinal is None else device_ordinal
        # Budgets below a few GiB get 2 MiB frames (the VMM granularity) so they still
        # hold enough frames for a panel schedule; larger ones keep 64 MiB frames.
        chunk = (2 << 20) if 0 < budget_bytes < (4 << 30) else (64 << 20)
        self.s = sdk.Sdk(sdk.session_config(cache_target_bytes=budget_bytes,
                                            device_ordinal=ordinal, chunk_size_bytes=chunk))
        self.lock = threading.Lock()

    def close(self) -> None:
        self.s.close()

    def _upload(self, t: torch.Tensor):
        t = t.contiguous()
        alloc = self.s.alloc(max(t.numel() * t.element_size(), 4))
        if t.numel():
            alloc.write(t)
        return alloc

    def mm(self, a, b, out=None, tensor_cores=False, b_transposed=False, bias=None,
           relu=False):
        """Row-major a (m x k) @ b (k x n), or a @ b^T for b (n x k) when b_transposed."""
        dtype = _dtype_of(a, b)
        if (tensor_cores or bias is not None or relu) and dtype != torch.float32:
            raise TypeError("tensor_cores, bias and ReLU apply to float32 matrices")
        dt = _TYPES[dtype]
        m, k = a.shape
        n = b.shape[0] if b_transposed else b.shape[1]
        if (b.shape[1] if b_transposed else b.shape[0]) != k:
            raise ValueError(f"shapes {tuple(a.shape)} and {tuple(b.shape)} do not multiply")
        if out is None:
            out = torch.empty((m, n), dtype=dtype)
        if m == 0 or n == 0:
            return out
        if k == 0:
            raise ValueError("the out-of-core path needs k > 0 (no host-side arithmetic)")
        with self.lock:
            A, B = self._upload(a), self._upload(b)
            C = self.s.alloc(max(m * n * a.element_size(), 4))
            allocs = [A, B, C]
            try:
                mode = (sdk.COMPUTE_FP64 if dt == sdk.FP64 else
                        sdk.COMPUTE_FP32_TF32 if tensor_cores else sdk.COMPUTE_FP32_STRICT)
                if b_transposed:  # b is (n x k) row-major; op(B) = T
                    bdesc = sdk.matrix(B, n, k, k, sdk.ROW_MAJOR, data_type=dt)
                else:
                    bdesc = sdk.matrix(B, k, n, n, sdk.ROW_MAJOR, data_type=dt)
                desc = self.s.gemm_desc(sdk.matrix(A, m, k, k, sdk.ROW_MAJOR, data_type=dt),
                                        bdesc, sdk.matrix(C, m, n, n, sdk.ROW_MAJOR, data_type=dt),
                                        sdk.OP_N, sdk.OP_T if b_transposed else sdk.OP_N,
                                        mode=mode)
                plan = self.s.plan(desc)
                try:
                    self.s.check("gemm_execute", self.s.t.gemm_execute(plan, sdk.TIMEOUT_INFINITE))
                finally:
                    self.s.t.gemm_plan_release(plan)
                if bias is not None or relu:
                    Bias = self._upload(bias.to(torch.float32)) if bias is not None else None
                    if Bias is not None:
                        allocs.append(Bias)
                    spec = [(C, 0, m * n * 4, sdk.READ_WRITE)]
                    if Bias is not None:
                        spec.append((Bias, 0, n * 4, sdk.READ))

                    def body(ctx):
                        y = ctx.ranges[0].device_address
                        bptr = ctx.ranges[1].device_address if Bias is not None else 0
                        # row-major (m, n) = column-major (n, m): n features x m rows
                        return sdk.bias_activation(y, n, n, m, bptr, relu, ctx.native_stream)
                    d = self.s.transaction_desc(spec, body)
                    self.s.check("transaction_execute",
                                 self.s.t.transaction_execute(self.s.session, ctypes.byref(d),
                                                              sdk.TIMEOUT_INFINITE))
                C.read(out)
                return out
            finally:
                for x in allocs:
                    x.release()

    def linear(self, x, weight, bias=None, relu=False, tensor_cores=False):
        return self.mm(x, weight, tensor_cores=tensor_cores, b_transposed=True, bias=bias,
                       relu=relu)


_host = None
_host_lock = threading.Lock()


def _close_host_session() -> None:
    """Closes the host-tensor session at interpreter exit, before the CUDA runtime's own
    teardown (its worker and budget sampler must not outlive the device)."""
    global _host
    with _host_lock:
        if _host is not None:
            _host.close()
            _host = None


atexit.register(_close_host_session)


def _host_session() -> HostGemm:
    global _host
    if not torch.cuda.is_available():
        raise RuntimeError("xvram_b200.torch_bridge needs a CUDA device (there is no CPU path)")
    with _host_lock:
        if _host is None:
            _host = HostGemm()
        return _host


def set_host_budget(budget_bytes: int) -> None:
    """Re-open the host-tensor session with a device budget (bytes; 0 = automatic)."""
    global _host
    with _host_lock:
        if _host is not None:
            _host.close()
        _host = HostGemm(budget_bytes)
