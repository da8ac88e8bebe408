"""A stand-in for the library's gated entries on host memory, in 64 bits, so that what the bridge
hands over (pointers, leading dimensions, transpositions) is checked without a GPU: every matrix
has to lie inside the storage of a live tensor, and 16-bit operands have to be aligned as the
tensor-core kernels want them."""
from __future__ import annotations

import contextlib
import ctypes as C
import gc

import numpy as np
import torch

from feed_util import ACTS, act_and_slope

TYPES = {0: np.float16, 2: np.float32}  # XVRAM_DATA_*


def room(ptr: int) -> int:
    """Bytes from ptr to the end of the live tensor storage that holds it."""
    for t in gc.get_objects():
        if issubclass(type(t), torch.Tensor) and t.device.type == "cpu":
            s = t.untyped_storage()
            if s.data_ptr() <= ptr < s.data_ptr() + s.nbytes():
                return s.data_ptr() + s.nbytes() - ptr
    raise AssertionError(f"{ptr:#x} is in no tensor")


def matrix(ptr: int, rows: int, cols: int, ld: int, kind: int, transposed=0) -> np.ndarray:
    """The rows x cols matrix at ptr as a writable view of its memory."""
    dtype = np.dtype(TYPES[kind])
    outer, inner = (cols, rows) if transposed else (rows, cols)
    assert ld >= inner, "leading dimension below the rows' length"
    count = (outer - 1) * ld + inner
    assert count * dtype.itemsize <= room(ptr), "the matrix ends outside its storage"
    flat = np.frombuffer((C.c_char * (count * dtype.itemsize)).from_address(ptr), dtype)
    item = dtype.itemsize
    view = np.lib.stride_tricks.as_strided(flat, (outer, inner), (ld * item, item))
    return view.T if transposed else view


class HostLibrary:
    def __init__(self):
        self.calls = []

    def _operands(self, d, backward):
        per = 16 // TYPES[d.data_type]().itemsize
        # The kernel for few rows reads any element-aligned row.
        few = not d.x_transposed and not d.w_transposed and (
            d.m == 1 or (d.m <= 4 and d.h * d.k <= 1 << 23))
        for p, ld in ((d.x, d.ldx), (d.w_gate, d.ld_gate), (d.w_up, d.ld_up)):
            if d.data_type != 2 and (backward or not few) and (p % 16 or ld % per):
                return None
        return (matrix(d.x, d.m, d.k, d.ldx, d.data_type, d.x_transposed).astype(np.float64),
                *(matrix(p, d.h, d.k, ld, d.data_type, d.w_transposed).astype(np.float64)
                  for p, ld in ((d.w_gate, d.ld_gate), (d.w_up, d.ld_up))))

    def xvram_b200_gated_workspace_bytes(self, problem, backward):
        return 0

    def xvram_b200_gated_forward(self, problem, out, ld_out):
        d = problem._obj
        self.calls.append("forward")
        if d.m == 0 or d.h == 0:
            return 0
        if (ops := self._operands(d, False)) is None:
            return 1
        x, wg, wu = ops
        g, u = x @ wg.T, x @ wu.T
        if d.bias_gate:
            g += matrix(d.bias_gate, 1, d.h, d.h, d.data_type)
        if d.bias_up:
            u += matrix(d.bias_up, 1, d.h, d.h, d.data_type)
        if d.pre_gate:
            matrix(d.pre_gate, d.m, d.h, d.ld_pre, 2)[:] = g
            matrix(d.pre_up, d.m, d.h, d.ld_pre, 2)[:] = u
        a, _ = act_and_slope(torch.from_numpy(g), ACTS[d.activation])
        matrix(out, d.m, d.h, ld_out, d.data_type)[:] = a.numpy() * u
        return 0

    def xvram_b200_gated_backward(self, problem, dout, ld_dout, dx, ld_dx, dw_gate, dw_up, ld_dw,
                                  db_gate, db_up):
        d = problem._obj
        self.calls.append("backward")
        if d.m == 0 or d.h == 0:
            return 0
        if (ops := self._operands(d, True)) is None:
            return 1
        x, wg, wu = ops
        g, u = (matrix(p, d.m, d.h, d.ld_pre, 2).astype(np.float64) for p in (d.pre_gate, d.pre_up))
        a, s = (t.numpy() for t in act_and_slope(torch.from_numpy(g), ACTS[d.activation]))
        dh = matrix(dout, d.m, d.h, ld_dout, d.data_type).astype(np.float64)
        dg, du = dh * u * s, dh * a
        kind = d.data_type
        for p, rows, cols, ld, v in ((dx, d.m, d.k, ld_dx, dg @ wg + du @ wu),
                                     (dw_gate, d.h, d.k, ld_dw, dg.T @ x),
                                     (dw_up, d.h, d.k, ld_dw, du.T @ x),
                                     (db_gate, 1, d.h, d.h, dg.sum(0)[None]),
                                     (db_up, 1, d.h, d.h, du.sum(0)[None])):
            if p:
                matrix(p, rows, cols, ld, kind)[:] = v
        return 0

    def xvram_b200_pack_rows(self, kind, items, count, stream):
        self.calls.append("pack")
        for t in items[:count]:
            if t.rows and t.cols:
                dst = matrix(t.dst, t.rows, t.ld_dst, t.ld_dst, kind)
                dst[:] = 0
                dst[:, :t.cols] = matrix(t.src, t.rows, t.cols, t.ld_src, kind)
        return 0


@contextlib.contextmanager
def installed(monkeypatch, tb):
    """Lets the bridge's gated calls take CPU tensors and hand them to a HostLibrary."""
    host = HostLibrary()
    monkeypatch.setattr(tb, "lib", host)
    monkeypatch.setattr(tb, "_stream", lambda index: 0)
    monkeypatch.setattr(tb, "_on_device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(tb, "_check_gated", lambda *a: None)
    gc.freeze()  # `room` looks through the objects made from here on
    yield host
    gc.unfreeze()


def layouts(t: torch.Tensor) -> list:
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
