"""Refusals of the feed-forward operators that need no GPU: the bridge's argument checks and
the C entries' INVALID_ARGUMENT, all before any device work."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from xvram_b200 import torch_bridge as tb  # noqa: E402
from xvram_b200._native import Gated, Mxfp4Product, Pack, lib  # noqa: E402

OK, INVALID = 0, 1


def ones(*shape, dtype=torch.float16):
    return torch.ones(shape, dtype=dtype)


def test_gated_linear_arguments():
    x, w = ones(2, 8), ones(4, 8)
    with pytest.raises(ValueError, match="activation"):
        tb.gated_linear(x, w, w, activation="tanh")
    with pytest.raises(TypeError):
        tb.gated_linear(x, w, w.float())
    with pytest.raises(TypeError):
        tb.gated_linear(*(t.double() for t in (x, w, w)))
    for bad in (ones(4, 7), ones(8), ones(4, 8, 1)):
        with pytest.raises(ValueError):
            tb.gated_linear(x, bad, bad)
    with pytest.raises(ValueError):
        tb.gated_linear(x, w, ones(5, 8))
    with pytest.raises(ValueError, match="input feature"):
        tb.gated_linear(ones(2, 0), ones(4, 0), ones(4, 0))
    with pytest.raises(RuntimeError, match="no CPU path"):
        tb.gated_linear(x, w, w)


def test_mxfp4_arguments():
    with pytest.raises(TypeError):
        tb.quantize_mxfp4(ones(2, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        tb.quantize_mxfp4(ones(8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        tb.quantize_mxfp4(ones(2, 8))
    codes, scales = torch.zeros(5 * 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    q = tb.Mxfp4Matrix(codes, scales, (5, 40))
    for args in ((codes[:-1], scales, (5, 40)), (codes, scales[:-16], (5, 40)),
                 (codes.char(), scales, (5, 40)), (codes, scales, (-1, 40)),
                 (codes.view(80, 2)[:, 0], scales, (5, 20))):
        with pytest.raises(ValueError):
            tb.Mxfp4Matrix(*args)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tb.dequantize_mxfp4(q)
    with pytest.raises(TypeError):
        tb.dequantize_mxfp4(q, torch.float64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tb.linear_mxfp4(ones(2, 40), q)
    with pytest.raises(ValueError):
        tb.linear_mxfp4(ones(2, 41), q)
    with pytest.raises(ValueError):
        tb.linear_mxfp4(ones(2, 40), ones(5, 40))
    with pytest.raises(TypeError):
        tb.linear_mxfp4(ones(2, 40, dtype=torch.float64), q)
    with pytest.raises(ValueError, match="activation"):
        tb.gated_linear_mxfp4(ones(2, 40), q, q, activation="none")


def gated(**changes):
    d = Gated(C.sizeof(Gated), 1, 0, 0, 0, 0, 4, 8, 16, 4096, 8192, 12288, 16, 16, 16)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("changes", [
    {"struct_size": 8}, {"data_type": 3}, {"activation": 5}, {"x_transposed": 2},
    {"w_transposed": 7}, {"m": -1}, {"h": -1}, {"k": 0}, {"m": 1 << 31}, {"h": (1 << 31) - 511},
    {"x": 0}, {"w_gate": 0},
    {"w_up": 0}, {"ldx": 15}, {"ld_gate": 15}, {"ld_up": 3}, {"x": 4097}, {"bias_gate": 3},
    {"pre_gate": 4096}, {"pre_gate": 4096, "pre_up": 4104, "ld_pre": 8},
    {"pre_gate": 4096, "pre_up": 8192, "ld_pre": 10},
    {"pre_gate": 4096, "pre_up": 8192, "ld_pre": 4}])
def test_gated_entry_refuses(changes):
    assert lib.xvram_b200_gated_forward(C.byref(gated(**changes)), 1 << 16, 8) == INVALID


def test_gated_entry_outputs():
    assert lib.xvram_b200_gated_forward(None, 1 << 16, 8) == INVALID
    assert lib.xvram_b200_gated_forward(C.byref(gated()), 0, 8) == INVALID
    assert lib.xvram_b200_gated_forward(C.byref(gated()), 1 << 16, 7) == INVALID
    assert lib.xvram_b200_gated_forward(C.byref(gated(m=0)), 0, 0) == OK
    back = lambda d, *a: lib.xvram_b200_gated_backward(C.byref(d), *a)
    kept = {"pre_gate": 4096, "pre_up": 8192, "ld_pre": 8}
    assert back(gated(), 65536, 8, 0, 0, 0, 0, 0, 0, 0) == INVALID  # nothing kept
    assert back(gated(**kept), 0, 8, 0, 0, 0, 0, 0, 0, 0) == INVALID
    assert back(gated(**kept), 65536, 7, 0, 0, 0, 0, 0, 0, 0) == INVALID
    assert back(gated(**kept), 65536, 8, 131072, 15, 0, 0, 0, 0, 0) == INVALID
    assert back(gated(**kept), 65536, 8, 0, 0, 131072, 0, 15, 0, 0) == INVALID
    assert lib.xvram_b200_gated_workspace_bytes(C.byref(gated(k=0)), 1) == 0
    assert lib.xvram_b200_gated_workspace_bytes(C.byref(gated()), 1) > 0


def product(**changes):
    d = Mxfp4Product(C.sizeof(Mxfp4Product), 1, 1, 0, 20, 8, 64, 4096, 64, 8192, 8192, 16384, 16384,
                     32768, 32768, 0, 0, 65536, 8, 0)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("changes", [
    {"struct_size": 4}, {"x_type": 3}, {"out_type": 3}, {"activation": 9}, {"m": -1}, {"k": 0},
    {"n": 1 << 31}, {"ldx": 63}, {"x": 4097}, {"x_codes": 8}, {"x_scales": 0}, {"w_codes0": 8200},
    {"w_scales0": 0}, {"out": 0}, {"ld_out": 7}, {"out": 65537}, {"bias0": 1}])
def test_product_entries_refuse(changes):
    for fn in (lib.xvram_b200_mxfp4_linear, lib.xvram_b200_mxfp4_gated):
        assert fn(C.byref(product(**changes))) == INVALID


def test_other_entries():
    assert lib.xvram_b200_mxfp4_linear(None) == INVALID
    assert lib.xvram_b200_mxfp4_linear(C.byref(product(activation=2))) == INVALID
    assert lib.xvram_b200_mxfp4_linear(C.byref(product(m=0))) == OK
    assert lib.xvram_b200_mxfp4_gated(C.byref(product(w_codes1=0))) == INVALID
    a, b = C.c_uint64(), C.c_uint64()
    assert lib.xvram_b200_mxfp4_bytes(129, 33, C.byref(a), C.byref(b)) == OK
    assert (a.value, b.value) == (129 * 32, 2 * 512)
    assert lib.xvram_b200_mxfp4_bytes(-1, 33, C.byref(a), C.byref(b)) == INVALID
    assert lib.xvram_b200_mxfp4_bytes(1, 33, None, C.byref(b)) == INVALID
    q = lib.xvram_b200_mxfp4_quantize
    assert q(1, 0, 8, 0, 0, 0, 0, 0) == OK
    for args in ((3, 2, 8, 4096, 8, 4096, 4096, 0), (1, 2, 8, 0, 8, 4096, 4096, 0),
                 (1, 2, 8, 4096, 7, 4096, 4096, 0), (1, 2, 8, 4096, 8, 4100, 4096, 0)):
        assert q(*args) == INVALID
        assert lib.xvram_b200_mxfp4_dequantize(args[0], args[1], args[2], args[5], args[6], args[3],
                                               args[4], 0) == INVALID
    pack = lib.xvram_b200_pack_rows
    good = (4096, 8192, 3, 8, 2, 3)
    assert pack(1, None, 1, 0) == INVALID
    assert pack(1, (Pack * 1)(good), 0, 0) == INVALID and pack(3, (Pack * 1)(good), 1, 0) == INVALID
    assert pack(1, (Pack * 5)(*[good] * 5), 5, 0) == INVALID
    for bad in ((0, 8192, 3, 8, 2, 3), (4097, 8192, 3, 8, 2, 3), (4096, 8200, 3, 8, 2, 3),
                (4096, 8192, 3, 7, 2, 3), (4096, 8192, -1, 8, 2, 3), (4096, 8192, 3, 2, 2, 3)):
        assert pack(1, (Pack * 1)(bad), 1, 0) == INVALID
