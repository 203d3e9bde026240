"""Addresses and sizes as the Python binding takes them (nothing is launched)."""
import ctypes
import enum

import numpy as np
import pytest

import varda_b200 as vb


class Address(enum.IntEnum):
    X = 1 << 20


class Tensor:
    def data_ptr(self):
        return 1 << 21


HOST = np.zeros(8, np.float32)


@pytest.mark.parametrize("a,want", [(None, None), (1 << 40, 1 << 40), (0, None), (Address.X, 1 << 20), (True, 1), (Tensor(), 1 << 21),
                                    (HOST, HOST.ctypes.data)])
def test_addresses(a, want):
    """None, integers and their subclasses, tensors, host arrays: as one argument, and packed into the norm's struct."""
    assert ctypes.c_void_p.from_param(vb._ptr(a)) is None or ctypes.cast(vb._ptr(a), ctypes.c_void_p).value == want
    assert vb._addr(a) == (want or 0)


@pytest.mark.parametrize("x", [Address.X, Tensor(), HOST])
def test_block_norm_takes_what_the_others_take(x, monkeypatch):
    """Every address in its place of the struct; a refusal is the library's, whatever holds the address."""
    seen = []
    monkeypatch.setitem(vb.lib.__dict__, "vb_block_norm", lambda dtype, a, stream: seen.append(vb.BLOCK_NORM_ARGS.unpack(a)) or 0)
    vb.block_norm(vb.FP16, 4, 64, x, 64, h=x, ldh=65, gate=x, ldgate=66, out=x, ldo=67, y=x, ldy=68, post_w=x, post_b=x, pre_w=x,
                  pre_b=x, scale=x, shift=x, ldmod=69, y_codes=x, ldc=32, y_scales=x)
    p = vb._addr(x)
    assert p and seen[0][:23] == (4, 64, p, 64, p, 65, p, p, p, 66, p, 67, p, p, p, p, 69, 0, p, 68, p, 32, p)
    monkeypatch.undo()
    with pytest.raises(vb.VardaError) as e:
        vb.block_norm(vb.FP16, 4, 64, x, 63, y=x, ldy=64)
    assert e.value.code == 1


@pytest.mark.parametrize("n", [1 << 30, (1 << 31) + 1, (1 << 63) - 1])
def test_sizes_that_no_function_takes(n):
    """No size for what quantise and product refuse, and no overflow on the way to it."""
    assert vb.mx4_row_bytes(n) == 0 and vb.mx4_scale_bytes(n, 64) == 0 and vb.mx4_scale_bytes(64, n) == 0
    assert vb.mx4_row_bytes((1 << 30) - 1) == 1 << 29
    with pytest.raises(vb.VardaError) as e:
        vb.mx4_quantize(vb.FP16, 1 << 20, n, 4, n, 1 << 20, 1 << 40, 1 << 20)
    assert e.value.code == 1
