"""The 4-bit Linear layers and the gated block norm on the CPU: sizes, and every refusal (made on the host,
before anything is launched)."""
import numpy as np
import pytest

import mx4_reference as ref
import varda_b200 as vb

P = 1 << 20  # stands for a device address, 16-byte aligned; no refused call uses it


def refused(fn, code=1):
    with pytest.raises(vb.VardaError) as e:
        fn()
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (1, 33), (128, 128), (129, 129), (189809, 1024), (5, 4096)])
def test_sizes(rows, K):
    nb = (K + 31) // 32
    assert vb.mx4_row_bytes(K) == 16 * nb
    assert vb.mx4_scale_bytes(rows, K) == len(ref.tile_scales(np.zeros((rows, nb), np.uint8)))


def test_sizes_of_nothing():
    assert vb.mx4_row_bytes(0) == 0 and vb.mx4_scale_bytes(0, 64) == 0 and vb.mx4_scale_bytes(4, -1) == 0


def test_reference_round_trip():
    """Values of the format come back as they are; the tiling is a permutation."""
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 256, (5, 48), dtype=np.uint8)
    codes[:, ::16] |= 7  # a 6 in each block, so that its scale is the one its values give
    sb = rng.integers(1, 250, (5, 3), dtype=np.uint8)
    v = ref.values(codes, sb, 96)
    c2, s2 = ref.quantize(v)
    assert np.array_equal(s2, sb) and np.array_equal(ref.values(c2, s2, 96), v)
    assert np.array_equal(ref.untile_scales(ref.tile_scales(sb), 5, 3), sb)


QUANT = dict(dtype=vb.FP16, x=P, ldx=64, rows=4, K=64, codes=P, ldc=32, scales=P)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(x=None), dict(ldx=63), dict(rows=-1), dict(K=0), dict(K=1 << 31),
                                 dict(codes=None), dict(codes=P + 8), dict(ldc=16), dict(ldc=40), dict(scales=None),
                                 dict(scales=P + 4)])
def test_quantize_refuses(bad):
    refused(lambda: vb.mx4_quantize(**{**QUANT, **bad}))
    d = {**QUANT, **bad}
    refused(lambda: vb.mx4_dequantize(d["dtype"], d["codes"], d["ldc"], d["scales"], d["rows"], d["K"], d["x"], d["ldx"]))


GEMM = dict(dtype=vb.FP16, A=P, lda=32, sA=P, W=P, ldw=32, sW=P, bias=P, Y=P, ldy=72, R=P, ldr=72, M=5, N=70, K=64, epilogue=2)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(A=None), dict(A=P + 1), dict(lda=16), dict(lda=36), dict(sA=None),
                                 dict(W=None), dict(ldw=16), dict(sW=P + 8), dict(Y=None), dict(Y=P + 8), dict(ldy=64),
                                 dict(ldy=74), dict(R=None), dict(R=P + 2), dict(ldr=64), dict(ldr=77), dict(M=-1),
                                 dict(N=-1), dict(K=0), dict(M=1 << 31), dict(epilogue=3), dict(epilogue=-1)])
def test_gemm_refuses(bad):
    refused(lambda: vb.gemm_mx4(**{**GEMM, **bad}))


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(A=None), dict(lda=16), dict(sA=P + 2), dict(W=P + 4), dict(ldw=0),
                                 dict(sW=None), dict(codes=None), dict(codes=P + 8), dict(ldc=32), dict(ldc=56),
                                 dict(scales=None), dict(scales=P + 8), dict(M=-1), dict(N=-1), dict(K=0), dict(epilogue=2)])
def test_gemm_quant_refuses(bad):
    good = dict(dtype=vb.FP16, A=P, lda=32, sA=P, W=P, ldw=32, sW=P, bias=P, codes=P, ldc=48, scales=P, M=5, N=70, K=64, epilogue=1)
    refused(lambda: vb.gemm_mx4_quant(**{**good, **bad}))


NORM = dict(dtype=vb.FP16, rows=4, C=64, x=P, ldx=64, h=P, ldh=64, post=1, gate=P, ldgate=64, out=P, ldo=64, pre=2,
            scale=P, shift=P, ldmod=64, rows_per_group=2, y=P, ldy=64)


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(rows=-1), dict(C=0), dict(x=None), dict(ldx=63), dict(ldh=60),
                                 dict(ldo=1), dict(ldy=0), dict(post=3), dict(pre=-1), dict(ldgate=0), dict(ldmod=63),
                                 dict(rows_per_group=-2), dict(out=None, y=None), dict(y_codes=P, ldc=32, y_scales=P),
                                 dict(y=None, y_codes=P, ldc=16, y_scales=P), dict(y=None, y_codes=P, ldc=32),
                                 dict(y=None, y_codes=P + 4, ldc=32, y_scales=P)])
def test_block_norm_refuses(bad):
    refused(lambda: vb.block_norm(**{**NORM, **bad}))


def test_block_norm_refuses_wide_rows_and_no_arguments():
    wide = dict(C=16385, ldx=16385, ldh=16385, ldgate=16385, ldo=16385, ldmod=16385, ldy=16385)
    refused(lambda: vb.block_norm(**{**NORM, **wide}), code=4)
    assert vb.lib.vb_block_norm(vb.FP16, None, None) == 1
    assert vb.BLOCK_NORM_ARGS.size == 23 * 8 + 16  # which the library checks of its struct


def test_nothing_to_do_is_no_error():
    vb.mx4_quantize(**{**QUANT, "rows": 0, "x": None})
    vb.gemm_mx4(**{**GEMM, "M": 0, "Y": None})
    vb.gemm_mx4(**{**GEMM, "N": 0, "W": None})
    vb.block_norm(**{**NORM, "rows": 0, "x": None})
