"""The 4-bit product's bounded waits, made to run out from the host without a GPU fault: VB_DEBUG_MX4_WITHHOLD=1 makes block 0
skip its first stage's codes, VB_DEBUG_WAIT_NS shortens the waits' limit. The kernel gives up and returns, vb_check_device
reports VB_ERR_TIMEOUT (code 6), and the same call without the hooks is right."""
import pytest

import test_mx4_gpu as t
import varda_b200 as vb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# (M, N, K) whose product takes tiles of 64 and 128 columns and the pairs' 256
TILES = [(130, 640, 600), (2000, 1024, 96), (9500, 4080, 544)]


def withhold(monkeypatch, on=True):
    for k, v in (("VB_DEBUG_WAIT_NS", "20000000"), ("VB_DEBUG_MX4_WITHHOLD", "1")):
        if on:
            monkeypatch.setenv(k, v)
        else:
            monkeypatch.delenv(k)


def timed_out(what):
    with pytest.raises(vb.VardaError, match=what) as e:
        vb.check_device()
    assert e.value.code == 6


@pytest.mark.parametrize("M,N,K", TILES)
@pytest.mark.parametrize("dt,epi,quant", [(vb.FP16, 0, False), (vb.FP16, 2, False), (vb.FP32, 2, False), (vb.FP16, 1, True)])
def test_waits_run_out_and_the_device_stays_usable(M, N, K, dt, epi, quant, monkeypatch):
    A, W, bias, R = t.product_case(M, N, K, dt, 2)
    b, r = torch.from_numpy(bias).to("cuda", t.tdt(dt)), t.put(R, dt)
    y, (codes, tiles) = torch.zeros(M, N, device="cuda", dtype=t.tdt(dt)), t.mx4_space(M, N)

    def run():
        a = (dt, A[0], A[0].stride(0), A[1], W[0], W[0].stride(0), W[1], b)
        if quant:
            vb.gemm_mx4_quant(*a, codes, codes.stride(0), tiles, M, N, K, epi)
        else:
            vb.gemm_mx4(*a, y, N, r, N, M, N, K, epi)

    withhold(monkeypatch)
    run()
    timed_out("4-bit GEMM")
    vb.check_device()  # reading the flag clears it
    withhold(monkeypatch, False)
    run()
    vb.check_device()
    if quant:
        want, err = t.product_exact(A[2], W[2], bias, None, epi, False)
        t.blocks_check((codes, tiles), M, N, want, err)
    else:
        t.product_check(t.get(y).astype(float), A[2], W[2], bias, R, dt, epi)


def test_a_timeout_beside_the_attention_s_is_not_lost(monkeypatch):
    """Both kernels' waits run out before anyone asks: vb_check_device reports one, then the other, then none."""
    import numpy as np
    rng = np.random.default_rng(1)
    n, C, heads = 300, 256, 4
    src, dst = [], []
    for i in range(n):
        s = np.unique(np.clip(i + rng.integers(-20, 20, 6), 0, n - 1))
        src += list(s)
        dst += [i] * len(s)
    rp, src, _, attr = vb.build_csr(np.array([src, dst], np.int64), rng.normal(size=(len(src), 3)).astype(np.float16).astype(np.float32), n, n)
    tiles = vb.Tiles(rp, src, attr, n, C // heads, kind=vb.Tiles.TC)
    q, k, v, xr, out = (torch.zeros(n, C, device="cuda", dtype=torch.float16) for _ in range(5))
    M, N, K = TILES[0]
    A, W, _, _ = t.product_case(M, N, K, vb.FP16, 2)
    y = torch.zeros(M, N, device="cuda", dtype=torch.float16)
    withhold(monkeypatch)
    monkeypatch.setenv("VB_DEBUG_TC_WITHHOLD", "1")
    tiles.attention(0, n, q, C, k, v, C, xr, C, out, C, torch.zeros(4, C, device="cuda"), C, heads, C // heads)
    vb.gemm_mx4(vb.FP16, A[0], A[0].stride(0), A[1], W[0], W[0].stride(0), W[1], None, y, N, None, 0, M, N, K)
    torch.cuda.synchronize()
    timed_out("4-bit GEMM")
    timed_out("attention")
    vb.check_device()
