"""The 4-bit Linear layers and the gated block norm on the B200, against plain forms in 64 bits.

Tolerances. Quantising and reading back are exact. A product's sum: at most K additions and a few operations
of the epilogue, each off by at most one unit of the last place (2^-23) of the sum of magnitudes, then half a
step of the type. A norm: a sum of C values is formed over at most 64 values per thread and 8 levels, so mean
and variance are off by at most 80 2^-24 of the mean magnitude; with the few operations after it, 128 2^-24 =
2^-17 of (|normalised value| + mean magnitude / spread + 1), then half a step of the type.
"""
import math

import numpy as np
import pytest

import mx4_reference as ref
import varda_b200 as vb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF_STEP = {vb.FP16: 2.0 ** -11, vb.FP32: 2.0 ** -24}
TINY = {vb.FP16: 2.0 ** -25, vb.FP32: 2.0 ** -149}  # half a step below the normal numbers


def tdt(dt):
    return torch.float16 if dt == vb.FP16 else torch.float32


def put(a, dt, ld=None, pad=float("nan"), skew=0):
    """Rows on the device, ld elements apart (NaN between them), `skew` elements past an aligned address."""
    a = np.asarray(a)
    rows, k = a.shape
    ld = k if ld is None else ld
    buf = torch.full((skew + rows * ld,), pad, device="cuda", dtype=tdt(dt))
    v = buf[skew:].view(rows, ld)
    v[:, :k] = torch.from_numpy(np.ascontiguousarray(a)).to("cuda", tdt(dt))
    return v[:, :k]


def get(t):
    return t.detach().cpu().numpy()


def rounded(a, dt):
    return a.astype(np.float16 if dt == vb.FP16 else np.float32).astype(np.float64)


def blocks(x):
    """x in 64 bits -> (codes, tiles on the device, the values that they stand for)."""
    c, s = ref.quantize(x)
    return torch.from_numpy(c).cuda(), torch.from_numpy(ref.tile_scales(s)).cuda(), ref.values(c, s, x.shape[1])


# ------------------------------------------------------------------ quantising

@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 1024), (3, 31), (5, 32), (128, 33), (129, 127), (300, 129), (257, 1000),
                                    (40, 4096)])
def test_quantize_bits(rows, K, dt):
    rng = np.random.default_rng(rows * 7 + K)
    x = rounded(rng.normal(size=(rows, K)) * np.exp2(rng.integers(-20, 12, (rows, 1))), dt)
    x[rng.random(x.shape) < 0.1] *= 0
    x[0, 0] = -0.0
    for ld, skew in ((K, 0), (K + 8 + (-K) % 8, 0), (K + 3, 1)):
        d = put(x, dt, ld, skew=skew)
        ldc = vb.mx4_row_bytes(K) + 16
        codes = torch.full((rows + 1, ldc), 0xEE, device="cuda", dtype=torch.uint8)
        tiles = torch.full((vb.mx4_scale_bytes(rows, K) + 16,), 0xEE, device="cuda", dtype=torch.uint8)
        vb.mx4_quantize(dt, d, ld, rows, K, codes, ldc, tiles)
        rc, rs = ref.quantize(x)
        assert np.array_equal(get(codes)[:rows, :ldc - 16], rc)
        assert (get(codes)[:, ldc - 16:] == 0xEE).all() and (get(codes)[rows] == 0xEE).all()
        assert np.array_equal(get(tiles)[:-16], ref.tile_scales(rs)) and (get(tiles)[-16:] == 0xEE).all()
        y = torch.full((rows + 1, ld), 7.0, device="cuda", dtype=tdt(dt))
        vb.mx4_dequantize(dt, codes, ldc, tiles, rows, K, y, ld)
        assert np.array_equal(get(y)[:rows, :K].astype(np.float64), rounded(ref.values(rc, rs, K), dt))
        assert (get(y)[:, K:] == 7).all() and (get(y)[rows] == 7).all()


def test_quantize_ties_ends_and_not_finite():
    """Every tie and its neighbours, saturation, the ends of fp32, and blocks with Inf or NaN."""
    grid = np.concatenate([ref.E2M1, (ref.E2M1[1:] + ref.E2M1[:-1]) / 2, [6.5, 7, 7.99]])
    near = np.concatenate([grid, np.nextafter(grid.astype(np.float32), np.float32(9)), np.nextafter(grid.astype(np.float32), np.float32(0))])
    rows = []
    for e in (-126, -100, -1, 0, 5, 120, 125):
        for part in np.array_split(near, 3):
            r = np.zeros(32)
            r[:len(part)] = part * (1 - 2 * (np.arange(len(part)) % 2))
            r[31] = 4.0
            rows.append(r * np.exp2(float(e)))
    for lone in (2.0 ** -149, 2.0 ** -126, 2.0 ** -127, 3.4028234663852886e38, np.inf, -np.inf, np.nan):
        r = np.linspace(-1, 1, 32) * 2.0 ** -130
        r[5] = lone
        rows.append(r)
    x = np.array(rows, np.float32).astype(np.float64)
    n = len(x)
    codes, tiles = torch.zeros(n, 16, device="cuda", dtype=torch.uint8), torch.zeros(512, device="cuda", dtype=torch.uint8)
    vb.mx4_quantize(vb.FP32, put(x, vb.FP32), 32, n, 32, codes, 16, tiles)
    rc, rs = ref.quantize(x)
    assert np.array_equal(ref.untile_scales(get(tiles), n, 1), rs) and (rs[-3:] == 255).all()
    assert np.array_equal(get(codes), rc)
    y = torch.zeros(n, 32, device="cuda")
    vb.mx4_dequantize(vb.FP32, codes, 16, tiles, n, 32, y, 32)
    np.testing.assert_array_equal(get(y), ref.values(rc, rs, 32).astype(np.float32))


# ------------------------------------------------------------------ products

def gelu(v, tanh=False):
    if tanh:
        return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return 0.5 * v * torch.special.erfc(torch.from_numpy(-v * math.sqrt(0.5)).cuda()).cpu().numpy()


def product_case(M, N, K, dt, seed=0):
    rng = np.random.default_rng(seed + M * 31 + N * 7 + K)
    A = rng.normal(size=(M, K)) * np.exp(rng.normal(size=(M, 1)) + 0.5 * rng.normal(size=(1, K)))
    W = rng.normal(size=(N, K)) / math.sqrt(K)
    return blocks(A), blocks(W), rounded(rng.normal(size=N), dt), rounded(rng.normal(size=(M, N)), dt)


def matmul(a, w):
    """a w^T in 64 bits, by the device's 64-bit matrix product (small ones here)."""
    if len(a) * len(w) * a.shape[1] < 10 ** 9:
        return a @ w.T
    return (torch.from_numpy(a).cuda() @ torch.from_numpy(w).cuda().t()).cpu().numpy()


def product_exact(a, w, bias, R, epi, tanh):
    """(the result in 64 bits, the bound of an fp32 evaluation's error)."""
    K = a.shape[1]
    y, mag = matmul(a, w), matmul(np.abs(a), np.abs(w))
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    err = (K + 8) * 2.0 ** -23 * mag
    if epi == 1:  # |gelu'| <= 1.13; its own operations (erf within 2^-22 of 1, a handful of roundings)
        err = 1.13 * err + 2.0 ** -20 * np.abs(y)
        y = gelu(y, tanh)
    if epi == 2:
        y, err = y + R, err + 2.0 ** -23 * (np.abs(y) + np.abs(R))
    return y, err


def product_check(got, a, w, bias, R, dt, epi, tanh=False):
    y, err = product_exact(a, w, bias, R, epi, tanh)
    tol = err + HALF_STEP[dt] * (np.abs(y) + err) + TINY[dt]
    bad = np.abs(got - y) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - y) / tol):.2f} x the tolerance at {np.argwhere(bad)[0]}"


def product_run(A, W, bias, R, M, N, K, dt, epi, tanh=False, ld=None):
    ld = ld or (N + 7) // 8 * 8
    y = torch.full((M + 1, ld), 7.0, device="cuda", dtype=tdt(dt))
    r = put(R, dt, ld) if epi == 2 else None
    b = None if bias is None else torch.from_numpy(bias).to("cuda", tdt(dt))
    vb.gemm_mx4(dt, A[0], A[0].stride(0), A[1], W[0], W[0].stride(0), W[1], b, y, ld, r, ld, M, N, K, epi, tanh)
    vb.check_device()
    y = get(y).astype(np.float64)
    assert (y[M] == 7).all() and (y[:, N:] == 7).all(), "wrote past the output"
    return y[:M, :N]


SHAPES = [(1, 1, 1), (1, 80, 32), (1, 4096, 1024), (2, 129, 33), (3, 1000, 200), (4, 31, 64), (5, 256, 1024), (8, 70, 2100),
          (9, 1024, 4096), (17, 257, 96), (64, 512, 512), (127, 80, 184), (128, 128, 128), (129, 130, 160), (300, 1000, 1000),
          (512, 300, 320), (1000, 2048, 512), (2400, 1024, 544), (4600, 1024, 96), (5000, 1024, 1000), (20000, 800, 320),
          (40000, 80, 256), (3, 500, 2100), (4, 1000, 4096), (1, 40, 5000), (2, 300, 9000), (4, 33, 8200), (129, 1, 64),
          (130, 7, 33), (5, 3, 1), (40000, 1000, 96), (20000, 1000, 1100), (20001, 1001, 1100), (20000, 998, 1100)]


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, dt):
    A, W, bias, R = product_case(M, N, K, dt)
    epi = (M + N + K) % 3
    got = product_run(A, W, bias, R, M, N, K, dt, epi)
    product_check(got, A[2], W[2], bias, R, dt, epi)


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("epi,tanh,has_bias", [(0, False, False), (0, False, True), (1, False, True), (1, True, True),
                                               (2, False, False), (2, False, True)])
def test_product_epilogues(M, epi, tanh, has_bias):
    for dt in (vb.FP16, vb.FP32):
        N, K = 200, 352
        A, W, bias, R = product_case(M, N, K, dt, 3)
        bias = bias if has_bias else None
        got = product_run(A, W, bias, R, M, N, K, dt, epi, tanh, ld=208)
        product_check(got, A[2], W[2], bias, R, dt, epi, tanh)


@pytest.mark.parametrize("M", [2, 200])
def test_product_nan_blocks_and_zero_rows(M):
    """A NaN block makes its row (of A) or column (of W) NaN and nothing else; a row of zeros gives the bias."""
    N, K = 96, 256
    A, W, bias, R = product_case(M, N, K, vb.FP32, 5)
    a, w = A[2].copy(), W[2].copy()
    a[0] = 0
    a[1, 100] = np.nan
    w[7, 3] = np.inf
    A, W = blocks(a), blocks(w)
    got = product_run(A, W, bias, R, M, N, K, vb.FP32, 0)
    nan = np.zeros((M, N), bool)
    nan[1], nan[:, 7] = True, True
    assert np.array_equal(np.isnan(got), nan)
    keep = np.arange(N) != 7
    assert np.array_equal(got[0, keep], bias[keep])


@pytest.mark.parametrize("M,N,K", [(2, 70, 64), (5, 100, 96), (300, 1000, 1100), (20000, 1001, 1100)])
def test_product_ignores_the_scale_bytes_of_absent_rows(M, N, K):
    """Whatever the last tiles hold for rows past M and N: the same bits, in values and in 4-bit blocks."""
    A, W, bias, R = product_case(M, N, K, vb.FP16, 4)
    ld, ldc, z = (N + 7) // 8 * 8, vb.mx4_row_bytes(N), vb.mx4_scale_bytes(M, N)
    b = torch.from_numpy(bias).to("cuda", torch.float16)
    present = np.ones((M, -(-N // 32)), np.uint8)
    outs = []
    for byte in (0, 255):
        sc = []
        for t, rows in ((A[1], M), (W[1], N)):
            absent = ref.tile_scales(np.ones((rows, 4 * -(-K // 128)), np.uint8)) == 0
            t = t.clone()
            t[torch.from_numpy(absent).cuda()] = byte
            sc.append(t)
        y = torch.zeros(M, ld, device="cuda", dtype=torch.float16)
        vb.gemm_mx4(vb.FP16, A[0], A[0].stride(0), sc[0], W[0], W[0].stride(0), sc[1], b, y, ld, None, 0, M, N, K, 0)
        codes, tiles = torch.zeros(M, ldc, device="cuda", dtype=torch.uint8), torch.zeros(z, device="cuda", dtype=torch.uint8)
        vb.gemm_mx4_quant(vb.FP16, A[0], A[0].stride(0), sc[0], W[0], W[0].stride(0), sc[1], b, codes, ldc, tiles, M, N, K, 1)
        vb.check_device()
        outs.append((get(y), get(codes), get(tiles)[ref.tile_scales(present) == 1]))
    assert all(np.array_equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("M", [2, 200])
def test_product_of_extreme_scales(M):
    """Scales far from 1 whose products are not: 2^p in a row of A against 2^-p in all of W, and the other way round."""
    N, K, dt = 40, 160, vb.FP32
    rng = np.random.default_rng(6)
    a, w = rng.normal(size=(M, K)), rng.normal(size=(N, K))
    for p in (60, 100, 120, -60, -100, -118):
        A, W = blocks(a * 2.0 ** p), blocks(w * 2.0 ** -p)
        got = product_run(A, W, None, None, M, N, K, dt, 0)
        product_check(got, A[2], W[2], None, None, dt, 0)


@pytest.mark.parametrize("M", [2, 200])
def test_product_residual_in_place_and_strided_codes(M):
    """R is Y; codes whose rows are further apart than they need."""
    N, K, dt = 136, 224, vb.FP16
    A, W, bias, R = product_case(M, N, K, dt, 9)

    def wide(c):
        t = torch.full((c.shape[0], c.shape[1] + 48), 0xFF, device="cuda", dtype=torch.uint8)
        t[:, :c.shape[1]] = c
        return t

    ca, cw, y = wide(A[0]), wide(W[0]), put(R, dt)
    b = torch.from_numpy(bias).to("cuda", tdt(dt))
    vb.gemm_mx4(dt, ca, ca.stride(0), A[1], cw, cw.stride(0), W[1], b, y, N, y, N, M, N, K, 2)
    product_check(get(y).astype(np.float64), A[2], W[2], bias, R, dt, 2)


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 64, 64), (3, 70, 200), (7, 192, 96), (129, 100, 64), (300, 1000, 320),
                                   (2400, 1000, 224), (5000, 1024, 96), (20000, 800, 160), (40000, 1000, 96),
                                   (20001, 1000, 1100)])
def test_product_in_4_bits(M, N, K, dt):
    """The output blocks: scale and values are those of some number within the fp32 error of the exact one."""
    A, W, bias, _ = product_case(M, N, K, dt, 1)
    epi = (M + N) % 2
    nb, ldc = -(-N // 32), vb.mx4_row_bytes(N) + 16
    codes = torch.full((M + 1, ldc), 0xEE, device="cuda", dtype=torch.uint8)
    tiles = torch.full((vb.mx4_scale_bytes(M, N),), 0xEE, device="cuda", dtype=torch.uint8)
    b = torch.from_numpy(bias).to("cuda", tdt(dt))
    vb.gemm_mx4_quant(dt, A[0], A[0].stride(0), A[1], W[0], W[0].stride(0), W[1], b, codes, ldc, tiles, M, N, K, epi)
    vb.check_device()
    c = get(codes)
    assert (c[:, ldc - 16:] == 0xEE).all() and (c[M] == 0xEE).all()
    sb = ref.untile_scales(get(tiles), M, -(-nb // 4) * 4)
    assert (sb[:, nb:] == 0).all()
    y, err = product_exact(A[2], W[2], bias, None, epi, False)
    low, high = np.maximum(np.abs(y) - err, 0), np.abs(y) + err
    assert (ref.quantize(low)[1] <= sb[:, :nb]).all() and (sb[:, :nb] <= ref.quantize(high)[1]).all()
    v = ref.values(c[:M, :ldc - 16], sb[:, :nb], 32 * nb)
    assert (v[:, N:] == 0).all()
    assert (ref.round_to(y - err, sb[:, :nb]) <= v[:, :N]).all() and (v[:, :N] <= ref.round_to(y + err, sb[:, :nb])).all()


# ------------------------------------------------------------------ block norm

def norm_tol(v, n, size, w, b, dt):
    """|normalised value| etc. -> tolerance of the norm's fp32 result."""
    scale = 1.0 if w is None else np.abs(w)
    return 2.0 ** -17 * (scale * (np.abs(n) + size + 1) + (0 if b is None else np.abs(b)))


def norm_case(rows, C, dt, groups, rng, mean=0.0):
    x, h = (rounded(rng.normal(size=(rows, C)) * s + mean, dt) for s in (2.0, 0.7))
    g, sc, sh = (rounded(0.3 * rng.normal(size=(groups, C)), dt) for _ in range(3))
    w = [(1 + 0.2 * rng.normal(size=C)).astype(np.float32) for _ in range(2)]
    b = [(0.2 * rng.normal(size=C)).astype(np.float32) for _ in range(2)]
    return x, h, g, sc, sh, w, b


def norm_check(got_x, got_y, x, h, post, pw, pb, g, rs, pre, w, b, sc, sh, dt, eps=1e-5):
    """x' against 64 bits; y against 64 bits of the norm of the x' that the kernel stored."""
    t, e = rs * x, 2.0 ** -23 * np.abs(rs * x)
    if h is not None:
        n, size = ref.norm(h, post, None, None, eps)
        p, _ = ref.norm(h, post, pw, pb, eps)
        pe = norm_tol(h, n, size, pw, pb, dt) if post else 0
        if g is not None:
            p, pe = p * g, (pe + 2.0 ** -23 * np.abs(p)) * np.abs(g)
        t, e = t + p, e + pe + 2.0 ** -23 * (np.abs(t) + np.abs(p))
    tol = e + HALF_STEP[dt] * (np.abs(t) + e) + TINY[dt]
    assert (np.abs(got_x - t) <= tol).all(), f"x': {np.max(np.abs(got_x - t) / tol):.2f} x the tolerance"
    if got_y is None:
        return
    n, size = ref.norm(got_x, pre, None, None, eps)
    y, _ = ref.norm(got_x, pre, w, b, eps)
    e = norm_tol(got_x, n, size, w, b, dt) if pre else 0
    if sc is not None:
        y, e = y * (1 + sc), (e + 2.0 ** -22 * np.abs(y)) * (1 + np.abs(sc))
    if sh is not None:
        y, e = y + sh, e + 2.0 ** -23 * (np.abs(y) + np.abs(sh))
    tol = e + HALF_STEP[dt] * (np.abs(y) + e) + TINY[dt]
    assert (np.abs(got_y - y) <= tol).all(), f"y: {np.max(np.abs(got_y - y) / tol):.2f} x the tolerance"


def norm_run(x, h, post, pw, pb, g, rs, pre, w, b, sc, sh, group, dt, ld=None, skew=0):
    rows, C = x.shape
    ld = ld or C
    f32 = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    opt = lambda a: None if a is None else put(a, dt, ld, skew=skew)  # noqa: E731
    out, y = (torch.full((rows + 1, ld), 7.0, device="cuda", dtype=tdt(dt)) for _ in range(2))
    vb.block_norm(dt, rows, C, put(x, dt, ld, skew=skew), ld, h=opt(h), ldh=ld, post=post, post_w=f32(pw), post_b=f32(pb),
                  gate=opt(g), ldgate=ld, res_scale=rs, out=out, ldo=ld, pre=pre, pre_w=f32(w), pre_b=f32(b), scale=opt(sc),
                  shift=opt(sh), ldmod=ld, rows_per_group=group, y=y, ldy=ld)
    torch.cuda.synchronize()
    for t in (out, y):
        assert (t[rows] == 7).all() and (t[:, C:] == 7).all(), "wrote past the rows"
    return get(out)[:rows, :C].astype(np.float64), get(y)[:rows, :C].astype(np.float64)


NORM_SHAPES = [(1, 1), (2, 7), (9, 8), (5, 100), (3, 256), (1, 1024), (33, 1000), (7, 2048), (3, 2056), (2, 5000), (2, 16384),
               (1300, 264), (1200, 1024), (1201, 2000), (1199, 517), (1300, 700), (1250, 1404), (1205, 2800), (1300, 4104),
               (1190, 6004), (1195, 8192), (1189, 8200), (1204, 1404), (1204, 2800), (1300, 5000), (1300, 8096)]


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows,C", NORM_SHAPES)
def test_block_norm(rows, C, dt):
    rng = np.random.default_rng(rows + C)
    i = rows + C
    post, pre = i % 3, (i // 3) % 3
    group = [0, 1, 2, max(1, rows // 3)][i % 4]
    groups = -(-rows // group) if group else 1
    at = np.arange(rows) // group if group else np.zeros(rows, int)
    for ld, skew in ((C, 0), (C + 8 + (-C) % 8, 0), (C + 1, 1)):
        x, h, g, sc, sh, w, b = norm_case(rows, C, dt, groups, rng, mean=[0, 5.0][rows % 2])
        got = norm_run(x, h, post, w[0], b[0], g, 0.75, pre, w[1], b[1], sc, sh, group, dt, ld, skew)
        norm_check(*got, x, h, post, w[0], b[0], g[at], 0.75, pre, w[1], b[1], sc[at], sh[at], dt)


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows", [3, 1500])
def test_block_norm_without_parts(rows, dt):
    """Each part absent; x' alone; in place."""
    C = 384
    rng = np.random.default_rng(rows)
    x, h, g, sc, sh, w, b = norm_case(rows, C, dt, 1, rng)
    at = np.zeros(rows, int)
    for post in (0, 1, 2):
        for pre in (0, 1, 2):
            got = norm_run(x, None, post, w[0], b[0], g, 0.5, pre, None, b[1], sc, None, 0, dt)
            norm_check(*got, x, None, post, None, None, None, 0.5, pre, None, b[1], sc[at], None, dt)
            got = norm_run(x, h, post, None, None, None, 1.0, pre, w[1], None, None, sh, 0, dt)
            norm_check(*got, x, h, post, None, None, None, 1.0, pre, w[1], None, None, sh[at], dt)
    d, e, y = put(x, dt), put(h, dt), put(h, dt)
    vb.block_norm(dt, rows, C, d, C, h=y, ldh=C, post=1, out=d, ldo=C, pre=1, y=y, ldy=C)  # x' over x, y over h
    first = get(d).astype(np.float64), get(y).astype(np.float64)
    norm_check(*first, x, h, 1, None, None, None, 1.0, 1, None, None, None, None, dt)
    d = put(x, dt)
    vb.block_norm(dt, rows, C, d, C, h=e, ldh=C, post=1, out=d, ldo=C)
    assert np.array_equal(get(d).astype(np.float64), first[0])


def test_block_norm_constant_rows_and_not_finite():
    """A constant row normalises to zero (eps keeps it finite); NaN and Inf stay in their rows."""
    C, dt = 512, vb.FP32
    rng = np.random.default_rng(2)
    x = rng.normal(size=(6, C))
    x[1], x[2], x[3, 17], x[4, 3] = 0.0, 4.0, np.nan, np.inf
    y = torch.zeros(6, C, device="cuda")
    vb.block_norm(dt, 6, C, put(x, dt), C, pre=vb.NORM_LAYER, y=y, ldy=C)
    got = get(y)
    assert (got[1] == 0).all() and (got[2] == 0).all()
    assert np.isnan(got[3]).all() and np.isnan(got[4]).any() and np.isfinite(got[[0, 5]]).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows,C", [(1, 32), (3, 1000), (130, 96), (40, 1), (1300, 1024), (1250, 100), (5, 4100), (1200, 744),
                                    (1300, 5000), (1190, 8100)])
def test_block_norm_in_4_bits(rows, C, dt):
    """The 4-bit output is the quantised fp32 y: with fp32 storage, the same bits as quantising the y it stores."""
    rng = np.random.default_rng(rows + C)
    x, h, g, sc, sh, w, b = norm_case(rows, C, dt, 1, rng)
    f32 = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(h=put(h, dt), ldh=C, post=2, post_w=f32(w[0]), gate=put(g, dt), pre=1, pre_w=f32(w[1]), pre_b=f32(b[1]),
              scale=put(sc, dt), shift=put(sh, dt))
    y = torch.zeros(rows, C, device="cuda", dtype=tdt(dt))
    vb.block_norm(dt, rows, C, put(x, dt), C, y=y, ldy=C, **kw)
    nb, ldc = -(-C // 32), vb.mx4_row_bytes(C) + 16
    codes = torch.full((rows + 1, ldc), 0xEE, device="cuda", dtype=torch.uint8)
    tiles = torch.full((vb.mx4_scale_bytes(rows, C),), 0xEE, device="cuda", dtype=torch.uint8)
    out = torch.zeros(rows, C, device="cuda", dtype=tdt(dt))
    vb.block_norm(dt, rows, C, put(x, dt), C, y_codes=codes, ldc=ldc, y_scales=tiles, out=out, ldo=C, **kw)
    assert (get(codes)[:, ldc - 16:] == 0xEE).all() and (get(codes)[rows] == 0xEE).all()
    got_s = ref.untile_scales(get(tiles), rows, -(-nb // 4) * 4)
    assert (got_s[:, nb:] == 0).all()
    if dt == vb.FP32:
        rc, rs = ref.quantize(get(y))
        assert np.array_equal(got_s[:, :nb], rs) and np.array_equal(get(codes)[:rows, :ldc - 16], rc)
    else:  # quantised before the rounding to fp16: within a code's step of y, half of it and y's own rounding
        v = ref.values(get(codes)[:rows, :ldc - 16], got_s[:, :nb], C)
        step = np.repeat(np.exp2(got_s[:, :nb].astype(np.float64) - 127), 32, 1)[:, :C] * 2.0
        assert (np.abs(v - get(y)) <= step + 2.0 ** -10 * np.abs(get(y))).all()


# ------------------------------------------------------------------ together, streams, graphs, far rows

def linear(rng, n, k):
    w = blocks(rng.normal(size=(n, k)) / math.sqrt(k))
    return w, rounded(rng.normal(size=n) * 0.1, vb.FP16)


def mx4_space(rows, k):
    return (torch.zeros(rows, vb.mx4_row_bytes(k), device="cuda", dtype=torch.uint8),
            torch.zeros(vb.mx4_scale_bytes(rows, k), device="cuda", dtype=torch.uint8))


def held(space, rows, k):
    """The values in 64 bits that codes and scale tiles on the device stand for."""
    nb = -(-k // 32)
    return ref.values(get(space[0]), ref.untile_scales(get(space[1]), rows, -(-nb // 4) * 4)[:, :nb], k)


class Block:
    """A processor block with 4-bit Linear layers: norm -> q|k|v|self, edge attention, proj, norm with the gate,
    mlp1 with GELU, mlp2 + residual, on one stream's buffers."""

    def __init__(self, H, C, heads, seed=0):
        rng = np.random.default_rng(seed)
        self.H, self.C, self.heads, self.F = H, C, heads, 4 * C
        E = 5 * H
        ei = np.stack([rng.integers(0, H, E), rng.integers(0, H, E)]).astype(np.int64)
        self.rp, self.src, _, self.attr = vb.build_csr(ei, rounded(rng.normal(size=(E, 3)), vb.FP16).astype(np.float32), H, H)
        self.d_rp = torch.from_numpy(self.rp).cuda()
        self.d_ed = torch.from_numpy(vb.pack_edges(self.src, self.attr, True)).cuda()
        self.w4 = rounded(rng.normal(size=(4, C)) * 0.3, vb.FP16).astype(np.float32)
        self.d_w4 = torch.from_numpy(self.w4).cuda()
        self.lin = {n: linear(rng, o, i) for n, o, i in (("qkvs", 4 * C, C), ("proj", C, C), ("mlp1", self.F, C), ("mlp2", C, self.F))}
        self.x = rounded(rng.normal(size=(H, C)), vb.FP16)
        self.gate, self.scale, self.shift = (rounded(0.3 * rng.normal(size=(1, C)), vb.FP16) for _ in range(3))
        self.w = (1 + 0.1 * rng.normal(size=C)).astype(np.float32)
        d = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.float16)  # noqa: E731
        self.t = {"x": put(self.x, vb.FP16), "gate": put(self.gate, vb.FP16), "scale": put(self.scale, vb.FP16),
                  "shift": put(self.shift, vb.FP16), "w": torch.from_numpy(self.w).cuda(), "qkvs": d(H, 4 * C), "att": d(H, C),
                  "proj": d(H, C), "x1": d(H, C), "out": d(H, C), "n1": mx4_space(H, C), "a4": mx4_space(H, C),
                  "n2": mx4_space(H, C), "f4": mx4_space(H, self.F)}
        self.b = {n: torch.from_numpy(v[1]).to("cuda", torch.float16) for n, v in self.lin.items()}

    def run(self, stream):
        H, C, F, t = self.H, self.C, self.F, self.t

        def gemm(a, n, y, N, K, r=None, epi=0):
            w = self.lin[n][0]
            vb.gemm_mx4(vb.FP16, a[0], a[0].stride(0), a[1], w[0], w[0].stride(0), w[1], self.b[n], y, N, r, N, H, N, K, epi,
                        stream=stream)

        vb.block_norm(vb.FP16, H, C, t["x"], C, pre=vb.NORM_LAYER, pre_w=t["w"], scale=t["scale"], shift=t["shift"],
                      y_codes=t["n1"][0], ldc=t["n1"][0].stride(0), y_scales=t["n1"][1], stream=stream)
        gemm(t["n1"], "qkvs", t["qkvs"], 4 * C, C)
        q = t["qkvs"]
        vb.attention(vb.FP16, self.d_rp, self.d_ed, 0, H, q, 4 * C, q[:, C:], q[:, 2 * C:], 4 * C, q[:, 3 * C:], 4 * C, t["att"], C,
                     self.d_w4, C, self.heads, C // self.heads, stream=stream)
        vb.mx4_quantize(vb.FP16, t["att"], C, H, C, t["a4"][0], t["a4"][0].stride(0), t["a4"][1], stream=stream)
        gemm(t["a4"], "proj", t["proj"], C, C)
        vb.block_norm(vb.FP16, H, C, t["x"], C, h=t["proj"], ldh=C, post=vb.NORM_RMS, gate=t["gate"], out=t["x1"], ldo=C,
                      pre=vb.NORM_LAYER, pre_w=t["w"], scale=t["scale"], shift=t["shift"], y_codes=t["n2"][0],
                      ldc=t["n2"][0].stride(0), y_scales=t["n2"][1], stream=stream)
        w = self.lin["mlp1"][0]
        vb.gemm_mx4_quant(vb.FP16, t["n2"][0], t["n2"][0].stride(0), t["n2"][1], w[0], w[0].stride(0), w[1], self.b["mlp1"],
                          t["f4"][0], t["f4"][0].stride(0), t["f4"][1], H, F, C, 1, stream=stream)
        gemm(t["f4"], "mlp2", t["out"], C, F, t["x1"], 2)

    def verify(self):
        """Each stage against 64 bits of the stage's own inputs as the device holds them."""
        H, C, F, t, f64 = self.H, self.C, self.F, self.t, lambda k: get(self.t[k]).astype(np.float64)
        product_check(f64("qkvs"), held(t["n1"], H, C), self.lin["qkvs"][0][2], self.lin["qkvs"][1], None, vb.FP16, 0)
        q = f64("qkvs")
        att = attention(self.rp, self.src, self.attr, q, self.w4.astype(np.float64), self.heads, C)
        assert np.abs(f64("att") - att).max() <= 2e-3 * np.abs(att).max()
        rc, rs = ref.quantize(f64("att"))
        assert np.array_equal(held(t["a4"], H, C), ref.values(rc, rs, C))
        product_check(f64("proj"), held(t["a4"], H, C), self.lin["proj"][0][2], self.lin["proj"][1], None, vb.FP16, 0)
        norm_check(f64("x1"), None, f64("x"), f64("proj"), 2, None, None, self.gate, 1.0, 0, None, None, None, None, vb.FP16)
        for key, x in (("n1", f64("x")), ("n2", f64("x1"))):
            y, _ = ref.norm(x, 1, self.w, None, 1e-5)
            y = y * (1 + self.scale) + self.shift
            n, size = ref.norm(x, 1, None, None, 1e-5)
            e = norm_tol(x, n, size, self.w, None, vb.FP16) * (1 + np.abs(self.scale)) + 2.0 ** -21 * (np.abs(y) + np.abs(self.shift))
            blocks_check(t[key], H, C, y, e)
        y, err = product_exact(held(t["n2"], H, C), self.lin["mlp1"][0][2], self.lin["mlp1"][1], None, 1, False)
        blocks_check(t["f4"], H, F, y, err)
        product_check(f64("out"), held(t["f4"], H, F), self.lin["mlp2"][0][2], self.lin["mlp2"][1], f64("x1"), vb.FP16, 2)


def attention(rp, src, attr, qkvs, w4, heads, C):
    """Graph attention in 64 bits: scores and values with the edge term, + self."""
    q, k, v, xs = (qkvs[:, i * C:(i + 1) * C] for i in range(4))
    out, hd = xs.copy(), C // heads
    for i in range(len(rp) - 1):
        e = slice(rp[i], rp[i + 1])
        if rp[i] == rp[i + 1]:
            continue
        term = attr[e].astype(np.float64) @ w4[:3] + w4[3]
        kk, vv = (k[src[e]] + term).reshape(-1, heads, hd), (v[src[e]] + term).reshape(-1, heads, hd)
        s = np.einsum("ehd,hd->eh", kk, q[i].reshape(heads, hd)) / math.sqrt(hd)
        p = np.exp(s - s.max(0))
        out[i] += np.einsum("eh,ehd->hd", p / p.sum(0), vv).ravel()
    return out


def blocks_check(space, rows, k, y, err):
    """4-bit blocks that some number within err of y quantises to."""
    nb = -(-k // 32)
    sb = ref.untile_scales(get(space[1]), rows, -(-nb // 4) * 4)[:, :nb]
    assert (ref.quantize(np.maximum(np.abs(y) - err, 0))[1] <= sb).all() and (sb <= ref.quantize(np.abs(y) + err)[1]).all()
    v = ref.values(get(space[0]), sb, k)
    assert (ref.round_to(y - err, sb) <= v).all() and (v <= ref.round_to(y + err, sb)).all()


@pytest.mark.parametrize("H,C,heads", [(1, 128, 4), (300, 256, 4), (2600, 512, 8)])
def test_block_of_4_bit_layers(H, C, heads):
    b = Block(H, C, heads)
    b.run(torch.cuda.current_stream().cuda_stream)
    vb.check_device()
    b.verify()


def test_block_captured_replayed_and_two_at_once():
    """A captured block replayed on new inputs, and two blocks on two streams at once, give an eager run's bits."""
    blk = [Block(700, 256, 4, seed=i) for i in range(2)]
    for b in blk:
        b.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = [get(b.t["out"]).copy() for b in blk]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for b in blk:
            b.t["out"].zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for b, s in zip(blk, streams):
                b.run(s.cuda_stream)
        torch.cuda.synchronize()
        for b, w in zip(blk, want):
            assert np.array_equal(get(b.t["out"]), w)
    graphs = []
    for b, s in zip(blk, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.run(s.cuda_stream)
        graphs.append(g)
    x = [b.t["x"].clone() for b in blk]
    blk[0].t["x"].copy_(x[1]), blk[1].t["x"].copy_(x[0])  # other inputs
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    swapped = [get(b.t["out"]).copy() for b in blk]
    for b, w in zip(blk, swapped):
        b.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert np.array_equal(get(b.t["out"]), w) and not np.array_equal(w, want[0])
    vb.check_device()


def test_rows_past_32_bit_offsets():
    """Rows whose element and byte offsets pass 2^32: a stride of 2^20 elements, 4200 rows (8.8 GB)."""
    rows, K, N, ld = 4200, 64, 64, 1 << 20
    rng = np.random.default_rng(4)
    x = rounded(rng.normal(size=(rows, K)), vb.FP16)
    big = torch.zeros(rows, ld, device="cuda", dtype=torch.float16)
    big[:, :K] = torch.from_numpy(x).to("cuda", torch.float16)
    codes, tiles = mx4_space(rows, K)
    vb.mx4_quantize(vb.FP16, big, ld, rows, K, codes, K // 2, tiles)
    rc, rs = ref.quantize(x)
    assert np.array_equal(get(codes), rc) and np.array_equal(get(tiles), ref.tile_scales(rs))
    W = blocks(rng.normal(size=(N, K)))
    y = big[:, 128:]
    vb.gemm_mx4(vb.FP16, codes, K // 2, tiles, W[0], W[0].stride(0), W[1], None, y, ld, None, 0, rows, N, K)
    product_check(get(big[:, 128:128 + N]).astype(np.float64), ref.values(rc, rs, K), W[2], None, None, vb.FP16, 0)
    o = big[:, 256:]
    vb.block_norm(vb.FP16, rows, K, big, ld, pre=vb.NORM_LAYER, y=o, ldy=ld)
    z = big[:, 384:]
    vb.mx4_dequantize(vb.FP16, codes, K // 2, tiles, rows, K, z, ld)
    torch.cuda.synchronize()
    norm_check(x, get(big[:, 256:256 + K]).astype(np.float64), x, None, 0, None, None, None, 1.0, 1, None, None, None, None, vb.FP16)
    assert np.array_equal(get(big[:, 384:384 + K]).astype(np.float64), rounded(ref.values(rc, rs, K), vb.FP16))
    assert not big[:, 64:128].any() and not big[:, 192:256].any() and not big[:, 320:384].any() and not big[:, 448:].any()


def test_first_calls_inside_a_capture():
    """A process whose first calls are made inside a stream capture: nothing in them is forbidden there."""
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = %r
import numpy as np, torch, varda_b200 as vb
import test_mx4_gpu as t
b = t.Block(2600, 512, 8)
s = torch.cuda.Stream(); torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    b.run(s.cuda_stream)
with torch.cuda.stream(s):
    g.replay()
torch.cuda.synchronize(); vb.check_device(); b.verify(); print("verified")
""" % [p for p in sys.path if p]
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "verified" in r.stdout, r.stderr[-2000:]
