"""Edges of the 4-bit product and the block norm on the B200: GELU's tails and its tanh form on every tile, NaN and
Inf into 4-bit blocks, modulations of several groups, groups without a modulation, what is past the last column.

Tolerances as in test_mx4_gpu.py. GELU alone (a product of zeros and a bias x) is max(x, 0) - t, t = |x| Phi(-|x|) as
|x| 2^P: 2^P within 2^-22 (ex2) and ln 2 times P's rounding, 2^-22 (1 + |P|), of itself, P's fit (2e-7 of t's largest
error for fp16 and 4-bit output, 5e-9 for fp32 output), and half a step of fp32 of the result. Past -5.6, where the fit is
only bounded, the values must fall as the true ones do: at most 16 times them, and nothing below -14. Of -Inf it is 0.
"""
import math

import numpy as np
import pytest
from scipy.special import erfc, log_ndtr

import mx4_reference as ref
import test_mx4_gpu as t
import varda_b200 as vb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# (M, N, K) whose product takes tiles of 64 and 128 columns and the pairs' 256
TILES = [(130, 641, 96), (2000, 1021, 96), (9500, 4075, 544)]


def quantized(dt, A, W, bias, M, N, K, epi, tanh=False):
    """vb_gemm_mx4_quant -> (codes [M, 16 nb], scale bytes [M, nb])."""
    nb = -(-N // 32)
    codes, tiles = t.mx4_space(M, N)
    b = None if bias is None else torch.from_numpy(bias).to("cuda", t.tdt(dt))
    vb.gemm_mx4_quant(dt, A[0], A[0].stride(0), A[1], W[0], W[0].stride(0), W[1], b, codes, codes.stride(0), tiles, M, N, K, epi,
                      tanh)
    vb.check_device()
    return t.get(codes), ref.untile_scales(t.get(tiles), M, -(-nb // 4) * 4)[:, :nb]


def zeros(rows, K):
    return (torch.zeros(rows, vb.mx4_row_bytes(K), device="cuda", dtype=torch.uint8),
            torch.zeros(vb.mx4_scale_bytes(rows, K), device="cuda", dtype=torch.uint8))


# ------------------------------------------------------------------ GELU

def sweep(N, dt):
    """N pre-activations in order (blocks of like sizes), dense over GELU's range, -Inf, Inf and NaN at the end."""
    n = N - 35
    x = np.sort(np.concatenate([np.linspace(-40, 40, n // 4), np.linspace(-16, -5, n // 4), np.linspace(-6, 6, n - n // 4 * 2)]))
    x[n // 2] = 0.0
    return t.rounded(np.concatenate([x, np.full(32, 1.0), [-np.inf, np.inf, np.nan]]), dt)


def gelu_bounds(x, dt):
    """(GELU in 64 bits, the bound of its error before the rounding to the output's type)."""
    with np.errstate(invalid="ignore"):
        y = 0.5 * x * erfc(-x / math.sqrt(2))
        tail, P = np.abs(x) * np.exp(log_ndtr(-np.abs(x))), -log_ndtr(-np.abs(x)) / math.log(2)
        err = 2.0 ** -24 * np.abs(y) + tail * (1 + math.log(2) * (1 + P)) * 2.0 ** -22 + (5e-9 if dt == vb.FP32 else 2e-7)
    return np.where(x == -np.inf, 0.0, y), np.where(x == -np.inf, 0.0, err)


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("M,N,K", TILES + [(2, 4000, 64), (1, 900, 64)])
def test_gelu_alone(M, N, K, dt):
    x = sweep(N, dt)
    got = t.product_run(zeros(M, K), zeros(N, K), x, None, M, N, K, dt, 1)
    assert (got == got[0])[:, ~np.isnan(got[0])].all() and (np.isnan(got) == np.isnan(got[0])).all()
    y, err = gelu_bounds(x, dt)
    assert np.array_equal(np.isnan(got[0]), np.isnan(y)) and got[0, N - 2] == np.inf
    ok = np.isfinite(y)
    g, y, err, x = got[0][ok], y[ok], err[ok], x[ok]
    tol = err + t.HALF_STEP[dt] * (np.abs(y) + err) + t.TINY[dt]
    assert (np.abs(g - y) <= tol).all(), f"{np.max(np.abs(g - y) / tol):.2f} x the tolerance at {x[np.argmax(np.abs(g - y) / tol)]}"
    far = x < -5.6
    assert (np.abs(g[far]) <= 16 * np.abs(y[far]) + 2.0 ** -126 + t.TINY[dt]).all(), "the tail does not vanish"
    assert (g[x < -14] == 0).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
def test_gelu_does_not_depend_on_the_rows(dt):
    """The few-row kernel and every tile apply the same GELU."""
    N, K = 4075, 544
    x = sweep(N, dt)
    rows = [t.product_run(zeros(M, K), zeros(N, K), x, None, M, N, K, dt, 1)[0] for M in (1, 2, 3, 1000, 9500)]
    for r in rows[1:]:
        np.testing.assert_array_equal(r, rows[0])


@pytest.mark.parametrize("M,N,K", TILES)
def test_gelu_alone_in_4_bits(M, N, K):
    x = sweep(N, vb.FP16)
    codes, sb = quantized(vb.FP16, zeros(M, K), zeros(N, K), x, M, N, K, 1)
    assert (codes == codes[0]).all() and (sb == sb[0]).all()
    codes, sb, nb = codes[:1], sb[:1], sb.shape[1]
    y, err = gelu_bounds(x, vb.FP16)
    bad = np.array([not np.isfinite(y[32 * b:32 * b + 32]).all() for b in range(nb)])
    assert np.array_equal(sb[0] == 255, bad) and (codes.reshape(nb, 16)[bad] == 0).all()
    y, err = np.where(np.isfinite(y), y, 0), np.where(np.isfinite(y), err, 0)
    v, keep = ref.values(codes, sb, N)[0], np.repeat(~bad, 32)[:N]
    assert (ref.round_to((y - err)[None], sb)[0] <= v)[keep].all() and (v <= ref.round_to((y + err)[None], sb)[0])[keep].all()
    far = keep & (x < -5.6)  # a block of the tail: at most 16 times its values, each then rounded by half of itself at most
    top = np.repeat([np.abs(y[32 * b:32 * b + 32]).max() for b in range(nb)], 32)[:N]
    assert (np.abs(v[far]) <= 24 * top[far] + 2.0 ** -126).all() and (v[keep & (x < -17)] == 0).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("M,N,K", TILES)
def test_tanh_gelu_on_every_tile(M, N, K, dt):
    A, W, bias, _ = t.product_case(M, N, K, dt, 11)
    got = t.product_run(A, W, bias, None, M, N, K, dt, 1, tanh=True)
    t.product_check(got, A[2], W[2], bias, None, dt, 1, tanh=True)
    codes, sb = quantized(dt, A, W, bias, M, N, K, 1, tanh=True)
    y, err = t.product_exact(A[2], W[2], bias, None, 1, True)
    assert (ref.quantize(np.maximum(np.abs(y) - err, 0))[1] <= sb).all() and (sb <= ref.quantize(np.abs(y) + err)[1]).all()
    v = ref.values(codes, sb, N)
    assert (ref.round_to(y - err, sb) <= v).all() and (v <= ref.round_to(y + err, sb)).all()


# ------------------------------------------------------------------ NaN and Inf

@pytest.mark.parametrize("epi,tanh", [(0, False), (1, False), (1, True)])
@pytest.mark.parametrize("M,N,K", TILES)
def test_product_not_finite_in_4_bits(M, N, K, epi, tanh):
    """A NaN block of A makes its row's blocks NaN, one of W or a bias of +-Inf the blocks of its column, and none else."""
    rng = np.random.default_rng(M)
    a, w, bias = rng.normal(size=(M, K)), rng.normal(size=(N, K)) / math.sqrt(K), t.rounded(rng.normal(size=N), vb.FP16)
    a[M // 2, 40], w[70, 3], bias[N - 1], bias[200], bias[300] = np.nan, np.inf, np.inf, -np.inf, np.nan  # (GELU of -Inf is 0)
    codes, sb = quantized(vb.FP16, t.blocks(a), t.blocks(w), bias, M, N, K, epi, tanh)
    bad = np.zeros(sb.shape, bool)
    bad[M // 2] = True
    bad[:, [70 // 32, (N - 1) // 32, 300 // 32] + [200 // 32] * (epi == 0 or tanh)] = True
    assert np.array_equal(sb == 255, bad)
    assert (codes.reshape(*sb.shape, 16)[bad] == 0).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("kind", [vb.NORM_LAYER, vb.NORM_RMS])
@pytest.mark.parametrize("rows,C", [(7, 700), (1300, 60), (1300, 700), (1250, 1024), (1205, 2800), (1195, 5001)])
def test_block_norm_not_finite(rows, C, kind, dt):
    """NaN and Inf of x or h stay in their rows, and reach y and its 4-bit blocks as the definition has them."""
    rng = np.random.default_rng(rows + C)
    x, h, g, _, _, w, b = t.norm_case(rows, C, dt, 1, rng)
    x[1, C // 2], x[3, 0], h[4, C - 1], h[rows - 1, 1] = np.nan, np.inf, -np.inf, np.nan
    with np.errstate(invalid="ignore", over="ignore"):
        want_x = x + g * ref.norm(h, kind, w[0], b[0], 1e-5)[0]
        want_y = ref.norm(want_x, kind, w[1], b[1], 1e-5)[0]
    f32 = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(h=t.put(h, dt), ldh=C, post=kind, post_w=f32(w[0]), post_b=f32(b[0]), gate=t.put(g, dt), pre=kind, pre_w=f32(w[1]),
              pre_b=f32(b[1]))
    out, y = (torch.zeros(rows, C, device="cuda", dtype=t.tdt(dt)) for _ in range(2))
    vb.block_norm(dt, rows, C, t.put(x, dt), C, out=out, ldo=C, y=y, ldy=C, **kw)
    codes, tiles = t.mx4_space(rows, C)
    vb.block_norm(dt, rows, C, t.put(x, dt), C, y_codes=codes, ldc=codes.stride(0), y_scales=tiles, **kw)
    out, y = t.get(out).astype(np.float64), t.get(y).astype(np.float64)
    assert np.array_equal(np.isnan(out), np.isnan(want_x)) and np.array_equal(np.isinf(out), np.isinf(want_x))
    assert np.array_equal(np.isnan(y), np.isnan(want_y)) and not np.isinf(y).any()
    fine = np.setdiff1d(np.arange(rows), [1, 3, 4, rows - 1])
    t.norm_check(out[fine], y[fine], x[fine], h[fine], kind, w[0], b[0], g, 1.0, kind, w[1], b[1], None, None, dt)
    nb = -(-C // 32)
    sb = ref.untile_scales(t.get(tiles), rows, -(-nb // 4) * 4)[:, :nb]
    bad = ~np.isfinite(np.pad(want_y, ((0, 0), (0, 32 * nb - C)))).reshape(rows, nb, 32).all(-1)
    assert np.array_equal(sb == 255, bad) and (t.get(codes).reshape(rows, nb, 16)[bad] == 0).all()


@pytest.mark.parametrize("rows", [5, 1300])
def test_block_norm_infinite_modulation_without_bias(rows):
    """gate and 1 + scale of Inf times a value that is not zero are Inf, where no bias is multiplied with them."""
    C, dt = 256, vb.FP32
    rng = np.random.default_rng(rows)
    x, h, g, sc, _, w, _ = t.norm_case(rows, C, dt, 1, rng)
    g[0, 5], sc[0, 9] = np.inf, -np.inf
    out, y = (torch.zeros(rows, C, device="cuda") for _ in range(2))
    f32 = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    vb.block_norm(dt, rows, C, t.put(x, dt), C, h=t.put(h, dt), ldh=C, post=2, post_w=f32(w[0]), gate=t.put(g, dt), out=out, ldo=C)
    vb.block_norm(dt, rows, C, t.put(x, dt), C, pre=2, pre_w=f32(w[1]), scale=t.put(sc, dt), y=y, ldy=C)
    with np.errstate(invalid="ignore"):
        want_x, want_y = x + g * ref.norm(h, 2, w[0], None, 1e-5)[0], ref.norm(x, 2, w[1], None, 1e-5)[0] * (1 + sc)
    for got, want in ((t.get(out), want_x), (t.get(y), want_y)):
        assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any()
        assert np.array_equal(np.sign(got[np.isinf(want)]), np.sign(want[np.isinf(want)]))


# ------------------------------------------------------------------ groups, ends of rows

def run_norm(dt, x, C, group, y4, **kw):
    """vb_block_norm -> [x', y] or [x', codes, scale tiles] on the host."""
    rows = x.shape[0]
    out = torch.zeros(rows, C, device="cuda", dtype=t.tdt(dt))
    if y4:
        codes, tiles = t.mx4_space(rows, C)
        vb.block_norm(dt, rows, C, x, C, out=out, ldo=C, y_codes=codes, ldc=codes.stride(0), y_scales=tiles, rows_per_group=group, **kw)
        return [t.get(out), t.get(codes), t.get(tiles)]
    y = torch.zeros(rows, C, device="cuda", dtype=t.tdt(dt))
    vb.block_norm(dt, rows, C, x, C, out=out, ldo=C, y=y, ldy=C, rows_per_group=group, **kw)
    return [t.get(out), t.get(y)]


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows,C,group", [(5000, 64, 1024), (5000, 64, 1700), (5000, 700, 1024), (5000, 704, 1700), (5000, 1024, 1024),
                                          (4999, 1024, 1700), (3100, 5000, 1024), (2050, 8192, 1025), (20000, 100, 1033)])
def test_block_norm_of_several_groups(rows, C, group, dt):
    """Modulations of more than one group folded into the vectors: groups that divide neither the rows nor a CTA's."""
    rng = np.random.default_rng(rows + C + group)
    groups, at = -(-rows // group), np.arange(rows) // group
    x, h, g, sc, sh, w, b = t.norm_case(rows, C, dt, groups, rng)
    f32 = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(h=t.put(h, dt), ldh=C, post=1, post_w=f32(w[0]), post_b=f32(b[0]), gate=t.put(g, dt), ldgate=C, res_scale=0.75, pre=2,
              pre_w=f32(w[1]), pre_b=f32(b[1]), scale=t.put(sc, dt), shift=t.put(sh, dt), ldmod=C)
    d = t.put(x, dt)
    out, y = run_norm(dt, d, C, group, False, **kw)
    t.norm_check(out.astype(np.float64), y.astype(np.float64), x, h, 1, w[0], b[0], g[at], 0.75, 2, w[1], b[1], sc[at], sh[at], dt)
    out4, codes, tiles = run_norm(dt, d, C, group, True, **kw)
    assert np.array_equal(out4, out)
    nb = -(-C // 32)
    sb = ref.untile_scales(tiles, rows, -(-nb // 4) * 4)[:, :nb]
    if dt == vb.FP32:
        rc, rs = ref.quantize(y)
        assert np.array_equal(sb, rs) and np.array_equal(codes, rc)
    else:  # quantised before the rounding to fp16
        step = np.repeat(np.exp2(sb.astype(np.float64) - 127), 32, 1)[:, :C] * 2.0
        assert (np.abs(ref.values(codes, sb, C) - y) <= step + 2.0 ** -10 * np.abs(y)).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows,C", [(9, 100), (1300, 40), (1300, 1024), (1250, 2000)])
@pytest.mark.parametrize("group", [1, 3, 1100])
def test_groups_without_a_modulation(rows, C, group, dt):
    """rows_per_group says nothing where nothing is modulated: the bits of rows_per_group = 0. A gate without h, scale and
    shift without y, strides and a norm's weight without what they belong to are not read."""
    rng = np.random.default_rng(rows + C)
    x, h, _, _, _, w, b = t.norm_case(rows, C, dt, 1, rng)
    f32 = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(post=1, post_w=f32(w[0]), post_b=f32(b[0]), pre=2, pre_w=f32(w[1]), pre_b=f32(b[1]))
    d, e = t.put(x, dt), t.put(h, dt)
    for y4 in (False, True):
        for more in (dict(h=e, ldh=C), dict(gate=e, ldgate=C)):
            for p, q in zip(run_norm(dt, d, C, group, y4, **kw, **more), run_norm(dt, d, C, 0, y4, **kw, **{**more, "gate": None})):
                assert np.array_equal(p, q)
    kw = dict(pre=2, pre_w=f32(w[1]))
    for p, q in zip(run_norm(dt, d, C, group, False, **kw, ldh=C + 1, ldgate=C + 1, ldmod=C + 1, post=1, post_w=f32(np.ones(C + 1, np.float32))[1:]),
                    run_norm(dt, d, C, 0, False, **kw)):
        assert np.array_equal(p, q)
    outs = []
    for g, m in ((group, e), (0, None)):
        out = torch.zeros(rows, C, device="cuda", dtype=t.tdt(dt))
        vb.block_norm(dt, rows, C, d, C, h=e, ldh=C, post=1, out=out, ldo=C, scale=m, shift=m, ldmod=C, rows_per_group=g)
        outs.append(t.get(out))
    assert np.array_equal(*outs)


def test_groups_without_a_modulation_cost_nothing():
    """A group per row without a modulation takes no longer than none (three times it at most)."""
    rows, C, dt = 20000, 1024, vb.FP16
    x, h, y, out = (torch.randn(rows, C, device="cuda").half() for _ in range(4))
    w = torch.ones(C, device="cuda")
    s = torch.cuda.current_stream().cuda_stream

    def best(group):
        times = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                vb.block_norm(dt, rows, C, x, C, h=h, ldh=C, post=1, post_w=w, out=out, ldo=C, pre=1, pre_w=w, y=y, ldy=C,
                              rows_per_group=group, stream=s)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert best(1) <= 3 * best(0)


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("rows", [3, 1300])
@pytest.mark.parametrize("C", [1, 40, 301])
@pytest.mark.parametrize("pre", [0, 1, 2])
def test_codes_past_the_last_column_are_zero(rows, C, pre, dt):
    """... whatever the signs before it: res_scale < 0 and no h."""
    x = np.random.default_rng(C).normal(size=(rows, C))
    _, codes, tiles = run_norm(dt, t.put(x, dt), C, 0, True, res_scale=-1.0, pre=pre)
    c = np.stack((codes & 15, codes >> 4), -1).reshape(rows, -1)
    assert (c[:, C:] == 0).all()


@pytest.mark.parametrize("dt", [vb.FP16, vb.FP32])
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 9, 11])
@pytest.mark.parametrize("group", [0, 1])
def test_block_norm_of_narrow_rows(C, group, dt):
    """Many rows of a few columns, the last vector of a row reaching into the next."""
    rows, ld = 1300, -(-C // 4) * 4 if dt == vb.FP32 else -(-C // 8) * 8
    rng = np.random.default_rng(C)
    groups = rows if group else 1
    at = np.arange(rows) if group else np.zeros(rows, int)
    x, h, g, sc, sh, w, b = t.norm_case(rows, C, dt, groups, rng)
    got = t.norm_run(x, h, 1, w[0], b[0], g, 0.75, 2, w[1], b[1], sc, sh, group, dt, ld)
    t.norm_check(*got, x, h, 1, w[0], b[0], g[at], 0.75, 2, w[1], b[1], sc[at], sh[at], dt)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("rows,C,group", [(4100, 512, 1025), (2500, 256, 0), (40968, 512, 10242)])
def test_mlp_of_several_members(rows, C, group):
    """norm with a modulation per member -> product with GELU in 4 bits -> product + residual: every stage against 64 bits of
    what the device holds, and the same bits each time, with other inputs in between."""
    F, dt = 4 * C, vb.FP16
    rng = np.random.default_rng(rows)
    groups = -(-rows // group) if group else 1
    at = np.arange(rows) // group if group else np.zeros(rows, int)
    sets = [t.norm_case(rows, C, dt, groups, rng) for _ in range(2)]
    (W1, b1), (W2, b2) = t.linear(rng, F, C), t.linear(rng, C, F)
    db1, db2 = (torch.from_numpy(v).to("cuda", torch.float16) for v in (b1, b2))
    x, h, g, sc, sh = (torch.empty(n, C, device="cuda", dtype=torch.float16) for n in (rows, rows, groups, groups, groups))
    w = torch.empty(C, device="cuda")
    out, z = (torch.empty(rows, C, device="cuda", dtype=torch.float16) for _ in range(2))
    a, u = t.mx4_space(rows, C), t.mx4_space(rows, F)

    def run(s):
        for d, v in zip((x, h, g, sc, sh), s[:5]):
            d.copy_(torch.from_numpy(v))
        w.copy_(torch.from_numpy(s[5][1]))
        torch.cuda.synchronize()
        vb.block_norm(dt, rows, C, x, C, h=h, ldh=C, gate=g, ldgate=C, out=out, ldo=C, pre=1, pre_w=w, scale=sc, shift=sh, ldmod=C,
                      rows_per_group=group, y_codes=a[0], ldc=a[0].stride(0), y_scales=a[1])
        vb.gemm_mx4_quant(dt, a[0], a[0].stride(0), a[1], W1[0], W1[0].stride(0), W1[1], db1, u[0], u[0].stride(0), u[1], rows, F, C, 1)
        vb.gemm_mx4(dt, u[0], u[0].stride(0), u[1], W2[0], W2[0].stride(0), W2[1], db2, z, C, out, C, rows, C, F, 2)
        vb.check_device()
        return [t.get(v).copy() for v in (out, a[0], a[1], u[0], u[1], z)]

    first = run(sets[0])
    for _ in range(6):
        run(sets[1])
        for p, q in zip(first, run(sets[0])):
            assert np.array_equal(p, q)
    s, held = sets[0], first[0].astype(np.float64)
    t.norm_check(held, None, s[0], s[1], 0, None, None, s[2][at], 1.0, 0, None, None, None, None, dt)
    part = slice(rows - 2500 if rows > 2500 else 0, rows)  # (64-bit products of the last rows only)
    part = slice(part.start // 128 * 128, rows)
    y, _ = ref.norm(held[part], 1, s[5][1], None, 1e-5)
    n, size = ref.norm(held[part], 1, None, None, 1e-5)
    y, one = y * (1 + s[3][at][part]) + s[4][at][part], 1 + np.abs(s[3][at][part])
    e = t.norm_tol(None, n, size, s[5][1], None, dt) * one + 2.0 ** -21 * (np.abs(y) + np.abs(s[4][at][part]))
    m = rows - part.start

    def tail(space, k):
        return space[0][part], space[1][part.start // 128 * (-(-k // 128)) * 512:]

    t.blocks_check(tail(a, C), m, C, y, e)
    y, err = t.product_exact(t.held(tail(a, C), m, C), W1[2], b1, None, 1, False)
    t.blocks_check(tail(u, F), m, F, y, err)
    t.product_check(first[5][part].astype(np.float64), t.held(tail(u, F), m, F), W2[2], b2, held[part], dt, 2)
