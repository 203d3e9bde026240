"""Edges of the 4-bit product and the block norm on the B200: GELU's tails on every tile, Inf,
groups without a modulation, what is past the last column,
narrow rows.

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


# ------------------------------------------------------------------ NaN and Inf

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
