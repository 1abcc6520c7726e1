"""8-bit rows at the ends of the number range, at the borders of the launch rules and in the forms that only the engine calls, against their definitions in
float64 (U = 2^-24, the rounding of fp32)."""
import math
import os
import subprocess
import sys

import pytest
import torch

from tests.test_gpu_rows8 import ROOT, U, _h16, _half_step, _make, _phi, _tiny, dev, ref_checkpoint, ref_row_codes          # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ int8 product: scales far from one
def _linear64(x, w, bias=None):
    q, sx = ref_row_codes(x)
    wq, sw = ref_row_codes(w)
    acc = (q.double() @ wq.double().t()) * sx.double()[:, None] * sw.double()[None, :]
    z = acc + (bias.double() if bias is not None else 0.0)
    return z, 4 * U * acc.abs() + U * z.abs() + 2.0 ** -149          # the sum, two products, one of them with the addition; the last may be subnormal


# one launch for few tokens, 64 x 64 tiles, 128 x 128, 192 x 192; whole tiles and ragged ones
SHAPES = [(3, 3000, 48), (40, 3000, 48), (64, 4096, 128), (2560, 3000, 1280), (3264, 3000, 2304), (2500, 3000, 1201)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_a_scale_product_below_the_range(dev, M, K, N):
    """x w of ~1e-41 summed 3000 times: ordinary numbers of ~3e-38, while the product of the two scales has two bits at most"""
    from climb_amd import rows8
    g = torch.Generator().manual_seed(M)
    x, w = (1 + torch.rand(M, K, generator=g)) * 3e-21, (1 + torch.rand(N, K, generator=g)) * 2e-21
    z, tol = _linear64(x, w)
    assert float(ref_row_codes(x)[1].double().max() * ref_row_codes(w)[1].double().max()) < 2.0 ** -147 and float(z.min()) > 2.0 ** -126
    y = rows8.linear_i8(x.cuda(), rows8.quantize_rows(w.cuda())).cpu().double()
    assert ((y - z).abs() <= tol).all()


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_scales_at_the_top_of_the_range(dev, M, K, N):
    """a few tokens of 1e35 (a scale beyond 2^96) times channels of 1e-30: finite; times channels of 1e10: infinite, but a sum of 0 stays 0; the other tokens keep
    their bits"""
    from climb_amd import rows8
    g = torch.Generator().manual_seed(M + 1)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * 1e-30
    bias = torch.randn(N, generator=g)
    w[0] = torch.rand(K, generator=g) * 1e10
    w[1, : K // 2 * 2] = 1e10          # (and the rest, if any, stays tiny: its codes are 0)
    clean = rows8.linear_i8(x.cuda(), rows8.quantize_rows(w.cuda()), bias.cuda())
    far = torch.tensor([0, M // 2, M - 1])
    x[far] = torch.randn(3, K, generator=g) * 1e35
    x[0] = 1e35
    x[0, 1::2] = -1e35
    x[0, K // 2 * 2:] = 0
    z, tol = _linear64(x, w, bias)
    assert float(ref_row_codes(x)[1].double()[far].min()) > 2.0 ** 96
    y = rows8.linear_i8(x.cuda(), rows8.quantize_rows(w.cuda()), bias.cuda())
    keep = torch.ones(M, dtype=torch.bool)
    keep[far] = False
    assert torch.equal(y[keep.cuda()], clean[keep.cuda()])
    y = y.cpu().double()
    over = z.abs() > 3.5e38
    assert over[M - 1, 0] and not over[:, 2:].any()
    assert (y[over] == torch.sign(z[over]) * math.inf).all() and ((y - z).abs()[~over] <= tol[~over]).all()
    assert y[0, 1] == bias[1]          # a sum of 0 under a scale product beyond fp32


# ------------------------------------------------------------------------------------------------ GELU in 16 bits
def test_gelu_of_every_16_bit_number(dev):
    """all 65536 arguments, through gelu_fwd and through the product's epilogue (tokens of zeros: the argument is the bias).  x q, q = Phi(-|x|) = 2^p: the fit of p gives q to
    2e-5 below 2, 9e-5 below 3 and 4e-4 beyond (half: 2.7e-5), Horner's roundings of p 8 U x^2 and the rest 20 U, as in test_gelu; 2^p ends at 2^-126, times |x| <= 14.5"""
    from climb_amd import rows8
    dt = _h16()
    u = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dt)
    x = u.double()
    ref = torch.where(x == -math.inf, torch.zeros_like(x), torch.where(x == math.inf, x, x * _phi(x)))
    z = x.abs().clamp(max=40.0)
    tail = z * _phi(-z)
    fit = torch.where(z < 2, 2e-5, torch.where(z < 3, 9e-5, 4e-4)) if dt is torch.bfloat16 else torch.full_like(z, 2.7e-5)
    tol = tail * (fit + U * (20 + 8 * z * z)) + U * ref.abs().nan_to_num(posinf=0.0) + _half_step(dt) * ref.abs().nan_to_num(posinf=0.0) + max(_tiny(dt), 2.0 ** -122)
    nan = torch.isnan(x)
    a, _ = rows8.gelu_fwd(u.cuda().view(256, 256))
    w8 = rows8.quantize_rows(torch.ones(65536, 16, device="cuda"))
    y = rows8.linear_i8(torch.zeros(9, 16, dtype=dt, device="cuda"), w8, u.float().cuda(), epi="gelu")
    few = rows8.linear_i8(torch.zeros(2, 16, dtype=dt, device="cuda"), w8, u.float().cuda(), epi="gelu")
    for got in (a.view(-1), y[0], y[8], few[1]):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), nan)
        ok = (got == ref) | ((got - ref).abs() <= tol) | nan
        assert ok.all(), (x[~ok][:5], got[~ok][:5], ref[~ok][:5])


# ------------------------------------------------------------------------------------------------ checkpoints at the top of the 16-bit type
@pytest.mark.parametrize("M,K,N", [(70, 130, 48), (7000, 768, 2304)])          # both kernels of the weight gradient
def test_the_largest_16_bit_activations_stay_finite(dev, M, K, N):
    """a finite activation next to the largest of its type reads back finite, in a load, as a recomputed activation and as an operand; beyond it, it is infinite"""
    from climb_amd import rows8
    dt = _h16()
    half = dt is torch.float16
    top = 65504.0 if half else torch.finfo(torch.bfloat16).max
    x = _make(M, K, dt, 5)[0]
    for r, f in ((3, 1.0), (4, -1.0), (5, 0.9985), (6, -0.994)):          # (of half: 65504, 65408, 65120)
        x[r, 7 * r] = f * top
    assert torch.isfinite(x).all()
    _, _, v = ref_checkpoint(x, half)
    if half:
        assert (v.abs() == 65536).any()
        v = torch.where(v.abs() == 65536, torch.sign(v) * top, v)
    ck = rows8.checkpoint_save(x.cuda())
    assert torch.equal(ck.load().cpu().double(), v)
    da = torch.ones(M, K, dtype=dt, device="cuda")
    du, a = rows8.gelu_bwd(da, ck, recompute=True)
    assert torch.isfinite(a).all() and torch.isfinite(du).all() and float(a[3, 21]) == float(v[3, 21])
    dy = _make(M, N, dt, 6)[0]
    dy[3:7] = (2.0 ** -13 if half else 2.0 ** -100)
    dw, _ = rows8.weight_grad(dy.cuda(), ck)
    ref, mag = dy.double().t() @ v, dy.double().abs().t() @ v.abs()
    assert ((dw.cpu().double() - ref).abs() <= 2 * (M + 16) * U * mag + 1e-30).all()
    if half:          # fp32 numbers beyond the type are what they were: infinite in 16 bits
        y = torch.full((2, 64), 66100.0, device="cuda")
        y[1] = -70000.0
        assert torch.isinf(rows8.checkpoint_save(y).load(dt)).all()


# ------------------------------------------------------------------------------------------------ weight gradient at the borders of its plan
# 256-tile kernel from 12 tiles of 64 tokens a range on (25 tiles: ten ranges, 27: nine, 36: seven); one token more than whole ranges leaves a last one of 193
@pytest.mark.parametrize("M,K,N", [(7616, 1280, 1280), (7617, 1280, 1280), (7680, 1280, 1280), (7681, 1280, 1280), (6848, 768, 2304), (6912, 768, 2304), (6913, 768, 2304), (5377, 1281, 1288)])
def test_weight_gradient_ranges(dev, M, K, N):
    from climb_amd import rows8
    x, d = _make(M, K, _h16(), M + K)
    dy, dd = _make(M, N, _h16(), M + N + 1)
    v = ref_checkpoint(x, _h16() is torch.float16)[2].cuda()
    dw, db = rows8.weight_grad(dd, rows8.checkpoint_save(d))
    g = dd.double().t().contiguous()
    ref, mag = g @ v, g.abs() @ v.abs()
    assert ((dw.double() - ref).abs() <= 2 * (M + 16) * U * mag + 1e-30).all()          # exact products, at most M + 16 additions (twice: MFMA sums may truncate)
    assert ((db.double() - g.sum(1)).abs() <= (M + 16) * U * g.abs().sum(1) + 1e-30).all()
    # the sum over whole ranges alone cannot hide a token: one gradient row at a time
    for t in (0, M - 1, M // 2):
        one = torch.zeros_like(dd)
        one[t] = dd[t]
        w1, b1 = rows8.weight_grad(one, rows8.checkpoint_save(d))
        want = one[t].double()[:, None] * v[t][None]
        assert ((w1.double() - want).abs() <= U * want.abs()).all() and torch.equal(b1, dd[t].float())


# ------------------------------------------------------------------------------------------------ LayerNorm backward as the engine calls it
def _layernorm_bwd(M, C, dt, seed, colsum, beta, gamma_off=0):
    """climb_act8_layernorm_bwd in place (dx over dres_in) with a 16-bit copy of dx and, if asked for, its column sums"""
    from climb_amd import _lib, rows8
    g = torch.Generator().manual_seed(seed)
    x, dy, res = torch.randn(M, C, generator=g).cuda(), torch.randn(M, C, generator=g).to(dt).cuda(), torch.randn(M, C, generator=g).cuda()
    gamma = torch.empty(C + gamma_off, device="cuda")[gamma_off:]          # (an offset of one float: the unaligned path)
    gamma.copy_(1 + 0.1 * torch.randn(C, generator=g))
    _, ck = rows8.layernorm_fwd(x, gamma, gamma, 1e-5)
    v, mu, rs = ck.load(torch.float32).double(), ck.mean.double()[:, None], ck.rstd.double()[:, None]
    sums = [torch.full((C,), float(i + 2), device="cuda") for i in range(3)]
    dx, cast = res.clone(), torch.empty(M, C, dtype=dt, device="cuda")
    n = _lib.query_arg("climb_act8_layernorm_bwd_workspace", M, C, 1 if colsum else 0)
    part = torch.full((max(n // 4, 1),), float("nan"), device="cuda")
    code = 0 if dt is torch.float32 else 1
    _lib.call("climb_act8_layernorm_bwd", dy, C, code, *ck._args(), ck.mean, ck.rstd, gamma, dx, C, dx, C, cast, C, part if n else None, sums[0], sums[1], sums[2] if colsum else None,
              beta, M, C, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    d, ga = dy.double(), gamma.double()
    xh, G = (v - mu) * rs, d * ga
    want = res.double() + rs * (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True))
    wide = (v.abs() + mu.abs()) * rs
    mag = res.double().abs() + rs * (G.abs() + G.abs().mean(1, keepdim=True) + wide * (G.abs() * wide).mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= 96 * U * mag + 1e-30).all()          # (as in test_layernorm: ~30 additions on a path, twice, and a handful)
    assert torch.equal(cast, dx.to(dt))
    # column sums: at most M + 96 additions on a path (dx itself errs by 96 U of its terms), one fma with the old value
    for i, (terms, size) in enumerate(((d * xh, d.abs() * wide), (d, d.abs()), (want, mag))[:3 if colsum else 2]):
        old = beta * (i + 2)
        assert ((sums[i].double() - old - terms.sum(0)).abs() <= (M + 200) * U * size.sum(0) + 4 * U * abs(old) + 1e-30).all(), i
    if not colsum:
        assert (sums[2] == 4).all()          # not asked for, not touched
    return dx, sums


# three rows a wave from 8192 on (24 a workgroup), one below; one launch up to 768 rows without column sums; all widths a wave holds, ragged and whole
@pytest.mark.parametrize("M,C", [(8191, 70), (8192, 768), (8209, 129), (12301, 768), (8200, 1536), (8215, 3), (8193, 257), (769, 768), (768, 768), (5, 1535), (1, 1)])
@pytest.mark.parametrize("name", ["f32", "h16"])
def test_layernorm_backward_in_place_with_a_copy_and_column_sums(dev, M, C, name):
    dt = torch.float32 if name == "f32" else _h16()
    for colsum in (True, False):
        a = _layernorm_bwd(M, C, dt, M + C, colsum, 1.0)
        b = _layernorm_bwd(M, C, dt, M + C, colsum, 1.0)
        assert torch.equal(a[0], b[0]) and all(torch.equal(s, t) for s, t in zip(a[1], b[1]))          # no atomics: the same bits
        _layernorm_bwd(M, C, dt, M + C, colsum, 0.0, gamma_off=1)


@pytest.mark.skipif(os.environ.get("CLIMB_AMD_H16") == "fp16", reason="this is the child run")
def test_the_half_build(dev):
    """this file on the library build whose 16-bit type is IEEE half (a process holds one of them)"""
    env = dict(os.environ, CLIMB_AMD_H16="fp16", CLIMB_AMD_BACKGROUND_CHILD="1")
    env.pop("CLIMB_AMD_LIB", None)
    r = subprocess.run([sys.executable, "-m", "pytest", "tests/test_gpu_rows8_edges.py", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"], cwd=ROOT, env=env, capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
