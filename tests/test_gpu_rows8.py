"""8-bit rows on the MI355X against their definitions in float64.  Codes and scales have to be EQUAL to the definition's; computed results are held to bounds
counted in roundings (U = 2^-24, the rounding of fp32; EPS16 = half a step of the 16-bit type), written beside each check."""
import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def _h16():
    from climb_amd import _lib
    return _lib.torch_h16()


def _dt(name):
    return torch.float32 if name == "f32" else _h16()


def _half_step(dt):
    return torch.finfo(dt).eps / 2 if dt is not torch.float32 else U


def _tiny(dt):          # absolute half step at the bottom of the type's range (fp16 stores subnormals)
    return 2.0 ** -25 if dt is torch.float16 else 1e-38


def _make(M, C, dt, seed, layout="plain"):
    """[M, C] on the CPU (values of `dt`, a few columns 20 times the rest) and the same values on the GPU in the given layout"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, C, generator=g)
    x[:, ::97] *= 20.0
    x = x.to(dt)
    if layout == "plain":
        d = x.cuda()
    elif layout == "wide":          # rows of a wider, aligned matrix
        d = torch.full((M, C + 24), 777.0, dtype=dt, device="cuda")[:, 8:8 + C]
        d.copy_(x)
    elif layout == "odd":           # odd row stride and a base that is aligned to its element only
        d = torch.full((M, C + 3), 777.0, dtype=dt, device="cuda")[:, 1:1 + C]
        d.copy_(x)
    else:                           # column-strided: the calls copy it
        d = x.cuda().t().contiguous().t()
    return x, d


def ref_row_codes(x):
    x = x.double()
    amax = x.abs().amax(1)
    bad = ~torch.isfinite(amax)
    s = (amax / 127).float().clamp(min=2.0 ** -126)
    q = torch.round(x / s.double()[:, None])
    q[bad] = 0
    s[bad] = float("nan")
    return q.to(torch.int8), s


def ref_checkpoint(x, half):
    """(codes, exponent bytes, values) of the definition, group by group"""
    x = x.double()
    M, C = x.shape
    q, es, v = torch.zeros(M, C, dtype=torch.int8), [], torch.zeros(M, C, dtype=torch.float64)
    emin = -24 if half else -126
    for c in range(0, C, 64):
        p = x[:, c:c + 64]
        top = p.abs().amax(1)
        bad = ~torch.isfinite(top)
        t = torch.where(bad, torch.ones_like(top), top)
        e = torch.full((M,), float(emin), dtype=torch.float64)
        k = torch.ceil(torch.log2(t.clamp(min=1e-300) / 127)).clamp(min=emin)
        for cand in (k - 1, k, k + 1):          # the smallest that satisfies the definition, whatever log2 rounded to
            cand = cand.clamp(min=emin)
            okc = 127 * torch.exp2(cand) >= t
            e = torch.where(okc & (~(127 * torch.exp2(e) >= t) | (cand < e)), cand, e)
        assert (127 * torch.exp2(e) >= t).all()
        code = torch.round(p * torch.exp2(-e)[:, None])
        code[e == 122] = code[e == 122].clamp(-63, 63)          # 64 * 2^122 is beyond fp32
        code[bad] = 0
        val = code * torch.exp2(e)[:, None]
        val[bad] = float("nan")
        q[:, c:c + 64] = code.to(torch.int8)
        v[:, c:c + 64] = val
        eb = (e + 127).to(torch.uint8)
        eb[bad] = 255
        es.append(eb)
    return q, torch.stack(es, 1), v


def _awkward(M, C, dt, seed):
    """rows of zeros, of one value, of the type's largest and smallest numbers, of exact halves, with NaN and infinities"""
    x = _make(M, C, dt, seed)[0]
    big = torch.finfo(dt).max
    x[0] = 0
    x[1] = 1.0
    x[2, 0] = big
    x[3] = torch.finfo(dt).smallest_normal
    x[4] = 2.0 ** -133 if dt is not torch.float16 else 2.0 ** -24
    x[5] = torch.arange(C).to(dt) % 2 + 0.5          # halves of the step for scale 1: ties
    x[5, 0] = 127.0
    x[6, C // 2] = float("nan")
    x[7, C - 1] = float("inf")
    x[8, 0] = -float("inf")
    x[9] = 3.0
    x[9, :: 2] = 1.5                                  # x = amax / 2: quotient next to 63.5
    return x


SIZES = [(1, 1), (3, 17), (5, 64), (2, 65), (33, 127), (4, 128), (7, 129), (10, 300), (13, 768), (6, 1000), (9, 1536), (5, 2000), (3, 3100), (2, 5001)]


# ------------------------------------------------------------------------------------------------ formats
@pytest.mark.parametrize("name", ["f32", "h16"])
@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("layout", ["plain", "wide", "odd", "columns"])
def test_row_codes_equal_the_definition(dev, M, C, name, layout):
    from climb_amd import rows8
    x, d = _make(M, C, _dt(name), 3 * M + C, layout)
    q, s = ref_row_codes(x)
    r = rows8.quantize_rows(d)
    assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q[:, :C].cpu(), q)
    assert not r.q[:, C:].any()


@pytest.mark.parametrize("name", ["f32", "h16"])
@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("layout", ["plain", "wide", "odd", "columns"])
def test_checkpoints_equal_the_definition(dev, M, C, name, layout):
    from climb_amd import rows8
    dt = _dt(name)
    x, d = _make(M, C, dt, 5 * M + C, layout)
    q, e, v = ref_checkpoint(x, _h16() is torch.float16)
    ck = rows8.checkpoint_save(d)
    assert torch.equal(ck.exps.cpu(), e) and torch.equal(ck.q[:, :C].cpu(), q)
    assert torch.equal(ck.load(torch.float32).cpu().double(), v)
    assert torch.equal(ck.load(_h16()).cpu().double(), v)          # a code times its step is a number of the 16-bit type


@pytest.mark.parametrize("name", ["f32", "h16"])
@pytest.mark.parametrize("C", [70, 256, 768, 3333])
def test_awkward_rows(dev, name, C):
    from climb_amd import rows8
    x = _awkward(12, C, _dt(name), C)
    q, s = ref_row_codes(x)
    r = rows8.quantize_rows(x.cuda())
    assert torch.equal(r.scale.cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0)) and torch.equal(r.q[:, :C].cpu(), q)
    half = _h16() is torch.float16
    if half and name == "f32":
        x[2, 0] = 60000.0           # beyond IEEE half a 16-bit load of the checkpoint is infinite; the codes are checked all the same
    q, e, v = ref_checkpoint(x, half)
    ck = rows8.checkpoint_save(x.cuda())
    assert torch.equal(ck.exps.cpu(), e) and torch.equal(ck.q[:, :C].cpu(), q)
    assert torch.equal(torch.isnan(ck.load(torch.float32)).cpu(), torch.isnan(v))
    assert torch.equal(ck.load(torch.float32).cpu().double().nan_to_num(nan=-1.0), v.nan_to_num(nan=-1.0))


# ------------------------------------------------------------------------------------------------ int8 linear layer
def _phi(x):
    return torch.special.erfc(-x / math.sqrt(2.0)) / 2


def _gelu_tol(x, h16):
    """x q, q = Phi(-|x|).  fp32: a rational argument and a polynomial (relative error 1.5e-7), ~16 roundings, an exponential whose argument x^2 / 2 is rounded
    three times.  16 bits: 2^p with p a polynomial of degree 8 (fitted to 1.66e-5); Horner's roundings of p are below 2 U sum |c_k| |x|^k, and that sum is
    below 5.8 x^2 for 1 <= |x| <= 10 (34 at 5, 400 at 10), times ln 2: 8 U x^2."""
    tail = (x * _phi(-x.abs())).abs()
    return tail * ((1.7e-5 if h16 else 1.5e-7) + U * (20 + (8 if h16 else 3) * x * x)) + 2 * U * x.abs()


def _check_linear(x, w, bias, resid, epi, out_dt, y, s=None):
    q, sx = ref_row_codes(x)
    wq, sw = ref_row_codes(w)
    acc = (q.double() @ wq.double().t()) * sx.double()[:, None] * sw.double()[None, :]
    z = acc + (bias.double() if bias is not None else 0.0)
    tol = 4 * U * acc.abs() + 2 * U * z.abs()          # the int32 sum to fp32, two scale products, one fma
    if epi == "gelu":
        tol = 1.13 * tol + _gelu_tol(z, out_dt is not torch.float32)          # |gelu'| <= 1.13
        z = z * _phi(z)
    elif epi == "resid":
        z = z + resid.double()
        tol = tol + U * z.abs()
    tol = tol * 1.01 + _half_step(out_dt) * z.abs() + _tiny(out_dt)
    got = y.cpu().double()
    assert got.shape == z.shape
    worst = ((got - z).abs() / tol).max().item()
    assert worst <= 1.0, worst


LINEAR = [(1, 768, 768), (7, 5000, 33), (33, 1500, 50), (49, 3200, 17), (64, 4, 5), (12288, 200, 192), (1, 16, 17), (2, 100, 33), (15, 768, 96), (16, 2000, 40), (17, 129, 65), (40, 128, 128), (64, 1536, 3129), (185, 768, 768), (200, 77, 130),
          (333, 640, 1001), (1000, 256, 1100), (2500, 384, 1200)]


@pytest.mark.parametrize("M,K,N", LINEAR)
@pytest.mark.parametrize("xn,yn,epi", [("h16", "h16", "none"), ("f32", "f32", "none"), ("h16", "h16", "gelu"), ("f32", "f32", "gelu"), ("h16", "f32", "resid"), ("f32", "h16", "none")])
def test_linear(dev, M, K, N, xn, yn, epi):
    from climb_amd import rows8
    x, d = _make(M, K, _dt(xn), M + K, "odd" if N % 2 else "plain")
    g = torch.Generator().manual_seed(N)
    w = torch.randn(N, K, generator=g) * 0.05
    bias = torch.randn(N, generator=g)
    resid = torch.randn(M, N, generator=g) if epi == "resid" else None
    y = rows8.linear_i8(d, rows8.quantize_rows(w.cuda()), bias.cuda(), epi=epi, resid=resid.cuda() if resid is not None else None, out_dtype=_dt(yn))
    assert y.dtype is _dt(yn)
    _check_linear(x, w, bias, resid, epi, _dt(yn), y)


# every tile size of the product, whole and ragged: 256 tiles of 192 x 192 in one round; more of them with a long reduction; 128 x 128; 64 x 64
@pytest.mark.parametrize("M,K,N", [(12288, 130, 768), (12101, 256, 581), (10000, 1600, 800), (10000, 200, 800), (1000, 260, 777)])
@pytest.mark.parametrize("epi", ["none", "gelu", "resid"])
def test_linear_tiles(dev, M, K, N, epi):
    from climb_amd import rows8
    g = torch.Generator().manual_seed(M + K)
    x, w, bias = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * 0.05, torch.randn(N + 1, generator=g)[1:]
    resid = torch.randn(M, N, generator=g) if epi == "resid" else None
    out_dtype = torch.float32 if epi == "resid" else _h16()
    b = torch.zeros(N + 1, device="cuda")[1:]          # (a base that is aligned to its element only)
    b.copy_(bias)
    y = rows8.linear_i8(x.cuda(), rows8.quantize_rows(w.cuda()), b, epi=epi, resid=resid.cuda() if resid is not None else None, out_dtype=out_dtype)
    _check_linear(x, w, bias, resid, epi, out_dtype, y)


def test_linear_leading_dims_codes_out_and_residual_in_place(dev):
    from climb_amd import rows8
    x, d = _make(6 * 7, 96, torch.float32, 1)
    w = torch.randn(50, 96, generator=torch.Generator().manual_seed(2))
    w8 = rows8.quantize_rows(w.cuda())
    d3 = d.view(6, 7, 96)
    y = rows8.linear_i8(d3, w8)
    assert y.shape == (6, 7, 50)
    _check_linear(x, w, None, None, "none", torch.float32, y.view(42, 50))
    codes = rows8.quantize_rows(d3)
    assert torch.equal(rows8.linear_i8(codes, w8), y)                       # shared codes: the same bits ...
    assert torch.equal(rows8.linear_i8(d[:8], w8), y.view(42, 50)[:8])      # ... and few tokens in their one launch
    wide = torch.full((42, 60), 5.0, device="cuda")
    res = torch.randn(42, 50, generator=torch.Generator().manual_seed(3))
    wide[:, 4:54] = res.cuda()
    out = rows8.linear_i8(d, w8, epi="resid", resid=wide[:, 4:54], out=wide[:, 4:54])
    _check_linear(x, w, None, res, "resid", torch.float32, out)
    assert (wide[:, :4] == 5).all() and (wide[:, 54:] == 5).all()           # columns beside the result stay as they were


def test_linear_rows_with_nan_and_no_rows(dev):
    from climb_amd import rows8
    x, d = _make(40, 200, torch.float32, 4)
    w8 = rows8.quantize_rows(torch.randn(30, 200, generator=torch.Generator().manual_seed(5)).cuda())
    clean = rows8.linear_i8(d, w8)
    d[3, 7], d[9, 0], d[20] = float("nan"), float("inf"), 0.0
    y = rows8.linear_i8(d, w8)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 9]] = True
    assert torch.isnan(y[bad]).all() and (y[20] == 0).all()
    keep = ~bad
    keep[20] = False
    assert torch.equal(y[keep], clean[keep])
    assert rows8.linear_i8(d[:0], w8).shape == (0, 30)


def test_tensor_call_refusals_on_the_gpu(dev):
    from climb_amd import rows8
    x = torch.zeros(4, 8, device="cuda")
    w8 = rows8.quantize_rows(torch.zeros(3, 8, device="cuda"))
    for bad, exc in ((lambda: rows8.linear_i8(x[:, :7], w8), ValueError), (lambda: rows8.linear_i8(x.cpu(), w8), ValueError), (lambda: rows8.linear_i8(x.double(), w8), TypeError),
                     (lambda: rows8.linear_i8(x, w8, bias=torch.zeros(4, device="cuda")), ValueError), (lambda: rows8.linear_i8(x, w8, out=torch.zeros(4, 4, device="cuda")), ValueError),
                     (lambda: rows8.linear_i8(x, w8, epi="resid", resid=torch.zeros(5, 3, device="cuda")), ValueError), (lambda: rows8.linear_i8(x, w8, out_dtype=torch.float64), TypeError),
                     (lambda: rows8.layernorm_fwd(torch.zeros(2, 1600, device="cuda"), torch.ones(1600, device="cuda"), torch.ones(1600, device="cuda"), 1e-5), ValueError),
                     (lambda: rows8.weight_grad(torch.zeros(5, 3, dtype=_h16(), device="cuda"), rows8.checkpoint_save(x)), ValueError),
                     (lambda: rows8.weight_grad(torch.zeros(4, 3, device="cuda"), rows8.checkpoint_save(x)), TypeError),
                     (lambda: rows8.gelu_bwd(torch.zeros(4, 9, device="cuda"), rows8.checkpoint_save(x)), ValueError)):
        with pytest.raises(exc):
            bad()


# ------------------------------------------------------------------------------------------------ weight gradient
WGRAD = [(1, 1, 1), (1, 768, 40), (3, 17, 130), (63, 64, 64), (64, 1536, 3129), (65, 129, 127), (185, 768, 768), (511, 100, 200), (512, 33, 77), (700, 384, 260), (3000, 200, 90),
         (12288, 130, 140), (8195, 1000, 1288), (4097, 768, 2304), (12290, 1536, 768), (4609, 768, 2304), (12290, 1536, 1024)]


@pytest.mark.parametrize("M,K,N", WGRAD)
def test_weight_gradient(dev, M, K, N):
    from climb_amd import rows8
    x, d = _make(M, K, torch.float32, M + K, "odd" if K % 2 else "wide")
    dy, dd = _make(M, N, _h16(), M + N + 1, "odd" if N % 2 else "plain")
    _, _, v = ref_checkpoint(x, _h16() is torch.float16)
    dw, db = rows8.weight_grad(dd, rows8.checkpoint_save(d))
    ref, mag = dy.double().t() @ v, dy.double().abs().t() @ v.abs()
    tol = 2 * (M + 16) * U * mag + 1e-30          # exact products, at most M + 16 additions on a path (twice: MFMA sums may truncate)
    assert ((dw.cpu().double() - ref).abs() <= tol).all(), ((dw.cpu().double() - ref).abs() / tol).max()
    tol = (M + 16) * U * dy.double().abs().sum(0) + 1e-30
    assert ((db.cpu().double() - dy.double().sum(0)).abs() <= tol).all()
    again = rows8.weight_grad(dd, rows8.checkpoint_save(d))
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)          # no atomics: the same bits


@pytest.mark.parametrize("M", [0, 30, 2000])
def test_weight_gradient_accumulates_into_strided_targets(dev, M):
    from climb_amd import rows8
    K, N = 70, 90
    _, d = _make(M, K, _h16(), 1)
    _, dd = _make(M, N, _h16(), 2)
    ck = rows8.checkpoint_save(d)
    dw, db = rows8.weight_grad(dd, ck)
    wide = torch.full((N, K + 5), 2.0, device="cuda")
    b = torch.full((N,), 3.0, device="cuda")
    got, gb = rows8.weight_grad(dd, ck, dw=wide[:, 2:2 + K], dbias=b)
    assert got.data_ptr() == wide[:, 2:].data_ptr() and gb is b
    assert ((wide[:, 2:2 + K] - (dw + 2.0)).abs() <= 2 * U * (dw.abs() + 2)).all() and ((b - (db + 3.0)).abs() <= 2 * U * (db.abs() + 3)).all()
    assert (wide[:, :2] == 2).all() and (wide[:, 2 + K:] == 2).all()
    only, none = rows8.weight_grad(dd, ck, bias=False)
    assert torch.equal(only, dw) and none is None
    if M == 0:
        assert not dw.any() and not db.any()


def test_weight_gradient_keeps_nan_in_its_columns(dev):
    """a NaN in a group makes that group's 64 columns NaN and no others; gradient rows of zeros stay apart from a neighbour's NaN"""
    from climb_amd import rows8
    x, d = _make(100, 200, torch.float32, 9)
    _, dd = _make(100, 50, _h16(), 10)
    d[5, 70] = float("nan")
    dw, db = rows8.weight_grad(dd, rows8.checkpoint_save(d))
    nan = torch.isnan(dw).any(0)
    assert nan[64:128].all() and not nan[:64].any() and not nan[128:].any() and not torch.isnan(db).any()


@pytest.mark.parametrize("M,K,N", [(100, 200, 50), (4609, 768, 2304), (7000, 768, 2304)])
def test_weight_gradient_of_the_largest_numbers(dev, M, K, N):
    """groups whose step is 2^121 or 2^122 (fp32 numbers next to the top of the range): 128 steps are beyond fp32, the values are not"""
    from climb_amd import rows8
    x, _ = _make(M, K, torch.float32, 20)
    x[5, 3], x[7, 3], x[9, 70], x[M - 1, K - 1] = 3.3e38, -1.6e38, -3.4e38, 2.0e38
    x[11] = torch.linspace(-1.0, 1.0, K) * 3e38
    dy = _make(M, N, _h16(), 21)[0]
    dy[[5, 7, 9, 11, M - 1]] = 2.0 ** -14
    _, _, v = ref_checkpoint(x, _h16() is torch.float16)
    dw, _ = rows8.weight_grad(dy.cuda(), rows8.checkpoint_save(x.cuda()))
    if _h16() is torch.float16:          # (numbers beyond 65504 are infinite operands: zero codes stay zeros, columns without such a number stay finite)
        v = torch.where(v.abs() > 65504, torch.sign(v) * math.inf, v)
        finite = torch.isfinite(v).all(0)
        assert torch.isfinite(dw.cpu()[:, finite]).all() and not torch.isfinite(dw.cpu()[:, ~finite]).any()
        return
    ref, mag = dy.double().t() @ v, dy.double().abs().t() @ v.abs()
    assert ((dw.cpu().double() - ref).abs() <= 2 * (M + 16) * U * mag + 1e-30).all()


# ------------------------------------------------------------------------------------------------ LayerNorm and GELU
LN = [(1, 1), (1, 5), (3, 64), (4, 70), (25, 129), (185, 768), (50, 767), (23, 770), (333, 1536), (24, 1535), (1000, 100)]


@pytest.mark.parametrize("M,C", LN)
@pytest.mark.parametrize("name", ["f32", "h16"])
@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_layernorm(dev, M, C, name, layout):
    from climb_amd import rows8
    dt = _dt(name)
    x, d = _make(M, C, torch.float32, M + C, layout)
    dy, dd = _make(M, C, dt, M + C + 1, layout)
    res, dres = _make(M, C, torch.float32, M + C + 2, layout)
    g = torch.Generator().manual_seed(C)
    gamma, beta = 1 + 0.1 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g)
    eps = 1e-5
    y, ck = rows8.layernorm_fwd(d, gamma.cuda(), beta.cuda(), eps, out_dtype=dt)
    dx, dg, db = rows8.layernorm_bwd(dd, ck, gamma.cuda(), dres=dres)
    x, dy, res, gamma, beta = x.double(), dy.double(), res.double(), gamma.double(), beta.double()
    mu = x.mean(1, keepdim=True)
    rs = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    ref = (x - mu) * rs * gamma + beta
    q, e, v = ref_checkpoint(x.float(), _h16() is torch.float16)
    assert torch.equal(ck.q[:, :C].cpu(), q) and torch.equal(ck.exps.cpu(), e)
    # the mean: at most 24 additions in a lane and 6 across, so 32 U of the largest |x|, times rs; 1 / sqrt(variance): half of as many; the rest a handful
    xm = x.abs().amax(1, keepdim=True)
    err = 48 * U * (((xm + mu.abs()) * rs + ((x - mu) * rs).abs()) * gamma.abs() + beta.abs())
    assert ((y.cpu().double() - ref).abs() <= err + _half_step(dt) * ref.abs() + _tiny(dt)).all()
    xh, G = (v - mu) * rs, dy * gamma
    want = res + rs * (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True))
    wide = ((v.abs() + xm) * rs)
    mag = res.abs() + rs * (G.abs() + G.abs().mean(1, keepdim=True) + wide * (G.abs() * wide).mean(1, keepdim=True))
    assert ((dx.cpu().double() - want).abs() <= 96 * U * mag + 1e-30).all()
    assert ((dg.cpu().double() - (dy * xh).sum(0)).abs() <= (M + 96) * U * (dy.abs() * wide).sum(0) + 1e-30).all()
    assert ((db.cpu().double() - dy.sum(0)).abs() <= (M + 16) * U * dy.abs().sum(0) + 1e-30).all()
    dx2, dg2, db2 = rows8.layernorm_bwd(dd, ck, gamma.float().cuda(), dgamma=torch.ones(C, device="cuda"))          # no residual, accumulating
    assert ((dg2 - 1 - dg).abs() <= 4 * U * (1 + dg.abs())).all() and torch.equal(db2, db)
    assert ((dx2.cpu().double() - (want - res)).abs() <= 96 * U * mag + 1e-30).all()


GELU = [(1, 1), (2, 7), (3, 64), (5, 65), (12, 200), (33, 1000), (185, 3100)]


@pytest.mark.parametrize("M,C", GELU)
@pytest.mark.parametrize("name", ["f32", "h16"])
@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_gelu(dev, M, C, name, layout):
    from climb_amd import rows8
    dt = _dt(name)
    u, d = _make(M, C, dt, M + C, layout)
    da, dd = _make(M, C, dt, M + C + 1, layout)
    a, ck = rows8.gelu_fwd(d)
    du, a2 = rows8.gelu_bwd(dd, ck, recompute=True)
    assert torch.equal(rows8.gelu_bwd(dd, ck), du)
    q, e, v = ref_checkpoint(u, _h16() is torch.float16)
    assert torch.equal(ck.q[:, :C].cpu(), q) and torch.equal(ck.exps.cpu(), e)
    deg6 = dt is not torch.float32
    for got, x in ((a, u.double()), (a2, v)):
        ref = x * _phi(x)
        assert ((got.cpu().double() - ref).abs() <= _gelu_tol(x, deg6) + _half_step(dt) * ref.abs() + _tiny(dt)).all()
    pdf = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    d1 = _phi(v) + v * pdf
    tol = _phi(-v.abs()) * ((8.3e-6 if deg6 else 1.5e-7) + U * (20 + 3 * v * v)) + (v * pdf).abs() * U * (8 + 3 * v * v) + 4 * U
    ref = da.double() * d1
    assert ((du.cpu().double() - ref).abs() <= da.double().abs() * tol + 2 * U * ref.abs() + _half_step(dt) * ref.abs() + _tiny(dt)).all()


def test_gelu_limits(dev):
    from climb_amd import rows8
    u = torch.tensor([[0.0, -0.0, 40.0, -40.0, 3e38, -3e38, float("inf"), -float("inf"), float("nan")]], device="cuda")
    a, _ = rows8.gelu_fwd(u)
    a = a[0].tolist()
    assert a[:8] == [0.0, 0.0, 40.0, 0.0, u[0, 4].item(), 0.0, float("inf"), 0.0] and math.isnan(a[8])


def test_gradients_against_differences(dev):
    """inputs that the checkpoint holds exactly (multiples of its step): the backward is then the derivative of the forward's formula, here by central
    differences of that formula in float64"""
    from climb_amd import rows8
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-127, 128, (3, 128), generator=g).float() / 32
    x[:, ::64] = 127 / 32
    dy = torch.randn(3, 128, generator=g)
    gamma, beta = 1 + 0.1 * torch.randn(128, generator=g), torch.randn(128, generator=g)

    def ln(t, ga, be):
        mu = t.mean(1, keepdim=True)
        return ((t - mu) / torch.sqrt(((t - mu) ** 2).mean(1, keepdim=True) + 1e-5)) * ga + be

    def diff(f, t, h=1e-5):
        out = torch.zeros_like(t)
        for i in range(t.numel()):
            p, m = t.clone(), t.clone()
            p.view(-1)[i] += h
            m.view(-1)[i] -= h
            out.view(-1)[i] = (f(p) - f(m)) / (2 * h)
        return out
    xd, dyd, gd, bd = x.double(), dy.double(), gamma.double(), beta.double()
    y, ck = rows8.layernorm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5)
    assert torch.equal(ck.load().cpu(), x)
    dx, dg, db = rows8.layernorm_bwd(dy.cuda(), ck, gamma.cuda())
    # the differences' own error: h^2 times a third derivative of order 10, and 1e-16 / h
    for got, want in ((dx, diff(lambda t: (ln(t, gd, bd) * dyd).sum(), xd)), (dg, diff(lambda t: (ln(xd, t, bd) * dyd).sum(), gd)), (db, diff(lambda t: (ln(xd, gd, t) * dyd).sum(), bd))):
        assert (got.cpu().double() - want).abs().max() < 1e-5
    a, ck = rows8.gelu_fwd(x.cuda())
    du = rows8.gelu_bwd(dy.cuda(), ck)
    assert (du.cpu().double() - diff(lambda t: (t * _phi(t) * dyd).sum(), xd)).abs().max() < 1e-5
    h = dy.to(_h16())
    w = torch.randn(128, 128, generator=g).double()
    dw, dbias = rows8.weight_grad(h.cuda(), rows8.checkpoint_save(x.cuda()))
    eye = torch.zeros(128, 128, dtype=torch.float64)
    for n, k in ((0, 0), (5, 77), (127, 127)):
        p = eye.clone()
        p[n, k] = 1e-3
        num = (((xd @ (w + p).t()) - (xd @ (w - p).t())) * h.double()).sum() / 2e-3
        assert abs(float(num) - float(dw[n, k])) < 1e-4
    assert (dw.cpu().double() - h.double().t() @ xd).abs().max() < 1e-4


def test_broadcast_gradients(dev):
    """a gradient that is a broadcast view (all rows, or all columns, one number in memory) gives what its copy gives"""
    from climb_amd import rows8
    M, C, N = 40, 96, 64
    _, x = _make(M, C, torch.float32, 1)
    g, b = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    _, ck = rows8.layernorm_fwd(x, g, b, 1e-5)
    _, uk = rows8.gelu_fwd(x)
    for view in (torch.randn(1, C, device="cuda").expand(M, C), torch.randn(M, 1, device="cuda").expand(M, C), torch.randn((), device="cuda").expand(M, C)):
        for got, want in zip(rows8.layernorm_bwd(view, ck, g, dres=view), rows8.layernorm_bwd(view.contiguous(), ck, g, dres=view.contiguous())):
            assert torch.equal(got, want)
        assert torch.equal(rows8.gelu_bwd(view, uk), rows8.gelu_bwd(view.contiguous(), uk))
    dy = torch.randn(1, N, device="cuda").to(_h16()).expand(M, N)
    for got, want in zip(rows8.weight_grad(dy, uk), rows8.weight_grad(dy.contiguous(), uk)):
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ as they are used together
def _block(rows8, x, p, dy):
    """x + W2 gelu(W1 LN(x) + b1) + b2, forward on the int8 product, backward from the checkpoints (the input gradients' products in fp32)"""
    y, lnck = rows8.layernorm_fwd(x, p["g"], p["b"], 1e-5, out_dtype=_h16())
    yck = rows8.checkpoint_save(y)
    u = rows8.linear_i8(y, p["w1q"], p["b1"])
    a, uck = rows8.gelu_fwd(u)
    out = rows8.linear_i8(a, p["w2q"], p["b2"], epi="resid", resid=x, out_dtype=torch.float32)
    d16 = dy.to(_h16())
    da = (d16.float() @ p["w2"]).to(_h16())
    du, a2 = rows8.gelu_bwd(da, uck, recompute=True)
    dw2, db2 = rows8.weight_grad(d16, rows8.checkpoint_save(a2))
    dw1, db1 = rows8.weight_grad(du, yck)
    dx, dg, db = rows8.layernorm_bwd((du.float() @ p["w1"]).to(_h16()), lnck, p["g"], dres=dy)
    return out, dw2, db2, dw1, db1, dx, dg, db


def _block_params(H, F, seed=0):
    g = torch.Generator().manual_seed(seed)
    p = dict(g=1 + 0.1 * torch.randn(H, generator=g), b=0.1 * torch.randn(H, generator=g), w1=torch.randn(F, H, generator=g) * H ** -0.5, b1=0.1 * torch.randn(F, generator=g),
             w2=torch.randn(H, F, generator=g) * F ** -0.5, b2=0.1 * torch.randn(H, generator=g))
    return {k: v.cuda() for k, v in p.items()}


@pytest.mark.parametrize("M,H,F", [(185, 96, 384), (37, 65, 130)])
def test_an_mlp_block_forward_and_backward(dev, M, H, F):
    """the operators together against float64 autograd of the same block without 8-bit steps: what is left is the quantisation itself.  Uniform rounding to
    steps of max / 127 (rows) and at most max / 63.5 (groups) of normal data, whose largest of H values is ~3 sigma: relative r.m.s. 3 / 127 / sqrt 12 =
    0.7 % an int8 operand, 1.4 % a checkpoint; a product adds its two operands', a gradient passes through up to four of them: 8 % bounds every result's
    relative error in the Frobenius norm, and a wrong scale, layout or formula is beyond it"""
    from climb_amd import rows8
    p = _block_params(H, F)
    p["w1q"], p["w2q"] = rows8.quantize_rows(p["w1"]), rows8.quantize_rows(p["w2"])
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(M, H, generator=g).cuda(), torch.randn(M, H, generator=g).cuda()
    got = _block(rows8, x, p, dy)
    r = {k: p[k].double().cpu().requires_grad_() for k in ("g", "b", "w1", "b1", "w2", "b2")}
    xr = x.double().cpu().requires_grad_()
    y = torch.nn.functional.layer_norm(xr, (H,), r["g"], r["b"], 1e-5)
    u = y @ r["w1"].t() + r["b1"]
    out = xr + (u * _phi(u)) @ r["w2"].t() + r["b2"]
    out.backward(dy.double().cpu())
    want = (out.detach(), r["w2"].grad, r["b2"].grad, r["w1"].grad, r["b1"].grad, xr.grad, r["g"].grad, r["b"].grad)
    for a, b in zip(got, want):
        assert float((a.cpu().double() - b).norm() / b.norm()) < 0.08


def test_captured_and_replayed_beside_eager_work(dev):
    """two graphs of the same calls, replayed in turn with eager calls of other sizes between them: each replay equals the eager result of its inputs"""
    from climb_amd import rows8
    p = _block_params(96, 384)
    p["w1q"], p["w2q"] = rows8.quantize_rows(p["w1"]), rows8.quantize_rows(p["w2"])
    g = torch.Generator().manual_seed(2)
    graphs = []
    for M in (700, 530):
        x, dy = torch.randn(M, 96, generator=g).cuda(), torch.randn(M, 96, generator=g).cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                _block(rows8, x, p, dy)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = _block(rows8, x, p, dy)
        graphs.append((gr, x, dy, outs))
    for rep in range(3):
        for gr, x, dy, outs in graphs:
            x.copy_(torch.randn(x.shape, generator=g).cuda())
            dy.copy_(torch.randn(dy.shape, generator=g).cuda())
            want = _block(rows8, x, p, dy)
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_large_products_captured_without_a_run_before(dev):
    """the kernels that ask for more than 64 KB of LDS, first called inside a capture; replayed three times beside eager work"""
    from climb_amd import rows8
    M, K, N = 12290, 768, 768
    x, dy = torch.randn(M, K, device="cuda"), torch.randn(M, 3 * N, device="cuda").to(_h16())
    w8, ck = rows8.quantize_rows(torch.randn(N, K, device="cuda")), rows8.checkpoint_save(x)
    codes = rows8.quantize_rows(x)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = rows8.linear_i8(codes, w8)
        dw, db = rows8.weight_grad(dy, ck)
    for rep in range(3):
        dy.copy_(torch.randn(M, 3 * N, device="cuda"))
        want = (rows8.linear_i8(codes, w8), *rows8.weight_grad(dy, ck))
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dw, db), want):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(dev):
    """matrices of more than 2^32 elements: the last rows come out as they do alone"""
    from climb_amd import rows8
    M, C, t = 5_600_000, 768, 40
    assert M * C > 2 ** 32
    tail = torch.randn(t, C, device="cuda")
    h = torch.zeros(M, C, dtype=_h16(), device="cuda")
    h[-t:] = tail.to(_h16())
    last = h[-t:].clone()
    codes, few = rows8.quantize_rows(h), rows8.quantize_rows(last)
    assert torch.equal(codes.q[-t:], few.q) and torch.equal(codes.scale[-t:], few.scale)
    w8 = rows8.quantize_rows(torch.randn(900, C, device="cuda"))
    y = rows8.linear_i8(codes, w8, epi="gelu", out_dtype=_h16())          # [M, 900]
    assert torch.equal(y[-t:], rows8.linear_i8(few, w8, epi="gelu", out_dtype=_h16()))
    del codes, y
    a, ck = rows8.gelu_fwd(h)
    a1, ck1 = rows8.gelu_fwd(last)
    assert torch.equal(a[-t:], a1) and torch.equal(ck.q[-t:], ck1.q) and torch.equal(ck.exps[-t:], ck1.exps)
    assert torch.equal(ck.load()[-t:], ck1.load())
    du, a2 = rows8.gelu_bwd(h, ck, recompute=True)
    du1, a3 = rows8.gelu_bwd(last, ck1, recompute=True)
    assert torch.equal(du[-t:], du1) and torch.equal(a2[-t:], a3)
    del a, du, a2
    for N in (64, 2304):          # both kernels of the weight gradient; rows of zeros add nothing
        d = torch.zeros(M, N, dtype=_h16(), device="cuda")
        d[-t:] = torch.randn(t, N, device="cuda").to(_h16())
        dw, db = rows8.weight_grad(d, ck)
        dw1, db1 = rows8.weight_grad(d[-t:], ck1)
        mag = d[-t:].float().abs().t() @ ck1.load(torch.float32).abs()
        assert ((dw - dw1).abs() <= 4 * (t + 16) * U * mag).all()          # two orders of at most t + 16 additions
        assert ((db - db1).abs() <= 4 * (t + 16) * U * d[-t:].float().abs().sum(0)).all()
        del d
    del h, ck
    x = torch.zeros(M, C, device="cuda")
    x[-t:] = tail
    g, b = torch.rand(C, device="cuda") + 0.5, torch.randn(C, device="cuda")
    y, ck = rows8.layernorm_fwd(x, g, b, 1e-5, out_dtype=_h16())
    y1, ck1 = rows8.layernorm_fwd(tail, g, b, 1e-5, out_dtype=_h16())
    assert torch.equal(y[-t:], y1) and torch.equal(ck.q[-t:], ck1.q) and torch.equal(ck.rstd[-t:], ck1.rstd)
    dx, _, _ = rows8.layernorm_bwd(y, ck, g, dres=x)
    assert torch.equal(dx[-t:], rows8.layernorm_bwd(y1, ck1, g, dres=tail)[0])


@pytest.mark.parametrize("lead", [(0,), (3, 0)])
def test_no_rows_at_all(dev, lead):
    from climb_amd import rows8
    C = 70
    x, h = torch.zeros(*lead, C, device="cuda"), torch.zeros(*lead, C, device="cuda", dtype=_h16())
    g = torch.ones(C, device="cuda")
    y, ck = rows8.layernorm_fwd(x, g, g, 1e-5)
    dx, dg, db = rows8.layernorm_bwd(x, ck, g, dres=x)
    acc = rows8.layernorm_bwd(x, ck, g, dgamma=torch.full((C,), 2.0, device="cuda"))[1]
    assert y.shape == dx.shape == x.shape and not dg.any() and not db.any() and (acc == 2).all() and ck.mean.shape == ck.rstd.shape == (0,)
    a, uk = rows8.gelu_fwd(h)
    du, a2 = rows8.gelu_bwd(h, uk, recompute=True)
    assert a.shape == du.shape == a2.shape == uk.load().shape == h.shape and a.dtype is _h16()
    w8 = rows8.quantize_rows(torch.ones(5, C, device="cuda"))
    assert rows8.linear_i8(h, w8).shape == (*lead, 5) and rows8.linear_i8(rows8.quantize_rows(h), w8).shape == (*lead, 5)


@pytest.mark.parametrize("M,C", [(1, 64), (30, 768), (767, 100), (768, 1536), (769, 1536), (200, 3)])
def test_layernorm_gradients_in_one_launch_and_in_two(dev, M, C):
    """column sums of dx wanted (two launches) or not (one, for few rows): the same dx, and dgamma, dbeta up to the order of their sums"""
    from climb_amd import _lib, rows8
    _, x = _make(M, C, torch.float32, M)
    _, dy = _make(M, C, torch.float32, M + 1)
    g = torch.rand(C, device="cuda") + 0.5
    _, ck = rows8.layernorm_fwd(x, g, g, 1e-5)
    dx, dg, db = rows8.layernorm_bwd(dy, ck, g, dgamma=torch.full((C,), 3.0, device="cuda"))
    dx2, dg2, db2, cs = torch.empty_like(x), torch.full((C,), 3.0, device="cuda"), torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    part = torch.empty(_lib.query_arg("climb_act8_layernorm_bwd_workspace", M, C, 1) // 4, device="cuda")
    assert part.numel() == _lib.query_arg("climb_act8_layernorm_bwd_blocks", M) * 3 * C
    _lib.call("climb_act8_layernorm_bwd", dy, C, 0, *ck._args(), ck.mean, ck.rstd, g, None, 0, dx2, C, None, 0, part, dg2, db2, cs, 1.0, M, C, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(dx, dx2)
    xh = (ck.load() - ck.mean[:, None]) * ck.rstd[:, None]
    for got, want, mag in ((dg, dg2, (dy * xh).abs().sum(0) + 3), (db, db2, dy.abs().sum(0)), (cs, dx.sum(0), dx.abs().sum(0))):
        assert ((got - want).abs() <= 2 * (M + 8) * U * mag + 1e-30).all()          # two orders of M additions
    again = rows8.layernorm_bwd(dy, ck, g, dgamma=torch.full((C,), 3.0, device="cuda"))
    assert torch.equal(again[1], dg) and torch.equal(again[2], db)


def test_rows_that_are_not_numbers_stay_in_their_rows(dev):
    """LayerNorm and GELU of rows with a NaN or an infinity: those rows' gradients are NaN where their groups are, the other rows' bits stay as they were"""
    from climb_amd import rows8
    M, C = 50, 200
    _, x = _make(M, C, torch.float32, 30)
    _, dy = _make(M, C, torch.float32, 31)
    g, b = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    clean_y, ck = rows8.layernorm_fwd(x, g, b, 1e-5)
    clean_dx = rows8.layernorm_bwd(dy, ck, g)[0]
    clean_du = rows8.gelu_bwd(dy, rows8.gelu_fwd(x)[1])
    x[3, 70], x[44, 199] = float("nan"), float("inf")
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[[3, 44]] = False
    y, ck = rows8.layernorm_fwd(x, g, b, 1e-5)
    dx, dg, _ = rows8.layernorm_bwd(dy, ck, g)
    for got, want in ((y, clean_y), (dx, clean_dx)):
        assert torch.equal(got[keep], want[keep]) and torch.isnan(got[~keep]).all()
    assert torch.isnan(dg).all()
    du = rows8.gelu_bwd(dy, rows8.gelu_fwd(x)[1])
    bad = torch.zeros(M, C, dtype=torch.bool, device="cuda")
    bad[3, 64:128] = bad[44, 192:] = True
    assert torch.isnan(du[bad]).all() and torch.equal(du[~bad], clean_du[~bad])


def test_two_streams_at_once(dev):
    from climb_amd import rows8
    work = []
    for i in range(2):
        _, d = _make(3000, 200, _h16(), i)
        _, dd = _make(3000, 260, _h16(), i + 5)
        ck = rows8.checkpoint_save(d)
        work.append((dd, ck, rows8.weight_grad(dd, ck)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    outs = [[] for _ in work]
    for _ in range(4):
        for s, (dd, ck, _), o in zip(streams, work, outs):
            with torch.cuda.stream(s):
                o.append(rows8.weight_grad(dd, ck))
    torch.cuda.synchronize()
    for (_, _, want), o in zip(work, outs):
        for got in o:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.skipif(os.environ.get("CLIMB_AMD_H16") == "fp16", reason="this is the child run")
def test_the_half_build(dev):
    """the same suite on the library build whose 16-bit type is IEEE half (a process holds one of them)"""
    env = dict(os.environ, CLIMB_AMD_H16="fp16", CLIMB_AMD_BACKGROUND_CHILD="1")
    env.pop("CLIMB_AMD_LIB", None)
    r = subprocess.run([sys.executable, "-m", "pytest", "tests/test_gpu_rows8.py", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"], cwd=ROOT, env=env, capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
