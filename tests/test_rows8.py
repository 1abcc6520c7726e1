"""8-bit rows, host side: what the C entry points and the tensor calls refuse (nothing here reaches a GPU)."""
import ctypes
import importlib.util
import os
import re

import pytest
import torch

from climb_amd import _lib, rows8

EINVAL, EUNSUPPORTED = -1, -2


def _rc(name, *args):
    return int(getattr(_lib.load(), name)(*args))


@pytest.fixture(scope="module")
def mem():
    """a host address that stands for a device buffer: every call below must return before it touches one"""
    buf = ctypes.create_string_buffer(4096)
    return (ctypes.addressof(buf) + 63) & ~63, buf


@pytest.mark.parametrize("change", [dict(M=-1), dict(C=0), dict(ldx=99), dict(ldq=100), dict(ldq=120), dict(dtype=2), dict(x=None), dict(q=None), dict(s=None), dict(qoff=1)])
def test_quantiser_refuses(mem, change):
    p = mem[0]
    a = dict(M=4, C=100, ldx=100, ldq=128, dtype=1, x=p, q=p, s=p, qoff=0)
    a.update(change)
    q = None if a["q"] is None else a["q"] + a["qoff"]
    assert _rc("climb_rows8_quant", a["x"], a["ldx"], a["dtype"], q, a["ldq"], a["s"], a["M"], a["C"], None) == EINVAL


@pytest.mark.parametrize("change,rc", [(dict(M=-1), EINVAL), (dict(N=0), EINVAL), (dict(K=0), EINVAL), (dict(lda=64), EINVAL), (dict(ldb=120), EINVAL), (dict(lda=136), EINVAL),
                                       (dict(ldc=31), EINVAL), (dict(epi=3), EINVAL), (dict(epi=2), EINVAL), (dict(epi=2, aux=1, ldaux=8), EINVAL), (dict(c_dtype=2), EINVAL),
                                       (dict(sa=None), EINVAL), (dict(A=None), EINVAL), (dict(C=None), EINVAL), (dict(aoff=8), EINVAL),
                                       (dict(K=(1 << 17) + 1, lda=1 << 18, ldb=1 << 18), EUNSUPPORTED), (dict(lda=1 << 22), EUNSUPPORTED)])
def test_int8_product_refuses(mem, change, rc):
    p = mem[0]
    a = dict(M=4, N=32, K=100, lda=128, ldb=128, ldc=32, epi=0, aux=None, ldaux=0, c_dtype=0, A=p, B=p, C=p, sa=p, sb=p, aoff=0)
    a.update(change)
    A = None if a["A"] is None else a["A"] + a["aoff"]
    aux = p if a["aux"] else None
    assert _rc("climb_gemm_i8_nt", A, a["lda"], a["sa"], a["B"], a["ldb"], a["sb"], a["C"], a["ldc"], a["c_dtype"], a["M"], a["N"], a["K"], None, a["epi"], aux, a["ldaux"],
               None) == rc
    # ... and so does the call that quantises its tokens (A as a 16-bit matrix), with few tokens and with many
    if "lda" in change and "K" not in change or "aoff" in change or "sa" in change:
        return
    for M in (a["M"], a["M"] * 100):
        assert _rc("climb_linear_i8", A, max(a["K"], 1), 1, a["B"], a["ldb"], a["sb"], a["C"], a["ldc"], a["c_dtype"], M, a["N"], a["K"], None, a["epi"], aux, a["ldaux"], p, 1 << 30,
                   None) == rc


def test_linear_asks_for_its_workspace(mem):
    p = mem[0]
    assert _rc("climb_linear_i8_workspace", 1, 768) == 0 and _rc("climb_linear_i8_workspace", 64, 100) == 64 * 132 and _rc("climb_linear_i8_workspace", -1, 8) == EINVAL
    need = 64 * 132
    for ws, nb in ((None, need), (p + 4, need), (p, need - 1)):
        assert _rc("climb_linear_i8", p, 100, 0, p, 128, p, p, 32, 0, 64, 32, 100, None, 0, None, 0, ws, nb, None) == EINVAL
    for dtype, ldx in ((2, 100), (0, 99)):
        assert _rc("climb_linear_i8", p, ldx, dtype, p, 128, p, p, 32, 0, 64, 32, 100, None, 0, None, 0, p, need, None) == EINVAL


@pytest.mark.parametrize("change", [dict(M=-1), dict(C=0), dict(ldq=96), dict(ldq=104), dict(lde=1), dict(dtype=2), dict(x=None), dict(q=None), dict(e=None), dict(ldx=99)])
def test_checkpoint_calls_refuse(mem, change):
    p = mem[0]
    a = dict(M=4, C=100, ldx=100, ldq=112, lde=2, dtype=0, x=p, q=p, e=p)
    a.update(change)
    ck = (a["q"], a["ldq"], a["e"], a["lde"])
    mc = (a["M"], a["C"], None)
    assert _rc("climb_act8_save", a["x"], a["ldx"], a["dtype"], *ck, *mc) == EINVAL
    assert _rc("climb_act8_load", *ck, a["x"], a["ldx"], a["dtype"], *mc) == EINVAL
    assert _rc("climb_act8_gelu_fwd", a["x"], a["ldx"], a["dtype"], p, 100, *ck, *mc) == EINVAL
    assert _rc("climb_act8_gelu_bwd", a["x"], a["ldx"], a["dtype"], *ck, p, 100, None, 0, *mc) == EINVAL
    assert _rc("climb_act8_layernorm_fwd", p, 100, p, p, 1e-5, a["x"], a["ldx"], a["dtype"], p, p, *ck, *mc) == EINVAL
    assert _rc("climb_act8_layernorm_bwd", a["x"], a["ldx"], a["dtype"], *ck, p, p, p, None, 0, p, 100, None, 0, p, p, p, None, 0.0, *mc) == EINVAL


def test_layernorm_refuses_rows_it_cannot_hold(mem):
    p = mem[0]
    assert _rc("climb_act8_layernorm_fwd", p, 1540, p, p, 1e-5, p, 1540, 0, p, p, p, 1552, p, 25, 4, 1540, None) == EUNSUPPORTED
    assert _rc("climb_act8_layernorm_bwd", p, 1540, 0, p, 1552, p, 25, p, p, p, None, 0, p, 1540, None, 0, p, p, p, None, 0.0, 4, 1540, None) == EUNSUPPORTED


def test_weight_gradient_refuses_and_asks_for_its_workspace(mem):
    p = mem[0]
    ok = dict(dY=p, lddy=96, q=p, ldq=112, e=p, lde=2, C=p, ldc=100, M=4096, N=96, K=100, ws=p)
    need = _rc("climb_act8_weight_grad_workspace", 4096, 96, 100)
    assert need > 0 and need % (4 * (96 * 100 + 96)) == 0
    assert _rc("climb_act8_weight_grad_workspace", 100, 96, 100) == 0          # one token range: straight into C
    assert _rc("climb_act8_weight_grad_workspace", -1, 96, 100) == EINVAL
    assert _rc("climb_act8_weight_grad_workspace", 64, 2 ** 31 - 1, 100) == EINVAL and _rc("climb_act8_weight_grad_workspace", 64, 96, 2 ** 31 - 1) == EINVAL

    def call(nbytes=need, **change):
        a = dict(ok, **change)
        return _rc("climb_act8_weight_grad", a["dY"], a["lddy"], a["q"], a["ldq"], a["e"], a["lde"], a["C"], a["ldc"], None, a["M"], a["N"], a["K"], 0.0, a["ws"], nbytes, None)
    for change in (dict(M=-1), dict(N=0), dict(K=0), dict(lddy=95), dict(ldq=96), dict(ldq=104), dict(lde=1), dict(ldc=99), dict(dY=None), dict(q=p + 1), dict(e=None),
                   dict(C=None), dict(C=p + 2), dict(dY=p + 1), dict(ws=None), dict(ws=p + 4)):
        assert call(**change) == EINVAL, change
    assert call(nbytes=need - 1) == EINVAL


def test_sizes_beyond_a_launch_are_refused(mem):
    p = mem[0]
    big = (1 << 30) + 1
    assert _rc("climb_rows8_quant", p, 64, 0, p, 128, p, big, 64, None) == EINVAL
    assert _rc("climb_rows8_quant", p, 64, 0, p, 128, p, 1 << 28, 64, None) == EUNSUPPORTED
    assert _rc("climb_act8_save", p, 64, 0, p, 64, p, 1, 1 << 29, 64, None) == EUNSUPPORTED
    assert _rc("climb_act8_gelu_fwd", p, 64, 0, p, 64, p, 64, p, 1, 1 << 29, 64, None) == EUNSUPPORTED
    assert _rc("climb_act8_layernorm_fwd", p, 64, p, p, 1e-5, p, 64, 0, p, p, p, 64, p, 1, 1 << 26, 64, None) == EUNSUPPORTED
    assert _rc("climb_gemm_i8_nt", p, 128, p, p, 128, p, p, 1 << 20, 0, 1 << 24, 1 << 20, 64, None, 0, None, 0, None) == EUNSUPPORTED
    assert _rc("climb_act8_weight_grad", p, 1 << 20, p, 1 << 20, p, 1 << 14, p, 1 << 20, None, 64, 1 << 20, 1 << 20, 0.0, p, 1 << 60, None) == EUNSUPPORTED


def test_nothing_is_launched_for_no_rows():
    z = (0, 64, None)
    assert _rc("climb_rows8_quant", None, 64, 0, None, 128, None, *z) == 0
    assert _rc("climb_act8_save", None, 64, 0, None, 64, None, 1, *z) == 0
    assert _rc("climb_gemm_i8_nt", None, 128, None, None, 128, None, None, 32, 0, 0, 32, 64, None, 0, None, 0, None) == 0


def test_tensor_calls_refuse():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="HIP device"):
        rows8.quantize_rows(x)
    with pytest.raises(ValueError, match="HIP device"):
        rows8.checkpoint_save(x)
    with pytest.raises(ValueError, match="HIP device"):
        rows8.gelu_fwd(x)
    with pytest.raises(TypeError, match="tensor"):
        rows8.checkpoint_save([1.0])
    with pytest.raises(RuntimeError, match="autograd"):
        rows8.gelu_fwd(torch.zeros(4, 8, requires_grad=True))
    w = rows8.RowCodes(3, 8, (3,), torch.device("cpu"))
    assert w.q.shape == (3, 128) and w.scale.shape == (3,)
    with pytest.raises(ValueError, match="epilogue"):
        rows8.linear_i8(x, w, epi="tanh")
    with pytest.raises(ValueError, match="resid"):
        rows8.linear_i8(x, w, epi="resid")
    with pytest.raises(TypeError, match="RowCodes"):
        rows8.linear_i8(x, x)
    ck = rows8.Checkpoint(4, 8, (4,), torch.float32, torch.device("cpu"))
    with pytest.raises(ValueError, match="row statistics"):
        rows8.layernorm_bwd(x, ck, torch.ones(8))
    assert ck.nbytes == 4 * 16 + 4 * 4 and ck.q.shape == (4, 16) and ck.exps.shape == (4, 1) and ck.mean is None
    ck = rows8.Checkpoint(3, 70, (3,), torch.float32, torch.device("cpu"), stats=True)
    assert ck.nbytes == 3 * 84 + 4 + 24 and ck.mean.shape == ck.rstd.shape == (3,)
    assert rows8.GROUP == _lib.query("climb_act8_group")


def test_the_backward_takes_the_mode_of_its_forward():
    """`act8` switched between a forward and its backward: whether weight gradients are deferred (and where d(x_L) goes) follows what the forward kept"""
    from types import SimpleNamespace
    from climb_amd.engine import ViltEngine
    eng = object.__new__(ViltEngine)
    eng.precision, eng.split, eng.overlap_dw, eng.grad_ready_hook, eng.cfg = "bf16", False, False, None, dict(layers=12)
    ws = SimpleNamespace(M=256)
    for kept in (False, True):
        eng.saved = dict(act8=kept)
        sizes = []
        for now in (False, True):
            eng.act8 = now
            sizes.append(eng._dw_group_size(ws, None))
        assert sizes[0] == sizes[1] and (sizes[0] == 0) == kept


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name", ["gemm_i8.hip", "act8_wgrad.hip"])
def test_a_stage_is_refilled_only_behind_its_last_reads(name):
    """behind a raw barrier DMA overwrites the stage that was just read: the source itself asks for the LDS reads in front of each (a barrier waits for none)"""
    lines = open(os.path.join(ROOT, "climb_amd", "csrc", name)).read().splitlines()
    at = [i for i, l in enumerate(lines) if "__builtin_amdgcn_s_barrier()" in l]
    assert at
    for i in at:
        before = [l.strip() for l in lines[max(0, i - 2):i]]
        assert any("s_waitcnt lgkmcnt(0)" in l for l in before), (name, i + 1)


def test_the_built_kernels_meet_with_their_reads_back():
    """... and so it stands in the libraries: between a barrier of the int8 product or the large weight gradient and the last LDS read before it lies lgkmcnt(0)"""
    spec = importlib.util.spec_from_file_location("check_store_hazard", os.path.join(ROOT, "tools", "check_store_hazard.py"))
    ch = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ch)
    libs = [l for l in (os.path.join(ROOT, "climb_amd", "csrc", f) for f in ("libclimb_hip.so", "libclimb_hip_f16.so")) if os.path.exists(l)]
    if not libs or not os.path.exists(ch.HIPCC):
        pytest.skip("needs the built libraries and the ROCm llvm tools")
    for lib in libs:
        kernels, barriers = set(), 0
        for code in ch.library_code(lib):
            kern, waited = None, True
            for k, l in code:
                if "gemm_i8_kernel" not in k and "act8_wgrad_big_kernel" not in k:
                    continue
                if k != kern:
                    kern, waited = k, True
                if l.startswith("ds_read"):
                    waited = False
                elif l.startswith("s_waitcnt") and re.search(r"lgkmcnt\(0\)", l):
                    waited = True
                elif l.startswith("s_barrier"):
                    assert waited, k
                    kernels.add(k)
                    barriers += 1
        assert len(kernels) == 19 and barriers >= 3 * 18, (lib, len(kernels), barriers)          # (18 instantiations of the product)


def test_forward_mode_tangents_are_refused():
    """a tangent that a call would drop without a word: for matrices, vectors and tensors that are written in place"""
    import torch.autograd.forward_ad as fwd
    x, v, dev = torch.ones(4, 8), torch.ones(8), torch.device("cpu")
    with fwd.dual_level():
        for call in (lambda: rows8.gelu_fwd(fwd.make_dual(x, x)), lambda: rows8.quantize_rows(fwd.make_dual(x, x)), lambda: rows8._vec(fwd.make_dual(v, v), "bias", 8, dev),
                     lambda: rows8._target(fwd.make_dual(x, x), "out", (4, 8), torch.float32, dev)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert rows8._vec(v, "bias", 8, dev) is v          # inside a level, but without a tangent
        with pytest.raises(ValueError, match="HIP device"):
            rows8.gelu_fwd(x)
    assert rows8._vec(v, "bias", 8, dev) is v


def test_arguments_of_another_kind_are_named(mem):
    x = torch.zeros(4, 8)
    for call in (lambda: rows8.weight_grad(x, x), lambda: rows8.layernorm_bwd(x, None, x[0]), lambda: rows8.gelu_bwd(x, x), lambda: rows8.gelu_bwd(x, rows8.RowCodes(4, 8, (4,), torch.device("cpu")))):
        with pytest.raises(TypeError, match="Checkpoint"):
            call()
    w = rows8.RowCodes(3, 8, (3,), torch.device("cpu"))
    with pytest.raises(TypeError, match="out"):
        rows8.linear_i8(rows8.RowCodes(4, 8, (4,), torch.device("cpu")), w, out=[1.0])
    p = mem[0]
    for K in ((1 << 30) + 1, 2 ** 31 - 1):          # rounding them up would leave the type
        assert _rc("climb_gemm_i8_nt", p, 1 << 32, p, p, 1 << 32, p, p, 32, 0, 4, 32, K, None, 0, None, 0, None) == EUNSUPPORTED
        assert _rc("climb_linear_i8", p, 1 << 32, 1, p, 1 << 32, p, p, 32, 0, 4, 32, K, None, 0, None, 0, p, 1 << 30, None) == EUNSUPPORTED
