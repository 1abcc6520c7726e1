"""Rows in 8 bits on tensors: the int8 linear layer and 8-bit activation checkpoints (include/climb_hip.h, "8-bit rows").

Two formats.  `RowCodes` -- one fp32 scale a row, what the int8 product multiplies.  `Checkpoint` -- a power-of-two scale for each 64 columns, what a forward
pass keeps for its backward: half the bytes of a 16-bit activation, a quarter of an fp32 one.  A row (group) that holds a NaN or an infinity reads as NaN.

    w8 = quantize_rows(weight)                          # once, for as long as the weight stands
    y  = linear_i8(x, w8, bias, epi="gelu")             # evaluation

    y, ck = layernorm_fwd(x, gamma, beta, eps)          # training: keep `ck`, drop `x`
    dx, dgamma, dbeta = layernorm_bwd(dy, ck, gamma, dres=dres)
    a, ck = gelu_fwd(u);   du, a = gelu_bwd(da, ck, recompute=True)
    ck = checkpoint_save(x);   dw, db = weight_grad(dy, ck)

Matrices are [..., C] in fp32 or the library's 16-bit type, on one HIP device, any row stride; an input whose last dimension is strided or whose rows overlap
(a broadcast view) is copied first.  Work goes to the current stream of the inputs' device; nothing synchronises, and every scratch buffer is the call's
own (torch's allocator), so the calls can be captured.  Forward and backward are explicit calls as in climb_amd.engine: inputs that require grad are
refused while autograd records."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

GROUP = 64          # columns of a checkpoint that share a scale (climb_act8_group)
_EPI = {"none": 0, "gelu": 1, "resid": 2}


class RowCodes:
    """int8 codes [rows, ld] (columns cols .. ld are zero) and one fp32 scale a row"""
    __slots__ = ("q", "scale", "cols", "lead")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, cols: int, lead: Tuple[int, ...]):
        self.q, self.scale, self.cols, self.lead = q, scale, cols, lead

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    def dequantize(self) -> torch.Tensor:
        """the fp32 values the codes stand for"""
        return (self.q[:, :self.cols].float() * self.scale[:, None]).view(*self.lead, self.cols)


class Checkpoint:
    """int8 codes [rows, ld], a biased exponent byte for each row and 64 columns, and the dtype the activation had"""
    __slots__ = ("q", "exps", "cols", "lead", "dtype", "mean", "rstd")

    def __init__(self, rows: int, cols: int, lead: Tuple[int, ...], dtype: torch.dtype, device: torch.device):
        self.q = torch.empty((rows, _up(cols, 16)), dtype=torch.int8, device=device)
        self.exps = torch.empty((rows, _up(cols, GROUP) // GROUP), dtype=torch.uint8, device=device)
        self.cols, self.lead, self.dtype = cols, lead, dtype
        self.mean: Optional[torch.Tensor] = None          # LayerNorm's row statistics (layernorm_fwd)
        self.rstd: Optional[torch.Tensor] = None

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.exps.numel()

    def load(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """the activation the codes stand for (default: in the dtype it was saved from)"""
        dtype = dtype or self.dtype
        y = torch.empty((*self.lead, self.cols), dtype=dtype, device=self.q.device)
        _launch(self.q.device, "climb_act8_load", self.q, self.q.shape[1], self.exps, self.exps.shape[1], y, self.cols, _code(dtype), self.rows, self.cols)
        return y


def _up(x: int, m: int) -> int:
    return -(-x // m) * m


def _code(dtype: torch.dtype) -> int:
    if dtype is torch.float32:
        return 0
    if dtype is _lib.torch_h16():
        return 1
    raise TypeError(f"rows8: {dtype} is not a type of this library build (torch.float32 or {_lib.torch_h16()})")


def _launch(dev: torch.device, name: str, *args):
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


def _mat(x: torch.Tensor, what: str, cols: Optional[int] = None, rows: Optional[int] = None, dtype: Optional[torch.dtype] = None,
         dev: Optional[torch.device] = None) -> torch.Tensor:
    """x as [rows, cols] with unit column stride and rows that do not overlap"""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"rows8: {what} must be a tensor")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"rows8: {what} requires grad, and these calls record nothing for autograd: detach it (forward and backward are explicit calls)")
    if not x.is_cuda or (dev is not None and x.device != dev):
        raise ValueError(f"rows8: {what} is on {x.device}; every tensor of a call must be on one HIP device")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"rows8: {what} has shape {tuple(x.shape)}; a last dimension of at least 1 is needed")
    if cols is not None and x.shape[-1] != cols:
        raise ValueError(f"rows8: {what} has {x.shape[-1]} columns, {cols} expected")
    if dtype is not None and x.dtype is not dtype:
        raise TypeError(f"rows8: {what} is {x.dtype}, {dtype} expected")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if rows is not None and x.shape[0] != rows:
        raise ValueError(f"rows8: {what} has {x.shape[0]} rows, {rows} expected")
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    return max(x.stride(0), x.shape[1]) if x.shape[0] > 1 else x.shape[1]


def _vec(x: Optional[torch.Tensor], what: str, n: int, dev: torch.device) -> Optional[torch.Tensor]:
    if x is None:
        return None
    return _mat(x.reshape(1, -1) if isinstance(x, torch.Tensor) else x, what, cols=n, rows=1, dtype=torch.float32, dev=dev)


def _target(x: torch.Tensor, what: str, shape: Tuple[int, ...], dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """a tensor that the call writes: never copied"""
    if not isinstance(x, torch.Tensor) or tuple(x.shape) != shape or x.dtype is not dtype or x.device != dev:
        raise ValueError(f"rows8: {what} must be a {dtype} tensor of shape {shape} on {dev}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"rows8: {what} requires grad and would be written in place")
    if (x.shape[-1] > 1 and x.stride(-1) != 1) or (x.dim() == 2 and x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise ValueError(f"rows8: {what} needs unit column stride and rows that do not overlap")
    return x


# ------------------------------------------------------------------------------------------------ int8 linear layer
def quantize_rows(x: torch.Tensor) -> RowCodes:
    """Row codes of x: the tokens of an activation, or the output channels of a weight [N, K]."""
    m = _mat(x, "x")
    M, C = m.shape
    code = _code(m.dtype)
    q = torch.empty((M, _up(C, 128)), dtype=torch.int8, device=m.device)
    s = torch.empty((M,), dtype=torch.float32, device=m.device)
    _launch(m.device, "climb_rows8_quant", m, _ld(m), code, q, q.shape[1], s, M, C)
    return RowCodes(q, s, C, tuple(x.shape[:-1]))


def linear_i8(x: Union[torch.Tensor, RowCodes], w: RowCodes, bias: Optional[torch.Tensor] = None, epi: str = "none", resid: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = epi(x8 w8^T + bias): x quantised by token here (or handed over as RowCodes, which several products can share), w by output channel.
    epi: "none", "gelu" (erf form) or "resid" (+ resid, fp32; `out` may be `resid` itself).  The products' sum is exact, the rest is fp32, y is rounded once
    to out_dtype (default: x's)."""
    if epi not in _EPI:
        raise ValueError(f"rows8: unknown epilogue {epi!r} (one of {sorted(_EPI)})")
    if (resid is not None) != (epi == "resid"):
        raise ValueError('rows8: `resid` goes with epi="resid"')
    if not isinstance(w, RowCodes):
        raise TypeError("rows8: w must be RowCodes (quantize_rows(weight))")
    dev, N, K = w.q.device, w.rows, w.cols
    if isinstance(x, RowCodes):
        if x.q.device != dev:
            raise ValueError(f"rows8: x is on {x.q.device}, w on {dev}")
        if x.cols != K:
            raise ValueError(f"rows8: x has {x.cols} columns, {K} expected")
        xq, lead, dt = x, x.lead, torch.float32
    else:
        _mat(x, "x", cols=K, dev=dev)
        xq, lead, dt = quantize_rows(x), tuple(x.shape[:-1]), x.dtype
    if N == 0:
        raise ValueError("rows8: w has no rows")
    M = xq.rows
    if out is not None:
        y = _target(out, "out", (*lead, N), out_dtype or out.dtype, dev)
        if y.dim() != 2 and not y.is_contiguous():
            raise ValueError("rows8: out with more than two dimensions must be contiguous")
        y2 = y.view(-1, N) if y.dim() != 2 else y
    else:
        y = torch.empty((*lead, N), dtype=out_dtype or dt, device=dev)
        y2 = y.view(M, N)
    code = _code(y.dtype)
    b = _vec(bias, "bias", N, dev)
    r = _mat(resid, "resid", cols=N, rows=M, dtype=torch.float32, dev=dev) if resid is not None else None
    _launch(dev, "climb_gemm_i8_nt", xq.q, xq.q.shape[1], xq.scale, w.q, w.q.shape[1], w.scale, y2, _ld(y2), code, M, N, K, b, _EPI[epi], r, _ld(r) if r is not None else 0)
    return y


# ------------------------------------------------------------------------------------------------ checkpoints
def checkpoint_save(x: torch.Tensor) -> Checkpoint:
    """Keep x in 8 bits."""
    m = _mat(x, "x")
    M, C = m.shape
    code = _code(m.dtype)
    ck = Checkpoint(M, C, tuple(x.shape[:-1]), m.dtype, m.device)
    _launch(m.device, "climb_act8_save", m, _ld(m), code, ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], M, C)
    return ck


def weight_grad(dy: torch.Tensor, ck: Checkpoint, dw: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None,
                bias: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dw [N, K], dbias [N]) of y = x w^T + b from dy (16 bit) and the checkpoint of x.  Given `dw` / `dbias` are added to (fp32, in place); `bias` False:
    no bias gradient."""
    dev, K = ck.q.device, ck.cols
    d = _mat(dy, "dy", rows=ck.rows, dtype=_lib.torch_h16(), dev=dev)
    M, N = d.shape
    if dbias is not None and not bias:
        raise ValueError("rows8: dbias given, bias=False")
    beta = 0.0 if dw is None and dbias is None else 1.0
    new = torch.empty if beta == 0.0 else torch.zeros
    dw = new((N, K), dtype=torch.float32, device=dev) if dw is None else _target(dw, "dw", (N, K), torch.float32, dev)
    if bias:
        dbias = new((N,), dtype=torch.float32, device=dev) if dbias is None else _target(dbias, "dbias", (N,), torch.float32, dev)
    nb = _lib.query_arg("climb_act8_weight_grad_workspace", M, N, K)
    ws = torch.empty((nb,), dtype=torch.uint8, device=dev) if nb > 0 else None
    _launch(dev, "climb_act8_weight_grad", d, _ld(d), ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], dw, _ld(dw), dbias, M, N, K, beta, ws, max(nb, 0))
    return dw, dbias


def layernorm_fwd(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Checkpoint]:
    """y = LayerNorm(x) (x fp32, at most 1536 columns; y in out_dtype, default fp32) and the checkpoint of x with its row statistics."""
    m = _mat(x, "x", dtype=torch.float32)
    M, C = m.shape
    if C > 1536:
        raise ValueError(f"rows8: LayerNorm of {C} columns; this build holds rows of at most 1536 in registers")
    dev = m.device
    y = torch.empty(x.shape, dtype=out_dtype or torch.float32, device=dev)
    code = _code(y.dtype)
    g, b = _vec(gamma, "gamma", C, dev), _vec(beta, "beta", C, dev)
    ck = Checkpoint(M, C, tuple(x.shape[:-1]), torch.float32, dev)
    st = torch.empty((2, M), dtype=torch.float32, device=dev)
    ck.mean, ck.rstd = st[0], st[1]
    _launch(dev, "climb_act8_layernorm_fwd", m, _ld(m), g, b, float(eps), y, C, code, ck.mean, ck.rstd, ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], M, C)
    return y, ck


def layernorm_bwd(dy: torch.Tensor, ck: Checkpoint, gamma: torch.Tensor, dres: Optional[torch.Tensor] = None, dgamma: Optional[torch.Tensor] = None,
                  dbeta: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgamma, dbeta), dx = dres + d(LayerNorm)/dx^T dy in fp32; given `dgamma` / `dbeta` are added to."""
    if ck.mean is None:
        raise ValueError("rows8: this checkpoint holds no row statistics (layernorm_fwd makes one that does)")
    dev, M, C = ck.q.device, ck.rows, ck.cols
    d = _mat(dy, "dy", cols=C, rows=M, dev=dev)
    code = _code(d.dtype)
    g = _vec(gamma, "gamma", C, dev)
    r = _mat(dres, "dres", cols=C, rows=M, dtype=torch.float32, dev=dev) if dres is not None else None
    acc = dgamma is not None or dbeta is not None
    new = torch.zeros if acc or M == 0 else torch.empty
    dgamma = new((C,), dtype=torch.float32, device=dev) if dgamma is None else _target(dgamma, "dgamma", (C,), torch.float32, dev)
    dbeta = new((C,), dtype=torch.float32, device=dev) if dbeta is None else _target(dbeta, "dbeta", (C,), torch.float32, dev)
    dx = torch.empty((*ck.lead, C), dtype=torch.float32, device=dev)
    if M == 0:
        return dx, dgamma, dbeta
    rpb = _lib.query("climb_act8_layernorm_bwd_rows_per_block")
    nblk = -(-M // rpb)
    part = torch.empty((nblk, 3, C), dtype=torch.float32, device=dev)
    _launch(dev, "climb_act8_layernorm_bwd", d, _ld(d), code, ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], ck.mean, ck.rstd, g, r, _ld(r) if r is not None else 0,
            dx, C, None, 0, part, M, C)
    _launch(dev, "climb_colreduce3", part, 3 * C, nblk, dgamma, dbeta, None, C, 1.0 if acc else 0.0)
    return dx, dgamma, dbeta


def gelu_fwd(u: torch.Tensor) -> Tuple[torch.Tensor, Checkpoint]:
    """a = gelu(u) (erf form) in u's dtype, and the checkpoint of u."""
    m = _mat(u, "u")
    M, C = m.shape
    code = _code(m.dtype)
    a = torch.empty(u.shape, dtype=m.dtype, device=m.device)
    ck = Checkpoint(M, C, tuple(u.shape[:-1]), m.dtype, m.device)
    _launch(m.device, "climb_act8_gelu_fwd", m, _ld(m), code, a, C, ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], M, C)
    return a, ck


def gelu_bwd(da: torch.Tensor, ck: Checkpoint, recompute: bool = False):
    """du = da gelu'(u) in da's dtype; recompute: (du, gelu(u)) -- the activation itself, which the next layer's weight gradient reads, is not kept."""
    dev, M, C = ck.q.device, ck.rows, ck.cols
    d = _mat(da, "da", cols=C, rows=M, dev=dev)
    code = _code(d.dtype)
    du = torch.empty((*ck.lead, C), dtype=d.dtype, device=dev)
    a = torch.empty_like(du) if recompute else None
    _launch(dev, "climb_act8_gelu_bwd", d, _ld(d), code, ck.q, ck.q.shape[1], ck.exps, ck.exps.shape[1], du, C, a, C, M, C)
    return (du, a) if recompute else du
