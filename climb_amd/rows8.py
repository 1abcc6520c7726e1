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
refused while autograd records, and so are forward-mode tangents.

The host's share of a call is kept small (a launch alone is 3 us, and a batch of one sequence runs in less): one allocation per code matrix with its scales,
contiguous inputs taken as they are, the stream read as a plain number."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as _fwd

from . import _lib

GROUP = 64          # columns of a checkpoint that share a scale (climb_act8_group)
_EPI = {"none": 0, "gelu": 1, "resid": 2}
_F32 = torch.float32


class RowCodes:
    """int8 codes [rows, ld] (columns cols .. ld are zero) and one fp32 scale a row, in one buffer"""
    __slots__ = ("buf", "rows", "cols", "ld", "lead", "device")

    def __init__(self, rows: int, cols: int, lead: Tuple[int, ...], device: torch.device):
        self.rows, self.cols, self.ld, self.lead, self.device = rows, cols, _up(cols, 128), lead, device
        self.buf = torch.empty(rows * (self.ld + 4), dtype=torch.int8, device=device)

    @property
    def q(self) -> torch.Tensor:
        return self.buf[:self.rows * self.ld].view(self.rows, self.ld)

    @property
    def scale(self) -> torch.Tensor:
        return self.buf[self.rows * self.ld:].view(_F32)

    def dequantize(self) -> torch.Tensor:
        """the fp32 values the codes stand for"""
        return (self.q[:, :self.cols].float() * self.scale[:, None]).view(*self.lead, self.cols)


class Checkpoint:
    """int8 codes [rows, ld], an exponent byte for each row and 64 columns, LayerNorm's row statistics if layernorm_fwd made it, in one buffer, and the dtype the
    activation had"""
    __slots__ = ("buf", "rows", "cols", "ld", "groups", "lead", "dtype", "device", "_stats")

    def __init__(self, rows: int, cols: int, lead: Tuple[int, ...], dtype: torch.dtype, device: torch.device, stats: bool = False):
        ld, groups = (cols + 15) & ~15, ((cols + GROUP - 1) // GROUP + 3) & ~3          # (whole words of exponents: the weight gradient fetches four at a time)
        self.rows, self.cols, self.ld, self.groups, self.lead, self.dtype, self.device = rows, cols, ld, groups, lead, dtype, device
        n = rows * (ld + groups)
        if stats:          # byte offset of mean [rows], rstd [rows]
            self._stats = n = (n + 15) & ~15
            n += 8 * rows
        else:
            self._stats = None
        self.buf = torch.empty(n, dtype=torch.uint8, device=device)

    @property
    def q(self) -> torch.Tensor:
        return self.buf[:self.rows * self.ld].view(torch.int8).view(self.rows, self.ld)

    @property
    def exps(self) -> torch.Tensor:
        n = self.rows * self.ld
        return self.buf[n:n + self.rows * self.groups].view(self.rows, self.groups)[:, :-(-self.cols // GROUP)]

    @property
    def mean(self) -> Optional[torch.Tensor]:
        return self.buf[self._stats:self._stats + 4 * self.rows].view(_F32) if self._stats is not None else None

    @property
    def rstd(self) -> Optional[torch.Tensor]:
        return self.buf[self._stats + 4 * self.rows:].view(_F32) if self._stats is not None else None

    @property
    def nbytes(self) -> int:
        return self.buf.numel()

    def _args(self) -> Tuple[int, int, int, int]:
        p = self.buf.data_ptr()
        return p, self.ld, p + self.rows * self.ld, self.groups

    def load(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """the activation the codes stand for (default: in the dtype it was saved from)"""
        dtype = dtype or self.dtype
        code = _code(dtype)
        y = torch.empty((*self.lead, self.cols), dtype=dtype, device=self.device)
        _launch(self.device, "climb_act8_load", *self._args(), y.data_ptr(), self.cols, code, self.rows, self.cols)
        return y


def _up(x: int, m: int) -> int:
    return -(-x // m) * m


_h16 = None


def _h16_type() -> torch.dtype:
    global _h16
    if _h16 is None:
        _h16 = _lib.torch_h16()
    return _h16


def _code(dtype: torch.dtype) -> int:
    if dtype is _F32:
        return 0
    if dtype is _h16_type():
        return 1
    raise TypeError(f"rows8: {dtype} is not a type of this library build (torch.float32 or {_h16})")


_fns = {}


def _launch(dev: torch.device, name: str, *args):
    """the launcher on the current stream of `dev` (also where another device is the current one); arguments are plain numbers"""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = _lib.bound(name)
    i = dev.index
    if i == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))          # (what torch.cuda.current_stream(dev).cuda_stream holds, without the object: 0.1 against 1.9 us)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc != 0:
        _lib.check(name, rc)


def _query(name: str, *args) -> int:
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = _lib.bound(name)
    return fn(*args)


def _recorded(x: torch.Tensor) -> bool:
    """whether autograd would have to see what is done with x, in reverse mode or (inside forward_ad.dual_level()) in forward mode"""
    return (x.requires_grad and torch.is_grad_enabled()) or (_fwd._current_level >= 0 and _fwd.unpack_dual(x).tangent is not None)


def _mat(x: torch.Tensor, what: str, cols: Optional[int] = None, rows: Optional[int] = None, dtype: Optional[torch.dtype] = None,
         dev: Optional[torch.device] = None) -> Tuple[torch.Tensor, int, int, int]:
    """(x, rows, cols, row stride) of x as a matrix with unit column stride and rows that do not overlap"""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"rows8: {what} must be a tensor")
    if _recorded(x):
        raise RuntimeError(f"rows8: {what} requires grad or carries a forward-mode tangent, and these calls record nothing for autograd: detach it (forward and backward are "
                           "explicit calls)")
    if not x.is_cuda or (dev is not None and x.device != dev):
        raise ValueError(f"rows8: {what} is on {x.device}; every tensor of a call must be on one HIP device")
    shape = x.shape
    C = shape[-1] if shape else 0
    if C == 0:
        raise ValueError(f"rows8: {what} has shape {tuple(shape)}; a last dimension of at least 1 is needed")
    if cols is not None and C != cols:
        raise ValueError(f"rows8: {what} has {C} columns, {cols} expected")
    if dtype is not None and x.dtype is not dtype:
        raise TypeError(f"rows8: {what} is {x.dtype}, {dtype} expected")
    if x.is_contiguous():
        M, ld = x.numel() // C, C
    else:
        if len(shape) != 2:
            x = x.reshape(-1, C)
        M = x.shape[0]
        if (C > 1 and x.stride(1) != 1) or (M > 1 and x.stride(0) < C):
            x = x.contiguous()
        ld = x.stride(0) if M > 1 else C
    if rows is not None and M != rows:
        raise ValueError(f"rows8: {what} has {M} rows, {rows} expected")
    return x, M, C, ld


def _kept(ck: "Checkpoint") -> "Checkpoint":
    if not isinstance(ck, Checkpoint):
        raise TypeError(f"rows8: ck must be a Checkpoint (checkpoint_save, gelu_fwd and layernorm_fwd make one), not {type(ck).__name__}")
    return ck


def _like(x: torch.Tensor, shape) -> torch.Tensor:
    """an empty contiguous tensor of x's dtype (empty_like is the cheapest of torch's allocations)"""
    return torch.empty_like(x) if x.shape == shape and x.is_contiguous() else x.new_empty(shape)


def _vec(x: torch.Tensor, what: str, n: int, dev: torch.device) -> torch.Tensor:
    if isinstance(x, torch.Tensor) and x.dtype is _F32 and x.device == dev and x.numel() == n and x.is_contiguous() and not _recorded(x):
        return x
    x, M, C, ld = _mat(x, what, dtype=_F32, dev=dev)
    if M * C != n:
        raise ValueError(f"rows8: {what} has {M * C} elements, {n} expected")
    return x if M == 1 or ld == C else x.contiguous()


def _target(x: torch.Tensor, what: str, shape: Tuple[int, ...], dtype: torch.dtype, dev: torch.device) -> int:
    """row stride of a tensor that the call writes: never copied"""
    if not isinstance(x, torch.Tensor) or tuple(x.shape) != tuple(shape) or x.dtype is not dtype or x.device != dev:
        raise ValueError(f"rows8: {what} must be a {dtype} tensor of shape {tuple(shape)} on {dev}")
    if _recorded(x):
        raise RuntimeError(f"rows8: {what} requires grad or carries a forward-mode tangent, and would be written in place")
    if x.is_contiguous():
        return shape[-1]
    if x.dim() != 2 or (shape[1] > 1 and x.stride(1) != 1) or (shape[0] > 1 and x.stride(0) < shape[1]):
        raise ValueError(f"rows8: {what} needs unit column stride and rows that do not overlap (more than two dimensions: contiguous)")
    return x.stride(0) if shape[0] > 1 else shape[1]


# ------------------------------------------------------------------------------------------------ int8 linear layer
def quantize_rows(x: torch.Tensor) -> RowCodes:
    """Row codes of x: the tokens of an activation, or the output channels of a weight [N, K]."""
    m, M, C, ld = _mat(x, "x")
    code = _code(m.dtype)
    r = RowCodes(M, C, tuple(x.shape[:-1]), m.device)
    p = r.buf.data_ptr()
    _launch(m.device, "climb_rows8_quant", m.data_ptr(), ld, code, p, r.ld, p + M * r.ld, M, C)
    return r


def linear_i8(x: Union[torch.Tensor, RowCodes], w: RowCodes, bias: Optional[torch.Tensor] = None, epi: str = "none", resid: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = epi(x8 w8^T + bias): x quantised by token here (or handed over as RowCodes, which several products can share), w by output channel.
    epi: "none", "gelu" (erf form) or "resid" (+ resid, fp32; `out` may be `resid` itself).  The products' sum is exact, the rest is fp32, y is rounded once
    to out_dtype (default: x's; fp32 for RowCodes).  `out` must not overlap x, w or bias."""
    e = _EPI.get(epi)
    if e is None:
        raise ValueError(f"rows8: unknown epilogue {epi!r} (one of {sorted(_EPI)})")
    if (resid is not None) != (e == 2):
        raise ValueError('rows8: `resid` goes with epi="resid"')
    if not isinstance(w, RowCodes):
        raise TypeError("rows8: w must be RowCodes (quantize_rows(weight))")
    dev, N, K = w.device, w.rows, w.cols
    if N == 0:
        raise ValueError("rows8: w has no rows")
    codes = isinstance(x, RowCodes)
    if codes:
        if x.device != dev:
            raise ValueError(f"rows8: x is on {x.device}, w on {dev}")
        if x.cols != K:
            raise ValueError(f"rows8: x has {x.cols} columns, {K} expected")
        M, lead, dt = x.rows, x.lead, _F32
    else:
        m, M, _, ldx = _mat(x, "x", cols=K, dev=dev)
        lead, dt = x.shape[:-1], m.dtype
        xcode = _code(dt)
    if out is None:
        dt = out_dtype or dt
        ycode = _code(dt)
        y, ldy = (m.new_empty((*lead, N)) if not codes and dt is m.dtype else torch.empty((*lead, N), dtype=dt, device=dev)), N
    else:
        if not isinstance(out, torch.Tensor):
            raise TypeError("rows8: out must be a tensor")
        y, dt = out, out_dtype or out.dtype
        ycode, ldy = _code(dt), _target(out, "out", (*lead, N), dt, dev)
    b = 0
    if bias is not None:
        bias = _vec(bias, "bias", N, dev)
        b = bias.data_ptr()
    r = ldr = 0
    if resid is not None:
        resid, _, _, ldr = _mat(resid, "resid", cols=N, rows=M, dtype=_F32, dev=dev)
        r = resid.data_ptr()
    wp = w.buf.data_ptr()
    if codes:
        xp = x.buf.data_ptr()
        _launch(dev, "climb_gemm_i8_nt", xp, x.ld, xp + M * x.ld, wp, w.ld, wp + N * w.ld, y.data_ptr(), ldy, ycode, M, N, K, b, e, r, ldr)
    else:
        nb = _query("climb_linear_i8_workspace", M, K)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb > 0 else None
        _launch(dev, "climb_linear_i8", m.data_ptr(), ldx, xcode, wp, w.ld, wp + N * w.ld, y.data_ptr(), ldy, ycode, M, N, K, b, e, r, ldr,
                ws.data_ptr() if nb > 0 else 0, nb)
    return y


# ------------------------------------------------------------------------------------------------ checkpoints
def checkpoint_save(x: torch.Tensor) -> Checkpoint:
    """Keep x in 8 bits."""
    m, M, C, ld = _mat(x, "x")
    code = _code(m.dtype)
    ck = Checkpoint(M, C, tuple(x.shape[:-1]), m.dtype, m.device)
    _launch(m.device, "climb_act8_save", m.data_ptr(), ld, code, *ck._args(), M, C)
    return ck


def weight_grad(dy: torch.Tensor, ck: Checkpoint, dw: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None,
                bias: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dw [N, K], dbias [N]) of y = x w^T + b from dy (16 bit) and the checkpoint of x.  Given `dw` / `dbias` are added to (fp32, in place); `bias` False:
    no bias gradient."""
    dev, K = _kept(ck).device, ck.cols
    d, M, N, ld = _mat(dy, "dy", rows=ck.rows, dtype=_h16_type(), dev=dev)
    if dbias is not None and not bias:
        raise ValueError("rows8: dbias given, bias=False")
    beta = 0.0 if dw is None and dbias is None else 1.0
    new = torch.empty if beta == 0.0 else torch.zeros
    if dw is None:
        dw, ldw = new((N, K), dtype=_F32, device=dev), K
    else:
        ldw = _target(dw, "dw", (N, K), _F32, dev)
    if dbias is not None:
        _target(dbias, "dbias", (N,), _F32, dev)
    elif bias:
        dbias = new((N,), dtype=_F32, device=dev)
    nb = _query("climb_act8_weight_grad_workspace", M, N, K)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb > 0 else None
    _launch(dev, "climb_act8_weight_grad", d.data_ptr(), ld, *ck._args(), dw.data_ptr(), ldw, dbias.data_ptr() if dbias is not None else 0, M, N, K, beta,
            ws.data_ptr() if nb > 0 else 0, nb)
    return dw, dbias


def layernorm_fwd(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Checkpoint]:
    """y = LayerNorm(x) (x fp32, at most 1536 columns; y in out_dtype, default fp32) and the checkpoint of x with its row statistics."""
    m, M, C, ld = _mat(x, "x", dtype=_F32)
    if C > 1536:
        raise ValueError(f"rows8: LayerNorm of {C} columns; this build holds rows of at most 1536 in registers")
    dev, dt = m.device, out_dtype or _F32
    code = _code(dt)
    g, b = _vec(gamma, "gamma", C, dev), _vec(beta, "beta", C, dev)
    y = torch.empty_like(x, dtype=dt) if x.is_contiguous() else torch.empty(x.shape, dtype=dt, device=dev)
    ck = Checkpoint(M, C, tuple(x.shape[:-1]), _F32, dev, stats=True)
    q, ldq, e, lde = ck._args()
    st = q + ck._stats
    _launch(dev, "climb_act8_layernorm_fwd", m.data_ptr(), ld, g.data_ptr(), b.data_ptr(), eps, y.data_ptr(), C, code, st, st + 4 * M, q, ldq, e, lde, M, C)
    return y, ck


def layernorm_bwd(dy: torch.Tensor, ck: Checkpoint, gamma: torch.Tensor, dres: Optional[torch.Tensor] = None, dgamma: Optional[torch.Tensor] = None,
                  dbeta: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgamma, dbeta), dx = dres + d(LayerNorm)/dx^T dy in fp32; given `dgamma` / `dbeta` are added to."""
    if _kept(ck)._stats is None:
        raise ValueError("rows8: this checkpoint holds no row statistics (layernorm_fwd makes one that does)")
    dev, M, C = ck.device, ck.rows, ck.cols
    d, _, _, ld = _mat(dy, "dy", cols=C, rows=M, dev=dev)
    code = _code(d.dtype)
    g = _vec(gamma, "gamma", C, dev)
    r = ldr = 0
    if dres is not None:
        dres, _, _, ldr = _mat(dres, "dres", cols=C, rows=M, dtype=_F32, dev=dev)
        r = dres.data_ptr()
    acc = dgamma is not None or dbeta is not None
    new = torch.zeros_like if acc or M == 0 else torch.empty_like
    if g.dim() != 1:
        g = g.view(C)
    if dgamma is None:
        dgamma = new(g)
    else:
        _target(dgamma, "dgamma", (C,), _F32, dev)
    if dbeta is None:
        dbeta = new(g)
    else:
        _target(dbeta, "dbeta", (C,), _F32, dev)
    dx = _like(g if dres is None else dres, (*ck.lead, C))
    if M == 0:
        return dx, dgamma, dbeta
    nb = _query("climb_act8_layernorm_bwd_workspace", M, C, 0)
    part = torch.empty(nb, dtype=torch.uint8, device=dev) if nb > 0 else None
    q, ldq, e, lde = ck._args()
    st = q + ck._stats
    _launch(dev, "climb_act8_layernorm_bwd", d.data_ptr(), ld, code, q, ldq, e, lde, st, st + 4 * M, g.data_ptr(), r, ldr, dx.data_ptr(), C, 0, 0, part.data_ptr() if nb > 0 else 0,
            dgamma.data_ptr(), dbeta.data_ptr(), 0, 1.0 if acc else 0.0, M, C)
    return dx, dgamma, dbeta


def gelu_fwd(u: torch.Tensor) -> Tuple[torch.Tensor, Checkpoint]:
    """a = gelu(u) (erf form) in u's dtype, and the checkpoint of u."""
    m, M, C, ld = _mat(u, "u")
    code = _code(m.dtype)
    a = _like(u, u.shape)
    ck = Checkpoint(M, C, tuple(u.shape[:-1]), m.dtype, m.device)
    _launch(m.device, "climb_act8_gelu_fwd", m.data_ptr(), ld, code, a.data_ptr(), C, *ck._args(), M, C)
    return a, ck


def gelu_bwd(da: torch.Tensor, ck: Checkpoint, recompute: bool = False):
    """du = da gelu'(u) in da's dtype; recompute: (du, gelu(u)) -- the activation itself, which the next layer's weight gradient reads, is not kept."""
    dev, M, C = _kept(ck).device, ck.rows, ck.cols
    d, _, _, ld = _mat(da, "da", cols=C, rows=M, dev=dev)
    code = _code(d.dtype)
    du = _like(d, (*ck.lead, C))
    a = torch.empty_like(du) if recompute else None
    _launch(dev, "climb_act8_gelu_bwd", d.data_ptr(), ld, code, *ck._args(), du.data_ptr(), C, a.data_ptr() if recompute else 0, C, M, C)
    return (du, a) if recompute else du
