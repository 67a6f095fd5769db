"""Operators beside the network, on torch CUDA tensors: 4-bit microscaled
matrices and the move sampler (include/azb200.h, "device operators").

    q = mx4_quantise(w)                        # Mx4: codes and block scales
    mx4_values(q, torch.float32)               # the values q holds, exactly
    y = mx4_product(x, q, bias=b, relu=True)   # Q(x) . q^T on the tensor cores
    moves, logprob = sample_moves(y, noise, legal=mask, temperature=0.8, top_k=40, top_p=0.95)

Every call runs on the tensors' device in torch's current stream, does not
synchronise and can be captured into a CUDA graph after a first call on the
device. Tensors are float32 or bfloat16; a matrix's rows may be any distance
apart (0 for a broadcast source), its columns are adjacent. There is no
backward pass: a source that requires a gradient is refused. Bad arguments
raise ValueError, failures of the device azb200.CudaError.
"""
from __future__ import annotations

import ctypes as C

import torch

import azb200
from azb200 import CudaError, SampleArgs

_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _fail(fn: str, e) -> None:
    msg = e.value.decode()
    raise (CudaError(msg) if msg.startswith("cuda") or ": cuda" in msg else ValueError(msg))


def _type(t, what: str) -> int:
    code = _TYPES.get(t)
    if code is None:
        raise ValueError(f"{what}: float32 or bfloat16, not {t}")
    return code


def _matrix(t: torch.Tensor, what: str):
    """(type, rows, cols, row stride) of a 2-D source on a GPU."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: a CUDA tensor is needed")
    code = _type(t.dtype, what)
    if t.dim() != 2:
        raise ValueError(f"{what}: a matrix is needed, not {t.dim()} dimensions")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and there is no backward pass (detach it)")
    rows, cols = t.shape
    if cols < 1:
        raise ValueError(f"{what}: at least one column is needed")
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{what}: columns must be adjacent (stride {inner})")
    return code, rows, cols, ld


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _same_device(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


class Mx4:
    """A rows x cols matrix in the 4-bit microscaled form: `codes` (uint8
    [rows, 16 * ceil(cols / 32)]) and `scales` (uint8, in the tensor core's
    tile order), as azb_mx4_quantise lays them out."""

    __slots__ = ("codes", "scales", "rows", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        need, got = _sizes(rows, cols), (codes.numel(), scales.numel())
        if need != got or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"Mx4 of {rows} x {cols}: {need} bytes of codes and scales, not {got}")
        if not (codes.is_cuda and codes.is_contiguous() and scales.is_contiguous() and codes.device == scales.device):
            raise ValueError("Mx4: codes and scales must be contiguous and on one GPU")
        self.codes, self.scales, self.rows, self.cols = codes, scales, rows, cols

    @property
    def device(self):
        return self.codes.device

    @property
    def shape(self):
        return (self.rows, self.cols)

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _sizes(rows: int, cols: int):
    nc, ns, e = C.c_size_t(), C.c_size_t(), azb200._err()
    if azb200.lib().azb_mx4_sizes(rows, cols, C.byref(nc), C.byref(ns), e, 1024) != 0:
        _fail("azb_mx4_sizes", e)
    return nc.value, ns.value


def mx4_quantise(x: torch.Tensor) -> Mx4:
    """The 4-bit microscaled form of a matrix."""
    code, rows, cols, ld = _matrix(x, "x")
    nc, ns = _sizes(rows, cols)
    q = object.__new__(Mx4)
    q.codes = torch.empty((rows, nc // rows if rows else 0), dtype=torch.uint8, device=x.device)
    q.scales = torch.empty(ns, dtype=torch.uint8, device=x.device)
    q.rows, q.cols = rows, cols
    e = azb200._err()
    if azb200.lib().azb_mx4_quantise(x.device.index, x.data_ptr(), code, rows, cols, ld, q.codes.data_ptr(),
                                     q.scales.data_ptr(), _stream(x.device), e, 1024) != 0:
        _fail("azb_mx4_quantise", e)
    return q


def mx4_values(q: Mx4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values q holds; exact in either type."""
    code = _type(dtype, "dtype")
    out = torch.empty((q.rows, q.cols), dtype=dtype, device=q.device)
    e = azb200._err()
    if azb200.lib().azb_mx4_values(q.device.index, q.codes.data_ptr(), q.scales.data_ptr(), q.rows, q.cols,
                                   out.data_ptr(), code, q.cols, _stream(q.device), e, 1024) != 0:
        _fail("azb_mx4_values", e)
    return out


def mx4_product(x, w: Mx4, *, bias: torch.Tensor | None = None, relu: bool = False,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(x . w^T + bias) with both factors in the 4-bit form, summed in
    fp32 and rounded once to `dtype` (default: x's, float32 for an Mx4). x: an
    Mx4, or a matrix or vector that is quantised on the way."""
    if not isinstance(w, Mx4):
        raise ValueError("w: an Mx4 is needed (mx4_quantise)")
    quantised = isinstance(x, Mx4)
    vector = False
    if quantised:
        m, k, x_type = x.rows, x.cols, 0
    else:
        vector = isinstance(x, torch.Tensor) and x.dim() == 1
        if vector:
            x = x.unsqueeze(0)
        x_type, m, k, x_ld = _matrix(x, "x")
    if k != w.cols:
        raise ValueError(f"x has {k} columns, w {w.cols}")
    dtype = dtype or (torch.float32 if quantised else x.dtype)
    code = _type(dtype, "dtype")
    device = x.device
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (w.rows,) or not bias.is_contiguous()):
        raise ValueError(f"bias: {w.rows} adjacent float32 numbers are needed")
    _same_device(device, w=w, bias=bias)
    n = w.rows
    out = torch.empty((m, n), dtype=dtype, device=device)
    L, e = azb200.lib(), azb200._err()
    tail = (n, None if bias is None else bias.data_ptr(), int(relu), out.data_ptr(), code, n)
    if quantised:
        rc = L.azb_mx4_product(device.index, x.codes.data_ptr(), x.scales.data_ptr(), m, w.codes.data_ptr(),
                               w.scales.data_ptr(), n, k, *tail[1:], _stream(device), e, 1024)
    else:
        need = L.azb_mx4_linear_workspace(m, k)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        rc = L.azb_mx4_linear(device.index, x.data_ptr(), x_type, m, k, x_ld, w.codes.data_ptr(), w.scales.data_ptr(),
                              *tail, ws.data_ptr(), need, _stream(device), e, 1024)
    if rc != 0:
        _fail("azb_mx4_product", e)
    return out[0] if vector else out


def _per_row(v, name: str, rows: int, device, dtype):
    """(number, pointer) of a setting: one number, or one per row."""
    if not isinstance(v, torch.Tensor):
        return v, None
    if v.dtype != dtype or v.shape != (rows,) or v.device != device or not v.is_contiguous():
        raise ValueError(f"{name}: a number, or {rows} adjacent {dtype} numbers on {device}")
    return 0, v.data_ptr()


def sample_moves(logits: torch.Tensor, noise: torch.Tensor | None, *, legal: torch.Tensor | None = None,
                 temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One move per row: (moves int64 [rows], logprob float32 [rows]).

    noise: uniform numbers on (0, 1), float32 of logits' shape (None only at
    temperature 0); legal: bool or uint8 of that shape. temperature (0: the
    largest logit), top_k (0: off), top_p (1: off) and min_p (0: off) are
    numbers, or tensors of one per row (float32; top_k int32). A row with
    nothing legal gives -1 and -inf. azb_sample_moves states the arithmetic."""
    code, rows, cols, ld = _matrix(logits, "logits")
    device = logits.device
    a = SampleArgs()
    a.logits, a.type, a.rows, a.cols, a.ld = logits.data_ptr(), code, rows, cols, ld
    if noise is not None:
        if noise.dtype != torch.float32 or noise.shape != logits.shape or (cols > 1 and noise.stride(1) != 1):
            raise ValueError("noise: float32 of logits' shape, columns adjacent")
        a.noise, a.noise_ld = noise.data_ptr(), noise.stride(0)
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != logits.shape or (cols > 1 and legal.stride(1) != 1):
            raise ValueError("legal: bool or uint8 of logits' shape, columns adjacent")
        a.legal, a.legal_ld = legal.data_ptr(), legal.stride(0)
    _same_device(device, noise=noise, legal=legal)
    a.temperature, a.temperature_rows = _per_row(temperature, "temperature", rows, device, torch.float32)
    a.top_k, a.top_k_rows = _per_row(top_k, "top_k", rows, device, torch.int32)
    a.top_p, a.top_p_rows = _per_row(top_p, "top_p", rows, device, torch.float32)
    a.min_p, a.min_p_rows = _per_row(min_p, "min_p", rows, device, torch.float32)
    moves = torch.empty(rows, dtype=torch.int64, device=device)
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    a.moves, a.logprob = moves.data_ptr(), logprob.data_ptr()
    e = azb200._err()
    if azb200.lib().azb_sample_moves(device.index, C.byref(a), _stream(device), e, 1024) != 0:
        _fail("azb_sample_moves", e)
    return moves, logprob


def check(device: int = 0) -> None:
    """Waits for the device; raises CudaError if a product kernel's bounded wait ran out since the last check."""
    e = azb200._err()
    if azb200.lib().azb_ops_check(device, e, 1024) != 0:
        raise CudaError(e.value.decode())
