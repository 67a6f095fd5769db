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

import functools
import struct

import torch

import azb200
from azb200 import CudaError

# azb_sample_args (azb200.SampleArgs), packed in one step.
_SAMPLE_ARGS = struct.Struct("@PiqqqPqPqfffiPPPPPP")
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


_stream = torch._C._cuda_getCurrentRawStream   # of a device index: its current stream's handle


def _empty(rows: int, cols: int, dtype, device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


class Mx4:
    """A rows x cols matrix in the 4-bit microscaled form, as azb_mx4_quantise
    lays it out: `codes` (uint8 [rows, 16 * ceil(cols / 32)]) and `scales`
    (uint8, in the tensor core's tile order) in one allocation. Mx4(codes,
    scales, rows, cols) takes existing ones."""

    __slots__ = ("_data", "_split", "_scales", "rows", "cols", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        need, got = _sizes(rows, cols), (codes.numel(), scales.numel())
        if need != got or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"Mx4 of {rows} x {cols}: {need} bytes of codes and scales, not {got}")
        if not (codes.is_cuda and codes.is_contiguous() and scales.is_contiguous() and codes.device == scales.device):
            raise ValueError("Mx4: codes and scales must be contiguous and on one GPU")
        self._data, self._split, self._scales = codes, need[0], scales
        self.rows, self.cols, self.device = rows, cols, codes.device

    @property
    def codes(self) -> torch.Tensor:
        return self._data.flatten()[:self._split].view(self.rows, -1 if self.rows else 0)

    @property
    def scales(self) -> torch.Tensor:
        return self._scales if self._scales is not None else self._data[-(-self._split // 256) * 256:]

    def pointers(self) -> tuple[int, int]:
        p = self._data.data_ptr()
        return p, (p + -(-self._split // 256) * 256 if self._scales is None else self._scales.data_ptr())

    @property
    def shape(self):
        return (self.rows, self.cols)

    def nbytes(self) -> int:
        return sum(_sizes(self.rows, self.cols))


def _sizes(rows: int, cols: int) -> tuple[int, int]:
    """azb_mx4_sizes."""
    blocks = -(-cols // 32)
    return rows * blocks * 16, -(-rows // 128) * -(-blocks // 4) * 512


@functools.lru_cache(maxsize=4096)
def _workspace(m: int, n: int, k: int) -> int:
    return azb200.lib().azb_mx4_linear_workspace(m, n, k)


def mx4_quantise(x: torch.Tensor) -> Mx4:
    """The 4-bit microscaled form of a matrix."""
    code, rows, cols, ld = _matrix(x, "x")
    device = x.device
    index, e = device.index, azb200._err()
    blocks = -(-cols // 32)
    nc = rows * blocks * 16
    at = -(-nc // 256) * 256   # the scales' place
    q = object.__new__(Mx4)
    q.rows, q.cols, q.device, q._split, q._scales = rows, cols, device, nc, None
    q._data = data = torch.empty_strided((at + -(-rows // 128) * -(-blocks // 4) * 512,), (1,), dtype=torch.uint8,
                                         device=device)
    p = data.data_ptr()
    if azb200.lib().azb_mx4_quantise(index, x.data_ptr(), code, rows, cols, ld, p, p + at, _stream(index), e, 1024) != 0:
        _fail("azb_mx4_quantise", e)
    return q


def mx4_values(q: Mx4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values q holds; exact in either type."""
    code = _type(dtype, "dtype")
    device, rows, cols = q.device, q.rows, q.cols
    out = _empty(rows, cols, dtype, device)
    e = azb200._err()
    if azb200.lib().azb_mx4_values(device.index, *q.pointers(), rows, cols, out.data_ptr(), code, cols,
                                   _stream(device.index), e, 1024) != 0:
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
    if w.device != device or (bias is not None and bias.device != device):
        raise ValueError(f"x is on {device}, w on {w.device}" + (f", bias on {bias.device}" if bias is not None else ""))
    n = w.rows
    out = _empty(m, n, dtype, device)
    L, e = azb200.lib(), azb200._err()
    b = None if bias is None else bias.data_ptr()
    if quantised:
        rc = L.azb_mx4_product(device.index, *x.pointers(), m, *w.pointers(), n, k, b, relu, out.data_ptr(), code, n,
                               _stream(device.index), e, 1024)
    else:
        need, ws = _workspace(m, n, k), None
        if need:
            ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device)
        rc = L.azb_mx4_linear(device.index, x.data_ptr(), x_type, m, k, x_ld, *w.pointers(), n, b, relu,
                              out.data_ptr(), code, n, ws.data_ptr() if ws is not None else None, need,
                              _stream(device.index), e, 1024)
    if rc != 0:
        _fail("azb_mx4_product", e)
    return out[0] if vector else out


def _per_row(v, name: str, rows: int, device, dtype):
    """(number, pointer) of a setting: one number, or one per row."""
    if not isinstance(v, torch.Tensor):
        return v, 0
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
    n_at = n_ld = l_at = l_ld = 0
    if noise is not None:
        if noise.dtype != torch.float32 or noise.shape != logits.shape:
            raise ValueError("noise: float32 of logits' shape is needed")
        n_at, (n_ld, inner) = noise.data_ptr(), noise.stride()
        if (inner != 1 and cols > 1) or noise.device != device:
            raise ValueError(f"noise: adjacent columns on {device} are needed (stride {inner}; it is on {noise.device})")
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != logits.shape:
            raise ValueError("legal: bool or uint8 of logits' shape is needed")
        l_at, (l_ld, inner) = legal.data_ptr(), legal.stride()
        if (inner != 1 and cols > 1) or legal.device != device:
            raise ValueError(f"legal: adjacent columns on {device} are needed (stride {inner}; it is on {legal.device})")
    temperature, t_at = _per_row(temperature, "temperature", rows, device, torch.float32)
    top_k, k_at = _per_row(top_k, "top_k", rows, device, torch.int32)
    top_p, p_at = _per_row(top_p, "top_p", rows, device, torch.float32)
    min_p, m_at = _per_row(min_p, "min_p", rows, device, torch.float32)
    moves = torch.empty_strided((rows,), (1,), dtype=torch.int64, device=device)
    logprob = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device)
    args = _SAMPLE_ARGS.pack(logits.data_ptr(), code, rows, cols, ld, n_at, n_ld, l_at, l_ld, temperature, top_p, min_p,
                             top_k, t_at, p_at, m_at, k_at, moves.data_ptr(), logprob.data_ptr())
    index, e = device.index, azb200._err()
    if azb200.lib().azb_sample_moves(index, args, _stream(index), e, 1024) != 0:
        _fail("azb_sample_moves", e)
    return moves, logprob


def check(device: int = 0) -> None:
    """Waits for the device; raises CudaError if a product kernel's bounded wait ran out since the last check."""
    e = azb200._err()
    if azb200.lib().azb_ops_check(device, e, 1024) != 0:
        raise CudaError(e.value.decode())
