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
backward pass: an argument that requires a gradient or carries a forward-mode
tangent is refused, and so are a negated view, a tensor that stands for others
and a call under a trace (the calls run below torch's dispatcher). Bad
arguments raise ValueError, failures of the device azb200.CudaError.

The calls go through _azb_torch.so (binding/azb_torch.cpp); importing this
module fails loudly when it is missing.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch

import azb200
from azb200 import CudaError

_BINDING = os.path.join(azb200.HERE, "_azb_torch.so")
if not os.path.exists(_BINDING):
    raise RuntimeError(f"{_BINDING} is not built: run `python {os.path.join(azb200.HERE, 'build_ext.py')}`")
azb200.lib()   # the engine's library, which the binding links against
_spec = importlib.util.spec_from_file_location("_azb_torch", _BINDING,
                                               loader=importlib.machinery.ExtensionFileLoader("_azb_torch", _BINDING))
_T = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_T)

_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _type(dtype) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"dtype: float32 or bfloat16, not {dtype}")
    return code


class Mx4:
    """A rows x cols matrix in the 4-bit microscaled form, as azb_mx4_quantise
    lays it out, in one allocation: `codes` (uint8 [rows, 16 * ceil(cols /
    32)]), then `scales` (uint8, in the tensor core's tile order). Mx4(codes,
    scales, rows, cols) holds a copy of given ones."""

    __slots__ = ("data", "rows", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        need, got = _sizes(rows, cols), (codes.numel(), scales.numel())
        if need != got or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"Mx4 of {rows} x {cols}: {need} bytes of codes and scales, not {got}")
        if not codes.is_cuda or codes.device != scales.device:
            raise ValueError("Mx4: codes and scales must be on one GPU")
        self.rows, self.cols = rows, cols
        self.data = codes.new_empty(-(-need[0] // 256) * 256 + need[1])
        self.codes.copy_(codes.view(self.codes.shape))
        self.scales.copy_(scales.flatten())

    @property
    def codes(self) -> torch.Tensor:
        blocks = -(-self.cols // 32)
        return self.data[:self.rows * blocks * 16].view(self.rows, blocks * 16)

    @property
    def scales(self) -> torch.Tensor:
        return self.data[self.data.numel() - _sizes(self.rows, self.cols)[1]:]

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.cols)

    def pointers(self) -> tuple[int, int]:
        """The device addresses of codes and scales, for the C ABI."""
        return self.data.data_ptr(), self.scales.data_ptr()

    def nbytes(self) -> int:
        return sum(_sizes(self.rows, self.cols))


def _sizes(rows: int, cols: int) -> tuple[int, int]:
    """azb_mx4_sizes."""
    blocks = -(-cols // 32)
    return rows * blocks * 16, -(-rows // 128) * -(-blocks // 4) * 512


def mx4_quantise(x: torch.Tensor) -> Mx4:
    """The 4-bit microscaled form of a matrix."""
    q = Mx4.__new__(Mx4)
    q.data, q.rows, q.cols = _T.mx4_quantise(x)
    return q


def mx4_values(q: Mx4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values q holds; exact in either type."""
    return _T.mx4_values(q.data, q.rows, q.cols, _type(dtype))


def mx4_product(x, w: Mx4, *, bias: torch.Tensor | None = None, relu: bool = False,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(x . w^T + bias) with both factors in the 4-bit form, summed in
    fp32 and rounded once to `dtype` (default: x's, float32 for an Mx4). x: an
    Mx4, or a matrix or vector that is quantised on the way."""
    if type(w) is not Mx4:
        raise ValueError("w: an Mx4 is needed (mx4_quantise)")
    code = -1 if dtype is None else _type(dtype)
    if type(x) is Mx4:
        return _T.mx4_product(x.data, x.rows, x.cols, w.data, w.rows, w.cols, bias, relu, code)
    return _T.mx4_product(x, -1, 0, w.data, w.rows, w.cols, bias, relu, code)


def sample_moves(logits: torch.Tensor, noise: torch.Tensor | None, *, legal: torch.Tensor | None = None,
                 temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One move per row: (moves int64 [rows], logprob float32 [rows]).

    noise: uniform numbers on (0, 1), float32 of logits' shape (None only at
    temperature 0); legal: bool or uint8 of that shape. temperature (0: the
    largest logit), top_k (0: off), top_p (1: off) and min_p (0: off) are
    numbers, or tensors of one per row (float32; top_k int32). A row with
    nothing legal gives -1 and -inf. azb_sample_moves states the arithmetic."""
    return _T.sample_moves(logits, noise, legal, temperature, top_k, top_p, min_p)


def check(device: int = 0) -> None:
    """Waits for the device; raises CudaError if a product kernel's bounded wait ever ran out on it (and again in every
    later call: that product's outputs are not valid, whoever's they were)."""
    e = azb200._err()
    if azb200.lib().azb_ops_check(device, e, 1024) != 0:
        raise CudaError(e.value.decode())
