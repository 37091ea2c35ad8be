"""Weights in microscaled 4-bit floating point (MXFP4): quantising rows, reading rows back (also the lookup in an embedding table), and the
contractions of a decoder on such weights.

A number is a sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6); 32 neighbours along a row share a power of two
``2 ** (e - 127)``, ``e`` a byte (255: the block is no number).  ``Mxfp4`` holds a matrix [rows, K], or a stack [X, rows, K]:

* ``data`` uint8 [.., rows, K / 2]: number 2 i of a row in the low half of byte i, number 2 i + 1 in the high half;
* ``scales`` uint8 [.., ceil(rows / 128), ceil(K / 128), 32, 4, 4]: the exponent of block b of row r at
  [r // 128, b // 4, r % 32, r // 32 % 4, b % 4].  Exponents of rows and blocks past the matrix are padding, any byte but 255.

``Mxfp4.from_exponents`` takes exponents row by row, ``exponents`` gives them so.

What a call writes may be any input of the next call on the stream, the weights of another operator included.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from .lib import FG_BF16, FG_F32, KernelError, check, lib, register_signatures, require_cuda

register_signatures("mx", {
    "fg_mxfp4_quantize": [c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p],
    "fg_mxfp4_rows": [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_float, c_void_p],
    "fg_gemm_mxfp4": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_void_p],
    "fg_gemm_mxfp4_ext": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_int, c_int, c_int,
                          c_void_p],
    "fg_gemm_mxfp4_grouped": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int,
                              c_void_p],
    "fg_gemm_mxfp4_both": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_void_p],
    "fg_gemm_mxfp4_both_ext": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p],
    "fg_gemm_mxfp4_error": [],
})

BLOCK = 32
MOST = 2 ** 31 - 1                               # of the launchers' C integers (their own limits are finer)
_CODES = {torch.float32: FG_F32, torch.bfloat16: FG_BF16}


def _scale_shape(rows: int, k: int) -> tuple:
    return (rows + 127) // 128, (k + 127) // 128, 32, 4, 4


class Mxfp4:
    """A matrix [rows, k], or a stack of them, in MXFP4 (layout: the module's text)."""

    __slots__ = ("data", "scales", "rows", "k")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        if data.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise KernelError(f"Mxfp4: data and scales are uint8, got {data.dtype} and {scales.dtype}")
        shape = data.shape
        if len(shape) not in (2, 3):
            raise KernelError(f"Mxfp4: data is [rows, K / 2] or [X, rows, K / 2], got {tuple(shape)}")
        self.rows, self.k = shape[-2], 2 * shape[-1]
        if self.k == 0 or self.k % BLOCK:
            raise KernelError(f"Mxfp4: rows of {self.k} numbers are not whole blocks of {BLOCK}")
        want = (*shape[:-2], *_scale_shape(self.rows, self.k))
        if scales.shape != want:
            raise KernelError(f"Mxfp4: scales of {tuple(shape[:-1])} rows of {self.k} numbers are {want}, got {tuple(scales.shape)}")
        if not data.is_contiguous() or not scales.is_contiguous():
            raise KernelError("Mxfp4: data and scales must be contiguous")
        if data.device != scales.device:
            raise KernelError(f"Mxfp4: data is on {data.device}, scales on {scales.device}")
        self.data, self.scales = data, scales

    @property
    def shape(self) -> tuple:
        return (*self.data.shape[:-1], self.k)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def __getitem__(self, i: int) -> "Mxfp4":
        """Matrix i of a stack."""
        if self.data.dim() != 3:
            raise KernelError("Mxfp4: only a stack of matrices has members")
        return Mxfp4(self.data[i], self.scales[i])

    @classmethod
    def from_exponents(cls, data: torch.Tensor, exponents: torch.Tensor) -> "Mxfp4":
        """From exponents row by row, uint8 [.., rows, K / 32].

        Model files may order a block's sixteen bytes otherwise: where byte j holds number j in its low half and number j + 16 in its high half (GGUF's
        MXFP4 blocks, whose exponent is this one), ``raw`` [.., rows, K / 32, 16] of such bytes becomes ``data`` by

            codes = torch.cat([raw & 15, raw >> 4], -1)
            data = (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(-2)
        """
        rows, k = data.shape[-2], 2 * data.shape[-1]
        if exponents.dtype != torch.uint8 or k % BLOCK or exponents.shape != (*data.shape[:-1], k // BLOCK):
            raise KernelError(f"Mxfp4: exponents are uint8 [.., rows, K / {BLOCK}], got {exponents.dtype} {tuple(exponents.shape)} for data {tuple(data.shape)}")
        lead, n = data.shape[:-2], data.dim() - 2
        tr, tk = _scale_shape(rows, k)[:2]
        full = torch.zeros((*lead, tr * 128, tk * 4), dtype=torch.uint8, device=data.device)
        full[..., :rows, :k // BLOCK] = exponents
        full = full.reshape(*lead, tr, 4, 32, tk, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
        return cls(data.contiguous(), full.contiguous())

    def exponents(self) -> torch.Tensor:
        """The exponents row by row, uint8 [.., rows, K / 32]."""
        n = self.data.dim() - 2
        tr, tk = self.scales.shape[n:n + 2]
        full = self.scales.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*self.data.shape[:n], tr * 128, tk * 4)
        return full[..., :self.rows, :self.k // BLOCK].contiguous()


_launchers: dict = {}
_current_device, _raw_stream = torch.cuda.current_device, getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _launch(name: str, device: int, *args) -> None:
    """Calls a launcher on the tensors' device, whichever is current, and on that device's current stream.  (A small step's time is the host's: what a
    call needs is looked up once.)"""
    fn = _launchers.get(name)
    if fn is None:
        fn = _launchers[name] = getattr(lib("mx"), "fg_" + name)
    if device == _current_device():
        code = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _raw_stream(device))
    check(code, name)


def _on_one_device(what: str, *tensors) -> int:
    """The CUDA device that holds all of the tensors (None: left out)."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != device or device < 0):
            require_cuda(*tensors)
            raise KernelError(f"{what}: tensors on {tensors[0].device} and {t.device}")
    return device


def _too_large(what: str, *sizes: int) -> None:
    """(a size that passes 31 bits would reach the kernels as another one)"""
    raise KernelError(f"{what}: sizes go up to {MOST}, got {max(sizes)}")


def mxfp4_quantize(x: torch.Tensor) -> Mxfp4:
    """x [rows, K] or [X, rows, K], float32 or bfloat16, K a multiple of 32, to MXFP4.

    A block's exponent is the one with which its largest number lies in [4, 8) (at least 2^-127); numbers are rounded to the nearest that the
    format holds, ties to the even code, beyond 6 to 6.  A block that holds an infinity or no number becomes no number as a whole."""
    require_cuda(x)
    code = _CODES.get(x.dtype)
    if code is None:
        raise KernelError(f"mxfp4_quantize: rows are float32 or bfloat16, got {x.dtype}")
    if x.dim() not in (2, 3):
        raise KernelError(f"mxfp4_quantize: x is [rows, K] or [X, rows, K], got {tuple(x.shape)}")
    rows, k = x.shape[-2:]
    if k == 0 or k % BLOCK:
        raise KernelError(f"mxfp4_quantize: rows of {k} numbers are not whole blocks of {BLOCK}")
    if x.stride(-1) != 1:
        raise KernelError("mxfp4_quantize: the numbers of a row must be contiguous")
    lead = x.shape[:-2]
    if rows > MOST or k > MOST or (lead and lead[0] > MOST):
        _too_large("mxfp4_quantize", *x.shape)
    q = Mxfp4.__new__(Mxfp4)                     # (as its constructor would leave it)
    q.rows, q.k = rows, k
    q.data = data = x.new_empty((*lead, rows, k // 2), dtype=torch.uint8)
    q.scales = scales = x.new_empty((*lead, *_scale_shape(rows, k)), dtype=torch.uint8)
    _launch("mxfp4_quantize", x.get_device(), x.data_ptr(), code, x.stride(-2), x.stride(0) if lead else 0, data.data_ptr(), scales.data_ptr(),
            lead[0] if lead else 1, rows, k)
    return q


def mxfp4_rows(w: Mxfp4, rows: Optional[torch.Tensor] = None, *, scale: float = 1.0, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out[i, :] = scale * w[rows[i], :] (without ``rows``: every row), float32 or bfloat16: what the matrix stands for, or the lookup in an
    embedding table.  rows: [n] int32.  A row index outside the matrix gives a row of NaN."""
    device = _on_one_device("mxfp4_rows", w.data, rows, out)
    if w.data.dim() != 2:
        raise KernelError("mxfp4_rows: w is one matrix, not a stack")
    if rows is not None and (rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous()):
        raise KernelError(f"mxfp4_rows: rows must be a contiguous int32 vector, got {rows.dtype} {tuple(rows.shape)}")
    n = w.rows if rows is None else rows.numel()
    if n > MOST or w.rows > MOST or w.k > MOST:
        _too_large("mxfp4_rows", n, w.rows, w.k)
    if out is None:
        out = w.data.new_empty((n, w.k), dtype=out_dtype or torch.float32)
    elif out.shape != (n, w.k) or out.stride(1) != 1 or (n > 1 and out.stride(0) < w.k) or (out_dtype is not None and out.dtype != out_dtype):
        raise KernelError(f"mxfp4_rows: out must be [{n}, {w.k}] with contiguous rows")
    code = _CODES.get(out.dtype)
    if code is None:
        raise KernelError(f"mxfp4_rows: cannot write {out.dtype}")
    _launch("mxfp4_rows", device, w.data.data_ptr(), w.scales.data_ptr(), rows.data_ptr() if rows is not None else None, out.data_ptr(), code,
            max(out.stride(0), w.k), n, w.rows, w.k, scale)
    return out


def _output(what: str, M: int, N: int, K: int, like: torch.Tensor, out, out_dtype, accumulate: bool) -> tuple:
    if M > MOST or N > MOST or K > MOST:
        _too_large(what, M, N, K)
    if out is None:
        if accumulate:
            raise KernelError(f"{what}: accumulate needs the tensor to accumulate into")
        out = like.new_empty((M, N), dtype=out_dtype or torch.bfloat16)
    elif out.shape != (M, N) or out.stride(1) != 1 or (M > 1 and out.stride(0) < N) or (out_dtype is not None and out.dtype != out_dtype):
        raise KernelError(f"{what}: out must be [{M}, {N}] with contiguous rows")
    code = _CODES.get(out.dtype)
    if code is None:
        raise KernelError(f"{what}: cannot write {out.dtype}")
    if accumulate and code != FG_F32:
        raise KernelError(f"{what}: the residual sum is 32-bit; accumulate needs a float32 output")
    return out, code


def _activations(what: str, x: torch.Tensor, k: int) -> None:
    if x.dtype != torch.bfloat16:
        raise KernelError(f"{what}: activations are bfloat16, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] != k:
        raise KernelError(f"{what}: activations are [rows, {k}], got {tuple(x.shape)}")
    if x.stride(1) != 1:
        raise KernelError(f"{what}: the reduction dimension must be contiguous")


def gemm_mxfp4(x: torch.Tensor, w: Mxfp4, *, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               accumulate: bool = False) -> torch.Tensor:
    """out[m, n] (+)= sum_k x[m, k] w[n, k]: bfloat16 activations [M, K] on a matrix [N, K] in MXFP4, float32 sums.  Output bfloat16 (default) or
    float32; ``accumulate`` adds into a float32 ``out``."""
    data = w.data
    device = _on_one_device("gemm_mxfp4", x, data, out)
    if data.dim() != 2:
        raise KernelError("gemm_mxfp4: w is one matrix, not a stack (see gemm_mxfp4_grouped)")
    _activations("gemm_mxfp4", x, w.k)
    M = x.shape[0]
    out, code = _output("gemm_mxfp4", M, w.rows, w.k, data, out, out_dtype, accumulate)
    _launch("gemm_mxfp4", device, x.data_ptr(), x.stride(0), data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), code, out.stride(0),
            accumulate, M, w.rows, w.k)
    return out


def gemm_mxfp4_both(x: Mxfp4, w: Mxfp4, *, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                    accumulate: bool = False) -> torch.Tensor:
    """The same with the activations [M, K] in MXFP4 too (``mxfp4_quantize``)."""
    device = _on_one_device("gemm_mxfp4_both", x.data, w.data, out)
    if w.data.dim() != 2 or x.data.dim() != 2:
        raise KernelError("gemm_mxfp4_both: x and w are one matrix each, not stacks")
    if x.k != w.k:
        raise KernelError(f"gemm_mxfp4_both: x is {x.shape} but w is {w.shape}")
    M = x.rows
    out, code = _output("gemm_mxfp4_both", M, w.rows, w.k, w.data, out, out_dtype, accumulate)
    _launch("gemm_mxfp4_both", device, x.data.data_ptr(), x.scales.data_ptr(), w.data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), code,
            out.stride(0), accumulate, M, w.rows, w.k)
    return out


def gemm_mxfp4_grouped(x: torch.Tensor, w: Mxfp4, offsets: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                       out_dtype: Optional[torch.dtype] = None, accumulate: bool = False) -> torch.Tensor:
    """Rows grouped by expert: out[m, n] (+)= sum_k x[m, k] w[e, n, k] for the rows offsets[e] <= m < offsets[e + 1] of expert e.

    x: [M, K] bfloat16; w: a stack [X, N, K]; offsets: [X + 1] int32 on the device, rising from the first row.  Runs may be empty.  Rows of no
    run (before the first offset, behind the last) are not written: they keep what ``out`` held, which is undefined without an ``out``."""
    device = _on_one_device("gemm_mxfp4_grouped", x, w.data, offsets, out)
    if w.data.dim() != 3:
        raise KernelError("gemm_mxfp4_grouped: w is a stack of matrices")
    X = w.data.shape[0]
    if offsets.dtype != torch.int32 or offsets.shape != (X + 1,) or not offsets.is_contiguous():
        raise KernelError(f"gemm_mxfp4_grouped: offsets must be contiguous int32 [{X + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    _activations("gemm_mxfp4_grouped", x, w.k)
    M = x.shape[0]
    out, code = _output("gemm_mxfp4_grouped", M, w.rows, w.k, w.data, out, out_dtype, accumulate)
    _launch("gemm_mxfp4_grouped", device, x.data_ptr(), x.stride(0), w.data.data_ptr(), w.scales.data_ptr(), offsets.data_ptr(), X, out.data_ptr(),
            code, out.stride(0), accumulate, M, w.rows, w.k)
    return out
