"""The 8-bit operators on torch CUDA tensors (kk_fp8_* of include/kokoro_b200.h): rows and weights held
as e4m3 values with a power-of-two scale for each block of 128, and the linear layer over them.

    q = fp8.quantize(x)                       # activations: a scale per 128 columns of each row
    w = fp8.quantize(weight, block_rows=128)  # weights: a scale per 128 x 128 block
    y = fp8.linear(q, w, bias, act="gelu")    # act(x W^T + bias) + residual
    x2 = fp8.dequantize(q)

Calls enqueue on the current stream of their tensors' device and allocate only their results (give
``out`` to have none); they may be captured into a CUDA graph. Tensors made or last used on another
stream are the caller's to order, as for any torch operator. There is no gradient: a tensor that
requires one is refused while gradients are being recorded. ``KokoroError`` carries the status of a
refused call.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .engine import KK_ERR_INVALID_ARG, KK_OK, KokoroError, load_library

E4M3 = torch.float8_e4m3fn
_TYPES = {torch.float32: 0, torch.bfloat16: 1, E4M3: 2}  # kk_fp8_type
_ACTS = {None: 0, "gelu": 1}  # kk_fp8_act


def _refuse(msg: str):
    raise KokoroError(KK_ERR_INVALID_ARG, msg)


def _ld(t: torch.Tensor, unit: int = 1) -> int:
    """Row stride; a single row's is whatever holds its columns."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // unit) * unit


def _check_rows(t: torch.Tensor, name: str, dtypes) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _refuse(f"{name}: a tensor of {' or '.join(str(d) for d in dtypes)} is wanted")
    if t.dim() != 2:
        _refuse(f"{name}: rows are wanted, [rows, columns]")
    if t.shape[1] > 1 and t.stride(1) != 1:
        _refuse(f"{name}: a row's columns must be adjacent")
    if not t.is_cuda:
        _refuse(f"{name}: a CUDA tensor is wanted")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name}: the 8-bit operators have no gradient")


class Fp8Tensor:
    """A store of ``rows`` x ``k`` values: ``values`` (float8_e4m3fn [rows, k], rows a multiple of 16
    bytes apart) and ``exps`` (uint8 [ceil(rows / block_rows), ceil(k / 128)], rows a multiple of 4
    bytes apart): a block stands for value * 2^(E - 127). block_rows is 1 (activations) or 128 (weights)."""

    __slots__ = ("values", "exps", "block_rows")

    def __init__(self, values: torch.Tensor, exps: torch.Tensor, block_rows: int = 1):
        _check_rows(values, "values", (E4M3,))
        _check_rows(exps, "exps", (torch.uint8,))
        if block_rows not in (1, 128):
            _refuse("block_rows must be 1 or 128")
        rows, k = values.shape
        if exps.shape[0] != -(-rows // block_rows) or exps.shape[1] != -(-k // 128):
            _refuse(f"exps: [{-(-rows // block_rows)}, {-(-k // 128)}] is wanted for values [{rows}, {k}]")
        if exps.device != values.device:
            _refuse("values and exps must be on one device")
        self.values, self.exps, self.block_rows = values, exps, block_rows

    @classmethod
    def empty(cls, rows: int, k: int, block_rows: int = 1, device="cuda") -> "Fp8Tensor":
        """A store with its rows padded to the alignment that the operators want; not initialised."""
        kb = -(-k // 128)
        v = torch.empty(rows, -(-k // 16) * 16, dtype=E4M3, device=device)
        e = torch.empty(-(-rows // block_rows) if block_rows in (1, 128) else 0, -(-kb // 4) * 4, dtype=torch.uint8,
                        device=device)
        return cls(v[:, :k], e[:, :kb], block_rows)

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def __getitem__(self, rows: slice) -> "Fp8Tensor":
        """A view of some of an activation store's rows (to read them, or to quantise into them)."""
        if not isinstance(rows, slice) or self.block_rows != 1:
            _refuse("a store is cut by a slice of rows, and only with block_rows 1")
        return Fp8Tensor(self.values[rows], self.exps[rows])

    def _args(self):
        v, e = self.values, self.exps
        return v.data_ptr(), _ld(v, 16), e.data_ptr(), _ld(e, 4)


def _run(status: int) -> None:
    if status != KK_OK:
        raise KokoroError(status, load_library().kk_fp8_error().decode())


def _same_device(dev: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != dev:
            _refuse(f"tensors on {dev} and {t.device}: one device is wanted")


def quantize(x: torch.Tensor, block_rows: int = 1, out: Optional[Fp8Tensor] = None) -> Fp8Tensor:
    """x [rows, k] (float32 or bfloat16) as a store; into ``out`` when given (its other rows are left)."""
    _check_rows(x, "x", (torch.float32, torch.bfloat16))
    if out is None:
        out = Fp8Tensor.empty(x.shape[0], x.shape[1], block_rows, x.device)
    elif not isinstance(out, Fp8Tensor) or out.shape != x.shape or out.block_rows != block_rows:
        _refuse("out: a store of x's shape and of the same block_rows is wanted")
    dev = x.device
    _same_device(dev, out.values)
    _run(load_library().kk_fp8_quantize(dev.index, torch.cuda.current_stream(dev).cuda_stream, x.data_ptr(),
                                        _TYPES[x.dtype], x.shape[0], x.shape[1], _ld(x), block_rows, *out._args()))
    return out


def dequantize(q: Fp8Tensor, dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that a store stands for, as ``dtype`` (float32 or bfloat16; both hold them exactly,
    but for bfloat16 below its normal numbers)."""
    if not isinstance(q, Fp8Tensor):
        _refuse("q: a store is wanted")
    if out is None:
        if dtype not in (torch.float32, torch.bfloat16):
            _refuse("dtype: float32 or bfloat16 is wanted")
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
    else:
        _check_rows(out, "out", (dtype,) if dtype in (torch.float32, torch.bfloat16) else (torch.float32,))
        if out.shape != q.shape:
            _refuse("out: the store's shape is wanted")
    dev = q.device
    _same_device(dev, out)
    _run(load_library().kk_fp8_dequantize(dev.index, torch.cuda.current_stream(dev).cuda_stream, *q._args(),
                                          q.block_rows, q.shape[0], q.shape[1], out.data_ptr(), _TYPES[out.dtype],
                                          _ld(out)))
    return out


def linear(x: Fp8Tensor, w: Fp8Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
           out: Union[torch.Tensor, Fp8Tensor, None] = None) -> Union[torch.Tensor, Fp8Tensor]:
    """act(x w^T + bias) + residual: x [m, k] a store with block_rows 1, w [n, k] one with block_rows
    128, bias float32 [n], act None or "gelu" (the tanh form). The result is float32, bfloat16 (with a
    residual of the same type, which may be ``out`` itself), or with float8_e4m3fn a store that the next
    layer reads (without a residual)."""
    if not isinstance(x, Fp8Tensor) or x.block_rows != 1:
        _refuse("x: a store with block_rows 1 is wanted")
    if not isinstance(w, Fp8Tensor) or w.block_rows != 128:
        _refuse("w: a store with block_rows 128 is wanted")
    m, k = x.values.shape
    n = w.values.shape[0]
    if w.values.shape[1] != k:
        _refuse(f"x has {k} columns and w {w.values.shape[1]}")
    if act not in _ACTS:
        _refuse("act: None or 'gelu' is wanted")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            _refuse(f"bias: adjacent float32 [{n}] is wanted")
        if bias.requires_grad and torch.is_grad_enabled():
            _refuse("bias: the 8-bit operators have no gradient")
    dev = x.values.device
    if out is None:
        if out_dtype == E4M3:
            out = Fp8Tensor.empty(m, n, 1, dev)
        elif out_dtype in (torch.float32, torch.bfloat16):
            out = torch.empty((m, n), dtype=out_dtype, device=dev)
        else:
            _refuse("out_dtype: float32, bfloat16 or float8_e4m3fn is wanted")
    if isinstance(out, Fp8Tensor):
        if out.block_rows != 1 or out.shape != (m, n) or out_dtype != E4M3:
            _refuse(f"out: a store [{m}, {n}] with block_rows 1 goes with out_dtype float8_e4m3fn")
        if residual is not None:
            _refuse("an e4m3 result takes no residual")
        y_type, y = 2, out._args()
        _same_device(dev, w.values, bias, out.values)
        r = (None, 0)
    else:
        _check_rows(out, "out", (out_dtype,) if out_dtype in (torch.float32, torch.bfloat16) else ())
        if out.shape != (m, n):
            _refuse(f"out: [{m}, {n}] is wanted")
        y_type, y = _TYPES[out_dtype], (out.data_ptr(), _ld(out), None, 0)
        _same_device(dev, w.values, bias, out, residual)
        r = (None, 0)
        if residual is not None:
            _check_rows(residual, "residual", (out_dtype,))
            if residual.shape != (m, n):
                _refuse(f"residual: [{m}, {n}] is wanted")
            r = (residual.data_ptr(), _ld(residual))
    _run(load_library().kk_fp8_linear(dev.index, torch.cuda.current_stream(dev).cuda_stream, m, n, k, *x._args(),
                                      *w._args(), None if bias is None else bias.data_ptr(), _ACTS[act], *r, y_type,
                                      *y))
    return out


def check(device=None) -> None:
    """Waits for the current stream and raises if a bounded in-kernel wait of a linear layer on this
    device gave up since the last check (its results are then not valid)."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    idx = torch.cuda.current_device() if dev.index is None else dev.index
    _run(load_library().kk_fp8_check(idx, torch.cuda.current_stream(idx).cuda_stream))
