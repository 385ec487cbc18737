"""The 8-bit operators on torch CUDA tensors (kk_fp8_* of include/kokoro_b200.h): rows and weights held
as e4m3 values with a power-of-two scale for each block of 128, and the linear layer over them.

    q = fp8.quantize(x)                       # activations: a scale per 128 columns of each row
    w = fp8.quantize(weight, block_rows=128)  # weights: a scale per 128 x 128 block
    y = fp8.linear(q, w, bias, act="gelu")    # act(x W^T + bias) + residual
    x2 = fp8.dequantize(q)

Calls enqueue on the current stream of their tensors' device and allocate only their results (give
``out`` to have none); they may be captured into a CUDA graph. Tensors made or last used on another
stream are the caller's to order, as for any torch operator. There is no gradient: a tensor that
requires one is refused while gradients are being recorded, and so is one with a forward-mode tangent.
``KokoroError`` carries the status of a refused call.
"""
from __future__ import annotations

import struct
from typing import Optional, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .engine import KK_ERR_INVALID_ARG, KokoroError, load_library

E4M3 = torch.float8_e4m3fn
_F32, _BF16 = torch.float32, torch.bfloat16
_TYPES = {_F32: 0, _BF16: 1, E4M3: 2}  # kk_fp8_type
_ACTS = {None: 0, "gelu": 1}  # kk_fp8_act


def _refuse(msg: str):
    raise KokoroError(KK_ERR_INVALID_ARG, msg)


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the current stream's handle without the object around it, where torch offers that (2 us of a small call)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _no_gradient(t: torch.Tensor, name: str):
    """For a tensor that requires a gradient, or while a dual level is open (tangents live inside one; -1 is outside of all):
    asked for beforehand, which is 0.03 us where unpacking is 0.5."""
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name}: the 8-bit operators have no gradient")
    if forward_ad.unpack_dual(t).tangent is not None:
        _refuse(f"{name}: the 8-bit operators have no gradient, in forward mode either")


def _rows(t: torch.Tensor, name: str, dtypes, unit: int = 1):
    """(rows, columns, row stride) of a CUDA tensor of rows whose columns are adjacent; a single row's
    stride is whatever holds its columns."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _refuse(f"{name}: a tensor of {' or '.join(str(d) for d in dtypes)} is wanted")
    shape = t.shape
    if len(shape) != 2:
        _refuse(f"{name}: rows are wanted, [rows, columns]")
    rows, k = shape
    ld, inner = t.stride()
    if inner != 1 and k > 1:
        _refuse(f"{name}: a row's columns must be adjacent")
    if k == 1 and t.is_neg():  # (the imaginary part of a conjugate, whose columns are never adjacent)
        _refuse(f"{name}: its negation is still to be done (resolve_neg)")
    if t.requires_grad or forward_ad._current_level >= 0:
        _no_gradient(t, name)
    if not t.is_cuda:
        _refuse(f"{name}: a CUDA tensor is wanted")
    return rows, k, ld if rows > 1 else -(-k // unit) * unit


class Fp8Tensor:
    """A store of ``rows`` x ``k`` values: ``values`` (float8_e4m3fn [rows, k], rows a multiple of 16
    bytes apart) and ``exps`` (uint8 [ceil(rows / block_rows), ceil(k / 128)], rows a multiple of 4
    bytes apart): a block stands for value * 2^(E - 127). block_rows is 1 (activations) or 128 (weights).
    It is a view of the tensors' memory and keeps it, but not over a storage's own ``resize_``."""

    __slots__ = ("shape", "block_rows", "device", "_values", "_exps", "_buf", "_args")

    def __init__(self, values: torch.Tensor, exps: torch.Tensor, block_rows: int = 1):
        rows, k, ldv = _rows(values, "values", (E4M3,), 16)
        erows, kb, lde = _rows(exps, "exps", (torch.uint8,), 4)
        if block_rows != 1 and block_rows != 128:
            _refuse("block_rows must be 1 or 128")
        if erows != -(-rows // block_rows) or kb != -(-k // 128):
            _refuse(f"exps: [{-(-rows // block_rows)}, {-(-k // 128)}] is wanted for values [{rows}, {k}]")
        self.device = values.device
        if exps.device != self.device:
            _refuse("values and exps must be on one device")
        self.shape, self.block_rows, self._values, self._exps = values.shape, block_rows, values, exps
        # the memory that the calls are given stays, whatever becomes of the two tensors (set_, .data)
        self._buf = values.untyped_storage(), exps.untyped_storage()
        self._args = (values.data_ptr(), ldv, exps.data_ptr(), lde)

    @classmethod
    def empty(cls, rows: int, k: int, block_rows: int = 1, device="cuda") -> "Fp8Tensor":
        """A store with its rows padded to the alignment that the operators want (or do best with); not initialised."""
        if block_rows != 1 and block_rows != 128:
            _refuse("block_rows must be 1 or 128")
        if rows < 0 or k < 0:
            _refuse("rows and columns must not be negative")
        # Rows of values begin on the largest of 128, 64 or 32 bytes that pads them by at most an eighth: L2 gives whole
        # sectors of 32 (33,104 x 770 -> 2304: 81 us in rows of 784 bytes, 69 in 800, 66 in 832, 64 in 896).
        ldv, lde = -(-k // 16) * 16, -(-k // 512) * 4
        for unit in (128, 64, 32):
            if -k % unit * 8 <= k:
                ldv = -(-k // unit) * unit
                break
        self = cls.__new__(cls)
        # one allocation: the values, then the exponents; the views are made when they are asked for
        self._buf = torch.empty(rows * ldv + -(-rows // block_rows) * lde, dtype=torch.uint8, device=device)
        if not self._buf.is_cuda:
            _refuse("a store is held on a CUDA device")
        at = self._buf.data_ptr()
        self.shape, self.block_rows, self.device = torch.Size((rows, k)), block_rows, self._buf.device
        self._values = self._exps = None
        self._args = (at, ldv, at + rows * ldv, lde)
        return self

    @property
    def values(self) -> torch.Tensor:
        if self._values is None:
            self._values = self._buf.view(E4M3).as_strided(self.shape, (self._args[1], 1))
        return self._values

    @property
    def exps(self) -> torch.Tensor:
        if self._exps is None:
            (rows, k), (_, ldv, _, lde) = self.shape, self._args
            self._exps = self._buf.as_strided((-(-rows // self.block_rows), -(-k // 128)), (lde, 1), rows * ldv)
        return self._exps

    def __reduce__(self):  # a copy (copy.deepcopy, torch.save) is a store over copied tensors, with addresses of its own
        return Fp8Tensor, (self.values, self.exps, self.block_rows)

    def __getitem__(self, rows: slice) -> "Fp8Tensor":
        """A view of some of an activation store's rows (to read them, or to quantise into them)."""
        if not isinstance(rows, slice) or self.block_rows != 1:
            _refuse("a store is cut by a slice of rows, and only with block_rows 1")
        return Fp8Tensor(self.values[rows], self.exps[rows])


# the arguments of the C calls, packed (kk_fp8_call)
_args12, _args22 = struct.Struct("12q").pack, struct.Struct("22q").pack


def _run(status: int) -> None:
    if status != 0:
        raise KokoroError(status, load_library().kk_fp8_error().decode())


def _one_device(dev: torch.device, other: torch.device) -> None:
    if other != dev:
        _refuse(f"tensors on {dev} and {other}: one device is wanted")


def quantize(x: torch.Tensor, block_rows: int = 1, out: Optional[Fp8Tensor] = None) -> Fp8Tensor:
    """x [rows, k] (float32 or bfloat16) as a store; into ``out`` when given (its other rows are left)."""
    rows, k, ld = _rows(x, "x", (_F32, _BF16))
    dev = x.device
    if out is None:
        out = Fp8Tensor.empty(rows, k, block_rows, dev)
    elif not isinstance(out, Fp8Tensor) or out.shape != x.shape or out.block_rows != block_rows:
        _refuse("out: a store of x's shape and of the same block_rows is wanted")
    elif out.device != dev:
        _one_device(dev, out.device)
    _run(load_library().kk_fp8_call(0, _args12(dev.index, _stream(dev.index), x.data_ptr(), _TYPES[x.dtype], rows, k, ld,
                                               block_rows, *out._args), 12))
    return out


def dequantize(q: Fp8Tensor, dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that a store stands for, as ``dtype`` (float32 or bfloat16; both hold them exactly,
    but for bfloat16 below its normal numbers, and for 2^128, which magnitudes from 3.2965e38 on are held as
    and which reads back as infinity)."""
    if not isinstance(q, Fp8Tensor):
        _refuse("q: a store is wanted")
    if dtype is not _F32 and dtype is not _BF16:
        _refuse("dtype: float32 or bfloat16 is wanted")
    (rows, k), dev = q.shape, q.device
    if out is None:
        out, ld = torch.empty(rows, k, dtype=dtype, device=dev), k
    else:
        ld = _rows(out, "out", (dtype,))[2]
        if out.shape != q.shape:
            _refuse("out: the store's shape is wanted")
        _one_device(dev, out.device)
        increment_version(out)  # (a backward pass that saved it says so, as for any operator in place)
    _run(load_library().kk_fp8_call(1, _args12(dev.index, _stream(dev.index), *q._args, q.block_rows, rows, k,
                                               out.data_ptr(), _TYPES[dtype], ld), 12))
    return out


def linear(x: Fp8Tensor, w: Fp8Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
           out: Union[torch.Tensor, Fp8Tensor, None] = None) -> Union[torch.Tensor, Fp8Tensor]:
    """act(x w^T + bias) + residual: x [m, k] a store with block_rows 1, w [n, k] one with block_rows
    128, bias float32 [n], act None or "gelu" (the tanh form). The result is float32, bfloat16 (with a
    residual of the same type, which may be ``out`` itself or not overlap it), or with float8_e4m3fn a store that the next
    layer reads (without a residual). ``out`` may not overlap x, w or bias."""
    if not isinstance(x, Fp8Tensor) or x.block_rows != 1:
        _refuse("x: a store with block_rows 1 is wanted")
    if not isinstance(w, Fp8Tensor) or w.block_rows != 128:
        _refuse("w: a store with block_rows 128 is wanted")
    m, k = x.shape
    n, kw = w.shape
    if kw != k:
        _refuse(f"x has {k} columns and w {kw}")
    if act not in _ACTS:
        _refuse("act: None or 'gelu' is wanted")
    if out_dtype not in _TYPES:
        _refuse("out_dtype: float32, bfloat16 or float8_e4m3fn is wanted")
    dev = x.device
    if w.device != dev:
        _one_device(dev, w.device)
    b = 0
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype is not _F32 or bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            _refuse(f"bias: adjacent float32 [{n}] is wanted")
        if bias.requires_grad or forward_ad._current_level >= 0:
            _no_gradient(bias, "bias")
        if n == 1 and bias.is_neg():
            _refuse("bias: its negation is still to be done (resolve_neg)")
        if bias.device != dev:
            _one_device(dev, bias.device)
        b = bias.data_ptr()
    res, ldr = 0, 0
    if residual is not None:
        if out_dtype is E4M3:
            _refuse("an e4m3 result takes no residual")
        ldr = _rows(residual, "residual", (out_dtype,))[2]
        if residual.shape != (m, n):
            _refuse(f"residual: [{m}, {n}] is wanted")
        if residual.device != dev:
            _one_device(dev, residual.device)
        res = residual.data_ptr()
    if out_dtype is E4M3:
        if out is None:
            out = Fp8Tensor.empty(m, n, 1, dev)
        elif not isinstance(out, Fp8Tensor) or out.block_rows != 1 or out.shape != (m, n):
            _refuse(f"out: a store [{m}, {n}] with block_rows 1 is wanted")
        elif out.device != dev:
            _one_device(dev, out.device)
        y = out._args
    elif out is None:
        out = torch.empty(m, n, dtype=out_dtype, device=dev)
        y = (out.data_ptr(), n, 0, 0)
    else:
        ldy = _rows(out, "out", (out_dtype,))[2]
        if out.shape != (m, n):
            _refuse(f"out: [{m}, {n}] is wanted")
        if out.device != dev:
            _one_device(dev, out.device)
        increment_version(out)
        y = (out.data_ptr(), ldy, 0, 0)
    _run(load_library().kk_fp8_call(2, _args22(dev.index, _stream(dev.index), m, n, k, *x._args, *w._args, b, _ACTS[act],
                                               res, ldr, _TYPES[out_dtype], *y), 22))
    return out


def _current(device):
    """(ordinal, handle of the current stream) of a CUDA device."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    if dev.type != "cuda":
        _refuse(f"device: a CUDA device is wanted, not {dev}")
    idx = torch.cuda.current_device() if dev.index is None else dev.index
    return idx, _stream(idx)


def check(device=None) -> None:
    """Waits for the current stream and raises if a bounded in-kernel wait of a linear layer on this
    device, of whichever stream, gave up since this host thread last checked this stream (or since the
    process began): the stream's results since then are not valid. Every thread and stream is told.
    Refused while the stream is being captured."""
    _run(load_library().kk_fp8_check(*_current(device)))


def wait_selftest(device=None, cluster: bool = False, limit_ns: int = 5000) -> None:
    """Diagnostics: a kernel on the current stream waits in vain for limit_ns and gives up, which ``check``
    reports (kk_fp8_wait_selftest)."""
    _run(load_library().kk_fp8_wait_selftest(*_current(device), int(cluster), int(limit_ns)))
