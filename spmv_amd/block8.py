"""Matrices of 128 x 128 blocks in 8 bits: a layer's product, both its gradients, and 8-bit checkpoints of activations.

The host side of the `spmv_hip_block8_*` / `_quantize8_` / `_restore8_` calls of include/spmv_hip.h on torch tensors.
Vectors are the rows of a tensor [..., columns]; every call runs on the device of its tensors, on torch's current stream
there, and is checked here before the library sees an address.

    A = Block8(rows, columns, block_ptr, block_col)   # which blocks are stored, as a CSR pattern of blocks
    A.set_values(w)                                   # w [blocks, 128, 128], rounded to 8 bits block by block
    y = A.linear(x)                                   # differentiable in x and w; keeps x in 8 bits until backward
    y = A.product(x)                                  # the product alone

Number format (include/spmv_hip.h has the definition): e4m3 values, one power-of-two scale per block of the matrix and per
128 consecutive entries of a vector, kept as the byte b of 2^(b-127), 1 to 247.  Gradients are those of the product with the
rounded operands (the rounding itself counts as the identity).
"""
from __future__ import annotations

import math

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .matrix import Matrix

BLOCK = 128
MAX_WIDE = 1024                       # vectors a product rounds to 8 bits by itself (SPMV_HIP_BLOCK8_MAX_WIDE)
MAX_APART = 1 << 23                   # entries between vectors of dy, less than
MAX_INT = (1 << 31) - 1               # of the library's sizes; ctypes would cut a larger one off without a word
_DTYPE = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


# torch's current stream on a device, as an address.  The public torch.cuda.current_stream(device).cuda_stream builds a
# Stream object for it: 1.5 us, against 5 us for a whole call with few vectors.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)


def _dual_level() -> int:
    """negative outside of forward-mode differentiation"""
    return getattr(forward_ad, "_current_level", 0)


def _stream(index: int) -> int:
    """The stream of a call.  torch.jit.trace would record the tensors made for the results, and not the calls that fill them."""
    if _tracing():
        raise RuntimeError("products with 8-bit blocks cannot be traced by torch.jit")
    return _raw_stream(index)


def _call(device: torch.device, f, *args) -> None:
    """A library call without a handle, which knows no device of its own, on `device`."""
    if torch.cuda.current_device() == device.index:
        L.check(f(*args))
    else:
        with torch.cuda.device(device):
            L.check(f(*args))


def _wide(name: str, x: torch.Tensor, length: int | None = None) -> torch.Tensor:
    """x, without its history, as [n, length] rows that are contiguous inside (any distance apart); copies only what has no
    such view."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPE:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 tensor")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a GPU; there is no CPU path")
    if x.dim() < 1 or (length is not None and x.shape[-1] != length):
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected (..., {length})")
    if x.requires_grad:
        x = x.detach()
    if x.is_neg():                               # the memory holds the negated numbers
        x = x.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if x.shape[0] > MAX_INT or x.shape[1] > MAX_INT:
        raise ValueError(f"{name} holds {x.shape[0]} vectors of {x.shape[1]}, more than 2^31 - 1")
    if not x.is_contiguous():
        n, columns = x.shape
        if columns > 1 and x.stride(1) != 1 or n > 1 and x.stride(0) < columns:
            x = x.contiguous()                   # transposed or broadcast rows
    return x


def _ld(x: torch.Tensor) -> int:
    return max(x.stride(0), x.shape[1])


def _meets(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Does the contiguous `out` share memory with the rows of t (contiguous inside, any distance apart)?"""
    if out.numel() == 0 or t.numel() == 0:
        return False
    o, p, size = out.data_ptr(), t.data_ptr(), t.element_size()
    n, row = (t.shape[0], t.shape[1] * size) if t.dim() == 2 else (1, t.numel() * size)
    apart = max(t.stride(0) * size, row) if n > 1 else row
    i = max((o - p - row) // apart + 1, 0)       # the first row that ends behind out's beginning
    return i < n and p + i * apart < o + out.numel() * out.element_size()


class Packed8:
    """n vectors in 8 bits: `values` uint8 [n, columns rounded up to 128] (zero past `columns`), `scale` uint8
    [groups, n], `dtype` of the vectors it was made from, `shape` (..., columns) of the tensor that held them: n vectors in
    all.  The calls that take it trust these to fit each other, so none can be replaced."""

    __slots__ = ("values", "scale", "columns", "dtype", "shape")

    def __init__(self, values: torch.Tensor, scale: torch.Tensor, columns: int, dtype: torch.dtype, shape=None):
        if columns < 0:
            raise ValueError(f"columns is {columns}, must not be negative")
        groups = -(-columns // BLOCK)
        if dtype not in _DTYPE:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        if values.dtype != torch.uint8 or values.dim() != 2 or values.shape[1] != groups * BLOCK or not values.is_contiguous():
            raise ValueError(f"values must be a contiguous uint8 tensor [n, {groups * BLOCK}]")
        if scale.dtype != torch.uint8 or tuple(scale.shape) != (groups, values.shape[0]) or not scale.is_contiguous():
            raise ValueError(f"scale must be a contiguous uint8 tensor [{groups}, {values.shape[0]}]")
        n = values.shape[0]
        if n > MAX_INT or columns > MAX_INT:
            raise ValueError(f"{n} vectors of {columns} are more than 2^31 - 1")
        shape = tuple(shape) if shape is not None else (n, columns)
        if not shape or shape[-1] != columns or min(shape) < 0 or math.prod(shape[:-1]) != n:
            raise ValueError(f"shape {shape} does not hold {n} vectors of {columns}")
        if not values.is_cuda or scale.device != values.device:
            raise ValueError("values and scale must be on one GPU")
        self._fill(values, scale, columns, dtype, shape)

    def __setattr__(self, name, value):
        raise AttributeError(f"Packed8.{name} cannot be replaced")

    def __delattr__(self, name):
        raise AttributeError(f"Packed8.{name} cannot be removed")

    def __reduce__(self):
        return Packed8._made, (self.values, self.scale, self.columns, self.dtype, self.shape)

    @classmethod
    def _made(cls, values, scale, columns, dtype, shape):
        """Of tensors made here: nothing to check."""
        q = object.__new__(cls)
        q._fill(values, scale, columns, dtype, shape)
        return q

    def _fill(self, values, scale, columns, dtype, shape) -> None:
        _put_values(self, values)
        _put_scale(self, scale)
        _put_columns(self, columns)
        _put_dtype(self, dtype)
        _put_shape(self, shape)

    @property
    def n(self) -> int:
        return self.values.shape[0]

    def restore(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The vectors their 8-bit form stands for, in the shape they came in."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPE:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        device, (n, ld8) = self.values.device, self.values.shape
        x = self.values.new_empty(self.shape, dtype=dtype)
        _call(device, L.lib().spmv_hip_restore8_dev, n, self.columns, self.values.data_ptr(), ld8, self.scale.data_ptr(), n,
              x.data_ptr(), _DTYPE[dtype], self.columns, _stream(device.index))
        return x


_put_values, _put_scale, _put_columns, _put_dtype, _put_shape = (getattr(Packed8, name).__set__ for name in Packed8.__slots__)


def _rounded(rows: torch.Tensor, shape) -> Packed8:
    n, columns = rows.shape
    groups = -(-columns // BLOCK)
    device = rows.device
    values = rows.new_empty((n, groups * BLOCK), dtype=torch.uint8)
    scale = rows.new_empty((groups, n), dtype=torch.uint8)
    _call(device, L.lib().spmv_hip_quantize8_dev, n, columns, rows.data_ptr(), _DTYPE[rows.dtype], _ld(rows), values.data_ptr(),
          groups * BLOCK, scale.data_ptr(), n, _stream(device.index))
    return Packed8._made(values, scale, columns, rows.dtype, shape)


def quantize(x: torch.Tensor) -> Packed8:
    """x [..., columns] to 8 bits."""
    return _rounded(_wide("x", x), x.shape)


def _whole(name: str, a) -> np.ndarray:
    """a as the library's 32-bit integers, refused where that would change a number."""
    a = np.asarray(a)
    with np.errstate(invalid="ignore"):
        whole = np.ascontiguousarray(a, np.int32)
    if not np.array_equal(a, whole):
        raise ValueError(f"{name} must hold whole numbers of 32 bits")
    return whole


def _inside(n: int, size: int, rows: int, nblocks: int, cus: int) -> bool:
    """Are n vectors rounded inside the product, by every workgroup again, or by a call to quantize before?  Inside where that
    costs less (bf16, 1920 blocks: 16 vectors 11 us inside, 17 before; 32 vectors 26 and 17 us; 4096 blocks, 16 vectors 17
    and 17 us), and more than 64 vectors only where the library takes those in 8 bits by the same kernel (tiles of 64 for an
    eighth of the CUs): the same bits either way."""
    if n > 64 and (n > MAX_WIDE or -(-rows // BLOCK) * -(-n // 64) * 8 > cus):
        return False
    return nblocks * (-(-n // 16) * size) < (8500 if n <= 16 else 7500)


class Block8(Matrix):
    """A handle of 8-bit blocks on the current device.  block_ptr [ceil(rows / 128) + 1] and block_col are host integers
    like the row_ptr and col of a CSR matrix, in units of blocks."""

    def __init__(self, rows: int, columns: int, block_ptr, block_col):
        if max(rows, columns) > MAX_INT:
            raise ValueError(f"{rows} x {columns} is more than 2^31 - 1 a side")
        ptr, col = _whole("block_ptr", block_ptr), _whole("block_col", block_col)
        if ptr.shape != (-(-max(rows, 0) // BLOCK) + 1,) or col.ndim != 1:
            raise ValueError(f"block_ptr has shape {ptr.shape} for {rows} rows, block_col {col.shape}")
        super().__init__(L.lib().spmv_hip_create_block8(rows, columns, len(col), ptr.ctypes.data, col.ctypes.data))
        self.rows, self.columns, self.nblocks = rows, columns, len(col)
        self._index = torch.cuda.current_device()
        self.device = torch.device("cuda", self._index)
        self._cus = torch.cuda.get_device_properties(self._index).multi_processor_count
        self.values = None               # the tensor set_values last took: the leaf that linear() differentiates
        self._version = 0                # set_values / load calls so far

    @classmethod
    def full(cls, rows: int, columns: int) -> "Block8":
        """Every block stored."""
        brows, bcols = -(-rows // BLOCK), -(-columns // BLOCK)
        return cls(rows, columns, np.arange(brows + 1) * bcols, np.tile(np.arange(bcols), brows))

    def download(self, which: int) -> np.ndarray:
        """The pattern (ARR_ROW_PTR: block_ptr, ARR_COL: block_col); store has the values."""
        size = {L.ARR_ROW_PTR: -(-self.rows // BLOCK) + 1, L.ARR_COL: self.nblocks}.get(which)
        if size is None:
            return super().download(which)       # refused there
        out = np.empty(size, np.int32)
        L.check(L.lib().spmv_hip_download(self._h, which, out.ctypes.data, out.nbytes))
        return out

    def _here(self, name: str, t: torch.Tensor) -> None:
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the matrix on {self.device}")

    def _blocks(self, name: str, t: torch.Tensor, dtypes) -> None:
        if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
            raise TypeError(f"{name} must be a tensor of one of {sorted(str(d) for d in dtypes)}")
        if tuple(t.shape) != (self.nblocks, BLOCK, BLOCK) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [{self.nblocks}, 128, 128], has shape {tuple(t.shape)}")
        self._here(name, t)

    def _out(self, out, shape, dtype, *operands: torch.Tensor):
        if dtype not in _DTYPE:
            raise TypeError("the result's type must be float32, bfloat16 or float16")
        if out is None:
            return operands[0].new_empty(shape, dtype=dtype)
        if tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_contiguous() or out.is_neg():
            raise ValueError(f"out must be contiguous {tuple(shape)} of {dtype}")
        self._here("out", out)
        if any(_meets(out, t) for t in operands):
            raise ValueError("out shares memory with an operand, which is still read while it is written")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out requires grad, and results written into it have no history")
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)      # for passes that saved it
        return out

    def set_values(self, values: torch.Tensor) -> None:
        """Rounds values [blocks, 128, 128] into the matrix, on the current stream (products on others have to wait for
        it).  linear() returns the gradient of this tensor."""
        self._blocks("values", values, _DTYPE)
        data = values.detach().resolve_neg() if values.is_neg() else values
        L.check(L.lib().spmv_hip_block8_set_values_dev(self._h, data.data_ptr(), _DTYPE[values.dtype], _stream(self._index)))
        self.values = values
        self._version += 1

    def load(self, values8: torch.Tensor, scale: torch.Tensor) -> None:
        """8-bit values [blocks, 128, 128] (uint8 or float8_e4m3fn) and scale bytes uint8 [blocks] as they are."""
        self._blocks("values8", values8, (torch.uint8, torch.float8_e4m3fn))
        if scale.dtype != torch.uint8 or tuple(scale.shape) != (self.nblocks,) or not scale.is_contiguous():
            raise ValueError(f"scale must be a contiguous uint8 tensor [{self.nblocks}]")
        self._here("scale", scale)
        L.check(L.lib().spmv_hip_block8_load_dev(self._h, values8.data_ptr(), scale.data_ptr(), _stream(self._index)))
        self.values = None
        self._version += 1

    def store(self):
        """(values8 uint8 [blocks, 128, 128], scale uint8 [blocks]): what load takes."""
        values8 = torch.empty((self.nblocks, BLOCK, BLOCK), dtype=torch.uint8, device=self.device)
        scale = torch.empty(self.nblocks, dtype=torch.uint8, device=self.device)
        L.check(L.lib().spmv_hip_block8_store_dev(self._h, values8.data_ptr(), scale.data_ptr(), _stream(self._index)))
        return values8, scale

    def product(self, x, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """y[..., rows] = A x for the vectors of x: a tensor [..., columns] (rounded to 8 bits on the way in) or a
        Packed8.  `dtype` of y: that of x unless given.  y has no history (linear has).

        Sums are 32 bits wide, with one exception: bfloat16 results of more than 64 vectors come from the 8-bit matrix
        instruction, at twice the rate, and may be off by 7 * 2^-13 of the sum of the terms' magnitudes before they are
        rounded, so that a vector's last bits depend on how many others come with it.  dtype=torch.float32 avoids that."""
        if not isinstance(x, Packed8):
            rows = _wide("x", x, self.columns)
            self._here("x", rows)
            shape = (*x.shape[:-1], self.rows)
            n = rows.shape[0]
            if _inside(n, rows.element_size(), self.rows, self.nblocks, self._cus):
                y = self._out(out, shape, dtype or rows.dtype, rows)
                L.check(L.lib().spmv_hip_block8_mult_dev(self._h, n, rows.data_ptr(), _DTYPE[rows.dtype], _ld(rows),
                                                         None, 0, y.data_ptr(), _DTYPE[y.dtype], self.rows, _stream(self._index)))
                return y
            dtype = dtype or rows.dtype
            x = _rounded(rows, rows.shape)
        else:
            if x.columns != self.columns:
                raise ValueError(f"x has {x.columns} columns, the matrix {self.columns}")
            self._here("x", x.values)
            shape = (*x.shape[:-1], self.rows)
        y = self._out(out, shape, dtype or x.dtype, x.values, x.scale)
        L.check(L.lib().spmv_hip_block8_mult_dev(self._h, x.n, x.values.data_ptr(), L.E4M3, x.values.shape[1], x.scale.data_ptr(),
                                                 x.n, y.data_ptr(), _DTYPE[y.dtype], self.rows, _stream(self._index)))
        return y

    def product_t(self, dy: torch.Tensor, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """dx[..., columns] = A^T dy for dy [..., rows]; dy is not rounded."""
        d = self._dy(dy)
        dx = self._out(out, (*dy.shape[:-1], self.columns), dtype or d.dtype, d)
        self._backward(d, None, dx, None, False)
        return dx

    def gradient(self, dy: torch.Tensor, x: Packed8, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                 accumulate: bool = False) -> torch.Tensor:
        """The gradient of the stored blocks [blocks, 128, 128] from dy [..., rows] and the 8-bit x of the product."""
        d = self._dy(dy)
        if not isinstance(x, Packed8):
            raise TypeError("x must be a Packed8 (quantize)")
        if x.columns != self.columns or x.n != d.shape[0]:
            raise ValueError(f"x holds {x.n} vectors of {x.columns}, dy {d.shape[0]} for a matrix of {self.columns} columns")
        self._here("x", x.values)
        if accumulate and out is None:
            raise ValueError("accumulate adds to out, which is missing")
        dv = self._out(out, (self.nblocks, BLOCK, BLOCK), out.dtype if out is not None else dtype, d, x.values, x.scale)
        self._backward(d, x, None, dv, accumulate)
        return dv

    def _dy(self, dy) -> torch.Tensor:
        d = _wide("dy", dy, self.rows)
        if _ld(d) >= MAX_APART:
            d = d.contiguous()
        self._here("dy", d)
        return d

    def _backward(self, d, x, dx, dv, accumulate) -> None:
        """dx and dv, either None, from checked operands."""
        lib, n, ld = L.lib(), d.shape[0], _ld(d)
        p, t, work = d.data_ptr(), _DTYPE[d.dtype], None
        size = lib.spmv_hip_block8_backward_work(self._h, n, p, t, ld, dx is not None, dv is not None)
        if size:
            work = d.new_empty(size, dtype=torch.uint8)
        L.check(lib.spmv_hip_block8_backward_dev(
            self._h, n, p, t, ld,
            *((x.values.data_ptr(), x.values.shape[1], x.scale.data_ptr(), x.n) if dv is not None else (None, 0, None, 0)),
            *((dx.data_ptr(), _DTYPE[dx.dtype], self.columns) if dx is not None else (None, 0, 0)),
            *((dv.data_ptr(), _DTYPE[dv.dtype]) if dv is not None else (None, 0)), accumulate,
            work.data_ptr() if work is not None else None, _stream(self._index)))

    def linear(self, x: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
        """y = A x, differentiable in x and in the tensor that set_values took.  `dtype` of y as in product: float32 for sums of
        32 bits whatever the number of vectors.  Between the passes x is kept in 8 bits; the backward pass refuses a matrix
        whose values were set again meanwhile (not by the replay of a graph, which is not seen here).  Forward-mode
        differentiation is refused."""
        if not isinstance(x, torch.Tensor):
            raise TypeError("x must be a tensor")
        if _dual_level() >= 0:
            for t in (x, self.values):
                if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                    raise NotImplementedError("linear has no forward-mode derivative")
        if torch.is_grad_enabled() and (x.requires_grad or self.values is not None and self.values.requires_grad):
            return _Linear.apply(x, self.values, self, dtype)
        return self.product(x, dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, matrix, dtype):
        rows = _wide("x", x, matrix.columns)
        matrix._here("x", rows)
        q = _rounded(rows, x.shape)
        ctx.save_for_backward(q.values, q.scale)
        ctx.matrix, ctx.version, ctx.x_shape, ctx.x_dtype = matrix, matrix._version, x.shape, x.dtype
        ctx.values_dtype = values.dtype if values is not None else None
        return matrix.product(q, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        values8, scale = ctx.saved_tensors
        matrix = ctx.matrix
        if matrix._version != ctx.version:
            raise RuntimeError("the values of the 8-bit matrix were set again between forward and backward")
        d = matrix._dy(dy)
        dx = d.new_empty(ctx.x_shape, dtype=ctx.x_dtype) if ctx.needs_input_grad[0] else None
        dv = None
        if ctx.needs_input_grad[1]:
            dv = d.new_empty((matrix.nblocks, BLOCK, BLOCK), dtype=ctx.values_dtype)
        matrix._backward(d, Packed8._made(values8, scale, matrix.columns, ctx.x_dtype, ctx.x_shape), dx, dv, False)
        return dx, dv, None, None
