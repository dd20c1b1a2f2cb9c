"""Products with 8-bit block matrices on the GPU against the 64-bit oracle (tests/block8_oracle.py).

Tolerances.  Rounding to 8 bits is compared exactly.  A product's operands are exact numbers (8-bit values times powers of
two; dy as it is), so what remains is the sum of K terms t_i in 32 bits, in whatever order: every one of its at most K
additions is off by at most 2^-23 of the partial sum (the matrix instruction does not promise round-to-nearest), and a partial
sum is at most sum|t_i|: K * 2^-23 * sum|t_i|.  Rounding the result to its type adds half a step, finfo.eps / 2 * |y|.

Products with more than 64 vectors into bf16 run on the 8-bit matrix instruction, which sums 8 products at a time after
aligning them to the largest exponent e of the 8 and dropping what lies below 2^(e-13) (a lone 2^-13 beside 1 - 1
survives, 2^-14 does not, in the same 8; in different 8s it does).  The largest product itself has 8 significant bits and loses
nothing, so 8 products lose less than 7 * 2^(e-13) <= 7 * 2^-13 * max|t_i| of them, and all of them less than
7 * 2^-13 * sum|t_i|: EIGHT below.
"""
import numpy as np
import pytest
import torch

import spmv_amd as S
from spmv_amd import block8
from spmv_amd.block8 import Block8, Packed8, quantize
from tests import block8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
EIGHT = 7 * 2.0 ** -13


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _same(got, want):
    """equal numbers, NaN where NaN"""
    got = _np(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok]), np.abs(got[ok] - want[ok]).max()


def _close(got, want, terms, magnitude, extra=0.0):
    """`terms` additions of terms whose magnitudes add up to `magnitude`, then one rounding to got's type; `extra`: what
    else a sum may be off, as a share of `magnitude`"""
    eps = torch.finfo(got.dtype).eps / 2
    g = _np(got)
    assert g.shape == want.shape
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * eps            # half a step among the subnormals
    err, tol = np.abs(g - want), (terms * 2.0 ** -23 + extra) * magnitude * (1 + eps) + eps * np.abs(want) + tiny
    assert np.all(err <= tol), (float((err / np.maximum(tol, 1e-300)).max()), np.unravel_index(np.argmax(err - tol), err.shape))


def _mat(a, b):
    """a @ b in 64 bits"""
    return torch.mm(torch.from_numpy(np.ascontiguousarray(a)), torch.from_numpy(np.ascontiguousarray(b))).numpy()


def _vectors(n, columns, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, columns, generator=g) * torch.exp(spread * torch.randn(columns, generator=g))
    return x.to(dtype).to(DEV)


class Case:
    def __init__(self, rows, columns, keep, seed, values_dtype=F32):
        self.rows, self.columns = rows, columns
        self.ptr, self.col = O.pattern(rows, columns, keep, seed)
        g = torch.Generator().manual_seed(seed)
        nb = len(self.col)
        self.values = (torch.randn(nb, 128, 128, generator=g) * torch.exp2(torch.randint(-9, 3, (nb, 1, 1), generator=g).float())).to(values_dtype)
        self.A = Block8(rows, columns, self.ptr, self.col)
        self.A.set_values(self.values.to(DEV))
        self.blocks, self.scale = O.quantized_blocks(_np(self.values), self.ptr, self.col, rows, columns)
        self.dense = O.dense(self.blocks, self.ptr, self.col, rows, columns)
        self.dense_abs = O.dense(np.abs(self.blocks), self.ptr, self.col, rows, columns)


# ---- 8 bits and back ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,columns", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 1000), (300, 384), (2, 5000), (1000, 130)])
def test_quantize_and_restore_equal_the_oracle(dtype, n, columns):
    x = _vectors(n, columns, dtype, n + columns, 2.0)
    if n > 2:
        x[1] = 0                                             # a vector of zeros: scale 1
        x[2] *= 2.0 ** -10
    q = quantize(x)
    want, b = O.quantize(_np(x))
    _same(O.decode(q.values.cpu().numpy()), want)
    assert np.array_equal(q.scale.cpu().numpy(), b)
    assert q.restore().dtype == dtype
    _same(q.restore(F32), O.quantized(_np(x)))
    _same(q.restore(), _np(torch.from_numpy(O.quantized(_np(x))).to(dtype)))


def test_quantize_extremes():
    top = torch.finfo(F32).max
    rows = [[448.0, 1.0], [448.0 * (1 + 2.0 ** -23), 1.0], [top, 1.0], [1e-45, 0.0], [2.0 ** -126, -2.0 ** -130], [float("inf"), 3.0],
            [float("nan"), -3.0], [-float("inf"), float("nan")], [0.0, -0.0], [464.0, 17.0], [1.0625, 1.1875], [1e38, 1e-38]]
    x = torch.zeros(len(rows), 200)
    x[:, 0], x[:, 150] = torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])
    x[:, 1] = torch.tensor([r[1] for r in rows])
    q = quantize(x.to(DEV))
    want, b = O.quantize(_np(x))
    _same(O.decode(q.values.cpu().numpy()), want)
    assert np.array_equal(q.scale.cpu().numpy(), b)
    back = _np(q.restore())
    assert back[2, 0] == top                                  # 256 * 2^120 does not exist in 32 bits
    h = torch.full((1, 4), 65504.0, dtype=F16, device=DEV)
    assert np.all(_np(quantize(h).restore()) == 65504.0)      # 256 * 2^8 does not exist in fp16
    h = torch.full((1, 4), torch.finfo(BF16).max, dtype=BF16, device=DEV)
    assert np.all(_np(quantize(h).restore()) == torch.finfo(BF16).max)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_shifted_and_broadcast_vectors(dtype):
    big = _vectors(40, 700, dtype, 3)
    for view in (big[::2, 5:305], big[:, 1:258], big.t()[10:300], big[:1].expand(7, 700), big[:, ::2], big.view(4, 10, 700)[:, 3]):
        q = quantize(view)
        want, b = O.quantize(_np(view))
        _same(O.decode(q.values.cpu().numpy()), want)
        assert np.array_equal(q.scale.cpu().numpy(), b)
        assert q.restore().shape == view.shape
        _same(q.restore(F32), O.quantized(_np(view)))
    cube = big.view(4, 10, 700)
    assert quantize(cube).restore().shape == cube.shape
    _same(quantize(cube).restore(F32).view(40, 700), O.quantized(_np(big)))
    assert quantize(big[3]).restore().shape == (700,)
    assert quantize(big[:0]).restore().shape == (0, 700)


def test_abi_strides_leave_the_gaps_alone():
    """vectors and scales further apart than they are long; nothing between them is written"""
    n, columns, ldx, ld8, lds = 9, 300, 333, 512, 21
    x = _vectors(n, ldx, BF16, 1)
    x8 = torch.full((n, ld8), 7, dtype=torch.uint8, device=DEV)
    sc = torch.full((3, lds), 7, dtype=torch.uint8, device=DEV)
    L, st = S.lib(), torch.cuda.current_stream().cuda_stream
    S.check(L.spmv_hip_quantize8_dev(n, columns, x.data_ptr(), S.BF16, ldx, x8.data_ptr(), ld8, sc.data_ptr(), lds, st))
    want, b = O.quantize(_np(x)[:, :columns])
    _same(O.decode(x8.cpu().numpy()[:, :384]), want)
    assert np.array_equal(sc.cpu().numpy()[:, :n], b)
    assert torch.all(x8[:, 384:] == 7) and torch.all(sc[:, n:] == 7)
    back = torch.full((n, ldx), -5.0, device=DEV)
    S.check(L.spmv_hip_restore8_dev(n, columns, x8.data_ptr(), ld8, sc.data_ptr(), lds, back.data_ptr(), S.F32, ldx, st))
    _same(back[:, :columns], O.quantized(_np(x)[:, :columns]))
    assert torch.all(back[:, columns:] == -5.0)
    # the three products on the same padded operands
    c = Case(260, columns, 0.9, 4)
    xq = O.quantized(_np(x)[:, :columns])
    for k in (n, 1):
        y = torch.full((n, 301), -5.0, device=DEV)
        S.check(L.spmv_hip_block8_mult_dev(c.A._h, k, x8.data_ptr(), S.E4M3, ld8, sc.data_ptr(), lds, y.data_ptr(), S.F32, 301, st))
        _close(y[:k, :260], _mat(xq[:k], c.dense.T), columns, _mat(np.abs(xq[:k]), c.dense_abs.T))
        assert torch.all(y[:, 260:] == -5.0) and torch.all(y[k:] == -5.0)
    dy = _vectors(n, 277, F16, 2)
    dx = torch.full((n, 301), -5.0, device=DEV)
    size = L.spmv_hip_block8_backward_work(c.A._h, n, dy.data_ptr(), S.F16, 277, 1, 1)
    assert size >= 2 * n * 384 * 2
    work = torch.zeros(size + 16, dtype=torch.uint8, device=DEV)
    args = (c.A._h, n, dy.data_ptr(), S.F16, 277)
    S.check(L.spmv_hip_block8_backward_dev(*args, None, 0, None, 0, dx.data_ptr(), S.F32, 301, None, 0, 0, work.data_ptr(), st))
    d = _np(dy)[:, :260]
    _close(dx[:, :columns], _mat(d, c.dense), 260, _mat(np.abs(d), c.dense_abs))
    assert torch.all(dx[:, columns:] == -5.0)
    dv = torch.full((c.A.nblocks + 1, 128, 128), -5.0, device=DEV)
    S.check(L.spmv_hip_block8_backward_dev(*args, x8.data_ptr(), ld8, sc.data_ptr(), lds, None, 0, 0, dv.data_ptr(), S.F32, 0,
                                           work.data_ptr(), st))
    assert torch.all(work[-16:] == 0)
    _close(dv[:-1], O.sampled(_mat(d.T, xq), c.ptr, c.col), n, O.sampled(_mat(np.abs(d).T, np.abs(xq)), c.ptr, c.col))
    assert torch.all(dv[-1] == -5.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_abi_one_vector_needs_no_distance(dtype):
    """n = 1: whatever stands for the distance to the next vector"""
    c = Case(600, 300, 0.9, 6)
    x, dy = _vectors(1, 300, dtype, 1), _vectors(1, 600, dtype, 2)
    q, L, st = quantize(x), S.lib(), torch.cuda.current_stream().cuda_stream
    code = {F32: S.F32, BF16: S.BF16, F16: S.F16}[dtype]
    want_dx, want_dv = c.A.product_t(dy), c.A.gradient(dy, q)
    for ld in (0, 600, 1 << 40):
        dx, dv = torch.full_like(want_dx, -5.0), torch.full_like(want_dv, -5.0)
        work = torch.empty(L.spmv_hip_block8_backward_work(c.A._h, 1, dy.data_ptr(), code, ld, 1, 1) + 16, dtype=torch.uint8, device=DEV)
        S.check(L.spmv_hip_block8_backward_dev(c.A._h, 1, dy.data_ptr(), code, ld, q.values.data_ptr(), 384, q.scale.data_ptr(), 1, dx.data_ptr(),
                                               code, ld, dv.data_ptr(), S.F32, 0, work.data_ptr(), st))
        assert torch.equal(dx, want_dx) and torch.equal(dv, want_dv)
        y = torch.full((1, 600), -5.0, dtype=dtype, device=DEV)
        S.check(L.spmv_hip_block8_mult_dev(c.A._h, 1, x.data_ptr(), code, ld, None, 0, y.data_ptr(), code, ld, st))
        assert torch.equal(y, c.A.product(x))
        x8, sc = torch.zeros_like(q.values), torch.zeros_like(q.scale)
        S.check(L.spmv_hip_quantize8_dev(1, 300, x.data_ptr(), code, ld, x8.data_ptr(), 384, sc.data_ptr(), 1, st))
        assert torch.equal(x8, q.values) and torch.equal(sc, q.scale)


# ---- the matrix -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (128, 128), (130, 255), (500, 700)])
def test_set_values_store_and_load(dtype, rows, columns):
    c = Case(rows, columns, 1.0, 5, dtype)
    v8, sc = c.A.store()
    assert np.array_equal(sc.cpu().numpy(), c.scale)
    s = np.exp2(c.scale.astype(np.float64) - 127)[:, None, None]
    _same(O.decode(v8.cpu().numpy()) * s, c.blocks)
    other = Block8(rows, columns, c.ptr, c.col)
    assert torch.all(other.store()[0] == 0)
    other.load(v8, sc)
    w8, wc = other.store()
    assert torch.equal(w8, v8) and torch.equal(wc, sc)
    # what lies beyond the edge is not taken over
    other.load(torch.full_like(v8, 0x38), sc)
    inside = O.quantized_blocks(np.ones_like(c.blocks), c.ptr, c.col, rows, columns)[0] != 0
    assert np.array_equal(other.store()[0].cpu().numpy() == 0x38, inside)
    info = c.A.info
    assert (info.format, info.rows, info.columns, info.nnz) == (S.BLOCK8, rows, columns, int(inside.sum()))
    assert info.stored == c.A.nblocks * 16384
    assert np.array_equal(_download(c.A, S.ARR_ROW_PTR, len(c.ptr)), c.ptr)
    assert np.array_equal(_download(c.A, S.ARR_COL, len(c.col)), c.col)


def _download(A, which, count):
    out = np.empty(count, np.int32)
    S.check(S.lib().spmv_hip_download(A._h, which, out.ctypes.data, out.nbytes))
    return out


def test_values_that_are_not_finite():
    c = Case(200, 200, 1.0, 6)
    c.values[0, 3, 5], c.values[1, 0, 0] = float("inf"), float("nan")
    c.A.set_values(c.values.to(DEV))
    x = torch.ones(2, 200, device=DEV)
    for n in (2, 70):
        y = _np(c.A.product(x[:1].expand(n, 200)))
        bad = np.zeros(200, bool)
        for r in range(len(c.ptr) - 1):
            for k in range(c.ptr[r], c.ptr[r + 1]):
                if k in (0, 1):
                    bad[r * 128 + (3 if k == 0 else 0)] = True
        assert np.array_equal(np.isnan(y[0]), bad) and np.array_equal(np.isnan(y[-1]), bad)


# ---- products -------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1.0), (128, 128, 1.0), (129, 127, 1.0), (300, 1000, 0.6), (1000, 300, 0.6), (700, 640, 0.3), (2000, 1500, 0.5)]
COUNTS = [1, 2, 13, 16, 17, 33, 64, 65, 127, 128, 200, 515]


@pytest.mark.parametrize("rows,columns,keep", SHAPES)
@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, F16)])
def test_product(rows, columns, keep, x_dtype, y_dtype):
    c = Case(rows, columns, keep, rows + columns)
    for n in COUNTS:
        x = _vectors(n, columns, x_dtype, n)
        xq = O.quantized(_np(x))
        want, magnitude = _mat(xq, c.dense.T), _mat(np.abs(xq), c.dense_abs.T)
        extra = EIGHT if y_dtype == BF16 and n > 64 else 0.0
        _close(c.A.product(x, y_dtype), want, columns, magnitude, extra)
        q = quantize(x)
        _close(c.A.product(q, y_dtype), want, columns, magnitude, extra)
        if n <= 64:                                          # rounding inside the product or before it: the same product
            assert torch.equal(c.A.product(x, y_dtype), c.A.product(q, y_dtype))


@pytest.mark.parametrize("rows,columns,keep", SHAPES)
@pytest.mark.parametrize("dy_dtype,dx_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F16, F32), (F32, BF16)])
def test_product_t(rows, columns, keep, dy_dtype, dx_dtype):
    c = Case(rows, columns, keep, rows + columns)
    for n in COUNTS:
        dy = _vectors(n, rows, dy_dtype, n)
        d = _np(dy)
        _close(c.A.product_t(dy, dx_dtype), _mat(d, c.dense), rows * (3 if dy_dtype == F32 else 2), _mat(np.abs(d), c.dense_abs))


@pytest.mark.parametrize("dy_dtype", TYPES)
@pytest.mark.parametrize("n", [3, 80])
def test_product_t_small_entries_and_far_scales(dy_dtype, n):
    """dy among its type's subnormals (fp16; 2^-100 for the others), blocks of one column 2^-60 to 2^60 apart"""
    rows, columns = 520, 140
    ptr, col = O.pattern(rows, columns, 1.0, 3)
    values = torch.randn(len(col), 128, 128) * torch.exp2(torch.tensor([[-60.0, 60.0, -3.0, 0.0, 20.0][k % 5] for k in range(len(col))]))[:, None, None]
    A = Block8(rows, columns, ptr, col)
    A.set_values(values.to(DEV))
    blocks, _ = O.quantized_blocks(_np(values), ptr, col, rows, columns)
    a, mag = O.dense(blocks, ptr, col, rows, columns), O.dense(np.abs(blocks), ptr, col, rows, columns)
    dy = (torch.randn(n, rows) * (2.0 ** -17 if dy_dtype == F16 else 2.0 ** -40)).to(dy_dtype)
    dy[:, 1::7] = (torch.randn(n, len(range(1, rows, 7))) * (2.0 ** -23 if dy_dtype == F16 else 2.0 ** -60)).to(dy_dtype)
    d = _np(dy)
    assert dy_dtype != F16 or (np.abs(d[d != 0]) < 2.0 ** -14).mean() > 0.9
    _close(A.product_t(dy.to(DEV), F32), _mat(d, a), rows * (3 if dy_dtype == F32 else 2), _mat(np.abs(d), mag))


@pytest.mark.parametrize("rows,columns,keep", SHAPES)
@pytest.mark.parametrize("dy_dtype,dv_dtype", [(F32, F32), (BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
def test_gradient(rows, columns, keep, dy_dtype, dv_dtype):
    c = Case(rows, columns, keep, rows + columns)
    for n in COUNTS:
        x, dy = _vectors(n, columns, dy_dtype, n), _vectors(n, rows, dy_dtype, n + 1, 0.5)
        q = quantize(x)
        xq, d = O.quantized(_np(x)), _np(dy)
        want, magnitude = _mat(d.T, xq), _mat(np.abs(d).T, np.abs(xq))
        want, magnitude = O.sampled(want, c.ptr, c.col), O.sampled(magnitude, c.ptr, c.col)
        dv = c.A.gradient(dy, q, dv_dtype)
        _close(dv, want, n * (3 if dy_dtype == F32 else 2), magnitude)
        if n in (13, 128):
            base = torch.randn(dv.shape, device=DEV).to(dv_dtype)
            out = base.clone()
            assert c.A.gradient(dy, q, out=out, accumulate=True) is out
            _close(out, want + _np(base), n * 3 + 1, magnitude + np.abs(_np(base)))


# ---- the larger tiles, pairs of blocks and cut sums -------------------------------------------------------------------

def _close_64(got, want, terms, magnitude, extra=0.0):
    """_close with 64-bit tensors on the GPU"""
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * eps
    err = (got.double() - want).abs()
    tol = (terms * 2.0 ** -23 + extra) * magnitude * (1 + eps) + eps * want.abs() + tiny
    assert got.shape == want.shape and bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())


def _on_gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


# rows, columns, share of blocks, vectors: 33 block rows (or columns) x 4, 8 or 16 tiles of vectors a workgroup, and 18
# blocks a row for the 16 waves of few vectors
@pytest.mark.parametrize("rows,columns,keep,counts", [(700, 2300, 1.0, [1, 13, 31, 64]), (4200, 500, 0.7, [1000, 2050]), (4100, 150, 1.0, [700])])
@pytest.mark.parametrize("dtype", TYPES)
def test_product_larger(rows, columns, keep, counts, dtype):
    c = Case(rows, columns, keep, rows + columns)
    a, mag = _on_gpu(c.dense.T), _on_gpu(c.dense_abs.T)
    for n in counts:
        x = _vectors(n, columns, dtype, n)
        xq = _on_gpu(O.quantized(_np(x)))
        extra = EIGHT if dtype == BF16 and n > 64 else 0.0
        _close_64(c.A.product(x), torch.mm(xq, a), columns, torch.mm(xq.abs(), mag), extra)


@pytest.mark.parametrize("rows,columns,keep,counts", [(500, 4200, 0.7, [700, 1500, 2900]), (5200, 200, 0.8, [1, 5, 40, 130]), (3001, 130, 1.0, [3, 65, 700]),
                                                      (9000, 64, 0.5, [2, 20])])
@pytest.mark.parametrize("dy_dtype,dx_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_product_t_larger_and_cut(rows, columns, keep, counts, dy_dtype, dx_dtype):
    c = Case(rows, columns, keep, rows + columns)
    a, mag = _on_gpu(c.dense), _on_gpu(c.dense_abs)
    for n in counts:
        # beyond a row's end lies what must not be read, or not be used
        wide = torch.full((n, rows + 24), float("nan"), dtype=dy_dtype, device=DEV)
        for dy in (_vectors(n, rows, dy_dtype, n), wide[:, :rows]):
            dy.copy_(_vectors(n, rows, dy_dtype, n))
            got = c.A.product_t(dy, dx_dtype)
            _close_64(got, torch.mm(dy.double(), a), rows * (3 if dy_dtype == F32 else 2), torch.mm(dy.double().abs(), mag))
            assert torch.equal(c.A.product_t(dy, dx_dtype), got)


@pytest.mark.parametrize("rows,columns,keep,counts", [(4200, 4200, 0.5, [1, 33, 70, 200]), (130, 300, 1.0, [512, 1000, 2111]), (100, 1, 1.0, [4000]),
                                                      (2001, 1500, 0.6, [1999])])
@pytest.mark.parametrize("dy_dtype,dv_dtype", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
def test_gradient_larger_and_cut(rows, columns, keep, counts, dy_dtype, dv_dtype):
    c = Case(rows, columns, keep, rows + columns)
    for n in counts:
        x = _vectors(n, columns, dy_dtype, n)
        q = quantize(x)
        xq = _on_gpu(O.quantized(_np(x)))
        wide = torch.full((n, rows + 24), float("nan"), dtype=dy_dtype, device=DEV)
        for dy in (_vectors(n, rows, dy_dtype, n), wide[:, :rows]):
            dy.copy_(_vectors(n, rows, dy_dtype, n + 1, 0.5))
            d = dy.double()
            want = _on_gpu(O.sampled(torch.mm(d.t().contiguous(), xq).cpu().numpy(), c.ptr, c.col))
            magnitude = _on_gpu(O.sampled(torch.mm(d.abs().t().contiguous(), xq.abs()).cpu().numpy(), c.ptr, c.col))
            dv = c.A.gradient(dy, q, dv_dtype)
            _close_64(dv, want, n * (3 if dy_dtype == F32 else 2), magnitude)
            assert torch.equal(c.A.gradient(dy, q, dv_dtype), dv)
        base = torch.randn(dv.shape, device=DEV).to(dv_dtype)
        out = base.clone()
        c.A.gradient(dy, q, out=out, accumulate=True)
        _close_64(out, want + base.double(), n * 3 + 1, magnitude + base.double().abs())


def test_a_cut_gradient_replays_and_does_not_share_its_workspace():
    """Two captured graphs and an eager call, all of cut sums on one handle, replayed in turn."""
    c = Case(1500, 250, 0.9, 21)
    runs = []
    for k, n in enumerate((900, 4)):
        x, dy = _vectors(n, 250, F16, k), _vectors(n, 1500, F16, 10 + k)
        q = quantize(x)
        f = lambda q=q, dy=dy: (c.A.product_t(dy), c.A.gradient(dy, q))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        runs.append((graph, out, f, dy))
    for k in range(4):
        for graph, out, f, dy in runs:
            dy.copy_(_vectors(dy.shape[0], 1500, F16, 30 + k))
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, f, dy in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, f())), k


def test_dy_vectors_far_apart():
    c = Case(200, 300, 1.0, 23)
    wide = torch.zeros(3, (1 << 23) + 8, dtype=F16, device=DEV)
    dy = wide[:, :200]
    dy.copy_(_vectors(3, 200, F16, 1))
    q = quantize(_vectors(3, 300, F16, 2))
    assert torch.equal(c.A.product_t(dy), c.A.product_t(dy.contiguous()))
    assert torch.equal(c.A.gradient(dy, q), c.A.gradient(dy.contiguous(), q))


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_together_from_vectors_at_odd_addresses(dtype):
    """dx and the blocks' gradient of one backward pass against the two by themselves, dy not 16-byte aligned"""
    c = Case(389, 517, 0.8, 24)
    w = c.values.to(DEV).requires_grad_()
    c.A.set_values(w)
    for n in (1, 70):
        x = _vectors(n, 517, dtype, 1).requires_grad_()
        dy = _vectors(n + 1, 389, dtype, 2).flatten()[1:1 + n * 389].view(n, 389)
        dx, dw = torch.autograd.grad(c.A.linear(x), (x, w), dy)
        assert torch.equal(dx, c.A.product_t(dy)) and torch.equal(dw, c.A.gradient(dy, quantize(x)))


def test_offsets_past_32_bits():
    """a matrix of 2.2 GB and blocks of vectors past 2 GB: the last block row, block column, block and vectors"""
    k = 370
    A = Block8.full(128 * k, 128 * k)
    g = torch.Generator(device=DEV).manual_seed(1)
    v8 = torch.randint(0, 256, (A.nblocks, 128, 128), generator=g, device=DEV, dtype=torch.uint8)
    v8[(v8 & 127) == 127] = 5                                # no NaN
    scale = torch.randint(118, 124, (A.nblocks,), generator=g, device=DEV, dtype=torch.uint8)
    A.load(v8, scale)
    code = torch.from_numpy(O.decode(np.arange(256, dtype=np.uint8))).to(DEV)

    def blocks(ids):                                         # in 64 bits
        return code[v8[ids].long()] * torch.exp2(scale[ids].double() - 127)[:, None, None]

    last_row = blocks(torch.arange(A.nblocks - k, A.nblocks, device=DEV)).permute(1, 0, 2).reshape(128, -1)
    last_col = blocks(torch.arange(k - 1, A.nblocks, k, device=DEV)).reshape(-1, 128)
    n = 46000
    x = torch.randn(n, 128 * k, generator=g, device=DEV, dtype=BF16)
    q = quantize(x)
    tail = quantize(x[-200:])
    assert torch.equal(tail.values, q.values[-200:]) and torch.equal(tail.scale, q.scale[:, -200:])
    back = q.restore(F32)
    assert torch.equal(back[-200:], tail.restore(F32))
    xq = back[-200:].double()
    del back
    for m, p, dtype, extra in ((3, quantize(x[-3:]), F32, 0.0), (200, tail, F32, 0.0), (200, q, BF16, EIGHT)):
        y = A.product(p, dtype)
        a = xq[-m:]
        _close_64(y[-m:, -128:], torch.mm(a, last_row.t().contiguous()), 128 * k, torch.mm(a.abs(), last_row.abs().t().contiguous()), extra)
    dy = y                                                   # [46000, 47360] of bf16
    d = dy[-200:].double()
    for p, m in ((dy, 200), (dy[-3:], 3)):
        dx = A.product_t(p, BF16)
        _close_64(dx[-m:, -128:], torch.mm(d[-m:], last_col), 2 * 128 * k, torch.mm(d[-m:].abs(), last_col.abs()))
    del dx
    dv = A.gradient(dy[-200:], tail, BF16)
    t = d[:, -128:].t().contiguous()
    _close_64(dv[-1], torch.mm(t, xq[:, -128:].contiguous()), 200, torch.mm(t.abs(), xq[:, -128:].abs().contiguous()))


@pytest.mark.parametrize("dtype,n", [(F32, 5500), (BF16, 9000)])
def test_results_larger_than_the_last_cache(dtype, n):
    """restore past the caches against restore through them, of the same vectors in two halves"""
    columns = 7700
    q = quantize(torch.randn(n, columns, device=DEV).to(dtype))
    back = q.restore()
    half = n // 2
    for rows in (slice(0, half), slice(half, n)):
        part = Packed8(q.values[rows], q.scale[:, rows].contiguous(), columns, dtype)
        assert torch.equal(part.restore(), back[rows])


@pytest.mark.parametrize("dtype", TYPES)
def test_few_vectors_and_many_blocks(dtype):
    """from some size on x is rounded before the product: the same bits as inside it"""
    c = Case(4000, 3900, 1.0, 22)
    a, mag = _on_gpu(c.dense.T), _on_gpu(c.dense_abs.T)
    code = {F32: S.F32, BF16: S.BF16, F16: S.F16}[dtype]
    for n in (1, 8, 16, 17, 33, 64):
        x = _vectors(n, 3900, dtype, n)
        y = c.A.product(x)
        inside = torch.empty_like(y)
        S.check(S.lib().spmv_hip_block8_mult_dev(c.A._h, n, x.data_ptr(), code, 3900, None, 0, inside.data_ptr(), code, 4000,
                                                 torch.cuda.current_stream().cuda_stream))
        assert torch.equal(y, inside)
        xq = _on_gpu(O.quantized(_np(x)))
        _close_64(y, torch.mm(xq, a), 3900, torch.mm(xq.abs(), mag))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns,n", [(300, 700, 65), (300, 700, 515), (130, 200, 1024), (250, 130, 1025), (128, 1000, 777)])
def test_many_wide_vectors_and_few_rows(rows, columns, n, dtype):
    """rounded inside the product or before it: the same bits"""
    c = Case(rows, columns, 0.9, rows + n)
    x = _vectors(n, columns, dtype, n)
    xq = _on_gpu(O.quantized(_np(x)))
    y = c.A.product(x)
    _close_64(y, torch.mm(xq, _on_gpu(c.dense.T)), columns, torch.mm(xq.abs(), _on_gpu(c.dense_abs.T)), EIGHT if dtype == BF16 else 0.0)
    assert torch.equal(y, c.A.product(quantize(x)))


def test_two_blocks_at_one_place_add_up_and_get_a_gradient_each():
    ptr, col = np.array([0, 3], np.int32), np.array([1, 0, 1], np.int32)
    A = Block8(100, 200, ptr, col)
    v = torch.randn(3, 128, 128)
    A.set_values(v.to(DEV))
    blocks, _ = O.quantized_blocks(_np(v), ptr, col, 100, 200)
    a, mag = O.dense(blocks, ptr, col, 100, 200), O.dense(np.abs(blocks), ptr, col, 100, 200)
    for n in (3, 100):
        x, dy = _vectors(n, 200, F32, 1), _vectors(n, 100, F32, 2)
        xq = O.quantized(_np(x))
        _close(A.product(x), _mat(xq, a.T), 400, _mat(np.abs(xq), mag.T))
        _close(A.product_t(dy), _mat(_np(dy), a), 600, _mat(np.abs(_np(dy)), mag))
        dv = A.gradient(dy, quantize(x))
        assert torch.equal(dv[0], dv[2])


def test_no_blocks_no_rows_no_columns_no_vectors():
    A = Block8(300, 200, np.zeros(4, np.int32), np.zeros(0, np.int32))
    A.set_values(torch.zeros(0, 128, 128, device=DEV))
    for n in (0, 1, 100):
        x, dy = torch.ones(n, 200, device=DEV), torch.ones(n, 300, device=DEV)
        assert A.product(x).shape == (n, 300) and torch.all(A.product(x) == 0)
        assert A.product_t(dy).shape == (n, 200) and torch.all(A.product_t(dy) == 0)
        assert A.gradient(dy, quantize(x)).shape == (0, 128, 128)
    A = Block8(300, 0, np.zeros(4, np.int32), np.zeros(0, np.int32))
    for n in (3, 100):
        assert torch.all(A.product(torch.ones(n, 0, device=DEV)) == 0) and A.product(torch.ones(n, 0, device=DEV)).shape == (n, 300)
    A = Block8(0, 200, np.zeros(1, np.int32), np.zeros(0, np.int32))
    assert torch.all(A.product_t(torch.ones(3, 0, device=DEV)) == 0)
    c = Case(200, 300, 1.0, 1)
    empty = c.A.gradient(torch.ones(0, 200, device=DEV), quantize(torch.ones(0, 300, device=DEV)))
    assert empty.shape == (c.A.nblocks, 128, 128) and torch.all(empty == 0)


def test_rows_of_a_tensor_of_any_rank_and_stride():
    c = Case(260, 390, 0.7, 8)
    x = _vectors(30, 390, BF16, 1).view(2, 15, 390)
    y = c.A.product(x)
    assert y.shape == (2, 15, 260) and y.dtype == BF16
    assert torch.equal(y.view(30, 260), c.A.product(x.view(30, 390)))
    assert torch.equal(c.A.product(x[0, 3]), y[0, 3])
    wide = _vectors(30, 900, BF16, 2)
    for view in (wide[:, 7:397], wide[::3, 100:490], wide.t()[:30].t()[:, :30].repeat(1, 13)):
        assert torch.equal(c.A.product(view), c.A.product(view.contiguous()))
    wide = _vectors(90, 900, BF16, 2)
    for view in (wide[:, 7:267], wide[::3, 100:360], wide[:1, :260].expand(70, 260)):
        assert torch.equal(c.A.product_t(view), c.A.product_t(view.contiguous()))
        q = quantize(_vectors(view.shape[0], 390, BF16, 3))
        assert torch.equal(c.A.gradient(view, q), c.A.gradient(view.contiguous(), q))


def test_non_finite_vectors_stay_in_their_rows():
    c = Case(256, 256, 1.0, 9)
    for n in (5, 90):
        x = _vectors(n, 256, BF16, 1)
        clean = c.A.product(x)
        x[1, 7], x[3, 200] = float("inf"), float("nan")
        y = c.A.product(x)
        rest = [v for v in range(n) if v not in (1, 3)]
        assert torch.equal(y[rest], clean[rest]) and torch.all(torch.isnan(y[[1, 3]]))
        # tensors padded with NaN behind their last vector and column are never read there
        wide = torch.full((n + 3, 300), float("nan"), dtype=BF16, device=DEV)
        wide[:n, :256] = _vectors(n, 256, BF16, 1)
        assert torch.equal(c.A.product(wide[:n, :256]), clean)
        d = _vectors(n, 256, BF16, 2)
        wide[:n, :256] = d
        q = quantize(_vectors(n, 256, BF16, 1))
        assert torch.equal(c.A.product_t(wide[:n, :256]), c.A.product_t(d))
        assert torch.equal(c.A.gradient(wide[:n, :256], q), c.A.gradient(d, q))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 90])
def test_infinities_in_dy_reach_what_they_multiply(dtype, n):
    """inf * a is inf or, where a is 0, NaN: never NaN because dy was split into parts"""
    c = Case(300, 256, 1.0, 9)
    x, dy = _vectors(n, 256, dtype, 1), _vectors(n, 300, dtype, 2)
    x[x == 0] = 1.0
    dy[1, 7], dy[3, 299], dy[4, 130] = float("inf"), -float("inf"), float("nan")
    xq, d = O.quantized(_np(x)), _np(dy)
    with np.errstate(invalid="ignore"):
        dx = np.zeros((n, 256))                              # block by block: what no stored block touches is not multiplied
        for r in range(len(c.ptr) - 1):
            for k in range(c.ptr[r], c.ptr[r + 1]):
                rows, j = d[:, r * 128:(r + 1) * 128], c.col[k] * 128
                dx[:, j:j + 128] += np.einsum("tr,rc->tc", rows, c.blocks[k][:rows.shape[1]])
        for got, want in ((_np(c.A.product_t(dy, F32)), dx),
                          (_np(c.A.gradient(dy, quantize(x))), O.sampled(np.einsum("tr,tc->rc", d, xq), c.ptr, c.col))):
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
            assert np.array_equal(np.sign(got[np.isinf(got)]), np.sign(want[np.isinf(want)]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 90])
def test_the_largest_numbers_in_dy(dtype, n):
    """finite results of the largest finite dy: no part of it may overflow on the way"""
    rows, columns = 260, 140
    ptr, col = O.pattern(rows, columns, 1.0, 3)
    values = torch.randn(len(col), 128, 128) * 2.0 ** -20
    A = Block8(rows, columns, ptr, col)
    A.set_values(values.to(DEV))
    blocks, _ = O.quantized_blocks(_np(values), ptr, col, rows, columns)
    a, mag = O.dense(blocks, ptr, col, rows, columns), O.dense(np.abs(blocks), ptr, col, rows, columns)
    top = torch.finfo(dtype).max
    dy = torch.randn(n, rows).to(dtype)
    dy[0, 3], dy[1, 200], dy[n - 1, 259] = top, -top, top
    x = _vectors(n, columns, dtype, 4) * 2.0 ** -20
    q, d = quantize(x), _np(dy)
    xq = O.quantized(_np(x))
    _close(A.product_t(dy.to(DEV), F32), _mat(d, a), 3 * rows, _mat(np.abs(d), mag))
    want, magnitude = O.sampled(_mat(d.T, xq), ptr, col), O.sampled(_mat(np.abs(d).T, np.abs(xq)), ptr, col)
    _close(A.gradient(dy.to(DEV), q), want, 3 * n, magnitude)


def test_general_entry_points_take_a_block8_handle():
    """mult, mult_dev, mult_mv, mult_mv_dev and bench of any handle (F32 vectors)"""
    c = Case(390, 390, 0.8, 10)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((70, 390)).astype(np.float32).astype(np.float64)
    xq = O.quantized(x)
    want, mag = _mat(xq, c.dense.T), _mat(np.abs(xq), c.dense_abs.T)
    tol = 390 * 2.0 ** -23 * mag + 2.0 ** -24 * np.abs(want)
    assert np.all(np.abs(c.A.mult(x[0]) - want[0]) <= tol[0])
    assert np.all(np.abs(c.A.mult_mv(x) - want) <= tol)
    xd, yd = torch.from_numpy(x).float().to(DEV), torch.full((70, 400), -3.0, device=DEV)
    c.A.mult_mv_dev(70, xd.data_ptr(), 390, yd.data_ptr(), 400, torch.cuda.current_stream().cuda_stream)
    assert np.all(np.abs(_np(yd)[:, :390] - want) <= tol) and torch.all(yd[:, 390:] == -3.0)
    iters, seconds, _, last = c.A.bench(x[0], 3, 0.0)
    assert iters >= 3 and seconds > 0 and abs(np.linalg.norm(last) - 1) < 1e-5
    assert c.A.analyze(1) == 0
    for name in ("variant", "block_map", "hot_columns"):
        with pytest.raises(S.SpmvHipError, match="does not apply"):
            c.A.set_option(name, 1)


# ---- training -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 40, 130])
def test_linear_gradients(dtype, n):
    c = Case(300, 400, 0.7, 11)
    w = c.values.to(DEV).requires_grad_(True)
    c.A.set_values(w)
    x = _vectors(n, 400, dtype, 1).requires_grad_(True)
    dy = _vectors(n, 300, dtype, 2)
    y = c.A.linear(x)
    assert y.dtype == dtype
    y.backward(dy)
    assert x.grad.dtype == dtype and w.grad.dtype == F32
    xq, d = O.quantized(_np(x)), _np(dy)
    _close(y, _mat(xq, c.dense.T), 400, _mat(np.abs(xq), c.dense_abs.T), EIGHT if dtype == BF16 and n > 64 else 0.0)
    _close(x.grad, _mat(d, c.dense), 900, _mat(np.abs(d), c.dense_abs))
    _close(w.grad, O.sampled(_mat(d.T, xq), c.ptr, c.col), 3 * n, O.sampled(_mat(np.abs(d).T, np.abs(xq)), c.ptr, c.col))
    # a broadcast dy (the gradient of a sum), and only one of the two gradients asked for
    x2 = x.detach().requires_grad_(True)
    c.A.set_values(w.detach())
    c.A.linear(x2).sum().backward()
    one = np.ones((n, 300))
    _close(x2.grad, _mat(one, c.dense), 900, _mat(one, c.dense_abs))
    c.A.set_values(w)
    g, = torch.autograd.grad(c.A.linear(x.detach()).sum(), w)
    _close(g, O.sampled(_mat(one.T, xq), c.ptr, c.col), 3 * n, O.sampled(_mat(one.T, np.abs(xq)), c.ptr, c.col))
    with torch.no_grad():
        assert not c.A.linear(x).requires_grad


def test_linear_gradients_against_differences():
    """Numbers that 8 bits hold exactly before and after the step, so that rounding does not hide the difference; the loss
    sum(y^2) / 2 is quadratic, its central difference exact but for the 32-bit sums."""
    g = torch.Generator().manual_seed(1)
    A = Block8.full(130, 140)
    w = torch.randint(-4, 5, (A.nblocks, 128, 128), generator=g).float()
    x = torch.randint(-4, 5, (9, 140), generator=g).float()
    w[:, 0, 0], x[:, 0], x[:, 128] = 8.0, 8.0, 8.0             # the scales do not change with a step of 1
    def loss(w, x):
        A.set_values(w.to(DEV))
        return float((A.product(x.to(DEV)).double() ** 2).sum() / 2)
    wd, xd = w.to(DEV).requires_grad_(True), x.to(DEV).requires_grad_(True)
    A.set_values(wd)
    y = A.linear(xd)
    (y ** 2 / 2).sum().backward()
    for t, c in ((0, 5), (3, 139), (8, 77)):
        a, b = x.clone(), x.clone()
        a[t, c] += 1; b[t, c] -= 1
        assert abs((loss(w, a) - loss(w, b)) / 2 - float(xd.grad[t, c])) < 0.51      # whole numbers all along
    for k, r, c in ((0, 3, 4), (1, 100, 11), (2, 1, 127), (3, 0, 3)):
        a, b = w.clone(), w.clone()
        a[k, r, c] += 1; b[k, r, c] -= 1
        assert abs((loss(a, x) - loss(b, x)) / 2 - float(wd.grad[k, r, c])) < 0.51


def test_two_layers_share_a_matrix_and_a_changed_one_is_refused():
    c = Case(256, 256, 1.0, 12)
    w = c.values.to(DEV).requires_grad_(True)
    c.A.set_values(w)
    x = _vectors(20, 256, F32, 1).requires_grad_(True)
    y1 = c.A.linear(x)
    y2 = c.A.linear(y1)
    y2.sum().backward()
    q1, q2 = quantize(x), quantize(y1)
    d2 = torch.ones(20, 256, device=DEV)
    d1 = c.A.product_t(d2)
    want = c.A.gradient(d2, q2) + c.A.gradient(d1, q1)
    # two gradients of at most 20 terms each, added in either order
    assert torch.allclose(w.grad, want, rtol=2.0 ** -22, atol=0)
    assert torch.equal(x.grad, c.A.product_t(d1))
    y = c.A.linear(x)
    c.A.set_values(w)
    with pytest.raises(RuntimeError, match="set again between forward and backward"):
        y.sum().backward()


def test_checkpoint_holds_8_bits_only():
    c = Case(128, 1024, 1.0, 13)
    c.A.set_values(c.values.to(DEV).requires_grad_(True))
    x = _vectors(4096, 1024, BF16, 1)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = c.A.linear(x)
    held = torch.cuda.memory_allocated() - before - y.numel() * y.element_size()
    assert held <= 4096 * (1024 + 8) + 4096                   # bytes of the 8-bit copy and its scales, not 2 per entry


# ---- streams, graphs, refusals --------------------------------------------------------------------------------------

def test_a_run_on_a_side_stream():
    c = Case(500, 600, 0.6, 14)
    x, dy = _vectors(150, 600, BF16, 1), _vectors(150, 500, BF16, 2)
    want = (c.A.product(x), c.A.product_t(dy), c.A.gradient(dy, quantize(x)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = (c.A.product(x), c.A.product_t(dy), c.A.gradient(dy, quantize(x)))
    st.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_products_on_one_handle_overlap_on_two_streams():
    c = Case(1000, 1000, 0.8, 15)
    xs = [_vectors(n, 1000, BF16, n) for n in (1, 7, 64, 300)]
    want = [c.A.product(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(c.A.product(xs[k]))
    torch.cuda.synchronize()
    for k in range(len(xs)):
        assert all(torch.equal(y, want[k]) for y in got[k])


def test_captured_step_replays_with_new_inputs():
    """set_values, checkpoint, product and both gradients in one graph, replayed with other inputs and eager work between"""
    c = Case(390, 520, 0.7, 16)
    n = 100
    w, x, dy = c.values.to(DEV), _vectors(n, 520, BF16, 1), _vectors(n, 390, BF16, 2)
    few = _vectors(3, 520, BF16, 3)

    def step():
        c.A.set_values(w)
        q = quantize(x)
        return c.A.product(q), c.A.product_t(dy), c.A.gradient(dy, q), q.restore(), c.A.product(few)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        w.copy_(torch.randn(w.shape) * 2.0 ** (k - 2))
        x.copy_(_vectors(n, 520, BF16, 20 + k))
        dy.copy_(_vectors(n, 390, BF16, 30 + k))
        few.copy_(_vectors(3, 520, BF16, 40 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), k


def test_captured_training_step_through_linear():
    """set_values, linear and its backward pass in one graph; nothing of an eager pass alive meanwhile"""
    c = Case(390, 520, 0.7, 19)
    n = 100
    w = c.values.to(DEV).requires_grad_()
    x, dy = _vectors(n, 520, BF16, 1).requires_grad_(), _vectors(n, 390, BF16, 2)

    def step():
        c.A.set_values(w)
        y = c.A.linear(x)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            w.copy_(torch.randn(w.shape) * 2.0 ** (k - 2))
            x.copy_(_vectors(n, 520, BF16, 20 + k))
        dy.copy_(_vectors(n, 390, BF16, 30 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), k


def test_repeated_calls_give_the_same_bits():
    c = Case(1500, 1300, 0.5, 17)
    x, dy = _vectors(333, 1300, BF16, 1), _vectors(333, 1500, BF16, 2)
    q = quantize(x)
    for f in (lambda: c.A.product(q), lambda: c.A.product_t(dy), lambda: c.A.gradient(dy, q), lambda: c.A.product(x[:5])):
        first = f()
        for _ in range(5):
            assert torch.equal(f(), first)


def test_refusals():
    c = Case(200, 300, 1.0, 18)
    A, L = c.A, S.lib()
    x = torch.zeros(2, 300, device=DEV)
    with pytest.raises(ValueError, match="expected"):
        A.product(torch.zeros(2, 299, device=DEV))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        A.product(torch.zeros(2, 300, device=DEV, dtype=torch.float64))
    with pytest.raises(ValueError, match="no CPU path"):
        A.product(torch.zeros(2, 300))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        A.product(x, torch.float64)
    with pytest.raises(ValueError, match="out must be"):
        A.product(x, out=torch.zeros(2, 201, device=DEV))
    with pytest.raises(ValueError, match="columns"):
        A.product(quantize(torch.zeros(2, 128, device=DEV)))
    with pytest.raises(ValueError, match="vectors of"):
        A.gradient(torch.zeros(3, 200, device=DEV), quantize(x))
    with pytest.raises(TypeError, match="Packed8"):
        A.gradient(torch.zeros(2, 200, device=DEV), x)
    with pytest.raises(ValueError, match="accumulate"):
        A.gradient(torch.zeros(2, 200, device=DEV), quantize(x), accumulate=True)
    with pytest.raises(ValueError, match="contiguous"):
        A.set_values(torch.zeros(A.nblocks, 128, 64, device=DEV))
    with pytest.raises(ValueError, match="the matrix on"):
        A.set_values(torch.zeros(A.nblocks, 128, 128))
    with pytest.raises(TypeError):
        A.set_values(torch.zeros(A.nblocks, 128, 128, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="scale"):
        A.load(torch.zeros(A.nblocks, 128, 128, device=DEV, dtype=torch.uint8), torch.zeros(A.nblocks + 1, device=DEV, dtype=torch.uint8))

    def fails(rc, text):
        assert rc != 0 and text in L.spmv_hip_last_error().decode()

    p, h = x.data_ptr(), A._h
    fails(L.spmv_hip_block8_mult_dev(h, 1025, p, S.F32, 300, None, 0, p, S.F32, 200, None), "at most 1024")
    fails(L.spmv_hip_block8_mult_dev(h, 1, p, S.F32, 300, p, 0, p, S.F32, 200, None), "scales belong")
    fails(L.spmv_hip_block8_mult_dev(h, 1, p, S.F64, 300, None, 0, p, S.F32, 200, None), "F32, BF16, F16 or E4M3")
    fails(L.spmv_hip_block8_mult_dev(h, 1, p, S.F32, 300, None, 0, p, S.E4M3, 200, None), "must be F32, BF16 or F16")
    fails(L.spmv_hip_block8_mult_dev(h, 1, p, S.E4M3, 300, p, 1, p, S.F32, 200, None), "multiple of 128")
    fails(L.spmv_hip_block8_mult_dev(h, 2, p, S.F32, 300, None, 0, p, S.F32, 199, None), "shorter than their length")
    fails(L.spmv_hip_block8_mult_dev(h, -1, p, S.F32, 300, None, 0, p, S.F32, 200, None), "negative vector count")
    back = lambda n=2, dy=p, dt=S.F32, ld=200, x8=p, ld8=384, sc=p, lds=2, dx=p, xt=S.F32, ldx=300, dv=p, vt=S.F32, work=p: \
        L.spmv_hip_block8_backward_dev(h, n, dy, dt, ld, x8, ld8, sc, lds, dx, xt, ldx, dv, vt, 0, work, None)
    fails(back(ld=199), "shorter than their length")
    fails(back(ldx=299), "shorter than their length")
    fails(back(ld=1 << 23), "at most 2^23 - 1")
    fails(back(dy=None), "NULL vector block")
    fails(back(dt=S.E4M3), "must be F32, BF16 or F16")
    fails(back(xt=S.F64), "must be F32, BF16 or F16")
    fails(back(vt=9), "must be F32, BF16 or F16")
    fails(back(n=-1), "negative vector count")
    fails(back(lds=1), "1 scales per group")
    fails(back(x8=None), "NULL 8-bit")
    fails(back(work=None), f"NULL workspace, {3 * 2 * 256 * 2} bytes needed")
    fails(back(work=p + 8), "workspace is not 16-byte aligned")
    assert back(dx=None, dv=None) == 0                       # neither asked for: nothing to do
    m = S.Matrix.csr(2, 2, S.make_coo([0, 1], [0, 1], [1.0, 2.0]))
    fails(L.spmv_hip_block8_mult_dev(m._h, 1, p, S.F32, 2, None, 0, p, S.F32, 2, None), "needs a handle of 8-bit blocks")
    m.free()
    fails(L.spmv_hip_download(h, S.ARR_VAL, p, 4), "not part of format")
