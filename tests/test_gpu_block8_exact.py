"""Products with 8-bit block matrices whose exact results are known: equality, no tolerance.

Whole numbers up to 8 are exact in 8 bits (a group's scale is at least 2^-5 where its largest is 8: four significant
bits from 2^-5 on), their products are at most 64, and sums of up to 2^18 of them stay below 2^24: every addition in 32 bits is
exact, in whatever order, and so is the 8-bit matrix instruction (it drops what lies 13 bits below the largest of 8 products, and
64 * 2^-13 < 1).  A lost, doubled or misplaced term changes the result.
"""
import numpy as np
import pytest
import torch

import spmv_amd as S
from spmv_amd.block8 import Block8, Packed8, quantize
from tests import block8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def _whole(seed, *shape, top=8):
    """whole numbers -top .. top, none of them zero"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = torch.randint(1, top + 1, shape, generator=g, device=DEV)
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.5, -a, a).double()


def _equal(got, want, *what):
    got = got.double()
    assert got.shape == want.shape
    wrong = int((got != want).sum())
    assert wrong == 0, (*what, f"{wrong} of {got.numel()}, the first at {torch.nonzero(got != want)[0].tolist()}")


class Whole:
    """A matrix of whole numbers: its blocks, and the dense matrix in 64 bits."""

    def __init__(self, rows, columns, keep, seed):
        self.rows, self.columns = rows, columns
        self.ptr, self.col = O.pattern(rows, columns, keep, seed)
        self.values = _whole(seed, len(self.col), 128, 128)
        self.A = Block8(rows, columns, self.ptr, self.col)
        self.A.set_values(self.values.float())
        self.dense = torch.from_numpy(O.dense(self.values.cpu().numpy(), self.ptr, self.col, rows, columns)).to(DEV)

    def sampled(self, full):
        return torch.from_numpy(O.sampled(full.cpu().numpy(), self.ptr, self.col)).to(DEV)


def _in_place(a, gap):
    """a, its vectors a multiple of 8 entries apart and 16-byte aligned, NaN between them"""
    n, length = a.shape
    wide = torch.full((n, -(-length // 8) * 8 + gap), float("nan"), dtype=a.dtype, device=DEV)
    wide[:, :length] = a
    view = wide[:, :length]
    assert view.data_ptr() % 16 == 0 and view.stride(0) % 8 == 0
    return view


# ---- dy where it lies -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,columns,keep", [(129, 130, 1.0), (300, 260, 0.9), (501, 300, 0.9), (2001, 300, 0.7), (2500, 4100, 0.4), (8199, 900, 1.0)])
def test_gradients_from_dy_in_place_that_ends_inside_16_bytes(rows, columns, keep, dtype):
    """the last vector of every 32 ends where the loads' bound lies"""
    c = Whole(rows, columns, keep, rows)
    for n in (31, 32, 33, 64, 1000):
        x, dy = _whole(n, n, columns), _whole(n + 1, n, rows)
        q = quantize(x.float())
        for gap in (0, 8):
            d = _in_place(dy.to(dtype), gap)
            _equal(c.A.gradient(d, q), c.sampled(torch.mm(dy.t().contiguous(), x)), n, gap)
            _equal(c.A.product_t(d, F32), torch.mm(dy, c.dense), n, gap)


# ---- the largest and the smallest numbers ---------------------------------------------------------------------------

def _close(got, want, terms, magnitude, extra=0.0, floor=0.0):
    """`terms` additions in 32 bits of terms whose magnitudes add up to `magnitude` (each off by at most 2^-23 of the partial
    sum), `extra` more of `magnitude` and `floor` whatever it is, then one rounding to got's type"""
    eps, least = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal
    g = got.double()
    want, magnitude = want.to(DEV), magnitude.to(DEV)
    tol = (terms * 2.0 ** -23 + extra) * magnitude * (1 + eps) + eps * want.abs() + 2 * eps * least + floor
    over = want.abs() > torch.finfo(got.dtype).max
    off = torch.where(over, torch.zeros_like(want), (g - want).abs() - tol)
    assert bool((off <= 0).all()), (float(off.max()), torch.nonzero(~(off <= 0))[0].tolist())
    assert bool(torch.isinf(g[over]).all())


EIGHT = 7 * 2.0 ** -13             # the 8-bit matrix instruction: what it drops of 8 products, each below 2^-13 of the largest


def _blocks(c, values):
    """the numbers the matrix's 8-bit blocks stand for, dense, and the same of their magnitudes"""
    blocks, _ = O.quantized_blocks(values.double().cpu().numpy(), c.ptr, c.col, c.rows, c.columns)
    dense = lambda b: torch.from_numpy(O.dense(b, c.ptr, c.col, c.rows, c.columns)).to(DEV)
    return dense(blocks), dense(np.abs(blocks))


@pytest.mark.parametrize("y_dtype", TYPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 64, 90, 700])
def test_the_largest_numbers_in_x(n, dtype, y_dtype):
    """their 8-bit form is 2^128; times small values, or zero, that is finite, in every path alike"""
    c = Whole(700, 260, 1.0, 1)
    values = _whole(2, len(c.col), 128, 128).float() * 2.0 ** -122
    values[:, ::3, :] = 0
    c.A.set_values(values)
    a, mag = _blocks(c, values)
    top = torch.finfo(dtype).max
    x = _whole(3, n, 260).to(dtype)
    x[0, 5], x[1, 200], x[n - 1, 259], x[n - 1, 0] = top, -top, top, top
    xq = torch.from_numpy(O.quantized(x.double().cpu().numpy())).to(DEV)
    assert float(xq.max()) == 2.0 ** 128
    want, magnitude = torch.mm(xq, a.t().contiguous()), torch.mm(xq.abs(), mag.t().contiguous())
    for given in (x, quantize(x)):
        extra = EIGHT if y_dtype == BF16 and n > 64 else 0.0
        _close(c.A.product(given, y_dtype), want, 260, magnitude, extra)
    # the gradient of the blocks, from dy small enough for it
    for dy_dtype in (F32, BF16):
        dy = (_whole(4, n, 700) * 2.0 ** -30).to(dy_dtype)
        dy[:, 10] = 0
        d = dy.double()
        want, magnitude = (c.sampled(torch.mm(t.t().contiguous(), u)) for t, u in ((d, xq), (d.abs(), xq.abs())))
        _close(c.A.gradient(dy, quantize(x)), want, 3 * n, magnitude)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 64, 90, 700])
def test_the_largest_numbers_in_the_matrix(n, dtype):
    c = Whole(700, 260, 1.0, 1)
    values = _whole(2, len(c.col), 128, 128).float()
    values[:, 3, 5], values[:, 100, 100] = torch.finfo(F32).max, -torch.finfo(F32).max
    c.A.set_values(values)
    a, mag = _blocks(c, values)
    assert float(a.max()) == 2.0 ** 128
    x = (_whole(3, n, 260) * 2.0 ** (-10 if dtype == F16 else -60)).to(dtype)
    x[:, 4] = 0
    xq = torch.from_numpy(O.quantized(x.double().cpu().numpy())).to(DEV)
    want, magnitude = torch.mm(xq, a.t().contiguous()), torch.mm(xq.abs(), mag.t().contiguous())
    for y_dtype in TYPES:
        extra = EIGHT if y_dtype == BF16 and n > 64 else 0.0
        _close(c.A.product(x, y_dtype), want, 260, magnitude, extra)
    dy = (_whole(4, n, 700) * 2.0 ** -20).to(dtype)
    dy[:, 10] = 0
    d = dy.double()
    _close(c.A.product_t(dy, F32), torch.mm(d, a), 2100, torch.mm(d.abs(), mag))


@pytest.mark.parametrize("n", [5, 90])
@pytest.mark.parametrize("size", [-100, -114, -120, -130])
def test_the_smallest_numbers_in_x_and_the_matrix(n, size):
    """exact down to groups of 2^-115; below, an entry counts with an error of at most 2^-133"""
    c = Whole(300, 260, 1.0, 1)
    small, large = _whole(2, len(c.col), 128, 128).float() * 2.0 ** (size - 3), _whole(3, len(c.col), 128, 128).float() * 2.0 ** 90
    tiny = lambda seed, *shape: _whole(seed, *shape).float() * 2.0 ** (size - 3)
    off = 0.0 if size >= -114 else 2.0 ** -133
    x = tiny(4, n, 260)
    c.A.set_values(large)
    a, _ = _blocks(c, large)
    xq = torch.from_numpy(O.quantized(x.double().cpu().numpy())).to(DEV)
    # sums of whole numbers times one power of two: exact but for what the entries lose
    want, lost = torch.mm(xq, a.t().contiguous()), off * a.abs().sum(1)
    for given in (x, quantize(x)):
        got = c.A.product(given).double()
        assert bool(((got - want).abs() <= lost + 2.0 ** -23 * lost).all())
    dy = _whole(5, n, 300).float() * 2.0 ** 90
    want = c.sampled(torch.mm(dy.double().t().contiguous(), xq))
    assert bool(((c.A.gradient(dy, quantize(x)).double() - want).abs() <= off * 1.001 * n * 2.0 ** 93).all())
    c.A.set_values(small)
    a, _ = _blocks(c, small)
    assert bool(((c.A.product_t(dy).double() - torch.mm(dy.double(), a)).abs() <= off * 1.001 * 300 * 2.0 ** 93).all())


# ---- refusals -------------------------------------------------------------------------------------------------------

def test_more_vectors_than_32_bits_count_are_refused():
    """without memory for them: one entry, broadcast"""
    A = Block8.full(1, 1)
    for n in (2 ** 31, 2 ** 32 + 5):
        many = torch.ones(1, 1, device=DEV, dtype=BF16).expand(n, 1)
        for f in (quantize, A.product, A.linear, A.product_t, lambda x: A.gradient(x, quantize(x[:1]))):
            with pytest.raises(ValueError, match="more than 2"):
                f(many)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_calls_are_not_traced():
    """a trace would hold the results' allocations alone"""
    c = Whole(200, 300, 1.0, 1)
    x, dy, w = _whole(2, 3, 300).float(), _whole(3, 3, 200).float(), c.values.float()
    q = quantize(x)

    def load(scale):
        c.A.load(torch.zeros(c.A.nblocks, 128, 128, dtype=torch.uint8, device=DEV), scale)
        return scale

    def set_values(v):
        c.A.set_values(v)
        return v

    for f, a in ((lambda t: quantize(t).values, x), (lambda t: q.restore() + t, x), (c.A.product, x), (c.A.linear, x), (lambda t: c.A.product(q) + t, dy),
                 (c.A.product_t, dy), (lambda t: c.A.gradient(t, q), dy), (set_values, w),
                 (load, torch.full((c.A.nblocks,), 127, dtype=torch.uint8, device=DEV)), (lambda t: c.A.store()[0] + t, torch.zeros(1, device=DEV))):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (a,), check_trace=False)
    _equal(c.A.product(x), torch.mm(_whole(2, 3, 300), c.dense.t().contiguous()))


# ---- views ----------------------------------------------------------------------------------------------------------

def test_negated_views():
    """z.conj().imag and its like: the memory holds the numbers with the other sign"""
    c = Whole(200, 300, 1.0, 1)
    x, dy = _whole(2, 3, 300), _whole(3, 3, 200)
    neg = lambda a: torch.complex(torch.zeros_like(a), -a).conj().imag
    flat = lambda a: torch._neg_view(-a)
    for view in (neg, flat):
        xv, dv = view(x.float()), view(dy.float())
        assert xv.is_neg() and dv.is_neg()
        q = quantize(xv)
        _equal(q.restore(), x)
        _equal(c.A.product(xv), torch.mm(x, c.dense.t().contiguous()))
        _equal(c.A.product_t(dv), torch.mm(dy, c.dense))
        _equal(c.A.gradient(dv, q), c.sampled(torch.mm(dy.t().contiguous(), x)))
    w = flat(-c.values.float())
    c.A.set_values(w)
    assert c.A.values is w
    _equal(c.A.product(x.float()), -torch.mm(x, c.dense.t().contiguous()))
    with pytest.raises(ValueError, match="out must be"):
        c.A.product(x.float(), out=torch._neg_view(torch.zeros(3, 200, device=DEV)))


# ---- which kernel ---------------------------------------------------------------------------------------------------

def test_wide_and_packed_vectors_change_kernels_together():
    """bf16 results on both sides of the border between the kernels, an eighth of the CUs in tiles of 64 vectors"""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for brows in (1, 2, 5):
        c = Whole(128 * brows - 3, 300, 1.0, brows)
        c.A.set_values(torch.randn(c.values.shape, device=DEV))
        tiles = cus // 8 // brows
        for n in (64, 65, 64 * tiles, 64 * tiles + 1):
            x = torch.randn(n, 300, device=DEV).to(BF16)
            assert torch.equal(c.A.product(x), c.A.product(quantize(x))), (brows, n)


@pytest.mark.parametrize("n", [5, 90, 700])
def test_linear_in_32_bits(n):
    """bf16 vectors into fp32 results: 32-bit sums for any number of them, where the 8-bit instruction would lose the 2^-13 beside 1 - 1"""
    A = Block8.full(128, 128)
    w = torch.ones(1, 128, 128, device=DEV, requires_grad=True)
    A.set_values(w)
    x = torch.zeros(n, 128, dtype=BF16, device=DEV)
    x[:, 0::8], x[:, 1::8], x[:, 2::8] = 1.0, -1.0, 2.0 ** -16
    x.requires_grad_(True)
    y = A.linear(x, F32)
    assert y.dtype == F32 and bool((y == 16 * 2.0 ** -16).all())
    with torch.no_grad():
        assert torch.equal(A.linear(x, F32), y)
    dy = _whole(1, n, 128).float()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dx.dtype == BF16 and dw.dtype == F32
    assert torch.equal(dx, A.product_t(dy, BF16)) and torch.equal(dw, A.gradient(dy, quantize(x)))
    assert A.linear(x).dtype == BF16
