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


# ---- no term lost ---------------------------------------------------------------------------------------------------

# rows, columns, share of blocks, vectors: a block and less, ragged edges, 16 waves a row, more block rows than CUs / 8 in every tile size,
# pairs of blocks, cut sums
SHAPES = [(1, 1, 1.0, [1, 33, 70]), (129, 127, 1.0, [1, 17, 64, 65, 128, 515]), (700, 2300, 1.0, [1, 13, 31, 64, 200]), (2000, 1500, 0.5, [3, 33, 130, 777]),
          (4200, 500, 0.7, [40, 1000, 2050]), (500, 4200, 0.7, [16, 700, 2900]), (4100, 4100, 0.6, [5, 64, 333, 1500]), (5200, 200, 0.8, [5, 130, 4000])]


@pytest.mark.parametrize("rows,columns,keep,counts", SHAPES)
def test_whole_numbers_through_every_product(rows, columns, keep, counts):
    """at most 4: sums stay below fp16's largest number too; rounding the exact sum is all that is left"""
    c = Whole(rows, columns, keep, rows + columns)
    c.values = c.values.sign() * (c.values.abs() % 4 + 1)
    c.A.set_values(c.values.float())
    c.dense = torch.from_numpy(O.dense(c.values.cpu().numpy(), c.ptr, c.col, rows, columns)).to(DEV)
    for n in counts:
        x, dy = _whole(n, n, columns, top=4), _whole(n + 1, n, rows, top=4)
        want_y, want_dx, want_dv = torch.mm(x, c.dense.t().contiguous()), torch.mm(dy, c.dense), c.sampled(torch.mm(dy.t().contiguous(), x))
        for dtype in TYPES:
            xt, dt = x.to(dtype), dy.to(dtype)
            q = quantize(xt)
            _equal(q.restore(), x)
            for y_dtype in TYPES:
                want = want_y.to(y_dtype).double()
                _equal(c.A.product(xt, y_dtype), want, n, dtype, y_dtype)
                _equal(c.A.product(q, y_dtype), want, n, dtype, y_dtype)
            for to in (F32, dtype):
                _equal(c.A.product_t(dt, to), want_dx.to(to).double(), n, dtype, to)
                _equal(c.A.gradient(dt, q, to), want_dv.to(to).double(), n, dtype, to)


def _full_mantissas(dtype, seed, *shape):
    """numbers whose last mantissa bit is set, so that every bf16 part of them is needed"""
    bits = {F32: 23, F16: 10, BF16: 7}[dtype]
    g = torch.Generator(device=DEV).manual_seed(seed)
    m = torch.randint(0, 1 << (bits - 1), shape, generator=g, device=DEV).double() * 2 + 1 + 2.0 ** bits
    e = torch.randint(-4, 5, shape, generator=g, device=DEV).double()
    sign = torch.randint(0, 2, shape, generator=g, device=DEV).double() * 2 - 1
    a = (sign * m * torch.exp2(e - bits)).to(dtype)
    assert bool((a.double() == sign * m * torch.exp2(e - bits)).all())
    return a


def _powers(seed, *shape):
    g = torch.Generator(device=DEV).manual_seed(seed)
    e = torch.randint(-3, 4, shape, generator=g, device=DEV).double()
    return torch.exp2(e) * (torch.randint(0, 2, shape, generator=g, device=DEV).double() * 2 - 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns,keep,counts", [(129, 127, 1.0, [1, 31, 32, 33, 128, 2000]), (300, 260, 0.9, [32, 64, 95, 128, 2000]), (2001, 1500, 0.6, [33, 256, 2000]),
                                                      (4200, 4200, 0.7, [32, 70, 1000]), (5200, 200, 0.8, [5, 40, 130]), (500, 4200, 0.7, [64, 1500])])
def test_every_bit_of_dy_reaches_both_gradients(rows, columns, keep, counts, dtype):
    """one entry of dy to a sum, times a power of two: the product is the sum, and needs all of dy's bits.  (The tolerance of K
    additions hides the last part of an fp32 entry, 2^-16 of it, from K = 33 on.)"""
    c = Whole(rows, columns, keep, rows)
    values = _powers(1, len(c.col), 128, 128)
    c.A.set_values(values.float())
    dense = torch.from_numpy(O.dense(values.cpu().numpy(), c.ptr, c.col, rows, columns)).to(DEV)
    for n in counts:
        for seed in (1, 2):
            g = torch.Generator(device=DEV).manual_seed(seed + n)
            # the gradient: every row of A has its one vector
            dy, at = torch.zeros(n, rows, dtype=dtype, device=DEV), torch.randint(0, n, (rows,), generator=g, device=DEV)
            dy[at, torch.arange(rows, device=DEV)] = _full_mantissas(dtype, seed, rows)
            x = _powers(seed + 1, n, columns)
            want = c.sampled(torch.mm(dy.double().t().contiguous(), x))
            _equal(c.A.gradient(dy, quantize(x.float())), want, n, seed)
            # dx: every vector has its one row
            dy, at = torch.zeros(n, rows, dtype=dtype, device=DEV), torch.randint(0, rows, (n,), generator=g, device=DEV)
            dy[torch.arange(n, device=DEV), at] = _full_mantissas(dtype, seed, n)
            _equal(c.A.product_t(dy, F32), torch.mm(dy.double(), dense), n, seed)


def test_no_term_is_lost_past_32_bit_offsets():
    """a matrix of 2.2 GB and blocks of vectors past 2 GB, in whole numbers: sums of 47360 products of at most 64"""
    k = 370
    g = torch.Generator(device=DEV).manual_seed(1)

    def whole(*shape):
        a = torch.randint(-8, 9, shape, generator=g, device=DEV, dtype=torch.int8)
        return a

    A = Block8.full(128 * k, 128 * k)
    v = whole(A.nblocks, 128, 128)
    codes = torch.arange(-8, 9, device=DEV).float().to(torch.float8_e4m3fn).view(torch.uint8)
    v8 = torch.empty(v.shape, dtype=torch.uint8, device=DEV)
    for at in range(0, A.nblocks, 10000):
        v8[at:at + 10000] = codes[v[at:at + 10000].int() + 8]
    A.load(v8, torch.full((A.nblocks,), 127, dtype=torch.uint8, device=DEV))
    del v8
    rows = lambda i: v[i * k:(i + 1) * k].double().permute(1, 0, 2).reshape(128, -1)
    cols = lambda j: v[j::k].double().reshape(-1, 128)
    n = 46000
    x, dy = whole(n, 128 * k).to(BF16), whole(n, 128 * k).to(BF16)
    x[:, ::128] = 8                                          # the scale of every group: all its whole numbers are exact
    q = quantize(x)
    part = {200: quantize(x[-200:]), 3: quantize(x[-3:])}
    y = A.product(q)
    for i in (0, k // 2, k - 1):
        at = slice(128 * i, 128 * (i + 1))
        r, c = rows(i).t().contiguous(), cols(i)
        for m, p in part.items():
            _equal(A.product(p, F32)[:, at], torch.mm(x[-m:].double(), r), "product", i, m)
        dx = A.product_t(dy)
        for t in (slice(0, 300), slice(n - 300, n)):
            _equal(y[t, at], torch.mm(x[t].double(), r).to(BF16).double(), "product", i, t)
            _equal(dx[t, at], torch.mm(dy[t].double(), c).to(BF16).double(), "product_t", i, t)
        _equal(A.product_t(dy[-3:], F32)[:, at], torch.mm(dy[-3:].double(), c), "product_t", i)
        del dx
    del y
    dv = A.gradient(dy, q, BF16)
    for i, j in ((0, 0), (0, k - 1), (k // 2, 7), (k - 1, 0), (k - 1, k - 1)):
        a, b = dy[:, 128 * i:128 * (i + 1)].double().t().contiguous(), x[:, 128 * j:128 * (j + 1)].double().contiguous()
        _equal(dv[i * k + j], torch.mm(a, b).to(BF16).double(), "gradient", i, j)


def test_download_gives_the_pattern():
    c = Whole(700, 520, 0.6, 3)
    assert np.array_equal(c.A.download(S.ARR_ROW_PTR), c.ptr) and np.array_equal(c.A.download(S.ARR_COL), c.col)
    for which in (S.ARR_VAL, S.ARR_SLICE_PTR, S.ARR_ROW_ORDER, S.ARR_TILE_COORD):
        with pytest.raises(S.SpmvHipError, match="not part of format"):
            c.A.download(which)
    empty = Block8(300, 200, [0, 0, 0, 0], [])
    assert np.array_equal(empty.download(S.ARR_ROW_PTR), np.zeros(4)) and empty.download(S.ARR_COL).shape == (0,)


# ---- the pipelines' ends --------------------------------------------------------------------------------------------

def _rows_of(lengths, bcols, seed):
    """a pattern whose block rows hold `lengths` blocks"""
    rng = np.random.default_rng(seed)
    col = [sorted(rng.permutation(bcols)[:k]) for k in lengths]
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32), np.concatenate(col).astype(np.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [130, 1000, 2100, 4103])
def test_block_rows_and_columns_of_every_length_give_the_same_bits(n, dtype):
    """1 to 13 blocks: whole rounds of 2, 3 or 4 stages and every number of steps after them, in tiles of 64, 128 and 256 vectors;
    a stage read before its loads have arrived is wrong now and then, so every product is repeated"""
    lengths = [5, 1, 2, 3, 4, 5, 0, 6, 7, 8, 9, 10, 11, 12, 13, 5, 8]
    for turned in (False, True):
        ptr, col = _rows_of(lengths, 16, n)
        rows, columns = 128 * len(lengths) - 70, 16 * 128 - 30
        if turned:                                           # the lengths are those of block columns
            place = sorted((c, r) for r in range(len(lengths)) for c in col[ptr[r]:ptr[r + 1]])
            rows, columns = columns, rows
            ptr = np.array([sum(1 for p in place if p[0] < r) for r in range(17)], np.int32)
            col = np.array([p[1] for p in place], np.int32)
        values = _whole(n, len(col), 128, 128, top=4)
        A = Block8(rows, columns, ptr, col)
        A.set_values(values.float())
        a = torch.from_numpy(O.dense(values.cpu().numpy(), ptr, col, rows, columns)).to(DEV)
        x, dy = _whole(n, n, columns, top=4), _whole(n + 1, n, rows, top=4)
        q, d = quantize(x.to(dtype)), dy.to(dtype)
        y, dx = torch.mm(x, a.t().contiguous()), torch.mm(dy, a)
        for k in range(20):
            for to in TYPES:
                _equal(A.product(q, to), y.to(to).double(), to, k)
            _equal(A.product_t(d, dtype), dx.to(dtype).double(), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(128, 128), (1300, 1300), (2600, 2600), (4200, 4200)])
def test_gradients_of_every_number_of_vectors_give_the_same_bits(rows, columns, dtype):
    """1 to 9 steps of 32 vectors and what is left, single blocks and pairs"""
    c = Whole(rows, columns, 0.7 if rows > 2600 else 1.0, rows)
    for n in [32 * k + r for k in range(1, 10) for r in (0, 5)]:
        x, dy = _whole(n, n, columns), _whole(n + 1, n, rows)
        q, d = quantize(x.to(dtype)), dy.to(dtype)
        want = c.sampled(torch.mm(dy.t().contiguous(), x))
        for k in range(4):
            _equal(c.A.gradient(d, q), want, n, k)


def test_the_largest_number_of_vectors():
    """2^31 - 1: rounding their number up to whole tiles passes 32 bits"""
    n = 2 ** 31 - 1
    A = Block8(1, 0, [0, 0], [])                            # neither product here reads or writes past 2^31 - 1 vectors
    q = Packed8(torch.empty(n, 0, dtype=torch.uint8, device=DEV), torch.empty(0, n, dtype=torch.uint8, device=DEV), 0, BF16)
    y = torch.full((n, 1), float("nan"), dtype=BF16, device=DEV)
    A.product(q, out=y)
    assert int(torch.count_nonzero(y)) == 0
    del y
    A = Block8.full(8, 1)
    A.set_values(torch.ones(1, 128, 128, device=DEV))
    dy = torch.zeros(n, 8, dtype=BF16, device=DEV)
    dy[0, 3], dy[n - 1, 7], dy[n - 1, 0], dy[2 ** 30, 5] = 1, 2, 3, 4
    dx = A.product_t(dy)
    assert int(torch.count_nonzero(dx)) == 3 and [float(dx[k, 0]) for k in (0, n - 1, 2 ** 30)] == [1, 5, 4]


# ---- every number ---------------------------------------------------------------------------------------------------

def _same_numbers(got, want):
    """equal, NaN where NaN"""
    got = got.double().cpu().numpy()
    assert got.shape == want.shape and np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok]), (int((got[ok] != want[ok]).sum()), got[ok][got[ok] != want[ok]][:3], want[ok][got[ok] != want[ok]][:3])


@pytest.mark.parametrize("dtype", TYPES)
def test_every_number_to_8_bits(dtype):
    """all 16-bit numbers (of fp32 a million bit patterns), alone and beside larger ones that set the scale"""
    if dtype == F32:
        g = torch.Generator().manual_seed(1)
        bits = torch.randint(-2 ** 31, 2 ** 31, (1 << 20,), generator=g).to(torch.int32)
        bits[:1 << 19] &= ~0xfffff                           # near the borders of 8 bits
        x = bits.view(F32)
    else:
        x = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16).view(dtype)
    for up in (0, 1, 4, 9, 18):
        big = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).double()
        beside = torch.minimum(big * 1.5 * 2.0 ** up, torch.full_like(big, torch.finfo(dtype).max)).to(dtype) if up else torch.zeros_like(x)
        v = torch.stack((x, beside), 1)
        q = quantize(v.to(DEV))
        want, b = O.quantize(v.double().numpy())
        assert np.array_equal(q.scale.cpu().numpy(), b)
        _same_numbers(q.values.view(torch.float8_e4m3fn), want)
        A = Block8.full(1, 2)                                # rounded inside the product: the same
        w = torch.zeros(1, 128, 128)
        w[0, 0, 0] = 1
        A.set_values(w.to(DEV))
        ok = torch.isfinite(v).all(1) & torch.from_numpy(b[0] >= 4)
        y = torch.cat([A.product(p, F32) for p in v[ok].to(DEV).split(1024)])
        exact = O.quantized(v[ok].double().numpy())[:, :1]
        _same_numbers(y, np.where(np.abs(exact) > torch.finfo(F32).max, np.copysign(np.inf, exact), exact))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_back(dtype):
    """256 codes times 247 scales; past the type's largest number that number"""
    code, byte = torch.arange(256, dtype=torch.uint8), torch.arange(1, 248, dtype=torch.uint8)
    q = Packed8(code.repeat(247, 1).to(DEV), byte.repeat(2, 1).contiguous().to(DEV), 256, dtype)
    want = O.decode(code.numpy())[None] * np.exp2(byte.numpy().astype(np.float64) - 127)[:, None]
    top = torch.finfo(dtype).max
    with np.errstate(invalid="ignore"):
        want = torch.from_numpy(np.clip(want, -top, top)).to(dtype).double().numpy()
    _same_numbers(q.restore(), want)
