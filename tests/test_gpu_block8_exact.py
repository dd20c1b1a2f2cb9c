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
