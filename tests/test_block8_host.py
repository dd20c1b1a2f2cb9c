"""8-bit block matrices without a GPU: the oracle against torch's own e4m3 conversion, and every refusal that the library
or the Python layer makes before it needs a device."""
import copy
import ctypes as C
import pickle

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import spmv_amd as S
from spmv_amd import block8
from tests import block8_oracle as O


def _fails(rc, text):
    assert rc != 0
    assert text in S.lib().spmv_hip_last_error().decode(), S.lib().spmv_hip_last_error()


def test_oracle_rounds_like_torchs_e4m3():
    x = np.concatenate([np.linspace(-448, 448, 20001), np.exp2(np.linspace(-12, 8, 4001)), [0.0, -0.0, 2.0 ** -10, 1.5 * 2.0 ** -9]])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(O.nearest(x), want)
    codes = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(codes).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(np.nan_to_num(O.decode(codes), nan=-1e9), np.nan_to_num(t, nan=-1e9))


def test_oracle_scale_is_the_least_power_of_two_that_fits():
    rng = np.random.default_rng(0)
    a = np.abs(rng.standard_normal(1000)) * np.exp2(rng.integers(-130, 120, 1000))
    a = np.concatenate([a, [448.0, 448.0 * (1 + 2.0 ** -20), 449.0, 3.4e38, 1e-45]])
    b = O.scale_byte(a[:, None]).astype(np.float64)
    assert np.all(a <= 448 * np.exp2(b - 127))
    assert np.all((a > 448 * np.exp2(b - 128)) | (b == 1))
    assert O.scale_byte(np.zeros((1, 4)))[0] == 127
    assert O.scale_byte(np.array([[np.inf, np.nan, 2.0]]))[0] == O.scale_byte(np.array([[2.0]]))[0]


def _create(rows, columns, ptr, col):
    ptr, col = np.array(ptr, np.int32), np.array(col, np.int32)
    return S.lib().spmv_hip_create_block8(rows, columns, len(col), ptr.ctypes.data, col.ctypes.data)


@pytest.mark.parametrize("rows,columns,ptr,col,text", [
    (-1, 5, [0], [], "negative dimension"),
    (130, 130, [0, 1, 1], [2], "block column 2 out of range"),
    (130, 130, [0, 1, 1], [-1], "block column -1 out of range"),
    (130, 130, [0, 2, 1], [0], "block_ptr decreases"),
    (130, 130, [0, 0, 2], [0], "must equal nblocks"),
    (130, 130, [1, 1, 1], [0], "block_ptr[0] must be 0"),
    (130, 0, [0, 1, 1], [0], "out of range"),
])
def test_creator_refuses_bad_patterns(rows, columns, ptr, col, text):
    assert not _create(rows, columns, ptr, col)
    assert text in S.lib().spmv_hip_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_no_gpu_is_an_error():
    assert not _create(130, 130, [0, 1, 1], [0])
    assert "no HIP device" in S.lib().spmv_hip_last_error().decode()


def test_vector_calls_refuse_bad_arguments():
    L = S.lib()
    p = 4096                                                 # an address that no refused call touches
    q = lambda n=2, cols=200, x=p, dt=S.F32, ldx=200, x8=p, ld8=256, sc=p, lds=2: L.spmv_hip_quantize8_dev(n, cols, x, dt, ldx, x8, ld8, sc, lds, None)
    _fails(q(dt=S.F64), "must be F32, BF16 or F16")
    _fails(q(dt=S.E4M3), "must be F32, BF16 or F16")
    _fails(q(n=-1), "negative vector count")
    _fails(q(cols=-1), "negative length")
    _fails(q(x=None), "NULL vector block")
    _fails(q(ldx=199), "shorter than their length")
    _fails(q(x8=None), "NULL 8-bit")
    _fails(q(sc=None), "NULL 8-bit")
    _fails(q(ld8=128), "multiple of 128 of at least 256")
    _fails(q(ld8=300), "multiple of 128")
    _fails(q(x8=p + 8), "16-byte aligned")
    _fails(q(lds=1), "1 scales per group for 2 vectors")
    r = lambda n=2, cols=200, x8=p, ld8=256, sc=p, lds=2, x=p, dt=S.F32, ldx=200: L.spmv_hip_restore8_dev(n, cols, x8, ld8, sc, lds, x, dt, ldx, None)
    _fails(r(dt=9), "must be F32, BF16 or F16")
    _fails(r(ldx=3), "shorter than their length")
    _fails(r(ld8=255), "multiple of 128")
    assert q(n=0) == 0 and r(n=0) == 0 and q(cols=0) == 0    # nothing to do
    for name, args in (("mult", (None, 1, p, S.F32, 9, None, 0, p, S.F32, 9, None)), ("backward", (None, 1, p, S.F32, 9, p, 128, p, 1, p, S.F32, 9, p, S.F32, 0, p, None)),
                       ("set_values", (None, p, S.F32, None)),
                       ("load", (None, p, p, None)), ("store", (None, p, p, None))):
        _fails(getattr(L, f"spmv_hip_block8_{name}_dev")(*args), "NULL handle")
    assert L.spmv_hip_block8_backward_work(None, 1, p, S.F32, 9, 1, 1) == 0


def test_python_layer_refuses_what_is_not_on_a_gpu():
    with pytest.raises(ValueError, match="no CPU path"):
        block8.quantize(torch.zeros(2, 128))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        block8.quantize(torch.zeros(2, 128, dtype=torch.float64))
    with pytest.raises(TypeError):
        block8.quantize([1.0, 2.0])
    with pytest.raises(ValueError, match="on one GPU"):
        block8.Packed8(torch.zeros(2, 256, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 200, torch.float32)
    with pytest.raises(ValueError, match="contiguous uint8"):
        block8.Packed8(torch.zeros(2, 200, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 200, torch.float32)
    with pytest.raises(ValueError, match="block_ptr has shape"):
        block8.Block8(300, 300, [0, 1], [0])
    assert C.sizeof(S._lib.Info) > 0 and S.FORMAT_NAMES[S.BLOCK8] == "block8"


@pytest.mark.parametrize("columns,shape", [(200, (1, 200)), (200, (3, 200)), (200, (2, 199)), (200, (2, 201)), (200, (400,)), (200, ()), (200, (200,)),
                                           (200, (2, 2, 200)), (200, (-1, -2, 200)), (200, (0, 200)), (-5, None)])
def test_packed_vectors_refuse_a_shape_of_other_vectors(columns, shape):
    """restore() and product() size their results by the shape and write one vector for each of values' rows"""
    groups = max(-(-columns // 128), 0)
    values, scale = torch.zeros(2, groups * 128, dtype=torch.uint8), torch.zeros(groups, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="does not hold 2 vectors|must not be negative"):
        block8.Packed8(values, scale, columns, torch.float32, shape)


def test_packed_vectors_keep_their_parts():
    q = block8.Packed8._made(torch.zeros(2, 256, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 200, torch.float32, (2, 200))
    for name in ("values", "scale", "columns", "dtype", "shape"):
        with pytest.raises(AttributeError, match=name):
            setattr(q, name, (1, 200))
        with pytest.raises(AttributeError, match=name):
            delattr(q, name)
    assert q.shape == (2, 200) and q.n == 2
    for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert other.shape == q.shape and other.dtype == q.dtype and other.columns == 200 and torch.equal(other.values, q.values)


@pytest.mark.parametrize("rows,columns,ptr,col,text", [
    (130, 2 ** 32 + 128, [0, 1, 1], [0], "more than 2\\^31"),     # would be a matrix of 128 columns
    (2 ** 31, 128, [0, 1], [0], "more than 2\\^31"),
    (130, 130, [0, 1, 1], [2 ** 32], "block_col must hold"),      # would be block column 0
    (130, 130, [0, 1, 2 ** 32 + 1], [0], "block_ptr must hold"),
    (130, 130, [0, 1, 1], [0.5], "block_col must hold"),
    (130, 130, [0, 1, float("nan")], [0], "block_ptr must hold"),
])
def test_sizes_that_32_bits_would_change_are_refused(rows, columns, ptr, col, text):
    with pytest.raises(ValueError, match=text):
        block8.Block8(rows, columns, ptr, col)


def test_whole_numbers_of_any_type_make_a_pattern():
    for a in ([0, 1, 2], np.arange(3), np.arange(3, dtype=np.uint64), torch.arange(3), np.array([0.0, 1.0, 2.0])):
        assert np.array_equal(block8._whole("a", a), np.arange(3)) and block8._whole("a", a).dtype == np.int32
    assert block8._whole("a", []).shape == (0,)


def test_linear_refuses_forward_mode():
    """a dual tensor does not require grad: without this its tangent would be dropped"""
    A = object.__new__(block8.Block8)
    A._h, A.columns = None, 128
    t = torch.ones(2, 128)
    with forward_ad.dual_level():
        for x, A.values in ((forward_ad.make_dual(t, t), None), (t, forward_ad.make_dual(torch.ones(1, 128, 128), torch.ones(1, 128, 128)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.linear(x)
    A.values = None
    with pytest.raises(ValueError, match="no CPU path"):
        A.linear(t)


def test_a_result_on_top_of_an_operand_is_refused():
    """where the operand's rows lie, its gaps left out"""
    rng = np.random.default_rng(1)
    buf = torch.zeros(4000, dtype=torch.uint8)
    for k in range(3000):
        dtype = [torch.float32, torch.float16][k % 2]
        size = torch.finfo(dtype).bits // 8
        n, length, gap, at = rng.integers(1, 6), rng.integers(1, 20), rng.integers(0, 30), 4 * rng.integers(0, 200)
        t = buf[at:at + n * (length + gap) * size].view(dtype).view(n, length + gap)[:, :length]
        first, count = 4 * rng.integers(0, 300), rng.integers(1, 60)
        out = buf[first:first + 4 * count].view(torch.float32)
        held = {int(t.data_ptr()) + int(v) * (length + gap) * size + b for v in range(n) for b in range(length * size)}
        want = any(b in held for b in range(out.data_ptr(), out.data_ptr() + 4 * count))
        assert block8._meets(out, t) == want
    A = object.__new__(block8.Block8)
    A._h, A.device = None, torch.device("cpu")
    x = torch.zeros(6, 64)
    assert A._out(None, (3, 64), torch.float32, x).shape == (3, 64)
    assert A._out(x[3:], (3, 64), torch.float32, x[:3]) is not None
    for out in (x[:3], x[2:5]):
        with pytest.raises(ValueError, match="shares memory"):
            A._out(out, (3, 64), torch.float32, x[:3])
    scale = torch.zeros(2, 3, dtype=torch.uint8)
    with pytest.raises(ValueError, match="shares memory"):
        A._out(x[3:], (3, 64), torch.float32, x[:3], x.view(torch.uint8)[5:6, 8:11])
    assert not block8._meets(x[3:], scale) and not block8._meets(x[:0], x) and not block8._meets(x, x[:0])


def test_out_counts_as_changed_in_place():
    """a backward pass that saved the tensor has to notice"""
    A = object.__new__(block8.Block8)
    A._h, A.device = None, torch.device("cpu")
    x, out, w = torch.zeros(3, 64), torch.ones(3, 64), torch.ones(3, 64, requires_grad=True)
    loss = (out * w).sum()
    assert A._out(out, (3, 64), torch.float32, x) is out
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(ValueError, match="requires grad"):
        A._out(w, (3, 64), torch.float32, x)
    with torch.no_grad():
        assert A._out(w, (3, 64), torch.float32, x) is w
    with torch.inference_mode():
        out = torch.ones(3, 64)
        assert A._out(out, (3, 64), torch.float32, x) is out


def test_rounding_inside_the_product_follows_the_devices_cus():
    """more than 64 vectors inside only where the library takes their 8-bit form by the same kernel: block rows times tiles of
    64 vectors at most an eighth of the CUs (spmv_hip_block8_mult_dev)"""
    for cus in (256, 128, 64, 32):
        for rows in (1, 128, 300, 2000, 4096):
            for n in (1, 16, 64, 65, 128, 300, 1024, 1025):
                same = n <= 64 or -(-rows // 128) * -(-n // 64) * 8 <= cus
                assert block8._inside(n, 2, rows, 1, cus) == (same and n <= 1024)
    assert not block8._inside(65, 2, 128, 1, 15) and block8._inside(64, 2, 128, 1, 15)
    assert block8._inside(16, 2, 128, 4249, 256) and not block8._inside(16, 2, 128, 4250, 256)
    assert block8._inside(32, 4, 128, 937, 256) and not block8._inside(32, 4, 128, 938, 256)


def test_more_than_one_launch_takes_is_refused():
    """2^31 - 1 vectors of one entry: 2^27 workgroups of 256 threads"""
    L, p, n = S.lib(), 4096, 2 ** 31 - 1
    _fails(L.spmv_hip_quantize8_dev(n, 1, p, S.BF16, 1, p, 128, p, n, None), "more than one launch takes")
    _fails(L.spmv_hip_restore8_dev(n, 1, p, 128, p, n, p, S.BF16, 1, None), "more than one launch takes")
