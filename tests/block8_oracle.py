"""The 8-bit block format and its products in 64 bits with numpy: what tests/test_gpu_block8.py compares with."""
import numpy as np

B = 128


def decode(codes):
    """e4m3 bytes -> float64 (0x7f and 0xff are NaN)"""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * np.exp2(e - 7.0), m / 8.0 * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(s == 1, -v, v)


def scale_byte(groups):
    """groups [..., k] -> byte b: the least power of two 2^(b-127) >= 2^-126 with max |finite| <= 448 * 2^(b-127)"""
    g = np.asarray(groups, np.float64)
    a = np.where(np.isfinite(g), np.abs(g), 0.0).max(-1)
    m, e = np.frexp(a)                                       # a = m 2^e, 448 = 0.875 * 2^9
    k = np.where(m <= 0.875, e - 9, e - 8)
    return np.where(a == 0, 127, np.maximum(k, -126) + 127).astype(np.uint8)


def nearest(x):
    """float64 -> the nearest e4m3 number, ties to even; NaN for anything not finite"""
    x = np.asarray(x, np.float64)
    fin = np.isfinite(x)
    a = np.where(fin, np.abs(x), 0.0)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))
    step = np.exp2(e - 4.0)
    return np.where(fin, np.copysign(np.rint(a / step) * step, np.where(fin, x, 0.0)), np.nan)


def quantize(x):
    """x [n, columns] -> (values [n, groups * 128] before scaling, scale bytes [groups, n])"""
    x = np.asarray(x, np.float64)
    n, columns = x.shape
    groups = -(-columns // B)
    p = np.zeros((n, groups * B))
    p[:, :columns] = x
    p = p.reshape(n, groups, B)
    b = scale_byte(p)
    return nearest(p / np.exp2(b.astype(np.float64) - 127)[..., None]).reshape(n, groups * B), np.ascontiguousarray(b.T)


def quantized(x):
    """the numbers that the 8-bit form of x stands for"""
    v, b = quantize(x)
    return (v.reshape(v.shape[0], -1, B) * np.exp2(b.T.astype(np.float64) - 127)[..., None]).reshape(v.shape[0], -1)[:, :np.shape(x)[1]]


def quantized_blocks(blocks, ptr, col, rows, columns):
    """blocks [nb, 128, 128] -> the numbers their 8-bit form stands for, zero beyond the matrix's edge; scale bytes"""
    v = np.array(blocks, np.float64)
    for r in range(len(ptr) - 1):
        for k in range(ptr[r], ptr[r + 1]):
            v[k, max(rows - r * B, 0):, :] = 0
            v[k, :, max(columns - col[k] * B, 0):] = 0
    b = scale_byte(v.reshape(len(v), B * B)) if len(v) else np.zeros(0, np.uint8)
    s = np.exp2(b.astype(np.float64) - 127)[:, None, None]
    return nearest(v / s) * s, b


def dense(blocks, ptr, col, rows, columns):
    """the matrix [rows, columns]; blocks at one place add up"""
    a = np.zeros((-(-rows // B) * B, -(-columns // B) * B))
    for r in range(len(ptr) - 1):
        for k in range(ptr[r], ptr[r + 1]):
            a[r * B:(r + 1) * B, col[k] * B:(col[k] + 1) * B] += blocks[k]
    return a[:rows, :columns]


def sampled(full, ptr, col):
    """full [rows, columns] at the stored blocks, zero beyond its edge"""
    rows, columns = full.shape
    p = np.zeros((-(-rows // B) * B, -(-columns // B) * B))
    p[:rows, :columns] = full
    out = [p[r * B:(r + 1) * B, col[k] * B:(col[k] + 1) * B] for r in range(len(ptr) - 1) for k in range(ptr[r], ptr[r + 1])]
    return np.stack(out) if out else np.zeros((0, B, B))


def pattern(rows, columns, keep, seed):
    """A random pattern of blocks with an empty block row and an empty block column where there is room for them."""
    rng = np.random.default_rng(seed)
    brows, bcols = -(-rows // B), -(-columns // B)
    ptr, col = [0], []
    for r in range(brows):
        here = [c for c in range(bcols) if rng.random() < keep]
        if brows > 2 and r == 1:
            here = []
        if bcols > 2:
            here = [c for c in here if c != 1]
        rng.shuffle(here)                                    # any order inside a block row
        col += here
        ptr.append(len(col))
    return np.array(ptr, np.int32), np.array(col, np.int32)
