"""What is measured of the products with a matrix of 128 x 128 blocks held in 8 bits.

Five kinds of pass, each as a program makes it:

  checkpoint   activations to 8 bits (e4m3, one power-of-two scale per 128 along a vector) and back
  product      y = A x for n vectors: one token, a handful, a prompt
  transposed   dx = A^T dy, the gradient of the product's input
  gradient     the gradient of A's stored blocks, from dy and the 8-bit checkpoint of x
  step         a linear layer's whole training step: the values to 8 bits, the product, both gradients

With `own` false the passes are computed in elementary torch operations in 32 bits; with `own` true they are calls of
spmv_amd.block8.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token's activations on their way into a checkpoint: all latency
        dict(name="checkpoint_one_token", kind="checkpoint", n=1, columns=4096, dtype="bf16"),
        # a training batch's activations, 16 k tokens wide 8 k: all bandwidth
        dict(name="checkpoint_batch", kind="checkpoint", n=16384, columns=8192, dtype="bf16"),
        # answering token by token with every block of the layer stored
        dict(name="product_one_token", kind="product", n=1, rows=4096, columns=4096, keep=1.0, dtype="bf16", packed=False),
        # thirteen sequences answered together; a pruned layer with ragged edges
        dict(name="product_thirteen_tokens", kind="product", n=13, rows=14000, columns=5000, keep=0.25, dtype="f16", packed=False),
        # a prompt of odd length through a half-full layer, its activations in 8 bits already
        dict(name="product_prompt", kind="product", n=777, rows=5000, columns=2900, keep=0.5, dtype="f32", packed=True),
        # a training batch through a full layer
        dict(name="product_batch", kind="product", n=8192, rows=8192, columns=8192, keep=1.0, dtype="bf16", packed=False),
        # the input's gradient of a short odd batch in 32 bits
        dict(name="transposed_ragged", kind="transposed", n=333, rows=2500, columns=4100, keep=0.4, dtype="f32"),
        # the input's gradient of a training batch
        dict(name="transposed_batch", kind="transposed", n=8192, rows=8192, columns=8192, keep=1.0, dtype="bf16"),
        # the values' gradient of a pruned layer, odd batch
        dict(name="gradient_ragged", kind="gradient", n=1001, rows=2500, columns=4100, keep=0.4, dtype="f16"),
        # the values' gradient of a training batch, into 32-bit master gradients
        dict(name="gradient_batch", kind="gradient", n=8192, rows=8192, columns=8192, keep=1.0, dtype="bf16"),
        # a small layer's training step: many launches, little work
        dict(name="step_small", kind="step", n=64, rows=1024, columns=1024, keep=0.5, dtype="bf16"),
        # a large pruned layer's training step
        dict(name="step_pruned", kind="step", n=4096, rows=8192, columns=8192, keep=0.25, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["checkpoint", "product", "transposed", "gradient", "step"])
    case = dict(kind=kind, n=_spread(rng, 1, 8192), columns=_spread(rng, 100, 8192), dtype=rng.choice(["bf16", "f16", "f32"]))
    if kind != "checkpoint":
        case.update(rows=_spread(rng, 100, 8192), keep=rng.choice([0.1, 0.25, 0.5, 0.75, 1.0]))
    if kind == "product":
        case["packed"] = rng.random() < 0.5
    if kind == "step":
        case["n"] = min(case["n"], 2500)        # three products
    return case


def _groups(length):
    return (length + BLOCK - 1) // BLOCK


def _blocks_per_row(case):
    """Stored blocks of every block row: about `keep` of them, uneven, with empty block rows among them."""
    brows, bcols = _groups(case["rows"]), _groups(case["columns"])
    if case["keep"] >= 1.0:
        return [bcols] * brows
    k = max(1, round(case["keep"] * bcols))
    return [0 if i % 11 == 10 else min(bcols, max(0, k + (i * 7 + 1) % 3 - 1)) for i in range(brows)]


def _pattern(case, seed):
    bcols = _groups(case["columns"])
    gen = torch.Generator().manual_seed(seed * 7919 + 13)
    ptr, col = [0], []
    for k in _blocks_per_row(case):
        col += sorted(torch.randperm(bcols, generator=gen)[:k].tolist())
        ptr.append(len(col))
    return ptr, col


# ---- the number format in elementary operations --------------------------------------------------------------------

def _power(exponent):
    """2^exponent as float32, exactly, for -126 <= exponent <= 127."""
    return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _scale_exponent(groups):
    """Least e >= -126 with the largest finite magnitude of the last axis <= 448 * 2^e; 0 for a group of zeros."""
    finite = torch.where(torch.isfinite(groups), groups.abs(), torch.zeros_like(groups))
    mantissa, exponent = torch.frexp(finite.amax(-1))
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-126)
    return torch.where(mantissa == 0, torch.zeros_like(e), e).to(torch.int32)


def _to8(groups):
    """groups [..., 128 or more] in 32 bits -> (e4m3 tensor, exponent per group)"""
    e = _scale_exponent(groups)
    return (groups * _power(-e)[..., None]).to(torch.float8_e4m3fn), e


def _pack_vectors(x):
    n, columns = x.shape
    pad = _groups(columns) * BLOCK - columns
    wide = torch.nn.functional.pad(x.float(), (0, pad)) if pad else x.float()
    return _to8(wide.view(n, _groups(columns), BLOCK))


def _unpack_vectors(x8, e, columns):
    wide = x8.float() * _power(e)[..., None]
    return wide.reshape(x8.shape[0], -1)[:, :columns]


def _dense(case, ptr, col, values8, exponents):
    """The matrix [rows, columns] in 32 bits."""
    brows, bcols = _groups(case["rows"]), _groups(case["columns"])
    dense = torch.zeros(brows, BLOCK, bcols, BLOCK, dtype=torch.float32, device="cuda")
    block_row = torch.repeat_interleave(torch.arange(brows, device="cuda"), ptr[1:] - ptr[:-1], output_size=len(col))
    dense[block_row, :, col.long(), :] = values8.float() * _power(exponents)[:, None, None]
    return dense.view(brows * BLOCK, bcols * BLOCK)[:case["rows"], :case["columns"]]


def _sampled(case, ptr, col, dy, x):
    """(dy^T x) at the stored blocks, [blocks, 128, 128], zero beyond the matrix's edges."""
    brows, bcols = _groups(case["rows"]), _groups(case["columns"])
    full = torch.zeros(brows * BLOCK, bcols * BLOCK, dtype=torch.float32, device="cuda")
    full[:case["rows"], :case["columns"]] = dy.t() @ x
    block_row = torch.repeat_interleave(torch.arange(brows, device="cuda"), ptr[1:] - ptr[:-1], output_size=len(col))
    return full.view(brows, BLOCK, bcols, BLOCK)[block_row, :, col.long(), :]


# ---- inputs --------------------------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """Tensors of the case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, n, columns = TYPES[case["dtype"]], case["n"], case["columns"]
    t = {}
    # activations: channels of unlike size, a few far larger than the rest
    channel = torch.exp(0.5 * _normal(gen, columns))
    channel[torch.rand(columns, generator=gen, device="cuda") < 0.004] *= 20.0
    t["x"] = (_normal(gen, n, columns) * channel).to(dt)
    if case["kind"] == "checkpoint":
        return t
    ptr, col = _pattern(case, seed)
    t["host_ptr"], t["host_col"] = ptr, col
    t["ptr"] = torch.tensor(ptr, dtype=torch.int32, device="cuda")
    t["col"] = torch.tensor(col, dtype=torch.int32, device="cuda")
    # the layer's values, blocks of unlike size
    size = 0.02 * torch.exp2(2.0 * torch.rand(len(col), 1, 1, generator=gen, device="cuda") - 1.0)
    t["values"] = _normal(gen, len(col), BLOCK, BLOCK) * size
    if case["kind"] != "step":
        v8, e = _to8(t.pop("values").view(len(col), BLOCK * BLOCK))
        t["values8"], t["exponents"] = v8.view(len(col), BLOCK, BLOCK), e
    if case["kind"] in ("transposed", "gradient", "step"):
        token = 1e-2 * torch.exp2(2.0 * _normal(gen, n, 1))
        t["dy"] = (_normal(gen, n, case["rows"]) * token).to(dt)
    if case.get("packed") or case["kind"] == "gradient":
        t["x8"], t["x_exponents"] = _pack_vectors(t.pop("x"))
    return t


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["kind"] == "step":
        state["x"].requires_grad_(True)
        state["values"].requires_grad_(True)
    if own:
        from spmv_amd import block8
        if case["kind"] != "checkpoint":
            a = block8.Block8(case["rows"], case["columns"], state["host_ptr"], state["host_col"])
            if "values8" in state:
                a.load(state["values8"], (state["exponents"] + 127).to(torch.uint8))
            state["matrix"] = a
        if "x8" in state:
            n = case["n"]
            state["packed"] = block8.Packed8(state["x8"].view(torch.uint8).view(n, -1),
                                             (state["x_exponents"] + 127).to(torch.uint8).t().contiguous(),
                                             case["columns"], TYPES[case["dtype"]])
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(s):
    case = s["case"]
    kind, dt, columns = case["kind"], TYPES[case["dtype"]], case["columns"]
    with torch.no_grad():
        if kind == "checkpoint":
            x8, e = _pack_vectors(s["x"])
            return _unpack_vectors(x8, e, columns).to(dt), (e + 127).t().to(torch.uint8)
        if kind == "step":
            blocks = len(s["host_col"])
            v8, ve = _to8(s["values"].view(blocks, BLOCK * BLOCK))
            a = _dense(case, s["ptr"], s["col"], v8.view(blocks, BLOCK, BLOCK), ve)
            x = _unpack_vectors(*_pack_vectors(s["x"]), columns)
            dy = s["dy"].float()
            return (x @ a.t()).to(dt), (dy @ a).to(dt), _sampled(case, s["ptr"], s["col"], dy, x)
        if kind == "gradient":
            return _sampled(case, s["ptr"], s["col"], s["dy"].float(), _unpack_vectors(s["x8"], s["x_exponents"], columns))
        a = _dense(case, s["ptr"], s["col"], s["values8"], s["exponents"])
        if kind == "transposed":
            return (s["dy"].float() @ a).to(dt)
        x8, e = (s["x8"], s["x_exponents"]) if case["packed"] else _pack_vectors(s["x"])
        return (_unpack_vectors(x8, e, columns) @ a.t()).to(dt)


def _run_own(s):
    from spmv_amd import block8
    kind = s["case"]["kind"]
    if kind == "checkpoint":
        q = block8.quantize(s["x"])
        return q.restore(), q.scale
    a = s["matrix"]
    if kind == "product":
        return a.product(s["packed"] if "packed" in s else s["x"])
    if kind == "transposed":
        return a.product_t(s["dy"])
    if kind == "gradient":
        return a.gradient(s["dy"], s["packed"])
    a.set_values(s["values"])
    y = a.linear(s["x"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["values"]), s["dy"]))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    n, columns, size = case["n"], case["columns"], SIZE[case["dtype"]]
    wide = n * columns * size
    eight = n * columns + n * _groups(columns)
    if case["kind"] == "checkpoint":
        # in, out, and the 8-bit form that lies in memory between the two
        return {"bytes": 2 * wide + 2 * eight, "flops": 4 * n * columns}
    rows = case["rows"]
    blocks = sum(_blocks_per_row(case))
    matrix = blocks * (BLOCK * BLOCK + 1)
    out = n * rows * size
    flops = 2 * n * blocks * BLOCK * BLOCK
    if case["kind"] == "product":
        return {"bytes": matrix + (eight if case["packed"] else wide) + out, "flops": flops}
    if case["kind"] == "transposed":
        return {"bytes": matrix + wide + out, "flops": flops}
    if case["kind"] == "gradient":
        return {"bytes": 4 * blocks * BLOCK * BLOCK + eight + out, "flops": flops}
    # x, the values and dy in; y, dx and the values' gradient out
    return {"bytes": 2 * wide + 2 * out + 8 * blocks * BLOCK * BLOCK, "flops": 3 * flops}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _power64(e):
    """2^e as float64 for whole e, exactly"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest8(x):
    """Scaled values (64 bits, |x| <= 448) to the nearest e4m3 number, ties to even: steps of 2^(k-3) between 2^k and
    2^(k+1), of 2^-9 below 2^-6."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = _power64(e - 4)
    return torch.round(x / step) * step


def _rounded(groups):
    """groups [..., k] -> the numbers their 8-bit form stands for, in 64 bits, and log2 of the scales"""
    g = groups.double()
    largest = g.abs().amax(-1)
    s = torch.ceil(torch.log2(torch.where(largest > 0, largest, torch.full_like(largest, 448.0)) / 448.0))
    # log2 may be off by an ulp beside a power of two
    s = torch.where(largest > 448.0 * _power64(s), s + 1, s)
    s = torch.where((largest > 0) & (largest <= 448.0 * _power64(s - 1)), s - 1, s).clamp(min=-126)
    scale = _power64(s)[..., None]
    return _nearest8(g / scale) * scale, s


def _rounded_vectors(x):
    n, columns = x.shape
    wide = torch.zeros(n, _groups(columns) * BLOCK, dtype=torch.float64, device=x.device)
    wide[:, :columns] = x
    value, s = _rounded(wide.view(n, -1, BLOCK))
    return value.view(n, -1)[:, :columns], s


def exact(case, seed):
    t = _inputs(case, seed)
    kind, rows, columns = case["kind"], case.get("rows"), case["columns"]
    if kind == "checkpoint":
        value, s = _rounded_vectors(t["x"])
        return value, (s + 127).t().to(torch.uint8)
    if "x8" in t:
        x = (t["x8"].double() * _power64(t["x_exponents"])[..., None]).flatten(1)[:, :columns]
    else:
        x, _ = _rounded_vectors(t["x"])
    if kind == "step":
        blocks, _ = _rounded(t["values"].flatten(1))
        blocks = blocks.view(-1, BLOCK, BLOCK)
    else:
        blocks = t["values8"].double() * _power64(t["exponents"])[:, None, None]
    a = torch.zeros(_groups(rows) * BLOCK, _groups(columns) * BLOCK, dtype=torch.float64, device="cuda")
    places = [(i, j) for i in range(_groups(rows)) for j in t["host_col"][t["host_ptr"][i]:t["host_ptr"][i + 1]]]
    if kind != "gradient":
        for k, (i, j) in enumerate(places):
            a[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] = blocks[k]
    a = a[:rows, :columns]
    if kind == "product":
        return torch.mm(x, a.t())
    dy = t["dy"].double()
    if kind == "transposed":
        return torch.mm(dy, a)
    whole = torch.zeros(_groups(rows) * BLOCK, _groups(columns) * BLOCK, dtype=torch.float64, device="cuda")
    whole[:rows, :columns] = torch.mm(dy.t(), x)
    dv = torch.stack([whole[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] for i, j in places])
    return dv if kind == "gradient" else (torch.mm(x, a.t()), torch.mm(dy, a), dv)
