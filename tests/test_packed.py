"""Packed 4-bit weights: layout, products with their gradients, lookups, and the embedding's gradient.

Plain implementations in 64 bits stand beside every call.  Two kinds of check:

- exact: integer activations and scales that are powers of two make every product and sum exact in the
  kernels' arithmetic (all partial sums are integers times one power of two below 2^24), so the result is
  the 64-bit one rounded once to its type, bit for bit, on every path;
- bounded: for general values the distance is at most what the roundings allow, with S = sum |x| |W|:
  half a step of the result, 2^-23 S per term summed (the tensor cores truncate their fp32 sums, so a
  whole step), and where W itself is rounded to 16 bits half a step of S, twice 2^-11 more for the
  second part of its scale.
"""

import ctypes as C

import pytest
import torch

ROOT_DEV = "cuda:0"


def entry(m, n, strategy="group", group=128, sym=False, bits=4, seed=0, pow2=False, device="cpu"):
    """Random codes of an [m, n] weight as the quantisers write them, and W in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    groups = {"tensor": 1, "channel": 1, "group": -(-n // group)}[strategy]
    rows = 1 if strategy == "tensor" else m
    if pow2:
        scales = torch.exp2(torch.randint(-6, -2, (rows, groups), generator=g).float())
    else:
        scales = (torch.rand(rows, groups, generator=g) + 0.1) * 0.02
    top = 2 ** (bits - 1) - 1 if sym else 2 ** bits - 1
    zps = torch.zeros(rows, groups, dtype=torch.int32) if sym else torch.randint(0, top + 1, (rows, groups), generator=g, dtype=torch.int32)
    col = torch.arange(n) // group if strategy == "group" else torch.zeros(n, dtype=torch.long)
    q = torch.randint(-top if sym else 0, top + 1, (m, n), generator=g, dtype=torch.int32)
    z, s = zps.expand(m, groups)[:, col], scales.expand(m, groups)[:, col]
    stored = (q - z) & 0xF
    if n % 2:
        stored = torch.cat([stored, torch.zeros(m, 1, dtype=torch.int32)], 1)
    codes = (stored[:, 0::2] * 16 + stored[:, 1::2]).to(torch.uint8)
    shape = {"tensor": (1,), "channel": (m,), "group": (m, groups)}[strategy]
    e = {"codes": codes.to(device), "scales": scales.reshape(shape).to(device), "zero_points": zps.reshape(shape).to(device),
         "num_bits": bits, "symmetric": sym, "strategy": strategy, "group_size": group}
    return e, (q - z).double() * s.double()


def half_step(t):
    return torch.finfo(t).eps / 2


def weight(e, n):
    from llmcompressorsharp_b200 import Int4Weight

    return Int4Weight.from_entry(e, n)


def check_product(got, x, w, bias=None, rounded=False):
    """got against x W^T + bias (x, W in 64 bits on the CPU)."""
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, s = y + bias, s + bias.abs()
    bound = half_step(got.dtype) * y.abs() + (x.shape[1] + 8) * 2.0 ** -23 * s + 1e-30
    if rounded and got.dtype != torch.float32:
        bound += (half_step(got.dtype) + 2 * half_step(got.dtype) ** 2) * s * (1 + half_step(got.dtype))
    bound += torch.finfo(got.dtype).tiny
    bad = (got.double().cpu() - y).abs() - bound
    assert not bool((bad > 0).any()), f"off by {bad.max().item():.3g} more than the roundings allow"


# ------------------------------------------------------------------------------ refusals (CPU)
def test_layout_sizes_and_their_refusals():
    from llmcompressorsharp_b200 import _lib

    lib = _lib.load()
    p, x = C.c_int64(), C.c_int64()

    def sizes(rows, cols, group):
        return lib.llmc_int4_layout_sizes(rows, cols, group, C.byref(p), C.byref(x))

    # records of 16 rows x 128 columns: 1,024 bytes of codes, 80 for each group in the 128 columns
    assert sizes(100, 576, 128) == 0 and (p.value, x.value) == (8 * 5 * 1104, 128 + 5)
    # twelve groups of 50 columns take 64 each: two to a record
    assert sizes(129, 600, 50) == 0 and (p.value, x.value) == (16 * 6 * 1184, 256 + 12)
    assert sizes(16, 96, 32) == 0 and (p.value, x.value) == (8 * 1344, 128 + 4)
    assert sizes(1, 5, 8) == 0 and (p.value, x.value) == (8 * 1104, 128 + 1)
    assert sizes(0, 5, 8) == 2 and sizes(5, 0, 8) == 2  # LLMC_ERR_SHAPE
    assert sizes(5, 64, 15) == 3  # LLMC_ERR_UNSUPPORTED
    assert sizes(1 << 31, 64, 64) == 10  # LLMC_ERR_OUT_OF_RANGE
    assert lib.llmc_int4_layout_sizes(4, 4, 4, None, None) == 1


def test_null_arguments_are_statuses():
    from llmcompressorsharp_b200 import _lib

    lib = _lib.load()
    n = C.c_int64()
    assert lib.llmc_int4_layout(None, None, None, 1, None, None, 0, 1, None) == 1
    assert lib.llmc_int4_dequantize(None, None, None, 0, None, 1) == 1
    assert lib.llmc_int4_linear(None, None, None, None, 0, 1, 1, None, None, 1, None, 0) == 1
    assert lib.llmc_int4_linear_grad(None, None, None, None, 0, 1, 1, None, 1, None, 0) == 1
    assert lib.llmc_int4_linear_workspace(None, None, None, 0, 1, 1, C.byref(n)) == 1
    assert lib.llmc_int4_linear_grad_workspace(None, None, None, 0, 1, 1, C.byref(n)) == 1
    assert lib.llmc_col_sum(None, None, None, 0, 1, 1, 1, None, None, 0) == 1
    assert lib.llmc_embedding(None, None, None, 1, 1, None, 0, 1, 1, 1, 1.0, None, 1) == 1
    assert lib.llmc_int4_embedding(None, None, None, 1, 1, None, 0, 1.0, None, 1) == 1
    assert lib.llmc_embedding_grad(None, None, None, 1, 1, None, 0, 1, 1, 1, 1.0, -1, None, None, 0) == 1
    assert lib.llmc_embedding_grad_workspace(None, 1, 1, 1, C.byref(n)) == 1


def test_weight_refusals():
    from llmcompressorsharp_b200 import Int4Weight
    from llmcompressorsharp_b200.errors import ArgumentError, InvalidOperationError, NotSupportedError, ShapeError

    e, _ = entry(8, 64, group=32)
    for key, value, error in (("num_bits", 8, NotSupportedError), ("strategy", "token", NotSupportedError),
                              ("zero_points", None, ArgumentError), ("codes", None, ArgumentError),
                              ("codes", e["codes"][:, :-1], ShapeError), ("codes", e["codes"].int(), ShapeError),
                              ("scales", e["scales"][:, :1], ShapeError), ("zero_points", e["zero_points"][:3], ShapeError),
                              ("group_size", 8, NotSupportedError),
                              ("scales", e["scales"].clone().requires_grad_(True), InvalidOperationError)):
        with pytest.raises(error):
            Int4Weight.from_entry({**e, key: value}, 64)
    with pytest.raises(ArgumentError):
        Int4Weight.from_entry(None, 64)


def test_call_refusals_without_a_device():
    from llmcompressorsharp_b200 import embedding, int4_linear
    from llmcompressorsharp_b200.errors import ArgumentError, ShapeError

    x = torch.zeros(2, 4)
    for call, error in ((lambda: int4_linear(None, None), ArgumentError), (lambda: int4_linear(x, x), ArgumentError),
                        (lambda: embedding(None, x), ArgumentError), (lambda: embedding(x, x), ArgumentError),
                        (lambda: embedding(x.long(), x[0]), ShapeError), (lambda: embedding(x.long(), x.double()), ArgumentError),
                        (lambda: embedding(x.long(), x), ArgumentError),  # a table on the CPU
                        (lambda: embedding(x.long(), x, dtype=torch.float16), ArgumentError)):
        with pytest.raises(error):
            call()


# ------------------------------------------------------------------------------ GPU
GRIDS = [("group", 128, False, 4), ("group", 64, True, 4), ("group", 32, False, 4), ("group", 96, True, 3), ("group", 50, False, 4),
         ("group", 16, False, 2), ("channel", 1, False, 4), ("tensor", 1, True, 4)]
SHAPES = [(1, 1), (16, 32), (37, 100), (128, 128), (131, 577), (300, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("strategy,group,sym,bits", GRIDS)
@pytest.mark.parametrize("m,n", SHAPES)
def test_layout_reads_back(m, n, strategy, group, sym, bits):
    e, w = entry(m, n, strategy, group, sym, bits, seed=m + n, device=ROOT_DEV)
    p = weight(e, n)
    assert p.shape == (m, n)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(p.dequantize(t).cpu(), w.float().to(t))
    ids = torch.randint(0, m, (3, 5), generator=torch.Generator().manual_seed(1))
    from llmcompressorsharp_b200 import embedding

    for t in (torch.float32, torch.bfloat16):
        got = embedding(ids.to(ROOT_DEV), p, scale=0.5, dtype=t)
        assert got.shape == (3, 5, n) and torch.equal(got.cpu(), (w.float() * 0.5).to(t)[ids])


@pytest.mark.gpu
@pytest.mark.parametrize("strategy,group,sym,bits", GRIDS)
@pytest.mark.parametrize("tokens", [1, 8, 9, 16, 17, 129, 257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_products_of_exact_numbers_are_exact(tokens, dtype, strategy, group, sym, bits):
    """Also at the joins of 128 rows and columns, with and without a bias, and for the gradients."""
    from llmcompressorsharp_b200 import int4_linear

    for m, n in ((1, 1), (37, 100), (129, 577), (260, 256)):
        e, w = entry(m, n, strategy, group, sym, bits, seed=tokens + m, pow2=True, device=ROOT_DEV)
        g = torch.Generator().manual_seed(tokens)
        x = torch.randint(-4, 5, (tokens, n), generator=g).double()
        b = torch.randint(-4, 5, (m,), generator=g).double()
        dy = torch.randint(-4, 5, (tokens, m), generator=g).double()
        p = weight(e, n)
        xd, bd = x.to(ROOT_DEV, dtype).requires_grad_(True), b.to(ROOT_DEV, dtype).requires_grad_(True)
        y = int4_linear(xd, p, bd)
        assert torch.equal(y.detach().cpu(), (x @ w.t() + b).float().to(dtype))
        dx, db = torch.autograd.grad(y, [xd, bd], dy.to(ROOT_DEV, dtype))
        assert torch.equal(dx.cpu(), (dy @ w).float().to(dtype))
        assert torch.equal(db.cpu(), dy.sum(0).float().to(dtype))
        assert torch.equal(int4_linear(xd.detach(), p).cpu(), (x @ w.t()).float().to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,m,n", [(1, 300, 2048), (5, 131, 577), (16, 300, 1000), (17, 131, 577), (128, 300, 1000),
                                        (200, 400, 2048), (300, 1531, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("strategy,group,sym", [("group", 128, False), ("group", 100, True), ("channel", 1, False)])
def test_products_and_gradients(tokens, m, n, dtype, strategy, group, sym):
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(m, n, strategy, group, sym, seed=m, device=ROOT_DEV)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, n, generator=g).to(dtype)
    b = torch.randn(m, generator=g).to(dtype)
    dy = torch.randn(tokens, m, generator=g).to(dtype)
    p = weight(e, n)
    xd, bd = x.to(ROOT_DEV).requires_grad_(True), b.to(ROOT_DEV).requires_grad_(True)
    y = int4_linear(xd, p, bd)
    check_product(y.detach(), x.double(), w, b.double(), rounded=tokens > 16)
    dx, db = torch.autograd.grad(y, [xd, bd], dy.to(ROOT_DEV))
    check_product(dx, dy.double(), w.t(), rounded=True)
    check_product(db[None], torch.ones(1, tokens, dtype=torch.float64), dy.double().t())
    again = int4_linear(xd, p, bd)
    assert torch.equal(again, y) and torch.equal(torch.autograd.grad(again, xd, dy.to(ROOT_DEV))[0], dx)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products_of_few_tokens_on_the_tensor_cores(dtype):
    """A weight large enough that 40 tokens leave the few-row kernel, rows and columns off the tiles."""
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(4201, 4103, group=64, pow2=True, device=ROOT_DEV)
    x = torch.randint(-4, 5, (40, 4103), generator=torch.Generator().manual_seed(0)).double()
    b = torch.randint(-4, 5, (4201,), generator=torch.Generator().manual_seed(1)).double()
    y = int4_linear(x.to(ROOT_DEV, dtype), weight(e, 4103), b.to(ROOT_DEV, dtype))
    assert torch.equal(y.cpu(), (x @ w.t() + b).float().to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,tokens", [(19001, 130, 1), (3601, 130, 5), (9601, 130, 7), (9601, 1100, 8), (4801, 1100, 12), (4801, 1100, 32),
                                        (4801, 1100, 48), (601, 1030, 250), (9601, 70, 30)])
@pytest.mark.parametrize("group", [32, 64, 130])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_that_share_x_are_exact(m, n, tokens, dtype, group):
    """Weights of enough rows for each number of record rows to a CTA, the last of them partly past the weight; sums of
    1,100 terms of at most 60 in steps of 2^-6 are exact in fp32."""
    from llmcompressorsharp_b200 import _lib, int4_linear

    code = _lib.dtype_code(dtype)
    e, w = entry(m, n, group=group, pow2=True, seed=m, device=ROOT_DEV)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randint(-4, 5, (tokens, n), generator=g).double()
    b = torch.randint(-4, 5, (m,), generator=g).double()
    p = weight(e, n)
    assert torch.equal(int4_linear(x.to(ROOT_DEV, dtype), p, b.to(ROOT_DEV, dtype)).cpu(), (x @ w.t() + b).float().to(dtype))
    y = torch.full((tokens + 1, m + 3), 7.0, dtype=dtype, device=ROOT_DEV)
    xd = x.to(ROOT_DEV, dtype)
    ws = p._workspace("llmc_int4_linear_workspace", xd.data_ptr(), code, tokens, n)
    _lib.call("llmc_int4_linear", p._ctx, _lib.stream(0), p._ref, xd.data_ptr(), code, tokens, n, None, y.data_ptr(), m + 3,
              ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0)
    assert torch.equal(y[:tokens, :m].cpu(), (x @ w.t()).float().to(dtype))
    assert bool((y[tokens:] == 7).all()) and bool((y[:, m:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,m,n", [(1300, 1801, 260), (1300, 260, 1801), (2100, 1801, 1030)])
@pytest.mark.parametrize("group", [32, 64, 100, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products_of_many_tiles_are_exact(tokens, m, n, dtype, group):
    """More tiles of 128 x 128 than SMs in the product, its gradient or both, the last ones ragged.  Sums of up to 1,801
    terms below 8 in steps of 2^-6 are exact in fp32."""
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(m, n, group=group, pow2=True, seed=m, device=ROOT_DEV)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randint(-4, 5, (tokens, n), generator=g).double()
    b = torch.randint(-4, 5, (m,), generator=g).double()
    dy = torch.randint(-4, 5, (tokens, m), generator=g).double()
    xd = x.to(ROOT_DEV, dtype).requires_grad_(True)
    wd = w.to(ROOT_DEV)
    y = int4_linear(xd, weight(e, n), b.to(ROOT_DEV, dtype))
    assert torch.equal(y, (x.to(ROOT_DEV) @ wd.t() + b.to(ROOT_DEV)).float().to(dtype))
    assert torch.equal(torch.autograd.grad(y, xd, dy.to(ROOT_DEV, dtype))[0], (dy.to(ROOT_DEV) @ wd).float().to(dtype))


@pytest.mark.gpu
def test_gradient_against_differences():
    """The product is linear in x: a step of t along d changes it by t (d W^T), whatever x is."""
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(70, 130, group=64, device=ROOT_DEV)
    p = weight(e, 130)
    g = torch.Generator().manual_seed(3)
    x, d, c = torch.randn(5, 130, generator=g), torch.randn(5, 130, generator=g), torch.randn(5, 70, generator=g)
    xd = x.to(ROOT_DEV).requires_grad_(True)
    (int4_linear(xd, p) * c.to(ROOT_DEV)).sum().backward()
    got = (xd.grad.double().cpu() * d.double()).sum()
    diff = (int4_linear((x + d).to(ROOT_DEV), p).double().cpu() - int4_linear((x - d).to(ROOT_DEV), p).double().cpu()) / 2
    s = ((x.abs() + d.abs()).double() @ w.abs().t() * c.abs().double()).sum()
    assert abs(float((diff * c.double()).sum() - got)) <= 4 * (130 + 70 + 16) * 2.0 ** -23 * float(s)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 40])
def test_strides_alignment_and_surroundings(tokens):
    """Rows of a wider tensor, a base off 16 bytes, a transposed and an expanded x; and rows of y with a pitch,
    whose gaps and following rows keep what they held."""
    from llmcompressorsharp_b200 import _lib, int4_linear

    m, n = 70, 200
    e, w = entry(m, n, group=64, pow2=True, device=ROOT_DEV)
    p = weight(e, n)
    g = torch.Generator().manual_seed(5)
    big = torch.randint(-4, 5, (tokens, n + 24), generator=g).to(ROOT_DEV, torch.bfloat16)
    for x in (big[:, :n], big[:, 8:n + 8], big[:, 3:n + 3], big[:, :n].t().contiguous().t(), big[:1, :n].expand(tokens, n)):
        want = (x.double().cpu() @ w.t()).float().to(torch.bfloat16)
        assert torch.equal(int4_linear(x, p).cpu(), want)
        assert torch.equal(int4_linear(x.reshape(1, tokens, n), p).cpu(), want[None])
    x = big[:, :n].contiguous()
    y = torch.full((tokens + 2, m + 5), 7.0, dtype=torch.bfloat16, device=ROOT_DEV)
    ws = p._workspace("llmc_int4_linear_workspace", x.data_ptr(), _lib.DTYPE_BF16, tokens, n)
    _lib.call("llmc_int4_linear", p._ctx, _lib.stream(0), p._ref, x.data_ptr(), _lib.DTYPE_BF16, tokens, n, None, y.data_ptr(), m + 5,
              ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0)
    assert torch.equal(y[:tokens, :m].cpu(), (x.double().cpu() @ w.t()).float().to(torch.bfloat16))
    assert bool((y[tokens:] == 7).all()) and bool((y[:, m:] == 7).all())
    d = torch.full((tokens + 2, n + 3), 7.0, dtype=torch.bfloat16, device=ROOT_DEV)
    dy = y[:tokens, :m].contiguous()
    ws = p._workspace("llmc_int4_linear_grad_workspace", dy.data_ptr(), _lib.DTYPE_BF16, tokens, m)
    _lib.call("llmc_int4_linear_grad", p._ctx, _lib.stream(0), p._ref, dy.data_ptr(), _lib.DTYPE_BF16, tokens, m, d.data_ptr(), n + 3,
              ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0)
    assert bool((d[tokens:] == 7).all()) and bool((d[:, n:] == 7).all())
    check_product(d[:tokens, :n], dy.double().cpu(), w.t(), rounded=True)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinities_and_nan_stay_in_their_row(tokens, dtype):
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(50, 256, group=64, seed=9, device=ROOT_DEV)
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean = int4_linear(x.to(ROOT_DEV), weight(e, 256)).cpu()
    x[0, 17] = float("inf")
    x[1, 200] = float("nan")
    got = int4_linear(x.to(ROOT_DEV), weight(e, 256)).cpu()
    assert torch.equal(got[2:], clean[2:])
    assert bool(got[1].isnan().all())
    v = w[:, 17]
    assert bool(got[0][v == 0].isnan().all())
    assert bool((got[0][v > 0] == float("inf")).all()) and bool((got[0][v < 0] == -float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("magnitude", [1e-7, 3e4])
def test_fp16_keeps_small_and_large_scales(magnitude):
    """Scales below fp16's normal range (or whose products pass its largest value) lose nothing."""
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(40, 256, group=64, pow2=True, device=ROOT_DEV)
    f = 2.0 ** torch.tensor(magnitude).log2().round().item()
    e = {**e, "scales": e["scales"] * f}
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(-4, 5, (30, 256), generator=g) / 4096.0).half() if magnitude > 1 else torch.randint(-4, 5, (30, 256), generator=g).half() * 4096
    dy = (torch.randint(-4, 5, (30, 40), generator=g) / 4096.0).half() if magnitude > 1 else torch.randint(-4, 5, (30, 40), generator=g).half() * 4096
    xd = x.to(ROOT_DEV).requires_grad_(True)
    y = int4_linear(xd, weight(e, 256))
    assert torch.equal(y.detach().cpu(), (x.double() @ (w * f).t()).to(torch.float16))
    (dx,) = torch.autograd.grad(y, xd, dy.to(ROOT_DEV))
    assert torch.equal(dx.cpu(), (dy.double() @ (w * f)).to(torch.float16))


@pytest.mark.gpu
def test_empty_inputs():
    from llmcompressorsharp_b200 import embedding, int4_linear

    e, _ = entry(20, 64, group=32, device=ROOT_DEV)
    p = weight(e, 64)
    x = torch.zeros(0, 64, device=ROOT_DEV, requires_grad=True)
    b = torch.ones(20, device=ROOT_DEV, requires_grad=True)
    y = int4_linear(x, p, b)
    assert y.shape == (0, 20)
    dx, db = torch.autograd.grad(y, [x, b], torch.zeros(0, 20, device=ROOT_DEV))
    assert dx.shape == (0, 64) and bool((db == 0).all())
    assert int4_linear(torch.zeros(3, 0, 64, device=ROOT_DEV), p).shape == (3, 0, 20)
    ids = torch.zeros(0, dtype=torch.long, device=ROOT_DEV)
    assert embedding(ids, p).shape == (0, 64)
    t = torch.randn(9, 5, device=ROOT_DEV, requires_grad=True)
    (dt,) = torch.autograd.grad(embedding(ids, t), t, torch.zeros(0, 5, device=ROOT_DEV))
    assert dt.shape == (9, 5) and bool((dt == 0).all())


@pytest.mark.gpu
def test_from_float_is_the_quantiser():
    from llmcompressorsharp_b200 import Int4Weight, RtnConfig, rtn_quantize

    w = torch.randn(70, 333, generator=torch.Generator().manual_seed(0)).to(ROOT_DEV)
    for cfg in (RtnConfig(4, False, "group", group_size=100), RtnConfig(3, True, "channel"), RtnConfig(2, False, "tensor")):
        deq = rtn_quantize(w, cfg)[0]
        assert torch.equal(Int4Weight.from_float(w, cfg).dequantize(), deq)


# ------------------------------------------------------------------------------ embedding
def plain_grad(ids, dy, vocab, scale, padding):
    out = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for i, v in enumerate(ids.tolist()):
        if v != padding and 0 <= v < vocab:
            out[v] += dy[i].double() * scale
            size[v] += dy[i].double().abs() * abs(scale)
    return out, size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,vocab,hidden", [(1, 1, 1), (1, 7, 8), (33, 5, 64), (100, 3, 65), (1000, 50, 24), (700, 100000, 16),
                                                 (5000, 600, 40), (9000, 2, 129), (20000, 40, 8)])
@pytest.mark.parametrize("ids64", [True, False])
def test_embedding_and_gradient(tokens, vocab, hidden, dtype, ids64):
    from llmcompressorsharp_b200 import embedding

    g = torch.Generator().manual_seed(tokens + hidden)
    ids = (torch.rand(tokens, generator=g) ** 3 * vocab).long()  # low ids are frequent
    table = torch.randn(vocab, hidden, generator=g).to(dtype)
    dy = torch.randn(tokens, hidden, generator=g).to(dtype)
    idd = ids.to(ROOT_DEV, torch.int64 if ids64 else torch.int32)
    td = table.to(ROOT_DEV).requires_grad_(True)
    for scale, padding in ((1.0, None), (1.5, vocab - 1), (0.5, 0)):
        y = embedding(idd, td, scale, padding_idx=padding)
        assert torch.equal(y.detach().cpu(), (table.float() * scale).to(dtype)[ids])
        (got,) = torch.autograd.grad(y, td, dy.to(ROOT_DEV))
        want, size = plain_grad(ids, dy, vocab, scale, padding)
        # one rounding per addition of a row's run (2^-24 of the absolute sum each), of the scale, and of the result
        count = torch.bincount(ids, minlength=vocab).double()[:, None]
        bound = half_step(dtype) * want.abs() + (count + 1) * 2.0 ** -24 * size * 1.01 + torch.finfo(dtype).tiny
        assert bool(((got.double().cpu() - want).abs() <= bound).all())
        y2 = embedding(idd, td, scale, padding_idx=padding)
        assert torch.equal(torch.autograd.grad(y2, td, dy.to(ROOT_DEV))[0], got)


@pytest.mark.gpu
def test_embedding_gradient_of_integers_is_exact_over_long_runs():
    from llmcompressorsharp_b200 import embedding

    g = torch.Generator().manual_seed(0)
    vocab, hidden, tokens = 300, 72, 70000  # eight CTAs sort, three passes' worth of runs per row
    ids = torch.where(torch.rand(tokens, generator=g) < 0.5, torch.zeros(tokens, dtype=torch.long), torch.randint(0, vocab, (tokens,), generator=g))
    dy = torch.randint(-8, 9, (tokens, hidden), generator=g).float()
    t = torch.zeros(vocab, hidden, device=ROOT_DEV, requires_grad=True)
    (got,) = torch.autograd.grad(embedding(ids.to(ROOT_DEV), t), t, dy.to(ROOT_DEV))
    assert torch.equal(got.cpu(), torch.zeros(vocab, hidden).index_add_(0, ids, dy))


@pytest.mark.gpu
def test_ids_outside_the_table():
    from llmcompressorsharp_b200 import _lib, embedding
    from llmcompressorsharp_b200.errors import ArgumentOutOfRangeError

    e, w = entry(20, 64, group=32, device=ROOT_DEV)
    t = torch.randn(20, 64, device=ROOT_DEV, requires_grad=True)
    ids = torch.tensor([3, -1, 20, 1 << 40, 5], device=ROOT_DEV)
    sync = lambda: _lib.call("llmc_sync", _lib.ctx_for(0))  # noqa: E731
    sync()
    y = embedding(ids, t)
    with pytest.raises(ArgumentOutOfRangeError):
        sync()
    sync()  # reported once
    assert torch.equal(y[[0, 4]], t[[3, 5]]) and bool((y[1:4] == 0).all())
    (dt,) = torch.autograd.grad(y, t, torch.ones_like(y))
    with pytest.raises(ArgumentOutOfRangeError):
        sync()
    assert bool((dt[[3, 5]] == 1).all()) and float(dt.sum()) == 2 * 64
    p = embedding(ids, weight(e, 64), dtype=torch.float32)
    with pytest.raises(ArgumentOutOfRangeError):
        sync()
    assert torch.equal(p[0].cpu(), w[3].float()) and bool((p[1:4] == 0).all())


# ------------------------------------------------------------------------------ refusals on the device
@pytest.mark.gpu
def test_call_refusals():
    from llmcompressorsharp_b200 import _lib, embedding, int4_linear
    from llmcompressorsharp_b200.errors import ArgumentError, LlmcError, NotSupportedError, ShapeError

    e, _ = entry(20, 64, group=32, device=ROOT_DEV)
    p = weight(e, 64)
    x = torch.zeros(3, 64, device=ROOT_DEV)
    ids = torch.zeros(3, dtype=torch.long, device=ROOT_DEV)
    for call, error in ((lambda: int4_linear(x[:, :63], p), ShapeError), (lambda: int4_linear(x.double(), p), ArgumentError),
                        (lambda: int4_linear(x.cpu(), p), ArgumentError), (lambda: int4_linear(x, p, torch.zeros(19, device=ROOT_DEV)), ShapeError),
                        (lambda: int4_linear(x, p, torch.zeros(20, device=ROOT_DEV).half()), ArgumentError),
                        (lambda: int4_linear(torch.zeros((), device=ROOT_DEV), p), ShapeError),
                        (lambda: embedding(ids.cpu(), p), ArgumentError), (lambda: embedding(ids.half(), p), ArgumentError),
                        (lambda: embedding(ids, p, padding_idx=20), ArgumentError), (lambda: embedding(ids, p, dtype=torch.int8), ArgumentError),
                        (lambda: embedding(ids, torch.zeros(0, 4, device=ROOT_DEV)), ShapeError), (lambda: p.dequantize(torch.float64), ArgumentError)):
        with pytest.raises(error):
            call()
    out = torch.zeros(3, 20, device=ROOT_DEV)
    args = (p._ctx, _lib.stream(0), p._ref, x.data_ptr(), _lib.DTYPE_F32, 3, 64, None, out.data_ptr(), 20)
    with pytest.raises(LlmcError, match="workspace"):  # fp32 needs scratch
        _lib.call("llmc_int4_linear", *args, None, 0)
    with pytest.raises(ShapeError):
        _lib.call("llmc_int4_linear", *args[:6], 63, *args[7:], None, 0)
    bad = _lib.Int4WeightC(p.packed.data_ptr(), p.exps.data_ptr(), 20, 64, 8)
    with pytest.raises(NotSupportedError):
        _lib.call("llmc_int4_linear", *args[:2], C.byref(bad), *args[3:], None, 0)
