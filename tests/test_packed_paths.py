"""The many-row kernel where the dispatch surely takes it (more than 256 tokens), and each path held to its own contract.

What the roundings allow, relative to a product x W or to S = sum |x| |W|:

- fp32, many rows: x1 w2 + x2 w1 are left out, 2^-23 + 2^-24 with x rounded and W truncated to 8 bits a piece, and less;
  W is rounded to fp32 (2^-24) and so is the result; the tensor cores truncate the addends and the sum of the last two
  pieces' products (2 x 2^-23) and of the smaller ones (2^-7 of that).  Of one product: 2^-22.4 + 2 x 2^-24 + 2.02 x 2^-23
  < 2^-20.8.
- 16-bit, many rows: W is rounded once, half a step, its scale's second part another 2^-11 of that twice.
"""

import pytest
import torch

from test_packed import ROOT_DEV, check_product, entry, weight

pytestmark = pytest.mark.gpu


def few_rows(f32, tokens, rows, cols):
    """The condition under which the codes enter as exact integers."""
    if tokens <= (64 if f32 else 32):
        return True
    if tokens > 256:
        return False
    return f32 and cols >= 1024 or -(-tokens // 16) * rows * cols <= 1 << (27 if f32 else 25)


@pytest.mark.parametrize("tokens,m,n", [(300, 300, 2048), (257, 131, 577), (1100, 900, 130)])
@pytest.mark.parametrize("strategy,group,sym", [("group", 128, False), ("group", 100, True), ("group", 32, False), ("channel", 1, False)])
def test_every_piece_of_a_product_counts(tokens, m, n, strategy, group, sym):
    """fp32: one full-mantissa x (or dy) to a row, scales of full mantissas, so that each result is one product; in the
    first, last and padded tiles and at random between."""
    e, w = entry(m, n, strategy, group, sym, seed=n, device=ROOT_DEV)
    p = weight(e, n)
    g = torch.Generator().manual_seed(tokens)
    for back, width in ((False, n), (True, m)):
        at = torch.randint(0, width, (tokens,), generator=g)
        at[:4] = torch.tensor([0, width - 1, width // 2, width - 1])
        x = torch.zeros(tokens, width)
        x[torch.arange(tokens), at] = (torch.rand(tokens, generator=g) + 1) * torch.exp2(torch.randint(-20, 20, (tokens,), generator=g).float())
        x *= torch.where(torch.rand(tokens, generator=g) < 0.5, -1, 1)[:, None]
        got = p._product(x.to(ROOT_DEV), None, back).double().cpu()
        want = x.double() @ (w if back else w.t())
        assert bool(((got - want).abs() <= 2.0 ** -20.8 * want.abs()).all())
        assert bool((got[want == 0] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strides_alignment_and_surroundings_of_many_rows(dtype):
    """x read in place by its pitch, from a base off 16 bytes, transposed and expanded; rows of y and dx with a pitch,
    whose gaps and following rows keep what they held."""
    from llmcompressorsharp_b200 import _lib, int4_linear

    m, n, tokens = 70, 200, 300
    code = _lib.dtype_code(dtype)
    e, w = entry(m, n, group=64, pow2=True, device=ROOT_DEV)
    p = weight(e, n)
    g = torch.Generator().manual_seed(5)
    big = torch.randint(-4, 5, (tokens, n + 24), generator=g).to(ROOT_DEV, dtype)
    for x in (big[:, :n], big[:, 8:n + 8], big[:, 3:n + 3], big[:, :n].t().contiguous().t(), big[:1, :n].expand(tokens, n)):
        want = (x.double().cpu() @ w.t()).float().to(dtype)
        assert torch.equal(int4_linear(x, p).cpu(), want)
        assert torch.equal(int4_linear(x.reshape(1, tokens, n), p).cpu(), want[None])
    for pitch in (n + 24, n + 7):  # rows that TMA reads in place, and that it cannot
        x = torch.randint(-4, 5, (tokens, pitch), generator=g).to(ROOT_DEV, dtype)
        dy = torch.randint(-4, 5, (tokens, m + pitch - n), generator=g).to(ROOT_DEV, dtype)
        for fn, a, width, out, want in (("llmc_int4_linear", x, n, m, x[:, :n].double().cpu() @ w.t()),
                                        ("llmc_int4_linear_grad", dy, m, n, dy[:, :m].double().cpu() @ w)):
            y = torch.full((tokens + 2, out + 8), 7.0, dtype=dtype, device=ROOT_DEV)
            for ldy in (out + 8, out + 5):
                ys = torch.as_strided(y, (tokens + 1, ldy), (ldy, 1)).fill_(7)
                ws = p._workspace(fn + "_workspace", a.data_ptr(), code, tokens, a.shape[1])
                bias = [None] if fn == "llmc_int4_linear" else []
                _lib.call(fn, p._ctx, _lib.stream(0), p._ref, a.data_ptr(), code, tokens, a.shape[1], *bias, y.data_ptr(), ldy,
                          ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0)
                assert torch.equal(ys[:tokens, :out].cpu(), want.float().to(dtype))
                assert bool((ys[tokens:] == 7).all()) and bool((ys[:, out:] == 7).all())


@pytest.mark.parametrize("tokens", [300, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinities_and_nan_stay_in_their_row_of_many(tokens, dtype):
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(150, 256, group=64, seed=9, device=ROOT_DEV)
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean = int4_linear(x.to(ROOT_DEV), weight(e, 256)).cpu()
    x[0, 17], x[1, 200], x[129, 3] = float("inf"), float("nan"), -float("inf")
    got = int4_linear(x.to(ROOT_DEV), weight(e, 256)).cpu()
    rest = [i for i in range(tokens) if i not in (0, 1, 129)]
    assert torch.equal(got[rest], clean[rest])
    assert bool(got[1].isnan().all())
    for row, col, sign in ((0, 17, 1), (129, 3, -1)):
        v = w[:, col] * sign
        assert bool(got[row][v == 0].isnan().all())
        assert bool((got[row][v > 0] == float("inf")).all()) and bool((got[row][v < 0] == -float("inf")).all())


@pytest.mark.parametrize("f", [2.0 ** -23, 2.0 ** 15])
def test_fp16_keeps_small_and_large_scales_over_many_rows(f):
    """Scales below fp16's normal range, or whose products pass its largest value, lose nothing."""
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(40, 256, group=64, pow2=True, device=ROOT_DEV)
    e = {**e, "scales": e["scales"] * f}
    g = torch.Generator().manual_seed(2)
    size = 1 / 4096.0 if f > 1 else 4096.0
    x = (torch.randint(-4, 5, (300, 256), generator=g) * size).half()
    dy = (torch.randint(-4, 5, (300, 40), generator=g) * size).half()
    xd = x.to(ROOT_DEV).requires_grad_(True)
    y = int4_linear(xd, weight(e, 256))
    assert torch.equal(y.detach().cpu(), (x.double() @ (w * f).t()).to(torch.float16))
    assert torch.equal(torch.autograd.grad(y, xd, dy.to(ROOT_DEV))[0].cpu(), (dy.double() @ (w * f)).to(torch.float16))


@pytest.mark.parametrize("ratio", [6, 12, 16, 20])
def test_fp16_scales_beside_far_larger_ones(ratio):
    """A group (forward) or a row (gradient) whose scales are 2^-ratio of the largest, alone in meeting x or dy.  The two
    halves of a scale near one and their products count to 2^-25 each (half of fp16's least step), so a weight of the
    small ones is off by 2^-11 of itself, with the second half's 2^-22, and by (15 + 1 + 1) x 2^-25 of the largest scale's
    power of two at most."""
    m, n, tokens = 64, 256, 300
    g = torch.Generator().manual_seed(ratio)
    e, w = entry(m, n, group=64, seed=ratio, device=ROOT_DEV)
    e["scales"], w = e["scales"] * 1024, w * 1024  # results in fp16's normal range
    small = 2.0 ** -ratio
    x, dy = torch.zeros(tokens, n), torch.zeros(tokens, m)
    x[:, 64:128] = torch.randn(tokens, 64, generator=g)  # only the second group of columns
    dy[:, 5] = torch.randn(tokens, generator=g)          # only the sixth row
    x, dy = x.half(), dy.half()
    fwd, back = e["scales"].clone(), e["scales"].clone()
    fwd[:, 1] *= small
    back[5] *= small
    column = torch.arange(n) // 64
    q = w / e["scales"].cpu().double()[:, column]
    for scales, a, grad in ((fwd, x, False), (back, dy, True)):
        ws = q * scales.cpu().double()[:, column]
        p = weight({**e, "scales": scales}, n)
        got = p._product(a.to(ROOT_DEV), None, grad).double().cpu()
        ad = a.double()
        mat = ws if grad else ws.t()
        want, size = ad @ mat, ad.abs() @ mat.abs()
        # the largest scale of the weight's row (forward) or of its group over all rows (gradient), as a power of two
        s = scales.cpu().double()
        top = torch.exp2(torch.floor(torch.log2(s.max(0).values[column] if grad else s.max(1).values)) + 1)
        bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -21 + (ad.shape[1] + 8) * 2.0 ** -23) * size
        bound += 17 * 2.0 ** -25 * ad.abs().sum(1, keepdim=True) * top[None] + 2.0 ** -25
        assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens,m,n", [(17, 131, 577), (128, 300, 1000), (128, 2000, 2048), (200, 400, 2048), (256, 131, 577), (300, 1531, 1000),
                                        (700, 257, 390)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_weight_is_rounded_only_where_the_dispatch_says(tokens, m, n, dtype):
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(m, n, "group", 64, False, seed=m, device=ROOT_DEV)
    g = torch.Generator().manual_seed(tokens)
    x, b = torch.randn(tokens, n, generator=g).to(dtype), torch.randn(m, generator=g).to(dtype)
    y = int4_linear(x.to(ROOT_DEV), weight(e, n), b.to(ROOT_DEV))
    check_product(y, x.double(), w, b.double(), rounded=not few_rows(dtype == torch.float32, tokens, m, n))


@pytest.mark.parametrize("limit", [1, 7])
def test_an_sm_limit_changes_no_result_of_many_rows(limit):
    from llmcompressorsharp_b200 import _lib

    p = weight(entry(400, 640, "group", 128, True)[0], 640)
    x = torch.randn(300, 640, generator=torch.Generator().manual_seed(2)).to(ROOT_DEV, torch.float16)
    want = p._product(x, None, False)
    ctx = _lib.ctx_handle(p.device.index)
    try:
        _lib.call("llmc_set_sm_limit", ctx, limit)
        assert torch.equal(p._product(x, None, False), want)
    finally:
        _lib.call("llmc_set_sm_limit", ctx, 0)


@pytest.mark.parametrize("value", [3.4028234e38, 3.3961775e38, 3.39e38])
def test_the_largest_fp32_values_stay_finite(value):
    """Values that bf16 would round to an infinity: their first piece is truncated."""
    e, w = entry(40, 64, group=64, pow2=True, device=ROOT_DEV)
    w = w * 2.0 ** -20
    p = weight({**e, "scales": e["scales"] * 2.0 ** -20}, 64)
    x = torch.zeros(300, 64)
    x[torch.arange(300), torch.arange(300) % 64] = value
    got, want = p._product(x.to(ROOT_DEV), None, False).double().cpu(), x.double() @ w.t()
    assert bool(((got - want).abs() <= 2.0 ** -20.8 * want.abs()).all())
