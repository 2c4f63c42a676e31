"""The packed operators as they are used: a compressed model run from its codes, quantisation-aware training of
an embedding, graphs, streams, threads, a wait that gives up, and offsets past 32 bits."""

import ctypes as C
import threading

import pytest
import torch

from test_packed import ROOT_DEV, check_product, entry, half_step, weight

pytestmark = pytest.mark.gpu


def tiny(dtype, device=ROOT_DEV, seed=3):
    from llmcompressorsharp_b200.calibration import LlamaForCalibration, LlamaShape

    return LlamaForCalibration(LlamaShape(hidden=96, intermediate=160, heads=4, kv_heads=2, layers=2, vocab=131), dtype=dtype,
                               device=device, seed=seed)


def plain_weight(e, n):
    """W in 64 bits of a compressed entry, from its definition."""
    codes = e["codes"].cpu().long()
    stored = torch.stack([codes >> 4, codes & 15], 2).reshape(codes.shape[0], -1)[:, :n]
    scale, zero = e["scales"].cpu().double(), e["zero_points"].cpu().long()
    if e["strategy"] == "group":
        col = torch.arange(n) // e["group_size"]
        scale, zero = scale[:, col], zero[:, col]
    else:
        scale, zero = scale.reshape(-1, 1), zero.reshape(-1, 1)
    if e["symmetric"]:
        return torch.where(stored >= 8, stored - 16, stored).double() * scale
    return (((stored + zero) & 15) - zero).double() * scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("config", [dict(num_bits=4, symmetric=False, strategy="group", group_size=32),
                                    dict(num_bits=4, symmetric=True, strategy="channel")])
def test_a_compressed_model_runs_from_its_codes(dtype, config):
    """RTN session -> state.compressed -> packed modules -> prompt and single-token forward.  Each packed
    module's output is checked against its own input; the embedding's against its table."""
    from llmcompressorsharp_b200 import CompressionSession, CompressionState, Int4Embedding, Int4Linear, RtnConfig, RtnModifier

    m = tiny(dtype)
    weights = m.linear_weights()
    weights["model.embed_tokens.weight"] = m.model.embed_tokens.weight
    state = CompressionState(weights)
    session = CompressionSession([RtnModifier(RtnConfig(**config))])
    session.run(state, [])
    assert session.failure is None
    done = m.load_compressed(state.compressed)
    assert sorted(done) == sorted(n[: -len(".weight")] for n in weights)
    assert isinstance(m.model.embed_tokens, Int4Embedding) and isinstance(m.model.layers[1].mlp.down_proj, Int4Linear)
    assert not m.linear_modules()
    seen = []
    for name, mod in m.named_modules():
        if isinstance(mod, (Int4Linear, Int4Embedding)):
            mod.register_forward_hook(lambda mod, args, out, name=name: seen.append((name, args[0].clone(), out.clone())))
    for shape in ((2, 37), (3, 1)):
        ids = torch.randint(0, 131, shape, generator=torch.Generator().manual_seed(1)).to(ROOT_DEV)
        out = m(ids)
        assert out.shape == (*shape, 96) and out.dtype == dtype and bool(out.isfinite().all())
    assert len(seen) == 2 * len(done)
    for name, x, y in seen:
        e = state.compressed[name + ".weight"]
        if name.endswith("embed_tokens"):
            assert torch.equal(y.cpu(), plain_weight(e, 96).float().to(dtype)[x.cpu()])
        else:
            w = plain_weight(e, x.shape[-1])
            check_product(y.reshape(-1, y.shape[-1]), x.reshape(-1, x.shape[-1]).double().cpu(), w, rounded=x.numel() // x.shape[-1] > 16)


def test_codes_of_gptq_and_of_a_tied_table():
    """GPTQ's codes multiply as its wq does; one packed weight serves the lookup and the output projection."""
    from llmcompressorsharp_b200 import GPTQConfig, Int4Weight, embedding, gptq_quantize_u, int4_linear

    cfg = GPTQConfig(num_bits=4, symmetric=False, strategy="group", group_size=64, block_size=128)
    w = (torch.randn(150, 256, generator=torch.Generator().manual_seed(0)) * 0.02).to(ROOT_DEV)
    res = gptq_quantize_u(w, torch.eye(256, device=ROOT_DEV), cfg)
    p = Int4Weight(res.codes, res.scales, res.zero_points, 256, "group", 64, False)
    assert torch.equal(p.dequantize(), res.wq)
    ids = torch.tensor([[0, 149, 7]], device=ROOT_DEV)
    h = embedding(ids, p, scale=2.0, dtype=torch.float32)
    assert torch.equal(h, (res.wq * 2)[ids])
    check_product(int4_linear(h, p).reshape(3, 150), h.reshape(3, 256).double().cpu(), res.wq.double().cpu())


def test_load_compressed_leaves_the_rest():
    from llmcompressorsharp_b200 import RtnConfig, load_compressed, rtn_quantize
    from llmcompressorsharp_b200.errors import ShapeError

    m = torch.nn.Sequential(torch.nn.Linear(32, 16), torch.nn.LayerNorm(16), torch.nn.Linear(16, 8)).to(ROOT_DEV)

    def made(w, bits):
        _, c, s, z = rtn_quantize(w, RtnConfig(bits, True, "channel"))
        return {"codes": c, "scales": s, "zero_points": z, "num_bits": bits, "symmetric": True, "strategy": "channel", "group_size": 128}

    state = {"0.weight": made(m[0].weight, 4), "2.weight": made(m[2].weight, 8), "1.weight": {"mask": None}, "9.weight": made(m[0].weight, 4)}
    bias = m[0].bias
    assert load_compressed(m, state) == ["0"]
    assert m[0].bias is bias and isinstance(m[2], torch.nn.Linear)
    x = torch.randn(4, 32, device=ROOT_DEV)
    m(x).sum().backward()
    assert bias.grad is not None and m[2].weight.grad is not None
    with pytest.raises(ShapeError):
        load_compressed(torch.nn.Sequential(torch.nn.Linear(32, 17)).to(ROOT_DEV), {"0.weight": state["0.weight"]})


def test_load_compressed_replaces_what_computes_the_same():
    """Subclasses, an Embedding with max_norm and a module elsewhere stay; a module held twice goes in both places."""
    from llmcompressorsharp_b200 import Int4Embedding, Int4Linear, RtnConfig, load_compressed, rtn_quantize

    class Doubled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def made(w):
        _, c, s, z = rtn_quantize(w, RtnConfig(4, True, "channel"))
        return {"codes": c, "scales": s, "zero_points": z, "num_bits": 4, "symmetric": True, "strategy": "channel", "group_size": 128}

    m = torch.nn.ModuleDict({"a": torch.nn.Linear(32, 32), "d": Doubled(32, 32), "n": torch.nn.Embedding(9, 32, max_norm=1.0),
                             "e": torch.nn.Embedding(9, 32)}).to(ROOT_DEV)
    m["b"] = torch.nn.Sequential(m["a"])
    state = {n + ".weight": made(m[n].weight) for n in ("a", "d", "n", "e")}
    assert sorted(load_compressed(m, state)) == ["a", "e"]
    assert type(m["d"]) is Doubled and type(m["n"]) is torch.nn.Embedding and type(m["e"]) is Int4Embedding
    assert type(m["a"]) is Int4Linear and m["b"][0] is m["a"]


@pytest.mark.parametrize("options", [{}, {"padding_idx": 3}, {"max_norm": 0.5}, {"scale_grad_by_freq": True}, {"dtype": torch.float64}])
def test_token_embedding_is_torchs(options):
    """The model's embedding keeps torch's values and gradients under each of torch's options.  Gradients are sums of
    up to 40 terms 2^-3 k of fp32 or wider, exact in any order; a division by a count is one rounding.  With max_norm
    both sides are torch's, which adds a row's 24 squares in no fixed order: a relative 23 x 2^-24 at most, half of it
    in the root, and with the root's, the quotient's and the product's roundings less than 2^-20 on each side."""
    from llmcompressorsharp_b200.calibration import TokenEmbedding

    gen = torch.Generator().manual_seed(0)
    ours, theirs = TokenEmbedding(11, 24, device=ROOT_DEV, **options), torch.nn.Embedding(11, 24, device=ROOT_DEV, **options)
    theirs.load_state_dict(ours.state_dict())
    ids = torch.randint(0, 11, (4, 10), generator=gen).to(ROOT_DEV)
    dy = (torch.randint(-8, 9, (4, 10, 24), generator=gen) * 0.125).to(ROOT_DEV, ours.weight.dtype)
    y, z = ours(ids), theirs(ids)
    if options.get("max_norm"):
        assert torch.allclose(y, z, rtol=2 ** -19, atol=0)
    else:
        assert torch.equal(y, z)
    y.backward(dy)
    z.backward(dy)
    if options.get("scale_grad_by_freq"):
        assert torch.allclose(ours.weight.grad, theirs.weight.grad, rtol=2 ** -20, atol=2 ** -20)
    else:
        assert torch.equal(ours.weight.grad, theirs.weight.grad)


@pytest.mark.parametrize("tokens,dtype", [(1, torch.bfloat16), (100, torch.float16), (300, torch.bfloat16), (300, torch.float32)])
def test_an_sm_limit_changes_no_result(tokens, dtype):
    """A context's limit of SMs leaves the size of a workspace asked for before it, and every bit, as they were."""
    from llmcompressorsharp_b200 import _lib, int4_linear

    p = weight(entry(400, 640, "group", 128, True)[0], 640)
    x = torch.randn(tokens, 640, generator=torch.Generator().manual_seed(2)).to(ROOT_DEV, dtype).requires_grad_(True)

    def both():
        y = int4_linear(x, p)
        return y.detach(), torch.autograd.grad(y, [x], torch.ones_like(y))[0]

    want = both()
    ctx = _lib.ctx_handle(p.device.index)
    try:
        for limit in (1, 7):
            _lib.call("llmc_set_sm_limit", ctx, limit)
            for got, w in zip(both(), want):
                assert torch.equal(got, w)
    finally:
        _lib.call("llmc_set_sm_limit", ctx, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantisation_aware_embedding_under_a_frozen_packed_layer(dtype):
    """Table -> FakeQuantize (straight through) -> embedding -> packed layer; every gradient against its formula."""
    from llmcompressorsharp_b200 import FakeQuantize, embedding, int4_linear

    e, w = entry(40, 64, group=32, device=ROOT_DEV)
    p = weight(e, 64)
    g = torch.Generator().manual_seed(0)
    table = (torch.randn(50, 64, generator=g) * 0.5).to(dtype).to(ROOT_DEV).requires_grad_(True)
    bias = torch.randn(40, generator=g).to(dtype).to(ROOT_DEV).requires_grad_(True)
    ids = torch.randint(0, 50, (6, 9), generator=g).to(ROOT_DEV)
    fq = FakeQuantize.apply(table, 0.1, 0, 4, True)
    h = embedding(ids, fq, scale=8.0, padding_idx=4)
    h.retain_grad()
    y = int4_linear(h, p, bias)
    dy = torch.randn(y.shape, generator=g).to(dtype)
    y.backward(dy.to(ROOT_DEV))
    assert torch.equal(h.detach().cpu(), (fq.detach().float() * 8).to(dtype)[ids].cpu())
    d2 = dy.reshape(-1, 40).double()
    check_product(y.detach().reshape(-1, 40), h.detach().reshape(-1, 64).double().cpu(), w, bias.detach().double().cpu(), rounded=True)
    check_product(h.grad.reshape(-1, 64), d2, w.t(), rounded=True)
    check_product(bias.grad[None], torch.ones(1, 54, dtype=torch.float64), d2.t())
    dh, flat = h.grad.reshape(-1, 64).double().cpu(), ids.flatten().cpu()
    want = torch.zeros(50, 64, dtype=torch.float64).index_add_(0, flat, dh * 8)
    size = torch.zeros(50, 64, dtype=torch.float64).index_add_(0, flat, dh.abs() * 8)
    want[4], size[4] = 0, 0
    bound = half_step(dtype) * want.abs() + 60 * 2.0 ** -24 * size + torch.finfo(dtype).tiny
    assert bool(((table.grad.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens", [1, 5, 16, 40, 200, 300, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_graphs_of_one_weight(tokens, dtype):
    """Two graphs of the same weight at once, replayed with new inputs on two streams: forward, and forward with backward."""
    from llmcompressorsharp_b200 import embedding, int4_linear

    e, _ = entry(300, 1000, group=128, device=ROOT_DEV)
    p = weight(e, 1000)
    g = torch.Generator().manual_seed(tokens)
    xs = [torch.randn(tokens, 1000, generator=g).to(ROOT_DEV, dtype).requires_grad_(True) for _ in range(2)]
    table = torch.randn(500, 1000, generator=g).to(ROOT_DEV, dtype).requires_grad_(True)
    ids = [torch.randint(0, 500, (tokens,), generator=g).to(ROOT_DEV) for _ in range(2)]
    dy = torch.randn(tokens, 300, generator=g).to(ROOT_DEV, dtype)

    def step(i):
        y = int4_linear(xs[i], p)
        (dx,) = torch.autograd.grad(y, xs[i], dy)
        h = embedding(ids[i], table, 2.0)
        (dt,) = torch.autograd.grad(h, table, dx)
        return y.detach(), dx, h.detach(), dt

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        with torch.no_grad():
            for i in range(2):
                xs[i].copy_(torch.randn(tokens, 1000, generator=g))
                ids[i].copy_(torch.randint(0, 500, (tokens,), generator=g))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], step(i)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [400, 20000])
def test_products_on_two_streams_at_once(tokens, dtype):
    """Two streams of products share the SMs and give, tile by tile, the bits that each gives alone."""
    p = weight(entry(300, 1000, group=128, device=ROOT_DEV)[0], 1000)
    g = torch.Generator().manual_seed(tokens)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for back, n in ((True, 300), (False, 1000)):
        src = [torch.randn(tokens, n, generator=g).to(ROOT_DEV, dtype) for _ in range(2)]
        want = [p._product(a, None, back) for a in src]
        torch.cuda.synchronize()
        for _ in range(12):
            got = []
            for i in (0, 1, 0, 1):
                with torch.cuda.stream(streams[i]):
                    got.append((i, p._product(src[i], None, back)))
            torch.cuda.synchronize()
            assert all(torch.equal(y, want[i]) for i, y in got)


def test_first_calls_inside_a_capture():
    """A process whose first call of the library is captured: the context, the attributes and the grids are set up then."""
    import subprocess
    import sys

    code = """
import torch
from llmcompressorsharp_b200 import embedding
t = torch.randn(40, 16, device="cuda", requires_grad=True)
ids = torch.randint(0, 40, (90,), device="cuda")
dy = torch.randn(90, 16, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = embedding(ids, t, 2.0)
    (dt,) = torch.autograd.grad(y, t, dy)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, t[ids] * 2)
want = torch.zeros(40, 16, dtype=torch.float64).index_add_(0, ids.cpu(), dy.double().cpu() * 2)
assert float((dt.double().cpu() - want).abs().max()) < 1e-4
print("captured")
"""
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_threads_on_streams_of_their_own():
    from llmcompressorsharp_b200 import embedding, int4_linear

    e, _ = entry(130, 256, group=64, device=ROOT_DEV)
    p = weight(e, 256)
    g = torch.Generator().manual_seed(0)
    table = torch.randn(300, 256, generator=g).to(ROOT_DEV)
    jobs = [(torch.randn(t, 256, generator=g).to(ROOT_DEV), torch.randint(0, 300, (t,), generator=g).to(ROOT_DEV)) for t in (1, 9, 40, 200)]
    want = [(int4_linear(x, p), embedding(i, table, 2.0)) for x, i in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        x, i = jobs[k]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                got = (int4_linear(x, p), embedding(i, table, 2.0))
                s.synchronize()
                if not (torch.equal(got[0], want[k][0]) and torch.equal(got[1], want[k][1])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_inputs_of_another_stream_are_waited_for_by_the_callers_event():
    """The call runs on the caller's current stream, whichever stream made the tensors."""
    from llmcompressorsharp_b200 import int4_linear

    e, _ = entry(64, 128, group=64, device=ROOT_DEV)
    p = weight(e, 128)
    s = torch.cuda.Stream()
    x = torch.zeros(4, 128, device=ROOT_DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            x.add_(torch.ones(4, 128, device=ROOT_DEV))
        y = int4_linear(x, p)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, int4_linear(torch.full((4, 128), 20.0, device=ROOT_DEV), p))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_non_finite_gradients_stay_in_their_row(dtype):
    from llmcompressorsharp_b200 import int4_linear

    e, w = entry(200, 96, group=32, seed=4, device=ROOT_DEV)
    p = weight(e, 96)
    x = torch.zeros(150, 96, device=ROOT_DEV, dtype=dtype, requires_grad=True)
    dy = torch.randn(150, 200, generator=torch.Generator().manual_seed(0)).to(dtype)
    clean = torch.autograd.grad(int4_linear(x, p), x, dy.to(ROOT_DEV))[0].cpu()
    dy[3, 7], dy[140, 199] = float("inf"), float("nan")
    got = torch.autograd.grad(int4_linear(x, p), x, dy.to(ROOT_DEV))[0].cpu()
    rest = [i for i in range(150) if i not in (3, 140)]
    assert torch.equal(got[rest], clean[rest]) and bool(got[140].isnan().all())
    v = w[7]
    assert bool(got[3][v == 0].isnan().all()) and bool((got[3][v > 0] == float("inf")).all()) and bool((got[3][v < 0] == -float("inf")).all())


@pytest.mark.parametrize("tokens,m,k,dtype", [(300, 300, 256, torch.bfloat16), (300, 300, 256, torch.float16), (300, 300, 256, torch.float32),
                                              (1300, 1801, 1792, torch.bfloat16), (1300, 1801, 1792, torch.float16)])
def test_a_wait_that_gives_up_is_reported_and_passes(tokens, m, k, dtype):
    """The limit of 0 makes the tensor-core kernel give up at its first wait, before it has issued a copy."""
    from llmcompressorsharp_b200 import _lib

    lib = _lib.load()
    ctx = C.c_void_p()
    assert lib.llmc_init(0, C.byref(ctx)) == 0
    try:
        e, _ = entry(m, k, group=64, device=ROOT_DEV)
        p = weight(e, k)
        x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(0)).to(ROOT_DEV, dtype)
        dy = torch.randn(tokens, m, generator=torch.Generator().manual_seed(1)).to(ROOT_DEV, dtype)
        torch.cuda.synchronize()
        for back in (False, True):
            a, n = (dy, k) if back else (x, m)
            want = p._product(a, None, back)
            out = torch.empty(tokens, n, dtype=dtype, device=ROOT_DEV)
            need = C.c_int64()
            fn = "llmc_int4_linear_grad" if back else "llmc_int4_linear"
            assert getattr(lib, fn + "_workspace")(ctx, p._ref, a.data_ptr(), _lib.dtype_code(dtype), tokens, a.shape[1], C.byref(need)) == 0
            ws = torch.empty(max(1, need.value), dtype=torch.uint8, device=ROOT_DEV)
            bias = [] if back else [None]

            def run():
                assert getattr(lib, fn)(ctx, C.c_void_p(1), p._ref, a.data_ptr(), _lib.dtype_code(dtype), tokens, a.shape[1], *bias,
                                        out.data_ptr(), n, ws.data_ptr(), ws.numel()) == 0
                torch.cuda.synchronize()

            assert lib.llmc_set_wait_limit(ctx, 0) == 0
            run()
            assert lib.llmc_sync(ctx) == 7 and lib.llmc_sync(ctx) == 0
            assert lib.llmc_set_wait_limit(ctx, -1) == 0
            run()
            assert lib.llmc_sync(ctx) == 0 and torch.equal(out, want)
    finally:
        lib.llmc_destroy(ctx)


def test_offsets_past_32_bits():
    """A packed weight of more than 2^31 bytes, a dense table of more than 2^31 elements and a product of more than
    2^31: rows at their far ends."""
    from llmcompressorsharp_b200 import Int4Weight, embedding, int4_linear

    m, n = 1 << 20, 4480
    codes = torch.randint(0, 256, (m, n // 2), dtype=torch.uint8, device=ROOT_DEV)
    p = Int4Weight(codes, torch.full((m,), 0.125, device=ROOT_DEV), None, n, "channel", symmetric=True)
    assert p.packed.numel() > 1 << 31
    tail = codes[-3:].cpu().long()
    stored = torch.stack([tail >> 4, tail & 15], 2).reshape(3, n)
    want = torch.where(stored >= 8, stored - 16, stored).double() * 0.125
    ids = torch.tensor([m - 3, m - 2, m - 1], device=ROOT_DEV)
    assert torch.equal(embedding(ids, p, dtype=torch.float32).cpu(), want.float())
    x = torch.randint(-2, 3, (20, n), generator=torch.Generator().manual_seed(0)).to(ROOT_DEV, torch.bfloat16)
    for t in (3, 20):
        assert torch.equal(int4_linear(x[:t], p)[:, -3:].cpu(), (x[:t].double().cpu() @ want.t()).float().bfloat16())
    del codes, p
    torch.cuda.empty_cache()
    rows = 600_000
    table = torch.empty(rows, 4096, dtype=torch.bfloat16, device=ROOT_DEV)
    table[-2:] = torch.randn(2, 4096, device=ROOT_DEV).bfloat16()
    table.requires_grad_(True)
    ids = torch.tensor([rows - 1, rows - 2, rows - 1], device=ROOT_DEV)
    y = embedding(ids, table)
    assert torch.equal(y, table[ids])
    dy = torch.randint(-4, 5, (3, 4096), generator=torch.Generator().manual_seed(1)).to(ROOT_DEV, torch.bfloat16)
    (dt,) = torch.autograd.grad(y, table, dy)
    assert torch.equal(dt[-1], dy[0] + dy[2]) and torch.equal(dt[-2], dy[1]) and not bool(dt[:-2].any())
    del table, y, dt
    torch.cuda.empty_cache()
    e, w = entry(31000, 128, "channel", pow2=True, device=ROOT_DEV)
    p = weight(e, 128)
    x = torch.randint(-4, 5, (70000, 128), generator=torch.Generator().manual_seed(2)).to(ROOT_DEV, torch.bfloat16)
    y = int4_linear(x, p)
    assert y.numel() > 1 << 31
    for rows in (slice(0, 2), slice(69990, 70000)):
        assert torch.equal(y[rows].cpu(), (x[rows].double().cpu() @ w.t()).float().bfloat16())


def test_copies_and_second_derivatives():
    import copy
    import pickle

    from llmcompressorsharp_b200 import Int4Linear, int4_linear

    e, w = entry(40, 64, group=32, device=ROOT_DEV)
    m = Int4Linear(weight(e, 64))
    x = torch.randn(3, 64, device=ROOT_DEV, requires_grad=True)
    y = m(x)
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert other.packed_weight.packed.data_ptr() != m.packed_weight.packed.data_ptr()
        m2 = other(x)
        assert torch.equal(m2, y)
    (dx,) = torch.autograd.grad(int4_linear(x, m.packed_weight).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
