"""The packed products and the embedding under torch's forward mode, its function transforms and its traces: a derivative
is given or the call is refused, never dropped."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_packed import ROOT_DEV, check_product, entry, weight


def stand_in(monkeypatch, w):
    """An Int4Weight of a dense matrix on the CPU: what is tested is what surrounds the product."""
    from llmcompressorsharp_b200 import Int4Weight

    p = object.__new__(Int4Weight)
    p.shape, p.device = tuple(w.shape), torch.device("cpu")

    def product(self, x, bias, back):  # of values alone, as a kernel's
        x, bias = torch.tensor(x.tolist()), None if bias is None else torch.tensor(bias.tolist())
        return x @ w if back else torch.nn.functional.linear(x, w, bias)

    monkeypatch.setattr(Int4Weight, "_product", product)
    return p


@pytest.fixture
def case(monkeypatch):
    g = torch.Generator().manual_seed(0)
    w = torch.randn(5, 7, generator=g)
    return stand_in(monkeypatch, w), w, torch.randn(3, 7, generator=g), torch.randn(5, generator=g), g


def test_tangents_of_a_product(case):
    """y = x W^T + b is linear: its tangent is dx W^T + db, of either alone too."""
    from llmcompressorsharp_b200 import int4_linear

    p, w, x, b, g = case
    dx, db = torch.randn(3, 7, generator=g), torch.randn(5, generator=g)
    with forward_ad.dual_level():
        for xs, bs, want in ((forward_ad.make_dual(x, dx), forward_ad.make_dual(b, db), dx @ w.t() + db),
                             (forward_ad.make_dual(x, dx), b, dx @ w.t()), (x, forward_ad.make_dual(b, db), db.expand(3, 5)),
                             (forward_ad.make_dual(x, dx), None, dx @ w.t())):
            y, dy = forward_ad.unpack_dual(int4_linear(xs, p, bs))
            assert torch.equal(y, torch.nn.functional.linear(x, w, None if bs is None else b))
            assert torch.allclose(dy, want, rtol=2 ** -20, atol=2 ** -20)
        assert forward_ad.unpack_dual(int4_linear(x, p, b)).tangent is None


def test_a_tangent_keeps_its_gradients(case):
    """Forward over reverse: y and its tangent both take gradients, dx's through W."""
    from llmcompressorsharp_b200 import int4_linear

    p, w, x, _, g = case
    x, dx = x.requires_grad_(True), torch.randn(3, 7, generator=g).requires_grad_(True)
    with forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(int4_linear(forward_ad.make_dual(x, dx), p))
        gx, gd = torch.autograd.grad((y + 2 * dy).sum(), [x, dx])
    assert torch.allclose(gx, w.sum(0).expand(3, 7)) and torch.allclose(gd, 2 * w.sum(0).expand(3, 7))


def test_transforms_and_traces_are_refused(case):
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from llmcompressorsharp_b200 import embedding, int4_linear
    from llmcompressorsharp_b200.errors import NotSupportedError

    p, _, x, b, _ = case
    ids, table = torch.tensor([0, 2]), torch.randn(4, 6)
    mode = FakeTensorMode()
    for f, t in ((lambda t: int4_linear(t, p), x), (lambda t: int4_linear(x, p, t), b), (lambda t: embedding(ids, t), table)):
        for call in (lambda: torch.func.grad(lambda t: f(t).sum())(t), lambda: torch.func.jvp(f, (t,), (t,)),
                     lambda: torch.jit.trace(f, (t,), check_trace=False), lambda: make_fx(f)(t), lambda: f(mode.from_tensor(t))):
            with pytest.raises(NotSupportedError):
                call()
    with pytest.raises(NotSupportedError):
        torch.func.vmap(lambda t: int4_linear(t, p))(torch.stack([x, x]))
    with pytest.raises(NotSupportedError):
        torch.func.vmap(lambda i: embedding(i, table))(torch.stack([ids, ids]))


def test_what_a_transform_does_not_touch_still_runs(case):
    """A product of tensors that are not the transform's own."""
    from llmcompressorsharp_b200 import int4_linear

    p, w, x, b, _ = case
    with torch.no_grad():
        assert torch.func.vmap(lambda t: t + 1, randomness="error")(int4_linear(x, p, b)).shape == (3, 5)
        assert torch.equal(int4_linear(x, p, b), torch.nn.functional.linear(x, w, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [3, 300])
def test_tangents_on_the_device(tokens, dtype):
    from llmcompressorsharp_b200 import embedding, int4_linear

    e, w = entry(70, 130, group=64, device=ROOT_DEV)
    p = weight(e, 130)
    g = torch.Generator().manual_seed(1)
    x, dx = (torch.randn(tokens, 130, generator=g).to(dtype).to(ROOT_DEV) for _ in range(2))
    b, db = (torch.randn(70, generator=g).to(dtype).to(ROOT_DEV) for _ in range(2))
    table, dt = (torch.randn(9, 16, generator=g).to(dtype).to(ROOT_DEV) for _ in range(2))
    ids = torch.randint(0, 9, (tokens,), generator=g).to(ROOT_DEV)
    with forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(int4_linear(forward_ad.make_dual(x, dx), p, forward_ad.make_dual(b, db)))
        h, dh = forward_ad.unpack_dual(embedding(ids, forward_ad.make_dual(table, dt), 2.0))
    assert torch.equal(y, int4_linear(x, p, b))
    check_product(dy, dx.double().cpu(), w, db.double().cpu(), rounded=True)
    assert torch.equal(h, (table * 2)[ids]) and torch.equal(dh, (dt * 2)[ids])


def test_the_calibration_model_asserts_on_ids_outside_its_table():
    """The model's embedding is torch's own, whose check of ids ends a session that calibrates on wrong ones: an
    error on the CPU, an assertion on a device."""
    from llmcompressorsharp_b200 import CompressionSession, CompressionState, RtnConfig, RtnModifier, SessionStatus
    from llmcompressorsharp_b200.calibration import LlamaForCalibration, LlamaShape, drive

    m = LlamaForCalibration(LlamaShape(hidden=32, intermediate=48, heads=2, kv_heads=2, layers=1, vocab=11), dtype=torch.float32)
    assert type(m.model.embed_tokens) is torch.nn.Embedding
    session = CompressionSession([RtnModifier(RtnConfig(4, True, "channel"))])
    state = CompressionState(m.linear_weights())
    assert session.run(state, drive(m, [torch.tensor([[1, 11]])])) == SessionStatus.FAILED and isinstance(session.failure, IndexError)


@pytest.mark.gpu
def test_token_embedding_leaves_to_torch_what_torch_transforms():
    """Values, tangents, gradients and graphs of an embedding that torch transforms or records are torch's."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.func import functional_call, grad, jvp, vmap

    from llmcompressorsharp_b200 import TokenEmbedding

    g = torch.Generator().manual_seed(0)
    ours, theirs = TokenEmbedding(11, 24, device=ROOT_DEV), torch.nn.Embedding(11, 24, device=ROOT_DEV)
    theirs.load_state_dict(ours.state_dict())
    ids, other = (torch.randint(0, 11, (4, 10), generator=g).to(ROOT_DEV) for _ in range(2))
    dw = torch.randn(11, 24, generator=g).to(ROOT_DEV)
    got = []
    for m in (ours, theirs):
        w = m.weight.detach()
        f = lambda w: functional_call(m, {"weight": w}, (ids,))  # noqa: B023, E731
        with forward_ad.dual_level():
            dual = forward_ad.unpack_dual(functional_call(m, {"weight": forward_ad.make_dual(w, dw)}, (ids,))).tangent
        got.append([dual, grad(lambda w: f(w).pow(2).sum())(w), *jvp(f, (w,), (dw,)), vmap(m)(ids),
                    torch.jit.trace(m, (ids,), check_trace=False)(other), make_fx(m)(ids)(other), torch.compile(m, backend="eager")(ids)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_compiled_callers_run_the_kernels():
    """torch.compile breaks its graph at the calls and runs them as they are."""
    from llmcompressorsharp_b200 import embedding, int4_linear

    p = weight(entry(64, 128, group=64, device=ROOT_DEV)[0], 128)
    x, table = torch.randn(4, 128, device=ROOT_DEV), torch.randn(40, 16, device=ROOT_DEV)
    ids = torch.randint(0, 40, (7,), device=ROOT_DEV)
    assert torch.equal(torch.compile(lambda x: int4_linear(x * 2, p) + 1, backend="eager")(x), int4_linear(x * 2, p) + 1)
    assert torch.equal(torch.compile(lambda i: embedding(i, table, 2.0) + 1, backend="eager")(ids), embedding(ids, table, 2.0) + 1)
    xs = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(torch.compile(lambda x: int4_linear(x * 2, p).sum(), backend="eager")(xs), xs)
    assert torch.equal(dx, torch.autograd.grad(int4_linear(xs * 2, p).sum(), xs)[0])


def test_forward_mode_over_a_backward_pass(case, monkeypatch):
    """The product of a second derivative with a vector: of sum (x W^T + b)^2 it is 2 (v W^T) W, and for b 2 sum v W^T."""
    from llmcompressorsharp_b200 import int4_linear, packed

    monkeypatch.setattr(packed, "_col_sum", lambda d: torch.tensor(d.tolist()).sum(0))
    p, w, x, b, g = case
    v = torch.randn(3, 7, generator=g)
    x, b = x.requires_grad_(True), b.requires_grad_(True)
    with forward_ad.dual_level():
        xs = forward_ad.make_dual(x, v)
        dx, db = torch.autograd.grad(int4_linear(xs, p, b).pow(2).sum(), [xs, b])
        dx, hx = forward_ad.unpack_dual(dx)
        db, hb = forward_ad.unpack_dual(db)
    y = x @ w.t() + b
    assert torch.allclose(dx, 2 * y @ w, atol=1e-4) and torch.allclose(db, 2 * y.sum(0), atol=1e-4)
    assert torch.allclose(hx, 2 * (v @ w.t()) @ w, atol=1e-4) and torch.allclose(hb, 2 * (v @ w.t()).sum(0), atol=1e-4)


@pytest.mark.gpu
def test_forward_mode_over_a_backward_pass_on_the_device():
    from llmcompressorsharp_b200 import embedding, int4_linear

    e, w = entry(70, 130, group=64, pow2=True, device=ROOT_DEV)
    p, w = weight(e, 130), w.float().to(ROOT_DEV)
    g = torch.Generator().manual_seed(1)
    x, v = (torch.randint(-3, 4, (9, 130), generator=g).float().to(ROOT_DEV) for _ in range(2))
    table, u = (torch.randint(-3, 4, (11, 16), generator=g).float().to(ROOT_DEV) for _ in range(2))
    b = torch.zeros(70, device=ROOT_DEV, requires_grad=True)
    ids = torch.randint(0, 11, (40,), generator=g).to(ROOT_DEV)
    x.requires_grad_(True), table.requires_grad_(True)
    with forward_ad.dual_level():
        xs, ts = forward_ad.make_dual(x, v), forward_ad.make_dual(table, u)
        got = [forward_ad.unpack_dual(d).tangent for d in torch.autograd.grad((int4_linear(xs, p, b).pow(2)).sum(), [xs, b])]
        got.append(forward_ad.unpack_dual(torch.autograd.grad(embedding(ids, ts, 2.0).pow(2).sum(), ts)[0]).tangent)
    s = (v.double() @ w.double().t())
    want = [2 * s @ w.double(), 2 * s.sum(0), 8 * u.double() * torch.bincount(ids, minlength=11)[:, None]]
    # s is exact (integers times powers of two); a sum of n terms is off by 2^-23 of its absolute terms for each and 8 more
    bounds = [78 * 2.0 ** -23 * (2 * s.abs() @ w.double().abs()), 17 * 2.0 ** -23 * 2 * s.abs().sum(0), torch.zeros(())]
    for a, c, bound in zip(got, want, bounds):
        assert bool(((a.double() - c).abs() <= bound.to(a.device)).all())
