"""Int4Linear, Int4Embedding and load_compressed: what the modules they replace did around their product goes on."""

import pytest
import torch

from test_packed import ROOT_DEV, check_product, entry, weight


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_casts_what_torch_casts(dtype):
    """Under autocast x and the bias are of its type, as torch.nn.Linear's, and their gradients of their own."""
    from llmcompressorsharp_b200 import Int4Linear, int4_linear

    e, w = entry(40, 64, group=32, device=ROOT_DEV)
    g = torch.Generator().manual_seed(0)
    m = Int4Linear(weight(e, 64), torch.nn.Parameter(torch.randn(40, generator=g).to(ROOT_DEV)))
    plain = torch.nn.Linear(64, 40, device=ROOT_DEV)
    x = torch.randn(50, 64, generator=g).to(ROOT_DEV)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        xs = x.to(t).requires_grad_(True)
        with torch.autocast("cuda", dtype):
            y = m(xs)
            assert y.dtype == plain(xs).dtype == dtype
        assert torch.equal(y, int4_linear(xs.to(dtype), m.packed_weight, m.bias.to(dtype)))
        dx, db = torch.autograd.grad(y, [xs, m.bias], torch.ones_like(y))
        assert dx.dtype == t and db.dtype == torch.float32
        check_product(y.detach(), xs.detach().to(dtype).double().cpu(), w, m.bias.detach().to(dtype).double().cpu(), rounded=True)
    with torch.autocast("cuda", dtype, enabled=False):
        assert m(x).dtype == torch.float32


@pytest.fixture
def made(monkeypatch):
    """load_compressed on the CPU: the packed weights are stand-ins that know their shape."""
    from llmcompressorsharp_b200 import Int4Weight

    def from_entry(e, cols):
        p = object.__new__(Int4Weight)
        p.shape, p.strategy, p.group_size = (e["rows"], cols), "channel", cols
        return p

    monkeypatch.setattr(Int4Weight, "from_entry", staticmethod(from_entry))
    return lambda m: {f"{n}.weight": {"codes": 1, "num_bits": 4, "rows": m.get_submodule(n).weight.shape[0]} for n in ("a", "b", "c", "d")}


def test_hooks_and_training_go_with_the_module(made):
    from llmcompressorsharp_b200 import Int4Embedding, Int4Linear, load_compressed

    m = torch.nn.ModuleDict({"a": torch.nn.Linear(8, 4), "b": torch.nn.Embedding(5, 8), "c": torch.nn.Linear(8, 4), "d": torch.nn.Linear(8, 4)})
    m["a"].eval()
    seen = []
    handles = [m["a"].register_forward_hook(lambda mod, args, kwargs, out: seen.append(("a", kwargs)), with_kwargs=True),
               m["a"].register_forward_pre_hook(lambda mod, args: seen.append("pre")),
               m["a"].register_full_backward_hook(lambda mod, gi, go: seen.append("back")),
               m["b"].register_forward_hook(lambda mod, args, out: out + 1)]
    assert load_compressed(m, made(m)) == ["a", "b", "c", "d"]
    assert type(m["a"]) is Int4Linear and type(m["b"]) is Int4Embedding
    assert not m["a"].training and m["b"].training and m["c"].training
    m["a"].forward = lambda x: x * 2
    m["b"].forward = lambda ids: ids * 2
    x = torch.ones(2, 8, requires_grad=True)
    m["a"](x).sum().backward()
    assert seen == ["pre", ("a", {}), "back"]
    assert torch.equal(m["b"](torch.tensor([1, 2])), torch.tensor([3, 5]))
    for h in handles:
        h.remove()
    m["a"](x)
    assert len(seen) == 3 and torch.equal(m["b"](torch.tensor([1, 2])), torch.tensor([2, 4]))


def test_what_a_packed_module_cannot_hold_stays_dense(made):
    """A type that the products do not take, and a weight that a hook computes before each call."""
    from llmcompressorsharp_b200 import load_compressed

    m = torch.nn.ModuleDict({"a": torch.nn.Linear(8, 4).double(), "b": torch.nn.Embedding(5, 8, dtype=torch.float64),
                             "c": torch.nn.utils.spectral_norm(torch.nn.Linear(8, 4)), "d": torch.nn.Linear(8, 4)})
    assert load_compressed(m, made(m)) == ["d"]
    assert m["a"](torch.ones(2, 8, dtype=torch.float64)).dtype == torch.float64 and m["c"](torch.ones(2, 8)).shape == (2, 4)


def test_a_layout_of_more_columns_than_32_bits_count_is_refused():
    """Groups of 16 columns take 32 of the layout: 2^30 columns would be 2^31 there."""
    import ctypes as C

    from llmcompressorsharp_b200 import _lib

    lib = _lib.load()
    p, x = C.c_int64(), C.c_int64()
    assert lib.llmc_int4_layout_sizes(1, 1 << 30, 16, C.byref(p), C.byref(x)) == 10  # LLMC_ERR_OUT_OF_RANGE
    assert lib.llmc_int4_layout_sizes(1, 1 << 30, 100, C.byref(p), C.byref(x)) == 10
    assert lib.llmc_int4_layout_sizes(1, 1 << 29, 16, C.byref(p), C.byref(x)) == 0
    assert lib.llmc_int4_layout_sizes(1, 1 << 30, 128, C.byref(p), C.byref(x)) == 0
    assert lib.llmc_int4_layout_sizes(1, 1 << 30, 1 << 30, C.byref(p), C.byref(x)) == 0


@pytest.mark.gpu
def test_a_session_over_a_packed_table_hears_of_a_bad_id():
    from llmcompressorsharp_b200 import (CompressionSession, CompressionState, Int4Embedding, Int4Weight, RtnConfig, RtnModifier, SessionStatus,
                                         embedding)
    from llmcompressorsharp_b200.calibration import drive
    from llmcompressorsharp_b200.errors import ArgumentOutOfRangeError

    lin = torch.nn.Linear(64, 32, bias=False, device=ROOT_DEV)
    w = torch.randn(20, 64, generator=torch.Generator().manual_seed(0)).to(ROOT_DEV)
    m = torch.nn.Sequential(Int4Embedding(Int4Weight.from_float(w, RtnConfig(4, True, "channel")), torch.float32), lin)

    def run(ids):
        s = CompressionSession([RtnModifier(RtnConfig(4, True, "channel"))])
        return s.run(CompressionState({"1.weight": lin.weight.detach()}), drive(m, [torch.tensor([i], device=ROOT_DEV) for i in ids])), s.failure

    assert run([3, 19]) == (SessionStatus.COMPLETED, None)
    status, failure = run([3, 20])
    assert status == SessionStatus.FAILED and isinstance(failure, ArgumentOutOfRangeError)
    assert run([3, 19]) == (SessionStatus.COMPLETED, None)
    embedding(torch.tensor([-1], device=ROOT_DEV), w)  # anyone's
    with pytest.warns(UserWarning, match="outside its table"):
        assert run([3, 19]) == (SessionStatus.COMPLETED, None)
