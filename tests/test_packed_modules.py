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
