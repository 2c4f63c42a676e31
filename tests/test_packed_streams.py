"""Products on two streams at once, many of them: the SMs pass from one kernel to the other in mid-run, copies come late
and early, and every product has the bits that it has alone."""

import pytest
import torch

from test_packed import ROOT_DEV, entry, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,group,tokens", [(300, 1000, 128, 20000), (300, 1000, 64, 5000), (1801, 1030, 128, 2100), (257, 640, 32, 400)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("back", [True, False])
def test_thousands_of_products_on_two_streams(m, n, group, tokens, dtype, back):
    p = weight(entry(m, n, group=group, device=ROOT_DEV)[0], n)
    g = torch.Generator().manual_seed(tokens)
    src = [torch.randn(tokens, m if back else n, generator=g).to(ROOT_DEV, dtype) for _ in range(2)]
    want = [p._product(a, None, back) for a in src]
    wrong = torch.zeros((), dtype=torch.int64, device=ROOT_DEV)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(100):
        got = []
        for i in (0, 1) * 4:
            with torch.cuda.stream(streams[i]):
                got.append((i, p._product(src[i], None, back)))
        torch.cuda.synchronize()
        for i, y in got:
            wrong += (y != want[i]).any()
        torch.cuda.synchronize()
    assert int(wrong) == 0, f"{int(wrong)} of 800 products differ from the one made alone"
