"""Errors that the device keeps for the next synchronisation: each is reported once, and none hides another."""

import ctypes as C

import pytest
import torch

from test_packed import ROOT_DEV

pytestmark = pytest.mark.gpu

OK, NOT_PD, OUT_OF_RANGE = 0, 4, 10


@pytest.fixture
def ctx():
    from llmcompressorsharp_b200 import _lib

    lib = _lib.load()
    c = C.c_void_p()
    assert lib.llmc_init(0, C.byref(c)) == 0
    assert lib.llmc_set_deferred_errors(c, 1) == 0
    yield lib, c
    lib.llmc_destroy(c)


def bad_id(lib, c):
    table, out = torch.ones(3, 8, device=ROOT_DEV), torch.empty(1, 8, device=ROOT_DEV)
    ids = torch.tensor([3], device=ROOT_DEV)
    assert lib.llmc_embedding(c, C.c_void_p(1), ids.data_ptr(), 1, 1, table.data_ptr(), 0, 3, 8, 8, 1.0, out.data_ptr(), 8) == 0
    torch.cuda.synchronize()
    assert not bool(out.any())


def not_pd(lib, c):
    h, u = -torch.eye(256, device=ROOT_DEV), torch.empty(256, 256, device=ROOT_DEV)
    torch.cuda.synchronize()
    assert lib.llmc_chol_inverse(c, h.data_ptr(), 256, 256, 0.0, 0, u.data_ptr(), 256, 1) == 0
    torch.cuda.synchronize()


def test_a_bad_id_outlives_the_error_that_is_reported_before_it(ctx):
    lib, c = ctx
    for first, second in ((bad_id, not_pd), (not_pd, bad_id)):
        first(lib, c)
        second(lib, c)
        assert [lib.llmc_sync(c) for _ in range(3)] == [NOT_PD, OUT_OF_RANGE, OK]
    bad_id(lib, c)
    assert [lib.llmc_sync(c) for _ in range(2)] == [OUT_OF_RANGE, OK]


def test_a_solve_leaves_an_id_of_another_lookup_pending(ctx):
    lib, c = ctx
    bad_id(lib, c)
    assert lib.llmc_wait(c) == OK
    not_pd(lib, c)
    assert [lib.llmc_wait(c), lib.llmc_wait(c), lib.llmc_sync(c), lib.llmc_sync(c)] == [NOT_PD, OK, OUT_OF_RANGE, OK]


def test_a_gptq_session_is_not_failed_by_an_id_of_another_lookup():
    from llmcompressorsharp_b200 import CompressionSession, CompressionState, GPTQConfig, GPTQModifier, SessionStatus, _lib, embedding
    from llmcompressorsharp_b200.errors import ArgumentOutOfRangeError

    embedding(torch.tensor([3], device=ROOT_DEV), torch.ones(3, 8, device=ROOT_DEV))
    lin = torch.nn.Linear(64, 32, bias=False, device=ROOT_DEV)
    state = CompressionState({"lin.weight": lin.weight.detach()})
    state.named_modules = {"lin": lin}

    def batches():
        for i in range(2):
            x = torch.randn(96, 64, generator=torch.Generator().manual_seed(i)).to(ROOT_DEV)
            lin(x)
            yield x

    session = CompressionSession([GPTQModifier(GPTQConfig(num_bits=4, symmetric=True, strategy="channel"))])
    assert session.run(state, batches()) == SessionStatus.COMPLETED, session.failure
    assert "lin.weight" in state.compressed
    with pytest.raises(ArgumentOutOfRangeError):
        _lib.call("llmc_sync", _lib.ctx_for(0))
