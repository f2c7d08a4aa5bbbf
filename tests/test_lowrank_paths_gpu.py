"""The adapter operators without adapters."""
import pytest
import torch

from eigen_amd import _lib, lowrank
from lowrank_ref import KINDS, NAME
from test_lowrank_gpu import Case

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------- no adapters
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("m, n, k, rank", [(64, 1, 96, 5), (64, 1, 96, 40), (64, 7, 96, 40), (64, 200, 96, 4), (1100, 1130, 72, 33), (2, 300, 24, 6),
                                           (2051, 1100, 72, 9), (16, 4, 0, 3)])
def test_without_adapters_p_is_zero(kind, opw, m, n, k, rank):
    """Every token is one without an adapter: a zero column of P."""
    c = Case(kind, m, n, k, rank, 0, opw + "TT", pad=3)
    c.P.as_strided().fill_(7.0)
    c.run().check()
    assert not c.P.as_strided().any()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n", [1, 40, 300])
def test_without_adapters_there_may_be_no_p(kind, n):
    c = Case(kind, 64, n, 96, 4, 0).run()
    y = c.Y.storage.clone()
    c.Y.as_strided().zero_()
    work = torch.empty(max(lowrank.lora_work_bytes("T", c.W, c.X), 1), dtype=torch.uint8, device="cuda")
    rc = _lib.lib.eigamd_lora_dev(kind, _lib.OP_T, _lib.OP_T, _lib.OP_T, 64, n, 96, 4, 0, c.W.ptr, c.W.ld, c.X.ptr, c.X.ld, 0, 1, 0, 0, 1, 0, 0,
                                  c.plan.storage.data_ptr(), 0, 1, c.Y.ptr, c.Y.ld, work.data_ptr(), work.numel(),
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.OK and torch.equal(c.Y.storage, y)
