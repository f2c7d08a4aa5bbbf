"""The adapter operators on paths that small shapes do not reach: no adapters, very many, wide projections, large calls in single
precision, and what lies around the gradients' matrices."""
import pytest
import torch

import eigen_amd
from eigen_amd import _lib, lowrank
from lowrank_ref import KINDS, NAME
from test_lowrank_gpu import MARK, Case, Grad, turned

pytestmark = pytest.mark.gpu
F32, BF16, F16 = eigen_amd.F32, eigen_amd.BF16, eigen_amd.F16


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


# ------------------------------------------------------------------------------------------------------------ many adapters
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("n, rank, count", [(2, 3, 65), (17, 64, 4096), (64, 20, 200), (130, 5, 65), (130, 40, 4096), (700, 20, 200), (700, 9, 4096)])
def test_lora_with_many_adapters(kind, opw, n, rank, count):
    c = Case(kind, 40, n, 72, rank, count, opw + "TT").run()
    c.check()
    # all tokens with the last ones, and none with any
    for ids in ([count - 1 - i % 2 for i in range(n)], [-1] * n):
        c.ids = torch.tensor(ids, dtype=torch.int32)
        c.plan = lowrank.lora_plan(c.ids.cuda(), count)
        c.run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n, rank, count", [(17, 33, 4096), (64, 5, 200), (700, 16, 65), (1500, 5, 4096), (5000, 7, 129)])
def test_lora_wgrad_with_many_adapters(kind, n, rank, count):
    for opg, beta in (("N", 0.0), ("T", 1.0)):
        c = Grad(kind, 40, n, rank, count, opg, beta).run()
        c.check()
        # a few long runs far apart among empty ones, in the order of their adapters and against it
        for ids in ([(0, 63, 64, count - 1)[i * 4 // n] for i in range(n)], [count - 1 - i * 3 // (2 * n) for i in range(n)]):
            c.ids = torch.tensor(ids, dtype=torch.int32)
            c.plan = lowrank.lora_plan(c.ids.cuda(), count)
            if beta:
                for j in range(count):
                    c.G.matrix(j).as_strided().copy_(turned(c.g0[j], opg))
            c.run().check()


@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("count", [61, 4096])
def test_lora_wgrad_of_runs_just_longer_than_a_piece(opg, count):
    """Pieces are 128 tokens here: runs of one token more, twice as many and one, one less, one by one behind each other."""
    ids = [j for j, length in enumerate([129, 257, 129, 128, 385, 1, 127, 129, 130, 255, 256, 257] * 5) for _ in range(length)]
    Grad(_lib.BF16, 40, len(ids), 5, count, opg, ids=ids).run().check()


# --------------------------------------------------------------------------------------------------------- wide projections
# With this many tokens the projection takes 32 ranks a workgroup (4100 tokens: rank 33, 40, 64) or 64 (8200 tokens, and rank 100 and
# 128), and the call is larger than the few-token form takes.
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("ops", ["TTT", "TNN"])
@pytest.mark.parametrize("n, rank, k", [(4100, 33, 72), (4100, 40, 200), (4100, 64, 1288), (8200, 40, 83), (8200, 64, 264), (4100, 100, 136), (4100, 128, 603)])
def test_wide_projections(kind, ops, n, rank, k):
    Case(kind, 520 if kind == F32 and n < 8000 else 264, n, k, rank, 3, ops).run().check()


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("ops", ["TTT", "NNN"])
def test_large_tiles_with_several_turns_of_ranks(kind, ops):
    Case(kind, 256 * 15 + 8, 256 * 14 + 37, 200, 100, 6, ops).run().check()


# ------------------------------------------------------------------------------------------------ large single precision calls
@pytest.mark.parametrize("ops", ["TTT", "NNN"])
@pytest.mark.parametrize("m, n, k, rank, count, pad", [(2051, 1100, 72, 7, 3, 0), (1030, 2047, 136, 40, 5, 3), (2048, 1024 + 64, 2056, 16, 2, 0), (2050, 1090, 1003, 16, 9, 1)])
def test_large_calls_in_single_precision(ops, m, n, k, rank, count, pad):
    """More than 512 blocks of 64 x 64: the library's product, and the low-rank part behind it."""
    Case(F32, m, n, k, rank, count, ops, pad=pad).run().check()


def test_large_single_precision_calls_repeat_in_graphs_and_on_streams():
    cases = [Case(F32, 2051, 1100, 264, 7, 3, "TTT", seed=s) for s in (1, 50)]
    want = []
    for c in cases:
        c.run().check()
        want.append((c.Y.storage.clone(), c.P.storage.clone()))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            c.run(stream=s)
    torch.cuda.synchronize()
    for c, (y, p) in zip(cases, want):
        assert torch.equal(c.Y.storage, y) and torch.equal(c.P.storage, p)
    c, (y, p) = cases[0], want[0]
    work = torch.empty(lowrank.lora_work_bytes("T", c.W, c.X), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(work=work)
    for _ in range(3):
        c.Y.as_strided().zero_()
        c.P.as_strided().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.Y.storage, y) and torch.equal(c.P.storage, p)
        c.run(work=work)
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------- around the gradients
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("rows, n, rank", [(1, 3, 1), (264, 70, 16), (261, 140, 7), (130, 1300, 33), (300, 90, 130)])
def test_lora_wgrad_writes_its_matrices_only(kind, packed, opg, rows, n, rank):
    """Rows below, columns behind and the gaps between neighbouring adapters' matrices: one with several pieces, one with one, one empty."""
    for beta, pad in ((0.0, 1), (0.5, 4)):
        c = Grad(kind, rows, n, rank, 4, opg, beta, pad, 0, packed, ids=[(0, 1, 1, 1, -1, 3)[i * 6 // n] for i in range(n)]).run()
        c.check()
        inside = torch.zeros(c.G.storage.numel(), dtype=torch.bool, device="cuda")
        for j in range(c.count):
            torch.as_strided(inside, (c.G.rows, c.G.cols), (1, c.G.ld), j * c.G.stride).fill_(True)
        assert bool((c.G.storage[~inside] == MARK).all())
