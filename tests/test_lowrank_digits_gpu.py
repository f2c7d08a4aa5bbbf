"""What the 16-bit forms of the adapter operators keep of P's 32 bits."""
import pytest
import torch

import eigen_amd
from eigen_amd import lowrank
import lowrank_ref as ref
from lowrank_ref import KINDS, NAME
from test_lowrank_gpu import Grad, store

pytestmark = pytest.mark.gpu
F32, BF16, F16 = eigen_amd.F32, eigen_amd.BF16, eigen_amd.F16


# ------------------------------------------------------------------------------------------------ gradients of the factors
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("rank", [6, 20, 40])
def test_quiet_ranks_beside_loud_ones_keep_their_digits(kind, packed, opg, rank):
    """Every rank is an output of its own: p of neighbouring ranks 2^10 apart, up to 2^60."""
    c = Grad(kind, 130, 300, rank, 2, opg, packed=packed)
    c.p = (c.p * 2.0 ** (20.0 - 10.0 * (torch.arange(rank) % 7).double().unsqueeze(1))).float().double()
    c.P = store(c.p, F32)
    c.run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("rank", [6, 40])
def test_quiet_tokens_beside_loud_ones_keep_their_digits(kind, packed, opg, rank):
    """Tokens whose p is up to 2^84 apart, and rows of u in which only the tokens of one magnitude are not zero."""
    c = Grad(kind, 64, 400, rank, 1, opg, ids=[0] * 400)
    which = torch.arange(400) % 8
    c.p = (c.p * 2.0 ** (24.0 - 12.0 * which.double())).float().double()
    c.u = torch.where((torch.arange(64) % 8).unsqueeze(1) == which, c.u, torch.zeros(()).double())
    c.P, c.U = store(c.p, F32), store(c.u, kind)
    if packed:
        ck = lowrank.Checkpoint8(64, 400, kind)
        lowrank.ckpt8_pack_dev(c.U, ck)
        back = store(torch.zeros(64, 400), kind)
        lowrank.ckpt8_unpack_dev(ck, back)
        c.u, c.U = back.as_strided().double().cpu(), ck
    c.run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opg", "NT")
def test_gradients_of_projections_at_both_ends_of_floats_range(kind, opg):
    for size in (2.0 ** 126, 2.0 ** -110):
        c = Grad(kind, 40, 70, 18, 2, opg)
        c.p = (c.p * size).float().double()
        c.u = c.u * 2.0 ** -6
        c.P, c.U = store(c.p, F32), store(c.u, kind)
        c.scale = torch.tensor([0.5, 1.0])
        g, ga = ref.wgrad(c.u.cuda(), c.p.cuda(), c.scale.double().cuda(), c.ids.cuda(), 2)
        c.run()
        assert bool(((c.got().double() - g).abs() <= ref.wgrad_tolerance(c.n, g, ga)).all())
