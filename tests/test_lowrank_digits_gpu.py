"""What the 16-bit forms of the adapter operators keep of P's 32 bits, and what they make of infinities."""
import pytest
import torch

import eigen_amd
from eigen_amd import lowrank
import lowrank_ref as ref
from lowrank_ref import KINDS, NAME, TORCH
from test_lowrank_gpu import Case, Grad, rand, store, store_stack, turned

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


# ------------------------------------------------------------------------------------------ the low-rank part of the product
def whole_numbers(shape, low, high, seed):
    return torch.randint(low, high + 1, shape, generator=torch.Generator().manual_seed(seed)).double()


# tiles of 256 x 256 and 128 x 128, a split reduction, extents that are copied first, the matrix-unit join of few tokens, and the
# joins that do without
SIZES = [(256 * 15 + 8, 256 * 14 + 37, 200, 16), (1100, 1130, 200, 40), (1101, 1130, 203, 7), (1096, 1130, 1288, 16), (1601, 130, 136, 100),
         (130, 70, 200, 33), (40, 17, 136, 16), (24, 1, 200, 4)]


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("m, n, k, rank", SIZES)
def test_the_low_rank_part_uses_all_of_p(kind, opw, m, n, k, rank):
    """Whole numbers, so that every sum is exact in 32 bits: P has 19 to 22 bits, neighbouring ranks of it differ by one entry of x and
    enter with opposite signs, and what is left has to be right to the last bit.  (P is about 255 / 2 * 31 / 2 * k, and half of the pairs of ranks
    take part: below 2^24 in every case.)"""
    c = Case(kind, m, n, k, rank, 3, opw + "TT")
    c.x = whole_numbers((k, n), 0, 255, 1)
    c.a = whole_numbers((3, rank, k), 0, 31, 2)
    c.b = torch.zeros(3, m, rank).double()
    pairs = rank // 2
    c.a[:, 1:2 * pairs:2] = c.a[:, 0:2 * pairs:2]
    for r in range(pairs):
        c.a[:, 2 * r + 1, (7 * r) % k] += 1
    some = whole_numbers((3, m, pairs), 0, 1, 3)
    c.b[:, :, 0:2 * pairs:2], c.b[:, :, 1:2 * pairs:2] = some, -some
    c.w = torch.zeros(m, k).double()
    c.w[:, ::16] = whole_numbers((m, (k + 15) // 16), -1, 1, 4)
    c.scale = torch.tensor([0.5, 1.0, -0.25])
    c.S = c.scale.cuda()
    c.W, c.X = store(turned(c.w, opw), kind), store(c.x, kind)
    c.A, c.B = store_stack(turned(c.a, "T"), kind), store_stack(turned(c.b, "T"), kind)
    c.run()
    d = [t.cuda() for t in (c.w, c.x, c.a, c.b)]
    y, p, _, _ = ref.lora(*d, c.scale.double().cuda(), c.ids.cuda())
    assert torch.equal(c.P.as_strided().double(), p)
    assert torch.equal(c.Y.as_strided(), y.to(TORCH[kind]))


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("m, n, k, rank", [(256 * 15 + 8, 256 * 14 + 37, 72, 12), (1100, 1130, 72, 40), (1601, 130, 136, 100), (130, 70, 72, 9)])
def test_quiet_ranks_beside_loud_ones_reach_y(kind, m, n, k, rank):
    """P of ranks 2^29 apart: the loud ones meet zeros, and a scale brings the quiet ones back."""
    c = Case(kind, m, n, k, rank, 2, "TTT")
    quiet = (torch.arange(rank) % 3 > 0).double()
    c.a = (rand(c.a.shape, kind, 31) * 2.0 ** (13.0 - 29.0 * quiet).unsqueeze(1)).to(TORCH[kind]).double()
    c.x = (c.x * 2.0 ** (torch.arange(n) % 3 - 1.0)).to(TORCH[kind]).double()
    c.b = c.b * quiet
    c.w = torch.zeros_like(c.w)
    c.scale = torch.tensor([2.0 ** 9, 2.0 ** 10])
    c.S = c.scale.cuda()
    c.W, c.X = store(turned(c.w, "T"), kind), store(c.x, kind)
    c.A, c.B = store_stack(turned(c.a, "T"), kind), store_stack(turned(c.b, "T"), kind)
    c.run()
    y, p, ya, pa = ref.lora(*[t.cuda() for t in (c.w, c.x, c.a, c.b)], c.scale.double().cuda(), c.ids.cuda())
    # as lora_tolerance, but nothing of P left out: k + rank products in 32 bits, and the one rounding
    tol = ref.HALF[kind] * y.abs() + (2 * k + rank + 32) * 2.0 ** -23 * ya * (1 + ref.HALF[kind]) + ref.SMALL[kind]
    err = (c.Y.as_strided().double() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


# --------------------------------------------------------------------------------------------------------------- infinities
@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("m, n, k, rank", [(1100, 1130, 72, 20), (1601, 130, 136, 100), (72, 40, 72, 9), (24, 1, 72, 9)])
def test_an_infinite_factor_gives_an_infinity_of_the_right_sign(kind, opw, m, n, k, rank):
    c = Case(kind, m, n, k, rank, 2, opw + "TT", ids=[i % 2 for i in range(n)])
    c.a[0, 3] = 0.0
    c.a[0, 3, 5] = 1.0                       # p of rank 3 is one entry of x: a few bits, the other pieces of it are empty
    c.x[5] = torch.where(torch.arange(n) % 4 < 2, 1.0, -1.5).double()
    c.A, c.X = store_stack(turned(c.a, "T"), kind), store(c.x, kind)
    c.b[0, 2, 3] = float("inf")
    c.b[0, 7, 4] = float("-inf")
    c.B = store_stack(turned(c.b, "T"), kind)
    c.run()
    on = c.ids.cuda() == 0
    y, p = c.Y.as_strided().double(), c.P.as_strided().double()
    assert torch.equal(y[2][on], torch.sign(p[3][on]) * float("inf") * float(c.scale[0]))
    assert torch.equal(y[7][on], -torch.sign(p[4][on]) * float("inf") * float(c.scale[0]))
    rest = torch.ones_like(y, dtype=torch.bool)
    rest[2, on] = rest[7, on] = False
    assert bool(torch.isfinite(y[rest]).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("m, n, k, rank", [(1100, 1130, 72, 20), (1601, 130, 136, 100), (72, 40, 72, 9), (24, 1, 72, 9)])
def test_an_infinite_projection_gives_infinities_of_the_right_sign(kind, opw, m, n, k, rank):
    c = Case(kind, m, n, k, rank, 2, opw + "TT", ids=[i % 2 for i in range(n)])
    c.a[0, 3, 5] = float("-inf")
    c.b[0, ::3, 3] = 0.5                     # (few bits, as above)
    c.b[0, 1, 3], c.b[0, 4, 3] = 0.0, float("inf")
    c.A, c.B = store_stack(turned(c.a, "T"), kind), store_stack(turned(c.b, "T"), kind)
    c.run()
    on = c.ids.cuda() == 0
    y, p = c.Y.as_strided().double(), c.P.as_strided().double()
    assert torch.equal(p[3][on], (-torch.sign(c.x[5]) * float("inf")).cuda()[on]) and bool(torch.isfinite(p[:, ~on]).all())
    want = torch.sign(c.b[0, :, 3]).cuda().unsqueeze(1) * p[3][on]            # 0 * inf: NaN
    got = y[:, on]
    assert torch.equal(torch.nan_to_num(got, nan=7.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(want, nan=7.0, posinf=1.0, neginf=-1.0))
    assert bool(torch.isfinite(y[:, ~on]).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_an_infinite_gradient_gives_an_infinity_of_the_right_sign(kind, opg, spread):
    """u of +-infinity: G's row is +-infinity by the sign of p (NaN where p is 0); and the other way round."""
    c = Grad(kind, 72, 90, 20, 1, opg, ids=[0] * 90)
    c.scale = torch.ones(1)
    c.p[:, 4] = torch.where(torch.arange(20) % 2 == 0, 1.0, -3.0).double()      # a few bits of 24
    c.p[7, 4] = 0.0
    c.p[:, 5:] *= 2.0 ** spread
    c.p[3, 8] = float("-inf")
    c.u[11, 4] = float("inf")
    c.u[5, 8] = 0.0
    c.P, c.U = store(c.p, F32), store(c.u, kind)
    c.run()
    got = c.got()[0].double().cpu()
    want = torch.sign(c.p[:, 4]) * float("inf")          # (0 * inf: NaN)
    other = torch.arange(20) != 3
    assert torch.equal(torch.nan_to_num(got[11][other], nan=7.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(want[other], nan=7.0, posinf=1.0, neginf=-1.0))
    rows = torch.arange(72) != 11
    column = -torch.sign(c.u[:, 8]) * float("inf")       # rank 3: p of token 8 is -infinity, u of row 5 is 0 there
    assert torch.equal(torch.nan_to_num(got[rows, 3], nan=7.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(column[rows], nan=7.0, posinf=1.0, neginf=-1.0))
    assert bool(torch.isfinite(got[rows][:, other]).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("m, n, k, rank", [(256 * 15 + 8, 256 * 14 + 37, 72, 12), (1100, 1130, 72, 40), (1601, 130, 136, 100), (72, 40, 72, 9)])
def test_what_a_request_gets_does_not_depend_on_infinities_beside_it(kind, m, n, k, rank):
    c = Case(kind, m, n, k, rank, 5).run()
    y, p = c.Y.as_strided().clone(), c.P.as_strided().clone()
    c.B.matrix(1).as_strided()[2, 3] = float("inf")
    c.A.matrix(3).as_strided()[5, 1] = float("nan")
    c.run()
    rest = ((c.ids != 1) & (c.ids != 3)).cuda()
    assert torch.equal(c.Y.as_strided()[:, rest], y[:, rest]) and torch.equal(c.P.as_strided()[:, rest], p[:, rest])
    assert not torch.equal(c.Y.as_strided(), y)


# ------------------------------------------------------------------------- where f16's pieces end and single precision begins
@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("m, n, rank", [(1100, 1130, 16), (1601, 130, 100)])
@pytest.mark.parametrize("spread", [10, 20, 23, 24, 25, 26, 27])
def test_quiet_ranks_at_every_distance_reach_y(kind, m, n, rank, spread):
    c = Case(kind, m, n, 72, rank, 2, "TTT")
    quiet = (torch.arange(rank) % 5 > 0).double()
    c.a = (rand(c.a.shape, kind, 41) * 2.0 ** (12.0 - spread * quiet).unsqueeze(1)).to(TORCH[kind]).double()
    c.b = c.b * quiet
    c.w = torch.zeros_like(c.w)
    c.scale = torch.tensor([2.0 ** (spread - 18), -2.0 ** (spread - 17)])
    c.S = c.scale.cuda()
    c.W, c.A, c.B = store(turned(c.w, "T"), kind), store_stack(turned(c.a, "T"), kind), store_stack(turned(c.b, "T"), kind)
    c.run()
    y, p, ya, pa = ref.lora(*[t.cuda() for t in (c.w, c.x, c.a, c.b)], c.scale.double().cuda(), c.ids.cuda())
    tol = ref.HALF[kind] * y.abs() + (2 * c.k + rank + 32) * 2.0 ** -23 * ya * (1 + ref.HALF[kind]) + ref.SMALL[kind]
    err = (c.Y.as_strided().double() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("opg", "NT")
@pytest.mark.parametrize("spread", [8, 13, 14, 15, 16, 17, 18, 25])
def test_quiet_tokens_at_every_distance_keep_their_digits(kind, opg, spread):
    """Every second token's p is 2^-spread times the others', and rows of u in which only these tokens are not zero."""
    c = Grad(kind, 80, 200, 20, 1, opg, ids=[0] * 200)
    quiet = torch.arange(200) % 2 == 1
    c.p = torch.where(quiet, c.p * 2.0 ** -spread, c.p).float().double()
    c.u = torch.where((torch.arange(80) % 2 == 0).unsqueeze(1) | quiet, c.u, torch.zeros(()).double())
    c.P, c.U = store(c.p, F32), store(c.u, kind)
    c.run().check()
