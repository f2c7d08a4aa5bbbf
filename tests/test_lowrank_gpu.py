"""Adapter and 8-bit checkpoint operators on the device against their formulas in 64 bits."""
import pytest
import torch

import eigen_amd
from eigen_amd import _lib, lowrank
from eigen_amd.device import DeviceMatrix
import lowrank_ref as ref
from lowrank_ref import KINDS, NAME, TORCH

pytestmark = pytest.mark.gpu
F32, BF16, F16 = eigen_amd.F32, eigen_amd.BF16, eigen_amd.F16
MARK = 12345.0     # stands in every element that no call may write


def rand(shape, kind, seed, scale=1.0):
    g = torch.Generator()
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(TORCH[kind]).double()


def store(t, kind, pad=0, shift=0):
    """t (rows, cols) as a DeviceMatrix with `pad` marked rows below and `shift` elements in front."""
    rows, cols = t.shape
    ld = max(rows + pad, 1)
    flat = torch.full((shift + ld * max(cols, 1),), MARK, dtype=TORCH[kind], device="cuda")
    m = DeviceMatrix(rows, cols, kind, ld=ld, storage=flat, offset=shift)
    m.as_strided().copy_(t.to(TORCH[kind]))
    return m


def store_stack(t, kind, pad=0):
    count, rows, cols = t.shape
    ld = max(rows + pad, 1)
    stride = ld * max(cols, 1) + pad
    flat = torch.full((stride * max(count, 1),), MARK, dtype=TORCH[kind], device="cuda")
    s = lowrank.MatrixStack(rows, cols, count, kind, ld=ld, stride=stride, storage=flat)
    for j in range(count):
        s.matrix(j).as_strided().copy_(t[j].to(TORCH[kind]))
    return s


def turned(t, op):
    return t if op == "N" else t.transpose(-1, -2)


def untouched(m, rows, cols):
    """Everything of the storage outside the matrix still holds the mark."""
    inside = torch.zeros(m.storage.numel(), dtype=torch.bool, device="cuda")
    torch.as_strided(inside, (rows, cols), (1, m.ld), m.offset).fill_(True)
    return bool((m.storage[~inside] == torch.tensor(MARK, dtype=m.storage.dtype)).all())


class Case:
    def __init__(self, kind, m, n, k, rank, count, ops="TTT", pad=0, shift=0, ids=None, seed=1):
        self.kind, self.m, self.n, self.k, self.rank, self.count, self.ops = kind, m, n, k, rank, count, ops
        self.w = rand((m, k), kind, seed, max(k, 1) ** -0.5)
        self.x = rand((k, n), kind, seed + 1)
        self.a = rand((count, rank, k), kind, seed + 2, max(k, 1) ** -0.5)
        self.b = rand((count, m, rank), kind, seed + 3)
        self.scale = (torch.arange(count) * 0.25 + 0.5).float()
        g = torch.Generator()
        g.manual_seed(seed + 4)
        self.ids = torch.randint(-1, max(count, 1), (n,), generator=g).to(torch.int32) if ids is None else torch.tensor(ids, dtype=torch.int32)
        self.W, self.X = store(turned(self.w, ops[0]), kind, pad, shift), store(self.x, kind, pad, shift)
        self.A, self.B = store_stack(turned(self.a, ops[1]), kind, pad), store_stack(turned(self.b, ops[2]), kind, pad)
        self.S = self.scale.cuda()
        self.plan = lowrank.lora_plan(self.ids.cuda(), count)
        self.P = store(torch.zeros(rank, n), F32, pad)
        self.Y = store(torch.zeros(m, n), kind, pad, shift)

    def run(self, **more):
        lowrank.lora_dev(self.ops[0], self.W, self.X, self.ops[1], self.A, self.ops[2], self.B, self.S, self.plan, self.P, self.Y, **more)
        return self

    def check(self):
        d = [t.cuda() for t in (self.w, self.x, self.a, self.b)]
        y, p, ya, pa = ref.lora(*d, self.scale.double().cuda(), self.ids.cuda())
        ty, tp = ref.lora_tolerance(self.kind, self.k, self.rank, y, ya, pa)
        gy, gp = self.Y.as_strided().double(), self.P.as_strided().double()
        if self.count:
            assert bool(((gp - p).abs() <= tp).all()), ("P", float(((gp - p).abs() - tp).max()))
        assert bool(((gy - y).abs() <= ty).all()), ("Y", float(((gy - y).abs() - ty).max()))
        assert untouched(self.Y, self.m, self.n) and untouched(self.P, self.rank, self.n)


# one element; fewer than a tile; whole tiles; extents that are multiples of nothing; a split reduction; both sides of 64 tokens
SHAPES = [(1, 1, 1, 1, 1), (16, 3, 8, 5, 2), (40, 17, 136, 16, 3), (128, 64, 128, 16, 1), (130, 70, 200, 33, 4), (257, 129, 264, 64, 5),
          (72, 300, 1288, 8, 7), (33, 65, 77, 100, 2), (256, 33, 1024, 256, 40)]


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("m, n, k, rank, count", SHAPES)
def test_lora_against_64_bits(kind, m, n, k, rank, count):
    for opw in "TN":
        Case(kind, m, n, k, rank, count, opw + "TT").run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("ops", ["TNT", "TTN", "NNN", "NTN"])
@pytest.mark.parametrize("m, n, k, rank", [(24, 20, 72, 12), (130, 150, 136, 33)])
def test_lora_forms_of_the_factors(kind, ops, m, n, k, rank):
    Case(kind, m, n, k, rank, 3, ops).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("pad, shift", [(8, 0), (3, 0), (8, 1), (0, 3)])
def test_lora_leading_dimensions_and_alignment(kind, opw, pad, shift):
    for n in (9, 140):
        Case(kind, 136, n, 72, 9, 3, opw + "TN", pad, shift).run().check()


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
def test_lora_large_tiles(kind, opw):
    # more than 200 tiles of 256 x 256, ragged both ways, a reduction that ends inside a slice
    Case(kind, 256 * 15 + 8, 256 * 14 + 37, 200, 16, 6, opw + "TT").run().check()


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("ops", ["TTT", "NTT", "TNN", "NNN"])
@pytest.mark.parametrize("m, n, k, rank", [(1100, 1130, 200, 40), (1101, 1130, 203, 7), (1096, 1130, 1288, 16), (2200, 2300, 264, 24), (1, 9000, 64, 3)])
def test_lora_small_tiles(kind, ops, m, n, k, rank):
    # tiles of 128 x 128, one or two to a compute unit, whole and split reductions, extents that are copied first
    Case(kind, m, n, k, rank, 5, ops).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("pad, shift", [(0, 0), (3, 1)])
@pytest.mark.parametrize("m, n, k, rank", [(130, 1, 2056, 32), (97, 1, 1003, 7), (16, 1, 7, 33), (520, 1, 4096, 16), (33, 2, 264, 9)])
def test_lora_single_tokens(kind, pad, shift, m, n, k, rank):
    # on both sides of 32 ranks; with and without an adapter
    for ids in ([0] * n, [-1] * n, [2, 9, 0, 2][:n]):
        Case(kind, m, n, k, rank, 3, "TTT", pad, shift, ids=ids).run().check()
    Case(kind, m, n, k, rank, 3, "TTN", pad, shift).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("pad, shift", [(0, 0), (1, 1), (8, 0)])
@pytest.mark.parametrize("m", [1, 7, 8, 9, 12, 63, 65, 68, 127])
def test_lora_few_tokens_and_rows_that_end_inside_a_chunk(kind, pad, shift, m):
    for n in (2, 70):
        Case(kind, m, n, 75, 5, 2, "NTT", pad, shift).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("ops", ["TTT", "NNN"])
@pytest.mark.parametrize("m, n, k, rank", [(1601, 130, 136, 100), (1600, 99, 520, 130)])
def test_lora_few_tokens_and_large_ranks(kind, ops, m, n, k, rank):
    Case(kind, m, n, k, rank, 9, ops).run().check()


@pytest.mark.parametrize("opw, ld", [("T", 2 ** 23 + 8), ("N", 2 ** 25 + 8)])
def test_a_leading_dimension_of_several_gigabytes_a_tile(opw, ld):
    # one tile's rows (lines) span more than 2^32 bytes
    c = Case(BF16, 260, 4100, 72, 16, 3, opw + "TT")
    c.W = store(turned(c.w, opw), BF16, ld - c.W.rows)
    c.run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n", [5, 130])
def test_lora_who_has_an_adapter(kind, n):
    for ids in ([-1] * n, [0] * n, [1] * (n - 1) + [99], [-7, 2, 0, 2, 5] * (n // 5), list(range(3)) * (n // 3) + [1] * (n % 3)):
        Case(kind, 48, n, 64, 4, 3, ids=ids).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
def test_lora_without_adapters_is_the_product(kind):
    for n in (7, 200):
        Case(kind, 64, n, 96, 1, 0).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
def test_lora_empty_extents(kind):
    c = Case(kind, 16, 4, 0, 2, 2).run()
    assert not c.Y.as_strided().any() and not c.P.as_strided().any()     # k = 0: nothing to add up
    Case(kind, 16, 0, 8, 2, 2).run()
    c = Case(kind, 0, 4, 8, 2, 2).run()
    torch.cuda.synchronize()
    want = ref.lora(c.w, c.x, c.a, c.b, c.scale.double(), c.ids)[1]
    assert torch.allclose(c.P.as_strided().cpu().double(), want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("opw", "TN")
@pytest.mark.parametrize("n", [20, 150])
def test_what_is_not_finite_stays_with_its_request(kind, opw, n):
    c = Case(kind, 136, n, 72, 5, 3, opw + "TT")
    ids = c.ids.cuda()
    for bad in (float("inf"), float("nan")):
        c.A.matrix(1).as_strided()[0, 0] = bad
        c.B.matrix(1).as_strided()[2, 3] = bad
        c.run()
        hit = ids == 1
        assert bool(hit.any()) and bool((~hit).any())
        assert bool(torch.isfinite(c.Y.as_strided()[:, ~hit]).all()) and bool(torch.isfinite(c.P.as_strided()[:, ~hit]).all())
        assert not bool(torch.isfinite(c.Y.as_strided()[:, hit]).all(dim=0).any())
    d = Case(kind, 136, n, 72, 5, 3, opw + "TT")
    d.X.as_strided()[3, 1] = float("nan")     # one token's activations
    d.run()
    rest = torch.arange(n, device="cuda") != 1
    assert bool(torch.isnan(d.Y.as_strided()[:, 1]).all()) and bool(torch.isfinite(d.Y.as_strided()[:, rest]).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
def test_a_single_token_meets_its_own_adapter_only(kind):
    for ids in ([0], [-1]):
        c = Case(kind, 40, 1, 72, 5, 2, ids=ids)
        c.A.matrix(1).as_strided().fill_(float("nan"))
        c.B.matrix(1).as_strided().fill_(float("inf"))
        c.run().check()
        c.A.matrix(0).as_strided()[0, 0] = float("nan")
        c.run()
        bad = ids == [0]
        assert bool(torch.isnan(c.Y.as_strided()).all()) == bad and bool(torch.isnan(c.P.as_strided()).any()) == bad


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("magnitude", [2.0 ** -40, 2.0 ** 40])
def test_projections_beyond_the_range_of_16_bits(kind, magnitude):
    """P outside f16's range (float keeps it) and scales that bring the result back."""
    c = Case(kind, 32, 100, 64, 8, 2)
    step = 2.0 ** 12 if magnitude > 1 else 2.0 ** -12
    c.a, c.x = c.a * step, c.x * step
    if kind == F16:   # what f16 can hold of it
        c.a, c.x = c.a.to(torch.float16).double(), c.x.to(torch.float16).double()
    c.w = torch.zeros_like(c.w)
    c.W, c.X, c.A = store(c.w.t(), kind), store(c.x, kind), store_stack(c.a.transpose(1, 2), kind)
    c.scale = torch.full((2,), step ** -2)
    c.S = c.scale.cuda()
    c.run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n", [33, 200])
def test_order_of_the_tokens_and_repetition(kind, n):
    c = Case(kind, 72, n, 264, 20, 5)
    c.run()
    y, p = c.Y.as_strided().clone(), c.P.as_strided().clone()
    c.run()
    assert torch.equal(y, c.Y.as_strided()) and torch.equal(p, c.P.as_strided())
    turn = torch.randperm(n, generator=torch.Generator().manual_seed(5))
    d = Case(kind, 72, n, 264, 20, 5)
    d.X = store(c.x[:, turn], kind)
    d.plan = lowrank.lora_plan(c.ids[turn].cuda(), 5)
    d.run()
    assert torch.equal(d.Y.as_strided(), y[:, turn.cuda()]) and torch.equal(d.P.as_strided(), p[:, turn.cuda()])


def test_plan():
    for n, count, seed in ((1, 1, 0), (64, 3, 1), (1000, 70, 2), (65, 0, 3), (0, 4, 4), (300, 4096, 5)):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(-2, count + 2, (n,), generator=g).to(torch.int32)
        plan = lowrank.lora_plan(ids.cuda(), count).storage.cpu()
        key = torch.where((ids >= 0) & (ids < count), ids, torch.tensor(count, dtype=torch.int32))
        order = torch.sort(key, stable=True).indices
        assert torch.equal(plan[:n].long(), order) and torch.equal(plan[n:2 * n], key[order])
        starts = torch.tensor([int((key < j).sum()) for j in range(count + 1)] + [n])
        assert torch.equal(plan[2 * n:].long(), starts)


# ------------------------------------------------------------------------------------------------ gradients of the factors
class Grad:
    def __init__(self, kind, rows, n, rank, count, opg, beta=0.0, pad=0, shift=0, packed=False, ids=None, seed=11):
        self.kind, self.rows, self.n, self.rank, self.count, self.opg, self.beta = kind, rows, n, rank, count, opg, beta
        self.u = rand((rows, n), kind, seed)
        self.p = rand((rank, n), F32, seed + 1, 0.3)
        self.scale = (torch.arange(count) * 0.5 - 0.75).float()
        g = torch.Generator()
        g.manual_seed(seed + 2)
        self.ids = torch.randint(-1, max(count, 1), (n,), generator=g).to(torch.int32) if ids is None else torch.tensor(ids, dtype=torch.int32)
        self.g0 = rand((count, rows, rank), F32, seed + 3)
        self.U, self.P = store(self.u, kind, pad, shift), store(self.p, F32, pad)
        if packed:
            c = lowrank.Checkpoint8(rows, n, kind, ld=max(rows, 1) + pad)
            lowrank.ckpt8_pack_dev(self.U, c)
            back = store(torch.zeros(rows, n), kind)
            lowrank.ckpt8_unpack_dev(c, back)
            self.u = back.as_strided().double().cpu()
            self.U = c
        self.G = store_stack(turned(self.g0 if beta else torch.full_like(self.g0, float("nan")), opg), F32, pad)
        self.plan = lowrank.lora_plan(self.ids.cuda(), count)

    def run(self, **more):
        lowrank.lora_wgrad_dev(self.opg, self.U, self.P, self.scale.cuda(), self.plan, self.beta, self.G, **more)
        return self

    def got(self):
        return torch.stack([turned(self.G.matrix(j).as_strided(), self.opg) for j in range(self.count)])

    def check(self):
        g, ga = ref.wgrad(self.u.cuda(), self.p.cuda(), self.scale.double().cuda(), self.ids.cuda(), self.count)
        old = self.beta * self.g0.cuda() if self.beta else torch.zeros_like(g)
        tol = ref.wgrad_tolerance(self.n, g, ga + old.abs())
        err = (self.got().double() - (g + old)).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows, n, rank, count", [(1, 1, 1, 1), (16, 33, 5, 2), (264, 200, 16, 3), (130, 97, 33, 4), (300, 1100, 64, 2), (257, 70, 100, 40)])
def test_lora_wgrad_against_64_bits(kind, packed, rows, n, rank, count):
    for opg, beta in (("N", 0.0), ("T", 0.0), ("N", 1.0), ("T", -0.5)):
        Grad(kind, rows, n, rank, count, opg, beta, packed=packed).run().check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("pad, shift", [(8, 0), (3, 0), (8, 1)])
def test_lora_wgrad_leading_dimensions_and_alignment(kind, packed, pad, shift):
    for opg in "NT":
        Grad(kind, 272, 150, 20, 3, opg, 1.0, pad, shift, packed).run().check()


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("packed", [False, True])
def test_lora_wgrad_long_runs(kind, packed):
    """Runs of many pieces beside short ones, empty ones and tokens without an adapter."""
    ids = [0] * 3000 + [2] * 40 + [-1] * 500 + [3] * 1025 + [0] * 435
    Grad(kind, 520, 5000, 24, 5, "N", packed=packed, ids=ids).run().check()
    Grad(kind, 520, 5000, 24, 5, "T", 2.0, packed=packed, ids=ids).run().check()


def test_lora_wgrad_without_tokens_keeps_beta_g():
    c = Grad(BF16, 40, 0, 4, 2, "N", 0.5).run()
    assert torch.equal(c.got().cpu().double(), 0.5 * c.g0)
    c = Grad(BF16, 40, 0, 4, 2, "N").run()
    assert not c.got().any()          # beta = 0: G is not read, NaN or not


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
def test_lora_wgrad_small_projections(kind):
    """p far below f16's smallest numbers keeps its digits; an infinity stays an infinity of its own adapter."""
    c = Grad(kind, 64, 90, 6, 3, "N")
    c.p = (c.p * 2.0 ** -30)
    c.P = store(c.p, F32)
    c.run().check()
    i = int((c.ids == 1).nonzero()[0])
    c.P.as_strided()[2, i] = float("inf")
    c.run()
    got = c.got()
    assert not bool(torch.isfinite(got[1][:, 2]).any())
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isfinite(got[2]).all())
    assert bool(torch.isfinite(got[1][:, :2]).all()) and bool(torch.isfinite(got[1][:, 3:]).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
def test_lora_wgrad_of_the_checkpoint_is_that_of_the_unpacked_matrix(kind):
    c = Grad(kind, 264, 700, 16, 3, "T", packed=True).run()
    d = Grad(kind, 264, 700, 16, 3, "T")
    d.U = store(c.u, kind)
    d.run()
    assert torch.equal(c.got(), d.got())


# ------------------------------------------------------------------------------------------------------------- checkpoints
def special_values(kind, k, n):
    t = TORCH[kind]
    x = rand((k, n), kind, 3)
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    low = tiny * torch.finfo(t).eps          # smallest subnormal
    for i, v in enumerate([0.0, big, -big, low, -3 * low, tiny, 127.0, 127.5, 128.0, 126.5, -0.5, 1e-3]):
        x[i % k, i % n] = v
    if n > 8:
        x[:, 2] = 0
        x[:, 3] *= low * 40 / max(float(x[:, 3].abs().max()), 1.0)
        x[:, 4] = torch.linspace(-127.0, 127.0, k).double() * 0.5         # ties
        x[:, 5] = big
        x[0, 6] = float("inf")
        x[k - 1, 7] = float("nan")
    return x.to(t)


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("k, n, pad", [(1, 1, 0), (31, 9, 0), (32, 12, 0), (70, 13, 0), (264, 11, 8), (100, 10, 3)])
def test_pack_is_exact(kind, k, n, pad):
    x = special_values(kind, k, n)
    X = store(x, kind, pad)
    c = lowrank.Checkpoint8(k, n, kind, ld=k + pad)
    c.storage.fill_(77)
    lowrank.ckpt8_pack_dev(X, c)
    back = store(torch.zeros(k, n), kind, pad)
    lowrank.ckpt8_unpack_dev(c, back)
    q, e, v = ref.pack(x, kind)
    whole = torch.as_strided(c.storage, (k, n), (1, c.ld)).cpu().double()
    assert torch.equal(whole, q)
    assert torch.equal(torch.as_strided(c.exponents, e.shape, (1, c.lde)).cpu().long() - 127, e)
    got = back.as_strided().cpu().double()
    assert torch.equal(torch.nan_to_num(got, nan=-1.0), torch.nan_to_num(v, nan=-1.0)) and torch.equal(torch.isnan(got), torch.isnan(v))
    assert untouched(back, k, n)
    if pad:
        assert bool((torch.as_strided(c.storage, (pad, n - 1), (1, c.ld), k) == 77).all())


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
def test_pack_of_a_packed_matrix_changes_nothing(kind):
    x = rand((520, 300), kind, 9).cuda()
    X, c = store(x, kind), lowrank.Checkpoint8(520, 300, kind)
    once, twice = store(x, kind), store(x, kind)
    lowrank.ckpt8_unpack_dev(lowrank.ckpt8_pack_dev(X, c), once)
    lowrank.ckpt8_unpack_dev(lowrank.ckpt8_pack_dev(once, c), twice)
    assert torch.equal(once.as_strided(), twice.as_strided())
    step = torch.exp2(torch.ceil(torch.log2(x.abs().amax() / 127)))
    assert float((once.as_strided().double() - x).abs().max()) <= float(step) / 2


def run_wgrad(kind, m, n, k, opw, beta, pad=0, shift=0, seed=21, dy_pad=None):
    dy, x = rand((m, n), kind, seed, 0.1), rand((k, n), kind, seed + 1)
    X, c = store(x, kind), lowrank.Checkpoint8(k, n, kind, ld=max(k + pad, 1), lde=(k + 31) // 32 + pad)
    lowrank.ckpt8_pack_dev(X, c)
    back = store(torch.zeros(k, n), kind)
    lowrank.ckpt8_unpack_dev(c, back)
    kept = back.as_strided().double()
    old = rand((m, k), F32, seed + 2)
    dw = store(turned(old if beta else torch.full_like(old, float("nan")), opw), F32, pad)
    lowrank.ckpt8_wgrad_dev(opw, store(dy, kind, pad if dy_pad is None else dy_pad, shift), c, beta, dw)
    dyd = dy.cuda()
    want = dyd @ kept.t().contiguous()
    mag = dyd.abs() @ kept.abs().t().contiguous()
    before = beta * old.cuda() if beta else torch.zeros_like(want)
    tol = ref.wgrad_tolerance(n, want + before, mag + before.abs())
    err = (turned(dw.as_strided(), opw).double() - (want + before)).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert untouched(dw, *turned(old, opw).shape)


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (8, 5, 40), (130, 70, 200), (136, 64, 264), (257, 129, 77), (128, 2100, 136), (264, 0, 40)])
def test_ckpt8_wgrad_against_64_bits(kind, m, n, k):
    for opw, beta in (("N", 0.0), ("T", 1.0), ("N", -0.5), ("T", 0.0)):
        run_wgrad(kind, m, n, k, opw, beta)


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("pad, shift", [(8, 0), (3, 0), (8, 1)])
def test_ckpt8_wgrad_leading_dimensions_and_alignment(kind, pad, shift):
    for opw in "NT":
        run_wgrad(kind, 136, 100, 72, opw, 1.0, pad, shift)


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("opw", "NT")
def test_ckpt8_wgrad_large_tiles(kind, opw):
    run_wgrad(kind, 256 * 14 + 40, 130, 256 * 15 + 8, opw, 1.0)


@pytest.mark.parametrize("kind", [BF16, F16], ids=NAME.get)
@pytest.mark.parametrize("opw", "NT")
def test_ckpt8_wgrad_small_tiles(kind, opw):
    run_wgrad(kind, 2300, 264, 2200, opw, 1.0)
    run_wgrad(kind, 1100, 1300, 1130, opw, 0.0)


def test_ckpt8_wgrad_with_a_leading_dimension_of_several_gigabytes_a_tile():
    run_wgrad(BF16, 136, 72, 264, "N", 1.0, dy_pad=2 ** 25 + 8 - 136)


# -------------------------------------------------------------------------------------------------- all of them, as they are used
def backward(kind, c, dy, saved):
    """dX, dA, dB of a Case through the library; saved: X or its checkpoint."""
    flip = {"N": "T", "T": "N"}
    dY = store(dy, kind)
    dX, Q = store(torch.zeros(c.k, c.n), kind), store(torch.zeros(c.rank, c.n), F32)
    lowrank.lora_dev(flip[c.ops[0]], c.W, dY, flip[c.ops[2]], c.B, flip[c.ops[1]], c.A, c.S, c.plan, Q, dX)
    dA = lowrank.MatrixStack(c.k, c.rank, c.count, F32)
    dB = lowrank.MatrixStack(c.m, c.rank, c.count, F32)
    lowrank.lora_wgrad_dev("N", saved, Q, c.S, c.plan, 0.0, dA)
    lowrank.lora_wgrad_dev("N", dY, c.P, c.S, c.plan, 0.0, dB)
    stack = lambda s: torch.stack([s.matrix(j).as_strided() for j in range(s.count)]).double()
    return dX.as_strided().double(), stack(dA).transpose(1, 2), stack(dB), Q


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("ops", ["TTT", "NNN"])
@pytest.mark.parametrize("m, n, k, rank", [(72, 50, 96, 6), (136, 200, 264, 16)])
def test_a_training_step(kind, ops, m, n, k, rank):
    """Forward, checkpoint, backward and the dense gradient, against differentiation of the formula in 64 bits."""
    c = Case(kind, m, n, k, rank, 3, ops).run()
    dy = rand((m, n), kind, 77, 0.1)
    ck = lowrank.ckpt8_pack_dev(c.X, lowrank.Checkpoint8(k, n, kind))
    kept = store(torch.zeros(k, n), kind)
    lowrank.ckpt8_unpack_dev(ck, kept)
    for saved, x in ((c.X, c.x), (ck, kept.as_strided().cpu().double())):
        w, a, b = (t.clone().requires_grad_(True) for t in (c.w, c.a, c.b))
        xin = c.x.clone().requires_grad_(True)
        p = torch.zeros((rank, n), dtype=torch.float64)
        cols = []
        for i in range(n):
            j = int(c.ids[i])
            y = w @ xin[:, i]
            cols.append(y + c.scale[j].double() * (b[j] @ (a[j] @ xin[:, i])) if 0 <= j else y)
        (torch.stack(cols, 1) * dy).sum().backward()
        dx, da, db, Q = backward(kind, c, dy, saved)
        dy_, q = dy.cuda(), Q.as_strided().double()
        # dX: the forward formula with the factors exchanged
        want, _, mag, _ = ref.lora(c.w.t().cuda(), dy_, c.b.transpose(1, 2).cuda(), c.a.transpose(1, 2).cuda(), c.scale.double().cuda(), c.ids.cuda())
        tol = ref.lora_tolerance(kind, m, rank, want, mag, mag)[0]
        assert bool((want - xin.grad.cuda()).abs().max() <= 1e-9)
        assert bool(((dx - want).abs() <= tol).all())
        # dA, dB: the segment sums of what they were given (Q and P with their own errors, bounded in the tests above)
        ga, gam = ref.wgrad(x.cuda(), q, c.scale.double().cuda(), c.ids.cuda(), 3)
        assert bool(((da - ga.transpose(1, 2)).abs() <= ref.wgrad_tolerance(n, ga, gam).transpose(1, 2)).all())
        gb, gbm = ref.wgrad(dy_, c.P.as_strided().double(), c.scale.double().cuda(), c.ids.cuda(), 3)
        assert bool(((db - gb).abs() <= ref.wgrad_tolerance(n, gb, gbm)).all())
        if saved is c.X:   # and those sums are the derivatives: P and Q off by k (m) steps of 2^-23 of their terms
            terms = lambda t, other, rest: (k + m + n + 64) * 2.0 ** -22 * float(t.abs().max()) * max(1.0, float(other.abs().max())) * rest
            assert float((da.cpu() - a.grad).abs().max()) <= terms(c.x, dy, m * rank ** 0.5)
            assert float((db.cpu() - b.grad).abs().max()) <= terms(c.x, dy, k * rank ** 0.5)
    dw = DeviceMatrix(*((m, k) if ops[0] == "N" else (k, m)), F32)
    lowrank.ckpt8_wgrad_dev(ops[0], store(dy, kind), ck, 0.0, dw)
    kx = kept.as_strided().double()
    want = dy.cuda() @ kx.t().contiguous()
    tol = ref.wgrad_tolerance(n, want, dy.cuda().abs() @ kx.abs().t().contiguous())
    assert bool(((turned(dw.as_strided(), ops[0]).double() - want).abs() <= tol).all())


def test_gradients_against_differences():
    """Single precision: the directional derivative of <Y, R>, by central differences of the formula in 64 bits.  The loss is
    quadratic in a step along A and B together, so central differences are exact but for 64-bit rounding; what is left is the
    kernels' 32 bits over k + m + n terms."""
    c = Case(F32, 40, 30, 56, 4, 2).run()
    r = rand((40, 30), F32, 5)
    dx, da, db, _ = backward(F32, c, r, c.X)
    ea, eb, ex = rand(c.a.shape, F32, 6), rand(c.b.shape, F32, 7), rand(c.x.shape, F32, 8)
    loss = lambda h, u: float((ref.lora(c.w, c.x + h * u[2], c.a + h * u[0], c.b + h * u[1], c.scale.double(), c.ids)[0] * r).sum())
    zero = (torch.zeros_like(ea), torch.zeros_like(eb), torch.zeros_like(ex))
    for i, (grad, e) in enumerate(((da, ea), (db, eb), (dx, ex))):
        u = list(zero)
        u[i] = e
        slope = (loss(0.5, u) - loss(-0.5, u))
        got = float((grad.cpu() * e).sum())
        terms = float((grad.cpu().abs() * e.abs()).sum())
        assert abs(got - slope) <= 200 * 2.0 ** -23 * terms * 8, (i, got, slope)


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n", [1, 24, 300, 4200])
def test_captured_and_replayed(kind, n):
    """Plan, forward, checkpoint and gradients in one graph; new tokens and adapters before every replay."""
    c = Case(kind, 136, n, 264, 16, 4)
    ids = c.ids.cuda()
    ck = lowrank.Checkpoint8(264, n, kind)
    G = lowrank.MatrixStack(136, 16, 4, F32)
    dw = DeviceMatrix(264, 136, F32)
    work = [torch.empty(1 << 24, dtype=torch.uint8, device="cuda") for _ in range(3)]

    def step(plan_of):
        plan = plan_of()
        lowrank.lora_dev("T", c.W, c.X, "T", c.A, "T", c.B, c.S, plan, c.P, c.Y, work=work[0])
        lowrank.ckpt8_pack_dev(c.X, ck)
        lowrank.lora_wgrad_dev("N", c.Y, c.P, c.S, plan, 0.0, G, work=work[1])
        lowrank.ckpt8_wgrad_dev("T", c.Y, ck, 0.0, dw, work=work[2])
        return plan
    plan_of = lambda: lowrank.lora_plan(ids, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(plan_of)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(plan_of)
    outs = (c.Y.storage, c.P.storage, G.storage, dw.storage, ck.storage, ck.exponents, kept.storage)
    for turn in range(4):
        g = torch.Generator().manual_seed(100 + turn)
        ids.copy_(torch.randint(-1, 4, (n,), generator=g).to(torch.int32))
        c.X.as_strided().copy_(rand((264, n), kind, 200 + turn))
        plan = step(plan_of)
        torch.cuda.synchronize()
        want = [t.clone() for t in outs[:-1]] + [plan.storage.clone()]
        for t in outs[:4]:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w)


def test_two_streams_at_once_and_a_stream_of_ones_own():
    cases = [Case(BF16, 520, 400, 1032, 16, 3, seed=s) for s in (1, 50)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            c.run(stream=s)
    torch.cuda.synchronize()
    for c in cases:
        c.check()


@pytest.mark.parametrize("kind", KINDS, ids=NAME.get)
@pytest.mark.parametrize("n", [1, 40, 200])
def test_gradients_on_two_streams_at_once(kind, n):
    cases, streams = [Case(kind, 520, n, 264, 16, 3, seed=s) for s in (1, 50)], [torch.cuda.Stream() for _ in range(2)]
    for c in cases:
        c.run()
    ck = [lowrank.ckpt8_pack_dev(c.X, lowrank.Checkpoint8(264, n, kind)) for c in cases]
    outs = [(lowrank.MatrixStack(264, 16, 3, F32), DeviceMatrix(520, 264, F32)) for _ in cases]
    def step(i, **more):
        lowrank.lora_wgrad_dev("N", ck[i], cases[i].P, cases[i].S, cases[i].plan, 0.0, outs[i][0], **more)
        lowrank.ckpt8_wgrad_dev("N", cases[i].Y, ck[i], 0.0, outs[i][1], **more)
    want = []
    for i in range(2):
        step(i)
        want.append([o.storage.clone() for o in outs[i]])
        for o in outs[i]:
            o.storage.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            step(i, stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o.storage, w) for o, w in zip(outs[i], want[i]))


def test_an_offset_beyond_32_bits():
    """Columns of X and Y more than 2^32 bytes into their storage."""
    m, k, n, ld = 40, 72, 70000, 32768 + 8
    c = Case(BF16, m, 64, k, 4, 2)
    X = DeviceMatrix(k, n, BF16, ld=ld)
    Y = DeviceMatrix(m, n, BF16, ld=ld)
    X.as_strided().zero_()
    cols = torch.tensor([0, 1, 65535, 65536, 69998, 69999], device="cuda")
    X.as_strided()[:, cols] = c.x[:, :6].to(torch.bfloat16).cuda()
    ids = torch.full((n,), -1, dtype=torch.int32)
    ids[cols.cpu()] = torch.tensor([0, 1, 0, 1, 1, 0], dtype=torch.int32)
    plan = lowrank.lora_plan(ids.cuda(), 2)
    P = DeviceMatrix(4, n, F32)
    lowrank.lora_dev("T", c.W, X, "T", c.A, "T", c.B, c.S, plan, P, Y)
    y, p, ya, pa = ref.lora(c.w, c.x[:, :6], c.a, c.b, c.scale.double(), ids[cols.cpu()])
    ty, tp = ref.lora_tolerance(BF16, k, 4, y, ya, pa)
    assert bool(((Y.as_strided()[:, cols].cpu().double() - y).abs() <= ty).all())
    ck = lowrank.Checkpoint8(k, n, BF16, ld=2 * ld, lde=ld)
    lowrank.ckpt8_pack_dev(X, ck)
    back = DeviceMatrix(k, n, BF16, ld=ld)
    lowrank.ckpt8_unpack_dev(ck, back)
    q, e, v = ref.pack(c.x[:, :6].to(torch.bfloat16), BF16)
    assert torch.equal(back.as_strided()[:, cols].cpu().double(), v)
    G = lowrank.MatrixStack(k, 4, 2, F32)
    lowrank.lora_wgrad_dev("N", ck, P, c.S, plan, 0.0, G)
    g, ga = ref.wgrad(v, P.as_strided()[:, cols].cpu().double(), c.scale.double(), ids[cols.cpu()], 2)
    got = torch.stack([G.matrix(j).as_strided() for j in range(2)]).cpu().double()
    assert bool(((got - g).abs() <= ref.wgrad_tolerance(n, g, ga)).all())
