"""Argument checks of the adapter and checkpoint entries, and calls with nothing to do: none of them needs a device."""
import ctypes

import numpy as np
import pytest
import torch

import eigen_amd
from eigen_amd import _lib, lowrank
from eigen_amd.device import DeviceMatrix

lib = _lib.lib
BUF = np.zeros(4096, dtype=np.float32)
P = ctypes.c_void_p(BUF.ctypes.data // 16 * 16 + 16)
Q = ctypes.c_void_p(BUF.ctypes.data // 16 * 16 + 4096)
NULL = ctypes.c_void_p(0)
ONE = np.ones(1, dtype=np.float32)
BETA = ctypes.c_void_p(ONE.ctypes.data)
# m, n, k, rank, adapters = 4, 3, 5, 2, 2 everywhere
LORA = dict(dtype=_lib.BF16, opw=0, opa=0, opb=0, m=4, n=3, k=5, rank=2, count=2, w=P, ldw=4, x=P, ldx=5, a=P, lda=2, sa=10, b=P, ldb=4, sb=8,
            scale=P, plan=P, p=P, ldp=2, y=Q, ldy=4, work=P, bytes=8192, stream=NULL)
GRAD = dict(dtype=_lib.F16, opg=0, rows=4, n=3, rank=2, count=2, u=P, ldu=4, e=NULL, lde=0, p=P, ldp=2, scale=P, plan=P, beta=BETA, g=Q, ldg=4,
            sg=8, work=NULL, bytes=0, stream=NULL)
WGRAD = dict(dtype=_lib.BF16, opw=0, m=4, n=3, k=5, dy=P, lddy=4, q=P, ldq=5, e=P, lde=1, beta=BETA, dw=Q, lddw=4, work=P, bytes=8192, stream=NULL)


def call(fn, base, **change):
    args = dict(base, **change)
    assert set(args) == set(base)
    return fn(*args.values())


@pytest.mark.parametrize("change", [
    dict(dtype=_lib.F64), dict(dtype=_lib.C32), dict(dtype=9), dict(opw=2), dict(opa=3), dict(opb=-1), dict(m=-1), dict(n=-1), dict(k=-1),
    dict(m=2 ** 21 + 1), dict(n=2 ** 24 + 1), dict(rank=0), dict(rank=257), dict(count=-1), dict(count=4097), dict(ldw=3), dict(opw=1, ldw=4),
    dict(ldx=4), dict(ldy=3), dict(lda=1), dict(opa=1, lda=4), dict(ldb=3), dict(opb=1, ldb=1), dict(ldp=1), dict(sa=-1), dict(sb=-1),
    dict(w=NULL), dict(x=NULL), dict(y=NULL), dict(a=NULL), dict(b=NULL), dict(p=NULL), dict(scale=NULL), dict(plan=NULL),
    dict(x=ctypes.c_void_p(P.value + 1)), dict(p=ctypes.c_void_p(P.value + 2)), dict(y=P), dict(work=NULL), dict(bytes=511),
    dict(work=ctypes.c_void_p(P.value + 4)), dict(dtype=_lib.F32, work=NULL)])
def test_lora_refuses(change):
    assert call(lib.eigamd_lora_dev, LORA, **change) == _lib.ERR_ARG
    assert b"eigamd_lora_dev" in lib.eigamd_last_error()


@pytest.mark.parametrize("change", [
    dict(dtype=_lib.C64), dict(opg=2), dict(rows=-1), dict(n=2 ** 24 + 1), dict(rank=0), dict(rank=300), dict(count=5000), dict(ldu=3), dict(ldp=1),
    dict(ldg=3), dict(opg=1, ldg=1), dict(sg=7), dict(u=NULL), dict(p=NULL), dict(g=NULL), dict(scale=NULL), dict(plan=NULL), dict(beta=NULL),
    dict(e=P, lde=0), dict(u=ctypes.c_void_p(P.value + 1)), dict(g=ctypes.c_void_p(Q.value + 2)), dict(n=5000, work=NULL)])
def test_lora_wgrad_refuses(change):
    assert call(lib.eigamd_lora_wgrad_dev, GRAD, **change) == _lib.ERR_ARG
    assert b"eigamd_lora_wgrad_dev" in lib.eigamd_last_error()


@pytest.mark.parametrize("change", [
    dict(dtype=_lib.F64), dict(opw=2), dict(m=-1), dict(n=-1), dict(k=2 ** 23), dict(lddy=3), dict(ldq=4), dict(lde=0), dict(lddw=3),
    dict(opw=1, lddw=4), dict(dy=NULL), dict(q=NULL), dict(e=NULL), dict(dw=NULL), dict(beta=NULL), dict(dtype=_lib.F32, work=NULL), dict(work=NULL),
    dict(dw=ctypes.c_void_p(Q.value + 1))])
def test_ckpt8_wgrad_refuses(change):
    assert call(lib.eigamd_ckpt8_wgrad_dev, WGRAD, **change) == _lib.ERR_ARG
    assert b"eigamd_ckpt8_wgrad_dev" in lib.eigamd_last_error()


@pytest.mark.parametrize("fn, order", [(lib.eigamd_ckpt8_pack_dev, "xqe"), (lib.eigamd_ckpt8_unpack_dev, "qex")])
def test_ckpt8_pack_and_unpack_refuse(fn, order):
    base = dict(x=(P, 40), q=(P, 40), e=(P, 2))

    def run(dtype=_lib.BF16, k=40, n=3, **change):
        both = dict(base, **change)
        return fn(dtype, k, n, *[v for name in order for v in both[name]], NULL)
    for change in (dict(dtype=_lib.F64), dict(k=-1), dict(n=2 ** 24 + 1), dict(x=(P, 39)), dict(q=(P, 39)), dict(e=(P, 1)), dict(x=(NULL, 40)),
                   dict(q=(NULL, 40)), dict(e=(NULL, 2)), dict(x=(ctypes.c_void_p(P.value + 1), 40))):
        assert run(**change) == _lib.ERR_ARG, change
    assert run(k=0) == _lib.OK and run(n=0) == _lib.OK


def test_plan_checks_and_sizes():
    assert lib.eigamd_lora_plan_ints(10, 3) == 25 and lib.eigamd_lora_plan_ints(0, 0) == 2
    assert lib.eigamd_lora_plan_ints(-1, 3) == -1 and lib.eigamd_lora_plan_ints(3, 4097) == -1
    assert lib.eigamd_lora_plan_dev(3, 2, NULL, P, NULL) == _lib.ERR_ARG
    assert lib.eigamd_lora_plan_dev(3, 2, P, NULL, NULL) == _lib.ERR_ARG
    assert lib.eigamd_lora_work_bytes(_lib.F64, 0, 4, 4, 4, P, 4, P, 4) == -1
    assert lib.eigamd_lora_work_bytes(_lib.BF16, 0, 0, 4, 4, P, 4, P, 4) == 0
    assert lib.eigamd_lora_wgrad_work_bytes(4, 4, 0, 1) == -1
    assert lib.eigamd_ckpt8_wgrad_work_bytes(_lib.BF16, -1, 4, 4, P, 4) == -1


def test_nothing_to_do_needs_no_device():
    assert call(lib.eigamd_lora_dev, LORA, n=0, x=NULL, y=NULL, p=NULL) == _lib.OK
    assert call(lib.eigamd_lora_dev, LORA, m=0, count=0, w=NULL, y=NULL) == _lib.OK
    assert call(lib.eigamd_lora_wgrad_dev, GRAD, rows=0) == _lib.OK
    assert call(lib.eigamd_lora_wgrad_dev, GRAD, count=0, g=NULL) == _lib.OK
    assert call(lib.eigamd_ckpt8_wgrad_dev, WGRAD, m=0, dw=NULL) == _lib.OK


@pytest.mark.skipif(lib.eigamd_device_ok() == 1, reason="a GPU is present")
def test_no_gpu_means_an_error():
    assert call(lib.eigamd_lora_dev, LORA) == _lib.ERR_NO_GPU
    assert call(lib.eigamd_lora_wgrad_dev, GRAD) == _lib.ERR_NO_GPU
    assert call(lib.eigamd_ckpt8_wgrad_dev, WGRAD) == _lib.ERR_NO_GPU
    assert lib.eigamd_ckpt8_pack_dev(_lib.F32, 4, 1, P, 4, Q, 4, Q, 1, NULL) == _lib.ERR_NO_GPU
    assert lib.eigamd_lora_plan_dev(3, 2, P, Q, NULL) == _lib.ERR_NO_GPU


def test_python_layer_refuses_what_does_not_fit():
    kind = eigen_amd.BF16
    m, n, k, r, count = 4, 3, 5, 2, 2
    mat = lambda rows, cols, kd=kind: DeviceMatrix(rows, cols, kd, device="cpu")
    st = lambda rows, cols, c=count, kd=kind: lowrank.MatrixStack(rows, cols, c, kd, device="cpu")
    plan = lowrank.LoraPlan(n, count, torch.zeros(2 * n + count + 2, dtype=torch.int32))
    scale = torch.ones(count)
    good = dict(opw="N", w=mat(m, k), x=mat(k, n), opa="N", a=st(r, k), opb="N", b=st(m, r), scale=scale, plan=plan, p=mat(r, n, eigen_amd.F32),
                y=mat(m, n))
    for change in (dict(opw="C"), dict(x=mat(k, n + 1)), dict(x=mat(k, n, eigen_amd.F16)), dict(y=mat(m + 1, n)), dict(a=st(r, k, 3)),
                   dict(b=st(m, r + 1)), dict(scale=torch.ones(3)), dict(scale=torch.ones(2, dtype=torch.float64)), dict(p=mat(r, n)),
                   dict(w=mat(m, k, eigen_amd.F64)), dict(a=lowrank.MatrixStack(r, k, count, kind, storage=torch.zeros(19, dtype=torch.bfloat16))),
                   dict()):   # the last one only lacks device memory
        with pytest.raises(ValueError):
            lowrank.lora_dev(**dict(good, **change))
    with pytest.raises(ValueError):
        lowrank.lora_plan(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(ValueError):
        lowrank.lora_plan(torch.zeros(3, dtype=torch.int32), 5000)
    with pytest.raises(ValueError):
        lowrank.Checkpoint8(40, 2, kind, lde=1, device="cpu")
    with pytest.raises(ValueError):
        lowrank.Checkpoint8(40, 2, kind, storage=torch.zeros(79, dtype=torch.int8))
    with pytest.raises(IndexError):
        st(r, k).matrix(2)


def test_leading_dimensions_and_strides_out_of_range():
    big = 2 ** 38 + 8
    for change in (dict(ldw=big), dict(ldx=big), dict(ldy=big), dict(lda=big), dict(ldb=big), dict(ldp=big), dict(sa=2 ** 49), dict(sb=2 ** 49)):
        assert call(lib.eigamd_lora_dev, LORA, **change) == _lib.ERR_ARG, change
    for change in (dict(ldu=big), dict(ldp=big), dict(ldg=big, sg=2 ** 41), dict(sg=2 ** 49), dict(e=P, lde=big)):
        assert call(lib.eigamd_lora_wgrad_dev, GRAD, **change) == _lib.ERR_ARG, change
    for change in (dict(lddy=big), dict(ldq=big), dict(lde=big), dict(lddw=big)):
        assert call(lib.eigamd_ckpt8_wgrad_dev, WGRAD, **change) == _lib.ERR_ARG, change


def test_a_checkpoint_of_strided_storage_is_refused():
    kind = _lib.BF16
    with pytest.raises(ValueError):
        lowrank.Checkpoint8(40, 2, kind, storage=torch.zeros(160, dtype=torch.int8)[::2])
    with pytest.raises(ValueError):
        lowrank.Checkpoint8(40, 2, kind, storage=torch.zeros(80, dtype=torch.int8), exponents=torch.zeros(8, dtype=torch.uint8)[::2])
