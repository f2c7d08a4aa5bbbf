"""More argument checks of the adapter and checkpoint entries that need no device."""
import ctypes

import pytest
import torch

from eigen_amd import _lib, device, lu
from eigen_amd.device import DeviceMatrix
from test_lowrank_cpu import LORA, NULL, P, call

lib = _lib.lib


def test_p_without_adapters_is_checked_if_it_is_there():
    for change in (dict(p=ctypes.c_void_p(P.value + 2)), dict(ldp=1)):
        assert call(lib.eigamd_lora_dev, LORA, count=0, **change) == _lib.ERR_ARG
    if lib.eigamd_device_ok() != 1:
        assert call(lib.eigamd_lora_dev, LORA, count=0, p=NULL) == _lib.ERR_NO_GPU


def test_scratch_of_the_factor_gradients_goes_by_what_runs_can_leave():
    """Only runs of more than a piece (128 tokens at least) leave sums: no more pieces than half pieces of the whole batch, however many
    adapters there are."""
    for rows, n, rank in ((8192, 2048, 64), (40, 5000, 7), (4096, 16384, 256)):
        for count in (1, 50, 4096):
            assert lib.eigamd_lora_wgrad_work_bytes(rows, n, rank, count) <= 2 * n // 128 * rows * rank * 4
    # few adapters: a place for every whole piece and one for every adapter's last
    assert lib.eigamd_lora_wgrad_work_bytes(4096, 8192, 16, 4) <= (8192 // 128 + 5) * 4096 * 16 * 4


@pytest.mark.parametrize("kind", [_lib.BF16, _lib.F16])
@pytest.mark.parametrize("call", [
    lambda h, f: device.gemm_dev("N", "N", 1.0, h(4, 4), h(4, 4), 0.0, h(4, 4)),
    lambda h, f: device.gemm_mixed_dev("N", "N", 1.0, h(4, 4), f(4, 4), 0.0, f(4, 4)),
    lambda h, f: device.trsm_dev("L", "U", "N", "N", 1.0, h(4, 4), h(4, 4)),
    lambda h, f: device.syrk_dev("U", "N", 1.0, h(4, 4), 0.0, h(4, 4)),
    lambda h, f: device.herk_dev("U", "N", 1.0, h(4, 4), 0.0, h(4, 4)),
    lambda h, f: device.syr2k_dev("U", "N", 1.0, h(4, 4), f(4, 4), 0.0, f(4, 4)),
    lambda h, f: device.symm_dev("L", "U", 1.0, h(4, 4), f(4, 4), 0.0, f(4, 4)),
    lambda h, f: device.trmm_dev("L", "U", "N", "N", 1.0, h(4, 4), f(4, 4)),
    lambda h, f: lu.trsm_llnu_dev(h(4, 4), f(4, 4)),
    lambda h, f: lu.getrs_dev("N", h(4, 4), torch.zeros(4, dtype=torch.int32), h(4, 1))],
    ids=["gemm", "gemm_mixed", "trsm", "syrk", "herk", "syr2k", "symm", "trmm", "trsm_llnu", "getrs"])
def test_the_dense_operations_refuse_16_bit_matrices(kind, call):
    """Also beside a matrix of another kind: its elements would be read as that kind's, past the end of its storage."""
    with pytest.raises(ValueError, match="16-bit"):
        call(lambda r, c: DeviceMatrix(r, c, kind, device="cpu"), lambda r, c: DeviceMatrix(r, c, _lib.F32, device="cpu"))


def test_16_bit_matrices_in_numpy():
    m = DeviceMatrix(2, 2, _lib.F16, device="cpu", storage=torch.arange(4).half())
    assert m.to_numpy().tolist() == [[0, 2], [1, 3]]
    with pytest.raises(ValueError, match="bf16"):
        DeviceMatrix(2, 2, _lib.BF16, device="cpu").to_numpy()
