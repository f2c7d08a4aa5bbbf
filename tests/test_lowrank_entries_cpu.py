"""More argument checks of the adapter and checkpoint entries that need no device."""
import ctypes


from eigen_amd import _lib
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
