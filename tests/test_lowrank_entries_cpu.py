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
