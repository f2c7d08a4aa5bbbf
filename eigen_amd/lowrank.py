"""Low-rank adapters of many requests beside a shared projection, and activations held in 8 bits for the backward pass, on
device-resident matrices (``eigamd_lora_*``, ``eigamd_ckpt8_*`` of ``include/eigen_amd_blas.h``).

Column-major, one token per column: a torch tensor of shape (tokens, features) is ``DeviceMatrix(features, tokens)`` on the
same storage.  Every call is asynchronous on ``stream`` (default: torch's current stream of the operands' device)."""
import contextlib
import ctypes
import functools

import torch

from . import _lib
from ._lib import lib
from .device import DeviceMatrix, _TORCH_OF_KIND

_KINDS = (_lib.F32, _lib.BF16, _lib.F16)
_BYTES = {_lib.F32: 4, _lib.BF16: 2, _lib.F16: 2}


class MatrixStack:
    """``count`` column-major rows x cols matrices of one kind in one storage (a 1-D torch tensor), ``stride`` elements apart."""

    def __init__(self, rows, cols, count, kind, ld=None, stride=None, device="cuda", storage=None, offset=0):
        self.rows, self.cols, self.count, self.kind = int(rows), int(cols), int(count), int(kind)
        self.ld = int(max(rows, 1) if ld is None else ld)
        if self.ld < max(self.rows, 1):
            raise ValueError("ld < rows")
        self.stride = int(self.ld * max(self.cols, 1) if stride is None else stride)
        self.offset = int(offset)
        if storage is None:
            storage = torch.empty(self.stride * max(self.count, 1), dtype=_TORCH_OF_KIND[self.kind], device=device)
        self.storage = storage

    @property
    def ptr(self):
        return self.storage.data_ptr() + self.offset * self.storage.element_size()

    def matrix(self, j):
        """Matrix j as a DeviceMatrix on the same storage."""
        if not 0 <= j < self.count:
            raise IndexError("matrix out of range")
        return DeviceMatrix(self.rows, self.cols, self.kind, ld=self.ld, storage=self.storage, offset=self.offset + j * self.stride)


class Checkpoint8:
    """The 8-bit form of a rows x cols matrix (features x tokens) of ``kind``: whole numbers (int8, leading dimension ``ld``)
    and one exponent byte per 32 features of a token (leading dimension ``lde``)."""

    def __init__(self, rows, cols, kind, ld=None, lde=None, device="cuda", storage=None, exponents=None):
        self.rows, self.cols, self.kind = int(rows), int(cols), int(kind)
        blocks = (self.rows + 31) // 32
        self.ld = int(max(rows, 1) if ld is None else ld)
        self.lde = int(max(blocks, 1) if lde is None else lde)
        if self.ld < max(self.rows, 1) or self.lde < max(blocks, 1):
            raise ValueError("leading dimension too small")
        if storage is None:
            storage = torch.empty(self.ld * max(self.cols, 1), dtype=torch.int8, device=device)
        if exponents is None:
            exponents = torch.empty(self.lde * max(self.cols, 1), dtype=torch.uint8, device=storage.device)
        if storage.dtype != torch.int8 or exponents.dtype != torch.uint8:
            raise ValueError("storage must be int8 and exponents uint8")
        if not storage.is_contiguous() or not exponents.is_contiguous():
            raise ValueError("storage and exponents must be contiguous")
        if self.rows and self.cols and (self.ld * (self.cols - 1) + self.rows > storage.numel()
                                        or self.lde * (self.cols - 1) + blocks > exponents.numel()):
            raise ValueError("storage or exponents are too small for the matrix")
        self.storage, self.exponents = storage, exponents

    @property
    def ptr(self):
        return self.storage.data_ptr()


class LoraPlan:
    """What ``lora_plan`` makes of a batch; belongs to its number of tokens and adapters."""

    def __init__(self, n, n_adapters, storage):
        self.n, self.n_adapters, self.storage = n, n_adapters, storage


def _check_matrix(m, kind, rows, cols, what, count=1):
    """Checks m (of a stack: its last matrix too) and returns its address.  Every operand of every call passes here, and a call's
    host time is what a single token waits for, so it is written out."""
    storage, offset = m.storage, m.offset
    if m.kind != kind:
        raise ValueError(f"{what} has the wrong scalar kind")
    if m.rows != rows or m.cols != cols:
        raise ValueError(f"{what} is {m.rows} x {m.cols}, expected {rows} x {cols}")
    if storage.dtype is not _TORCH_OF_KIND[kind] or not storage.is_contiguous():
        raise ValueError(f"{what}: the storage must be a contiguous tensor of the matrix's type")
    if rows and cols:
        last = offset + m.ld * (cols - 1) + rows
        if count > 1:
            last += (count - 1) * m.stride
        if offset < 0 or last > storage.numel():
            raise ValueError(f"{what}: the storage is too small for the matrix")
    return storage.data_ptr() + offset * _BYTES[kind] if offset else storage.data_ptr()


def _check_stack(m, kind, rows, cols, count, what):
    if m.count != count:
        raise ValueError(f"{what} has {m.count} matrices, expected {count}")
    return _check_matrix(m, kind, rows, cols, what, count) if count else 0


def _check_vector(v, n, dtype, what):
    if v.dtype is not dtype or v.numel() != n or not v.is_contiguous():
        raise ValueError(f"{what} must be {n} contiguous elements of {dtype}")
    return v.data_ptr()


_OPS = {"N": _lib.OP_N, "T": _lib.OP_T, "n": _lib.OP_N, "t": _lib.OP_T}


def _op(op):
    code = _OPS.get(op)
    if code is None:
        raise ValueError("op must be 'N' or 'T'")
    return code


def _turned(op, rows, cols):
    return (cols, rows) if op == _lib.OP_T else (rows, cols)


def _here(stream, *tensors):
    """The current stream's handle if this call can go straight there: no stream asked for, and the operands on the current
    device.  Otherwise None; the call is then made again inside ``_there``."""
    device = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != device:
            raise ValueError("operands lie on different devices")
    if device < 0:
        raise ValueError("operands must be in device memory")
    return torch._C._cuda_getCurrentRawStream(device) if stream is None and torch.cuda.current_device() == device else None


@contextlib.contextmanager
def _there(stream, tensor):
    """tensor's device and the stream (there, by default its current one) as the current ones: scratch memory is then allocated,
    and used again, in that stream's order."""
    device = tensor.device
    with torch.cuda.device(device):
        s = torch.cuda.current_stream(device) if stream is None else stream
        if s.device != device:
            raise ValueError("the stream belongs to another device than the operands")
        with torch.cuda.stream(s):
            yield


def _scratch(work, need, like):
    """(address, bytes) of the scratch memory, and the tensor that holds it."""
    if need < 0:
        raise ValueError("extent out of range")
    if not need:
        return 0, 0, None
    if work is None:
        work = torch.empty(need, dtype=torch.uint8, device=like.device)
    elif work.get_device() != like.get_device() or not work.is_contiguous() or work.numel() * work.element_size() < need:
        raise ValueError(f"work needs {need} contiguous bytes on the operands' device")
    return work.data_ptr(), need, work


# The queries depend on sizes and alignment alone (the pointers' last four bits stand for them), so a program's few answers are kept.
_lora_need = functools.lru_cache(maxsize=4096)(lib.eigamd_lora_work_bytes)
_lora_wgrad_need = functools.lru_cache(maxsize=4096)(lib.eigamd_lora_wgrad_work_bytes)
_ckpt8_wgrad_need = functools.lru_cache(maxsize=4096)(lib.eigamd_ckpt8_wgrad_work_bytes)


def lora_plan(adapter_of, n_adapters, stream=None):
    """Plan of a batch: ``adapter_of`` (int32, one per token; anything outside [0, n_adapters) means no adapter).  Made once per
    batch, used by every projection, forward and backward."""
    n, n_adapters = adapter_of.numel(), int(n_adapters)
    ids = _check_vector(adapter_of, n, torch.int32, "adapter_of")
    ints = lib.eigamd_lora_plan_ints(n, n_adapters)
    if ints < 0:
        raise ValueError("number of tokens or adapters out of range")
    s = _here(stream, adapter_of)
    if s is None:
        with _there(stream, adapter_of):
            return lora_plan(adapter_of, n_adapters)
    plan = torch.empty(ints, dtype=torch.int32, device=adapter_of.device)
    _lib.check(lib.eigamd_lora_plan_dev(n, n_adapters, ids, plan.data_ptr(), s), "eigamd_lora_plan_dev")
    return LoraPlan(n, n_adapters, plan)


def lora_work_bytes(opw, w, x):
    """Bytes of ``work`` that ``lora_dev`` needs for these operands."""
    o = _op(opw)
    return lib.eigamd_lora_work_bytes(w.kind, o, _turned(o, w.rows, w.cols)[0], x.cols, x.rows, w.ptr, w.ld, x.ptr, x.ld)


def lora_dev(opw, w, x, opa, a, opb, b, scale, plan, p, y, work=None, stream=None):
    """p <- op(a_j) x, y <- op(w) x + scale_j op(b_j) p column by column, j the adapter of the column's token.

    w, x, y: DeviceMatrix of one kind (F32, BF16, F16); a, b: MatrixStack of the same kind, one factor per adapter; scale:
    float32 per adapter; plan: from ``lora_plan``; p: F32 DeviceMatrix (rank x tokens), kept for the backward pass.  dX is
    this call with every op flipped, the roles of a and b exchanged and dY as x.  ``work``: scratch memory of
    ``lora_work_bytes`` bytes (default: from torch's allocator)."""
    ow, oa, ob = _op(opw), _op(opa), _op(opb)
    kind = w.kind
    if kind not in _KINDS:
        raise ValueError("the kind must be F32, BF16 or F16")
    m, k = (w.cols, w.rows) if ow else (w.rows, w.cols)
    n, rank, count = plan.n, p.rows, plan.n_adapters
    at_w = _check_matrix(w, kind, w.rows, w.cols, "w")
    at_x = _check_matrix(x, kind, k, n, "x")
    at_y = _check_matrix(y, kind, m, n, "y")
    at_p = _check_matrix(p, _lib.F32, rank, n, "p")
    at_a = _check_stack(a, kind, *_turned(oa, rank, k), count, "a")
    at_b = _check_stack(b, kind, *_turned(ob, m, rank), count, "b")
    at_s = _check_vector(scale, count, torch.float32, "scale")
    s = _here(stream, x.storage, w.storage, a.storage, b.storage, scale, plan.storage, p.storage, y.storage)
    if s is None:
        with _there(stream, x.storage):
            return lora_dev(opw, w, x, opa, a, opb, b, scale, plan, p, y, work)
    at, have, work = _scratch(work, _lora_need(kind, ow, m, n, k, at_w & 15, w.ld, at_x & 15, x.ld), x.storage)
    rc = lib.eigamd_lora_dev(kind, ow, oa, ob, m, n, k, rank, count, at_w, w.ld, at_x, x.ld, at_a, a.ld, a.stride, at_b, b.ld, b.stride, at_s,
                             plan.storage.data_ptr(), at_p, p.ld, at_y, y.ld, at, have, s)
    if rc:
        _lib.check(rc, "eigamd_lora_dev")
    return y


def lora_wgrad_dev(opg, u, p, scale, plan, beta, g, work=None, stream=None):
    """g_j <- beta g_j + scale_j sum over j's tokens of u_i p_i^T (rows x rank; stored transposed with opg 'T').

    u: DeviceMatrix (rows x tokens) or its Checkpoint8; p: F32 DeviceMatrix (rank x tokens); g: F32 MatrixStack, one matrix per
    adapter.  The gradient of b from u = dY and the forward pass's p; of a^T from u = x and the p of the call that made dX."""
    og = _op(opg)
    kind = u.kind
    if kind not in _KINDS:
        raise ValueError("the kind must be F32, BF16 or F16")
    rows, n, rank, count = u.rows, plan.n, p.rows, plan.n_adapters
    if u.cols != n:
        raise ValueError("u and the plan have different numbers of tokens")
    tensors, exps, lde = (u.storage, p.storage, scale, plan.storage, g.storage), 0, 0
    if isinstance(u, Checkpoint8):
        tensors, at_u, exps, lde = tensors + (u.exponents,), u.ptr, u.exponents.data_ptr(), u.lde
    else:
        at_u = _check_matrix(u, kind, rows, n, "u")
    at_p = _check_matrix(p, _lib.F32, rank, n, "p")
    at_g = _check_stack(g, _lib.F32, *_turned(og, rows, rank), count, "g")
    at_s = _check_vector(scale, count, torch.float32, "scale")
    s = _here(stream, *tensors)
    if s is None:
        with _there(stream, u.storage):
            return lora_wgrad_dev(opg, u, p, scale, plan, beta, g, work)
    at, have, work = _scratch(work, _lora_wgrad_need(rows, n, rank, count), u.storage)
    rc = lib.eigamd_lora_wgrad_dev(kind, og, rows, n, rank, count, at_u, u.ld, exps, lde, at_p, p.ld, at_s, plan.storage.data_ptr(),
                                   ctypes.byref(ctypes.c_float(beta)), at_g, g.ld, g.stride, at, have, s)
    if rc:
        _lib.check(rc, "eigamd_lora_wgrad_dev")
    return g


def _ckpt8(entry, x, c, stream, pack):
    at_x = _check_matrix(x, c.kind, c.rows, c.cols, "x")
    s = _here(stream, x.storage, c.storage, c.exponents)
    if s is None:
        with _there(stream, x.storage):
            return _ckpt8(entry, x, c, None, pack)
    at_q, at_e = c.storage.data_ptr(), c.exponents.data_ptr()
    if pack:
        rc = lib.eigamd_ckpt8_pack_dev(x.kind, x.rows, x.cols, at_x, x.ld, at_q, c.ld, at_e, c.lde, s)
    else:
        rc = lib.eigamd_ckpt8_unpack_dev(x.kind, x.rows, x.cols, at_q, c.ld, at_e, c.lde, at_x, x.ld, s)
    if rc:
        _lib.check(rc, entry)


def ckpt8_pack_dev(x, c, stream=None):
    """The DeviceMatrix x (features x tokens) into the Checkpoint8 c of the same kind and shape."""
    _ckpt8("eigamd_ckpt8_pack_dev", x, c, stream, True)
    return c


def ckpt8_unpack_dev(c, x, stream=None):
    """The values the Checkpoint8 c stands for into the DeviceMatrix x of the same kind and shape."""
    _ckpt8("eigamd_ckpt8_unpack_dev", x, c, stream, False)
    return x


def ckpt8_wgrad_dev(opw, dy, c, beta, dw, work=None, stream=None):
    """dw <- beta dw + dy x^T (opw 'N': features out x features in) or its transpose (opw 'T'), x the matrix that the
    Checkpoint8 c stands for; dy DeviceMatrix of c's kind, dw F32 DeviceMatrix."""
    ow = _op(opw)
    kind, m, n, k = c.kind, dy.rows, c.cols, c.rows
    if kind not in _KINDS:
        raise ValueError("the kind must be F32, BF16 or F16")
    at_dy = _check_matrix(dy, kind, m, n, "dy")
    at_dw = _check_matrix(dw, _lib.F32, *_turned(ow, m, k), "dw")
    s = _here(stream, dy.storage, c.storage, c.exponents, dw.storage)
    if s is None:
        with _there(stream, dy.storage):
            return ckpt8_wgrad_dev(opw, dy, c, beta, dw, work)
    at, have, work = _scratch(work, _ckpt8_wgrad_need(kind, m, n, k, at_dy & 15, dy.ld), dy.storage)
    rc = lib.eigamd_ckpt8_wgrad_dev(kind, ow, m, n, k, at_dy, dy.ld, c.storage.data_ptr(), c.ld, c.exponents.data_ptr(), c.lde,
                                    ctypes.byref(ctypes.c_float(beta)), at_dw, dw.ld, at, have, s)
    if rc:
        _lib.check(rc, "eigamd_ckpt8_wgrad_dev")
    return dw
