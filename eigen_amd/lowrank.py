"""Low-rank adapters of many requests beside a shared projection, and activations held in 8 bits for the backward pass, on
device-resident matrices (``eigamd_lora_*``, ``eigamd_ckpt8_*`` of ``include/eigen_amd_blas.h``).

Column-major, one token per column: a torch tensor of shape (tokens, features) is ``DeviceMatrix(features, tokens)`` on the
same storage.  Every call is asynchronous on ``stream`` (default: torch's current stream of the operands' device)."""
import ctypes

import torch

from . import _lib
from ._lib import lib
from .device import DeviceMatrix, _TORCH_OF_KIND

_KINDS = (_lib.F32, _lib.BF16, _lib.F16)


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
        _holds(storage, 0, self.ld, self.rows, self.cols, "storage")
        _holds(exponents, 0, self.lde, blocks, self.cols, "exponents")
        self.storage, self.exponents = storage, exponents

    @property
    def ptr(self):
        return self.storage.data_ptr()


class LoraPlan:
    """What ``lora_plan`` makes of a batch; belongs to its number of tokens and adapters."""

    def __init__(self, n, n_adapters, storage):
        self.n, self.n_adapters, self.storage = n, n_adapters, storage


def _holds(storage, offset, ld, rows, cols, what):
    if rows and cols and (offset < 0 or offset + ld * (cols - 1) + rows > storage.numel()):
        raise ValueError(f"{what}: the storage is too small for the matrix")


def _check_matrix(m, kind, rows, cols, what, count=1):
    if m.kind != kind:
        raise ValueError(f"{what} has the wrong scalar kind")
    if m.rows != rows or m.cols != cols:
        raise ValueError(f"{what} is {m.rows} x {m.cols}, expected {rows} x {cols}")
    storage = m.storage
    if storage.dtype is not _TORCH_OF_KIND[kind] or not storage.is_contiguous():
        raise ValueError(f"{what}: the storage must be a contiguous tensor of the matrix's type")
    _holds(storage, m.offset + (count - 1) * m.stride if count > 1 else m.offset, m.ld, rows, cols, what)


def _check_stack(m, kind, rows, cols, count, what):
    if m.count != count:
        raise ValueError(f"{what} has {m.count} matrices, expected {count}")
    if count:
        _check_matrix(m, kind, rows, cols, what, count)


def _check_vector(v, n, dtype, what):
    if v.dtype is not dtype or v.numel() != n or not v.is_contiguous():
        raise ValueError(f"{what} must be {n} contiguous elements of {dtype}")


_OPS = {"N": _lib.OP_N, "T": _lib.OP_T, "n": _lib.OP_N, "t": _lib.OP_T}


def _op(op):
    code = _OPS.get(op)
    if code is None:
        raise ValueError("op must be 'N' or 'T'")
    return code


def _turned(op, rows, cols):
    return (cols, rows) if op == _lib.OP_T else (rows, cols)


def _run(entry, stream, tensors, need, work, call):
    """call(stream handle, address of the scratch memory, its bytes) with the operands' device as the current one; the scratch
    memory is `work`, or allocated (and later used again) in the stream's own order."""
    device = tensors[0].get_device()
    if device < 0:
        raise ValueError("operands must be in device memory")
    for t in tensors:
        if t.get_device() != device:
            raise ValueError("operands lie on different devices")
    if need < 0:
        raise ValueError("extent out of range")
    if work is not None and (work.get_device() != device or not work.is_contiguous() or work.numel() * work.element_size() < need):
        raise ValueError(f"work needs {need} contiguous bytes on the operands' device")
    if stream is None and torch.cuda.current_device() == device:
        if work is None and need:
            work = torch.empty(need, dtype=torch.uint8, device=tensors[0].device)
        rc = call(torch._C._cuda_getCurrentRawStream(device), work.data_ptr() if need else 0, need)
    else:
        with torch.cuda.device(device):
            s = torch.cuda.current_stream(device) if stream is None else stream
            if s.device.index != device:
                raise ValueError("the stream belongs to another device than the operands")
            with torch.cuda.stream(s):
                if work is None and need:
                    work = torch.empty(need, dtype=torch.uint8, device=tensors[0].device)
                rc = call(s.cuda_stream, work.data_ptr() if need else 0, need)
    if rc != _lib.OK:
        _lib.check(rc, entry)


def lora_plan(adapter_of, n_adapters, stream=None):
    """Plan of a batch: ``adapter_of`` (int32, one per token; anything outside [0, n_adapters) means no adapter).  Made once per
    batch, used by every projection, forward and backward."""
    n, n_adapters = adapter_of.numel(), int(n_adapters)
    _check_vector(adapter_of, n, torch.int32, "adapter_of")
    ints = lib.eigamd_lora_plan_ints(n, n_adapters)
    if ints < 0:
        raise ValueError("number of tokens or adapters out of range")
    plan = []

    def call(s, work, have):
        plan.append(torch.empty(ints, dtype=torch.int32, device=adapter_of.device))
        return lib.eigamd_lora_plan_dev(n, n_adapters, adapter_of.data_ptr(), plan[0].data_ptr(), s)
    _run("eigamd_lora_plan_dev", stream, (adapter_of,), 0, None, call)
    return LoraPlan(n, n_adapters, plan[0])


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
    m, k = _turned(ow, w.rows, w.cols)
    n, rank = plan.n, p.rows
    _check_matrix(w, kind, w.rows, w.cols, "w")
    _check_matrix(x, kind, k, n, "x")
    _check_matrix(y, kind, m, n, "y")
    _check_matrix(p, _lib.F32, rank, n, "p")
    _check_stack(a, kind, *_turned(oa, rank, k), plan.n_adapters, "a")
    _check_stack(b, kind, *_turned(ob, m, rank), plan.n_adapters, "b")
    _check_vector(scale, plan.n_adapters, torch.float32, "scale")
    count = plan.n_adapters
    _run("eigamd_lora_dev", stream, (x.storage, w.storage, a.storage, b.storage, scale, plan.storage, p.storage, y.storage),
         lib.eigamd_lora_work_bytes(kind, ow, m, n, k, w.ptr, w.ld, x.ptr, x.ld), work,
         lambda s, at, have: lib.eigamd_lora_dev(kind, ow, oa, ob, m, n, k, rank, count, w.ptr, w.ld, x.ptr, x.ld, a.ptr, a.ld, a.stride,
                                                 b.ptr, b.ld, b.stride, scale.data_ptr(), plan.storage.data_ptr(), p.ptr, p.ld, y.ptr, y.ld,
                                                 at, have, s))
    return y


def lora_wgrad_dev(opg, u, p, scale, plan, beta, g, work=None, stream=None):
    """g_j <- beta g_j + scale_j sum over j's tokens of u_i p_i^T (rows x rank; stored transposed with opg 'T').

    u: DeviceMatrix (rows x tokens) or its Checkpoint8; p: F32 DeviceMatrix (rank x tokens); g: F32 MatrixStack, one matrix per
    adapter.  The gradient of b from u = dY and the forward pass's p; of a^T from u = x and the p of the call that made dX."""
    og = _op(opg)
    if u.kind not in _KINDS:
        raise ValueError("the kind must be F32, BF16 or F16")
    rows, n, rank = u.rows, plan.n, p.rows
    packed = isinstance(u, Checkpoint8)
    if u.cols != n:
        raise ValueError("u and the plan have different numbers of tokens")
    if not packed:
        _check_matrix(u, u.kind, rows, n, "u")
    _check_matrix(p, _lib.F32, rank, n, "p")
    _check_stack(g, _lib.F32, *_turned(og, rows, rank), plan.n_adapters, "g")
    _check_vector(scale, plan.n_adapters, torch.float32, "scale")
    be, count = ctypes.c_float(beta), plan.n_adapters
    tensors = (u.storage, p.storage, scale, plan.storage, g.storage)
    exps, lde = 0, 0
    if packed:
        tensors, exps, lde = tensors + (u.exponents,), u.exponents.data_ptr(), u.lde
    _run("eigamd_lora_wgrad_dev", stream, tensors, lib.eigamd_lora_wgrad_work_bytes(rows, n, rank, count), work,
         lambda s, at, have: lib.eigamd_lora_wgrad_dev(u.kind, og, rows, n, rank, count, u.ptr, u.ld, exps, lde, p.ptr, p.ld,
                                                       scale.data_ptr(), plan.storage.data_ptr(), ctypes.byref(be), g.ptr, g.ld, g.stride,
                                                       at, have, s))
    return g


def ckpt8_pack_dev(x, c, stream=None):
    """The DeviceMatrix x (features x tokens) into the Checkpoint8 c of the same kind and shape."""
    _check_matrix(x, c.kind, c.rows, c.cols, "x")
    _run("eigamd_ckpt8_pack_dev", stream, (x.storage, c.storage, c.exponents), 0, None,
         lambda s, at, have: lib.eigamd_ckpt8_pack_dev(x.kind, x.rows, x.cols, x.ptr, x.ld, c.ptr, c.ld, c.exponents.data_ptr(), c.lde, s))
    return c


def ckpt8_unpack_dev(c, x, stream=None):
    """The values the Checkpoint8 c stands for into the DeviceMatrix x of the same kind and shape."""
    _check_matrix(x, c.kind, c.rows, c.cols, "x")
    _run("eigamd_ckpt8_unpack_dev", stream, (x.storage, c.storage, c.exponents), 0, None,
         lambda s, at, have: lib.eigamd_ckpt8_unpack_dev(x.kind, x.rows, x.cols, c.ptr, c.ld, c.exponents.data_ptr(), c.lde, x.ptr, x.ld, s))
    return x


def ckpt8_wgrad_dev(opw, dy, c, beta, dw, work=None, stream=None):
    """dw <- beta dw + dy x^T (opw 'N': features out x features in) or its transpose (opw 'T'), x the matrix that the
    Checkpoint8 c stands for; dy DeviceMatrix of c's kind, dw F32 DeviceMatrix."""
    ow = _op(opw)
    m, n, k = dy.rows, c.cols, c.rows
    if c.kind not in _KINDS:
        raise ValueError("the kind must be F32, BF16 or F16")
    _check_matrix(dy, c.kind, m, n, "dy")
    _check_matrix(dw, _lib.F32, *_turned(ow, m, k), "dw")
    be = ctypes.c_float(beta)
    _run("eigamd_ckpt8_wgrad_dev", stream, (dy.storage, c.storage, c.exponents, dw.storage), lib.eigamd_ckpt8_wgrad_work_bytes(c.kind, m, n, k, dy.ptr, dy.ld), work,
         lambda s, at, have: lib.eigamd_ckpt8_wgrad_dev(c.kind, ow, m, n, k, dy.ptr, dy.ld, c.ptr, c.ld, c.exponents.data_ptr(), c.lde,
                                                        ctypes.byref(be), dw.ptr, dw.ld, at, have, s))
    return dw
