"""Low-rank adapters of many requests beside a shared projection, and activations held in 8 bits for the backward pass, on
device-resident matrices (``eigamd_lora_*``, ``eigamd_ckpt8_*`` of ``include/eigen_amd_blas.h``).

Column-major, one token per column: a torch tensor of shape (tokens, features) is ``DeviceMatrix(features, tokens)`` on the
same storage.  Every call is asynchronous on ``stream`` (default: torch's current stream of the operands' device)."""
import contextlib
import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import lib
from .device import DeviceMatrix, _OPCODE, _TORCH_OF_KIND

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


def _check_matrix(m, kind, rows, cols, what):
    if m.kind != kind:
        raise ValueError(f"{what} has the wrong scalar kind")
    if (m.rows, m.cols) != (rows, cols):
        raise ValueError(f"{what} is {m.rows} x {m.cols}, expected {rows} x {cols}")
    if m.storage.dtype != _TORCH_OF_KIND[kind] or not m.storage.is_contiguous():
        raise ValueError(f"{what}: the storage must be a contiguous tensor of the matrix's type")
    _holds(m.storage, m.offset, m.ld, rows, cols, what)


def _check_stack(m, kind, rows, cols, count, what):
    if m.count != count:
        raise ValueError(f"{what} has {m.count} matrices, expected {count}")
    _check_matrix(m, kind, rows, cols, what)
    if count:
        _holds(m.storage, m.offset + (count - 1) * m.stride, m.ld, rows, cols, what)


def _check_vector(v, n, dtype, what):
    if v.dtype != dtype or v.numel() != n or not v.is_contiguous():
        raise ValueError(f"{what} must be {n} contiguous elements of {dtype}")


def _op(op):
    op = op.upper()
    if op not in ("N", "T"):
        raise ValueError("op must be 'N' or 'T'")
    return _OPCODE[op]


def _turned(op, rows, cols):
    return (cols, rows) if op == _lib.OP_T else (rows, cols)


@contextlib.contextmanager
def _on(stream, *tensors):
    """The operands' device as the current one, and the stream (torch's current one there by default) with its handle."""
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError("operands must be in device memory")
    if any(t.device != device for t in tensors):
        raise ValueError("operands lie on different devices")
    with torch.cuda.device(device):
        s = torch.cuda.current_stream(device) if stream is None else stream
        if s.device != device:
            raise ValueError("the stream belongs to another device than the operands")
        with torch.cuda.stream(s):      # scratch memory is then allocated, and reused, in this stream's order
            yield ctypes.c_void_p(s.cuda_stream)


def _scratch(work, need, device):
    if need < 0:
        raise ValueError("extent out of range")
    if work is None:
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    elif not work.is_contiguous() or work.numel() * work.element_size() < need:
        raise ValueError(f"work needs {need} contiguous bytes")
    return work, work.numel() * work.element_size()


def _p(address):
    return ctypes.c_void_p(address)


def lora_plan(adapter_of, n_adapters, stream=None):
    """Plan of a batch: ``adapter_of`` (int32, one per token; anything outside [0, n_adapters) means no adapter).  Made once per
    batch, used by every projection, forward and backward."""
    n, n_adapters = adapter_of.numel(), int(n_adapters)
    _check_vector(adapter_of, n, torch.int32, "adapter_of")
    ints = lib.eigamd_lora_plan_ints(n, n_adapters)
    if ints < 0:
        raise ValueError("number of tokens or adapters out of range")
    with _on(stream, adapter_of) as s:
        plan = torch.empty(ints, dtype=torch.int32, device=adapter_of.device)
        _lib.check(lib.eigamd_lora_plan_dev(n, n_adapters, _p(adapter_of.data_ptr()), _p(plan.data_ptr()), s), "eigamd_lora_plan_dev")
    return LoraPlan(n, n_adapters, plan)


def lora_work_bytes(opw, w, x):
    """Bytes of ``work`` that ``lora_dev`` needs for these operands."""
    o = _op(opw)
    return lib.eigamd_lora_work_bytes(w.kind, o, _turned(o, w.rows, w.cols)[0], x.cols, x.rows)


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
    with _on(stream, x.storage, w.storage, a.storage, b.storage, scale, plan.storage, p.storage, y.storage) as s:
        work, have = _scratch(work, lib.eigamd_lora_work_bytes(kind, ow, m, n, k), x.storage.device)
        rc = lib.eigamd_lora_dev(kind, ow, oa, ob, m, n, k, rank, plan.n_adapters, _p(w.ptr), w.ld, _p(x.ptr), x.ld, _p(a.ptr), a.ld,
                                 a.stride, _p(b.ptr), b.ld, b.stride, _p(scale.data_ptr()), _p(plan.storage.data_ptr()), _p(p.ptr),
                                 p.ld, _p(y.ptr), y.ld, _p(work.data_ptr()), have, s)
    _lib.check(rc, "eigamd_lora_dev")
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
    be = np.array([beta], dtype=np.float32)
    with _on(stream, u.storage, p.storage, scale, plan.storage, g.storage, *([u.exponents] if packed else [])) as s:
        work, have = _scratch(work, lib.eigamd_lora_wgrad_work_bytes(rows, n, rank, plan.n_adapters), u.storage.device)
        rc = lib.eigamd_lora_wgrad_dev(u.kind, og, rows, n, rank, plan.n_adapters, _p(u.ptr), u.ld,
                                       _p(u.exponents.data_ptr()) if packed else None, u.lde if packed else 0, _p(p.ptr), p.ld,
                                       _p(scale.data_ptr()), _p(plan.storage.data_ptr()), _p(be.ctypes.data), _p(g.ptr), g.ld, g.stride,
                                       _p(work.data_ptr()), have, s)
    _lib.check(rc, "eigamd_lora_wgrad_dev")
    return g


def ckpt8_pack_dev(x, c, stream=None):
    """The DeviceMatrix x (features x tokens) into the Checkpoint8 c of the same kind and shape."""
    _check_matrix(x, c.kind, c.rows, c.cols, "x")
    with _on(stream, x.storage, c.storage, c.exponents) as s:
        rc = lib.eigamd_ckpt8_pack_dev(x.kind, x.rows, x.cols, _p(x.ptr), x.ld, _p(c.ptr), c.ld, _p(c.exponents.data_ptr()), c.lde, s)
    _lib.check(rc, "eigamd_ckpt8_pack_dev")
    return c


def ckpt8_unpack_dev(c, x, stream=None):
    """The values the Checkpoint8 c stands for into the DeviceMatrix x of the same kind and shape."""
    _check_matrix(x, c.kind, c.rows, c.cols, "x")
    with _on(stream, x.storage, c.storage, c.exponents) as s:
        rc = lib.eigamd_ckpt8_unpack_dev(x.kind, x.rows, x.cols, _p(c.ptr), c.ld, _p(c.exponents.data_ptr()), c.lde, _p(x.ptr), x.ld, s)
    _lib.check(rc, "eigamd_ckpt8_unpack_dev")
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
    be = np.array([beta], dtype=np.float32)
    with _on(stream, dy.storage, c.storage, c.exponents, dw.storage) as s:
        work, have = _scratch(work, lib.eigamd_ckpt8_wgrad_work_bytes(c.kind, m, n, k), dy.storage.device)
        rc = lib.eigamd_ckpt8_wgrad_dev(c.kind, ow, m, n, k, _p(dy.ptr), dy.ld, _p(c.ptr), c.ld, _p(c.exponents.data_ptr()), c.lde,
                                        _p(be.ctypes.data), _p(dw.ptr), dw.ld, _p(work.data_ptr()), have, s)
    _lib.check(rc, "eigamd_ckpt8_wgrad_dev")
    return dw
