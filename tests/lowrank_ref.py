"""64-bit formulas of the adapter and checkpoint operators, and the error each result may have."""
import torch

from eigen_amd import _lib

TORCH = {_lib.F32: torch.float32, _lib.BF16: torch.bfloat16, _lib.F16: torch.float16}
NAME = {_lib.F32: "f32", _lib.BF16: "bf16", _lib.F16: "f16"}
KINDS = [_lib.F32, _lib.BF16, _lib.F16]
HALF = {k: torch.finfo(t).eps / 2 for k, t in TORCH.items()}          # half a step, relative to the value
SMALL = {_lib.F32: 2.0 ** -150, _lib.BF16: 2.0 ** -134, _lib.F16: 2.0 ** -25}   # half a step below the normal numbers
EXP_MIN = {_lib.F32: -126, _lib.BF16: -126, _lib.F16: -24}


def lora(w, x, a, b, scale, ids):
    """w (m, k), x (k, n), a (count, rank, k), b (count, m, rank) in 64 bits -> y, p and the sums of the terms' magnitudes."""
    y, ya = w @ x, w.abs() @ x.abs()
    p = torch.zeros((a.shape[1], x.shape[1]), dtype=torch.float64, device=x.device)
    pa = p.clone()
    for j in range(a.shape[0]):
        on = (ids == j).nonzero().flatten()
        if on.numel():
            p[:, on] = a[j] @ x[:, on]
            pa[:, on] = a[j].abs() @ x[:, on].abs()
            y[:, on] += scale[j] * (b[j] @ p[:, on])
            ya[:, on] += scale[j].abs() * (b[j].abs() @ pa[:, on])
    return y, p, ya, pa


def lora_tolerance(kind, k, rank, y, ya, pa):
    """P: k products, sums in 32 bits (a step of 2^-23 a term, whichever way the unit rounds).  Y: the same over k + rank terms
    with P's own error inside, 2^-16 for P's two 16-bit pieces (2^-17 and 2^-23 are left out), and its one rounding."""
    tp = (k + 16) * 2.0 ** -23 * pa
    pieces = 0.0 if kind == _lib.F32 else 2.0 ** -16
    ty = HALF[kind] * y.abs() + ((2 * k + rank + 32) * 2.0 ** -23 + pieces) * ya * (1 + HALF[kind]) + SMALL[kind]
    return ty, tp


def wgrad(u, p, scale, ids, count):
    """G_j = s_j u p^T over j's columns (rows, rank), and the magnitudes' sums."""
    g = torch.zeros((count, u.shape[0], p.shape[0]), dtype=torch.float64, device=u.device)
    ga = g.clone()
    for j in range(count):
        on = (ids == j).nonzero().flatten()
        if on.numel():
            g[j] = scale[j] * (u[:, on] @ p[:, on].t().contiguous())
            ga[j] = scale[j].abs() * (u[:, on].abs() @ p[:, on].abs().t().contiguous())
    return g, ga


def wgrad_tolerance(n, g, ga):
    """n products and the joins of pieces in 32 bits, each of a p whose 16-bit pieces leave at most 2^-22 of it out; the scale
    and the sum with beta G round twice more."""
    return ((n + 64) * 2.0 ** -23 + 2.0 ** -22) * ga + 2.0 ** -22 * g.abs() + 1e-37


def pack(x, kind):
    """(whole numbers, exponents, values) of x (k, n) in 64 bits; blocks that are not finite: 0, 128, NaN."""
    k, n = x.shape
    finfo = torch.finfo(TORCH[kind])
    q = torch.zeros((k, n), dtype=torch.float64)
    e = torch.zeros(((k + 31) // 32, n), dtype=torch.int64)
    v = torch.zeros((k, n), dtype=torch.float64)
    for b in range(e.shape[0]):
        part = x[32 * b:32 * b + 32].double()
        for i in range(n):
            col = part[:, i]
            if not bool(torch.isfinite(col).all()):
                e[b, i] = 128
                v[32 * b:32 * b + 32, i] = float("nan")
                continue
            top = float(col.abs().max())
            s = EXP_MIN[kind]
            while top > 127 * 2.0 ** s:
                s += 1
            w = torch.round(col / 2.0 ** s)
            if 64 * 2.0 ** s > finfo.max:
                w = w.clamp(-63, 63)
            e[b, i] = s
            q[32 * b:32 * b + 32, i] = w
            v[32 * b:32 * b + 32, i] = w * 2.0 ** s
    return q, e, v
