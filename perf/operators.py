"""What the library's low-rank and checkpoint operators are measured on.

Column-major matrices, one token per column, as everywhere in the library; a torch tensor of shape (tokens, features) holds
exactly that storage.  The operators:

* ``lora``      Y = op(W) X + s_j op(B_j) P with P = op(A_j) X, j the adapter of the token's request (rank x k and m x rank
                factors of many adapters side by side), forward
* ``backward``  its gradients: dX, and dA_j, dB_j in 32 bits, X either as it was or from its 8-bit checkpoint
* ``ckpt8``     activations held in 8 bits with a power-of-two scale per 32 features of a token: pack and unpack
* ``wgrad``     dW += dY X^T of a dense layer, X read from its 8-bit checkpoint, dW in 32 bits
"""
import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_BLOCK = 32          # features that share a scale
# smallest exponent of a scale, and the largest binary exponent of a finite value
_EXP_MIN = {"bf16": -126, "f16": -24, "f32": -126}
_EXP_TOP = {"bf16": 127, "f16": 15, "f32": 127}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one request while answering: the call is all latency
        dict(name="lora_one_token", op="lora", dtype="bf16", n=1, m=2048, k=2048, rank=16, adapters=8, opw="T", order="mixed"),
        # a batch of requests while answering, one token each, most with an adapter of their own
        dict(name="lora_decode_48", op="lora", dtype="bf16", n=48, m=4096, k=4096, rank=16, adapters=32, opw="T", order="mixed"),
        # a few prompts of odd lengths through one projection whose weight is stored the other way round
        dict(name="lora_prompts_ragged", op="lora", dtype="f16", n=1237, m=4096, k=2048, rank=24, adapters=5, opw="N", order="runs"),
        # a full batch of prompt tokens through a wide projection
        dict(name="lora_prompts_large", op="lora", dtype="bf16", n=8192, m=8192, k=8192, rank=16, adapters=16, opw="T", order="runs"),
        # single precision, fine-tuning a small model with one adapter
        dict(name="lora_f32", op="lora", dtype="f32", n=777, m=1024, k=1536, rank=8, adapters=1, opw="T", order="runs"),
        # gradients of a small ragged batch with extents that are no multiples of anything
        dict(name="backward_odd", op="backward", dtype="f16", n=131, m=1003, k=1021, rank=7, adapters=3, opw="T", order="mixed",
             saved="x"),
        # gradients of one fine-tuning step, several adapters trained in one batch
        dict(name="backward_step", op="backward", dtype="bf16", n=8192, m=4096, k=4096, rank=16, adapters=4, opw="T",
             order="runs", saved="x"),
        # the same with the activations kept in 8 bits and a larger rank
        dict(name="backward_ckpt8", op="backward", dtype="bf16", n=4096, m=4096, k=8192, rank=64, adapters=3, opw="T",
             order="runs", saved="ckpt8"),
        # the activations of one short sequence
        dict(name="ckpt8_short", op="ckpt8", dtype="f16", n=33, k=1000),
        # the activations of one layer and one long batch
        dict(name="ckpt8_long", op="ckpt8", dtype="bf16", n=16384, k=8192),
        # weight gradient of a layer of a small model, a ragged batch
        dict(name="wgrad_ragged", op="wgrad", dtype="f16", n=1501, m=1032, k=2056, opw="N"),
        # weight gradient of a square projection over a long batch
        dict(name="wgrad_long", op="wgrad", dtype="bf16", n=16384, m=4096, k=4096, opw="T"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _extent(rng, low, high):
    """Feature counts: mostly multiples of 64, some of 8, some odd."""
    v = _spread(rng, low, high)
    step = rng.choice((64, 64, 64, 8, 1))
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(("lora", "lora", "backward", "ckpt8", "wgrad"))
    if op == "ckpt8":
        return dict(op=op, dtype=rng.choice(("bf16", "f16", "f32")), n=_spread(rng, 1, 16384), k=_extent(rng, 64, 8192))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op == "wgrad":
        return dict(op=op, dtype=dtype, n=_spread(rng, 64, 16384), m=_extent(rng, 256, 4096), k=_extent(rng, 256, 4096),
                    opw=rng.choice("NT"))
    case = dict(op=op, dtype=dtype, n=_spread(rng, 1, 8192) if op == "lora" else _spread(rng, 16, 8192),
                m=_extent(rng, 256, 8192 if op == "lora" else 4096), k=_extent(rng, 256, 8192 if op == "lora" else 4096),
                rank=rng.choice((1, 4, 8, 12, 16, 24, 32, 64, 128)), adapters=_spread(rng, 1, 48),
                opw=rng.choice("NTTT"), order=rng.choice(("runs", "runs", "mixed")))
    if op == "lora":
        if rng.random() < 0.2:
            case.update(dtype="f32", n=min(case["n"], 2048), m=min(case["m"], 2048), k=min(case["k"], 2048))
    else:
        case["saved"] = rng.choice(("x", "ckpt8"))
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _normal(shape, dtype, seed, salt, scale=1.0):
    return (torch.randn(shape, generator=_generator(seed, salt), device="cuda") * scale).to(dtype)


def _activations(n, k, dtype, seed):
    """Hidden states: unit normal, with a few features that are many times larger in every token."""
    x = torch.randn((n, k), generator=_generator(seed, 1), device="cuda")
    loud = torch.randint(0, k, (max(1, k // 512),), generator=_generator(seed, 2), device="cuda")
    x[:, loud] *= 20.0
    return x.to(dtype)


def _adapter_ids(case, seed):
    """Adapter of every token; -1 for a request that has none.  "runs": requests of uneven lengths one behind the other;
    "mixed": any order."""
    n, count = case["n"], case["adapters"]
    g = torch.Generator()
    g.manual_seed(seed * 7 + 3)
    if case["order"] == "runs":
        cuts = torch.sort(torch.randint(0, n + 1, (max(count, 2) - 1,), generator=g)).values
        ids = torch.bucketize(torch.arange(n), cuts, right=True) % count
        if count > 2:
            ids[ids == count - 1] = -1
    else:
        ids = torch.randint(-1 if n > 1 else 0, count, (n,), generator=g)
    return ids.to(torch.int32)


def _pack_plain(x, name):
    """(whole numbers in [-127, 127], exponents) of x (n, k), feature blocks of 32."""
    n, k = x.shape
    blocks = (k + _BLOCK - 1) // _BLOCK
    v = torch.zeros((n, blocks * _BLOCK), device=x.device)
    v[:, :k] = x.float()
    v = v.view(n, blocks, _BLOCK)
    frac, power = torch.frexp(v.abs().amax(dim=2))                       # amax = frac * 2^power, frac in [1/2, 1)
    e = torch.where(frac * 128 <= 127, power - 7, power - 6).clamp_(min=_EXP_MIN[name])
    e = torch.where(frac == 0, _EXP_MIN[name], e)
    q = torch.round(torch.ldexp(v, -e.unsqueeze(2)))
    top = torch.where(e > _EXP_TOP[name] - 6, 63, 127).unsqueeze(2)      # the value has to stay finite in its type
    q = torch.minimum(torch.maximum(q, -top), top)
    return q.view(n, -1)[:, :k], e


def _unpack_plain(q, e, dtype):
    wide = torch.repeat_interleave(e, _BLOCK, dim=1)[:, :q.shape[1]]
    return torch.ldexp(q.float(), wide).to(dtype)


def prepare(case, seed):
    op, dt = case["op"], _TORCH[case["dtype"]]
    n, k = case["n"], case["k"]
    s = {"case": case, "x": _activations(n, k, dt, seed)}
    if op == "ckpt8":
        if own:
            _prepare_own(s)
        return s
    m = case["m"]
    if op in ("backward", "wgrad"):
        s["dy"] = _normal((n, m), dt, seed, 3, 0.02)
    if op == "wgrad" or case.get("saved") == "ckpt8":
        q, e = _pack_plain(s["x"], case["dtype"])
        s["q"], s["e"] = q.to(torch.int8), (e + 127).to(torch.uint8)
        if op == "wgrad":
            s["w_shape"] = (k, m) if case["opw"] == "N" else (m, k)
            s["dw"] = _normal(s["w_shape"], torch.float32, seed, 4, 0.5)   # the sum over earlier micro-batches
            if own:
                _prepare_own(s)
            return s
    r, count = case["rank"], case["adapters"]
    s["w"] = _normal((m, k) if case["opw"] == "T" else (k, m), dt, seed, 5, k ** -0.5)
    s["a"] = _normal((count, r, k), dt, seed, 6, k ** -0.5)                # down-projections, features contiguous
    s["b"] = _normal((count, m, r), dt, seed, 7, 0.3 * r ** -0.5)          # up-projections, rank contiguous
    s["scale"] = torch.rand(count, generator=_generator(seed, 8), device="cuda") + 1.0
    ids = _adapter_ids(case, seed)
    s["ids"] = ids.cuda()
    s["groups"] = [(j, torch.nonzero(ids == j).flatten().cuda()) for j in range(count) if bool((ids == j).any())]
    if op == "backward":
        # what the forward pass keeps beside X: P, one short column per token
        s["p"] = _project_plain(s["x"].float(), s["a"].float(), s["groups"])
    if own:
        _prepare_own(s)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _project_plain(x, a, groups):
    p = torch.zeros((x.shape[0], a.shape[1]), dtype=x.dtype, device=x.device)
    for j, rows in groups:
        p[rows] = x[rows] @ a[j].t()
    return p


def _lora_plain(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    y = x @ (w.t() if case["opw"] == "T" else w)
    if case["n"] <= 64:
        # few tokens: every token takes copies of its factors, whatever the number of adapters
        j = s["ids"].clamp(min=0).long()
        live = (s["ids"] >= 0).unsqueeze(1)
        p = torch.where(live, (s["a"][j].float() * x.unsqueeze(1)).sum(2), 0.0)
        d = (s["b"][j].float() * p.unsqueeze(1)).sum(2) * s["scale"][j].unsqueeze(1)
        y = y + torch.where(live, d, 0.0)
    else:
        a, b = s["a"].float(), s["b"].float()
        p = _project_plain(x, a, s["groups"])
        for j, rows in s["groups"]:
            y[rows] += s["scale"][j] * (p[rows] @ b[j].t())
    return {"y": y.to(s["x"].dtype), "p": p}


def _backward_plain(s):
    case = s["case"]
    w, a, b = s["w"].float(), s["a"].float(), s["b"].float()
    dy, p = s["dy"].float(), s["p"]
    x = _unpack_plain(s["q"], s["e"].int() - 127, s["x"].dtype).float() if case["saved"] == "ckpt8" else s["x"].float()
    dx = dy @ (w if case["opw"] == "T" else w.t())
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for j, rows in s["groups"]:
        g, sj = dy[rows], s["scale"][j]
        q = g @ b[j]
        dx[rows] += sj * (q @ a[j])
        da[j] = sj * (q.t() @ x[rows])
        db[j] = sj * (g.t() @ p[rows])
    return {"dx": dx.to(s["dy"].dtype), "da": da, "db": db}


def _ckpt8_plain(s):
    q, e = _pack_plain(s["x"], s["case"]["dtype"])
    return {"x": _unpack_plain(q, e, s["x"].dtype), "e": e}


def _wgrad_plain(s):
    x = _unpack_plain(s["q"], s["e"].int() - 127, s["x"].dtype).float()
    dy = s["dy"].float()
    return {"dw": s["dw"] + (x.t() @ dy if s["case"]["opw"] == "N" else dy.t() @ x)}


# ------------------------------------------------------------------------------------------------------ the library's own
def _matrix(t, kind):
    from eigen_amd.device import DeviceMatrix
    return DeviceMatrix(t.shape[1], t.shape[0], kind, storage=t.view(-1))


def _stack(t, kind):
    from eigen_amd.lowrank import MatrixStack
    return MatrixStack(t.shape[2], t.shape[1], t.shape[0], kind, storage=t.view(-1))


def _prepare_own(s):
    import eigen_amd
    from eigen_amd import lowrank
    case = s["case"]
    kind = {"bf16": eigen_amd.BF16, "f16": eigen_amd.F16, "f32": eigen_amd.F32}[case["dtype"]]
    s["kind"] = kind
    s["X"] = _matrix(s["x"], kind)
    if case["op"] == "ckpt8":
        s["ckpt"] = lowrank.Checkpoint8(case["k"], case["n"], kind)
        s["back"] = _matrix(torch.empty_like(s["x"]), kind)
        return
    if "q" in s:
        s["ckpt"] = lowrank.Checkpoint8(case["k"], case["n"], kind, storage=s["q"].view(-1), exponents=s["e"].view(-1))
    if "dy" in s:
        s["dY"] = _matrix(s["dy"], kind)
    if case["op"] == "wgrad":
        return
    s["W"], s["A"], s["B"] = _matrix(s["w"], kind), _stack(s["a"], kind), _stack(s["b"], kind)
    # the batch's plan: made once per batch, used by every projection of every layer
    s["plan"] = lowrank.lora_plan(s["ids"], case["adapters"])
    if case["op"] == "backward":
        s["P"] = _matrix(s["p"], eigen_amd.F32)


def _run_own(s):
    import eigen_amd
    from eigen_amd import lowrank
    case, op = s["case"], s["case"]["op"]
    flip = {"N": "T", "T": "N"}
    if op == "lora":
        y = torch.empty((case["n"], case["m"]), dtype=s["x"].dtype, device="cuda")
        p = torch.empty((case["n"], case["rank"]), device="cuda")
        lowrank.lora_dev(case["opw"], s["W"], s["X"], "T", s["A"], "T", s["B"], s["scale"], s["plan"], _matrix(p, eigen_amd.F32),
                         _matrix(y, s["kind"]))
        return {"y": y, "p": p}
    if op == "backward":
        dx = torch.empty_like(s["x"])
        q = torch.empty((case["n"], case["rank"]), device="cuda")
        da = torch.empty(s["a"].shape, device="cuda")
        db = torch.empty(s["b"].shape, device="cuda")
        Q = _matrix(q, eigen_amd.F32)
        # dX is the same operator with every factor transposed and the two roles exchanged
        lowrank.lora_dev(flip[case["opw"]], s["W"], s["dY"], "N", s["B"], "N", s["A"], s["scale"], s["plan"], Q,
                         _matrix(dx, s["kind"]))
        saved = s["ckpt"] if case["saved"] == "ckpt8" else s["X"]
        lowrank.lora_wgrad_dev("N", saved, Q, s["scale"], s["plan"], 0.0, _stack(da, eigen_amd.F32))
        lowrank.lora_wgrad_dev("T", s["dY"], s["P"], s["scale"], s["plan"], 0.0, _stack(db, eigen_amd.F32))
        return {"dx": dx, "da": da, "db": db}
    if op == "ckpt8":
        lowrank.ckpt8_pack_dev(s["X"], s["ckpt"])
        lowrank.ckpt8_unpack_dev(s["ckpt"], s["back"])
        e = s["ckpt"].exponents.view(case["n"], -1)
        return {"x": s["back"].storage.view(case["n"], case["k"]), "e": e.to(torch.int32) - 127}
    dw = s["dw"].clone()
    lowrank.ckpt8_wgrad_dev(case["opw"], s["dY"], s["ckpt"], 1.0, _matrix(dw, eigen_amd.F32))
    return {"dw": dw}


def run(state):
    if own:
        return _run_own(state)
    return {"lora": _lora_plain, "backward": _backward_plain, "ckpt8": _ckpt8_plain, "wgrad": _wgrad_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op, es, n, k = case["op"], _BYTES[case["dtype"]], case["n"], case["k"]
    packed = n * k + n * ((k + _BLOCK - 1) // _BLOCK)
    if op == "ckpt8":      # pack reads X and writes the checkpoint, unpack the other way round
        return {"bytes": 2 * (n * k * es + packed), "flops": 4 * n * k}
    m = case["m"]
    if op == "wgrad":      # dW is read and written
        return {"bytes": packed + n * m * es + 8 * m * k, "flops": 2 * m * n * k}
    r = case["rank"]
    used = min(case["adapters"], n)
    factors = used * r * (m + k)
    if op == "lora":
        return {"bytes": es * (m * k + n * k + n * m + factors) + 4 * n * r, "flops": 2 * n * (m * k + r * (m + k))}
    saved = packed if case["saved"] == "ckpt8" else n * k * es
    return {"bytes": es * (m * k + n * m + n * k + factors) + saved + 4 * n * r + 4 * case["adapters"] * r * (m + k),
            "flops": 2 * n * (m * k + 2 * r * (m + k))}


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_block_values(x, name):
    """64-bit: the value every entry of x stands for after packing, and the exponents.  The exponent is the smallest whole e,
    not below the type's limit, with max|x| <= 127 2^e, found from the rounded-up logarithm and put right by comparing."""
    n, k = x.shape
    out = torch.empty((n, k), dtype=torch.float64, device=x.device)
    exps = torch.empty((n, (k + _BLOCK - 1) // _BLOCK), dtype=torch.int32, device=x.device)
    for b in range(exps.shape[1]):
        part = x[:, b * _BLOCK:(b + 1) * _BLOCK].double()
        top = part.abs().max(dim=1).values
        e = torch.ceil(torch.log2(top / 127)).clamp(min=float(_EXP_MIN[name]))
        e = torch.where(top > 127 * torch.exp2(e), e + 1, e)
        lower = torch.clamp(e - 1, min=float(_EXP_MIN[name]))
        e = torch.where(top <= 127 * torch.exp2(lower), lower, e)
        step = torch.exp2(e).unsqueeze(1)
        most = step * torch.where(e + 7 > _EXP_TOP[name] + 1, 63.0, 127.0).unsqueeze(1)
        v = torch.round(part / step) * step
        out[:, b * _BLOCK:(b + 1) * _BLOCK] = torch.clamp(v, -most, most)
        exps[:, b] = e.to(torch.int32)
    return out, exps


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "ckpt8":
        v, e = _exact_block_values(s["x"], case["dtype"])
        return {"x": v, "e": e}
    if "q" in s:
        e = torch.exp2(s["e"].double() - 127)
        col = torch.arange(case["k"], device="cuda") // _BLOCK
        kept = s["q"].double() * e[:, col]
    if op == "wgrad":
        dy = s["dy"].double()
        prod = torch.mm(dy.t().contiguous(), kept)                     # m x k
        return {"dw": s["dw"].double() + (prod if case["opw"] == "T" else prod.t())}
    w = s["w"].double()
    if case["opw"] == "N":
        w = w.t()
    w = w.contiguous()                                                 # m x k
    x, ids, sc = s["x"].double(), s["ids"], s["scale"].double()
    if op == "lora":
        y = torch.mm(x, w.t())
        p = torch.zeros((case["n"], case["rank"]), dtype=torch.float64, device="cuda")
        for j in range(case["adapters"]):
            on = (ids == j).nonzero().flatten()
            if on.numel():
                p[on] = torch.mm(x[on], s["a"][j].double().t())
                y[on] += torch.mm(p[on], s["b"][j].double().t() * sc[j])
        return {"y": y, "p": p}
    dy = s["dy"].double()
    if case["saved"] == "ckpt8":
        x = kept
    dx = torch.mm(dy, w)
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for j in range(case["adapters"]):
        on = (ids == j).nonzero().flatten()
        if on.numel():
            back = torch.mm(dy[on], s["b"][j].double()) * sc[j]
            dx[on] += torch.mm(back, s["a"][j].double())
            da[j] = torch.mm(back.t(), x[on])
            db[j] = torch.mm(dy[on].t(), s["p"][on].double()) * sc[j]
    return {"dx": dx, "da": da, "db": db}
