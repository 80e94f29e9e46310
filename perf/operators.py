"""Workloads of the frozen-teacher operators: 4-bit quantisation and products, top logits, distillation.

Every case exists in two forms: `run` with `own` false computes it with elementary torch operations in 32 bits, with
`own` true it makes the framework's own calls.  `exact` computes the same results in 64 bits from the definitions."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK, GROUP = 32, 256  # elements that share a scale; elements of a row that are stored together (128 bytes of codes)
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BIGGEST = 1 << 28  # logits of the largest case


def listed():
    return [
        # a ragged batch of pooled features on its way into a 4-bit layer (the format's error is what a user looks at)
        {"name": "quantize batch", "op": "quantize", "rows": 777, "cols": 1001, "dtype": "bf16"},
        # the widest fuser weight (18432 x 18432), once per checkpoint
        {"name": "quantize weight", "op": "quantize", "rows": 18432, "cols": 18432, "dtype": "fp32"},
        # a small head with odd sizes inside a training step
        {"name": "linear odd train", "op": "linear", "rows": 37, "k": 1001, "n": 1537, "dtype": "fp32", "bias": True, "train": True},
        # one region's features through the widest layer: latency of a single row
        {"name": "linear one row", "op": "linear", "rows": 1, "k": 18432, "n": 18432, "dtype": "bf16", "bias": True, "train": False},
        # the widest fuser layer at one view's 256 rows, with the gradient of its input
        {"name": "linear fuser train", "op": "linear", "rows": 256, "k": 18432, "n": 18432, "dtype": "bf16", "bias": False, "train": True},
        # a whole slide's regions through the second widest layer, with the gradient of its input
        {"name": "linear slide train", "op": "linear", "rows": 8192, "k": 9216, "n": 9216, "dtype": "fp16", "bias": True, "train": True},
        # a few embeddings against a wide set of prototypes
        {"name": "top few rows", "op": "top", "shape": "rows", "rows": 4, "classes": 65536, "hw": 1, "k": 16, "dtype": "fp32", "t": 1.0},
        # a teacher's batch against the same prototypes
        {"name": "top prototypes", "op": "top", "shape": "rows", "rows": 4096, "classes": 65536, "hw": 1, "k": 32, "dtype": "bf16", "t": 0.5},
        # a segmentation teacher's logit maps of 256 x 256
        {"name": "top maps", "op": "top", "shape": "maps", "rows": 16, "classes": 21, "hw": 65536, "k": 4, "dtype": "bf16", "t": 2.0},
        # a small batch of tile classes
        {"name": "distill tiles", "op": "distill", "shape": "rows", "rows": 64, "classes": 1000, "hw": 1, "k": 10, "dtype": "fp32", "t": 2.0, "rest": False, "mask": False},
        # the student's batch against the prototypes
        {"name": "distill prototypes", "op": "distill", "shape": "rows", "rows": 4096, "classes": 65536, "hw": 1, "k": 32, "dtype": "bf16", "t": 0.5, "rest": True, "mask": False},
        # a segmentation student's maps, unlabelled pixels masked
        {"name": "distill maps", "op": "distill", "shape": "maps", "rows": 32, "classes": 21, "hw": 65536, "k": 4, "dtype": "fp32", "t": 2.0, "rest": True, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "top", "distill"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "quantize":
        while True:
            rows, cols = _log(rng, 1, 18432), _log(rng, 32, 18432)
            if rows * cols <= 1 << 27:
                return {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op == "linear":
        while True:
            rows, k, n = _log(rng, 1, 16384), _log(rng, 64, 18432), _log(rng, 64, 18432)
            if rows * k * n <= 8192 * 9216 * 4608:
                break
        if rng.random() < 0.5:  # widths as heads have them
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        return {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.5, "train": rng.random() < 0.5}
    maps = rng.random() < 0.4
    while True:
        if maps:
            rows, classes, hw = _log(rng, 1, 64), _log(rng, 2, 64), _log(rng, 16, 256) * _log(rng, 16, 256)
        else:
            rows, classes, hw = _log(rng, 1, 8192), _log(rng, 2, 131072), 1
        if rows * classes * hw <= BIGGEST // 4:
            break
    k = min(classes, _log(rng, 1, 16 if maps else 64))
    case = {"op": op, "shape": "maps" if maps else "rows", "rows": rows, "classes": classes, "hw": hw, "k": k, "dtype": dtype,
            "t": rng.choice([0.5, 1.0, 2.0, 4.0])}
    if op == "distill":
        case["rest"] = rng.random() < 0.6
        case["mask"] = rng.random() < 0.4
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "quantize":
        x = normal(case["rows"], case["cols"])
        x *= torch.exp(0.5 * normal(case["cols"]))  # features (channels) of different size
        return {"case": case, "x": x.to(dt)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        codes, scales = [], []
        step = max(1, (1 << 25) // k)
        for a in range(0, n, step):  # in slices: the temporaries stay small
            c, s = _pack(normal(min(step, n - a), k) / math.sqrt(k))
            codes.append(c)
            scales.append(s)
        s = {"case": case, "codes": torch.cat(codes, 1).contiguous(), "scales": torch.cat(scales, 1).contiguous(),
             "x": normal(m, k).to(dt), "bias": 0.1 * normal(n) if case["bias"] else None}
        if case["train"]:
            s["x"].requires_grad_()
            s["dy"] = (normal(m, n) / 16).to(dt)
        return s
    r, c, hw = case["rows"], case["classes"], case["hw"]
    shape = (r, c, hw) if case["shape"] == "maps" else (r, c)
    dim = 1 if case["shape"] == "maps" else -1
    teacher = (3.0 * normal(*shape)).to(dt)
    s = {"case": case, "dim": dim}
    if case["op"] == "top":
        s["logits"] = teacher
        return s
    s["values"], s["indices"], rest = _top(teacher, case["k"], case["t"], dim)
    s["rest"] = rest if case["rest"] else None
    z = normal(*shape)
    z += 0.5 * teacher
    s["logits"] = z.to(dt).requires_grad_()
    counted = (r, hw) if case["shape"] == "maps" else (r,)
    s["mask"] = torch.rand(counted, generator=g, device="cuda") < 0.8 if case["mask"] else None
    # the gradient that arrives: a loss scaler's factor keeps fp16 gradients of a mean over many rows above the subnormals
    s["scale"] = torch.tensor(256.0 * 2.0 ** int(math.log2(r * hw)) if case["dtype"] == "fp16" else 1.0, device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _blocks(x):
    """[rows, cols] -> fp32 [rows, groups * 8, 32], zeros behind the last column"""
    rows, cols = x.shape
    pad = -cols % GROUP
    x = x.float()
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], 1)
    return x.reshape(rows, -1, BLOCK)


def _power(e):
    """2^(e - 127) of the scale codes e (int32); 255 stands for NaN"""
    bits = torch.where(e == 0, torch.full_like(e, 1 << 22), e << 23)
    return torch.where(e == 255, torch.full_like(e, 0x7FC00000), bits).view(torch.float32)


def _codes(x):
    """the 4-bit codes (uint8, one a byte) and scale codes (int32) of _blocks(x)"""
    b = _blocks(x)
    field = b.abs().amax(-1).contiguous().view(torch.int32) >> 23
    e = torch.where(field == 255, field, (field - 2).clamp(min=0))
    up = ((254 - e.clamp(max=253)) << 23).view(torch.float32)  # 2^(127 - e)
    a = b.abs() * up.unsqueeze(-1)
    c = (a > 0.25).to(torch.uint8)
    c += a >= 0.75
    c += a > 1.25
    c += a >= 1.75
    c += a > 2.5
    c += a >= 3.5
    c += a > 5.0
    c += torch.signbit(b).to(torch.uint8) * 8
    c *= (e != 255).unsqueeze(-1)
    return c, e


def _values(c, e):
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=c.device)
    return (table[c.int()] * _power(e).unsqueeze(-1)).reshape(c.shape[0], -1)


def _pack(x):
    """codes [groups, rows, 128] (the even element in the low four bits) and scales [groups, rows, 8], both uint8"""
    c, e = _codes(x)
    rows = c.shape[0]
    two = c.reshape(rows, -1, 2)
    codes = (two[..., 0] | (two[..., 1] << 4)).reshape(rows, -1, GROUP // 2).transpose(0, 1)
    return codes.contiguous(), e.to(torch.uint8).reshape(rows, -1, GROUP // BLOCK).transpose(0, 1).contiguous()


def _unpack(codes, scales, cols):
    groups, rows, _ = codes.shape
    c = codes.transpose(0, 1).reshape(rows, -1, 1)
    c = torch.cat([c & 15, c >> 4], -1).reshape(rows, -1, BLOCK)
    e = scales.transpose(0, 1).reshape(rows, -1).int()
    return _values(c, e)[:, :cols]


def _top(x, k, t, dim):
    """the k largest along dim (ties to the lowest index), their indices, log sum exp(x / t) of the others"""
    v = x.detach().movedim(dim, -1).float()
    n = v.shape[-1]
    bits = (v + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (order << 32) + (0x7FFFFFFF - torch.arange(n, device=v.device))
    at = 0x7FFFFFFF - (torch.topk(key, k, -1).values & 0xFFFFFFFF)
    values = torch.gather(v, -1, at)
    others = (v / t).scatter(-1, at, -math.inf)
    peak = others.amax(-1, keepdim=True)
    peak = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)
    rest = torch.log(torch.exp(others - peak).sum(-1)) + peak[..., 0]
    return values.movedim(-1, dim).contiguous(), at.int().movedim(-1, dim).contiguous(), rest


def _distill(z, values, indices, rest, mask, scale, t, dim):
    """mean loss over the rows that count, and scale * its gradient"""
    v = values.movedim(dim, -1).float() / t
    at = indices.movedim(dim, -1).long()
    a = z.detach().movedim(dim, -1).float()
    r = torch.full_like(v[..., :1], -math.inf) if rest is None else rest.unsqueeze(-1)
    peak = torch.maximum(v.amax(-1, keepdim=True), r)
    total = torch.exp(v - peak).sum(-1, keepdim=True) + torch.exp(r - peak)
    lse = torch.log(total) + peak
    p, pr = torch.exp(v - lse), torch.exp(r - lse)
    a = (a - a.amax(-1, keepdim=True)) / t
    grown = torch.exp(a)
    whole = grown.sum(-1, keepdim=True)
    spare = grown.scatter(-1, at, 0.0).sum(-1, keepdim=True)
    zero = torch.zeros_like(pr)
    loss = (p * (v - lse - torch.gather(a, -1, at) + torch.log(whole))).sum(-1, keepdim=True)
    loss = loss + torch.where(pr > 0, pr * (r - lse - torch.log(spare) + torch.log(whole)), zero)
    inside = torch.where(spare > 0, pr / spare, zero)
    grad = grown * (1.0 / whole - inside)
    grad.scatter_(-1, at, torch.gather(grown, -1, at) / whole - p)
    keep = torch.ones_like(loss, dtype=torch.bool) if mask is None else mask.unsqueeze(-1)
    loss, count = torch.where(keep, loss, zero), keep.sum().clamp(min=1)
    grad = torch.where(keep, grad, zero) * (t * scale / count)
    return (loss.sum() * (t * t)) / count, grad.movedim(-1, dim).contiguous().to(z.dtype)


def _plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        return _values(*_codes(s["x"]))[:, :case["cols"]].contiguous()
    if case["op"] == "linear":
        x = s["x"].detach()
        w = _unpack(s["codes"], s["scales"], case["k"])
        y = _values(*_codes(x))[:, :case["k"]] @ w.t()
        if s["bias"] is not None:
            y += s["bias"]
        y = y.to(x.dtype)
        return (y, (s["dy"].float() @ w).to(x.dtype)) if case["train"] else y
    if case["op"] == "top":
        return _top(s["logits"], case["k"], case["t"], s["dim"])
    return _distill(s["logits"], s["values"], s["indices"], s["rest"], s["mask"], s["scale"], case["t"], s["dim"])


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _framework(s):
    from msf_wsi_amd import losses, quant

    case = s["case"]
    if case["op"] == "quantize":
        return quant.quantize_mx4(s["x"]).dequantize()
    if case["op"] == "linear":
        w = quant.MX4Tensor(s["codes"], s["scales"], case["k"])
        y = quant.mx4_linear(s["x"], w, s["bias"])
        return (y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]) if case["train"] else y
    if case["op"] == "top":
        return tuple(losses.top_logits(s["logits"], case["k"], temperature=case["t"], dim=s["dim"]))
    loss = losses.TopLogitDistillLoss(temperature=case["t"], dim=s["dim"])(
        s["logits"], losses.TopLogits(s["values"], s["indices"], s["rest"]), mask=s["mask"])
    return loss.detach(), torch.autograd.grad(loss, s["logits"], s["scale"])[0]


def run(s):
    if own:
        return _framework(s)
    return _plain(s)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size + 4), "flops": 4 * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        passes = 2 if case["train"] else 1
        return {"bytes": n * k * 17 // 32 + passes * size * m * (k + n), "flops": passes * 2 * m * n * k}
    rows = case["rows"] * case["hw"]
    logits = rows * case["classes"]
    if case["op"] == "top":
        return {"bytes": logits * size + rows * (8 * case["k"] + 4), "flops": 4 * logits}
    return {"bytes": 2 * logits * size + rows * (8 * case["k"] + 5), "flops": 10 * logits}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_values(x):
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    big = x.abs().amax(-1, keepdim=True)
    e = (torch.frexp(big).exponent.double() - 3).clamp(min=-127)  # floor(log2 big) - 2
    unit = torch.pow(torch.full_like(e, 2.0), e)
    y = (x / unit).abs()
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = (torch.round(y / step) * step).clamp(max=6.0)  # torch.round: halves to even
    return (torch.copysign(y, x) * unit).reshape(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_values(s["x"])
    if case["op"] == "linear":
        k, x = case["k"], s["x"].detach()
        byte = torch.arange(256, device="cuda")
        code = torch.stack([byte % 16, byte // 16], 1)
        level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
        pair = torch.where(code > 7, -level[code % 8], level[code % 8])  # the two values of each byte
        w = torch.cat([(pair[c.long()].reshape(c.shape[0], GROUP // BLOCK, BLOCK) * torch.exp2(e.double() - 127).unsqueeze(-1)).flatten(1)
                       for c, e in zip(s["codes"], s["scales"])], 1)[:, :k]
        y = torch.matmul(_exact_values(x), w.t().contiguous())
        if s["bias"] is not None:
            y = y + s["bias"].double()
        return (y, torch.matmul(s["dy"].double(), w)) if case["train"] else y
    dim, k, t = s["dim"], case["k"], case["t"]
    if case["op"] == "top":
        v, at = torch.sort(s["logits"].double().movedim(dim, -1), dim=-1, descending=True, stable=True)
        rest = torch.logsumexp(v[..., k:] / t, -1) if k < case["classes"] else torch.full_like(v[..., 0], -math.inf)
        return v[..., :k].movedim(-1, dim).contiguous(), at[..., :k].int().movedim(-1, dim).contiguous(), rest
    z = s["logits"].detach().double().movedim(dim, -1).reshape(-1, case["classes"]).requires_grad_()
    at = s["indices"].long().movedim(dim, -1).reshape(-1, k)
    lt = s["values"].double().movedim(dim, -1).reshape(-1, k) / t
    if s["rest"] is not None:
        lt = torch.cat([lt, s["rest"].double().reshape(-1, 1)], 1)
    lt = torch.log_softmax(lt, 1)
    keep = torch.ones(z.shape[0], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"].reshape(-1)
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    grad = torch.zeros_like(z)
    for part in torch.arange(z.shape[0], device="cuda").split(max(1, (1 << 27) // case["classes"])):
        zi = z.detach()[part].requires_grad_()
        ls = torch.log_softmax(zi / t, 1)
        mine = torch.gather(ls, 1, at[part])
        if s["rest"] is not None:
            spare = torch.logsumexp(ls.scatter(1, at[part], -math.inf), 1, keepdim=True) if k < case["classes"] else torch.full_like(mine[:, :1], -math.inf)
            mine = torch.cat([mine, spare], 1)
        there = torch.exp(lt[part])
        row = torch.where(there > 0, there * (lt[part] - torch.where(there > 0, mine, torch.zeros_like(mine))), torch.zeros_like(mine)).sum(1)
        loss = t * t * row[keep[part]].sum() / keep.sum().clamp(min=1)
        if bool(keep[part].any()):
            grad[part] = torch.autograd.grad(loss, zi, s["scale"].double())[0]
        total = total + loss.detach()
    like = s["logits"].movedim(dim, -1).shape
    return total, grad.reshape(like).movedim(-1, dim).contiguous()
