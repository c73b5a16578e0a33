"""Workloads of the microscaled operators and of the router's balance loss.

Every case can be computed two ways on the same inputs: ``run`` in plain torch
operations (``own`` false), or through the framework's entry points (``own``
true). ``exact`` gives the results in 64 bits from the operators' definitions.

Formats (``fmt``): values in blocks along a row, one scale for each block.
  nvfp4   e2m1 values, blocks of 16, e4m3 scale, one float32 scale of the tensor
  mxfp4   e2m1 values, blocks of 32, power-of-two (e8m0) scale
  mxfp8   e4m3 values, blocks of 32, power-of-two (e8m0) scale
e2m1 values are packed two a byte, the even column in the low half.
"""
import importlib
import math

import torch

own = False

DEV = "cuda"
BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    """Widths 7168 and 2048, 4096 = 2 x 2048 gate and up rows, 256 experts,
    32 of them on a card and 8 per token are the layer's own geometry."""
    return [
        # one decoded token's hidden state to 4 bits and back: latency
        {"name": "quantize-1x7168", "op": "quantize", "fmt": "nvfp4", "rows": 1, "cols": 7168, "dtype": "bf16"},
        # the hidden states of a long prompt, 4 bits and back: bandwidth
        {"name": "quantize-16384x7168", "op": "quantize", "fmt": "nvfp4", "rows": 16384, "cols": 7168, "dtype": "bf16"},
        # an odd number of the experts' intermediate rows, the other 4-bit format
        {"name": "quantize-1009x2048", "op": "quantize", "fmt": "mxfp4", "rows": 1009, "cols": 2048, "dtype": "fp16"},
        # the step between two layers of a decode batch
        {"name": "norm-64x7168", "op": "norm", "fmt": "mxfp8", "rows": 64, "cols": 7168, "dtype": "bf16", "residual": True},
        # the same for a long prompt
        {"name": "norm-16384x7168", "op": "norm", "fmt": "mxfp8", "rows": 16384, "cols": 7168, "dtype": "bf16", "residual": True},
        # gate and up projection of one expert (the shared one) for a decode batch: weight streaming
        {"name": "matmul-8x7168x4096", "op": "matmul", "fmt": "nvfp4", "m": 8, "k": 7168, "n": 4096, "dtype": "bf16"},
        # the same for a long prompt: tensor cores
        {"name": "matmul-8192x7168x4096", "op": "matmul", "fmt": "nvfp4", "m": 8192, "k": 7168, "n": 4096, "dtype": "bf16"},
        # down projection, 8-bit values, a ragged number of tokens
        {"name": "matmul-1000x2048x7168", "op": "matmul", "fmt": "mxfp8", "m": 1000, "k": 2048, "n": 7168, "dtype": "bf16"},
        # gate and up products of 32 experts for 64 decoded tokens (64 x 8 x 32 / 256 rows)
        {"name": "experts-64x7168x4096", "op": "experts", "fmt": "nvfp4", "experts": 32, "m": 64, "k": 7168, "n": 4096,
         "hot": 0.0, "dtype": "bf16"},
        # down products of 32 experts for a prompt, 40% of the rows at 4 hot experts
        {"name": "experts-8192x2048x7168", "op": "experts", "fmt": "mxfp4", "experts": 32, "m": 8192, "k": 2048, "n": 7168,
         "hot": 0.4, "dtype": "bf16"},
        # a training step's balance loss over packed sequences, forward and backward
        {"name": "balance-16384x256", "op": "balance", "tokens": 16384, "experts": 256, "topk": 8, "seqs": 13,
         "score": "sigmoid", "dtype": "fp32"},
        # the softmax form on bf16 logits, a short batch
        {"name": "balance-200x256", "op": "balance", "tokens": 200, "experts": 256, "topk": 8, "seqs": 3,
         "score": "softmax", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "norm", "matmul", "experts", "balance"))
    if op in ("quantize", "norm"):
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        case = {"op": op, "rows": _log(rng, 1, 8192 if dtype == "fp32" else 16384), "cols": 32 * _log(rng, 1, 224), "dtype": dtype}
        if op == "norm":
            return dict(case, fmt="mxfp8", residual=rng.random() < 0.7)
        return dict(case, fmt=rng.choice(("nvfp4", "mxfp4")))
    if op == "matmul":
        return {"op": op, "fmt": rng.choice(("nvfp4", "mxfp4", "mxfp8")), "m": _log(rng, 1, 8192), "k": 32 * _log(rng, 4, 224),
                "n": _log(rng, 64, 4096), "dtype": rng.choice(("bf16", "fp16"))}
    if op == "experts":
        return {"op": op, "fmt": rng.choice(("nvfp4", "mxfp4", "mxfp8")), "experts": rng.randint(2, 32), "m": _log(rng, 1, 8192),
                "k": 32 * _log(rng, 4, 112), "n": _log(rng, 64, 4096), "hot": rng.choice((0.0, 0.4)), "dtype": "bf16"}
    return {"op": op, "tokens": _log(rng, 1, 16384), "experts": rng.choice((8, 60, 64, 160, 256)), "topk": rng.randint(1, 8),
            "seqs": _log(rng, 1, 64), "score": rng.choice(("sigmoid", "softmax")), "dtype": rng.choice(("fp32", "bf16"))}


# --------------------------------------------------------------------------
# the formats, in plain operations
# --------------------------------------------------------------------------
def _e2m1_code(t):
    """float32 -> 4-bit code, to nearest even, saturating at 6."""
    a = t.abs()
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return c + 8 * torch.signbit(t)


def _power(b):
    """2^(b - 127) of e8m0 bytes, float32 (0 stands for 2^-127, a subnormal number)."""
    b = b.to(torch.int32)
    return torch.where(b == 0, 1 << 22, b << 23).view(torch.float32)


def _quantize(x, fmt, g=None):
    """(packed values, scales) of a [rows, cols] float tensor."""
    rows, cols = x.shape
    xb = x.float().view(rows, cols // BLOCK[fmt], BLOCK[fmt])
    amax = xb.abs().amax(-1)
    fine = torch.isfinite(amax)
    if fmt == "nvfp4":
        g = 1.0 if g is None else g
        s = torch.where(fine, (amax / (amax.new_tensor(6.0) * g)).clamp(max=448.0), math.nan).to(torch.float8_e4m3fn)
        d = (s.float() * g)[..., None]
        t = torch.where(d > 0, xb / d, 0.0 * xb)
        scale = s
    else:
        e = (amax.view(torch.int32) >> 23) - (2 if fmt == "mxfp4" else 8)
        b = torch.where(fine, e.clamp(0, 254), 255)
        t = xb * _power(254 - b.clamp(max=254))[..., None]
        scale = b.to(torch.uint8).view(torch.float8_e8m0fnu)
    t = torch.where(fine[..., None], t, 0.0).view(rows, cols)
    if fmt == "mxfp8":
        return t.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale
    c = _e2m1_code(t)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8), scale


def _scale_values(scale):
    if scale.dtype == torch.float8_e8m0fnu:
        b = scale.view(torch.uint8)
        return torch.where(b == 255, math.nan, _power(b.clamp(max=254)))
    return scale.float()


def _values(q, scale, fmt):
    """float32 values of packed data and its scales (any leading dimensions)."""
    if fmt == "mxfp8":
        v = q.float()
    else:
        table = torch.tensor(E2M1 + tuple(-e for e in E2M1), device=q.device)
        v = table[torch.stack((q & 15, q >> 4), -1).int()].flatten(-2)
    return (v.unflatten(-1, (-1, BLOCK[fmt])) * _scale_values(scale)[..., None]).flatten(-2)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _hidden(gen, rows, cols):
    """Hidden states: normal, with a few columns that are an order larger."""
    x = torch.randn(rows, cols, generator=gen, device=DEV)
    hot = torch.rand(cols, generator=gen, device=DEV) < 0.01
    return torch.where(hot, 12.0 * x, x)


def _packed(x, fmt):
    """Quantised matrix and its tensor scale (None where the format has none)."""
    g = (x.abs().max() / (448.0 * 6.0)).reshape(1) if fmt == "nvfp4" else None
    return _quantize(x, fmt, g) + (g,)


def _offsets(gen, parts, total, hot):
    """Boundaries of `total` rows in `parts` runs: multinomial, `hot` of the rows in the first four, some runs empty."""
    w = torch.rand(parts, generator=gen, device=DEV) + 0.5
    w = w / w.sum() * (1.0 - hot)
    w[:4] += hot / min(4, parts)
    pick = torch.multinomial(w, total, replacement=True, generator=gen)
    return torch.cat((pick.new_zeros(1), torch.bincount(pick, minlength=parts).cumsum(0)))


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    st = dict(case)
    op = case["op"]
    if op == "quantize":
        x = _hidden(gen, case["rows"], case["cols"])
        st["g"] = (x.abs().max() / (448.0 * 6.0)).reshape(1) if case["fmt"] == "nvfp4" else None
        st["x"] = x.to(DTYPES[case["dtype"]])
    elif op == "norm":
        dt = DTYPES[case["dtype"]]
        st["x"] = (0.3 * _hidden(gen, case["rows"], case["cols"])).to(dt)
        st["res"] = _hidden(gen, case["rows"], case["cols"]).to(dt) if case["residual"] else None
        st["w"] = (1.0 + 0.1 * torch.randn(case["cols"], generator=gen, device=DEV)).to(dt)
    elif op in ("matmul", "experts"):
        fmt = case["fmt"]
        st["a"], st["sa"], ga = _packed(_hidden(gen, case["m"], case["k"]), fmt)
        many = case.get("experts", 1)
        parts = [_packed(0.02 * torch.randn(case["n"], case["k"], generator=gen, device=DEV), fmt) for _ in range(many)]
        st["b"] = torch.stack([p[0] for p in parts])
        st["sb"] = torch.stack([p[1].view(torch.uint8) for p in parts]).view(parts[0][1].dtype)
        st["alpha"] = torch.cat([ga * p[2] for p in parts]) if fmt == "nvfp4" else None
        if op == "matmul":
            st["b"], st["sb"] = st["b"][0], st["sb"][0]
        else:
            off = _offsets(gen, many, case["m"], case["hot"])
            st["off"] = off.int()
            # a padded batch for the plain form: row j of expert e, past the end the last row of all
            st["most"] = int((off[1:] - off[:-1]).max())
            at = off[:-1, None] + torch.arange(st["most"], device=DEV)
            st["valid"] = at < off[1:, None]
            st["at"] = at.clamp(max=case["m"] - 1)
        st["out"] = torch.zeros(case["m"], case["n"], dtype=DTYPES[case["dtype"]], device=DEV)
    else:
        t, e, s = case["tokens"], case["experts"], case["seqs"]
        x = torch.randn(t, e, generator=gen, device=DEV) + 0.5 * torch.randn(e, generator=gen, device=DEV)
        st["ids"] = x.topk(case["topk"], dim=1).indices.int()
        st["logits"] = x.to(DTYPES[case["dtype"]]).requires_grad_(True)
        st["off"] = _offsets(gen, s, t, 0.0).int()
        st["grad"] = torch.rand(s, generator=gen, device=DEV) + 0.5
        st["coeff"] = 1e-2
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _own(st):
    mx = importlib.import_module("flashinfer-mlsys_b200")
    op = st["op"]
    if op == "quantize":
        q, s = mx.quantize_mx(st["x"], st["fmt"], st["g"])
        return {"values": mx.dequantize_mx(q, s, st["fmt"], st["g"], st["x"].dtype), "scale": s}
    if op == "norm":
        q, s = mx.add_rmsnorm_quantize_mx(st["x"], st["res"], st["w"], EPS, st["fmt"])
        return {"q": q, "scale": s, "residual": st["res"]}
    if op == "matmul":
        return mx.matmul_mx(st["a"], st["sa"], st["b"], st["sb"], st["fmt"], st["alpha"], out=st["out"])
    if op == "experts":
        return mx.experts_matmul_mx(st["a"], st["sa"], st["b"], st["sb"], st["off"], st["fmt"], st["alpha"], out=st["out"])
    loss, counts = mx.balance_loss(st["logits"], st["ids"], st["off"], st["coeff"], st["score"])
    grad, = torch.autograd.grad(loss, st["logits"], st["grad"])
    return {"loss": loss, "counts": counts, "grad": grad}


def _plain_balance(st):
    x, ids, off = st["logits"].detach().float(), st["ids"], st["off"]
    t, e = x.shape
    s = st["seqs"]
    seq = torch.searchsorted(off[1:], torch.arange(t, device=DEV, dtype=torch.int32), right=True)
    member = (seq == torch.arange(s, device=DEV)[:, None]).float()
    counts = torch.zeros(s * e, dtype=torch.int32, device=DEV)
    counts.scatter_add_(0, (seq[:, None] * e + ids).flatten(), torch.ones(1, dtype=torch.int32, device=DEV).expand(ids.numel()))
    counts = counts.view(s, e)
    a = 1.0 / (1.0 + torch.exp(-x)) if st["score"] == "sigmoid" else torch.exp(x - x.amax(1, keepdim=True))
    p = a / a.sum(1, keepdim=True)
    length = (off[1:] - off[:-1]).float().clamp(min=1.0)
    f = counts.float() * (e / (ids.shape[1] * length))[:, None]
    loss = st["coeff"] * (f * (member @ p / length[:, None])).sum(1)
    ft = f[seq]
    d = p * (ft - (ft * p).sum(1, keepdim=True))
    d = d * (1.0 - a) if st["score"] == "sigmoid" else d
    grad = d * (st["coeff"] * st["grad"] / length)[seq][:, None]
    return {"loss": loss, "counts": counts, "grad": grad.to(st["logits"].dtype)}


def _plain(st):
    op = st["op"]
    if op == "quantize":
        q, s = _quantize(st["x"], st["fmt"], st["g"])
        v = _values(q, s, st["fmt"])
        return {"values": (v if st["g"] is None else v * st["g"]).to(st["x"].dtype), "scale": s}
    if op == "norm":
        h = st["x"].float()
        if st["res"] is not None:
            st["res"].copy_(h + st["res"].float())
            h = st["res"].float()
        y = h * (1.0 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)) * st["w"].float()
        q, s = _quantize(y, st["fmt"])
        return {"q": q, "scale": s, "residual": st["res"]}
    if op == "balance":
        return _plain_balance(st)
    a, b = _values(st["a"], st["sa"], st["fmt"]), _values(st["b"], st["sb"], st["fmt"])
    alpha = st["alpha"]
    if op == "matmul":
        y = a @ b.t()
        st["out"].copy_(y if alpha is None else y * alpha)
        return st["out"]
    y = torch.bmm(a[st["at"]], b.transpose(1, 2))
    y = y if alpha is None else y * alpha[:, None, None]
    # every row lies in one run: the padding adds zeros to a row that is written elsewhere
    rows = torch.zeros(st["out"].shape, device=DEV)
    rows.index_add_(0, st["at"].flatten(), torch.where(st["valid"][..., None], y, 0.0).flatten(0, 1))
    st["out"].copy_(rows)
    return st["out"]


def run(st):
    if own:
        return _own(st)
    return _plain(st)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _format_bytes(count, fmt):
    return count * (1.0 if fmt == "mxfp8" else 0.5) + count / BLOCK[fmt]


def work(case):
    op = case["op"]
    if op in ("quantize", "norm"):
        n = case["rows"] * case["cols"]
        size = DTYPES[case["dtype"]].itemsize
        if op == "quantize":  # the rows in, the format out, the values out
            return {"bytes": 2 * n * size + _format_bytes(n, case["fmt"]), "flops": 4.0 * n}
        return {"bytes": n * size * (3 if case["residual"] else 1) + case["cols"] * size + _format_bytes(n, case["fmt"]),
                "flops": 6.0 * n}
    if op in ("matmul", "experts"):
        m, n, k = case["m"], case["n"], case["k"]
        # an expert without rows need not be read: those that m draws are expected to reach
        many = case.get("experts", 1)
        used = many * (1.0 - (1.0 - (1.0 - case.get("hot", 0.0)) / many) ** m)
        return {"bytes": _format_bytes(m * k, case["fmt"]) + used * _format_bytes(n * k, case["fmt"]) + 2.0 * m * n,
                "flops": 2.0 * m * n * k}
    t, e, size = case["tokens"], case["experts"], DTYPES[case["dtype"]].itemsize
    # logits and ids in, gradient and counts out
    return {"bytes": 2.0 * t * e * size + 4.0 * t * case["topk"] + 4.0 * case["seqs"] * e, "flops": 20.0 * t * e}


# --------------------------------------------------------------------------
# 64 bits
# --------------------------------------------------------------------------
def _e2m1_exact(t):
    """Nearest e2m1 value of float64 numbers: the grid's step is 1/2 below 2, 1 below 4, 2 above."""
    a = t.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, t)


def _grid_exact(x, fmt, g=None):
    """(values in units of the scale, scale) in float64: [rows, blocks, block], [rows, blocks]."""
    xb = x.double().unflatten(1, (-1, BLOCK[fmt]))
    amax = xb.abs().amax(-1)
    if fmt == "nvfp4":
        g = 1.0 if g is None else g.double()
        want = (amax / (6.0 * g)).clamp(max=448.0)
        exp = torch.floor(torch.log2(want.clamp(min=2.0 ** -6)))
        s = torch.round(want / 2.0 ** (exp - 3)) * 2.0 ** (exp - 3)
        return _e2m1_exact(torch.where(s > 0, 1.0, 0.0)[..., None] * xb / (s * g).clamp(min=1e-300)[..., None]), s
    exp = torch.frexp(amax)[1].double() - 1.0
    s = 2.0 ** torch.where(amax > 0, exp - (2.0 if fmt == "mxfp4" else 8.0), -127.0).clamp(-127.0, 127.0)
    t = xb / s[..., None]
    if fmt == "mxfp4":
        return _e2m1_exact(t), s
    a = t.abs().clamp(max=448.0)
    ulp = 2.0 ** (torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / ulp) * ulp, t), s


def _values_exact(q, scale, fmt):
    if fmt == "mxfp8":
        v = q.double()
    else:
        c = torch.stack((q % 16, q // 16), -1).flatten(-2).int()
        exp, man = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(exp == 0, 0.5 * man, (1.0 + 0.5 * man) * 2.0 ** (exp.double() - 1.0))
        v = torch.where(c >= 8, -mag, mag)
    s = 2.0 ** (scale.view(torch.uint8).double() - 127.0) if scale.dtype == torch.float8_e8m0fnu else scale.double()
    return v * s.repeat_interleave(BLOCK[fmt], -1)


def exact(case, seed):
    st = prepare(case, seed)
    op, fmt = case["op"], case.get("fmt")
    if op == "quantize":
        v, s = _grid_exact(st["x"], fmt, st["g"])
        return {"values": (v * s[..., None]).flatten(1) * (1.0 if st["g"] is None else st["g"].double()), "scale": s}
    if op == "norm":
        h, res = st["x"].double(), None
        if st["res"] is not None:
            res = h + st["res"].double()
            h = res.to(st["x"].dtype).double()
        y = h * st["w"].double() / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
        v, s = _grid_exact(y, fmt)
        return {"q": v.flatten(1), "scale": s, "residual": res}
    if op == "matmul":
        y = _values_exact(st["a"], st["sa"], fmt) @ _values_exact(st["b"], st["sb"], fmt).t()
        return y if st["alpha"] is None else y * st["alpha"].double()
    if op == "experts":
        a, off = _values_exact(st["a"], st["sa"], fmt), st["off"].tolist()
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=DEV)
        for i in range(case["experts"]):
            if off[i] < off[i + 1]:
                w = _values_exact(st["b"][i], st["sb"][i], fmt)
                y[off[i]:off[i + 1]] = a[off[i]:off[i + 1]] @ w.t() * (1.0 if st["alpha"] is None else st["alpha"][i].double())
        return y
    x, off = st["logits"].detach().double().requires_grad_(True), st["off"].tolist()
    loss, e = [], case["experts"]
    for i in range(case["seqs"]):
        rows, ids = x[off[i]:off[i + 1]], st["ids"][off[i]:off[i + 1]]
        p = torch.softmax(rows, 1) if case["score"] == "softmax" else torch.sigmoid(rows) / torch.sigmoid(rows).sum(1, keepdim=True)
        n = max(1, rows.shape[0])
        f = torch.bincount(ids.flatten(), minlength=e).double() * e / (case["topk"] * n)
        loss.append(st["coeff"] * (f * p.sum(0) / n).sum())
    loss = torch.stack(loss)
    grad, = torch.autograd.grad(loss, x, st["grad"].double())
    return {"loss": loss.detach(), "counts": None, "grad": grad}
