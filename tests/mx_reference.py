"""The microscaled formats and the balance loss on the CPU, from their
definitions (test helpers). Quantisation follows the documented float32 steps
with float64 arithmetic rounded explicitly, products are float64."""
from __future__ import annotations

import torch

BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def e2m1_codes(t):
    """float64 -> codes: the nearest grid value, ties to the even code."""
    d = (t.abs().clamp(max=6.0)[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    even = torch.where(near, torch.arange(8) % 2 + torch.arange(8) / 100.0, torch.inf).argmin(-1)
    return (even + 8 * torch.signbit(t)).to(torch.uint8)


def quantize(x, fmt, g=None):
    """(codes uint8 [rows, cols] or e4m3 [rows, cols], scales) of a CPU tensor."""
    rows, cols = x.shape
    xb = x.float().view(rows, -1, BLOCK[fmt])
    amax = xb.abs().amax(-1)
    bad = ~torch.isfinite(xb).all(-1)
    if fmt == "nvfp4":
        gf = torch.ones(()) if g is None else g.float().reshape(())
        want = (amax.double() / (6.0 * gf).float().double()).float()   # one float32 rounding
        s = want.clamp(max=448.0).to(torch.float8_e4m3fn)
        s = torch.where(bad, torch.tensor(float("nan")), s.float()).to(torch.float8_e4m3fn)
        d = (s.float() * gf)[..., None]
        t = torch.where(d > 0, (xb.double() / d.double()).float(), torch.zeros(()))
    else:
        emax = 2 if fmt == "mxfp4" else 8
        b = ((amax.view(torch.int32) >> 23) - emax).clamp(0, 254)
        t = xb.double() * 2.0 ** (127.0 - b.double())[..., None]
        s = torch.where(bad, 255, b).to(torch.uint8).view(torch.float8_e8m0fnu)
    t = torch.where(bad[..., None], torch.zeros((), dtype=t.dtype), t).view(rows, cols)
    if fmt == "mxfp8":
        return t.float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s
    return e2m1_codes(t.double()), s


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(q):
    return torch.stack((q & 15, q >> 4), -1).flatten(-2)


def scale_values(scale):
    if scale.dtype == torch.float8_e8m0fnu:
        b = scale.view(torch.uint8).double()
        return torch.where(b == 255, torch.nan, 2.0 ** (b - 127.0))
    return scale.double()


def values(q, scale, fmt):
    """float64 values of packed CPU data (any leading dimensions)."""
    if fmt == "mxfp8":
        v = q.double()
    else:
        c = unpack(q).long()
        v = torch.where(c >= 8, -GRID[c & 7], GRID[c & 7])
    return v * scale_values(scale).repeat_interleave(BLOCK[fmt], -1)


def random_packed(gen, lead, rows, cols, fmt, spread=3):
    """Random codes with random scales (any bytes that are finite values)."""
    shape = (*lead, rows, cols // BLOCK[fmt])
    if fmt == "mxfp8":
        q = (torch.randn(*lead, rows, cols, generator=gen) * 64).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        q = torch.randint(0, 256, (*lead, rows, cols // 2), generator=gen, dtype=torch.uint8)
    if fmt == "nvfp4":
        s = (2.0 ** torch.randint(-spread, spread + 1, shape, generator=gen) * (1 + torch.rand(shape, generator=gen)))
        return q, s.to(torch.float8_e4m3fn)
    s = torch.randint(127 - spread, 128 + spread, shape, generator=gen, dtype=torch.uint8)
    return q, s.view(torch.float8_e8m0fnu)


def balance(logits, ids, off, coeff, score):
    """(loss [S], counts [S, E], gradient function of grad_loss) in float64."""
    x = logits.double().detach().requires_grad_(True)
    T, E = x.shape
    K = ids.shape[1]
    a = torch.sigmoid(x) if score == "sigmoid" else None
    off = [0, T] if off is None else off.tolist()
    losses, counts = [], []
    for lo, hi in zip(off[:-1], off[1:]):
        kept = ids[lo:hi].flatten()
        kept = kept[(kept >= 0) & (kept < E)].long()
        n = torch.bincount(kept, minlength=E)
        counts.append(n)
        if hi <= lo:
            losses.append(x.sum() * 0.0)
            continue
        rows = torch.softmax(x[lo:hi], 1) if score == "softmax" else a[lo:hi] / a[lo:hi].sum(1, keepdim=True)
        losses.append(coeff * (n.double() * E / (K * (hi - lo)) * rows.mean(0)).sum())
    loss = torch.stack(losses)
    return loss.detach(), torch.stack(counts), lambda g: torch.autograd.grad(loss, x, g.double(), retain_graph=True)[0]
