"""GPU: microscaled quantisation, residual + RMSNorm + quantisation and the
products, against plain CPU implementations (tests/mx_reference.py)."""
import pytest
import torch

import mx_reference as R
from conftest import pkg

pytestmark = pytest.mark.gpu

DEV = "cuda"
FMTS = list(R.BLOCK)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _hidden(rows, cols, dtype, seed):
    """Values over many binades, some zeros, a zero block, and (16-bit types
    apart) tiny and large ones."""
    g = _gen(seed)
    x = torch.randn(rows, cols, generator=g) * 2.0 ** torch.randint(-6, 7, (rows, cols // 32), generator=g).repeat_interleave(32, 1)
    x[torch.rand(rows, cols, generator=g) < 0.05] = 0.0
    x[0, :32] = 0.0
    x[-1, -32:] = torch.tensor([6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25]).repeat(4)  # ties of e2m1 at scale 1
    if rows > 2:
        x[1] *= 2.0 ** -13
        x[2, :16] = -0.0
    return x.to(dtype)


def _same(got, want):
    """Equal bytes (NaN scales included)."""
    assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


def _quantised(fmt, q, s, x, g=None):
    wq, ws = R.quantize(x, fmt, g)
    _same(s, ws)
    if fmt == "mxfp8":
        _same(q, wq)
    else:
        _same(q, R.pack(wq))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (17, 7168), (1000, 64)])
def test_quantize_bit_exact(gpu_available, fmt, dtype, rows, cols):
    x = _hidden(rows, cols, R.DTYPES[dtype], rows + cols)
    q, s = pkg().quantize_mx(x.to(DEV), fmt)
    _quantised(fmt, q, s, x)


@pytest.mark.parametrize("g", [1e-3, 0.37, 3.0, 1e-30, 1e25])
def test_quantize_global_scale(gpu_available, g):
    x = _hidden(9, 256, torch.float32, 5)
    gs = torch.tensor([g])
    q, s = pkg().quantize_mx(x.to(DEV), "nvfp4", gs.to(DEV))
    _quantised("nvfp4", q, s, x, gs)
    y = pkg().dequantize_mx(q, s, "nvfp4", gs.to(DEV), torch.float32)
    v = (R.values(q.cpu(), s.cpu(), "nvfp4").float() * gs).float()  # (value * scale) exact, one rounding
    torch.testing.assert_close(y.cpu(), v, rtol=0, atol=0)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_extreme_and_non_finite(gpu_available, fmt):
    x = torch.randn(6, 128, generator=_gen(2))
    x[0, 5] = float("inf")
    x[1, 40] = float("nan")
    x[2, 64:96] = 3.4e38
    x[3, :32] = 1e-45
    x[4, 32:64] = 1.2e-38
    x[5, 0] = -float("inf")
    q, s = pkg().quantize_mx(x.to(DEV), fmt)
    _quantised(fmt, q, s, x)
    y = pkg().dequantize_mx(q, s, fmt, dtype=torch.float32).cpu()
    v = R.values(q.cpu(), s.cpu(), fmt).float()
    torch.testing.assert_close(y, v, rtol=0, atol=0, equal_nan=True)
    blk = R.BLOCK[fmt]
    assert y[0, :blk].isnan().all() and y[1, 32:32 + blk].isnan().all() and y[2].isfinite().all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
def test_dequantize_rounds_once(gpu_available, fmt, dtype):
    q, s = R.random_packed(_gen(3), (), 37, 160, fmt)
    y = pkg().dequantize_mx(q.to(DEV), s.to(DEV), fmt, dtype=R.DTYPES[dtype])
    assert torch.equal(y.cpu(), R.values(q, s, fmt).to(R.DTYPES[dtype]))


def test_quantize_strides_outputs_and_empty(gpu_available):
    m = pkg()
    big = torch.randn(12, 512, generator=_gen(4)).to(torch.bfloat16)
    view = big.to(DEV)[1::2, 64:320]
    q, s = m.quantize_mx(view, "mxfp4")
    _quantised("mxfp4", q, s, big[1::2, 64:320])
    out, sc = torch.empty_like(q), torch.empty_like(s)
    a, b = m.quantize_mx(view, "mxfp4", None, out, sc)
    assert a is out and b is sc and torch.equal(out, q)
    back = torch.full((6, 512), 7.0, dtype=torch.float16, device=DEV)
    m.dequantize_mx(q, s, "mxfp4", out=back[:, 128:384])
    assert (back[:, :128] == 7).all() and (back[:, 384:] == 7).all()
    assert torch.equal(back[:, 128:384].cpu(), R.values(q.cpu(), s.cpu(), "mxfp4").half())
    e = torch.empty(0, 64, device=DEV)
    for fmt in FMTS:
        q0, s0 = m.quantize_mx(e, fmt)
        assert q0.shape[0] == 0 and m.dequantize_mx(q0, s0, fmt).shape == (0, 64)
        assert m.add_rmsnorm_quantize_mx(e, e.clone(), None, fmt=fmt)[0].shape[0] == 0


def test_more_than_2_31_elements(gpu_available):
    """Rows whose offsets pass 32 bits, in and out (about 10 GB)."""
    m = pkg()
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of free device memory")
    rows, cols = 310000, 7168
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[:2], x[-2:] = 1.0, _hidden(2, cols, torch.bfloat16, 6).to(DEV)
    q, s = m.quantize_mx(x, "mxfp4")
    _quantised("mxfp4", q[-2:], s[-2:], x[-2:].cpu())
    m.dequantize_mx(q, s, "mxfp4", out=x)
    assert torch.equal(x[-2:].cpu(), R.values(q[-2:].cpu(), s[-2:].cpu(), "mxfp4").bfloat16())
    b, sb = R.random_packed(_gen(7), (), cols, 32, "mxfp8")
    a = torch.zeros(rows, 32, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    sa = torch.full((rows, 1), 127, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    last, _ = R.random_packed(_gen(8), (), 2, 32, "mxfp8")
    a.view(torch.uint8)[-2:] = last.view(torch.uint8).to(DEV)
    m.matmul_mx(a, sa, b.to(DEV), sb.to(DEV), "mxfp8", out=x)
    assert (x[:-2:50000] == 0).all() and m.device_status() == 0
    _product_ok(x[-2:], last.double(), R.values(b, sb, "mxfp8"), 1.0, torch.bfloat16)


def test_refusals_on_the_device(gpu_available):
    m = pkg()
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    q, s = m.quantize_mx(x, "nvfp4")
    bad = [lambda: m.quantize_mx(x[:, :40], "mxfp4"), lambda: m.quantize_mx(x.t(), "mxfp4"),
           lambda: m.quantize_mx(x.long(), "mxfp4"), lambda: m.quantize_mx(x, "mxfp8", torch.ones(1, device=DEV)),
           lambda: m.quantize_mx(x, "nvfp4", torch.ones(1)), lambda: m.quantize_mx(x, "nvfp4", torch.ones(2, device=DEV)),
           lambda: m.quantize_mx(x.view(2, 2, 64)), lambda: m.quantize_mx(x, "nvfp4", out=q[:2]),
           lambda: m.quantize_mx(x[:, 4:36]), lambda: m.dequantize_mx(q, s, "mxfp4"), lambda: m.dequantize_mx(q, s[:2]),
           lambda: m.add_rmsnorm_quantize_mx(x, x.float()), lambda: m.add_rmsnorm_quantize_mx(x, None, x[0].float()),
           lambda: m.add_rmsnorm_quantize_mx(x, eps=-1.0), lambda: m.add_rmsnorm_quantize_mx(x, x[:2]),
           lambda: m.matmul_mx(q, s, q, s, "mxfp8"), lambda: m.matmul_mx(q, s, q[:, :16].contiguous(), s[:, :2].contiguous()),
           lambda: m.matmul_mx(q, s, q, s, out=torch.empty(4, 5, device=DEV)),
           lambda: m.matmul_mx(q, s, q, s, out=torch.empty(4, 4, device=DEV).t()[:, :4].long()),
           lambda: m.matmul_mx(q, s, q, s, out_dtype=torch.int32),
           lambda: m.matmul_mx(q, s, q, s, alpha=torch.ones(1)),
           lambda: m.experts_matmul_mx(q, s, q[None], s[None], torch.zeros(2, device=DEV)),
           lambda: m.experts_matmul_mx(q, s, q[None], s[None], torch.zeros(3, device=DEV, dtype=torch.int32)),
           lambda: m.experts_matmul_mx(q, s, q, s, torch.zeros(2, device=DEV, dtype=torch.int32))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# --------------------------------------------------------------------------
# residual + RMSNorm + quantisation
# --------------------------------------------------------------------------
def _check_rows(fmt, q, s, y):
    """Packed rows against float64 values y: within half a step of the format
    at the scale that came back, and that scale the one y asks for (or its
    neighbour where y's largest value is within the float32 error of a
    border). The float32 steps before quantisation: a sum of `cols` squares
    (<= 32 + 5 + 32 roundings), mean, add, root, reciprocal, two products:
    under 80 half-steps of 2^-24 each, i.e. 2^-17 relative."""
    err = 2.0 ** -17
    y = y.cpu()
    q, s = q.cpu(), s.cpu()
    lo, hi = [R.quantize((y * (1 + d)).float(), fmt)[1] for d in (-err, err)]
    sv, lo, hi = (R.scale_values(v) for v in (s, lo, hi))
    assert ((sv >= lo) & (sv <= hi)).all()
    sv = sv.repeat_interleave(R.BLOCK[fmt], 1)
    v = R.values(q, s, fmt)
    t = torch.where(sv > 0, y.abs() / sv, 0.0)
    if fmt == "mxfp8":
        step = torch.maximum(2.0 ** (torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3), torch.full_like(t, 2.0 ** -9))
        half = step / 2 + (t - 448).clamp(min=0)
    else:
        half = torch.where(t < 2, 0.25, torch.where(t < 4, 0.5, 1.0)) + (t - 6).clamp(min=0)
    assert ((v - y).abs() <= half * sv + err * y.abs() + 1e-300).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (9, 1024), (3, 1056), (33, 7168), (2, 8224), (2, 32768)])
def test_norm(gpu_available, fmt, dtype, rows, cols):
    dt = R.DTYPES[dtype]
    g = _gen(rows + cols)
    x, res = (torch.randn(rows, cols, generator=g).to(dt) for _ in range(2))
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dt)
    res_d = res.to(DEV)
    q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), res_d, w.to(DEV), 1e-5, fmt)
    h = (x.float() + res.float()).to(dt)
    assert torch.equal(res_d.cpu(), h)
    h = h.double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double()
    _check_rows(fmt, q, s, y)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
def test_norm_rounds_the_exact_value(gpu_available, dtype):
    """mxfp8 values and scales are those of the exact y (float64), rounded once:
    the sum's error of some 2^-30 moves one value in 10^8 across a border."""
    dt = R.DTYPES[dtype]
    g = _gen(77)
    x, w = torch.randn(40, 7168, generator=g).to(dt), (1 + 0.2 * torch.randn(7168, generator=g)).to(dt)
    x[3] = 1.0
    x[4] = 0.0
    w[:64] = 1.0
    q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, w.to(DEV), 2.0 ** -20, "mxfp8")
    h = x.double()
    y = h * w.double() / torch.sqrt(h.square().mean(1, keepdim=True) + 2.0 ** -20)
    amax = y.abs().view(40, -1, 32).amax(-1)
    e = torch.where(amax > 0, torch.floor(torch.log2(amax)) - 8 + 127, 0).clamp(0, 254)
    assert torch.equal(s.view(torch.uint8).cpu().double(), e)
    t = y / 2.0 ** (e - 127).repeat_interleave(32, 1)
    ulp = 2.0 ** (torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    want = (torch.round(t / ulp) * ulp).clamp(-448, 448)
    assert torch.equal(q.cpu().double(), want)


def test_norm_without_residual_or_weight(gpu_available):
    m = pkg()
    x = torch.randn(7, 256, generator=_gen(8)).to(torch.bfloat16)
    q, s = m.add_rmsnorm_quantize_mx(x.to(DEV), None, None, fmt="mxfp4")
    _quantised("mxfp4", q, s, x)                       # y = h = x
    w = torch.ones(256, dtype=torch.bfloat16)
    xd = x.to(DEV)
    q, s = m.add_rmsnorm_quantize_mx(xd, None, w.to(DEV), 1e-6, "mxfp8")
    assert torch.equal(xd.cpu(), x)
    h = x.double()
    _check_rows("mxfp8", q, s, h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6))


def test_norm_strides_global_scale_zero_row_and_nan_row(gpu_available):
    m = pkg()
    g = _gen(9)
    big = torch.randn(10, 640, generator=g)
    big[2] = 0.0
    big[4, 300] = float("nan")
    x = big.to(DEV)[::2, 128:512]
    res = torch.zeros(5, 400, device=DEV)
    res[:, 384:] = 3.0
    w = torch.rand(384, generator=g) + 0.5
    gs = torch.tensor([0.01])
    q, s = m.add_rmsnorm_quantize_mx(x, res[:, :384], w.to(DEV), 1e-6, "nvfp4", gs.to(DEV))
    assert (res[:, 384:] == 3).all()
    h = big[::2, 128:512].double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w.double()
    deq = m.dequantize_mx(q, s, "nvfp4", gs.to(DEV), torch.float32).cpu().double()
    assert (deq[1] == 0).all() and deq[2].isnan().all()
    ok = [0, 3, 4]
    # half a step of e2m1 (1/4 of the value at most, 1/12 of the block's largest) and the scale's 2^-4
    bound = y.abs() * (0.25 + 2.0 ** -4) + y.abs().view(5, -1, 16).amax(-1).repeat_interleave(16, 1) / 12
    assert ((deq - y).abs()[ok] <= bound[ok] * 1.01).all()


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------
def _product_ok(got, a, b, alpha, dt, note=""):
    """Against float64. The tensor core adds 32 or 64 exact products at a time
    to a float32 sum. Counted: one float32 step (2^-23) of the sum of
    magnitudes for every 32 values of K and 8 more for the alignment inside a
    step, the split's additions and alpha; then half a step of the output's type."""
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    tol = (a.shape[1] / 32 + 8) * 2.0 ** -23 * mag * abs(alpha) + torch.finfo(dt).eps / 2 * (ref * alpha).abs() * 1.01
    bad = (got.cpu().double() - ref * alpha).abs() > tol + 1e-30
    assert not bad.any(), f"{note}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


# rows x weight rows x width: one token, tile borders of both, K ends inside a
# stage and inside a scale word, K splits of 2..8, several tiles a CTA
SHAPES = [(1, 128, 256), (1, 1, 32), (1, 4096, 7168), (8, 130, 96), (16, 128, 512), (17, 300, 480), (33, 257, 2048), (64, 64, 1024),
          (65, 129, 736), (127, 512, 288), (200, 384, 4096), (256, 256, 256), (257, 128, 1184), (1000, 7168, 160), (700, 6000, 224)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(gpu_available, fmt, m, n, k):
    g = _gen(m + n + k)
    a, sa = R.random_packed(g, (), m, k, fmt)
    b, sb = R.random_packed(g, (), n, k, fmt)
    out = pkg().matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), fmt, out_dtype=torch.float32)
    assert pkg().device_status() == 0
    _product_ok(out, R.values(a, sa, fmt), R.values(b, sb, fmt), 1.0, torch.float32, f"{fmt} {m} {n} {k}")


@pytest.mark.parametrize("dtype", list(R.DTYPES))
def test_matmul_types_alpha_and_strided_output(gpu_available, dtype):
    dt = R.DTYPES[dtype]
    g = _gen(12)
    a, sa = R.random_packed(g, (), 70, 320, "nvfp4", 1)
    b, sb = R.random_packed(g, (), 201, 320, "nvfp4", 1)
    out = torch.full((72, 211), 9.0, dtype=dt, device=DEV)
    al = torch.tensor([0.0173])
    got = pkg().matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), "nvfp4", al.to(DEV), out=out[1:71, 3:204])
    assert got.data_ptr() == out[1:, 3:].data_ptr()
    _product_ok(got, R.values(a, sa, "nvfp4"), R.values(b, sb, "nvfp4"), float(al), dt)
    assert (out[0] == 9).all() and (out[71] == 9).all() and (out[:, :3] == 9).all() and (out[:, 204:] == 9).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_matmul_nan_scale_stays_in_its_row(gpu_available, fmt):
    g = _gen(13)
    a, sa = R.random_packed(g, (), 40, 512, fmt)
    b, sb = R.random_packed(g, (), 140, 512, fmt)
    nan = 0x7F if fmt == "nvfp4" else 255
    sa.view(torch.uint8)[7, 3] = nan
    sb.view(torch.uint8)[131, 9] = nan
    out = pkg().matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), fmt, out_dtype=torch.float32).cpu()
    nan = torch.zeros(40, 140, dtype=torch.bool)
    nan[7] = nan[:, 131] = True
    assert torch.equal(out.isnan(), nan)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("m,n,k", [(9, 70, 256), (150, 300, 416)])
def test_matmul_scales_at_any_address(gpu_available, fmt, shift, m, n, k):
    """Contiguous scales that start anywhere in memory, and rows of scales of any length."""
    g = _gen(m + shift)
    a, sa = R.random_packed(g, (), m, k, fmt)
    b, sb = R.random_packed(g, (), n, k, fmt)

    def moved(s):
        flat = torch.full((s.numel() + shift,), 0x7F, dtype=torch.uint8, device=DEV)
        flat[shift:] = s.view(torch.uint8).flatten().to(DEV)
        return flat[shift:].view(s.shape).view(s.dtype)

    out = pkg().matmul_mx(a.to(DEV), moved(sa), b.to(DEV), moved(sb), fmt, out_dtype=torch.float32)
    _product_ok(out, R.values(a, sa, fmt), R.values(b, sb, fmt), 1.0, torch.float32, f"{fmt} {shift}")


def test_matmul_empty(gpu_available):
    m = pkg()
    b, sb = (t.to(DEV) for t in R.random_packed(_gen(1), (), 8, 64, "nvfp4"))
    out = m.matmul_mx(b[:0], sb[:0], b, sb)
    assert out.shape == (0, 8)
    e = m.experts_matmul_mx(b[:0], sb[:0], b[None], sb[None], torch.zeros(2, dtype=torch.int32, device=DEV))
    assert e.shape == (0, 8)


def _runs(counts, first=0):
    off = torch.tensor([first] + list(counts)).cumsum(0).int()
    return off, int(off[-1])


EXPERTS = [([1], 128, 256), ([0, 0, 1, 0], 256, 7168), ([3, 0, 17, 1, 16], 130, 96), ([40, 0, 0, 250, 5, 129], 300, 480),
           ([1] * 40, 64, 512), ([2] * 33 + [0] * 70 + [300], 128, 736), ([500, 0, 1], 200, 2048), ([0, 0], 128, 64)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("counts,n,k", EXPERTS)
def test_experts_matmul(gpu_available, fmt, counts, n, k):
    """Ragged runs, empty ones among them, rows before and behind them left as they were."""
    off, end = _runs(counts, 2)
    rows, e = end + 3, len(counts)
    g = _gen(sum(counts) + n + k)
    a, sa = R.random_packed(g, (), rows, k, fmt)
    b, sb = R.random_packed(g, (e,), n, k, fmt)
    al = torch.rand(e, generator=g) + 0.5
    out = torch.full((rows, n), 5.0, device=DEV)
    pkg().experts_matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), off.to(DEV), fmt, al.to(DEV), out=out)
    assert pkg().device_status() == 0
    assert (out[:2] == 5).all() and (out[end:] == 5).all()
    av = R.values(a, sa, fmt)
    for i, c in enumerate(counts):
        if c:
            lo = int(off[i])
            _product_ok(out[lo:lo + c], av[lo:lo + c], R.values(b[i], sb[i], fmt), float(al[i]), torch.float32, f"expert {i}")


@pytest.mark.parametrize("offsets,runs", [([0, 6, 3, 9], [(0, 6), (6, 6), (6, 9)]), ([-4, 2, 1000, 7], [(0, 2), (2, 12), (12, 12)]),
                                          ([9, 4, 4, 4], [(9, 9)] * 3)])
def test_experts_matmul_keeps_bad_offsets_inside(gpu_available, offsets, runs):
    """Offsets that decrease or leave [0, m] are kept inside and in order."""
    g = _gen(22)
    a, sa = R.random_packed(g, (), 12, 96, "mxfp8")
    b, sb = R.random_packed(g, (3,), 40, 96, "mxfp8")
    out = torch.full((12, 40), 5.0, device=DEV)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    pkg().experts_matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), off, "mxfp8", out=out)
    assert pkg().device_status() == 0
    left = torch.ones(12, dtype=torch.bool)
    av = R.values(a, sa, "mxfp8")
    for e, (lo, hi) in enumerate(runs):
        left[lo:hi] = False
        if lo < hi:
            _product_ok(out[lo:hi], av[lo:hi], R.values(b[e], sb[e], "mxfp8"), 1.0, torch.float32)
    assert (out.cpu()[left] == 5).all()


def test_experts_matmul_more_experts_than_a_warp_scans(gpu_available):
    counts = [3 if i % 5 == 0 else 0 for i in range(300)]
    off, m = _runs(counts)
    g = _gen(23)
    a, sa = R.random_packed(g, (), m, 64, "mxfp4")
    b, sb = R.random_packed(g, (300,), 24, 64, "mxfp4")
    out = pkg().experts_matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), off.to(DEV), "mxfp4", out_dtype=torch.float32)
    av = R.values(a, sa, "mxfp4")
    for i in range(0, 300, 5):
        lo = int(off[i])
        _product_ok(out[lo:lo + 3], av[lo:lo + 3], R.values(b[i], sb[i], "mxfp4"), 1.0, torch.float32)


def test_experts_matmul_without_out_is_zero_outside(gpu_available):
    g = _gen(21)
    a, sa = (t.to(DEV) for t in R.random_packed(g, (), 9, 64, "nvfp4"))
    b, sb = (t.to(DEV) for t in R.random_packed(g, (2,), 8, 64, "nvfp4"))
    out = pkg().experts_matmul_mx(a, sa, b, sb, torch.tensor([2, 4, 4], dtype=torch.int32, device=DEV))
    assert out.dtype == torch.bfloat16 and (out[:2] == 0).all() and (out[4:] == 0).all() and (out[2:4] != 0).any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(3, 130, 1 << 20), (130, 130, 1 << 17), (2, 1 << 18, 32), (200, 1 << 18, 32)])
def test_matmul_longest_axes(gpu_available, fmt, m, n, k):
    g = _gen(n + m)
    a, sa = R.random_packed(g, (), m, k, fmt)
    b, sb = R.random_packed(g, (), n, k, fmt)
    out = pkg().matmul_mx(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), fmt, out_dtype=torch.float32)
    assert pkg().device_status() == 0
    pick = slice(None) if n < 1000 else slice(None, None, 997)
    av = R.values(a, sa, fmt)
    _product_ok(out[:, pick], av, R.values(b[pick], sb[pick], fmt), 1.0, torch.float32, f"{fmt} {m} {n} {k}")
    _product_ok(out[:, -1:], av, R.values(b[-1:], sb[-1:], fmt), 1.0, torch.float32, "last weight row")


def test_experts_matmul_weights_past_32_bits(gpu_available):
    """512 experts whose weights take 8 GB: the last ones' rows."""
    m = pkg()
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of free device memory")
    n, k = 1 << 16, 256
    b = torch.zeros(512, n, k, dtype=torch.uint8, device=DEV)
    sb = torch.full((512, n, k // 32), 127, dtype=torch.uint8, device=DEV)
    g = _gen(51)
    w, sw = R.random_packed(g, (2,), 300, k, "mxfp8")
    b[510:, -300:], sb[510:, -300:] = w.view(torch.uint8).to(DEV), sw.view(torch.uint8).to(DEV)
    a, sa = R.random_packed(g, (), 20, k, "mxfp8")
    off = torch.tensor([0] * 510 + [2, 3, 20], dtype=torch.int32, device=DEV)
    out = m.experts_matmul_mx(a.to(DEV), sa.to(DEV), b.view(torch.float8_e4m3fn), sb.view(torch.float8_e8m0fnu), off,
                              "mxfp8", out_dtype=torch.float32)
    assert m.device_status() == 0 and (out[:, :-300] == 0).all() and (out[:2] == 0).all()
    av = R.values(a, sa, "mxfp8")
    _product_ok(out[2:3, -300:], av[2:3], R.values(w[0], sw[0], "mxfp8"), 1.0, torch.float32)
    _product_ok(out[3:, -300:], av[3:], R.values(w[1], sw[1], "mxfp8"), 1.0, torch.float32)


def test_products_of_the_most_rows(gpu_available):
    """2^24 rows: their number of tiles, and outputs past 2^31 elements."""
    m = pkg()
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of free device memory")
    rows, n, k = 1 << 24, 192, 32
    g = _gen(52)
    a, sa = R.random_packed(g, (), 1000, k, "mxfp4")
    b, sb = R.random_packed(g, (2,), n, k, "mxfp4")
    big = torch.zeros(rows, k // 2, dtype=torch.uint8, device=DEV)
    sbig = torch.full((rows, 1), 127, dtype=torch.uint8, device=DEV)
    big[-1000:], sbig[-1000:] = a.to(DEV), sa.view(torch.uint8).to(DEV)
    sbig = sbig.view(torch.float8_e8m0fnu)
    out = torch.full((rows, n), 5.0, dtype=torch.bfloat16, device=DEV)
    m.matmul_mx(big, sbig, b[0].to(DEV), sb[0].to(DEV), "mxfp4", out=out)
    assert m.device_status() == 0 and not out[:-1000].any()
    av, bv = R.values(a, sa, "mxfp4"), R.values(b, sb, "mxfp4")
    _product_ok(out[-1000:], av, bv[0], 1.0, torch.bfloat16)
    out.fill_(5.0)
    off = torch.tensor([7, rows - 500, rows - 1], dtype=torch.int32, device=DEV)
    m.experts_matmul_mx(big, sbig, b.to(DEV), sb.to(DEV), off, "mxfp4", out=out)
    assert m.device_status() == 0 and (out[:7] == 5).all() and (out[-1] == 5).all() and not out[7:-1000].any()
    _product_ok(out[-1000:-500], av[:500], bv[0], 1.0, torch.bfloat16)
    _product_ok(out[-500:-1], av[500:-1], bv[1], 1.0, torch.bfloat16)


def test_products_are_repeatable_on_streams_and_in_graphs(gpu_available):
    """The same bits again, from two streams at once and from a replayed graph
    whose inputs have changed."""
    m = pkg()
    g = _gen(31)
    a, sa = (t.to(DEV) for t in R.random_packed(g, (), 24, 4096, "nvfp4"))
    b, sb = (t.to(DEV) for t in R.random_packed(g, (), 512, 4096, "nvfp4"))
    a2, sa2 = (t.to(DEV) for t in R.random_packed(g, (), 24, 4096, "nvfp4"))
    first, second = m.matmul_mx(a, sa, b, sb), m.matmul_mx(a2, sa2, b, sb)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(first) for _ in range(2)]
    for _ in range(10):
        for st, o, (x, sx) in zip(streams, outs, ((a, sa), (a2, sa2))):
            with torch.cuda.stream(st):
                m.matmul_mx(x, sx, b, sb, out=o)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], second)
    x, sx, o = a.clone(), sa.clone(), torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.matmul_mx(x, sx, b, sb, out=o)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, first)
    x.copy_(a2)
    sx.copy_(sa2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, second) and m.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_expert_mlp_after_routing(gpu_available, fmt):
    """The operators as a layer uses them: residual + norm + quantise, route,
    rows sorted by expert, gate and up products, SwiGLU, quantise, down
    products, weighted sum; against float64 of the same quantised values."""
    m = pkg()
    T, H, I, E = 24, 512, 256, 32
    g = _gen(41)
    x, res = (torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(torch.bfloat16).to(DEV)
    logits = torch.randn(T, 256, generator=g).to(DEV)
    bias = torch.zeros(256, dtype=torch.bfloat16, device=DEV)
    ids, wts, _ = m.route(logits, bias, 0, E, 2.5)
    loss, counts = m.balance_loss(logits, ids)
    flat = ids.flatten()
    local = flat < E
    order = torch.argsort(torch.where(local, flat, E), stable=True)[: int(local.sum())]
    tok, exp = order // 8, flat[order]
    off = torch.cat((counts.new_zeros(1, 1), counts[:, :E].cumsum(1)), 1).flatten().int()
    assert int(off[-1]) == order.numel()
    q, s = m.add_rmsnorm_quantize_mx(x, res, w, 1e-6, fmt)
    w13, s13 = (t.to(DEV) for t in R.random_packed(g, (E,), 2 * I, H, fmt))
    w2, s2 = (t.to(DEV) for t in R.random_packed(g, (E,), H, I, fmt))
    qa, sa = q[tok].contiguous(), s.view(torch.uint8)[tok].contiguous().view(s.dtype)
    h = m.experts_matmul_mx(qa, sa, w13, s13, off, fmt, out_dtype=torch.float32)
    act = h[:, :I] * (h[:, I:] * 2.0 ** -8).sigmoid()
    qi, si = m.quantize_mx(act, fmt)
    y = m.experts_matmul_mx(qi, si, w2, s2, off, fmt, out_dtype=torch.float32)
    out = torch.zeros(T, H, device=DEV).index_add_(0, tok, y * wts.flatten()[order][:, None])
    assert m.device_status() == 0
    av, iv = R.values(qa.cpu(), sa.cpu(), fmt), R.values(qi.cpu(), si.cpu(), fmt)
    for e in exp.unique().tolist():
        r = (exp == e).nonzero().flatten().cpu()
        _product_ok(h[r], av[r], R.values(w13[e].cpu(), s13[e].cpu(), fmt), 1.0, torch.float32)
        _product_ok(y[r], iv[r], R.values(w2[e].cpu(), s2[e].cpu(), fmt), 1.0, torch.float32)
    assert out.isfinite().all() and (out.abs().sum(1) > 0).any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("g", [None, 0.37, 1e-30])
def test_quantize_keeps_the_sign_of_zero(gpu_available, fmt, dtype, g):
    """x / s is -0 where x is: single -0 among ordinary values, in every branch of the scale."""
    x = _hidden(11, 256, R.DTYPES[dtype], 21)
    x[torch.rand(11, 256, generator=_gen(22)) < 0.2] = -0.0
    x[5] = 1.0
    x[5, ::3] = -0.0
    gs = torch.tensor([g]) if g and fmt == "nvfp4" else None
    q, s = pkg().quantize_mx(x.to(DEV), fmt, None if gs is None else gs.to(DEV))
    _quantised(fmt, q, s, x, gs)
    if gs is None:
        q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, None, fmt=fmt)
        _quantised(fmt, q, s, x)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("cols", [32, 96, 512, 1024, 7168, 32768])
def test_norm_of_exact_quotients(gpu_available, fmt, dtype, cols):
    """Rows whose y is a short number although 1 / sqrt(v) is none: +-c alone,
    one entry in four (y = 2 w), nine in sixteen (4/3 w), and c = 3, eps = 7 (3/4
    w), with weights that put y on borders and ties of the formats. Codes and
    scales are y's."""
    dt = R.DTYPES[dtype]
    g = _gen(cols)
    w = torch.tensor([1.0, 0.75, 1.0625, 1.1875, 1.25, 3.5, 5.0, 0.25])[torch.randint(0, 8, (cols,), generator=g)]
    w[:32] = 1.0
    for c in (7.0, 13.0, 14.0, 49.0, 0.1, 1e-3, 517.0):
        sign = torch.randint(0, 2, (6, cols), generator=g) * 2.0 - 1.0
        part = sign.clone()
        part.view(6, -1, 4)[:, :, 1:] = 0.0
        for rows, scale in ((sign, 1.0), (part, 2.0)):
            x = (rows * torch.tensor(c)).to(dt)
            q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, w.to(dt).to(DEV), 0.0, fmt)
            _quantised(fmt, q, s, rows * scale * w)
        nine = sign.clone()
        nine.view(6, -1, 16)[:, :, ::2] = 0.0
        nine.view(6, -1, 16)[:, :, 8] = 1.0
        q, s = pkg().add_rmsnorm_quantize_mx((nine * torch.tensor(c)).to(dt).to(DEV), None, (0.75 * w).to(dt).to(DEV), 0.0, fmt)
        _quantised(fmt, q, s, nine * w)
    x = (sign * 3.0).to(dt)
    q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, w.to(dt).to(DEV), 7.0, fmt)
    _quantised(fmt, q, s, sign * 0.75 * w)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,cols", [(40, 64), (40, 1024)])
def test_norm_keeps_the_sign_of_zero(gpu_available, fmt, dtype, rows, cols):
    """y = h w / sqrt(v) is -0 where h is -0 and w is positive, or the other way round."""
    g = _gen(80 + cols)
    x = torch.randn(rows, cols, generator=g).to(R.DTYPES[dtype])
    w = (torch.randint(0, 2, (cols,), generator=g) * 2.0 - 1.0).to(x.dtype)
    x[:, ::3] = -0.0
    x[:, 1::3] = 0.0
    q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, w.to(DEV), 1e-6, fmt)
    codes = q.cpu().view(torch.uint8) if fmt == "mxfp8" else R.unpack(q.cpu())
    minus = 0x80 if fmt == "mxfp8" else 8
    want = torch.where(torch.signbit(x.float() * w.float()), minus, 0).to(torch.uint8)
    zero = x == 0
    assert torch.equal(codes[zero], want[zero])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("cols", [64, 2048])
def test_norm_whose_product_with_the_weight_is_large(gpu_available, fmt, dtype, cols):
    """h w passes float32's range, y does not. One block has a y that does: its scale is NaN."""
    dt = R.DTYPES[dtype]
    g = _gen(60 + cols)
    x = (torch.randn(5, cols, generator=g) * 1e15).to(dt)
    x[1] *= 100.0
    w = ((1 + 0.2 * torch.randn(cols, generator=g)) * 1e28).to(dt)
    w[::7] = 1.0
    w[40] = 2.0 ** 127
    x[:, 40] = 0.0
    x[2, 40] = 5e15
    q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), None, w.to(DEV), 1e-5, fmt, *([torch.tensor([1e26], device=DEV)] if fmt == "nvfp4" else []))
    h = x.double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double()
    over = (y.abs() > torch.finfo(torch.float32).max).view(5, -1, R.BLOCK[fmt]).any(-1)
    assert over[2].any() and torch.equal(R.scale_values(s.cpu()).isnan(), over)
    y[over.repeat_interleave(R.BLOCK[fmt], 1)] = 0.0
    if fmt == "nvfp4":
        v = R.values(q.cpu(), s.cpu(), fmt) * 1e26
        ok = ~over.repeat_interleave(16, 1)
        # half a step of e2m1 and the scale's 2^-4, as above
        bound = y.abs() * (0.25 + 2.0 ** -4) + y.abs().view(5, -1, 16).amax(-1).repeat_interleave(16, 1) / 12
        assert ((v - y).abs()[ok] <= bound[ok] * 1.01).all()
    else:
        ok = ~over.any(1)
        _check_rows(fmt, q[ok.to(DEV)], s.view(torch.uint8)[ok.to(DEV)].view(s.dtype), y[ok])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(5, 32), (7, 96), (6, 512), (3, 7168)])
def test_norm_of_very_large_and_very_small_rows(gpu_available, fmt, dtype, rows, cols):
    """Squares that pass float32's range or fall below it, beside ordinary rows."""
    dt = R.DTYPES[dtype]
    g = _gen(rows + cols)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dt)
    for size, eps in ((1e20, 1e-5), (3e37, 1e-5), (1e-22, 0.0), (1e-30, 0.0), (1e-36, 1e-30), (1e-39, 0.0)):
        x = torch.randn(rows, cols, generator=g)
        x[::2] *= size
        x = x.to(dt)
        res = torch.zeros_like(x).to(DEV)
        q, s = pkg().add_rmsnorm_quantize_mx(x.to(DEV), res, w.to(DEV), eps, fmt)
        assert torch.equal(res.cpu(), x)
        h = x.double()
        e = float(torch.tensor(eps, dtype=torch.float32))
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + e) * w.double()
        if fmt == "nvfp4":
            # amax / 6 below 2^-10, half of e4m3's smallest number, is a scale of 0 and zeros: y ~ 1e-21 of size 1e-36
            none = y.view(rows, -1, 16).abs().amax(-1) / 6 < 2.0 ** -10 * (1 - 2.0 ** -16)
            assert (s.cpu().float()[none] == 0).all() and (R.unpack(q.cpu()).view(rows, -1, 16)[none] == 0).all()
            y[none.repeat_interleave(16, 1)] = 0.0
        _check_rows(fmt, q, s, y)


def test_written_tensors_are_known_to_autograd(gpu_available):
    """A tensor that autograd has saved and a call then writes: the backward
    pass refuses, as after any other write in place."""
    m = pkg()
    x = torch.randn(4, 64, generator=_gen(70)).to(DEV)
    q, s = m.quantize_mx(x, "mxfp8")
    leaf = torch.randn(4, 64, generator=_gen(71)).to(DEV).requires_grad_(True)
    for write in (lambda t: m.add_rmsnorm_quantize_mx(x, t, None), lambda t: m.dequantize_mx(q, s, "mxfp8", out=t),
                  lambda t: m.matmul_mx(q, s, torch.cat([q.view(torch.uint8)] * 16).view(q.dtype),
                                        torch.cat([s.view(torch.uint8)] * 16).view(s.dtype), "mxfp8", out=t)):
        t = leaf * 2.0
        loss = (t * t).sum()
        with torch.no_grad():
            write(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # tensors without a version are written all the same
        t = x * 1.0
        m.dequantize_mx(q, s, "mxfp8", out=t)
        assert torch.equal(t.cpu(), R.values(q.cpu(), s.cpu(), "mxfp8").float())


@pytest.mark.parametrize("fmt", FMTS)
def test_weighted_sum_of_the_experts_rows(gpu_available, fmt):
    """The chain of the test above, with its final output: token by token, slot
    by slot in float64 from the quantised values and the routing, without the
    sort and the offsets."""
    m = pkg()
    T, H, I, E = 24, 512, 256, 32
    g = _gen(43)
    x, res = (torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(torch.bfloat16).to(DEV)
    logits = torch.randn(T, 256, generator=g).to(DEV)
    ids, wts, n = m.route(logits, torch.zeros(256, dtype=torch.bfloat16, device=DEV), 0, E, 2.5)
    flat = ids.flatten()
    order = torch.argsort(torch.where(flat < E, flat, E), stable=True)[: int((flat < E).sum())]
    tok = order // 8
    off = torch.cat((n.new_zeros(1), n[:E].cumsum(0))).int()
    q, s = m.add_rmsnorm_quantize_mx(x, res, w, 1e-6, fmt)
    w13, s13 = (t.to(DEV) for t in R.random_packed(g, (E,), I, H, fmt))
    w2, s2 = (t.to(DEV) for t in R.random_packed(g, (E,), H, I, fmt))
    h = m.experts_matmul_mx(q[tok].contiguous(), s.view(torch.uint8)[tok].contiguous().view(s.dtype), w13, s13, off, fmt)
    qi, si = m.quantize_mx(h, fmt)
    y = m.experts_matmul_mx(qi, si, w2, s2, off, fmt, out_dtype=torch.float32)
    out = torch.zeros(T, H, device=DEV).index_add_(0, tok, y * wts.flatten()[order][:, None]).cpu().double()
    assert m.device_status() == 0
    a, up, down = R.values(q.cpu(), s.cpu(), fmt), R.values(w13.cpu(), s13.cpu(), fmt), R.values(w2.cpu(), s2.cpu(), fmt)
    hv, yv, wv = h.cpu().double(), R.values(qi.cpu(), si.cpu(), fmt), wts.cpu().double()
    row = {int(o): i for i, o in enumerate(order.tolist())}  # slot -> sorted row
    want, size = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for k in range(8):
            e = int(ids[t, k])
            if e >= E:
                continue
            i = row[8 * t + k]
            mag = a[t].abs() @ up[e].abs().t()
            assert ((hv[i] - a[t] @ up[e].t()).abs() <= (H / 32 + 8) * 2.0 ** -23 * mag + 2.0 ** -8 * 1.01 * hv[i].abs() + 1e-30).all()
            want[t] += wv[t, k] * (yv[i] @ down[e].t())
            size[t] += wv[t, k] * (yv[i].abs() @ down[e].abs().t())
    assert (size.amax(1) > 0).sum() > T // 2
    # the product's steps as in _product_ok, then a product and at most eight additions of 2^-24
    assert ((out - want).abs() <= ((I / 32 + 8) * 2.0 ** -23 + 10 * 2.0 ** -24) * size + 1e-30).all()
