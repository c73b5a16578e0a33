"""CPU: the microscaled operators' and the balance loss' refusals, and the
reference implementation that the GPU tests compare with."""
import pytest
import torch

import mx_reference as R
from conftest import pkg

OK, INVALID, ALIGN, NO_DEVICE = 0, 1, 2, 4
P = 1 << 20  # an aligned address that no call here reads: arguments are checked before any launch


def test_reference_rounding():
    t = torch.tensor([0.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.0, -0.25, -5.5], dtype=torch.float64)
    want = torch.tensor([0, 0, 1, 2, 2, 4, 4, 6, 6, 7, 7, 8, 15], dtype=torch.uint8)
    assert torch.equal(R.e2m1_codes(t), want)


@pytest.mark.parametrize("fmt", list(R.BLOCK))
def test_reference_round_trip_is_within_half_a_step(fmt):
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(1)) * 3
    q, s = R.quantize(x, fmt)
    v = R.values(q if fmt == "mxfp8" else R.pack(q), s, fmt)
    sv = R.scale_values(s).repeat_interleave(R.BLOCK[fmt], 1)
    t = (x.double() / sv).abs()
    if fmt == "mxfp8":  # half a step 2^-4 of the value, 2^-10 below the normal range; up to 512 saturates at 448
        half = torch.maximum(t * 2.0 ** -4, torch.full_like(t, 2.0 ** -10)) + (t - 448).clamp(min=0)
    else:               # half a step of 1/2, 1 or 2; nvfp4's scale may round down by 2^-4, mxfp4 saturates up to 8
        half = torch.where(t < 2, 0.25, torch.where(t < 4, 0.5, 1.0)) + (t - 6).clamp(min=0)
    assert ((v - x.double()).abs() <= half * sv * (1 + 1e-6)).all()


def _quant(lib, **k):
    a = dict(x=P, dt=0, rows=4, cols=64, ld=64, fmt=0, g=None, q=P, s=P)
    a.update(k)
    return lib.moe_fp8_ds_quantize_mx(a["x"], a["dt"], a["rows"], a["cols"], a["ld"], a["fmt"], a["g"], a["q"], a["s"], None)


def _dequant(lib, **k):
    a = dict(x=P, dt=0, rows=4, cols=64, ld=64, fmt=0, g=None, q=P, s=P)
    a.update(k)
    return lib.moe_fp8_ds_dequantize_mx(a["q"], a["s"], a["rows"], a["cols"], a["fmt"], a["g"], a["dt"], a["x"], a["ld"], None)


BAD_ROWS = [(dict(rows=-1), INVALID), (dict(rows=(1 << 24) + 1), INVALID), (dict(cols=0), INVALID), (dict(cols=48), INVALID),
            (dict(cols=1 << 21, ld=1 << 21), INVALID), (dict(fmt=3), INVALID), (dict(fmt=-1), INVALID), (dict(dt=3), INVALID),
            (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(s=None), INVALID), (dict(ld=32), INVALID),
            (dict(fmt=1, g=P), INVALID), (dict(x=P + 8), ALIGN), (dict(q=P + 8), ALIGN),
            (dict(ld=68), ALIGN), (dict(g=P + 2), ALIGN)]


@pytest.mark.parametrize("change,code", BAD_ROWS)
def test_c_abi_refuses_bad_rows(change, code):
    lib = pkg().load()
    assert _quant(lib, **change) == code
    assert _dequant(lib, **change) == code


def test_c_abi_norm_refusals():
    lib = pkg().load()

    def call(x=P, xl=64, r=P, rl=64, w=P, eps=1e-6, dt=0, rows=4, cols=64, fmt=2, g=None, q=P, s=P):
        return lib.moe_fp8_ds_add_norm_quantize_mx(x, xl, r, rl, w, eps, dt, rows, cols, fmt, g, q, s, None)

    assert call(cols=32800, xl=32800, rl=32800) == INVALID
    assert call(eps=-1.0) == INVALID and call(eps=float("nan")) == INVALID
    assert call(rl=32) == INVALID and call(g=P) == INVALID and call(x=None) == INVALID
    assert call(w=P + 2) == ALIGN and call(r=P + 2) == ALIGN and call(rl=68) == ALIGN


def test_c_abi_product_refusals():
    lib = pkg().load()

    def dense(a=P, sa=P, b=P, sb=P, m=4, n=8, k=64, fmt=0, al=None, out=P, dt=0, ld=8):
        return lib.moe_fp8_ds_matmul_mx(a, sa, b, sb, m, n, k, fmt, al, out, dt, ld, None)

    for bad in (dict(m=-1), dict(m=(1 << 24) + 1), dict(n=0), dict(n=(1 << 18) + 1, ld=1 << 19), dict(k=0), dict(k=40),
                dict(k=1 << 21), dict(fmt=5), dict(dt=7), dict(a=None), dict(sa=None), dict(b=None), dict(sb=None),
                dict(out=None), dict(ld=7)):
        assert dense(**bad) == INVALID, bad
    for bad in (dict(a=P + 8), dict(b=P + 8), dict(out=P + 1), dict(al=P + 2), dict(dt=2, out=P + 2)):
        assert dense(**bad) == ALIGN, bad

    def experts(off=P, e=3, m=4):
        return lib.moe_fp8_ds_experts_matmul_mx(P, P, P, P, off, e, m, 8, 64, 0, None, P, 0, 8, None)

    assert experts(off=None) == INVALID and experts(e=0) == INVALID and experts(e=513) == INVALID
    assert experts(off=P + 2) == ALIGN


def test_c_abi_balance_refusals():
    lib = pkg().load()

    def call(x=P, dt=2, ld=16, ids=P, off=P, t=8, e=16, k=4, s=2, score=0, work=P, loss=P, counts=P):
        return lib.moe_fp8_ds_balance_loss(x, dt, ld, ids, off, t, e, k, s, score, 1.0, work, loss, counts, None)

    for bad in (dict(t=-1), dict(e=0), dict(e=1025, ld=2000), dict(k=0), dict(k=17), dict(s=0), dict(score=2), dict(dt=4),
                dict(ld=15), dict(off=None), dict(x=None), dict(ids=None), dict(work=None), dict(loss=None), dict(counts=None)):
        assert call(**bad) == INVALID, bad
    assert call(x=P + 2) == ALIGN and call(work=P + 4) == ALIGN
    assert lib.moe_fp8_ds_balance_loss_work_bytes(8, 16, 0) == 0
    # a run of tokens and a sequence each may need a slot of sums and counts
    assert lib.moe_fp8_ds_balance_loss_work_bytes(1000, 16, 5) >= (1 + 5) * 16 * 8


def test_good_arguments_reach_the_device_check():
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    lib = pkg().load()
    assert _quant(lib) == NO_DEVICE and _dequant(lib) == NO_DEVICE and _quant(lib, rows=0, x=None) == NO_DEVICE


def test_binding_refuses_cpu_tensors_and_unknown_names():
    m = pkg()
    x = torch.zeros(4, 64)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.float8_e4m3fn)
    for call in (lambda: m.quantize_mx(x), lambda: m.dequantize_mx(q, s), lambda: m.add_rmsnorm_quantize_mx(x),
                 lambda: m.matmul_mx(q, s, q, s), lambda: m.experts_matmul_mx(q, s, q[None], s[None], torch.zeros(2)),
                 lambda: m.balance_loss(x, torch.zeros(4, 2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: m.quantize_mx(x, "fp4"), lambda: m.matmul_mx(q, s, q, s, None), lambda: m.dequantize_mx(q, s, "e2m1")):
        with pytest.raises(ValueError, match="fmt"):
            call()
