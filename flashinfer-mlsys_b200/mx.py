"""Microscaled formats: quantisation, residual + RMSNorm + quantisation, and
the products that read them, for torch tensors.

Formats (``fmt``): values in blocks along a row, one scale a block, as the
block-scaled tensor cores read them.

* ``"nvfp4"``: e2m1 values, blocks of 16, e4m3 scales, and one float32 scale of
  the tensor (``global_scale``, a 1-element CUDA tensor; None = 1)
* ``"mxfp4"``: e2m1 values, blocks of 32, e8m0 (power of two) scales
* ``"mxfp8"``: e4m3 values, blocks of 32, e8m0 scales

Packed data is ``torch.uint8 [rows, cols / 2]`` for the 4-bit formats (even
column in the low half of a byte) and ``torch.float8_e4m3fn [rows, cols]`` for
mxfp8; scales are ``torch.float8_e4m3fn [rows, cols / 16]`` (nvfp4) or
``torch.float8_e8m0fnu [rows, cols / 32]``. ``cols`` is a multiple of 32.

Every call runs in ``libmoe_fp8_ds.so`` on the current CUDA stream of the
tensors' device, keeps no state and needs no workspace, so calls may overlap
on different streams and be captured into CUDA graphs. There is no fallback:
bad arguments raise ``ValueError``, a failing call raises ``MoeError``. None of
them is differentiable: results carry no gradient, and a tensor that a call has
written cannot be used by an earlier graph's backward pass. Outputs must not
share memory with other arguments.
"""
from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .binding import _stream

_Tensor = torch.Tensor
_current_device = torch._C._cuda_getDevice
_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu

# fmt -> (C ABI code, packed dtype, values per stored element, scale dtype, block)
_FORMATS = {
    "nvfp4": (0, torch.uint8, 2, _E4M3, 16),
    "mxfp4": (1, torch.uint8, 2, _E8M0, 32),
    "mxfp8": (2, _E4M3, 1, _E8M0, 32),
}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_ROWS = 1 << 24
MAX_COLS = 1 << 20
MAX_N = 1 << 18
MAX_EXPERTS = 512
MAX_NORM_COLS = 32768

# The checks below build their messages only when they fail: these calls are
# short, and formatting took longer than the kernels of a decode step.


def _bad(msg):
    raise ValueError(msg)


def _run(dev, name, *args):
    """Calls a C-ABI function with `dev` current on its current stream."""
    fn = getattr(_lib._lib or _lib.load(), name)
    if dev.index == _current_device():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        _lib.check(rc, name)


def _wrote(t):
    """Counts a version of a tensor of the caller's that a call has written, so
    that autograd refuses a backward pass that would read it as it was (0.3 us)."""
    if t is not None and not t.is_inference():
        increment_version(t)


def _format(fmt):
    f = _FORMATS.get(fmt) if isinstance(fmt, str) else None
    return f or _bad(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")


def _cuda(t, name):
    if not isinstance(t, _Tensor):
        _bad(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        _bad(f"{name} must be a CUDA tensor")
    return t.device


def _matrix(t, name, dev, dtype=None, shape=None):
    """A 2-D bf16, fp16 or fp32 tensor on `dev` whose rows are contiguous and
    16-byte aligned (any row stride); returns (dtype code, row stride)."""
    if not isinstance(t, _Tensor) or t.device != dev:
        _cuda(t, name)
        _bad(f"{name} must be on {dev}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        _bad(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        _bad(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2:
        _bad(f"{name} must be 2-D, got {t.dim()}-D")
    rows, cols = t.shape
    if shape is not None and (rows, cols) != shape:
        _bad(f"{name} must have shape {shape}, got {(rows, cols)}")
    ld, inner = t.stride()
    if rows and cols:
        if inner != 1 and cols != 1:
            _bad(f"{name}'s rows must be contiguous")
        if rows == 1:
            ld = cols
        elif ld < cols:
            _bad(f"{name}'s rows must not overlap")
        if t.data_ptr() % 16 or (rows > 1 and ld * (4 if code == 2 else 2) % 16):
            _bad(f"{name}'s rows must be 16-byte aligned")
    return code, ld


def _exact(t, name, dtype, shape, dev):
    """A contiguous tensor of the given type, shape and device."""
    if (not isinstance(t, _Tensor) or t.dtype != dtype or t.shape != shape or t.device != dev
            or not t.is_contiguous()):
        _cuda(t, name)
        if t.dtype != dtype:
            _bad(f"{name} must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            _bad(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.device != dev:
            _bad(f"{name} must be on {dev}")
        _bad(f"{name} must be contiguous")
    return t.data_ptr()


def _exact16(t, name, dtype, shape, dev):
    p = _exact(t, name, dtype, shape, dev)
    if p % 16:
        _bad(f"{name} must be 16-byte aligned")
    return p


def _scalar(t, name, dev):
    """Address of a float32 tensor of one element, or None."""
    if t is None:
        return None
    if not isinstance(t, _Tensor) or t.dtype != torch.float32 or t.numel() != 1 or t.device != dev:
        _cuda(t, name)
        if t.device != dev:
            _bad(f"{name} must be on {dev}")
        _bad(f"{name} must be a float32 tensor of one element")
    return t.data_ptr()


def _global_scale(t, fmt, dev):
    if t is not None and fmt != "nvfp4":
        _bad(f"global_scale belongs to nvfp4, not to {fmt}")
    return _scalar(t, "global_scale", dev)


def _size(rows, cols, limit=MAX_COLS):
    if cols % 32 or not 0 < cols <= limit:
        _bad(f"the width must be a multiple of 32 in 32..{limit}, got {cols}")
    if rows > MAX_ROWS:
        _bad(f"at most {MAX_ROWS} rows, got {rows}")


def _packed_out(rows, cols, f, dev, out, out_scale):
    _, qt, per, st, block = f
    if out is None:
        out = torch.empty((rows, cols // per), dtype=qt, device=dev)
        qp = out.data_ptr()
    else:
        qp = _exact16(out, "out", qt, (rows, cols // per), dev)
    if out_scale is None:
        out_scale = torch.empty((rows, cols // block), dtype=st, device=dev)
        sp = out_scale.data_ptr()
    else:
        sp = _exact(out_scale, "out_scale", st, (rows, cols // block), dev)
    return out, out_scale, qp, sp


def quantize_mx(x: torch.Tensor, fmt: str = "nvfp4", global_scale: torch.Tensor | None = None,
                out: torch.Tensor | None = None, out_scale: torch.Tensor | None = None):
    """x [rows, cols] (bf16, fp16 or fp32, rows any stride apart) -> (packed
    values, scales). Float32 steps, every rounding to nearest even:

    * nvfp4: ``s = e4m3(min(448, amax / (6 g)))``, ``q = e2m1(x / (s g))`` (0
      where ``s g`` is 0), ``g`` = global_scale (positive and finite; the
      usual choice is amax of the tensor / (448 * 6))
    * mxfp4, mxfp8: ``s = 2 ** clamp(floor(log2(amax)) - emax, -127, 127)`` with
      emax 2 or 8, ``q = round(x / s)``, saturating

    A block with an infinity or a NaN gets a NaN scale (its values read back
    as NaN) and zeros."""
    f = _format(fmt)
    dev = _cuda(x, "x")
    code, ld = _matrix(x, "x", dev)
    rows, cols = x.shape
    _size(rows, cols)
    g = _global_scale(global_scale, fmt, dev)
    given, given_scale = out, out_scale
    out, out_scale, qp, sp = _packed_out(rows, cols, f, dev, out, out_scale)
    if rows:
        _run(dev, "moe_fp8_ds_quantize_mx", x.data_ptr(), code, rows, cols, ld, f[0], g, qp, sp)
        _wrote(given)
        _wrote(given_scale)
    return out, out_scale


def _packed_in(q, scale, f, dev, names, lead=()):
    """Checks packed data and its scales (leading dims `lead`); returns (rows, cols, addresses)."""
    _, qt, per, st, block = f
    if not isinstance(q, _Tensor) or q.dim() != 2 + len(lead):
        _cuda(q, names[0])
        _bad(f"{names[0]} must be {2 + len(lead)}-D, got {q.dim()}-D")
    rows, cols = q.shape[-2], q.shape[-1] * per
    _size(rows, cols)
    qp = _exact16(q, names[0], qt, (*lead, rows, cols // per), dev)
    return rows, cols, qp, _exact(scale, names[1], st, (*lead, rows, cols // block), dev)


def dequantize_mx(q: torch.Tensor, scale: torch.Tensor, fmt: str = "nvfp4", global_scale: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that packed data stands for, [rows, cols]: value * scale *
    global_scale in float32, rounded once to ``dtype`` (bf16, fp16 or fp32)."""
    f = _format(fmt)
    dev = _cuda(q, "q")
    rows, cols, qp, sp = _packed_in(q, scale, f, dev, ("q", "scale"))
    g = _global_scale(global_scale, fmt, dev)
    given = out
    if out is None:
        code, ld = _DTYPES.get(dtype), cols
        if code is None:
            _bad(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        out = torch.empty((rows, cols), dtype=dtype, device=dev)
    else:
        code, ld = _matrix(out, "out", dev, None, (rows, cols))
    if rows:
        _run(dev, "moe_fp8_ds_dequantize_mx", qp, sp, rows, cols, f[0], g, code, out.data_ptr(), ld)
        _wrote(given)
    return out


def add_rmsnorm_quantize_mx(x: torch.Tensor, residual: torch.Tensor | None = None,
                            norm_weight: torch.Tensor | None = None, eps: float = 1e-6, fmt: str = "mxfp8",
                            global_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                            out_scale: torch.Tensor | None = None):
    """``add_rmsnorm_quantize`` for any width up to 32768 and for the
    microscaled formats: ``h = residual + x`` rounded to x's type (written back
    into ``residual``), ``y = h / sqrt(mean(h^2) + eps) * norm_weight``, then
    the quantisation of y as in ``quantize_mx`` (y is rounded to odd in float32,
    so a value lands where the exact y would; the mean is taken in float64, so h
    may have any size; a y of float32's largest number or more counts as infinite). ``residual`` None: h = x;
    ``norm_weight`` None: y = h. All three tensors have x's type. Returns
    (packed values, scales)."""
    f = _format(fmt)
    dev = _cuda(x, "x")
    code, ld = _matrix(x, "x", dev)
    rows, cols = shape = x.shape
    _size(rows, cols, MAX_NORM_COLS)
    eps = float(eps)
    if not eps >= 0.0:
        _bad("eps must be >= 0")
    rp, rld, wp = None, 0, None
    if residual is not None:
        rld = _matrix(residual, "residual", dev, x.dtype, shape)[1]
        rp = residual.data_ptr()
    if norm_weight is not None:
        wp = _exact16(norm_weight, "norm_weight", x.dtype, (cols,), dev)
    g = _global_scale(global_scale, fmt, dev)
    given, given_scale = out, out_scale
    out, out_scale, qp, sp = _packed_out(rows, cols, f, dev, out, out_scale)
    if rows:
        _run(dev, "moe_fp8_ds_add_norm_quantize_mx", x.data_ptr(), ld, rp, rld, wp, eps, code, rows, cols, f[0], g, qp, sp)
        _wrote(residual)
        _wrote(given)
        _wrote(given_scale)
    return out, out_scale


def _product_out(m, n, dev, out, out_dtype, make):
    if out is None:
        code = _DTYPES.get(out_dtype)
        if code is None:
            _bad(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        return make((m, n), dtype=out_dtype, device=dev), code, n
    if not isinstance(out, _Tensor) or out.device != dev:
        _cuda(out, "out")
        _bad(f"out must be on {dev}")
    code = _DTYPES.get(out.dtype)
    if code is None:
        _bad(f"out must be bfloat16, float16 or float32, got {out.dtype}")
    if out.shape != (m, n):
        _bad(f"out must have shape {(m, n)}, got {tuple(out.shape)}")
    ld, inner = out.stride()
    if m and ((inner != 1 and n != 1) or (m > 1 and ld < n)):
        _bad("out's rows must be contiguous")
    return out, code, ld if m > 1 else n


def _same_width(k, kb, m, n):
    if k != kb:
        _bad(f"a and b must have the same width, got {k} and {kb}")
    if not 0 < n <= MAX_N:
        _bad(f"b must have 1..{MAX_N} rows, got {n}")


def matmul_mx(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, fmt: str = "nvfp4",
              alpha: torch.Tensor | None = None, out: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``out = alpha * A @ B.T`` of two microscaled matrices: a [m, k] and b
    [n, k], packed as ``quantize_mx`` returns them. float32 sums on the
    block-scaled tensor cores, rounded once to ``out``'s type (bf16, fp16 or
    fp32; its rows may lie any stride apart). ``alpha``: float32 tensor of one
    element, for nvfp4 the product of the two global scales; None = 1. e4m3
    scales must not be negative."""
    f = _format(fmt)
    dev = _cuda(a, "a")
    m, k, ap, asp = _packed_in(a, a_scale, f, dev, ("a", "a_scale"))
    n, kb, bp, bsp = _packed_in(b, b_scale, f, dev, ("b", "b_scale"))
    _same_width(k, kb, m, n)
    al = _scalar(alpha, "alpha", dev)
    given = out
    out, code, ld = _product_out(m, n, dev, out, out_dtype, torch.empty)
    if m:
        _run(dev, "moe_fp8_ds_matmul_mx", ap, asp, bp, bsp, m, n, k, f[0], al, out.data_ptr(), code, ld)
        _wrote(given)
    return out


def experts_matmul_mx(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                      expert_offsets: torch.Tensor, fmt: str = "nvfp4", alpha: torch.Tensor | None = None,
                      out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``matmul_mx`` with one weight matrix per run of rows, the experts'
    products of rows sorted by expert: rows ``expert_offsets[e]`` ..
    ``expert_offsets[e + 1] - 1`` of a use ``b[e]`` (b [experts, n, k]) and
    ``alpha[e]`` (float32 [experts] or None). expert_offsets: int32 [experts +
    1] on the device, not decreasing (values are kept inside [0, m]); nothing is
    copied to the host. Rows outside the runs are left as they were (zero where
    ``out`` is None)."""
    f = _format(fmt)
    dev = _cuda(a, "a")
    m, k, ap, asp = _packed_in(a, a_scale, f, dev, ("a", "a_scale"))
    _cuda(b, "b")
    if b.dim() != 3:
        _bad(f"b must be 3-D, got {b.dim()}-D")
    e = b.shape[0]
    if not 1 <= e <= MAX_EXPERTS:
        _bad(f"b must hold 1..{MAX_EXPERTS} experts, got {e}")
    n, kb, bp, bsp = _packed_in(b, b_scale, f, dev, ("b", "b_scale"), (e,))
    _same_width(k, kb, m, n)
    op = _exact(expert_offsets, "expert_offsets", torch.int32, (e + 1,), dev)
    al = None if alpha is None else _exact(alpha, "alpha", torch.float32, (e,), dev)
    given = out
    out, code, ld = _product_out(m, n, dev, out, out_dtype, torch.zeros)
    if m:
        _run(dev, "moe_fp8_ds_experts_matmul_mx", ap, asp, bp, bsp, op, e, m, n, k, f[0], al, out.data_ptr(), code, ld)
        _wrote(given)
    return out
