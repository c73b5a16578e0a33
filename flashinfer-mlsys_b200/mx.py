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
bad arguments raise ``ValueError``, a failing call raises ``MoeError``.
"""
from __future__ import annotations

import torch

from . import _lib
from .binding import _call, _need, _stream

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


def _format(fmt):
    f = _FORMATS.get(fmt) if isinstance(fmt, str) else None
    _need(f is not None, f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
    return f


def _is(t, name):
    _need(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _need(t.is_cuda, f"{name} must be a CUDA tensor")


def _matrix(t, name, dev=None, dtype=None, shape=None):
    """A 2-D bf16, fp16 or fp32 CUDA tensor whose rows are contiguous and
    16-byte aligned (any row stride); returns its dtype code."""
    _is(t, name)
    _need(t.dim() == 2, f"{name} must be 2-D, got {t.dim()}-D")
    code = _DTYPES.get(t.dtype)
    _need(code is not None, f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if dtype is not None:
        _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None:
        _need(tuple(t.shape) == shape, f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if dev is not None:
        _need(t.device == dev, f"{name} must be on {dev}")
    if t.numel():
        rows, cols = t.shape
        _need(cols == 1 or t.stride(1) == 1, f"{name}'s rows must be contiguous")
        _need(rows == 1 or t.stride(0) >= cols, f"{name}'s rows must not overlap")
        size = t.element_size()
        _need(t.data_ptr() % 16 == 0 and (rows == 1 or t.stride(0) * size % 16 == 0),
              f"{name}'s rows must be 16-byte aligned")
    return code


def _exact(t, name, dtype, shape, dev):
    """A contiguous tensor of the given type, shape and device."""
    _is(t, name)
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.device == dev, f"{name} must be on {dev}")
    _need(t.is_contiguous(), f"{name} must be contiguous")


def _scalar(t, name, dev, fmt=None):
    if t is None:
        return None
    _need(fmt is None or fmt == "nvfp4", f"{name} belongs to nvfp4, not to {fmt}")
    _is(t, name)
    _need(t.dtype == torch.float32 and t.numel() == 1, f"{name} must be a float32 tensor of one element")
    _need(t.device == dev, f"{name} must be on {dev}")
    return t.data_ptr()


def _width(cols, limit=MAX_COLS):
    _need(0 < cols <= limit and cols % 32 == 0, f"the width must be a multiple of 32 in 32..{limit}, got {cols}")


def _packed_out(rows, cols, f, dev, out, out_scale):
    _, qt, per, st, block = f
    if out is None:
        out = torch.empty((rows, cols // per), dtype=qt, device=dev)
    else:
        _exact(out, "out", qt, (rows, cols // per), dev)
        _need(out.data_ptr() % 16 == 0, "out must be 16-byte aligned")
    if out_scale is None:
        out_scale = torch.empty((rows, cols // block), dtype=st, device=dev)
    else:
        _exact(out_scale, "out_scale", st, (rows, cols // block), dev)
        _need(out_scale.data_ptr() % 2 == 0 or block != 16, "out_scale must be 2-byte aligned")
    return out, out_scale


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
    code = _matrix(x, "x")
    rows, cols = x.shape
    _width(cols)
    _need(rows <= MAX_ROWS, f"at most {MAX_ROWS} rows")
    dev = x.device
    g = _scalar(global_scale, "global_scale", dev, fmt)
    out, out_scale = _packed_out(rows, cols, f, dev, out, out_scale)
    if rows:
        rc = _call(dev, _lib.load().moe_fp8_ds_quantize_mx, x.data_ptr(), code, rows, cols, x.stride(0), f[0], g,
                   out.data_ptr(), out_scale.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_quantize_mx")
    return out, out_scale


def _packed_in(q, scale, f, dev, names, lead=()):
    """Checks packed data and its scales (leading dims `lead`); returns (rows, cols)."""
    _, qt, per, st, block = f
    _is(q, names[0])
    _need(q.dim() == 2 + len(lead), f"{names[0]} must be {2 + len(lead)}-D, got {q.dim()}-D")
    rows, cols = q.shape[-2], q.shape[-1] * per
    _width(cols)
    _exact(q, names[0], qt, (*lead, rows, cols // per), dev)
    _exact(scale, names[1], st, (*lead, rows, cols // block), dev)
    _need(q.data_ptr() % 16 == 0, f"{names[0]} must be 16-byte aligned")
    return rows, cols


def dequantize_mx(q: torch.Tensor, scale: torch.Tensor, fmt: str = "nvfp4", global_scale: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that packed data stands for, [rows, cols]: value * scale *
    global_scale in float32, rounded once to ``dtype`` (bf16, fp16 or fp32)."""
    f = _format(fmt)
    _is(q, "q")
    dev = q.device
    rows, cols = _packed_in(q, scale, f, dev, ("q", "scale"))
    _need(rows <= MAX_ROWS, f"at most {MAX_ROWS} rows")
    _need(f[4] != 16 or scale.data_ptr() % 2 == 0, "scale must be 2-byte aligned")
    g = _scalar(global_scale, "global_scale", dev, fmt)
    if out is None:
        _need(dtype in _DTYPES, f"dtype must be bfloat16, float16 or float32, got {dtype}")
        out = torch.empty((rows, cols), dtype=dtype, device=dev)
    code = _matrix(out, "out", dev, None, (rows, cols))
    if rows:
        rc = _call(dev, _lib.load().moe_fp8_ds_dequantize_mx, q.data_ptr(), scale.data_ptr(), rows, cols, f[0], g, code,
                   out.data_ptr(), out.stride(0), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_dequantize_mx")
    return out


def add_rmsnorm_quantize_mx(x: torch.Tensor, residual: torch.Tensor | None = None,
                            norm_weight: torch.Tensor | None = None, eps: float = 1e-6, fmt: str = "mxfp8",
                            global_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                            out_scale: torch.Tensor | None = None):
    """``add_rmsnorm_quantize`` for any width up to 32768 and for the
    microscaled formats: ``h = residual + x`` rounded to x's type (written back
    into ``residual``), ``y = h / sqrt(mean(h^2) + eps) * norm_weight`` in
    float32, then the quantisation of y as in ``quantize_mx``. ``residual``
    None: h = x; ``norm_weight`` None: y = h. All three tensors have x's type.
    Returns (packed values, scales)."""
    f = _format(fmt)
    code = _matrix(x, "x")
    rows, cols = x.shape
    _width(cols, MAX_NORM_COLS)
    _need(rows <= MAX_ROWS, f"at most {MAX_ROWS} rows")
    _need(float(eps) >= 0.0, "eps must be >= 0")
    dev = x.device
    if residual is not None:
        _matrix(residual, "residual", dev, x.dtype, (rows, cols))
    if norm_weight is not None:
        _exact(norm_weight, "norm_weight", x.dtype, (cols,), dev)
        _need(norm_weight.data_ptr() % 16 == 0, "norm_weight must be 16-byte aligned")
    g = _scalar(global_scale, "global_scale", dev, fmt)
    out, out_scale = _packed_out(rows, cols, f, dev, out, out_scale)
    if rows:
        rc = _call(dev, _lib.load().moe_fp8_ds_add_norm_quantize_mx, x.data_ptr(), x.stride(0),
                   None if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0),
                   None if norm_weight is None else norm_weight.data_ptr(), float(eps), code, rows, cols, f[0], g,
                   out.data_ptr(), out_scale.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_add_norm_quantize_mx")
    return out, out_scale


def _product_out(m, n, dev, out, out_dtype, make):
    if out is None:
        _need(out_dtype in _DTYPES, f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        return make((m, n), dtype=out_dtype, device=dev), _DTYPES[out_dtype]
    _is(out, "out")
    code = _DTYPES.get(out.dtype)
    _need(code is not None, f"out must be bfloat16, float16 or float32, got {out.dtype}")
    _need(tuple(out.shape) == (m, n), f"out must have shape {(m, n)}, got {tuple(out.shape)}")
    _need(out.device == dev, f"out must be on {dev}")
    _need(m == 0 or ((n == 1 or out.stride(1) == 1) and (m == 1 or out.stride(0) >= n)), "out's rows must be contiguous")
    return out, code


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
    _is(a, "a")
    dev = a.device
    m, k = _packed_in(a, a_scale, f, dev, ("a", "a_scale"))
    n, kb = _packed_in(b, b_scale, f, dev, ("b", "b_scale"))
    _need(k == kb, f"a and b must have the same width, got {k} and {kb}")
    _need(m <= MAX_ROWS and 0 < n <= MAX_N, f"a has at most {MAX_ROWS} rows and b 1..{MAX_N}")
    al = _scalar(alpha, "alpha", dev)
    out, code = _product_out(m, n, dev, out, out_dtype, torch.empty)
    if m:
        rc = _call(dev, _lib.load().moe_fp8_ds_matmul_mx, a.data_ptr(), a_scale.data_ptr(), b.data_ptr(),
                   b_scale.data_ptr(), m, n, k, f[0], al, out.data_ptr(), code, out.stride(0), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_matmul_mx")
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
    _is(a, "a")
    _is(b, "b")
    dev = a.device
    m, k = _packed_in(a, a_scale, f, dev, ("a", "a_scale"))
    _need(b.dim() == 3, f"b must be 3-D, got {b.dim()}-D")
    e = b.shape[0]
    _need(1 <= e <= MAX_EXPERTS, f"b must hold 1..{MAX_EXPERTS} experts, got {e}")
    n, kb = _packed_in(b, b_scale, f, dev, ("b", "b_scale"), (e,))
    _need(k == kb, f"a and b must have the same width, got {k} and {kb}")
    _need(m <= MAX_ROWS and 0 < n <= MAX_N, f"a has at most {MAX_ROWS} rows and b 1..{MAX_N}")
    _exact(expert_offsets, "expert_offsets", torch.int32, (e + 1,), dev)
    if alpha is not None:
        _exact(alpha, "alpha", torch.float32, (e,), dev)
    out, code = _product_out(m, n, dev, out, out_dtype, torch.zeros)
    if m:
        rc = _call(dev, _lib.load().moe_fp8_ds_experts_matmul_mx, a.data_ptr(), a_scale.data_ptr(), b.data_ptr(),
                   b_scale.data_ptr(), expert_offsets.data_ptr(), e, m, n, k, f[0],
                   None if alpha is None else alpha.data_ptr(), out.data_ptr(), code, out.stride(0), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_experts_matmul_mx")
    return out
