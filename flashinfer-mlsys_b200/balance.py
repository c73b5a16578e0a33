"""The router's balance loss and per-expert counts, with gradients.

DeepSeek-V3's sequence-wise balance loss over the routing logits and the
experts that ``route`` selected, for training next to the layer's routing. It
runs in ``libmoe_fp8_ds.so`` on the current CUDA stream; there is no fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from .binding import _call, _need, _stream

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCORES = {"sigmoid": 0, "softmax": 1}
MAX_EXPERTS = 1024
MAX_TOKENS = 1 << 24


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, offsets, coeff, score):
        T, E = logits.shape
        S = 1 if offsets is None else offsets.shape[0] - 1
        dev = logits.device
        lib = _lib.load()
        work = torch.empty(lib.moe_fp8_ds_balance_loss_work_bytes(T, E, S), dtype=torch.uint8, device=dev)
        loss = torch.empty(S, dtype=torch.float32, device=dev)
        counts = torch.empty((S, E), dtype=torch.int32, device=dev)
        off = None if offsets is None else offsets.data_ptr()
        rc = _call(dev, lib.moe_fp8_ds_balance_loss, logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0),
                   ids.data_ptr(), off, T, E, ids.shape[1], S, score, coeff, work.data_ptr(), loss.data_ptr(),
                   counts.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_balance_loss")
        ctx.save_for_backward(logits, ids, offsets, counts)
        ctx.coeff, ctx.score = coeff, score
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None
        logits, ids, offsets, counts = ctx.saved_tensors
        T, E = logits.shape
        dev = logits.device
        grad_loss = grad_loss.contiguous()
        grad = torch.empty((T, E), dtype=logits.dtype, device=dev)
        off = None if offsets is None else offsets.data_ptr()
        rc = _call(dev, _lib.load().moe_fp8_ds_balance_loss_backward, logits.data_ptr(), _DTYPES[logits.dtype],
                   logits.stride(0), ids.data_ptr(), off, T, E, ids.shape[1], counts.shape[0], ctx.score, ctx.coeff,
                   counts.data_ptr(), grad_loss.data_ptr(), grad.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc, "moe_fp8_ds_balance_loss_backward")
        return grad, None, None, None, None


def balance_loss(routing_logits: torch.Tensor, topk_ids: torch.Tensor, seq_offsets: torch.Tensor | None = None,
                 coeff: float = 1e-4, score_func: str = "sigmoid"):
    """Balance loss of every sequence and its per-expert counts.

    With T_s tokens in sequence s, K slots a token and E experts:
    ``f_i = E / (K T_s) * counts[s, i]``, ``p_ti = score(l_ti) / sum_j
    score(l_tj)`` and ``loss[s] = coeff * sum_i f_i * mean_t p_ti``.

    * routing_logits: [T, E] float32, bf16 or fp16 (E <= 1024, rows any stride
      apart); the loss is differentiable with respect to it, f is constant
    * topk_ids: int32 [T, K] (``route``'s ids). Ids outside [0, E) are not
      counted, an id that occurs twice counts twice
    * seq_offsets: int32 [S + 1] on the device, not decreasing: sequence s is
      tokens seq_offsets[s] .. seq_offsets[s + 1] - 1. None: one sequence
    * score_func: "sigmoid" (DeepSeek-V3) or "softmax"

    Returns (loss float32 [S], counts int32 [S, E]). An empty sequence has loss
    0; tokens of no sequence count nowhere and get a zero gradient; a token
    whose scores sum to zero in float32 has p = 0. ``counts.sum(0)`` is what a
    bias update of the no-aux router needs."""
    _need(isinstance(routing_logits, torch.Tensor) and routing_logits.is_cuda, "routing_logits must be a CUDA tensor")
    _need(isinstance(topk_ids, torch.Tensor) and topk_ids.is_cuda, "topk_ids must be a CUDA tensor")
    _need(routing_logits.dim() == 2 and topk_ids.dim() == 2, "routing_logits and topk_ids must be 2-D")
    _need(routing_logits.dtype in _DTYPES, f"routing_logits must be float32, bfloat16 or float16, got {routing_logits.dtype}")
    T, E = routing_logits.shape
    _need(1 <= E <= MAX_EXPERTS, f"1..{MAX_EXPERTS} experts, got {E}")
    _need(T <= MAX_TOKENS, f"at most {MAX_TOKENS} tokens")
    dev = routing_logits.device
    _need(topk_ids.dtype == torch.int32 and topk_ids.shape[0] == T and 1 <= topk_ids.shape[1] <= E,
          f"topk_ids must be int32 [{T}, 1..{E}], got {topk_ids.dtype} {tuple(topk_ids.shape)}")
    _need(topk_ids.device == dev, f"topk_ids must be on {dev}")
    _need(topk_ids.is_contiguous(), "topk_ids must be contiguous")
    _need(T == 0 or ((E == 1 or routing_logits.stride(1) == 1) and (T == 1 or routing_logits.stride(0) >= E)),
          "routing_logits' rows must be contiguous")
    _need(score_func in _SCORES, f"score_func must be one of {sorted(_SCORES)}, got {score_func!r}")
    if seq_offsets is not None:
        _need(isinstance(seq_offsets, torch.Tensor) and seq_offsets.dtype == torch.int32 and seq_offsets.dim() == 1
              and seq_offsets.shape[0] >= 2, "seq_offsets must be int32 [sequences + 1]")
        _need(seq_offsets.device == dev, f"seq_offsets must be on {dev}")
        _need(seq_offsets.is_contiguous(), "seq_offsets must be contiguous")
        _need(seq_offsets.shape[0] <= MAX_TOKENS, f"fewer than {MAX_TOKENS} sequences")
    return _BalanceLoss.apply(routing_logits, topk_ids, seq_offsets, float(coeff), _SCORES[score_func])
