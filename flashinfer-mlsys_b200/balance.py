"""The router's balance loss and per-expert counts, with gradients.

DeepSeek-V3's sequence-wise balance loss over the routing logits and the
experts that ``route`` selected, for training next to the layer's routing. It
runs in ``libmoe_fp8_ds.so`` on the current CUDA stream; there is no fallback.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from .mx import _bad, _cuda, _run

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCORES = {"sigmoid": 0, "softmax": 1}
MAX_EXPERTS = 1024
MAX_TOKENS = 1 << 24


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, offsets, coeff, score):
        loss, counts = _forward(logits, ids, offsets, coeff, score)
        ctx.save_for_backward(logits, ids, offsets, counts)
        ctx.args = coeff, score
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None
        if torch.is_grad_enabled():  # create_graph: the gradient's own gradient is not there
            raise RuntimeError("balance_loss can be differentiated once only")
        logits, ids, offsets, counts = ctx.saved_tensors
        coeff, score = ctx.args
        T, E = logits.shape
        dev = logits.device
        grad_loss = grad_loss.contiguous()
        grad = torch.empty((T, E), dtype=logits.dtype, device=dev)
        _run(dev, "moe_fp8_ds_balance_loss_backward", logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0),
             ids.data_ptr(), None if offsets is None else offsets.data_ptr(), T, E, ids.shape[1], counts.shape[0], score,
             coeff, counts.data_ptr(), grad_loss.data_ptr(), grad.data_ptr())
        return grad, None, None, None, None


def _forward(logits, ids, offsets, coeff, score):
    T, E = logits.shape
    S = 1 if offsets is None else offsets.shape[0] - 1
    dev = logits.device
    work = torch.empty(_lib.load().moe_fp8_ds_balance_loss_work_bytes(T, E, S), dtype=torch.uint8, device=dev)
    loss = torch.empty(S, dtype=torch.float32, device=dev)
    counts = torch.empty((S, E), dtype=torch.int32, device=dev)
    _run(dev, "moe_fp8_ds_balance_loss", logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), ids.data_ptr(),
         None if offsets is None else offsets.data_ptr(), T, E, ids.shape[1], S, score, coeff, work.data_ptr(),
         loss.data_ptr(), counts.data_ptr())
    return loss, counts


def balance_loss(routing_logits: torch.Tensor, topk_ids: torch.Tensor, seq_offsets: torch.Tensor | None = None,
                 coeff: float = 1e-4, score_func: str = "sigmoid"):
    """Balance loss of every sequence and its per-expert counts.

    With T_s tokens in sequence s, K slots a token and E experts:
    ``f_i = E / (K T_s) * counts[s, i]``, ``p_ti = score(l_ti) / sum_j
    score(l_tj)`` and ``loss[s] = coeff * sum_i f_i * mean_t p_ti``.

    * routing_logits: [T, E] float32, bf16 or fp16 (E <= 1024, rows any stride
      apart); the loss can be differentiated with respect to it once, in reverse
      mode (another derivative raises ``RuntimeError``); f is constant
    * topk_ids: int32 [T, K] (``route``'s ids). Ids outside [0, E) are not
      counted, an id that occurs twice counts twice
    * seq_offsets: int32 [S + 1] on the device, not decreasing: sequence s is
      tokens seq_offsets[s] .. seq_offsets[s + 1] - 1. None: one sequence
    * score_func: "sigmoid" (DeepSeek-V3) or "softmax"

    Returns (loss float32 [S], counts int32 [S, E]). Scores are within 5
    float32 steps of the exact ones (softmax: for the float32 difference to the
    row's largest logit). An empty sequence has loss 0; tokens of no sequence
    count nowhere and get a zero gradient; a token whose scores vanish in float32
    (sigmoids of logits under -87) has p = 0. Offsets that decrease give undefined
    numbers, not an access out of range. ``counts.sum(0)`` is what a bias update of
    the no-aux router needs."""
    dev = _cuda(routing_logits, "routing_logits")
    _cuda(topk_ids, "topk_ids")
    if routing_logits.dim() != 2 or topk_ids.dim() != 2:
        _bad("routing_logits and topk_ids must be 2-D")
    if routing_logits.dtype not in _DTYPES:
        _bad(f"routing_logits must be float32, bfloat16 or float16, got {routing_logits.dtype}")
    T, E = routing_logits.shape
    if not 1 <= E <= MAX_EXPERTS:
        _bad(f"1..{MAX_EXPERTS} experts, got {E}")
    if T > MAX_TOKENS:
        _bad(f"at most {MAX_TOKENS} tokens, got {T}")
    if topk_ids.dtype != torch.int32 or topk_ids.shape[0] != T or not 1 <= topk_ids.shape[1] <= E:
        _bad(f"topk_ids must be int32 [{T}, 1..{E}], got {topk_ids.dtype} {tuple(topk_ids.shape)}")
    if topk_ids.device != dev:
        _bad(f"topk_ids must be on {dev}")
    if not topk_ids.is_contiguous():
        _bad("topk_ids must be contiguous")
    ld, inner = routing_logits.stride()
    if T and ((inner != 1 and E != 1) or (T > 1 and ld < E)):
        _bad("routing_logits' rows must be contiguous")
    score = _SCORES.get(score_func)
    if score is None:
        _bad(f"score_func must be one of {sorted(_SCORES)}, got {score_func!r}")
    if seq_offsets is not None:
        _cuda(seq_offsets, "seq_offsets")
        if seq_offsets.dtype != torch.int32 or seq_offsets.dim() != 1 or not 2 <= seq_offsets.shape[0] <= MAX_TOKENS:
            _bad(f"seq_offsets must be int32 [sequences + 1], got {seq_offsets.dtype} {tuple(seq_offsets.shape)}")
        if seq_offsets.device != dev:
            _bad(f"seq_offsets must be on {dev}")
        if not seq_offsets.is_contiguous():
            _bad("seq_offsets must be contiguous")
    if forward_ad.unpack_dual(routing_logits).tangent is not None:
        raise RuntimeError("balance_loss has no forward-mode derivative")
    if routing_logits.requires_grad and torch.is_grad_enabled():
        return _BalanceLoss.apply(routing_logits, topk_ids, seq_offsets, float(coeff), score)
    return _forward(routing_logits, topk_ids, seq_offsets, float(coeff), score)
