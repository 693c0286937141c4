"""A whole MoE layer for a few tokens in two kernels, router included.

The reference composes the layer from its operators (bench/bench_mlp.py:60-96: router matmul, topk, two ragged matmuls, reduce); at a handful of
tokens those launches, and the kernels' waits for one another, take longer than the weights of the active experts."""
import torch

from . import _lib
from .matmul import _status_word
from .moe import MoeLayerWeights
from .router import prepare_router_weight
from .tensor_details.layout import B200MXScaleLayout, B200MXValueLayout

MAX_TOKENS = 16


def moe_layer_tokens(x: torch.Tensor, wg: torch.Tensor, bg, lw: MoeLayerWeights, k: int) -> torch.Tensor:
    """x [T, d_model] bf16 or fp16, T <= 16 -> [T, d_model]: sum over the k experts with the largest router logits x wg + bg of
    softmax-weight * (SwiGLU(x W1 + b1) W2 + b2).

    wg [d_model, E] bf16 in the memory order of `prepare_router_weight` (else it is re-laid-out on every call), bg [E] or None; `lw` in the default
    layouts.  Router logits, all sums and what is between the two products are fp32 (a hidden row enters the second as two fp16 terms, 2^-23 of a value, however many
    tokens its expert has) and the result is rounded once: `moe_layer_forward` on `router_topk`'s selection rounds the logits (by default), the hidden rows and every
    expert's output to bf16 too.  Equal logits go to the lower
    expert.  A sum of more than 2^114 times the largest element of its row is infinite.  At most 256 experts, k <= 16, widths that are multiples of 32 up to 8192 (4096 for more than 8 tokens); NotImplementedError
    beyond.  Runs on the current stream of x's device, which has to hold all tensors; every call has a workspace of its own, so calls may overlap and
    be captured in CUDA graphs."""
    if not isinstance(x, torch.Tensor) or x.ndim != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("moe_layer_tokens: x is a [tokens, d_model] tensor of bf16 or fp16")
    if not x.is_cuda:
        raise ValueError("triton_b200 operators take CUDA tensors only (no CPU path)")
    T, d = x.shape
    E = lw.n_expts
    if wg.ndim != 2 or tuple(wg.shape) != (d, E):
        raise ValueError(f"moe_layer_tokens: wg is [{d}, {E}] for these tokens and experts, got {list(wg.shape)}")
    if wg.dtype != torch.bfloat16:
        raise ValueError(f"moe_layer_tokens: wg is bf16, got {wg.dtype} (prepare_router_weight casts it)")
    if bg is not None and (bg.ndim != 1 or bg.shape[0] != E or bg.stride(0) != 1 or bg.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
        raise ValueError(f"moe_layer_tokens: bg is a contiguous vector of {E} floats")
    if not 0 < k <= E:
        raise ValueError(f"moe_layer_tokens: k = {k} of {E} experts")
    for w, s, b, K, what in ((lw.w1, lw.w1_scale, lw.b1, d, "W1"), (lw.w2, lw.w2_scale, lw.b2, lw.b1.shape[1] // 2, "W2")):
        if w is None or type(w.storage.layout) is not B200MXValueLayout or type(s.storage.layout) is not B200MXScaleLayout:
            raise NotImplementedError(f"moe_layer_tokens: {what} has to be in the default layouts (B200MXValueLayout / B200MXScaleLayout)")
        if len(w.shape) != 3 or w.shape[0] != E or w.shape[1] != K or tuple(b.shape) != (E, w.shape[2]) or b.stride(1) != 1:
            raise ValueError(f"moe_layer_tokens: {what} is {list(w.shape)} with a bias of {list(b.shape)}; expected [{E}, {K}, N] and [{E}, N]")
    if lw.w1.shape[2] % 2 or lw.w2.shape[2] != d:
        raise ValueError(f"moe_layer_tokens: W1 {list(lw.w1.shape)} and W2 {list(lw.w2.shape)} are no layer of width {d}")
    wg = prepare_router_weight(wg)
    if wg.data_ptr() % 16:
        wg = wg.t().clone(memory_format=torch.contiguous_format).t()
    return _lib.host().moe_tokens(x, wg, bg, k, (lw.w1.storage.data, lw.w1_scale.storage.data, lw.b1),
                                  (lw.w2.storage.data, lw.w2_scale.storage.data, lw.b2), lw.w1.shape[2] // 2, lw.alpha, lw.limit,
                                  _status_word(x.device))
