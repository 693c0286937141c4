"""A dense projection that all requests share, with each request's own low-rank adapter beside it.

The reference's `matmul` multiplies the rows of a ragged batch by their group's matrix (matmul.py:245-766); serving fine-tuned models puts one shared
matrix under all rows and a small product of two thin matrices, another per request, on top.  `matmul_lora` does both in two kernels (one for a single token's adapter of up to 16 ranks)."""
import itertools
from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib
from .matmul import _status_word

PIECE = 16                  # ranks that go together; an adapter's rank is padded with zeros to a multiple of it
MAX_RANK = 1024


@dataclass
class LoraAdapters:
    """Adapters as the kernels read them (`prepare_lora_adapters`); adapter i has the pieces first[i] .. first[i + 1]."""
    a: torch.Tensor         # [pieces * 16, d_in rounded up to 8]
    b: torch.Tensor         # [pieces, d_out rounded up to 128 / 8, 2, 8, 8]
    first: torch.Tensor     # int32 [adapters + 1]
    scale: torch.Tensor     # fp32 [adapters]
    ranks: tuple[int, ...]
    max_pieces: int         # of one adapter
    d_in: int
    d_out: int
    ranks_device: torch.Tensor | None = None        # `ranks` as int32 [adapters]; None: whole pieces

    @property
    def n_adapters(self):
        return len(self.ranks)


def prepare_lora_adapters(a: Sequence[torch.Tensor], b: Sequence[torch.Tensor], scale: Sequence[float]) -> LoraAdapters:
    """Adapters a[i] [d_in, rank_i] and b[i] [rank_i, d_out], scaled by scale[i], laid out once for `matmul_lora`: bf16 or fp16, all on one
    device; ranks may differ (1 to 1024).  Values of b have to be finite: a block of tokens multiplies the b of adapters that it does
    not have by zero."""
    if not len(a) == len(b) == len(scale) or len(a) == 0:
        raise ValueError(f"prepare_lora_adapters: as many a, b and scales, one at least (got {len(a)}, {len(b)}, {len(scale)})")
    d_in, d_out, dtype, device = a[0].shape[0], b[0].shape[1], a[0].dtype, a[0].device
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("prepare_lora_adapters: adapters are bf16 or fp16")
    for i, (ai, bi) in enumerate(zip(a, b)):
        r = ai.shape[-1]
        if tuple(ai.shape) != (d_in, r) or tuple(bi.shape) != (r, d_out) or {ai.dtype, bi.dtype} != {dtype} or {ai.device, bi.device} != {device}:
            raise ValueError(f"prepare_lora_adapters: adapter {i} is {list(ai.shape)} x {list(bi.shape)} in {ai.dtype} and {bi.dtype} on {ai.device} and {bi.device}; "
                             f"expected [{d_in}, r] x [r, {d_out}] in {dtype} on {device}")
        if not 1 <= r <= MAX_RANK:
            raise ValueError(f"prepare_lora_adapters: adapter {i} has rank {r}; ranks are 1 to {MAX_RANK}")
    ranks = tuple(ai.shape[1] for ai in a)
    pieces = [-(-r // PIECE) for r in ranks]
    first = [0, *itertools.accumulate(pieces)]
    rows, groups = -(-d_in // 8) * 8, -(-d_out // 128) * 16

    def stacked(parts, width, padded):                         # ranks one below the other, each adapter's up to a multiple of 16
        fill = {n: torch.zeros((n, width), dtype=dtype, device=device) for n in {-r % PIECE for r in ranks}}
        out = torch.zeros((first[-1] * PIECE, padded), dtype=dtype, device=device)
        out[:, :width] = torch.cat([t for part, r in zip(parts, ranks) for t in (part, fill[-r % PIECE])])
        return out

    pa = stacked([ai.t() for ai in a], d_in, rows)
    pb = stacked(b, d_out, groups * 8)
    if not bool(torch.isfinite(pb).all()):
        wrong = [i for i, bi in enumerate(b) if not bool(torch.isfinite(bi).all())]
        raise ValueError(f"prepare_lora_adapters: b of adapters {wrong} has values that are not finite")
    pb = pb.view(first[-1], 2, 8, groups, 8).permute(0, 3, 1, 4, 2).contiguous()
    counts = torch.tensor([*first, *ranks], dtype=torch.int32, device=device)
    return LoraAdapters(pa, pb, counts[:len(first)], torch.tensor([float(s) for s in scale], dtype=torch.float32, device=device), ranks, max(pieces), d_in, d_out,
                        counts[len(first):])


def prepare_projection_weight(w: torch.Tensor) -> torch.Tensor:
    """-> w as `matmul_lora` reads it: logical shape [d_in, d_out] kept, memory [d_out, d_in] with d_in contiguous and rows 16-byte aligned.  A weight that
    already has that memory order is returned as it is; do this once per weight, not per step."""
    if w.ndim != 2 or w.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("prepare_projection_weight: a [d_in, d_out] matrix of bf16 or fp16")
    K, N = w.shape
    if (K < 2 or w.stride(0) == 1) and (N < 2 or (w.stride(1) % 8 == 0 and w.stride(1) >= K)) and w.data_ptr() % 16 == 0 and (N > 1 or K % 8 == 0):
        return w
    out = torch.empty((N, -(-K // 8) * 8), dtype=w.dtype, device=w.device)[:, :K].t()
    out.copy_(w)
    return out


def matmul_lora(x: torch.Tensor, w: torch.Tensor, bias, adapters: LoraAdapters | None, indx) -> torch.Tensor:
    """y [T, d_out] = x w + bias, plus scale[a] * (x a[a]) b[a] for the rows whose index a = indx[t] is an adapter.

    x [T, d_in], w [d_in, d_out] (in the memory order of `prepare_projection_weight`, else it is re-laid-out on every call) and the adapters in one type,
    bf16 or fp16; bias [d_out] or None; indx [T] int32 or int64, any order: a negative index, or one past the last adapter, is a row without an adapter.
    Rows of a request that stand together share the reads of its adapter.  Sums are fp32 and y is rounded once; x a[a] goes into the
    second product in fp32, which with more than 128 tokens in bf16 is two bf16 terms, 2^-17 of a value off.  `adapters` None (then indx too) is the projection by
    itself.  Runs on the current stream of x's device, which has to hold all tensors; every call has a workspace of its own, so calls may overlap and be captured in CUDA graphs."""
    if not isinstance(x, torch.Tensor) or x.ndim != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("matmul_lora: x is a [tokens, d_in] tensor of bf16 or fp16")
    if not x.is_cuda:
        raise ValueError("triton_b200 operators take CUDA tensors only (no CPU path)")
    T, K = x.shape
    if K == 0 or w.ndim != 2 or w.shape[0] != K or w.dtype != x.dtype:
        raise ValueError(f"matmul_lora: w is [{K}, d_out] of {x.dtype} for this x, got {list(w.shape)} of {w.dtype}")
    N = w.shape[1]
    if bias is not None and (bias.ndim != 1 or bias.shape[0] != N or (N > 1 and bias.stride(0) != 1)
                             or bias.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
        raise ValueError(f"matmul_lora: bias is a contiguous vector of {N} floats")
    if (adapters is None) != (indx is None):
        raise ValueError("matmul_lora: adapters and indx go together")
    packed = None
    if adapters is not None:
        if adapters.d_in != K or adapters.d_out != N or adapters.a.dtype != x.dtype:
            raise ValueError(f"matmul_lora: adapters are [{adapters.d_in}, r] x [r, {adapters.d_out}] of {adapters.a.dtype}, the projection [{K}, {N}] of {x.dtype}")
        if indx.ndim != 1 or indx.shape[0] != T or indx.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"matmul_lora: indx is a vector of {T} int32 or int64")
        packed = (adapters.a, adapters.b, adapters.first, adapters.scale, adapters.n_adapters, adapters.max_pieces,
                  adapters.ranks_device)
    return _lib.host().lora(x, prepare_projection_weight(w), bias, packed, indx, _status_word(x.device))
