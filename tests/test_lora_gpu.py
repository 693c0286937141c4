"""`matmul_lora`: a shared projection with low-rank adapters of many requests, against the formula in 64 bits.

The bound of an element: a sum of n products in fp32, in any order, is off by at most (n / 16 + 32) 2^-23 times the sum of their magnitudes (16 exact
products an MMA, truncated to 24 bits as they are added); x A is taken in two 16-bit terms, off by 2^-16 of itself in bf16 (2^-22 in fp16) and, in
fp16, by 2^-25 where it is that small; the result by half a step of its type."""
import pytest
import torch

import triton_b200 as tb

gpu = pytest.mark.gpu


def make(T, K, N, ranks, dtype, seed, bias=True, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(T, K, device=device, generator=g).to(dtype)
    w = (torch.randn(K, N, device=device, generator=g) / K ** 0.5).to(dtype)
    b = torch.randn(N, device=device, generator=g).to(dtype) if bias else None
    la = [(torch.randn(K, r, device=device, generator=g) / K ** 0.5).to(dtype) for r in ranks]
    lb = [(torch.randn(r, N, device=device, generator=g) * 0.3).to(dtype) for r in ranks]
    scale = [0.5 + i % 3 for i in range(len(ranks))]
    return x, w, b, la, lb, scale


def reference(x, w, bias, la, lb, scale, indx):
    """-> (y, bound) in 64 bits"""
    X, W = x.double(), w.double()

    def rounding(n):
        return (n / 16 + 32) * 2.0 ** -23

    y, bound = X @ W, X.abs() @ W.abs()
    if bias is not None:
        y, bound = y + bias.double(), bound + bias.double().abs()
    bound = bound * rounding(X.shape[1])
    bf16 = x.dtype == torch.bfloat16
    for i, (a, b, s) in enumerate(zip(la, lb, scale)):
        at = torch.nonzero(indx == i).squeeze(1)
        t = s * (X[at] @ a.double())
        e_t = abs(s) * rounding(X.shape[1]) * (X[at].abs() @ a.double().abs()) + t.abs() * 2.0 ** (-16 if bf16 else -22) + (0 if bf16 else 2.0 ** -25)
        y[at] += t @ b.double()
        bound[at] += e_t @ b.double().abs() + rounding(X.shape[1] + 2 * a.shape[1]) * (t.abs() @ b.double().abs())
    return y, bound + (y.abs() + bound) * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).tiny


def check(y, ref, bound):
    assert torch.isfinite(y).all()
    worst = ((y.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, f"{worst} of the bound"


def indices(T, L, kind, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed + 99)
    if kind == "random":
        return torch.randint(-1, L, (T,), device=device, generator=g, dtype=torch.int32)
    if kind == "runs":
        return (torch.arange(T, device=device) * (L + 1) // max(T, 1)).to(torch.int32) - 1
    return torch.full((T,), {"none": -1, "last": L - 1}[kind], dtype=torch.int32, device=device)


def run_case(T, K, N, ranks, dtype=torch.bfloat16, kind="random", seed=0, bias=True):
    x, w, b, la, lb, scale = make(T, K, N, ranks, dtype, seed, bias)
    indx = indices(T, len(ranks), kind, seed)
    y = tb.matmul_lora(x, tb.prepare_projection_weight(w), b, tb.prepare_lora_adapters(la, lb, scale), indx)
    tb.matmul_check_status()
    assert y.shape == (T, N) and y.dtype == dtype
    check(y, *reference(x, w, b, la, lb, scale, indx))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 63, 64, 65, 130, 255, 256, 257, 300])
def test_token_counts(T, dtype):
    run_case(T, 512, 384, [16, 8, 40, 1], dtype)


@gpu
@pytest.mark.parametrize("kind", ["random", "runs", "none", "last"])
@pytest.mark.parametrize("T,K,N,ranks", [
    (1, 8, 1, [1]),                             # the smallest
    (5, 64, 130, [3, 17]),
    (33, 1000, 1001, [16] * 5),                 # extents that end inside tiles, odd rows of y
    (64, 2880, 640, [8, 16, 32, 64] * 16),      # as many adapters as tokens
    (19, 77, 65, [5, 31]),                      # rows of x that are not 16-byte aligned
    (600, 320, 500, [16, 64, 16]),
    (1000, 200, 300, [128, 16]),
])
def test_shapes(T, K, N, ranks, kind):
    run_case(T, K, N, ranks, kind=kind, seed=3, bias=N % 2 == 1)


@gpu
@pytest.mark.parametrize("T", [3, 500])
def test_high_rank(T):
    run_case(T, 256, 256, [1024, 200], kind="random", seed=5)
