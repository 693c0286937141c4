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
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,N", [(8, 8), (77, 300), (1000, 129), (2880, 5120)])
def test_one_token_of_small_ranks(K, N, dtype):
    x, w, b, la, lb, scale = make(1, K, N, [16, 3, 9], dtype, 13)
    pw, adapters = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale)
    for a in (-1, 0, 1, 2, 3):
        indx = torch.tensor([a], device="cuda", dtype=torch.int32)
        y = tb.matmul_lora(x, pw, b, adapters, indx)
        tb.matmul_check_status()
        check(y, *reference(x, w, b, la, lb, scale, indx))


@gpu
@pytest.mark.parametrize("T", [3, 500])
def test_high_rank(T):
    run_case(T, 256, 256, [1024, 200], kind="random", seed=5)


@gpu
@pytest.mark.parametrize("T,K,N,ranks", [(5000, 64, 5120, [16, 40]), (1500, 8, 9000, [16] * 9), (8200, 128, 300, [1])])
def test_more_tiles_than_pairs(T, K, N, ranks):
    run_case(T, K, N, ranks, kind="runs", seed=7)


@gpu
@pytest.mark.parametrize("T", [20, 200])
def test_many_adapters(T):
    run_case(T, 64, 200, [1 + i % 20 for i in range(300)], seed=9)


@gpu
@pytest.mark.parametrize("T", [64, 512, 1100])
@pytest.mark.parametrize("order", ["every", "turns", "back"])
def test_order_of_the_adapters(T, order):
    """as many adapters as tokens, one token each; three in turns; the last adapter's tokens first"""
    L = {"every": T, "turns": 3, "back": 5}[order]
    x, w, b, la, lb, scale = make(T, 64, 136, [1 + i % 17 for i in range(L)], torch.bfloat16, 11)
    at = torch.arange(T, device="cuda")
    indx = {"every": at * 37 % T, "turns": at % 3, "back": L - 1 - at * L // T}[order].to(torch.int32)
    assert order != "every" or indx.unique().numel() == T
    y = tb.matmul_lora(x, tb.prepare_projection_weight(w), b, tb.prepare_lora_adapters(la, lb, scale), indx)
    tb.matmul_check_status()
    check(y, *reference(x, w, b, la, lb, scale, indx))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_without_adapters(T, dtype):
    x, w, b, *_ = make(T, 200, 333, [], dtype, 4)
    w = tb.prepare_projection_weight(w)
    check(tb.matmul_lora(x, w, b, None, None), *reference(x, w, b, [], [], [], torch.full((T,), -1, device="cuda")))


@gpu
@pytest.mark.parametrize("T", [10, 300])
def test_a_request_that_is_not_finite_stays_by_itself(T):
    x, w, b, la, lb, scale = make(T, 256, 200, [16, 24, 8], torch.bfloat16, 5)
    indx = indices(T, 3, "random", 5)
    w, adapters = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale)
    want = tb.matmul_lora(x, w, b, adapters, indx)
    y = x.clone()
    y[3, 5] = float("nan")
    y[4, 6] = float("inf")
    got = tb.matmul_lora(y, w, b, adapters, indx)
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[5:], want[5:]) and not torch.isfinite(got[3:5]).any()
    broken = [la[0].clone(), *la[1:]]
    broken[0][2, 2] = float("inf")                             # an adapter that has gone wrong
    got = tb.matmul_lora(x, w, b, tb.prepare_lora_adapters(broken, lb, scale), indx)
    assert torch.equal(got[indx != 0], want[indx != 0]) and not torch.isfinite(got[indx == 0]).any()


@gpu
@pytest.mark.parametrize("T", [10, 300])
def test_layouts_of_the_inputs(T):
    x, w, b, la, lb, scale = make(T, 256, 200, [16, 24, 8], torch.bfloat16, 6)
    indx = indices(T, 3, "random", 6)
    pw, adapters = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale)
    want = tb.matmul_lora(x, pw, b, adapters, indx)
    wide = torch.full((T, 600), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, 129:385] = x
    assert torch.equal(tb.matmul_lora(wide[:, 129:385], pw, b, adapters, indx), want)
    assert torch.equal(tb.matmul_lora(x.t().contiguous().t(), pw, b, adapters, indx), want)
    assert torch.equal(tb.matmul_lora(x, w, b, adapters, indx), want)                                   # a weight not prepared
    assert torch.equal(tb.matmul_lora(x, pw, b.float(), adapters, indx), want)
    both = torch.stack((indx, indx), 1)[:, 0]
    assert torch.equal(tb.matmul_lora(x, pw, b, adapters, both), want)                                  # a strided index
    far = indx.long().masked_fill(indx == -1, 1 << 40)
    assert torch.equal(tb.matmul_lora(x, pw, b, adapters, far), want)                                   # past the last adapter is none
    assert torch.equal(tb.matmul_lora(x, pw, b, adapters, indx.masked_fill(indx == -1, 3)), want)
    assert torch.equal(tb.matmul_lora(x[:0], pw, b, adapters, indx[:0]), want[:0])


@gpu
@pytest.mark.parametrize("T", [10, 300])
def test_broadcast_inputs(T):
    x, w, b, la, lb, scale = make(T, 256, 200, [16, 24, 8], torch.bfloat16, 6)
    indx = indices(T, 3, "random", 6)
    adapters = tb.prepare_lora_adapters(la, lb, scale)
    row, column, one = x[:1].expand(T, -1), w[:, :1].expand(-1, 200), indx[:1].expand(T)
    got = tb.matmul_lora(row, column, b, adapters, indx)
    assert torch.equal(got, tb.matmul_lora(row.clone(memory_format=torch.contiguous_format), tb.prepare_projection_weight(column.clone(memory_format=torch.contiguous_format)), b, adapters, indx))
    assert torch.equal(tb.matmul_lora(x, w, b, adapters, one), tb.matmul_lora(x, w, b, adapters, one.clone(memory_format=torch.contiguous_format)))


@gpu
@pytest.mark.parametrize("T", [10, 300])
def test_captured_replayed_and_side_by_side(T):
    cases = []
    for seed in (1, 2):
        x, w, b, la, lb, scale = make(T, 512, 640, [16, 8, 32], torch.bfloat16, seed)
        cases.append((x, tb.prepare_projection_weight(w), b, tb.prepare_lora_adapters(la, lb, scale), indices(T, 3, "random", seed)))
    want = [tb.matmul_lora(*c) for c in cases]
    torch.cuda.synchronize()
    streams, graphs, out = [torch.cuda.Stream() for _ in cases], [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(tb.matmul_lora(*c))
        graphs.append(g)
    eager = [[], []]
    for _ in range(10):
        for c, s, g, e in zip(cases, streams, graphs, eager):
            with torch.cuda.stream(s):
                g.replay()
                e.append(tb.matmul_lora(*c))
    torch.cuda.synchronize()
    tb.matmul_check_status()
    for w_, y, e in zip(want, out, eager):
        assert torch.equal(w_, y) and all(torch.equal(w_, q) for q in e)
    for c in cases:                                            # new tokens and new adapters for the captured call
        c[0].normal_()
        c[4].copy_(torch.flip(c[4], (0,)))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for c, y in zip(cases, out):
        assert torch.equal(y, tb.matmul_lora(*c))


@gpu
def test_a_decode_step_projection_and_expert_layer():
    """A step of seven requests: attention's output projection with each request's adapter, the residual, the expert layer; eager and in one graph"""
    from test_moe_tokens_gpu import make_layer, router
    from test_moe_tokens_gpu import reference as layer_reference
    T, d, E, k = 7, 256, 16, 4
    x, w, b, la, lb, scale = make(T, 320, d, [8, 16], torch.bfloat16, 21)
    residual = torch.randn(T, d, device="cuda").bfloat16()
    indx = torch.tensor([0, 1, -1, 1, 0, 1, -1], device="cuda", dtype=torch.int32)
    pw, adapters = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale)
    lw, full1, full2 = make_layer(E, d, 192, 21)
    wg, bg = router(d, E, 21)

    def step():
        h = tb.matmul_lora(x, pw, b, adapters, indx) + residual
        return h, h + tb.moe_layer_tokens(h, wg, bg, lw, k)

    h, y = step()
    ref, bound = reference(x, w, b, la, lb, scale, indx)
    check(h, ref + residual.double(), bound + 2.0 ** -8 * (ref + residual.double()).abs() + 2.0 ** -8 * bound)
    ref, bound = layer_reference(h, wg, bg, lw, full1, full2, k)
    total = h.double() + ref
    check(y, total, bound + 2.0 ** -8 * (total.abs() + bound))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, again = step()
    g.replay()
    torch.cuda.synchronize()
    tb.matmul_check_status()
    assert torch.equal(again, y)


@gpu
def test_refusals():
    x, w, b, la, lb, scale = make(4, 64, 96, [16], torch.bfloat16, 0)
    adapters, indx = tb.prepare_lora_adapters(la, lb, scale), torch.zeros(4, dtype=torch.int32, device="cuda")
    good = {"x": x, "w": w, "bias": b, "adapters": adapters, "indx": indx}
    other = tb.prepare_lora_adapters([la[0][:32]], lb, scale)
    bad = [dict(x=x.float()), dict(x=x[0]), dict(x=x[:, :32]), dict(w=w.half()), dict(w=w[None]), dict(bias=b[:5]), dict(bias=b.double()), dict(indx=None),
           dict(adapters=None), dict(indx=indx[:2]), dict(indx=indx.to(torch.int16)), dict(adapters=other), dict(x=x.half(), w=w.half()), dict(indx=indx.cpu()),
           dict(w=w.cpu()), dict(bias=b.cpu())]
    for change in bad:
        with pytest.raises(ValueError):
            tb.matmul_lora(**{**good, **change})


def test_prepared_adapters():
    """Layout and refusals of the preparation, which runs anywhere"""
    x, w, b, la, lb, scale = make(1, 20, 130, [3, 17], torch.bfloat16, 0, device="cpu")
    p = tb.prepare_lora_adapters(la, lb, scale)
    assert p.first.tolist() == [0, 1, 3] and p.max_pieces == 2 and p.n_adapters == 2 and p.ranks == (3, 17)
    assert tuple(p.a.shape) == (48, 24) and tuple(p.b.shape) == (3, 32, 2, 8, 8)
    rows = p.b.permute(0, 2, 4, 1, 3).reshape(3, 16, 256)      # [piece, rank, output]
    for i, (r, f) in enumerate(((3, 0), (17, 1))):
        got = rows[f:f + -(-r // 16)].reshape(-1, 256)
        assert torch.equal(got[:r, :130], lb[i]) and got[r:].count_nonzero() == 0 and got[:, 130:].count_nonzero() == 0
        a = p.a[16 * f:16 * f + r]
        assert torch.equal(a[:, :20], la[i].t()) and a[:, 20:].count_nonzero() == 0
    nan = lb[0].clone()
    nan[0, 0] = float("inf")
    for args in (([], [], []), (la, lb[:1], scale), (la, [nan, lb[1]], scale), ([la[0].float(), la[1]], lb, scale), ([a.float() for a in la], [q.float() for q in lb], scale),
                 ([la[0][:10], la[1]], lb, scale), (la, [lb[0][:, :5], lb[1]], scale), ([la[0][:, :0], la[1]], [lb[0][:0], lb[1]], scale),
                 ([torch.zeros(20, 1025).bfloat16()], [torch.zeros(1025, 130).bfloat16()], [1.0])):
        with pytest.raises(ValueError):
            tb.prepare_lora_adapters(*args)


def test_prepared_weight():
    w = torch.randn(20, 6).bfloat16()
    p = tb.prepare_projection_weight(w)
    assert torch.equal(p, w) and p.stride(0) == 1 and p.stride(1) == 24
    assert tb.prepare_projection_weight(p) is p
    for bad in (w.float(), w[None]):
        with pytest.raises(ValueError):
            tb.prepare_projection_weight(bad)


def test_refuses_cpu_tensors_and_wrong_types():
    for x in (torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(1, 32), torch.zeros(32, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            tb.matmul_lora(x, None, None, None, None)


def test_refusals_of_the_c_entry_point():
    import ctypes
    from triton_b200 import _lib
    lib = _lib.load()
    assert lib.moe_lora_matmul(None, None) == 1 and b"NULL" in lib.moe_last_error()
    assert lib.moe_lora_matmul_workspace_bytes(None) == 0
    blank = (ctypes.c_uint8 * 512)()
    assert lib.moe_lora_matmul(ctypes.addressof(blank), None) == 1 and b"positive" in lib.moe_last_error()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,ranks", [(1, [5]), (1, [16, 7]), (1, [17, 40]), (10, [1, 24, 16]), (300, [1, 24, 16]), (4100, [3, 20])])
def test_infinities_keep_their_sign_whatever_the_rank(T, ranks, dtype):
    """Where the signs of x W and of every rank's share agree, a row with an infinite element is infinite with that sign: ranks that an adapter does not have add nothing."""
    x, w, b, la, lb, scale = make(T, 256, 200, ranks, dtype, 31)
    sign = torch.where(torch.arange(200, device="cuda") % 3 == 0, -1.0, 1.0).to(dtype)
    w[9] = (w[9].abs() + 0.01) * sign
    for a in la:
        a[9] = a[9].abs() + 0.01
    lb = [(q.abs() + 0.01) * sign for q in lb]
    indx = (torch.arange(T, device="cuda") % (len(ranks) + 1)).to(torch.int32) if T > 1 else torch.zeros(1, dtype=torch.int32, device="cuda")
    want = x.clone()
    rows = torch.arange(0, T, 3, device="cuda")
    x[rows, 9] = torch.where(rows % 2 == 0, float("inf"), float("-inf")).to(dtype)
    pw, adapters = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale)
    y = tb.matmul_lora(x, pw, b, adapters, indx)
    tb.matmul_check_status()
    assert torch.equal(y[rows], x[rows, 9:10] * sign)
    others = torch.ones(T, dtype=torch.bool, device="cuda")
    others[rows] = False
    assert torch.equal(y[others], tb.matmul_lora(want, pw, b, adapters, indx)[others])


@gpu
@pytest.mark.parametrize("scale,size", [(4.0e4, 2.0 ** -10), (1.0e-6, 2.0 ** 9), (1.0, 1.0)])
@pytest.mark.parametrize("T,N,ranks", [(128, 136, [16, 40, 5]), (129, 136, [16, 40, 5]), (300, 500, [16, 40, 5]), (1500, 900, [16, 40, 5]), (600, 200, [1000, 64])])
def test_x_a_outside_the_range_of_fp16(T, N, ranks, scale, size):
    """scale * x A of 1e5 and of 1e-6, beside B's that bring y back into range, in fp16: as with values near one, on both sides of 128 tokens.  x A is 24 bits there, of products
    that stay exact; what is left out of them is below 2^-22."""
    x, _, b, la, lb, _ = make(T, 96, N, ranks, torch.float16, 41)
    w = torch.zeros(96, N, device="cuda", dtype=torch.float16)
    lb = [(q.double() * size).half() for q in lb]
    scales = [scale * (1 + i) for i in range(len(ranks))]
    indx = indices(T, len(ranks), "random", 41)
    y = tb.matmul_lora(x, tb.prepare_projection_weight(w), None, tb.prepare_lora_adapters(la, lb, scales), indx)
    tb.matmul_check_status()
    ref, bound = torch.zeros(T, N, dtype=torch.float64, device="cuda"), torch.zeros(T, N, dtype=torch.float64, device="cuda")
    most = 0.0
    for i, (a, q, s) in enumerate(zip(la, lb, scales)):
        at = torch.nonzero(indx == i).squeeze(1)
        t = s * (x[at].double() @ a.double())
        e_t = s * (96 / 16 + 32) * 2.0 ** -23 * (x[at].abs().double() @ a.abs().double()) + 2.0 ** -22 * t.abs()
        ref[at] = t @ q.double()
        bound[at] = e_t @ q.double().abs() + ((96 + 5 * a.shape[1]) / 16 + 32) * 2.0 ** -23 * (t.abs() @ q.double().abs())
        most = max(most, t.abs().max().item())
    assert ref.abs().max() < 6e4 and (most > 65504 or scale < 4e4)
    bound += (ref.abs() + bound) * 2.0 ** -11 + 2.0 ** -25              # (half a step of fp16, or of its subnormals)
    check(y, ref, bound)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ["turns", "random", "runs", "back"])
@pytest.mark.parametrize("T,K,N,ranks", [
    # x A goes by blocks of 64 tokens beyond 1024 tokens of more than 3500 tokens times pieces, by eights below: both sides of either line
    (4500, 300, 136, [1 + i % 16 for i in range(64)]),          # as many adapters in a block as it has tokens
    (4100, 2001, 200, [16, 3, 40, 24, 8, 17, 64]),              # rows of x that are not 16-byte aligned
    (1030, 2888, 264, [64, 5, 33, 16, 48, 1]),                  # few blocks: k in four parts
    (1750, 520, 72, [32, 9, 17]), (1751, 520, 72, [32, 9, 17]),
    (1024, 1032, 72, [64, 30, 1, 16, 16]), (1025, 1032, 72, [64, 30, 1, 16, 16]),
    (3501, 96, 40, [7] * 130), (3500, 96, 40, [7] * 130),
])
def test_long_batches_of_mixed_adapters(T, K, N, ranks, order, dtype):
    L = len(ranks)
    x, w, b, la, lb, scale = make(T, K, N, ranks, dtype, 51)
    at = torch.arange(T, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(52)
    indx = {"turns": at % (L + 1) - 1, "random": torch.randint(-1, L + 1, (T,), device="cuda", generator=g), "runs": at * L // T, "back": (L - 1) - at * 37 % L}[order].to(torch.int32)
    y = tb.matmul_lora(x, tb.prepare_projection_weight(w), b, tb.prepare_lora_adapters(la, lb, scale), indx)
    tb.matmul_check_status()
    check(y, *reference(x, w, b, la, lb, scale, indx))


def test_prepared_adapters_carry_their_ranks():
    *_, la, lb, scale = make(1, 20, 130, [3, 17, 16], torch.float16, 0, device="cpu")
    p = tb.prepare_lora_adapters(la, lb, scale)
    assert p.ranks_device.tolist() == [3, 17, 16] and p.first.tolist() == [0, 1, 3, 4] and p.ranks_device.dtype == p.first.dtype == torch.int32


@gpu
@pytest.mark.parametrize("T", [1, 50, 400])
def test_adapters_without_ranks_are_whole_pieces(T):
    import dataclasses
    x, w, b, la, lb, scale = make(T, 128, 200, [5, 16, 9], torch.bfloat16, 61)
    pw, adapters, indx = tb.prepare_projection_weight(w), tb.prepare_lora_adapters(la, lb, scale), indices(T, 3, "random", 61)
    want = tb.matmul_lora(x, pw, b, adapters, indx)
    assert torch.equal(tb.matmul_lora(x, pw, b, dataclasses.replace(adapters, ranks_device=None), indx), want)
    with pytest.raises(ValueError):
        tb.matmul_lora(x, pw, b, dataclasses.replace(adapters, ranks_device=adapters.ranks_device.cpu()), indx)
