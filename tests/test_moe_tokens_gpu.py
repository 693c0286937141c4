"""`moe_layer_tokens`: a whole MoE layer for a few tokens, against the formula in 64 bits.

The bound of an element is made from the sizes that enter it.  A sum of n fp32 products in any of the kernels' orders is off by at most
(n / 32 + 64) 2^-23 times the sum of the products' magnitudes (a 32-k group is one exact-product sum of the tensor core, the groups follow one
another); what is between the sums is carried along by its derivatives; a hidden value as fp16 operand is off by 2^-12 of itself and 2^-24 of
its row's largest (elements that become subnormal), a token by the latter; the result by half a step of its type."""
import pytest
import torch

import triton_b200 as tb
from triton_b200.moe import MoeLayerWeights
from triton_b200.tensor_details.layout import make_default_matmul_mxfp4_w_layout, make_default_matmul_mxfp4_w_scale_layout

gpu = pytest.mark.gpu
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def make_layer(E, d, ff, seed, device="cuda", alpha=1.702, limit=7.0, bias_dtype=torch.bfloat16):
    """Random codes and scale bytes straight from a generator -> (MoeLayerWeights, fp64 W1 [E, d, 2 ff], fp64 W2 [E, ff, d])"""
    g = torch.Generator(device=device).manual_seed(seed)

    def weights(K, N):
        q = torch.randint(0, 256, (E, N, K // 2), device=device, generator=g, dtype=torch.uint8)
        s = torch.randint(118, 124, (E, N, K // 32), device=device, generator=g, dtype=torch.uint8)
        table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=device)
        codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).long()
        w = table[codes] * torch.exp2(s.double() - 127).repeat_interleave(32, -1)
        tq = tb.convert_layout(tb.wrap_torch_tensor(q.transpose(1, 2), dtype=tb.FP4), make_default_matmul_mxfp4_w_layout(mx_axis=-2))
        ts = tb.convert_layout(tb.wrap_torch_tensor(s.transpose(1, 2)), make_default_matmul_mxfp4_w_scale_layout(mx_axis=-2))
        return tq, ts, w.transpose(1, 2)

    w1, s1, full1 = weights(d, 2 * ff)
    w2, s2, full2 = weights(ff, d)
    b1 = (torch.randn(E, 2 * ff, device=device, generator=g) * 0.1).to(bias_dtype)
    b2 = (torch.randn(E, d, device=device, generator=g) * 0.1).to(bias_dtype)
    return MoeLayerWeights(w1, s1, b1, w2, s2, b2, alpha, limit), full1, full2


def router(d, E, seed, device="cuda", bias=True):
    g = torch.Generator(device=device).manual_seed(seed + 1000)
    wg = tb.prepare_router_weight((torch.randn(d, E, device=device, generator=g) / d ** 0.5).bfloat16())
    return wg, torch.randn(E, device=device, generator=g) if bias else None


def reference(x, wg, bg, lw, full1, full2, k):
    """-> (y, bound) in 64 bits; asserts that the selection is not a matter of rounding"""
    X, WG = x.double(), wg.double()
    T, d = X.shape
    ff = full2.shape[1]
    lim, al = lw.limit, lw.alpha

    def rounding(n):
        return (n / 32 + 64) * 2.0 ** -23

    # a logit: at most 8 ceil(d / 2048) products one after the other, then 5 steps of a warp, the warps' sums in pairs and the bias, half a step each
    router_terms = 8 * -(-d // 2048) + 14
    b = torch.zeros(wg.shape[1], dtype=torch.float64, device=x.device) if bg is None else bg.double()
    logits, e_logit = X @ WG + b, router_terms * 2.0 ** -24 * (X.abs() @ WG.abs() + b.abs())
    vals, indx = torch.sort(logits, dim=1, descending=True, stable=True)
    if k < logits.shape[1]:
        gap, err = vals[:, k - 1] - vals[:, k], e_logit.amax(1)
        assert bool(((gap > 2 * err) | (gap == 0)).all())
    gates = torch.softmax(vals[:, :k], 1)
    y, bound = torch.zeros(T, d, dtype=torch.float64, device=x.device), torch.zeros(T, d, dtype=torch.float64, device=x.device)
    for t in range(T):
        for j in range(k):
            e, g = int(indx[t, j]), gates[t, j]
            pre = X[t] @ full1[e] + lw.b1[e].double()
            e_pre = rounding(d) * (X[t].abs() @ full1[e].abs() + lw.b1[e].double().abs())
            e_pre = e_pre + 2.0 ** -24 * X[t].abs().max() * full1[e].abs().sum(0)
            gate, lin = pre[0::2], pre[1::2]
            if lim is not None:
                gate, lin = gate.clamp(max=lim), lin.clamp(-lim, lim)
            s = gate * torch.sigmoid(al * gate)
            h = s * (lin + 1)
            # |d s / d gate| <= 1.1; the exponential and the division are good to 2^-20 of s
            e_h = (lin + 1).abs() * (1.1 * e_pre[0::2] + 2.0 ** -20 * s.abs()) + (s.abs() + 1.1 * e_pre[0::2]) * e_pre[1::2]
            e_h = e_h + 2.0 ** -12 * h.abs() + 2.0 ** -24 * h.abs().max()
            o = h @ full2[e] + lw.b2[e].double()
            e_o = e_h @ full2[e].abs() + rounding(ff) * (h.abs() @ full2[e].abs() + lw.b2[e].double().abs())
            e_gate = 4 * e_logit[t].max() + 2.0 ** -20
            y[t] += g * o
            bound[t] += g * (e_o + e_gate * o.abs())
    return y, bound + (y.abs() + bound) * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).tiny


def check(y, ref, bound):
    assert torch.isfinite(y).all()
    off = (y.double() - ref).abs()
    worst = (off / bound).max().item()
    assert worst <= 1.0, f"{worst} of the bound"


def run_case(T, E, k, d, ff, dtype=torch.bfloat16, seed=0, bias=True, **layer):
    lw, full1, full2 = make_layer(E, d, ff, seed, **layer)
    wg, bg = router(d, E, seed, bias=bias)
    x = torch.randn(T, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 7)).to(dtype)
    y = tb.moe_layer_tokens(x, wg, bg, lw, k)
    tb.matmul_check_status()
    assert y.shape == x.shape and y.dtype == dtype
    ref, bound = reference(x, wg, bg, lw, full1, full2, k)
    check(y, ref, bound)
    return x, wg, bg, lw, y


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 13, 16])
def test_token_counts(T, dtype):
    run_case(T, 16, 4, 256, 192, dtype)


@gpu
@pytest.mark.parametrize("T,E,k,d,ff", [
    (1, 1, 1, 32, 32),              # one unit, one stage, one expert
    (16, 1, 1, 32, 64),             # every token at one expert
    (1, 2, 2, 512, 1024),           # fewer stages than SMs
    (3, 5, 3, 736, 1440),           # extents that end inside tiles
    (7, 8, 8, 96, 160),             # every expert of every token
    (16, 16, 16, 64, 96),
    (2, 256, 16, 64, 32),
    (16, 255, 7, 128, 96),
    (4, 8, 2, 2880, 2880),
    (16, 12, 4, 1024, 544),
    (8, 2, 2, 8192, 32),            # the widest
    (8, 2, 1, 32, 8192),
    (16, 3, 2, 4096, 64),
    (9, 3, 2, 64, 4096),
])
def test_shapes(T, E, k, d, ff):
    run_case(T, E, k, d, ff, seed=3)


@gpu
@pytest.mark.parametrize("T,E,k,d,ff", [(16, 64, 8, 1024, 96), (16, 8, 1, 2048, 1024), (11, 40, 3, 160, 1056)])
def test_popular_experts(T, E, k, d, ff):
    """some experts have one block of token columns and others two: the CTAs' shares differ"""
    lw, full1, full2 = make_layer(E, d, ff, 5)
    wg, bg = router(d, E, 5)
    bg = bg + torch.linspace(0, 3, E, device="cuda").to(bg.dtype).flip(0)
    x = torch.randn(T, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(12)).bfloat16()
    y = tb.moe_layer_tokens(x, wg, bg, lw, k)
    tb.matmul_check_status()
    check(y, *reference(x, wg, bg, lw, full1, full2, k))


@gpu
def test_without_router_bias_and_with_other_activation():
    run_case(3, 8, 2, 256, 256, bias=False)
    run_case(3, 8, 2, 256, 256, limit=None, alpha=1.0, seed=5)
    run_case(3, 8, 2, 256, 256, bias_dtype=torch.float32, limit=0.5, seed=6)


def small(T=5, E=8, k=3, d=128, ff=96, seed=11, dtype=torch.bfloat16):
    lw, full1, full2 = make_layer(E, d, ff, seed)
    wg, bg = router(d, E, seed)
    x = torch.randn(T, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)
    return x, wg, bg, lw, k, full1, full2


@gpu
def test_equal_logits_go_to_the_lower_expert():
    x, wg, bg, lw, k, full1, full2 = small()
    wg = tb.prepare_router_weight(torch.zeros_like(wg).contiguous())
    bg = torch.tensor([0.0, 1.0, 1.0, 1.0, 1.0, 0.5, 0.0, -1.0], device="cuda")            # four equal logits for three places
    check(tb.moe_layer_tokens(x, wg, bg, lw, k), *reference(x, wg, bg, lw, full1, full2, k))
    only = torch.full((8,), float("-inf"), device="cuda")
    only[6] = 0.25                                             # all but one expert closed: the others have no weight
    ref, bound = reference(x, wg, torch.where(only.isinf(), -100.0, only), lw, full1, full2, 1)
    check(tb.moe_layer_tokens(x, wg, only, lw, k), ref, bound)
    lowest = torch.where(only.isinf(), torch.finfo(torch.float32).min, only)
    check(tb.moe_layer_tokens(x, wg, lowest, lw, k), ref, bound)


@gpu
@pytest.mark.parametrize("T", [4, 12])
def test_a_row_that_is_not_finite_stays_by_itself(T):
    x, wg, bg, lw, k, full1, full2 = small(T)
    want = tb.moe_layer_tokens(x, wg, bg, lw, k)
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[1, 7] = bad
        got = tb.moe_layer_tokens(y, wg, bg, lw, k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
        assert not torch.isfinite(got[1]).all()
    y = x.clone()
    y[1] = 0
    y[2] *= 2.0 ** -100
    y[3] *= 2.0 ** 60
    assert torch.isfinite(tb.moe_layer_tokens(y, wg, bg, lw, k)).all()
    ref, bound = reference(y[1:3], wg, bg, lw, full1, full2, k)
    check(tb.moe_layer_tokens(y, wg, bg, lw, k)[1:3], ref, bound)


@gpu
def test_scale_bytes_at_their_ends():
    E, d, ff = 2, 128, 64
    g = torch.Generator(device="cuda").manual_seed(0)

    def laid_out(q, s):
        return (tb.convert_layout(tb.wrap_torch_tensor(q.transpose(1, 2), dtype=tb.FP4), make_default_matmul_mxfp4_w_layout(mx_axis=-2)),
                tb.convert_layout(tb.wrap_torch_tensor(s.transpose(1, 2)), make_default_matmul_mxfp4_w_scale_layout(mx_axis=-2)))

    def layer(s1, s2):
        return MoeLayerWeights(*laid_out(q1, s1), torch.zeros(E, 2 * ff, device="cuda").bfloat16(), *laid_out(q2, s2), torch.zeros(E, d, device="cuda").bfloat16())

    q1 = torch.randint(0, 256, (E, 2 * ff, d // 2), device="cuda", generator=g, dtype=torch.uint8) | 0x11          # no code is zero
    q2 = torch.randint(0, 256, (E, d, ff // 2), device="cuda", generator=g, dtype=torch.uint8) | 0x11
    s1 = torch.full((E, 2 * ff, d // 32), 122, device="cuda", dtype=torch.uint8)
    s2 = torch.full((E, d, ff // 32), 122, device="cuda", dtype=torch.uint8)
    x = torch.randn(3, d, device="cuda", generator=g).bfloat16()
    wg, bg = router(d, E, 0)
    want = tb.moe_layer_tokens(x, wg, bg, layer(s1, s2), 2)
    assert torch.isfinite(want).all()
    nan2 = s2.clone()
    nan2[:, 5, 1] = 255                                        # the dequantiser makes such a group NaN: one output of every expert
    got = tb.moe_layer_tokens(x, wg, bg, layer(s1, nan2), 2)
    assert got[:, 5].isnan().all() and torch.equal(torch.cat((got[:, :5], got[:, 6:]), 1), torch.cat((want[:, :5], want[:, 6:]), 1))
    nan1 = s1.clone()
    nan1[:, 9, 0] = 255                                        # a hidden value, and with it every output
    assert tb.moe_layer_tokens(x, wg, bg, layer(nan1, s2), 2).isnan().all()
    zero2 = s2.clone()
    zero2[:, 5, :] = 0                                         # byte 0 is the factor 0
    assert (tb.moe_layer_tokens(x, wg, bg, layer(s1, zero2), 2)[:, 5] == 0).all()


@gpu
def test_layouts_of_the_inputs():
    x, wg, bg, lw, k, _, _ = small()
    want = tb.moe_layer_tokens(x, wg, bg, lw, k)
    wide = torch.zeros(5, 3 * 128 + 1, device="cuda", dtype=x.dtype)
    wide[:, 129:257] = x
    assert torch.equal(tb.moe_layer_tokens(wide[:, 129:257], wg, bg, lw, k), want)                      # rows that start anywhere
    assert torch.equal(tb.moe_layer_tokens(x.t().contiguous().t(), wg, bg, lw, k), want)                # columns together
    assert torch.equal(tb.moe_layer_tokens(x, wg.contiguous(), bg, lw, k), want)                        # a router weight not prepared
    shifted = torch.zeros(8 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(8, 128)
    shifted.copy_(wg.t())
    assert torch.equal(tb.moe_layer_tokens(x, shifted.t(), bg, lw, k), want)
    assert torch.equal(tb.moe_layer_tokens(x[:0], wg, bg, lw, k), want[:0])
    for t in range(5):                                         # a token's result does not depend on the others but for the rounding of operands
        one = tb.moe_layer_tokens(x[t:t + 1], wg, bg, lw, k)
        assert (one - want[t]).float().norm() <= 2.0 ** -8 * want[t].float().norm()


@gpu
def test_the_same_bits_every_time_and_side_by_side():
    cases = [small(16, 32, 4, 512, 256, seed=1), small(3, 8, 2, 256, 512, seed=2)]
    want = [tb.moe_layer_tokens(*c[:5]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(30):
        for c, s, g in zip(cases, streams, got):
            with torch.cuda.stream(s):
                g.append(tb.moe_layer_tokens(*c[:5]))
    torch.cuda.synchronize()
    tb.matmul_check_status()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


@gpu
def test_two_captured_calls_replayed_side_by_side():
    cases = [small(4, 8, 2, 256, 128, seed=3), small(4, 8, 2, 256, 128, seed=4)]
    for c in cases:
        tb.moe_layer_tokens(*c[:5])
    torch.cuda.synchronize()
    graphs, out = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(tb.moe_layer_tokens(*c[:5]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for round_ in range(4):
        fresh = [torch.randn(4, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(100 + round_ + i)).bfloat16() for i in range(2)]
        for c, f in zip(cases, fresh):
            c[0].copy_(f)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        tb.matmul_check_status()
        for c, y in zip(cases, out):
            assert torch.equal(y, tb.moe_layer_tokens(*c[:5]))
        torch.cuda.synchronize()


@gpu
def test_agrees_with_the_layer_made_of_operators():
    x, wg, bg, lw, k, full1, full2 = small(9, 16, 4, 512, 320, seed=8)
    from triton_b200.moe import moe_layer_forward
    logits = (x.double() @ wg.double() + bg.double()).float()
    other = moe_layer_forward(x, logits, lw, k).float()
    mine = tb.moe_layer_tokens(x, wg, bg, lw, k).float()
    # the operators round the hidden rows, every expert's output and their sum to bf16: three half steps in the 2-norm, ours one
    assert (other - mine).norm() <= 4 * 2.0 ** -8 * mine.norm()


@gpu
def test_refusals():
    x, wg, bg, lw, k, _, _ = small()
    bad = [dict(x=x.float()), dict(x=x[0]), dict(wg=wg[:, :4]), dict(bg=bg[:4]), dict(bg=bg.double()), dict(bg=bg.repeat_interleave(2)[::2]), dict(k=0), dict(k=9),
           dict(x=x[:, :64].contiguous()), dict(wg=wg.cpu()), dict(bg=bg.cpu())]
    for change in bad:
        a = {"x": x, "wg": wg, "bg": bg, "lw": lw, "k": k, **change}
        with pytest.raises(ValueError):
            tb.moe_layer_tokens(a["x"], a["wg"], a["bg"], a["lw"], a["k"])
    with pytest.raises(NotImplementedError):
        tb.moe_layer_tokens(x.repeat(4, 1), wg, bg, lw, k)                                               # 20 tokens
    import dataclasses
    plain = dataclasses.replace(lw, w1=tb.wrap_torch_tensor(torch.zeros(8, 64, 192, device="cuda", dtype=torch.uint8), dtype=tb.FP4))
    with pytest.raises(NotImplementedError):
        tb.moe_layer_tokens(x, wg, bg, plain, k)
    with pytest.raises(ValueError):
        tb.moe_layer_tokens(x, wg, bg, dataclasses.replace(lw, b2=lw.b2[:, :64]), k)


def test_refuses_cpu_tensors():
    with pytest.raises(ValueError):
        tb.moe_layer_tokens(torch.zeros(1, 32, dtype=torch.bfloat16), None, None, None, 1)
    with pytest.raises(ValueError):
        tb.moe_layer_tokens(torch.zeros(1, 32), None, None, None, 1)


def test_refusals_of_the_c_entry_point():
    import ctypes
    from triton_b200 import _lib
    lib = _lib.load()
    assert lib.moe_layer_tokens(None, None) == 1 and b"NULL" in lib.moe_last_error()
    assert lib.moe_layer_tokens_workspace_bytes(None) == 0
    blank = (ctypes.c_uint8 * 512)()                           # all sizes zero
    assert lib.moe_layer_tokens(ctypes.addressof(blank), None) == 1 and b"positive" in lib.moe_last_error()


def layer_of_differences(E, d, ff, seed):
    """W1 = 0, so hidden value i is SwiGLU of its biases whatever the token; output o is h_i - h_j of two neighbours by size.  -> (MoeLayerWeights,
    h [E, ff] in 64 bits, i [d], j [d])"""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def laid_out(q, s):
        return (tb.convert_layout(tb.wrap_torch_tensor(q.transpose(1, 2), dtype=tb.FP4), make_default_matmul_mxfp4_w_layout(mx_axis=-2)),
                tb.convert_layout(tb.wrap_torch_tensor(s.transpose(1, 2)), make_default_matmul_mxfp4_w_scale_layout(mx_axis=-2)))

    b1 = torch.empty(E, 2 * ff, device="cuda")
    b1[:, 0::2] = torch.rand(E, ff, device="cuda", generator=g).sort(1).values * 0.02 + 1.0
    b1[:, 1::2] = 0.25
    gate, lin = b1[:, 0::2].double(), b1[:, 1::2].double()
    h = gate * torch.sigmoid(1.702 * gate) * (lin + 1)
    i = torch.randint(0, ff - 1, (d,), device="cuda", generator=g)
    codes = torch.zeros(E, d, ff, dtype=torch.uint8, device="cuda")
    codes.scatter_(2, i.view(1, d, 1).expand(E, -1, -1), 2)                    # 1.0
    codes.scatter_(2, (i + 1).view(1, d, 1).expand(E, -1, -1), 2 | 8)          # -1.0
    q1, s1 = torch.zeros(E, 2 * ff, d // 2, dtype=torch.uint8, device="cuda"), torch.full((E, 2 * ff, d // 32), 127, dtype=torch.uint8, device="cuda")
    q2, s2 = codes[..., 0::2] | codes[..., 1::2] << 4, torch.full((E, d, ff // 32), 127, dtype=torch.uint8, device="cuda")
    lw = MoeLayerWeights(*laid_out(q1, s1), b1, *laid_out(q2, s2), torch.zeros(E, d, device="cuda"))
    return lw, h, i, i + 1


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (4, 1, 1), (5, 1, 1), (8, 1, 1), (8, 2, 2), (9, 1, 1), (16, 1, 1), (16, 3, 3), (13, 6, 2)])
def test_hidden_rows_keep_their_bits_however_many_tokens_an_expert_has(T, E, k, dtype):
    """A hidden value is good to 2^-20 of itself (the exponential and the division), its two terms to 2^-22 and each of the sum's few roundings to 2^-23: less than
    2^-19 of the two values together, per expert; the gates sum to one within 2^-20 and weigh differences of some 2^-9; the result's own half step."""
    d, ff = 96, 160
    lw, h, i, j = layer_of_differences(E, d, ff, 3)
    wg, bg = router(d, E, 3)
    x = torch.randn(T, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(dtype)
    y = tb.moe_layer_tokens(x, wg, bg, lw, k).double()
    tb.matmul_check_status()
    logits = x.double() @ wg.double() + bg.double()
    vals, indx = torch.sort(logits, dim=1, descending=True, stable=True)
    gates = torch.softmax(vals[:, :k], 1)
    ref = torch.einsum("tk,tkd->td", gates, (h[:, i] - h[:, j])[indx[:, :k]])
    e_gates = 2.0 ** -18 * (h[:, i] - h[:, j]).abs().amax(0)          # (logits of some ten roundings of values below 8: 2^-18)
    bound = 2.0 ** -19 * (h[:, i] + h[:, j]).amax(0) + e_gates
    bound = bound + (ref.abs() + bound) * torch.finfo(dtype).eps / 2
    worst = ((y - ref).abs() / bound).max().item()
    assert worst <= 1.0, f"{worst} of the bound"


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,ff", [
    (16, 16, 16, 512, 1056),        # every expert has all tokens: two entries of fc2 each, 256 picks
    (8, 8, 8, 1440, 2880),          # fc2 in three stages, cut between CTAs
    (8, 3, 3, 64, 8192),
    (8, 3, 2, 8192, 64),
    (12, 4, 2, 2880, 1024),         # some experts in two entries, others in one
    (5, 2, 1, 736, 1440),
])
def test_experts_of_most_tokens(T, E, k, d, ff, dtype):
    run_case(T, E, k, d, ff, dtype, seed=17)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_router_weight_that_is_not_bf16_is_refused(dtype):
    """casting it would round the logits' factors, by which experts are picked, without the caller's knowing"""
    x, wg, bg, lw, k, _, _ = small()
    with pytest.raises(ValueError, match="bf16"):
        tb.moe_layer_tokens(x, wg.to(dtype), bg, lw, k)
    assert torch.isfinite(tb.moe_layer_tokens(x, tb.prepare_router_weight(wg.to(dtype)), bg, lw, k)).all()


@gpu
@pytest.mark.parametrize("T,E,k", [(16, 256, 16), (8, 128, 16), (16, 250, 15)])
def test_every_pick_another_expert(T, E, k):
    """as many active experts as there can be: the lists of experts are full"""
    d, ff = 64, 32
    lw, full1, full2 = make_layer(E, d, ff, 23)
    g = torch.Generator(device="cuda").manual_seed(24)
    x = torch.randn(T, d, device="cuda", generator=g) * 0.1
    x[:, :T] = torch.eye(T, device="cuda") * 4
    x = x.bfloat16()
    wg = torch.randn(d, E, device="cuda", generator=g) * 0.01
    experts = torch.randperm(E, device="cuda", generator=g)[:T * k].view(T, k)
    for t in range(T):
        wg[t, experts[t]] = 2.0 + torch.rand(k, device="cuda", generator=g)
    wg = tb.prepare_router_weight(wg.bfloat16())
    y = tb.moe_layer_tokens(x, wg, None, lw, k)
    tb.matmul_check_status()
    assert (x.double() @ wg.double()).topk(k, 1).indices.unique().numel() == T * k
    check(y, *reference(x, wg, None, lw, full1, full2, k))
