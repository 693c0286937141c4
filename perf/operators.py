"""Performance cases of the operators of a serving step over few tokens and many requests.

Kinds
  moe    `moe_layer_tokens`: a whole mixture-of-experts layer for up to 16 tokens -- router product, top-k, softmax over the selected
         logits, both expert products on MXFP4 weights with SwiGLU between them, and the weighted sum over the selected experts
  lora   `matmul_lora`: a projection that all requests share, with each request's own low-rank adapter added beside it

`listed()` names the cases that stand for the work, `draw(rng)` picks further ones from the same ranges, `prepare` makes what a program
holds before the call, `run` is one pass: in plain torch operations in 32 bits, rounded once at the end, or with `own` through the
package's entry points.  `exact` is the same from the definition in 64 bits, `work` the bytes and operations a pass cannot do without."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ALPHA, LIMIT = 1.702, 7.0                          # of SwiGLU: the layer's defaults
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)    # magnitudes of the codes 0 to 7; bit 3 is the sign


def _moe(name, tokens, experts, top_k, d_model, d_ff, dtype="bf16", skew=True):
    return {"name": name, "kind": "moe", "tokens": tokens, "experts": experts, "top_k": top_k, "d_model": d_model, "d_ff": d_ff,
            "dtype": dtype, "skew": skew}


def _lora(name, tokens, d_in, d_out, adapters, rank, mixed, form, dtype="bf16", bias=True):
    """rank: the largest; `mixed`: adapters of several ranks up to it.  form: "decode", every token a request of its own; "prompts", the
    tokens of a request stand together; "both", a batch of single tokens behind a few prompts."""
    return {"name": name, "kind": "lora", "tokens": tokens, "d_in": d_in, "d_out": d_out, "adapters": adapters, "rank": rank,
            "mixed": mixed, "form": form, "dtype": dtype, "bias": bias}


def listed():
    return [
        # decode of a single stream: four experts of 128 are read, latency counts
        _moe("moe 1 token", 1, 128, 4, 2880, 2880),
        # a few streams side by side, or a short run of drafted tokens that is being checked
        _moe("moe 4 tokens", 4, 128, 4, 2880, 2880),
        # a small serving batch of the smaller layer: most experts are read once, with one or two rows each
        _moe("moe 8 tokens 32 experts", 8, 32, 4, 2880, 2880),
        # a small model in fp16, odd count of tokens, extents that are no multiple of a tile
        _moe("moe 3 tokens small fp16", 3, 8, 2, 736, 1440, dtype="fp16", skew=False),
        # many picks per token over narrow experts
        _moe("moe 13 tokens top 8", 13, 64, 8, 2048, 1024),
        # the largest batch that this form takes: some fifty experts are streamed
        _moe("moe 16 tokens", 16, 128, 4, 2880, 2880),
        # one token of one request: the weight is read once, latency counts
        _lora("lora 1 token", 1, 2880, 5120, 8, 16, False, "decode"),
        # decode of a serving batch: nearly every token has another adapter
        _lora("lora 64 tokens 64 adapters", 64, 2880, 5120, 64, 64, True, "decode"),
        # a smaller batch through the projection back to the model's width, fp16, some requests without an adapter
        _lora("lora 23 tokens fp16", 23, 4096, 2880, 16, 32, True, "decode", dtype="fp16", bias=False),
        # single tokens and short prompts in one batch
        _lora("lora 300 tokens", 300, 2880, 5120, 12, 16, False, "both"),
        # a few prompts of ragged lengths, an output whose rows are odd
        _lora("lora 1200 tokens odd width", 1200, 2048, 1433, 8, 64, True, "prompts"),
        # prefill: the largest
        _lora("lora 8192 tokens", 8192, 2880, 5120, 4, 16, False, "prompts"),
    ]


MOE_MAX = 64 * 2880 * 2880                         # experts that can be active x d_model x d_ff of the largest listed case
MOE_MAX_WEIGHTS = 128 * 2880 * 2880
LORA_MAX = 8192 * 2880 * 5120


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    if rng.random() < 0.5:
        sizes = [512, 736, 1024, 1440, 2048, 2880, 2880, 4096]
        d_model, d_ff = rng.choice(sizes), rng.choice(sizes)
        experts = rng.choice([8, 16, 32, 60, 64, 128])
        while experts * d_model * d_ff > MOE_MAX_WEIGHTS:
            experts //= 2
        top_k = min(rng.choice([1, 2, 4, 4, 8]), experts)
        tokens = rng.randint(1, 16)
        while tokens > 1 and min(experts, tokens * top_k) * d_model * d_ff > MOE_MAX:
            tokens -= 1
        return _moe("", tokens, experts, top_k, d_model, d_ff, rng.choice(["bf16", "bf16", "bf16", "fp16"]), rng.random() < 0.75)
    d_in = rng.choice([512, 736, 1000, 1440, 2048, 2880, 4096, 5120])
    d_out = rng.choice([512, 736, 1001, 1433, 2048, 2880, 4096, 5120, 5760])
    tokens = _log_int(rng, 1, min(8192, LORA_MAX // (d_in * d_out)))
    form = "decode" if tokens < 16 else rng.choice(["decode", "both", "prompts"]) if tokens <= 256 else rng.choice(["both", "prompts"])
    return _lora("", tokens, d_in, d_out, _log_int(rng, 1, 64 if form == "decode" else 16), rng.choice([8, 16, 16, 32, 64]), rng.random() < 0.5,
                 form, rng.choice(["bf16", "bf16", "bf16", "fp16"]), rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _quantised(n_expts, n, k, g):
    """Weights N(0, 0.02) in MXFP4 along k: codes [E, n, k / 2], the even k in the low half of a byte, and scale bytes [E, n, k / 32]"""
    q = torch.empty((n_expts, n, k // 2), dtype=torch.uint8, device=DEV)
    s = torch.empty((n_expts, n, k // 32), dtype=torch.uint8, device=DEV)
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)          # half way between the magnitudes
    for e in range(n_expts):
        w = (torch.randn(n, k // 32, 32, device=DEV, generator=g) * 0.02)
        power = torch.ceil(torch.log2(w.abs().amax(2) / 6.0)).clamp(-120, 120)
        w = w / torch.exp2(power).unsqueeze(2)
        code = (torch.bucketize(w.abs(), steps, out_int32=True) + (w < 0) * 8).to(torch.uint8).view(n, k // 2, 2)
        q[e] = code[:, :, 0] | (code[:, :, 1] << 4)
        s[e] = (power + 127).to(torch.uint8)
    return q, s


def _moe_inputs(case, seed):
    T, E, d, ff = (case[n] for n in ("tokens", "experts", "d_model", "d_ff"))
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    x = torch.randn(T, d, device=DEV, generator=g).to(dt)
    wg = (torch.randn(E, d, device=DEV, generator=g) / d ** 0.5).bfloat16()            # [E, d]: d runs fastest, as the router reads it
    bg = torch.randn(E, device=DEV, generator=g) * (1.0 if case["skew"] else 0.1)
    w1, s1 = _quantised(E, 2 * ff, d, g)                                               # rows 2i and 2i + 1: gate and linear part of output i
    w2, s2 = _quantised(E, d, ff, g)
    b1 = (torch.randn(E, 2 * ff, device=DEV, generator=g) * 0.01).bfloat16()
    b2 = (torch.randn(E, d, device=DEV, generator=g) * 0.01).bfloat16()
    return {"x": x, "wg": wg, "bg": bg, "w1": w1, "s1": s1, "w2": w2, "s2": s2, "b1": b1, "b2": b2, "k": case["top_k"]}


def _lora_inputs(case, seed):
    T, K, N, L, R = (case[n] for n in ("tokens", "d_in", "d_out", "adapters", "rank"))
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    x = torch.randn(T, K, device=DEV, generator=g).to(dt)
    w = (torch.randn(N, K, device=DEV, generator=g) / K ** 0.5).to(dt)                 # [N, K]: K runs fastest
    bias = (torch.randn(N, device=DEV, generator=g) * 0.1).to(dt) if case["bias"] else None
    ranks = _ranks(case)
    a = torch.randn(L, R, K, device=DEV, generator=g) / K ** 0.5
    b = torch.randn(L, N, R, device=DEV, generator=g) * 0.1
    inside = torch.arange(R, device=DEV) < torch.tensor(ranks, device=DEV).unsqueeze(1)    # [L, R]
    a, b = (a * inside.unsqueeze(2)).to(dt), (b * inside.unsqueeze(1)).to(dt)
    scale = [32.0 / r for r in ranks]
    return {"x": x, "w": w, "bias": bias, "a": a, "b": b, "ranks": ranks, "scale": scale, "indx": _adapter_of(case, g)}


def _ranks(case):
    R, few = case["rank"], [r for r in (8, 16, 32, 64) if r <= case["rank"]]
    return [few[-1 - i % len(few)] if case["mixed"] else R for i in range(case["adapters"])]


def _adapter_of(case, g):
    """Adapter of every token, -1 for none (an eighth of the requests)"""
    T, L = case["tokens"], case["adapters"]
    single = torch.randint(0, L, (T,), device=DEV, generator=g, dtype=torch.int32)
    single = torch.where(torch.rand(T, device=DEV, generator=g) < 0.125, -1, single)
    if case["form"] == "decode":
        return single
    n = _requests(case)
    ends = torch.sort(torch.randint(1, T + 1, (n - 1,), device=DEV, generator=g)).values       # ragged prompts
    request = torch.bucketize(torch.arange(T, device=DEV), ends, right=True)
    indx = single[:n][request]
    if case["form"] == "both":
        indx = torch.where(torch.arange(T, device=DEV) >= T - T // 8, single, indx)
    return indx.to(torch.int32)


def _requests(case):
    return min(case["tokens"], case["adapters"] + 2)


def prepare(case, seed):
    if case["kind"] == "moe":
        s = _moe_inputs(case, seed)
        if own:
            s = _moe_handles(s)
    else:
        s = _lora_inputs(case, seed)
        if own:
            s = _lora_handles(s)
    return {"kind": case["kind"], **s}


def _moe_handles(s):
    import triton_b200 as tb
    from triton_b200.moe import MoeLayerWeights
    from triton_b200.tensor_details.layout import make_default_matmul_mxfp4_w_layout, make_default_matmul_mxfp4_w_scale_layout

    def laid_out(q, scale):
        return (tb.convert_layout(tb.wrap_torch_tensor(q.transpose(1, 2), dtype=tb.FP4), make_default_matmul_mxfp4_w_layout(mx_axis=-2)),
                tb.convert_layout(tb.wrap_torch_tensor(scale.transpose(1, 2)), make_default_matmul_mxfp4_w_scale_layout(mx_axis=-2)))

    lw = MoeLayerWeights(*laid_out(s["w1"], s["s1"]), s["b1"], *laid_out(s["w2"], s["s2"]), s["b2"], ALPHA, LIMIT)
    return {"x": s["x"], "wg": tb.prepare_router_weight(s["wg"].t()), "bg": s["bg"], "lw": lw, "k": s["k"]}


def _lora_handles(s):
    import triton_b200 as tb
    adapters = tb.prepare_lora_adapters([s["a"][i, :r].t() for i, r in enumerate(s["ranks"])],
                                        [s["b"][i, :, :r].t() for i, r in enumerate(s["ranks"])], s["scale"])
    return {"x": s["x"], "w": tb.prepare_projection_weight(s["w"].t()), "bias": s["bias"], "adapters": adapters, "indx": s["indx"]}


# ---------------------------------------------------------------------------------------------------------
# one pass

def run(state):
    if own:
        import triton_b200 as tb
        if state["kind"] == "moe":
            return tb.moe_layer_tokens(state["x"], state["wg"], state["bg"], state["lw"], state["k"])
        return tb.matmul_lora(state["x"], state["w"], state["bias"], state["adapters"], state["indx"])
    return _plain_moe(state) if state["kind"] == "moe" else _plain_lora(state)


def _values(q, scale):
    """Codes [.., n, k / 2] and scale bytes [.., n, k / 32] -> fp32 [.., n, k]"""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).int()
    v = table[codes].unflatten(-1, (-1, 32)) * torch.exp2(scale.float() - 127).unsqueeze(-1)
    return v.flatten(-2)


def _plain_moe(s):
    x, k = s["x"].float(), s["k"]
    T = x.shape[0]
    logits = x @ s["wg"].float().t() + s["bg"]
    vals, indx = torch.sort(logits, dim=1, descending=True, stable=True)               # equal logits: the lowest index first
    gates, expt = torch.softmax(vals[:, :k], dim=1), indx[:, :k].reshape(-1)
    rows = x.repeat_interleave(k, 0).unsqueeze(2)                                      # [T k, d, 1]
    h = torch.bmm(_values(s["w1"][expt], s["s1"][expt]), rows).squeeze(2) + s["b1"][expt].float()
    gate, lin = h[:, 0::2].clamp(max=LIMIT), h[:, 1::2].clamp(-LIMIT, LIMIT)
    h = gate * torch.sigmoid(ALPHA * gate) * (lin + 1)
    y = torch.bmm(_values(s["w2"][expt], s["s2"][expt]), h.unsqueeze(2)).squeeze(2) + s["b2"][expt].float()
    return (y.view(T, k, -1) * gates.unsqueeze(2)).sum(1).to(s["x"].dtype)


def _plain_lora(s):
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    L, R, _ = a.shape
    y = x @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    scale = torch.tensor(s["scale"], device=x.device)
    mine = (s["indx"].unsqueeze(1) == torch.arange(L, device=x.device)) * scale        # [T, L]
    t = (x @ a.reshape(L * R, -1).t()).view(-1, L, R) * mine.unsqueeze(2)
    return (y + t.view(-1, L * R) @ b.transpose(1, 2).reshape(L * R, -1)).to(s["x"].dtype)


# ---------------------------------------------------------------------------------------------------------
# from the definition, in 64 bits

def exact(case, seed):
    return _exact_moe(case, seed) if case["kind"] == "moe" else _exact_lora(case, seed)


def _exact_moe(case, seed):
    s = _moe_inputs(case, seed)
    x, logits = s["x"].double(), s["x"].double() @ s["wg"].double().t() + s["bg"].double()
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)

    def matrix(q, scale):                          # sign, exponent and fraction of every code
        out = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=DEV)
        for half in (0, 1):
            c = (q >> (4 * half)) & 15
            e, m = ((c >> 1) & 3).double(), (c & 1).double()
            mag = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))
            out[:, half::2] = torch.where(c >= 8, -mag, mag)
        return out * torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)

    for t, row in enumerate(logits.tolist()):
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:case["top_k"]]
        weight = [math.exp(row[e] - row[best[0]]) for e in best]
        for e, g in zip(best, weight):
            h = matrix(s["w1"][e], s["s1"][e]) @ x[t] + s["b1"][e].double()
            gate, lin = torch.clamp(h[0::2], max=LIMIT), torch.clamp(h[1::2], min=-LIMIT, max=LIMIT)
            h = gate / (1 + torch.exp(-ALPHA * gate)) * (lin + 1)
            y[t] += g / math.fsum(weight) * (matrix(s["w2"][e], s["s2"][e]) @ h + s["b2"][e].double())
    return y


def _exact_lora(case, seed):
    s = _lora_inputs(case, seed)
    x = s["x"].double()
    y = torch.matmul(x, s["w"].double().transpose(0, 1))
    if s["bias"] is not None:
        y += s["bias"].double()
    for i, (r, scale) in enumerate(zip(s["ranks"], s["scale"])):
        at = torch.nonzero(s["indx"] == i).squeeze(1)
        y[at] += scale * ((x[at] @ s["a"][i, :r].double().t()) @ s["b"][i, :, :r].double().t())
    return y


# ---------------------------------------------------------------------------------------------------------
def _active_experts(case):
    """Experts that get a token, from one simulated batch"""
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(case["tokens"], case["experts"], generator=g) + torch.randn(case["experts"], generator=g) * (1.0 if case["skew"] else 0.1)
    return int(logits.topk(case["top_k"], dim=1).indices.unique().numel())


def work(case):
    if case["kind"] == "moe":
        T, E, k, d, ff = (case[n] for n in ("tokens", "experts", "top_k", "d_model", "d_ff"))
        per_expert = 3 * d * ff // 2 + 3 * d * ff // 32 + (2 * ff + d) * 2              # packed codes, scales, biases
        return {"bytes": _active_experts(case) * per_expert + E * d * 2 + E * 4 + 2 * T * d * 2, "flops": 6 * T * k * d * ff + 2 * T * E * d}
    T, K, N, L = (case[n] for n in ("tokens", "d_in", "d_out", "adapters"))
    ranks = _ranks(case)
    mean = sum(ranks) / L
    picks = 0.875 * (T if case["form"] == "decode" else _requests(case) + (T // 8 if case["form"] == "both" else 0))
    used = L * (1 - (1 - 1 / L) ** picks) if L > 1 else min(1.0, picks)                 # adapters that some token has, on average
    nbytes = 2 * (T * K + N * K + T * N + (N if case["bias"] else 0)) + 4 * T + used * mean * (K + N) * 2
    return {"bytes": int(nbytes), "flops": int(2 * T * K * N + 0.875 * T * mean * 2 * (K + N))}
