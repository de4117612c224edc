"""The linears of a decoder layer in 8-bit integers (W8A8): activations quantised per token as they come in, weights
quantised per output channel when they were made.

A row v becomes codes q = rint(127 v / m), ties to even, with m = max(max|v|, 2^-40) and the scale s = m / 127, and

    out[i, n] = (sum_k q[i, k] w[n, k]) s[i] w_scale[n] + bias[n].

* `linear`: `gemm_int8` on 16-bit activations, or on codes and scales that the caller has already;
* `norm`: `resadd_norm_gemm_int8`: residual add and RMS norm in front of it;
* `silu`: `silu_mul_gemm_int8`: SiLU(gate) x up in front of it;
* `moe`: `moe_forward_full_int8`: selection, routed experts and a gated shared expert.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_FLOOR = 2.0 ** -40
_EPS = 1e-6
_MAX_FLOPS = 2.0 * 2048 * 4096 * 14336


def listed():
    return [
        # output projection of a 4096-wide model, one token: the smallest call of a decode step
        dict(name="linear_token", family="linear", M=1, K=4096, N=4096, codes=False, bias=False, dtype="f16"),
        # eight sequences on the gate and up projections, activations that the caller has quantised for several products
        dict(name="linear_batch8", family="linear", M=8, K=4096, N=14336, codes=True, bias=False, dtype="bf16"),
        # 64 sequences decoding together, with a bias
        dict(name="linear_batch64", family="linear", M=64, K=5120, N=5120, codes=False, bias=True, dtype="f16"),
        # a prefill chunk of ragged length onto an odd number of columns (a vocabulary's slice)
        dict(name="linear_ragged", family="linear", M=201, K=2048, N=12289, codes=True, bias=True, dtype="bf16"),
        # a long prompt on the same model's projections
        dict(name="linear_prefill", family="linear", M=2048, K=4096, N=14336, codes=False, bias=False, dtype="bf16"),
        # residual add, norm and projection of one token
        dict(name="norm_token", family="norm", M=1, K=4096, N=14336, bias=False, dtype="f16"),
        # the same of a prompt of ragged length in front of the fused q, k, v projection
        dict(name="norm_prefill", family="norm", M=1000, K=4096, N=6144, bias=True, dtype="bf16"),
        # the down projection of two sequences
        dict(name="silu_decode", family="silu", M=2, K=14336, N=4096, bias=False, dtype="bf16"),
        # and of a long prompt
        dict(name="silu_prefill", family="silu", M=2048, K=14336, N=4096, bias=False, dtype="f16"),
        # one token through a mixture-of-experts layer of 128 experts with its shared expert
        dict(name="moe_token", family="moe", T=1, E=128, k=8, H=2048, I=768, shared=1, dtype="bf16"),
        # 48 sequences decoding together: three rows per expert on average
        dict(name="moe_batch", family="moe", T=48, E=128, k=8, H=2048, I=768, shared=1, dtype="f16"),
        # a long prompt
        dict(name="moe_prefill", family="moe", T=4096, E=128, k=8, H=2048, I=768, shared=1, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["linear", "linear", "norm", "silu", "moe", "moe"])
    dtype = rng.choice(["f16", "bf16"])
    if family == "moe":
        E = rng.choice([8, 16, 32, 64, 128])
        k = rng.choice([j for j in (1, 2, 4, 6, 8) if j <= E])
        H, I = 64 * rng.randint(8, 64), 16 * _log(rng, 16, 128)
        while 3 * E * H * I > 3 * 128 * 2048 * 768:
            E //= 2
            k = min(k, E)
        shared = rng.randint(0, 1)
        T = _log(rng, 1, 4096)
        while 6.0 * T * (k + shared) * H * I > 6.0 * 4096 * 9 * 2048 * 768:
            T //= 2
        return dict(family=family, T=T, E=E, k=k, H=H, I=I, shared=shared, dtype=dtype)
    K, N = 16 * _log(rng, 32, 1024), _log(rng, 512, 16384)
    N = N | 1 if rng.random() < 0.2 else N // 8 * 8
    M = _log(rng, 1, 2048)
    while 2.0 * M * K * N > _MAX_FLOPS:
        M //= 2
    case = dict(family=family, M=M, K=K, N=N, bias=rng.random() < 0.3, dtype=dtype)
    if family == "linear":
        case["codes"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _codes_like_weights(g, *shape):
    """Codes of normally distributed weights: the largest of a row is about 3.7 standard deviations."""
    return torch.randn(*shape, generator=g, device="cuda").mul_(34.0).round_().clamp_(-127, 127).to(torch.int8)


def _scales(g, *shape):
    """max|w| / 127 of N(0, 0.02) weights, from channel to channel."""
    return 0.02 / 34.0 * (0.7 + 0.6 * torch.rand(*shape, generator=g, device="cuda"))


def _rows(g, rows, cols, dt):
    """Activations with a few columns far larger than the others, as hidden states have them."""
    wide = 1.0 + 7.0 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
    return (torch.randn(rows, cols, generator=g, device="cuda") * wide).to(dt)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    if case["family"] == "moe":
        T, E, H, I = case["T"], case["E"], case["H"], case["I"]
        s = dict(case, x=_rows(g, T, H, dt), logits=torch.randn(T, E, generator=g, device="cuda").to(dt),
                 w13=_codes_like_weights(g, E, 2 * I, H), s13=_scales(g, E, 2 * I), w2=_codes_like_weights(g, E, H, I),
                 s2=_scales(g, E, H), sw13=None, ss13=None, sw2=None, ss2=None, gw=None)
        if case["shared"]:
            s.update(sw13=_codes_like_weights(g, 2 * I, H), ss13=_scales(g, 2 * I), sw2=_codes_like_weights(g, H, I),
                     ss2=_scales(g, H), gw=(torch.randn(1, H, generator=g, device="cuda") * 0.02).to(dt))
        s["out"] = torch.empty(T, H, dtype=dt, device="cuda")
        return s
    M, K, N = case["M"], case["K"], case["N"]
    s = dict(case, w=_codes_like_weights(g, N, K), ws=_scales(g, N), xs=None, b=None)
    if case["bias"]:
        s["b"] = torch.randn(N, generator=g, device="cuda").to(dt)
    if case["family"] == "linear":
        s["x"] = _rows(g, M, K, dt)
        if case["codes"]:
            s["x"], s["xs"] = _codes_like_weights(g, M, K), 0.01 + 0.04 * torch.rand(M, generator=g, device="cuda")
    elif case["family"] == "norm":
        s["x"], s["res"] = _rows(g, M, K, dt), _rows(g, M, K, dt)
        s["nw"] = (1.0 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(dt)
        s["res_out"] = torch.empty(M, K, dtype=dt, device="cuda")
    else:
        s["x"] = _rows(g, M, 2 * K, dt)
    s["out"] = torch.empty(M, N, dtype=dt, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------- one pass
def _calls():
    package = os.path.abspath("llm-scaler_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import custom_esimd_kernels_vllm as v
    return v


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    v = _calls()
    if s["family"] == "linear":
        return v.gemm_int8(s["x"], s["xs"], s["w"], s["ws"], s["b"], s["out"])
    if s["family"] == "norm":
        out = v.resadd_norm_gemm_int8(s["x"], s["res"], s["res_out"], s["nw"], s["w"], s["ws"], s["b"], s["out"], _EPS)
        return {"out": out, "residual": s["res_out"]}
    if s["family"] == "silu":
        return v.silu_mul_gemm_int8(s["x"], s["w"], s["ws"], s["b"], s["out"])
    return v.moe_ops.moe_forward_full_int8(s["x"], s["logits"], s["out"], s["w13"], s["s13"], s["sw13"], s["ss13"], s["w2"],
                                           s["s2"], s["sw2"], s["ss2"], s["gw"], s["k"], s["shared"], s["E"])


def _quantised(v):
    """Codes (as 32-bit numbers) and scales of the rows of v."""
    m = v.abs().amax(-1, keepdim=True).clamp_min(_FLOOR)
    return torch.round(v * 127.0 / m), m / 127.0


def _product(q, s, w, ws):
    """Rows of q against rows of w, over any leading dimension; codes are whole, so 32-bit sums lose nothing that shows."""
    return torch.matmul(q, w.transpose(-1, -2).contiguous().float()) * s * ws.unsqueeze(-2)


def _silu_mul(gate_up):
    gate, up = gate_up.chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(s):
    if s["family"] == "moe":
        return _moe_plain(s)
    dt, x, residual = s["out"].dtype, s["x"].float(), None
    if s["family"] == "linear" and s["codes"]:
        q, sc = x, s["xs"].unsqueeze(1)
    else:
        if s["family"] == "norm":
            x = x + s["res"].float()
            residual = x.to(dt)
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * s["nw"].float()
        elif s["family"] == "silu":
            x = _silu_mul(x)
        q, sc = _quantised(x)
    out = _product(q, sc, s["w"], s["ws"])
    if s["b"] is not None:
        out = out + s["b"].float()
    return out.to(dt) if residual is None else {"out": out.to(dt), "residual": residual}


def _expert(q, sc, w13, s13, w2, s2):
    """One expert, or one per leading index, on rows of codes: 32-bit results."""
    return _product(*_quantised(_silu_mul(_product(q, sc, w13, s13))), w2, s2)


def _moe_plain(s):
    T, E, k, dt = s["T"], s["E"], s["k"], s["out"].dtype
    logits = s["logits"].float()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    top = torch.softmax(logits, 1).gather(1, ids)
    top = (top / top.sum(1, keepdim=True)).to(dt).float()
    q, sc = _quantised(s["x"].float())
    flat = ids.reshape(-1)
    token = torch.arange(T * k, device="cuda") // k
    if T * k <= E:                                        # a matrix per (token, route)
        y = _expert(q[token].unsqueeze(1), sc[token].unsqueeze(1), s["w13"][flat], s["s13"][flat], s["w2"][flat], s["s2"][flat]).squeeze(1)
    else:                                                 # rows of an expert together, padded to the most that one has
        order = torch.argsort(flat, stable=True)
        expert, counts = flat[order], torch.bincount(flat, minlength=E)
        place = torch.arange(T * k, device="cuda") - (counts.cumsum(0) - counts)[expert]
        most = int(counts.max())
        rows = torch.zeros(E, most, q.shape[1], device="cuda")
        scales = torch.zeros(E, most, 1, device="cuda")
        rows[expert, place], scales[expert, place] = q[token[order]], sc[token[order]]
        y = torch.empty(T * k, q.shape[1], device="cuda")
        y[order] = _expert(rows, scales, s["w13"], s["s13"], s["w2"], s["s2"])[expert, place]
    out = (y.view(T, k, -1) * top.unsqueeze(2)).sum(1)
    if s["shared"]:
        gate = torch.sigmoid((s["x"].float() * s["gw"].float()).sum(1, keepdim=True))
        out = out + gate * _expert(q, sc, s["sw13"], s["ss13"], s["sw2"], s["ss2"])
    return out.to(dt)


# ---------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["family"] == "moe":
        T, E, k, H, I, shared = (case[n] for n in ("T", "E", "k", "H", "I", "shared"))
        experts = E * (1.0 - (1.0 - k / E) ** T) + shared
        return {"bytes": experts * (3.0 * H * I + 4 * (2 * I + H)) + 2.0 * T * (2 * H + E), "flops": 6.0 * T * (k + shared) * H * I}
    M, K, N = case["M"], case["K"], case["N"]
    per = {"linear": 1 if case.get("codes") else 2, "norm": 6, "silu": 4}[case["family"]]     # bytes per activation
    return {"bytes": float(per) * M * K + N * K + 4.0 * N + 2.0 * M * N + (2.0 * N if case["bias"] else 0), "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def _int8_rows(v):
    largest = torch.maximum(v.abs().max(dim=1).values, torch.tensor(_FLOOR, dtype=torch.float64, device=v.device))
    return (127.0 * v / largest[:, None]).round(), largest / 127.0


def _linear64(codes, scale, w, ws):
    return (codes @ w.double().t()) * torch.outer(scale, ws.double())


def _gated64(rows, half):
    g = rows[:, :half]
    return g * torch.sigmoid(g) * rows[:, half:]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["family"] == "moe":
        k, I, dt = case["k"], case["I"], s["out"].dtype
        codes, scale = _int8_rows(x)

        def through(rows, w13, s13, w2, s2):
            h, hs = _int8_rows(_gated64(_linear64(codes[rows], scale[rows], w13, s13), I))
            return _linear64(h, hs, w2, s2)

        total = torch.zeros_like(x)
        prob = s["logits"].double().exp()
        chosen = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :k]
        weight = prob.gather(1, chosen)
        weight = (weight / weight.sum(1, keepdim=True)).to(dt).double()       # routing weights are 16-bit numbers by definition
        for e in range(case["E"]):
            rows, at = (chosen == e).nonzero(as_tuple=True)
            if rows.numel():
                total[rows] += weight[rows, at][:, None] * through(rows, s["w13"][e], s["s13"][e], s["w2"][e], s["s2"][e])
        if case["shared"]:
            every = torch.arange(case["T"], device=x.device)
            total += torch.sigmoid(x @ s["gw"].double().t()) * through(every, s["sw13"], s["ss13"], s["sw2"], s["ss2"])
        return total
    residual = None
    if case["family"] == "norm":
        residual = x + s["res"].double()
        x = residual / torch.sqrt(residual.pow(2).sum(1, keepdim=True) / case["K"] + _EPS) * s["nw"].double()
    elif case["family"] == "silu":
        x = _gated64(x, case["K"])
    codes, scale = (x, s["xs"].double()) if case.get("codes") else _int8_rows(x)
    out = _linear64(codes, scale, s["w"], s["ws"])
    if s["b"] is not None:
        out += s["b"].double()[None]
    return out if residual is None else {"out": out, "residual": residual}
