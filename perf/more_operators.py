"""Attention over a paged cache, as a decoder layer runs it: what lays queries, keys and values out, and what reads the cache.

* `rope`: `qk_norm_rope`: the rows of a fused q, k, v projection; an RMS norm per query and key head (where the layer has weights for
  it), the rotation of the token's position on the first `rot` elements of a head, keys and values into their slots of the cache;
* `attention`: `paged_attention`: the last n_b tokens of each sequence attend to its cache; causal, with an optional sliding window outside
  of which only the first `sinks` tokens stay visible;
* `tree`: `tree_attention`: the last n_b tokens of each sequence are drafted ones: each sees the whole context and, of the drafted tokens,
  those whose bits its mask has.

    out_i = sum_j p_ij v_j,    p_ij = exp(scale q_i . k_j) / sum_j' exp(scale q_i . k_j')    over the visible j.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_MAX_BYTES = 2.0 * 131072 * 8 * 128 * 4
_MAX_FLOPS = 4.0 * 8192 * 8192 / 2 * 32 * 128
_MAX_ROPE = 8192 * 80 * 128


def listed():
    return [
        # one token of a 4096-wide model with per-head norms: the smallest call of a decode step
        dict(name="rope_token", family="rope", T=1, Hq=32, Hkv=8, D=128, rot=128, norm=True, interleaved=False, page=16, table="f16", dtype="f16"),
        # a ragged batch on a model that rotates half of a head, neighbours in pairs, without norms; an fp32 table
        dict(name="rope_partial", family="rope", T=67, Hq=28, Hkv=4, D=128, rot=64, norm=False, interleaved=True, page=64, table="f32",
             dtype="bf16"),
        # a long prompt of an 8192-wide model
        dict(name="rope_prompt", family="rope", T=8192, Hq=64, Hkv=8, D=128, rot=128, norm=True, interleaved=False, page=128, table="bf16",
             dtype="bf16"),
        # one sequence decoding, a short context: the smallest call
        dict(name="decode_token", family="attention", B=1, query="one", length=700, ragged=0, Hq=32, Hkv=8, D=128, page=16, window=-1, sinks=0,
             dtype="f16"),
        # 64 sequences decoding together, contexts of one token to 8192
        dict(name="decode_batch", family="attention", B=64, query="one", length=8192, ragged=1, Hq=64, Hkv=8, D=128, page=64, window=-1, sinks=0,
             dtype="bf16"),
        # long conversations on a layer with a window of 4096 and four tokens that stay visible
        dict(name="decode_window", family="attention", B=32, query="one", length=32768, ragged=2, Hq=64, Hkv=8, D=64, page=32, window=4096, sinks=4,
             dtype="f16"),
        # two very long documents
        dict(name="decode_long", family="attention", B=2, query="one", length=131072, ragged=0, Hq=64, Hkv=8, D=128, page=128, window=-1, sinks=0,
             dtype="bf16"),
        # a prompt of 8192 tokens, causal
        dict(name="prompt_causal", family="attention", B=1, query="all", length=8192, ragged=0, Hq=32, Hkv=8, D=128, page=64, window=-1, sinks=0,
             dtype="bf16"),
        # a prompt of 16384 tokens on a layer with a window
        dict(name="prompt_window", family="attention", B=1, query="all", length=16384, ragged=0, Hq=64, Hkv=8, D=64, page=64, window=1024, sinks=4,
             dtype="bf16"),
        # a serving step: chunks of prompts between sequences that decode, heads of 256
        dict(name="chunks_mixed", family="attention", B=12, query="mixed", length=6000, ragged=3, Hq=16, Hkv=2, D=256, page=16, window=-1, sinks=0,
             dtype="f16"),
        # one sequence verifying eight drafted tokens
        dict(name="tree_token", family="tree", B=1, nodes=8, length=908, ragged=0, Hq=32, Hkv=8, D=128, page=16, dtype="f16"),
        # 24 sequences with up to 60 drafted tokens each, contexts up to 16384
        dict(name="tree_batch", family="tree", B=24, nodes=60, length=16384, ragged=4, Hq=32, Hkv=8, D=128, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["rope", "attention", "attention", "attention", "tree", "tree"])
    dtype = rng.choice(["f16", "bf16"])
    D, Hkv, G = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    page = rng.choice([1, 16, 16, 32, 48, 64, 128])
    case = dict(family=family, Hq=Hkv * G, Hkv=Hkv, D=D, page=page, dtype=dtype)
    if family == "rope":
        T = min(_log(rng, 1, 16384), _MAX_ROPE // ((Hkv * G + 2 * Hkv) * D))
        case.update(T=T, rot=rng.choice([D, D, D // 2, D // 4]), norm=rng.random() < 0.7, interleaved=rng.random() < 0.3,
                    table=rng.choice([dtype, "f32"]))
        return case
    case.update(B=_log(rng, 1, 64), length=_log(rng, 1, 131072), ragged=rng.randint(1, 10 ** 6))
    if family == "tree":
        case["nodes"] = _log(rng, 1, 128)
        case["length"] = max(case["length"], case["nodes"])
    else:
        case["query"] = rng.choice(["one", "one", "mixed", "all"])
        case["window"], case["sinks"] = (_log(rng, 1, 8192), rng.choice([0, 1, 4, 64])) if rng.random() < 0.5 else (-1, 0)
    while True:
        w = work(case)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS and case["B"] * case["length"] * Hkv * D <= _MAX_BYTES / 4:
            return case
        if case["B"] > 1:
            case["B"] //= 2
        else:
            case["length"] = max(case["length"] // 2, case.get("nodes", 1))


def _shape(case):
    """(tokens of the call, whole length) of each sequence."""
    B, top = case["B"], case["length"]
    if not case["ragged"]:
        lens = [top] * B
        news = [case["nodes"] if case["family"] == "tree" else top if case["query"] == "all" else 1] * B
        return news, lens
    rng = random.Random(case["ragged"])
    news, lens = [], []
    for b in range(B):
        if case["family"] == "tree":
            n = rng.randint(1, case["nodes"])
            lens.append(max(n, rng.randint(top // 2, top) if b else top))
        else:
            lens.append(_log(rng, 1, top) if b else top)
            long = case["query"] == "all" or (case["query"] == "mixed" and b % 3 == 0)
            n = rng.randint((lens[-1] + 1) // 2, lens[-1]) if long else 1
            if case["query"] == "one" and b and rng.random() < 0.03:
                lens[-1] = 0                              # an unused place of the batch: its row sees nothing
        news.append(n)
    return news, lens


# ---------------------------------------------------------------------------------------------- inputs
def _pages(g, count):
    """Page numbers in no order, from a cache with a few pages more."""
    return torch.randperm(count + 3, generator=g, device="cuda")[:count], count + 3


def _randn(g, dt, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(dt)


def _prepare_rope(case, g, dt):
    T, Hq, Hkv, D, rot, page = (case[n] for n in ("T", "Hq", "Hkv", "D", "rot", "page"))
    heads = Hq + 2 * Hkv
    wide = 1.0 + 7.0 * (torch.rand(heads * D, generator=g, device="cuda") < 0.01)        # a few elements far larger than the others
    s = dict(case, qkv=(torch.randn(T, heads * D, generator=g, device="cuda") * wide).to(dt), qw=None, kw=None)
    if case["norm"]:
        s["qw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        s["kw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
    places = 32768
    angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * \
        1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    s["table"] = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32 if case["table"] == "f32" else dt)
    s["positions"] = (torch.arange(T, device="cuda") + torch.randint(0, places - T, (1,), generator=g, device="cuda")) if T > 256 else \
        torch.randint(0, places, (T,), generator=g, device="cuda")
    ids, blocks = _pages(g, -(-T // page))
    t = torch.arange(T, device="cuda")
    s["slots"] = ids[t // page] * page + t % page
    s["kc"], s["vc"] = _randn(g, dt, blocks, page, Hkv, D), _randn(g, dt, blocks, page, Hkv, D)
    s["q"] = torch.empty(T, Hq, D, dtype=dt, device="cuda")
    return s


def _paths(g, n, words):
    """Masks of a tree of n nodes, a node behind its parent: the bits of a node are its parent's and its own."""
    parent = (torch.rand(n, generator=g, device="cuda") * torch.arange(n, device="cuda")).long().tolist()
    sees = []
    for i in range(n):
        sees.append((sees[parent[i]] if i else 0) | 1 << i)
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    return [[signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in sees]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    if case["family"] == "rope":
        return _prepare_rope(case, g, dt)
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    news, lens = _shape(case)
    T, most = sum(news), max(max(lens), 1)
    width = -(-most // page)
    ids, blocks = _pages(g, B * width)
    s = dict(case, news=news, lens=lens, most=most, scale=D ** -0.5, table=ids.view(B, width).int())
    s["q"] = 2 * _randn(g, dt, T, Hq, D)
    s["kc"] = _randn(g, dt, blocks, page, Hkv, D)
    s["vc"] = _randn(g, dt, blocks, page, Hkv, D) + _randn(g, dt, Hkv, D) / 2
    s["seq"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    if case["family"] == "tree":
        words = -(-max(news) // 64)
        s["mask"] = torch.tensor([row for n in news for row in _paths(g, n, words)], dtype=torch.int64, device="cuda").view(T, words)
    s["out"] = torch.empty(T, Hq, D, dtype=dt, device="cuda")
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
    if s["family"] == "rope":
        v.qk_norm_rope(s["qkv"], s["qw"], s["kw"], s["table"], s["positions"], s["q"], None, s["kc"], s["vc"], s["slots"], _EPS,
                       s["interleaved"])
        return {"q": s["q"], "key_cache": s["kc"], "value_cache": s["vc"]}
    if s["family"] == "tree":
        return v.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["seq"], s["cu"], s["mask"], s["out"], s["scale"], max(s["news"]),
                                s["most"])
    return v.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["seq"], s["cu"], s["out"], s["scale"], s["window"], s["sinks"],
                             max(s["news"]), s["most"])


def _head_norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rope_plain(s):
    T, Hq, Hkv, D, dt = s["T"], s["Hq"], s["Hkv"], s["D"], s["qkv"].dtype
    x = s["qkv"].view(T, Hq + 2 * Hkv, D)
    cos, sin = s["table"][s["positions"]].float().unsqueeze(1).chunk(2, -1)
    q = _rotate(_head_norm(x[:, :Hq].float(), s["qw"]), cos, sin, s["interleaved"]).to(dt)
    k = _rotate(_head_norm(x[:, Hq:Hq + Hkv].float(), s["kw"]), cos, sin, s["interleaved"]).to(dt)
    s["kc"].view(-1, Hkv, D)[s["slots"]] = k
    s["vc"].view(-1, Hkv, D)[s["slots"]] = x[:, Hq + Hkv:]
    return {"q": q, "key_cache": s["kc"], "value_cache": s["vc"]}


_SCORES = 1 << 28                                        # scores held at a time


def _run_plain(s):
    if s["family"] == "rope":
        return _rope_plain(s)
    Hq, Hkv, D, dt = s["Hq"], s["Hkv"], s["D"], s["q"].dtype
    G, out, at = Hq // Hkv, torch.zeros(s["q"].shape, device="cuda"), 0
    for b, (n, length) in enumerate(zip(s["news"], s["lens"])):
        first = length - n                                # place of the first token of the call
        step = max(1, min(n, _SCORES // (Hq * max(length, 1))))
        if s["family"] == "attention" and s["window"] > 0:
            step = max(1, min(n, max(s["window"], 256)))
        for i in range(0, n if length else 0, step):
            m = min(step, n - i)
            place = torch.arange(first + i, first + i + m, device="cuda")[:, None]
            keys = torch.arange(0, length if s["family"] == "tree" else max(first + i + m, 0), device="cuda")
            if s["family"] == "attention" and s["window"] > 0:
                low = max(0, first + i - s["window"] + 1)
                keys = torch.cat([keys[:min(s["sinks"], low)], keys[low:]])
            pages = s["table"][b].long()[keys // s["page"]] * s["page"] + keys % s["page"]
            k = s["kc"].view(-1, Hkv, D)[pages].permute(1, 2, 0).float().contiguous()      # Hkv, D, keys
            v = s["vc"].view(-1, Hkv, D)[pages].transpose(0, 1).float().contiguous()
            if s["family"] == "tree":
                node = keys - first
                word = s["mask"][at + i:at + i + m][:, (node.clamp_min(0) // 64)]
                visible = (node < 0) | ((word >> (node.clamp_min(0) % 64)) & 1).bool()
            else:
                visible = keys <= place
                if s["window"] > 0:
                    visible = visible & ((place - keys < s["window"]) | (keys < s["sinks"]))
            q = s["q"][at + i:at + i + m].view(m, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * m, D).float()
            score = torch.bmm(q, k).view(Hkv, G, m, -1) * s["scale"]
            score = score.masked_fill(~visible, -math.inf)
            weight = torch.exp(score - score.amax(-1, keepdim=True))
            sums = weight.sum(-1, keepdim=True)
            o = torch.bmm(weight.view(Hkv, G * m, -1), v).view(Hkv, G, m, D) / sums
            out[at + i:at + i + m] = o.permute(2, 0, 1, 3).reshape(m, Hq, D)
        at += n
    return out.to(dt)


# ---------------------------------------------------------------------------------------------- what a pass needs
def _seen(count, window, sinks, first):
    """Sum over i < count of the keys that place first + i sees."""
    if window < 0:
        return count * (first + 1) + count * (count - 1) / 2.0
    total = 0
    for i in range(count):
        p = first + i
        total += min(p + 1, window) + max(0, min(sinks, p + 1 - window))
    return total


def work(case):
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["family"] == "rope":
        elements = case["T"] * (Hq + 2 * Hkv) * D
        table = case["T"] * case["rot"] * (4 if case["table"] == "f32" else 2)
        return {"bytes": 4.0 * elements + table + 16.0 * case["T"], "flops": 8.0 * case["T"] * (Hq + Hkv) * D}
    news, lens = _shape(case)
    tree = case["family"] == "tree"
    keys, pairs = 0.0, 0.0
    for n, length in zip(news, lens):
        if not length:
            continue
        first = length - n
        if tree:
            keys += length
            pairs += n * (first + 0.6 + math.log(n))         # a node of a random tree sees about that many, itself among them
            continue
        low = 0 if case["window"] < 0 else max(0, first - case["window"] + 1)
        keys += length - low + min(case["sinks"], low)
        pairs += _seen(n, case["window"], case["sinks"], first)
    return {"bytes": 4.0 * sum(news) * Hq * D + 4.0 * keys * Hkv * D + (8.0 * sum(news) if tree else 0.0), "flops": 4.0 * pairs * Hq * D}


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_rope(case, seed):
    s = prepare(case, seed)
    Hq, Hkv, D, half = s["Hq"], s["Hkv"], s["D"], s["rot"] // 2
    rows = s["qkv"].double().view(s["T"], -1, D)
    angle = s["table"].double().index_select(0, s["positions"])
    turn = torch.complex(angle[:, :half], angle[:, half:])[:, None]

    def head(x, w):
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + _EPS) * w.double()
        y = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["interleaved"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    kc, vc = s["kc"].double(), s["vc"].double()
    kc.view(-1, Hkv, D).index_copy_(0, s["slots"], head(rows[:, Hq:Hq + Hkv], s["kw"]))
    vc.view(-1, Hkv, D).index_copy_(0, s["slots"], rows[:, Hq + Hkv:])
    return {"q": head(rows[:, :Hq], s["qw"]), "key_cache": kc, "value_cache": vc}


def exact(case, seed):
    if case["family"] == "rope":
        return _exact_rope(case, seed)
    s = prepare(case, seed)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, begin = s["Hq"] // s["Hkv"], 0
    for b in range(s["B"]):
        n, L = s["news"][b], s["lens"][b]
        if L == 0:
            begin += n
            continue
        blocks = s["table"][b, :-(-L // s["page"])].long()
        K = s["kc"].index_select(0, blocks).flatten(0, 1)[:L].double()
        V = s["vc"].index_select(0, blocks).flatten(0, 1)[:L].double()
        j = torch.arange(L, device="cuda").view(1, -1)
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            p = torch.arange(L - n + lo, L - n + hi, device="cuda").view(-1, 1)
            if s["family"] == "tree":
                bits = s["mask"][begin + lo:begin + hi]
                bits = (bits.unsqueeze(-1) >> torch.arange(64, device="cuda")).bitwise_and(1).flatten(1)[:, :n].bool()
                hidden = torch.cat([torch.zeros(hi - lo, L - n, dtype=torch.bool, device="cuda"), ~bits], 1)
            else:
                hidden = j > p
                if s["window"] > 0:
                    hidden = hidden | ((j <= p - s["window"]) & (j >= s["sinks"]))
            for h in range(s["Hq"]):
                logit = (s["q"][begin + lo:begin + hi, h].double() @ K[:, h // group].t()) * s["scale"]
                logit[hidden] = float("-inf")
                out[begin + lo:begin + hi, h] = torch.softmax(logit, 1) @ V[:, h // group]
        begin += n
    return out
