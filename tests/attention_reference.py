"""Attention over a paged cache in 64 bits, with how far a right result may be off.

A kernel's score is an fp32 sum of D products (each addition at most half a step of 2^-24 of the sum of magnitudes), scaled by a 32-bit factor; a
weight exp(s - m) carries the errors of its score and of the maximum, each rounded weight one half step u of the 16-bit type (fp16: or 2^-32 of
the row's largest, as they are raised by 2^7), and the sum of the weights is of the rounded ones.  Normalised weights are then off by 2 (u + e) relative at most, e
the error of the scores with a few steps of the exponential, the sums and the rescalings; the output is rounded once (u)."""
import torch


def half_step(dt):
    return torch.finfo(dt).eps / 2


def visible(kind, place, L, n, window, sinks, masks):
    """[n, L] of the tokens at places L - n .. (place: their places) against the keys 0 .. L - 1."""
    j = torch.arange(L, device=place.device)
    if kind == "tree":
        ok = (j < L - n).expand(n, L).clone()
        for u in range(n):
            if L - n + u >= 0 and u < 64 * masks.shape[1]:
                ok[:, L - n + u] = (masks[:, u // 64] >> (u % 64) & 1).bool()
        return ok
    ok = j <= place[:, None]
    if window > 0:
        ok = ok & ((place[:, None] - j < window) | (j < sinks))
    return ok


def gather(cache, row, L):
    """[L, heads, D] in 64 bits; second: which keys lie in the cache at all."""
    pages, page = cache.shape[:2]
    j = torch.arange(L, device=cache.device)
    inside = j // page < row.numel()
    ids = torch.where(inside, row.long()[(j // page).clamp_max(max(row.numel() - 1, 0))], -1)
    inside = inside & (ids >= 0) & (ids < pages)
    return cache[ids.clamp(0, pages - 1), j % page].double(), inside


def attention(q, kc, vc, table, lens, news, scale, window=-1, sinks=0, masks=None):
    """-> out, tolerance, both [T, Hq, D] in 64 bits; rows of tokens alone (the first sum(news))."""
    T, (Hq, D), Hkv, u = sum(news), q.shape[1:], kc.shape[2], half_step(q.dtype)
    G = Hq // Hkv
    out, tol = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device), torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    at = 0
    for b, (L, n) in enumerate(zip(lens, news)):
        if not n:
            continue
        rows = q[at:at + n].double()
        if L > 0:
            k, inside = gather(kc, table[b], L)
            v, _ = gather(vc, table[b], L)
            place = torch.arange(L - n, L, device=q.device)
            see = visible("causal" if masks is None else "tree", place, L, n, window, sinks, None if masks is None else masks[at:at + n]) & inside
            for h in range(Hq):
                kh, vh = k[:, h // G], v[:, h // G]
                kh, vh = torch.where(see.any(0)[:, None], kh, 0.0), torch.where(see.any(0)[:, None], vh, 0.0)
                s = (rows[:, h] @ kh.t()) * scale
                size = (rows[:, h].abs() @ kh.abs().t()) * scale
                e = torch.where(see, (D + 8) * 2.0 ** -24 * size, 0.0).amax(1, keepdim=True) + 2.0 ** -18
                s = s.masked_fill(~see, float("-inf"))
                m = s.amax(1, keepdim=True).clamp_min(-1e300)
                w = torch.exp(s - m)
                total = w.sum(1, keepdim=True)
                w = torch.where(total > 0, w / total.clamp_min(1e-300), 0.0)
                o = w @ vh
                parts = w @ vh.abs()
                small = 2.0 ** -32 * (see.double() @ vh.abs()) if q.dtype == torch.float16 else 0.0
                out[at:at + n, h] = o
                tol[at:at + n, h] = u * o.abs() + 2 * (u + 2 * e) * parts + 2 * small + (2.0 ** -24 if q.dtype == torch.float16 else 1e-38)
        at += n
    return out, tol


def tree_masks(g, n, words, own=True):
    """Random trees: the bits of a node are its parent's and its own."""
    sees = []
    for i in range(n):
        parent = int(torch.randint(0, max(i, 1), (1,), generator=g))
        sees.append((sees[parent] if i else 0) | 1 << i)
    if not own:
        sees = [m & ~(1 << i) for i, m in enumerate(sees)]
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    return torch.tensor([[signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in sees], dtype=torch.int64).view(n, words)


def make(dev, seed, lens, news, Hq, Hkv, D, page, dt, words=0, spare=2, spread=2.0):
    """q, key and value cache, table, seq_lens, cu_seqlens: pages in random order, NaN wherever no key lies."""
    g = torch.Generator().manual_seed(seed)
    B, T = len(lens), sum(news)
    width = max(1, -(-max(max(lens), 1) // page))
    used = [-(-max(L, 0) // page) for L in lens]
    ids = torch.randperm(sum(used) + spare, generator=g)
    kc = torch.full((sum(used) + spare, page, Hkv, D), float("nan"))
    vc = kc.clone()
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    for b, L in enumerate(lens):
        mine = ids[at:at + used[b]]
        at += used[b]
        table[b, :used[b]] = mine.int()
        if L > 0:
            k, v = torch.randn(used[b] * page, Hkv, D, generator=g), torch.randn(used[b] * page, Hkv, D, generator=g)
            k[L:], v[L:] = float("nan"), float("nan")
            kc[mine], vc[mine] = k.view(used[b], page, Hkv, D), v.view(used[b], page, Hkv, D)
    q = torch.randn(T, Hq, D, generator=g) * spread
    cu = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32)
    masks = torch.cat([tree_masks(g, n, words) for n in news if n] or [torch.zeros(0, words, dtype=torch.int64)]) if words else None
    move = lambda t: None if t is None else t.to(dev)
    return (move(q.to(dt)), move(kc.to(dt)), move(vc.to(dt)), move(table), torch.tensor(lens, dtype=torch.int32).to(dev), move(cu), move(masks))
