"""Norms of query and key heads with the rotation and the write to the cache, against 64-bit math.

Tolerance: an element passes through at most D / 16 + 5 additions of the sum of squares (half of whose relative error comes through the square
root), a root, a quotient and two products, below 24 steps of 2^-24 of itself; a rotated one is the sum of two such terms with two roundings more.
Then one rounding to 16 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTS = [torch.float16, torch.bfloat16]
EPS = 1e-6


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


def _table(places, rot, dtype, dev):
    angle = torch.arange(places, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype).to(dev)


def _head(x, w, cs, interleaved):
    """-> y, the sum of magnitudes of its terms."""
    x, half = x.double(), cs.shape[1] // 2
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
    y, size = x.clone(), x.abs()
    c, s = cs.double()[:, None, :half], cs.double()[:, None, half:]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size = size.clone()
    size[..., one], size[..., two] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def _check(got, ref, size, dt):
    tol = torch.finfo(dt).eps / 2 * ref.abs() * (1 + 2.0 ** -10) + 28 * 2.0 ** -24 * size + (2.0 ** -25 if dt == torch.float16 else 1e-40)
    worst = ((got.double() - ref).abs() / tol).max().item() if ref.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} of the tolerance"


def _inputs(dev, T, Hq, Hkv, D, rot, dt, seed, norm=True, places=500, page=16, table=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * (1 + 9 * (torch.rand((Hq + 2 * Hkv) * D, generator=g) < 0.02))).to(dt).to(dev)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dt).to(dev) for _ in range(2)) if norm else (None, None)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:T].to(dev)
    kc, vc = (torch.full((pages, page, Hkv, D), 3.0, dtype=dt, device=dev) for _ in range(2))
    return x, qw, kw, _table(places, rot, table or dt, dev), torch.randint(0, places, (T,), generator=g).to(dev), kc, vc, slots


def _compare(got_q, got_k, kc, vc, x, qw, kw, table, positions, slots, Hq, Hkv, D, interleaved):
    T, dt = x.shape[0], x.dtype
    heads = x.reshape(T, -1, D)
    _check(got_q, *_head(heads[:, :Hq], qw, table[positions], interleaved), dt)
    ref, size = _head(heads[:, Hq:Hq + Hkv], kw, table[positions], interleaved)
    if got_k is not None:
        _check(got_k, ref, size, dt)
    if kc is not None:
        _check(kc.reshape(-1, Hkv, D)[slots], ref, size, dt)
        assert torch.equal(vc.reshape(-1, Hkv, D)[slots], heads[:, Hq + Hkv:])
        rest = torch.ones(kc.shape[0] * kc.shape[1], dtype=torch.bool, device=kc.device)
        rest[slots] = False
        assert (kc.reshape(-1, Hkv, D)[rest] == 3).all() and (vc.reshape(-1, Hkv, D)[rest] == 3).all()


@pytest.mark.parametrize("T", [1, 2, 7, 33, 300])
@pytest.mark.parametrize("Hq,Hkv,D,rot", [(4, 1, 64, 64), (8, 8, 64, 16), (5, 2, 128, 128), (28, 4, 128, 64), (16, 2, 256, 64), (3, 1, 256, 256), (2, 1, 128, 0)])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_all_outputs(v, dev, T, Hq, Hkv, D, rot, dt, interleaved):
    for norm, table in ((True, dt), (False, torch.float32)):
        x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, T, Hq, Hkv, D, rot, dt, T + Hq + D + rot, norm, table=table)
        q, k = (torch.full((T, h, D), float("nan"), dtype=dt, device=dev) for h in (Hq, Hkv))
        before = x.clone()
        assert v.qk_norm_rope(x, qw, kw, cs, pos, q, k, kc, vc, slots, EPS, interleaved) is q
        assert torch.equal(x, before)
        _compare(q, k, kc, vc, x, qw, kw, cs, pos, slots, Hq, Hkv, D, interleaved)


@pytest.mark.parametrize("norms", [(True, False), (False, True)])
def test_one_norm_alone(v, dev, norms):
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, 9, 4, 2, 128, 64, torch.bfloat16, 1)
    qw, kw = qw if norms[0] else None, kw if norms[1] else None
    q = torch.empty(9, 4, 128, dtype=x.dtype, device=dev)
    v.qk_norm_rope(x, qw, kw, cs, pos, q, None, kc, vc, slots, EPS)
    _compare(q, None, kc, vc, x, qw, kw, cs, pos, slots, 4, 2, 128, False)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_in_place_and_strides(v, dev, dt, D):
    """Queries and keys over the projection's own columns, rows of a wider array, caches as halves of one array and with heads outside."""
    T, Hq, Hkv = 21, 6, 2
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, T, Hq, Hkv, D, D // 2, dt, D)
    q, k = (torch.empty(T, h, D, dtype=dt, device=dev) for h in (Hq, Hkv))
    v.qk_norm_rope(x, qw, kw, cs, pos, q, k, kc, vc, slots, EPS)
    wide = torch.full((T, 12 * D), 2.0, dtype=dt, device=dev)
    rows = wide[:, D:11 * D]
    rows.copy_(x)
    both = torch.full((kc.shape[0], 2, 16, Hkv, D), 3.0, dtype=dt, device=dev)
    v.qk_norm_rope(rows, qw, kw, cs, pos, rows[:, :Hq * D].unflatten(1, (Hq, D)), rows[:, Hq * D:-Hkv * D].unflatten(1, (Hkv, D)),
                   both[:, 0], both[:, 1], slots, EPS)
    assert torch.equal(rows[:, :Hq * D], q.flatten(1)) and torch.equal(rows[:, Hq * D:-Hkv * D], k.flatten(1))
    assert torch.equal(rows[:, -Hkv * D:], x[:, -Hkv * D:]) and (wide[:, :D] == 2).all() and (wide[:, 11 * D:] == 2).all()
    assert torch.equal(both[:, 0], kc) and torch.equal(both[:, 1], vc)
    heads = torch.full((2, kc.shape[0], Hkv, 16, D), 3.0, dtype=dt, device=dev).transpose(2, 3)
    turned = torch.empty(Hq, T, D, dtype=dt, device=dev).transpose(0, 1)
    v.qk_norm_rope(x, qw, kw, cs, pos, turned, None, heads[0], heads[1], slots, EPS)
    assert torch.equal(turned, q) and torch.equal(heads[0], kc) and torch.equal(heads[1], vc)


def test_slots_and_positions_outside(v, dev):
    T = 12
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, T, 4, 2, 128, 64, torch.float16, 4)
    places = kc.shape[0] * kc.shape[1]
    out = torch.tensor([-1, -2 ** 40, places, 2 ** 40], device=dev)
    slots[:4] = out
    pos[4:8] = torch.tensor([-1, 500, 2 ** 40, -2 ** 62], device=dev)
    q = torch.empty(T, 4, 128, dtype=x.dtype, device=dev)
    v.qk_norm_rope(x, qw, kw, cs, pos, q, None, kc, vc, slots, EPS)
    assert q[4:8, :, :64].isnan().all() and not q[4:8, :, 64:].isnan().any() and not q[:4].isnan().any() and not q[8:].isnan().any()
    written = kc.reshape(places, 2, 128)
    rest = torch.ones(places, dtype=torch.bool, device=dev)
    rest[slots[4:]] = False
    assert (written[rest] == 3).all() and written[slots[4:8]][..., :64].isnan().all() and not written[slots[8:]].isnan().any()
    assert torch.equal(vc.reshape(places, 2, 128)[slots[4:]], x.view(T, 8, 128)[4:, 6:])


def test_rows_of_any_size(v, dev):
    """Zeros, numbers whose squares leave 16 bits, NaN in one head alone."""
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, 4, 4, 2, 128, 128, torch.float16, 6)
    x[0] = 0
    x[1] = 60000
    x[2] = 6e-8
    x[3, 130] = float("nan")
    q, k = (torch.empty(4, h, 128, dtype=x.dtype, device=dev) for h in (4, 2))
    v.qk_norm_rope(x, qw, kw, cs, pos, q, k, kc, vc, slots, EPS)
    assert (q[0] == 0).all() and q[3, 1].isnan().all() and not q[3, [0, 2, 3]].isnan().any() and not k.isnan().any()
    heads = x.view(4, 8, 128)
    _check(q[:3], *_head(heads[:3, :4], qw, cs[pos[:3]], False), x.dtype)
    _check(k, *_head(heads[:, 4:6], kw, cs[pos], False), x.dtype)


def test_long_prompt(v, dev):
    T, Hq, Hkv, D = 9001, 8, 2, 128
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, T, Hq, Hkv, D, 128, torch.bfloat16, 8, places=20000, page=64)
    q = torch.empty(T, Hq, D, dtype=x.dtype, device=dev)
    v.qk_norm_rope(x, qw, kw, cs, pos, q, None, kc, vc, slots, EPS)
    _compare(q, None, kc, vc, x, qw, kw, cs, pos, slots, Hq, Hkv, D, False)


def test_cache_offsets_past_32_bits(v, dev):
    pages, page, Hkv, D = (1 << 32) // (64 * 2 * 128) + 40, 64, 2, 128
    x, qw, kw, cs, pos, _, _, _ = _inputs(dev, 3, 4, Hkv, D, 64, torch.bfloat16, 9)
    kc, vc = (torch.empty(pages, page, Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    slots = torch.tensor([pages * page - 1, 5, pages * page // 2 + 3], device=dev)
    q, k = (torch.empty(3, h, D, dtype=x.dtype, device=dev) for h in (4, Hkv))
    v.qk_norm_rope(x, qw, kw, cs, pos, q, k, kc, vc, slots, EPS)
    assert torch.equal(kc[slots // page, slots % page], k) and torch.equal(vc[slots // page, slots % page], x.view(3, 8, D)[:, 6:])


def test_a_decode_step_in_a_graph(v, dev):
    """The operators as a layer runs them: projection rows -> norm, rotation, cache -> attention, step after step from one graph, and drafted
    tokens behind it; every step against 64-bit math on the cache as it stands."""
    import attention_reference as R
    Hq, Hkv, D, page, B = 8, 2, 128, 16, 3
    g = torch.Generator().manual_seed(11)
    lens, width = [30, 1, 47], 8
    _, qw, kw, cs, _, _, _, _ = _inputs(dev, 1, Hq, Hkv, D, 64, torch.bfloat16, 12)
    kc, vc = (torch.full((B * width + 1, page, Hkv, D), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    table = torch.randperm(B * width, generator=g).view(B, width).int()

    def rows(places):
        """projection rows, positions and slots of tokens at those places of the sequences"""
        n = sum(len(p) for p in places)
        x = torch.randn(n, (Hq + 2 * Hkv) * D, generator=g).bfloat16()
        pos = torch.tensor([j for p in places for j in p])
        slots = torch.tensor([int(table[b, j // page]) * page + j % page for b, p in enumerate(places) for j in p])
        return x, pos, slots
    td = table.to(dev)
    scale = D ** -0.5

    def layer(x, pos, slots, q, seq, cu, out, most, longest, masks=None):
        v.qk_norm_rope(x, qw, kw, cs, pos, q, None, kc, vc, slots, EPS)
        if masks is None:
            return v.paged_attention(q, kc, vc, td, seq, cu, out, scale, 40, 4, most, longest)
        return v.tree_attention(q, kc, vc, td, seq, cu, masks, out, scale, most, longest)

    def buffers(n):
        return [torch.empty(n, Hq, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    # the prompts
    x, pos, slots = (t.to(dev) for t in rows([range(n) for n in lens]))
    q, out = buffers(sum(lens))
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 30, 31, 78], dtype=torch.int32, device=dev)
    layer(x, pos, slots, q, seq, cu, out, 47, 47)
    ref, tol = R.attention(q, kc, vc, td, lens, lens, scale, 40, 4)
    assert ((out.double() - ref).abs() <= tol).all()
    # single tokens from a graph
    x, pos, slots = (t.to(dev) for t in rows([[n] for n in lens]))
    q, out = buffers(B)
    seq, cu = seq + 1, torch.arange(B + 1, dtype=torch.int32, device=dev)
    layer(x, pos, slots, q, seq, cu, out, 1, width * page)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, pos, slots, q, seq, cu, out, 1, width * page)
    for step in range(20):
        now = [n + step for n in lens]
        for t, new in zip((x, pos, slots), rows([[n] for n in now])):
            t.copy_(new)
        seq.copy_(torch.tensor([n + 1 for n in now], dtype=torch.int32))
        graph.replay()
        ref, tol = R.attention(q, kc, vc, td, [n + 1 for n in now], [1] * B, scale, 40, 4)
        assert ((out.double() - ref).abs() <= tol).all(), step
    # drafted tokens: a node stands one place behind its parent, wherever its slot is
    base = [n + 20 for n in lens]
    x, pos, slots = (t.to(dev) for t in rows([range(n, n + 6) for n in base]))
    masks = torch.cat([R.tree_masks(g, 6, 1) for _ in range(B)])
    pos = torch.tensor([n + bin(int(m)).count("1") - 1 for n, part in zip(base, masks.view(B, 6)) for m in part], device=dev)
    q, out = buffers(6 * B)
    seq, cu = torch.tensor([n + 6 for n in base], dtype=torch.int32, device=dev), 6 * cu
    layer(x, pos, slots, q, seq, cu, out, 6, max(base) + 6, masks.to(dev))
    ref, tol = R.attention(q, kc, vc, td, [n + 6 for n in base], [6] * B, scale, masks=masks.to(dev))
    assert ((out.double() - ref).abs() <= tol).all()


def test_refusals(v, dev):
    T, Hq, Hkv, D = 5, 4, 2, 64
    x, qw, kw, cs, pos, kc, vc, slots = _inputs(dev, T, Hq, Hkv, D, 64, torch.float16, 2)
    q, k = (torch.empty(T, h, D, dtype=x.dtype, device=dev) for h in (Hq, Hkv))

    def call(x=x, qw=qw, kw=kw, cs=cs, pos=pos, q=q, k=k, kc=kc, vc=vc, slots=slots):
        return v.qk_norm_rope(x, qw, kw, cs, pos, q, k, kc, vc, slots, EPS)
    call()
    assert call(x=x[:0], pos=pos[:0], q=q[:0], k=k[:0], slots=slots[:0]).shape == (0, Hq, D)
    for kw_, why in ((dict(x=x.float()), "qkv must be"), (dict(x=x[0]), "qkv must be"), (dict(x=x[:, :-8]), r"\(Hq \+ 2 Hkv\) D columns"),
                     (dict(x=x[:, :-D]), "columns"), (dict(x=x[:, :Hq * D]), "columns"), (dict(x=x.t().contiguous().t()), "consecutive"),
                     (dict(x=x[:1].expand(T, -1)), "consecutive"), (dict(q=q[:4]), "q_out must be"), (dict(q=q.bfloat16()), "q_out must be"),
                     (dict(q=q.view(T, 2, 128)), "q_weight must have"), (dict(q=q.view(T, 8, 32)), "heads of 64"),
                     (dict(k=k[:, :1]), "k_out must be"), (dict(k=k.bfloat16()), "k_out must be"),
                     (dict(qw=qw[:32]), "q_weight must have"), (dict(kw=kw.float()), "k_weight must have"),
                     (dict(cs=cs.bfloat16()), "cos_sin must be"), (dict(cs=cs[0]), "cos_sin must be"), (dict(cs=cs[:, :24].contiguous()), "multiple of 16"),
                     (dict(cs=cs[:, :32]), "contiguous"), (dict(cs=cs[:0]), "no rows"), (dict(cs=torch.cat([cs, cs], 1)), "multiple of 16"),
                     (dict(pos=pos.int()), "positions must be"), (dict(pos=pos[:4]), "positions must be"),
                     (dict(kc=None), "together"), (dict(slots=None), "together"), (dict(vc=None), "together"),
                     (dict(k=None, kc=None, vc=None, slots=None), "nowhere"), (dict(slots=slots.int()), "slot_mapping must be"),
                     (dict(slots=slots[:3]), "slot_mapping must be"), (dict(kc=kc[:, :, :1], vc=vc[:, :, :1]), "kv heads"),
                     (dict(kc=kc.bfloat16(), vc=vc.bfloat16()), "input's type"), (dict(vc=kc), "overlap key_cache"),
                     (dict(q=q.as_strided((T, Hq, D), (0, D, 1))), "more than once"), (dict(q=q.as_strided((T, Hq, D), (Hq * D - 8, D, 1))), "more than once"),
                     (dict(kc=kc[:1].expand(kc.shape), vc=vc[:1].expand(vc.shape)), "more than once"),
                     (dict(q=x[:, D:(Hq + 1) * D].unflatten(1, (Hq, D))), "overlap qkv"), (dict(k=q[:, :Hkv]), "overlap q_out"),
                     (dict(pos=pos.cpu()), "same ROCm device"), (dict(q=q.cpu()), "same ROCm device")):
        with pytest.raises(RuntimeError, match=why):
            call(**kw_)
