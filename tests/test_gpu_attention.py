"""Attention over a paged cache against 64-bit math: single tokens, prompts, chunks, windows with first tokens that stay visible, drafted trees.
The tolerance of every element is derived in attention_reference."""
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu
DTS = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


def _check(got, ref, tol):
    worst = ((got.double() - ref).abs() / tol.clamp_min(1e-300)).max().item() if ref.numel() else 0.0
    assert not got.isnan().any() and worst <= 1.0, f"{worst:.2f} of the tolerance"


def _run(v, case, lens, news, D, window=-1, sinks=0, out=None, hint_q=None, hint_k=None, scale=None):
    q, kc, vc, table, seq, cu, masks = case
    out = torch.full_like(q, float("nan"), memory_format=torch.contiguous_format) if out is None else out
    scale = D ** -0.5 if scale is None else scale
    hint_q, hint_k = max(news) if hint_q is None else hint_q, max(max(lens), 0) if hint_k is None else hint_k
    if masks is None:
        got = v.paged_attention(q, kc, vc, table, seq, cu, out, scale, window, sinks, hint_q, hint_k)
    else:
        got = v.tree_attention(q, kc, vc, table, seq, cu, masks, out, scale, hint_q, hint_k)
    assert got is out
    return out


def _both(v, dev, seed, lens, news, Hq, Hkv, D, page, dt, window=-1, sinks=0, words=0, **kw):
    case = R.make(dev, seed, lens, news, Hq, Hkv, D, page, dt, words)
    out = _run(v, case, lens, news, D, window, sinks, **kw)
    ref, tol = R.attention(case[0], case[1], case[2], case[3], lens, news, D ** -0.5, window, sinks, case[6])
    _check(out[:sum(news)], ref, tol)
    return case, out


# lengths around a step of 32, a block of 64 and the shares of the workgroups; unused places of the batch; groups that do not divide 32
SINGLE = [([1], 1, 1), ([2, 33], 4, 2), ([31, 32, 33, 63, 64, 65], 8, 1), ([700], 32, 8), ([0, 5, 0, 129], 6, 2), ([1000, 1, 257], 15, 5), ([4097], 16, 1),
          ([64] * 70, 4, 4), ([300, 2000] * 40, 5, 1), ([130, 0, 64], 32, 1), ([77], 33, 1), ([500, 90], 80, 2)]


@pytest.mark.parametrize("lens,Hq,Hkv", SINGLE)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 1), (128, 48), (256, 32)])
@pytest.mark.parametrize("dt", DTS)
def test_single_tokens(v, dev, lens, Hq, Hkv, D, page, dt):
    _both(v, dev, len(lens) + Hq + D, lens, [1] * len(lens), Hq, Hkv, D, page, dt)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 64), (64, 63), (100, 65), (500, 4), (5000, 4), (2**31 - 1, 2**31 - 1), (2**40, 0)])
@pytest.mark.parametrize("D,page", [(64, 32), (128, 16), (256, 7)])
def test_single_tokens_in_a_window(v, dev, window, sinks, D, page):
    lens = [1, 31, 64, 65, 97, 128, 129, 600, 1100, 0]
    case = R.make(dev, window % 1000 + D, lens, [1] * len(lens), 16, 2, D, page, torch.bfloat16)
    out = _run(v, case, lens, [1] * len(lens), D, window, sinks)
    ref, tol = R.attention(*case[:4], lens, [1] * len(lens), D ** -0.5, min(window, 10 ** 6), sinks)
    _check(out, ref, tol)


# prompts: lengths around a block, rows around a tile of 256 (128), groups that do not divide a tile, sequences without tokens
PROMPTS = [([1], [1], 64, 1), ([65], [65], 4, 1), ([64, 128], [64, 128], 2, 2), ([300], [300], 8, 2), ([257, 0, 63], [257, 0, 63], 3, 1),
           ([1000, 70], [513, 70], 4, 2), ([2000], [40], 8, 1), ([900, 40, 300, 1], [1, 40, 200, 1], 4, 2), ([500, 600], [300, 1], 7, 1)]


@pytest.mark.parametrize("lens,news,Hq,Hkv", PROMPTS)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 24)])
@pytest.mark.parametrize("dt", DTS)
def test_prompts(v, dev, lens, news, Hq, Hkv, D, page, dt):
    _both(v, dev, sum(lens) + Hq + D, lens, news, Hq, Hkv, D, page, dt)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (17, 0), (63, 64), (64, 1), (65, 130), (200, 4), (3000, 4)])
@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 8, 1), (128, 64, 4, 4), (256, 16, 6, 2)])
def test_prompts_in_a_window(v, dev, window, sinks, D, page, Hq, Hkv):
    _both(v, dev, window + D, [700, 130, 450, 20], [700, 100, 30, 1], Hq, Hkv, D, page, torch.bfloat16, window, sinks)


TREES = [([8], [8], 4, 1), ([5, 100, 64], [5, 8, 3], 8, 2), ([300, 90, 64, 700], [33, 64, 64, 1], 8, 2), ([1000], [60], 32, 8), ([130, 400], [130, 100], 4, 2),
         ([2500, 1900], [20, 60], 4, 1), ([200, 0, 70], [7, 0, 70], 3, 1), ([6000], [64], 16, 1)]


@pytest.mark.parametrize("lens,news,Hq,Hkv", TREES)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (256, 5)])
@pytest.mark.parametrize("dt", DTS)
def test_trees(v, dev, lens, news, Hq, Hkv, D, page, dt):
    _both(v, dev, sum(lens) + Hq + D, lens, news, Hq, Hkv, D, page, dt, words=-(-max(news) // 64))


@pytest.mark.parametrize("n", [3, 40])
def test_a_chain_is_causal(v, dev, n):
    lens, news = [n + 200, n, 600], [n, n, n - 1]
    case = list(R.make(dev, n, lens, news, 8, 2, 128, 16, torch.bfloat16))
    causal = _run(v, case, lens, news, 128)
    case[6] = torch.tensor([[(2 << i) - 1] for k in news for i in range(k)], device=dev)
    ref, tol = R.attention(*case[:4], lens, news, 128 ** -0.5)
    _check(causal, ref, tol)
    _check(_run(v, case, lens, news, 128), ref, tol)


@pytest.mark.parametrize("D,n,G", [(64, 4, 2), (128, 4, 2), (256, 4, 2), (128, 50, 8)])
def test_rows_that_see_nothing(v, dev, D, n, G):
    """More tokens than keys, no keys, a tree whose nodes see nothing: zeros."""
    lens, news = [n - 2, 0, 1], [n, n, 1]
    case = list(R.make(dev, D, lens, news, 2 * G, 2, D, 16, torch.float16))
    out = _run(v, case, lens, news, D)
    assert (out[:2] == 0).all() and (out[n:2 * n] == 0).all() and (out[2] != 0).any()
    _check(out, *R.attention(*case[:4], lens, news, D ** -0.5))
    case[6] = torch.zeros(2 * n + 1, 1, dtype=torch.int64, device=dev)
    assert (_run(v, case, lens, news, D) == 0).all()


def test_calls_without_rows(v, dev):
    case = R.make(dev, 1, [10], [1], 4, 2, 64, 16, torch.float16)
    q, kc, vc, table, seq, cu, _ = case
    none = q[:0]
    assert v.paged_attention(none, kc, vc, table, seq, cu * 0, torch.empty_like(none), 0.1, -1, 0, 0, 10).shape == (0, 4, 64)
    out = torch.full_like(q, 7.0)
    v.paged_attention(q, kc, vc, table[:0], seq[:0], cu[:1], out, 0.1, -1, 0, 1, 10)
    v.paged_attention(q, kc, vc, table, seq, cu * 0, out, 0.1, -1, 0, 1, 10)          # a sequence without tokens
    assert (out == 7).all()


@pytest.mark.parametrize("n,splits", [(1, False), (9, False), (80, True)])
def test_rows_behind_the_last_sequence_stay(v, dev, n, splits):
    lens, news = [3000, 900], [n, n]
    q, kc, vc, table, seq, cu, _ = R.make(dev, n, lens, news, 8, 2, 128, 16, torch.bfloat16)
    more = torch.cat([q, torch.full((37, 8, 128), float("nan"), dtype=q.dtype, device=dev)])
    out = torch.full_like(more, 5.0)
    v.paged_attention(more, kc, vc, table, seq, cu, out, 0.1, -1, 0, n, 3000)
    assert (out[2 * n:] == 5).all()
    _check(out[:2 * n], *R.attention(q, kc, vc, table, lens, news, 0.1))


# [2600]: few tokens over a long context, in shares of its keys
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("kind", ["prompt", "window", "tree"])
@pytest.mark.parametrize("L,page", [(150, 16), (2600, 16), (2600, 12)])
def test_what_a_token_does_not_see_reaches_nothing(v, dev, D, dt, kind, L, page):
    """Infinities and NaN in keys and values that some tokens of a tile see and others do not: the others' rows keep their bits."""
    lens, news, words = [L, 90], [70, 20], 2 if kind == "tree" else 0
    window, sinks = (40, 3) if kind == "window" else (-1, 0)
    case = R.make(dev, D, lens, news, 4, 2, D, page, dt, words)
    clean = _run(v, case, lens, news, D, window, sinks)
    q, kc, vc, table, seq, cu, masks = case
    for value in (float("inf"), float("-inf"), float("nan")):
        for cache in (1, 2):
            dirty = list(case)
            dirty[cache] = case[cache].clone()
            j = L - 20                                  # of sequence 0, a key of the call's own tokens
            dirty[cache][table[0, j // page].long(), j % page, 0, 5] = value
            out = _run(v, dirty, lens, news, D, window, sinks)
            place = torch.arange(L - 70, L, device=dev)
            see = R.visible("causal" if masks is None else "tree", place, L, 70, window, sinks, None if masks is None else masks[:70])[:, j]
            rows = torch.zeros(90, 4, dtype=torch.bool, device=dev)
            rows[:70, :2] = see[:, None]                # heads 0 and 1 read kv head 0
            assert see.any() and not see.all()
            assert torch.equal(out[~rows], clean[~rows])
            if cache == 2:                              # a value: its column alone
                hit = out[rows]
                assert torch.equal(hit[:, 6:], clean[rows][:, 6:]) and torch.equal(hit[:, :5], clean[rows][:, :5])
                assert (hit[:, 5].isnan() if value != value else hit[:, 5] == value).all()
            else:                                       # a key: a score of -inf takes the key out, any other makes the row NaN
                lost = q[rows][:, 5].double() * value != float("-inf")
                assert torch.equal(out[rows].isnan().all(1), lost) and torch.equal(out[rows].isnan().any(1), lost)


@pytest.mark.parametrize("window,sinks", [(-1, 0), (300, 0), (700, 40), (1200, 129), (64, 1)])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 5), (128, 64), (128, 12), (256, 16), (256, 3)])
def test_few_tokens_over_long_contexts(v, dev, window, sinks, D, page):
    """Equal shares of the keys: tiles that end inside a share, sequences without tokens or with a single one between them, pages outside the cache."""
    lens, news = [2600, 30, 1500, 700, 2100, 64], [40, 30, 1, 0, 61, 3]
    case = R.make(dev, window + D, lens, news, 16, 2, D, page, torch.bfloat16)
    _check(_run(v, case, lens, news, D, window, sinks), *R.attention(*case[:4], lens, news, D ** -0.5, window, sinks))
    table, pages = case[3], case[1].shape[0]
    for b, key, bad in ((0, 1, -1), (0, 2500, pages), (2, 1499, -7), (4, 2040, 2 ** 31 - 1), (4, 1024, -2 ** 31)):
        table[b, key // page] = bad
    _check(_run(v, case, lens, news, D, window, sinks), *R.attention(*case[:4], lens, news, D ** -0.5, window, sinks))


@pytest.mark.parametrize("longest", [150, 2300])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_batches_of_more_sequences_than_lanes(v, dev, longest, D):
    lens = [(37 * i) % 140 for i in range(150)] + [longest, 100]
    news = [min(L, (1, 0, 40, 3)[i % 4]) for i, L in enumerate(lens)]
    _both(v, dev, longest + D, lens, news, 4, 2, D, 16, torch.float16)


@pytest.mark.parametrize("Hq,Hkv", [(300, 1), (129, 1), (514, 2)])
def test_groups_larger_than_a_tile(v, dev, Hq, Hkv):
    for D in (64, 256):
        _both(v, dev, Hq + D, [70, 200], [1, 3], Hq, Hkv, D, 16, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_tables_of_many_places(v, dev, D):
    """A table that could hold so many keys that their blocks are counted in 64 bits; all but the first columns are never used."""
    lens, news = [100, 1, 1030, 0] * 16, [1] * 64
    case = list(R.make(dev, D, lens, news, 8, 4, D, 512, torch.bfloat16))
    wide = torch.full((64, (1 << 28) // 512), -1, dtype=torch.int32, device=dev)
    wide[:, :case[3].shape[1]] = case[3]
    out = _run(v, case[:3] + [wide] + case[4:], lens, news, D)
    _check(out, *R.attention(*case[:4], lens, news, D ** -0.5))


@pytest.mark.parametrize("n,L", [(1, 900), (40, 300), (40, 2600)])
def test_starts_that_do_not_ascend_stay_inside(v, dev, n, L):
    lens, news = [L, 90, L], [n, n, n]
    q, kc, vc, table, seq, cu, _ = R.make(dev, n, lens, news, 8, 2, 128, 16, torch.bfloat16)
    for starts in ([0, 3 * n, 0, 3 * n], [2 * n, n, 0, 0], [-5, n, 2 * n, 10 ** 9], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0]):
        around = torch.full((5 * n, 8, 128), 3.0, dtype=q.dtype, device=dev)
        out = around[n:4 * n]
        v.paged_attention(q, kc, vc, table, seq, torch.tensor(starts, dtype=torch.int32, device=dev), out, 0.1, -1, 0, n, L)
        assert (around[:n] == 3).all() and (around[4 * n:] == 3).all()


@pytest.mark.parametrize("n", [1, 40])
def test_two_streams_at_once(v, dev, n):
    lens, news = [5000, 300], [n, n]
    cases = [R.make(dev, s, lens, news, 8, 2, 128, 16, torch.bfloat16) for s in range(2)]
    alone = [_run(v, c, lens, news, 128) for c in cases]
    outs = [[torch.empty_like(alone[0]) for _ in range(10)] for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for i in range(10):
        for s, c, o in zip(streams, cases, outs):
            with torch.cuda.stream(s):
                _run(v, c, lens, news, 128, out=o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for a, many in zip(alone, outs) for o in many)


def test_pages_outside_the_cache_are_not_seen(v, dev):
    for n in (1, 60):
        lens, news = [200, 130], [n, n]
        case = R.make(dev, n, lens, news, 8, 2, 128, 16, torch.bfloat16)
        table = case[3]
        table[0, 2], table[0, 5], table[1, 0] = -1, case[1].shape[0], 2 ** 31 - 1
        out = _run(v, case, lens, news, 128)
        _check(out, *R.attention(*case[:4], lens, news, 128 ** -0.5))


def test_lengths_behind_the_table_are_not_seen(v, dev):
    for n in (1, 60):
        lens, news = [200, 130], [n, n]
        case = list(R.make(dev, n, lens, news, 8, 2, 64, 16, torch.float16))
        case[3] = case[3][:, :6].contiguous()
        out = _run(v, case, lens, news, 64)
        _check(out, *R.attention(*case[:4], lens, news, 64 ** -0.5))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 50])
def test_strides(v, dev, D, n):
    """Queries as columns of a fused projection; caches as halves of one array and heads outside the places."""
    lens, news = [333, 90], [n, n]
    q, kc, vc, table, seq, cu, _ = R.make(dev, D + n, lens, news, 8, 2, D, 16, torch.bfloat16)
    plain = _run(v, (q, kc, vc, table, seq, cu, None), lens, news, D)
    wide = torch.randn(q.shape[0], 14 * D, device=dev).to(q.dtype)
    wide[:, D:9 * D] = q.flatten(1)
    strided = wide[:, D:9 * D].unflatten(1, (8, D))
    both = torch.stack([kc, vc], 1)
    heads = torch.stack([kc, vc]).permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
    inside = torch.cat([kc, vc], 3)
    for k2, v2 in (both.unbind(1), heads.unbind(0), (inside[..., :D], inside[..., D:])):
        assert torch.equal(_run(v, (strided, k2, v2, table, seq, cu, None), lens, news, D), plain)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(_run(v, (turned, kc, vc, table, seq, cu, None), lens, news, D), plain)


def test_offsets_past_32_bits(v, dev):
    """A cache of more than 2^32 elements, keys on its first and last pages."""
    pages, page, D = (1 << 32) // (64 * 2 * 128) + 40, 64, 128
    kc = torch.empty(pages, page, 2, D, dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    g = torch.Generator(device=dev).manual_seed(3)
    table = torch.tensor([[pages - 1, 0, pages - 2, pages // 2]], dtype=torch.int32, device=dev)
    for c in (kc, vc):
        c[table[0].long()] = torch.randn(4, page, 2, D, generator=g, device=dev).bfloat16()
    for n in (1, 200):
        q = torch.randn(n, 8, D, generator=g, device=dev).bfloat16()
        seq, cu = torch.tensor([250], dtype=torch.int32, device=dev), torch.tensor([0, n], dtype=torch.int32, device=dev)
        out = torch.empty_like(q)
        v.paged_attention(q, kc, vc, table, seq, cu, out, 0.1, -1, 0, n, 250)
        small = kc[table[0].long()], vc[table[0].long()]
        order = torch.arange(4, dtype=torch.int32, device=dev)[None]
        _check(out, *R.attention(q, *small, order, [250], [n], 0.1))


@pytest.mark.parametrize("hint_q,hint_k", [(0, 0), (1, 1), (10 ** 9, 10 ** 9), (2 ** 40, 2 ** 40), (33, 100), (90, 5000)])
def test_lengths_said_wrongly_change_no_result(v, dev, hint_q, hint_k):
    lens, news = [800, 90, 1500, 40], [70, 90, 1, 0]
    for kind in ("causal", "tree"):
        words = 0 if kind == "causal" else 2
        if kind == "tree" and hint_q > 128:
            continue
        case = R.make(dev, 5, lens, news, 8, 2, 128, 16, torch.bfloat16, words)
        out = _run(v, case, lens, news, 128, hint_q=hint_q, hint_k=hint_k)
        _check(out, *R.attention(*case[:4], lens, news, 128 ** -0.5, masks=case[6]))


def test_scores_of_any_size(v, dev):
    """Scores from far below to far above what an exponential holds: the largest one takes all."""
    for n in (1, 70):
        for spread in (1e-3, 30.0, 300.0):
            lens, news = [400, 100], [n, n]
            case = R.make(dev, n, lens, news, 4, 1, 64, 16, torch.bfloat16, spread=spread)
            _check(_run(v, case, lens, news, 64), *R.attention(*case[:4], lens, news, 64 ** -0.5))


@pytest.mark.parametrize("kind", ["single", "prompt", "tree", "mixed"])
def test_graphs_and_streams(v, dev, kind):
    """Captured on a side stream, replayed with other contents between eager calls; another graph beside it."""
    lens, news = dict(single=([900, 31], [1, 1]), prompt=([600, 80], [600, 80]), tree=([700, 64], [30, 30]), mixed=([700, 64, 40], [100, 1, 1]))[kind]
    words = 1 if kind == "tree" else 0
    cases = [R.make(dev, s, lens, news, 8, 2, 128, 16, torch.bfloat16, words) for s in range(3)]
    eager = [_run(v, c, lens, news, 128) for c in cases]
    again = [_run(v, c, lens, news, 128) for c in cases]
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    static = [t.clone() if t is not None else None for t in cases[0]]
    outs = [torch.empty_like(eager[0]) for _ in range(2)]
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(_run(v, static, lens, news, 128, out=outs[0]), eager[0])
    side.synchronize()
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _run(v, static, lens, news, 128, out=out)
        graphs.append(g)
    for turn in (1, 2, 0, 2):
        for t, c in zip(static, cases[turn]):
            if t is not None:
                t.copy_(c)
        for out in outs:
            out.fill_(float("nan"))
        for g in graphs:
            g.replay()
        assert torch.equal(_run(v, cases[turn - 1], lens, news, 128), eager[turn - 1])
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager[turn]) for out in outs)


def test_refusals(v, dev):
    q, kc, vc, table, seq, cu, masks = R.make(dev, 1, [40, 9], [2, 1], 8, 2, 64, 16, torch.float16, 1)

    def call(q=q, kc=kc, vc=vc, table=table, seq=seq, cu=cu, out=None, scale=0.1, window=-1, sinks=0, mq=2, mk=40, masks=None):
        out = torch.empty(q.shape, dtype=q.dtype, device=dev) if out is None else out
        if masks is not None:
            return v.tree_attention(q, kc, vc, table, seq, cu, masks, out, scale, mq, mk)
        return v.paged_attention(q, kc, vc, table, seq, cu, out, scale, window, sinks, mq, mk)
    call()
    call(masks=masks)
    deep = torch.empty(kc.numel() + 64, dtype=torch.float16, device=dev)
    shifted = deep[8:8 + kc.numel()].view_as(kc)
    for kw, why in ((dict(q=q.float()), "fp16 or bf16"), (dict(q=q[:, 0]), "fp16 or bf16"), (dict(q=q[..., :32].contiguous()), "heads of 64"),
                    (dict(q=q.bfloat16()), "cache must have the input's type"), (dict(vc=vc.bfloat16()), "input's type"),
                    (dict(kc=kc[..., :32]), "key_cache must be"), (dict(kc=kc[0]), "key_cache must be"), (dict(kc=kc[:0], vc=vc[:0]), "must have pages"),
                    (dict(vc=vc[:-1]), "sizes and strides"), (dict(vc=torch.stack([vc, vc], 1).unbind(1)[0]), "sizes and strides"),
                    (dict(kc=kc.transpose(1, 3).contiguous().transpose(1, 3)), "side by side"), (dict(vc=kc), "overlap key_cache"),
                    (dict(kc=deep[:kc.numel()].view_as(kc), vc=shifted), "overlap key_cache"),
                    (dict(q=q[:, :7]), "multiple of the cache's"), (dict(table=table.long()), "block_table must be int32"),
                    (dict(table=table[0]), "block_table must be int32"), (dict(table=table.t()), "contiguous"), (dict(seq=seq.long()), "seq_lens must be"),
                    (dict(seq=seq[:1]), "seq_lens must be"), (dict(cu=cu[:2]), "cu_seqlens_q must be"), (dict(cu=cu.long()), "cu_seqlens_q must be"),
                    (dict(out=torch.empty(3, 8, 64, dtype=torch.bfloat16, device=dev)), "output must have"),
                    (dict(out=torch.empty(2, 8, 64, dtype=torch.float16, device=dev)), "output must have"),
                    (dict(out=torch.empty(3, 64, 8, dtype=torch.float16, device=dev).transpose(1, 2)), "contiguous"), (dict(out=q), "overlap"),
                    (dict(scale=0.0), "scale must be"), (dict(scale=-1.0), "scale must be"), (dict(scale=float("nan")), "scale must be"),
                    (dict(scale=float("inf")), "scale must be"), (dict(window=0), "window must be"), (dict(window=-2), "window must be"),
                    (dict(sinks=-1), "sinks must"), (dict(mq=-1), "must not be negative"), (dict(mk=-1), "must not be negative"),
                    (dict(seq=seq.cpu()), "same ROCm device"), (dict(kc=kc.cpu()), "same ROCm device"),
                    (dict(q=deep[4:4 + q.numel()].view_as(q)), "16-byte boundary"),
                    (dict(q=deep[:3 * 8 * 68].view(3, 8, 68)[..., :64]), "multiples of 8"),
                    (dict(masks=masks.int()), "tree_mask must be"), (dict(masks=masks[:2]), "tree_mask must be"), (dict(masks=masks[:, :0]), "tree_mask must be"),
                    (dict(masks=masks, mq=65), "words for up to")):
        with pytest.raises(RuntimeError, match=why):
            call(**kw)


@pytest.mark.parametrize("dt", DTS)
def test_long_tails_keep_their_weight(v, dev, dt):
    """One key far above 100000 others whose weights are subnormal in 16 bits: together they count for more than the output's rounding."""
    L, D = 100000, 64
    for n in (1, 40):
        case = R.make(dev, 1, [L], [n], 1, 1, D, 64, dt)
        q, kc, vc, table = case[:4]
        q.zero_()
        q[..., 0] = 8.0
        flat = kc[table[0].long()]
        flat.view(-1, D)[:L] = 0
        flat.view(-1, D)[5, 0] = 11.0                   # a score of 11: the others have 2^-15.9 of its weight
        kc[table[0].long()] = flat
        vals = vc[table[0].long()]
        vals.view(-1, D)[:L] = 1.0
        vals.view(-1, D)[5] = -1.0
        vc[table[0].long()] = vals
        _check(_run(v, case, [L], [n], D), *R.attention(*case[:4], [L], [n], D ** -0.5))
