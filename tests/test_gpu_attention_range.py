"""Attention over a paged cache where scores or values are as large, or weights as small, as their types hold."""
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu
DTS = [torch.float16, torch.bfloat16]
# single tokens; tiles; few tokens over a long context, in shares of its keys; both kernels in one call
CALLS = [([700, 90], [1, 1]), ([300, 100], [70, 100]), ([2600, 1500], [40, 61]), ([2600, 40, 9000], [40, 1, 1])]


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


def _run(v, case, lens, news, scale):
    q, kc, vc, table, seq, cu, _ = case
    out = torch.full_like(q, float("nan"))
    return v.paged_attention(q, kc, vc, table, seq, cu, out, scale, -1, 0, max(news), max(lens))


def _check(got, ref, tol):
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert not got.isnan().any() and worst <= 1.0, f"{worst:.2f} of the tolerance"


def _keys(case, b, L):
    """Where keys 0 .. L - 1 of sequence b lie: page, place."""
    j = torch.arange(L, device=case[0].device)
    page = case[1].shape[1]
    return case[3][b].long()[j // page], j % page


def _exact_scores(case, lens, news, scale):
    """What the call returns where every score is exact in fp32, in any order of its sums.  Off is then, of a score, only what its distance to the
    largest one loses as it is scaled (three half steps of itself: the factor, the product, its use), and in a weight the exponential: 2^-18 as in
    attention_reference."""
    q, kc, vc, table = case[:4]
    u, G, at = R.half_step(q.dtype), q.shape[1] // kc.shape[2], 0
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, (L, n) in enumerate(zip(lens, news)):
        k, val = (c[_keys(case, b, L)].double() for c in (kc, vc))
        see = torch.arange(L, device=q.device) <= torch.arange(L - n, L, device=q.device)[:, None]
        for h in range(q.shape[1]):
            s = (q[at:at + n, h].double() @ k[:, h // G].t()).masked_fill(~see, float("-inf"))
            far = (s.amax(1, keepdim=True) - s) * scale
            w = torch.exp(-far)
            w = w / w.sum(1, keepdim=True)
            off = torch.where(w > 0, w * (2 * u + 2 * (2.0 ** -18 + 3 * 2.0 ** -24 * far.clamp_max(1e4))), 0.0)
            o, size = w @ val[:, h // G], val[:, h // G].abs()
            out[at:at + n, h] = o
            small = 2 * 2.0 ** -32 * (see.double() @ size) if q.dtype == torch.float16 else 0.0
            mean = (w * (2 * u + 2.0 ** -17)).sum(1, keepdim=True) * (w @ size)                  # of the sum that all are divided by
            tol[at:at + n, h] = u * o.abs() + off @ size + mean + small + (2.0 ** -24 if q.dtype == torch.float16 else 1e-38)
        at += n
    return out, tol


@pytest.mark.parametrize("lens,news", CALLS)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 12), (256, 16)])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("kind", ["high", "low", "mixed"])
def test_scores_of_2_to_the_30(v, dev, lens, news, D, page, dt, kind):
    """Scores of +-2^30 + 128 j, where a unit in fp32's last place is 128, at a scale of 1 / 64: exact, steps of 2 apart, where a unit in the last place of
    the scaled ones is 2 too.  Low: all of them far below zero.  Mixed: a third of the keys far below, a third around zero and a third far above, for heads that take them so, the other way
    round, and without the large part."""
    case = R.make(dev, D + len(lens), lens, news, 6, 2, D, page, dt)
    q, kc = case[:2]
    g = torch.Generator().manual_seed(D)
    q.zero_()
    q[..., 0], q[..., 1] = 32768.0, 128.0
    if kind != "high":
        q[:, 0::3, 0] = -32768.0
    if kind == "mixed":
        q[:, 1::3, 0] = 0.0
    for b, L in enumerate(lens):
        if not L:
            continue
        k = torch.zeros(L, 2, D)
        k[..., 1] = torch.randint(0, 16, (L, 2), generator=g)
        k[..., 0] = 32768.0
        if kind == "mixed":
            k[:L // 3, :, 0], k[L // 3:2 * L // 3, :, 0] = -32768.0, 0.0
        kc[_keys(case, b, L)] = k.to(dt).to(dev)
    _check(_run(v, case, lens, news, 1 / 64), *_exact_scores(case, lens, news, 1 / 64))


# one or few keys per row; a prompt whose first tokens see few; long contexts
LARGE = [([1, 2, 3, 70], [1, 1, 1, 1], 126), ([70, 1, 33], [70, 1, 33], 119), ([300, 100], [70, 100], 117), ([2600, 1500], [40, 61], 114),
         ([2600, 40, 9000], [40, 1, 1], 112)]


@pytest.mark.parametrize("lens,news,size", LARGE)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 12), (256, 16)])
def test_values_of_any_size(v, dev, lens, news, size, D, page):
    """bf16 values of 2^size (what keeps a sum of them under weights of 1 finite), and of 2^-size: exponents of fp32."""
    for exponent in (size, -size):
        case = R.make(dev, D + size, lens, news, 4, 2, D, page, torch.bfloat16)
        case[2].copy_((case[2].double().clamp(-3.9, 3.9) * 2.0 ** exponent).bfloat16())
        _check(_run(v, case, lens, news, D ** -0.5), *R.attention(*case[:4], lens, news, D ** -0.5))


@pytest.mark.parametrize("n", [1, 70])
def test_a_rising_maximum_under_large_values(v, dev, n):
    """Scores that rise by less than what moves the maximum, one key after the other: weights far above the first one's."""
    lens, news, D = [200], [n], 64
    case = R.make(dev, n, lens, news, 1, 1, D, 16, torch.bfloat16)
    q, kc, vc = case[:3]
    q.zero_()
    q[..., 0] = 8.0
    k = torch.zeros(200, 1, D)
    k[:, 0, 0] = torch.where(torch.arange(200) < 120, 0.0, 5.0)       # 2^7.2 of the first ones' weight
    at = _keys(case, 0, 200)
    kc[at] = k.bfloat16().to(dev)
    vc[at] = torch.full_like(vc[at], 2.0 ** 120)
    _check(_run(v, case, lens, news, D ** -0.5), *R.attention(*case[:4], lens, news, D ** -0.5))


@pytest.mark.parametrize("score", [14.75, 15.25, 16.75])
@pytest.mark.parametrize("n", [1, 40])
def test_tails_of_subnormal_weights(v, dev, n, score):
    """One key far above 100000 others, which have 2^-21.3, 2^-22 and 2^-24.2 of its weight: in fp16 subnormal (2^-14.3, 2^-15, 2^-17.2) as they are
    raised by 2^7.  Together they count for 2^-4.7, 2^-5.4 and 2^-7.6, twice that in the result: more than the tolerance, where a product or the sum of the
    weights lost them."""
    L, D = 100000, 64
    q, kc, vc, table, seq, cu, _ = case = R.make(dev, 1, [L], [n], 1, 1, D, 64, torch.float16)
    q.zero_()
    q[..., 0] = 8.0
    at = _keys(case, 0, L)
    k, val = torch.zeros(L, 1, D, dtype=torch.float16, device=dev), torch.ones(L, 1, D, dtype=torch.float16, device=dev)
    k[5, 0, 0], val[5] = score, -1.0
    kc[at], vc[at] = k, val
    _check(_run(v, case, [L], [n], D ** -0.5), *R.attention(*case[:4], [L], [n], D ** -0.5))
