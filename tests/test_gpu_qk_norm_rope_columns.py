"""qk_norm_rope with queries and keys as columns of one array of their own, and beside the projection's rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
T, HQ, HKV, D = 21, 6, 2, 128


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


def _inputs(dev):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, (HQ + 2 * HKV) * D, generator=g).bfloat16().to(dev)
    angle = torch.rand(40, D // 2, generator=g) * 6
    return x, torch.cat([angle.cos(), angle.sin()], 1).to(dev), torch.randint(0, 40, (T,), generator=g).to(dev)


def _columns(t, first, heads):
    return t[:, first * D:(first + heads) * D].unflatten(1, (heads, D))


def test_outputs_side_by_side(v, dev):
    x, cs, pos = _inputs(dev)
    q, k = (torch.empty(T, h, D, dtype=x.dtype, device=dev) for h in (HQ, HKV))
    v.qk_norm_rope(x, None, None, cs, pos, q, k, None, None, None, 1e-6)
    # [queries | keys], [keys | queries] with columns around them, [projection | queries | keys]
    for wide, first_q, first_k in ((torch.full((T, 8 * D), 3.0), 0, HQ), (torch.full((T, 11 * D), 3.0), 1 + HKV, 1), (torch.full((T, 19 * D), 3.0), 10, 17)):
        wide = wide.bfloat16().to(dev)
        rows = x
        if wide.shape[1] == 19 * D:
            rows = wide[:, :10 * D]
            rows.copy_(x)
        before = wide.clone()
        v.qk_norm_rope(rows, None, None, cs, pos, _columns(wide, first_q, HQ), _columns(wide, first_k, HKV), None, None, None, 1e-6)
        assert torch.equal(_columns(wide, first_q, HQ), q) and torch.equal(_columns(wide, first_k, HKV), k)
        for first, heads in ((first_q, HQ), (first_k, HKV)):
            _columns(before, first, heads).copy_(_columns(wide, first, heads))
        assert torch.equal(wide, before)                # nothing else


def test_columns_that_meet_are_refused(v, dev):
    x, cs, pos = _inputs(dev)
    wide = torch.empty(T, 24 * D, dtype=x.dtype, device=dev)
    wide[:, :10 * D] = x
    q, k = (torch.empty(T, h, D, dtype=x.dtype, device=dev) for h in (HQ, HKV))

    def call(x=x, q=q, k=k):
        return v.qk_norm_rope(x, None, None, cs, pos, q, k, None, None, None, 1e-6)
    last = torch.empty(T + 1, 8 * D, dtype=x.dtype, device=dev)
    for kw, why in ((dict(q=_columns(wide, 0, HQ), k=_columns(wide, HQ - 1, HKV)), "overlap q_out"),
                    (dict(q=_columns(wide, 1, HQ), k=_columns(wide, 0, HKV)), "overlap q_out"),
                    (dict(q=wide[:, 8:HQ * D + 8].unflatten(1, (HQ, D)), k=_columns(wide, HQ, HKV)), "overlap q_out"),
                    (dict(x=wide[:, :10 * D], q=_columns(wide, 9, HQ)), "overlap qkv"), (dict(x=wide[:, :10 * D], k=_columns(wide, 0, HKV)), "overlap qkv"),
                    # rows of the same stride that run into the next one's
                    (dict(q=last[:T, 4 * D:].as_strided((T, HQ, D), (8 * D, D, 1)), k=_columns(last[1:], 1, HKV)), "overlap q_out"),
                    # other strides: told by the spans alone
                    (dict(q=wide[:10].as_strided((T, HQ, D), (8 * D, D, 1)), k=_columns(wide, HQ, HKV)), "overlap q_out")):
        with pytest.raises(RuntimeError, match=why):
            call(**kw)


@pytest.mark.parametrize("head", [64, 128, 256])
def test_norm_of_elements_whose_squares_pass_fp32(v, dev, head):
    """bf16 rows from 1e15 to the type's largest number, beside rows of one: normed like any other; an infinity stays NaN."""
    g = torch.Generator().manual_seed(head)
    x = torch.randn(6, 4 * head, generator=g).double()
    x *= torch.tensor([1.0, 1e15, 1e19, 1e30, 8e37, 1.0])[:, None].double()
    x = x.clamp(-3.3e38, 3.3e38).bfloat16().to(dev)
    x[5, head + 3] = float("inf")
    q, k = (torch.empty(6, h, head, dtype=x.dtype, device=dev) for h in (2, 1))
    w = [(1 + 0.3 * torch.randn(head, generator=g)).bfloat16().to(dev) for _ in range(2)]
    v.qk_norm_rope(x, w[0], w[1], torch.empty(4, 0, device=dev), torch.zeros(6, dtype=torch.int64, device=dev), q, k, None, None, None, 1e-6)
    heads = x.double().view(6, 4, head)
    assert q[5, 1].isnan()[3] and not q[5, 0].isnan().any()
    for got, part, weight in ((q[:5], heads[:5, :2], w[0]), (k, heads[:, 2:3], w[1])):
        ref = part / torch.sqrt(part.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.double()
        # one rounding to bf16, and 28 steps of fp32 as for rows of ordinary size
        assert ((got.double() - ref).abs() <= (2.0 ** -8 * (1 + 2.0 ** -10) + 28 * 2.0 ** -24) * ref.abs() + 1e-40).all()
