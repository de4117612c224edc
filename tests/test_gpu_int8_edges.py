"""Edges of the 8-bit integer operators: what an expert's result keeps on its way to the weighted sum.  References in 64 bits, as in test_gpu_int8.py."""
import pytest
import torch

import int8_reference as R
from test_gpu_int8 import LOOSE, SILU, _moe, _moe_run, v  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ an expert's result
# tokens and experts, one route: the two launches for a few tokens, then 32, 64, 128, 192, 256, 320 and again 192 rows per tile
ROUTES = [(2, 3), (60, 3), (100, 6), (150, 3), (330, 3), (500, 3), (700, 3), (900, 3), (1100, 3)]


def _spread_check(dev, c):
    """One route per token (a weight of 1, whatever the arithmetic) against 64 bits.  With many tokens an expert's result passes to the sum as a
    float of 16 significant bits: off by 2^-16 of itself (half of its last place, 2^-15, at 1), of nothing else."""
    T, H = c["x"].shape
    out, slack, parts = (torch.zeros(T, H, dtype=torch.float64) for _ in range(3))
    q, s, near = R.quantise(c["x"].double())
    top = c["logits"].double().argmax(1)

    def expert(rows, w13, s13, w2, s2):
        gu, _ = R.product(q[rows], s[rows], near[rows], w13, s13)
        y, sl = R.product(*R.quantise(R.silu_mul(gu), LOOSE), w2, s2)
        return y, sl + 2.0 ** -16 * (y.abs() + sl)
    for e in range(c["w13"].shape[0]):
        rows = (top == e).nonzero(as_tuple=True)[0]
        if rows.numel():
            out[rows], slack[rows] = expert(rows, c["w13"][e], c["s13"][e], c["w2"][e], c["s2"][e])
            parts[rows] = out[rows].abs()
    if c["gw"] is not None:
        gate = torch.sigmoid(c["x"].double() @ c["gw"].double().t())
        y, sl = expert(torch.arange(T), c["sw13"], c["ss13"], c["sw2"], c["ss2"])
        # the gate's dot product in 32 bits: each of a lane's and a wavefront's H / 64 + 8 steps is off by 2^-24 of the terms' sizes at most
        dot = (c["x"].double().abs() @ c["gw"].double().abs().t()) * 2.0 ** -24 * (H / 64 + 8)
        out, slack, parts = out + gate * y, slack + gate * sl + dot * gate * y.abs(), parts + gate * y.abs()
    ok, worst = R.within(_moe_run(dev, c, 1), out, slack, c["x"].dtype, SILU, parts)
    assert ok, f"{worst:.2f} of the tolerance"


@pytest.mark.parametrize("T,E", ROUTES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_expert_columns_of_very_different_scales(v, dev, T, E, dt):  # noqa: F811
    """One output channel in 32 has a scale 1000 times its neighbours': they keep their bits."""
    c = _moe(T, E, 1, 272, 128, dt, T, T % 4 == 0)
    c["s2"][:, 5::32] *= 1000
    if c["gw"] is not None:
        c["ss2"][7::32] *= 1000
    _spread_check(dev, c)


@pytest.mark.parametrize("T,E", ROUTES)
def test_expert_columns_of_very_different_weights(v, dev, T, E):  # noqa: F811
    """Codes of one scale for all channels: a channel of large codes beside channels of -1, 0 and 1."""
    c = _moe(T, E, 1, 272, 128, torch.float16, T + 1, T % 4 == 0)
    for n in ("w2", "sw2"):
        if c[n] is not None:
            small = c[n].clamp(-1, 1)
            small[..., 5::32, :] = c[n][..., 5::32, :] * 3 // 4 + 31
            c[n] = small
    _spread_check(dev, c)


@pytest.mark.parametrize("T", [60, 330, 900])
def test_an_expert_scale_of_nan_stays_in_its_column(v, dev, T):  # noqa: F811
    """NaN scales, of every bit set too, reach their own columns of their expert's tokens and nothing else."""
    c = _moe(T, 3, 1, 272, 128, torch.bfloat16, T, False)
    want = _moe_run(dev, c, 1)
    c["s2"][1, 40] = float("nan")
    c["s2"].view(torch.int32)[1, 41] = -1
    c["s2"].view(torch.int32)[1, 43] = 0x7FFFFFFF
    got = _moe_run(dev, c, 1)
    bad = torch.zeros(T, 272, dtype=torch.bool)
    hit = (c["logits"].double().argmax(1) == 1).nonzero()
    assert len(hit)
    bad[hit, torch.tensor([40, 41, 43])] = True
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], want[~bad])
