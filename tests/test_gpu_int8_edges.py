"""Edges of the 8-bit integer operators: what an expert's result keeps on its way to the weighted sum, codes at ties, a norm's
row over batch sizes, row counts near the end of a grid.  References in 64 bits, as in test_gpu_int8.py."""
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


@pytest.mark.parametrize("T", [1, 2, 60, 330, 900])
def test_an_expert_scale_of_nan_stays_in_its_column(v, dev, T):  # noqa: F811
    """NaN scales, of every bit set too, reach their own columns of their expert's tokens and nothing else."""
    c = _moe(T, 3, 1, 272, 128, torch.bfloat16, T, False)
    c["logits"][0, 1] = 10                                # the first token takes it in any case
    want = _moe_run(dev, c, 1)
    c["s2"][1, 40] = float("nan")
    c["s2"].view(torch.int32)[1, 41] = -1
    c["s2"].view(torch.int32)[1, 43] = 0x7FFFFFFF
    got = _moe_run(dev, c, 1)
    bad = torch.zeros(T, 272, dtype=torch.bool)
    hit = (c["logits"].double().argmax(1) == 1).nonzero()
    bad[hit, torch.tensor([40, 41, 43])] = True
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("T", [1, 5, 120])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_expert_rows_longer_than_registers_hold(v, dev, T, dt):  # noqa: F811
    """H = 8208: rows of x are read again for their codes."""
    _spread_check(dev, _moe(T, 4, 1, 8208, 48, dt, T + 3, T % 2 == 1))


# ------------------------------------------------------------------------------------------------ codes at ties
def _ties(n, K, dt, seed):
    """Rows whose entries are halves of a step away from each other, or next to that (an entry of half the largest is 63.5 steps)."""
    g = torch.Generator().manual_seed(seed)
    m = (torch.rand(n, 1, generator=g) + 0.5).to(dt)
    x = (m.double() * torch.randint(-253, 254, (n, K), generator=g) / 254).to(dt)
    nudge = torch.where(x == 0, 0, torch.randint(-1, 2, x.shape, generator=g)).to(torch.int16)
    x = (x.view(torch.int16) + nudge).view(dt)
    x = torch.where(x.abs() > m, m, x)
    x[:, :1] = m
    return x


@pytest.mark.parametrize("K,rows", [(256, 16), (256, 3), (1040, 5), (2048, 8), (4096, 1)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_codes_of_few_rows_are_determined(v, dev, K, rows, dt):  # noqa: F811
    """The launch that quantises its rows itself, K in one part per wavefront and in several."""
    n = 40 * rows
    x = _ties(n, K, dt, K + rows)
    q, s, _ = R.quantise(x.double())
    eye, one = torch.eye(K, dtype=torch.int8, device=dev), torch.ones(K, device=dev)
    out, xd = torch.empty(n, K, dtype=dt, device=dev), x.to(dev)
    for i in range(0, n, rows):
        v.gemm_int8(xd[i:i + rows], None, eye, one, None, out[i:i + rows])
    # a code is at most 127: a 16-bit output is off by less than half a step, so the row's scale is taken out in 64 bits
    assert torch.equal(torch.round(out.cpu().double() / s[:, None]), q)


@pytest.mark.parametrize("T", [1, 3, 700])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_expert_codes_at_ties(v, dev, T, dt):  # noqa: F811
    """16 values of x: a code beside the right one changes a gate or an up by more than the outputs' tolerance."""
    for seed in range(20 if T < 16 else 2):
        c = _moe(T, 3, 1, 16, 64, dt, seed, False)
        c["x"] = _ties(T, 16, dt, seed)
        _spread_check(dev, c)


# ------------------------------------------------------------------------------------------------ rows over batch sizes
@pytest.mark.parametrize("K", [272, 512, 1024, 1040, 2048, 2064, 4096, 4112, 8192, 16384, 16400, 40000])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_a_row_behind_norm_or_silu_depends_on_itself_alone(v, dev, K, dt):  # noqa: F811
    """A row's bits are the same whichever launch quantises it: alone, among few or many, residual in place or not."""
    M, N = 400, 1000
    g = torch.Generator().manual_seed(K)
    x, res = (torch.randn(M, K, generator=g).to(dt).to(dev) for _ in range(2))
    nw = (1 + 0.1 * torch.randn(K, generator=g)).to(dt).to(dev)
    w, ws, b = R.codes_like_weights(g, N, K).to(dev), R.scales(g, N).to(dev), torch.randn(N, generator=g).to(dt).to(dev)
    gate_up = torch.cat([x, res], 1)

    def norm(lo, hi, in_place=False):
        out, r = x.new_empty(hi - lo, N), res[lo:hi].clone()
        r_out = r if in_place else torch.empty_like(r)
        v.resadd_norm_gemm_int8(x[lo:hi], r, r_out, nw, w, ws, b, out, 1e-6)
        return out

    def silu(lo, hi):
        out = x.new_empty(hi - lo, N)
        v.silu_mul_gemm_int8(gate_up[lo:hi], w, ws, b, out)
        return out
    whole, whole_silu = norm(0, M), silu(0, M)
    assert torch.equal(norm(0, M, True), whole)
    cuts = list(range(48)) + [50, 54, 62, 78, 110, 210, M]
    for lo, hi in zip(cuts, cuts[1:]):
        assert torch.equal(norm(lo, hi), whole[lo:hi]) and torch.equal(norm(lo, hi, True), whole[lo:hi])
        assert torch.equal(silu(lo, hi), whole_silu[lo:hi])


# ------------------------------------------------------------------------------------------------ many rows
@pytest.mark.parametrize("what,M,K", [("act", (1 << 23) + 5, 4112), ("act", (1 << 22) + 5, 8208), ("norm", (1 << 23) + 5, 4112), ("silu", (1 << 23) + 5, 2064)])
def test_rows_up_to_the_stated_limit(v, dev, what, M, K):  # noqa: F811
    """2^32 threads at 512 or 1024 per row are no launch: such a call takes fewer threads per row.  Few rows are filled and looked at."""
    dt, N = torch.bfloat16, 3
    row_bytes = {"act": 3 * K, "norm": 5 * K, "silu": 5 * K}[what] + 64
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < M * row_bytes * 1.05:
        pytest.skip("not enough free memory")
    g = torch.Generator().manual_seed(K)
    few = torch.tensor([0, 1, 2, (1 << 22) - 1, 1 << 22, M - 2, M - 1], device=dev)
    cols = 2 * K if what == "silu" else K
    rows = torch.randn(len(few), cols, generator=g).to(dt)
    w, ws = R.codes_like_weights(g, N, K), R.scales(g, N)
    nw = torch.ones(K, dtype=dt, device=dev)
    try:
        x = torch.zeros(M, cols, dtype=dt, device=dev)
        x[few] = rows.to(dev)
        out = torch.full((M, N), float("nan"), dtype=dt, device=dev)
        if what == "act":
            v.gemm_int8(x, None, w.to(dev), ws.to(dev), None, out)
            q, rel = R.quantise(rows.double()), 2.0 ** -21
        elif what == "norm":
            x_out = torch.empty_like(x)
            v.resadd_norm_gemm_int8(x, x, x_out, nw, w.to(dev), ws.to(dev), None, out, 1e-6)
            assert torch.equal(x_out[few], x[few] * 2)
            del x_out
            q, rel = R.quantise(R.norm(rows, rows, nw.cpu(), 1e-6)[1], LOOSE), 2.0 ** -15
        else:
            v.silu_mul_gemm_int8(x, w.to(dev), ws.to(dev), None, out)
            q, rel = R.quantise(R.silu_mul(rows.double()), LOOSE), SILU
        ref, slack = R.product(*q, w, ws)
        ok, worst = R.within(out[few].cpu(), ref, slack, dt, rel)
        assert ok, f"{worst:.2f} of the tolerance"
        rest = torch.ones(M, dtype=torch.bool, device=dev)
        rest[few] = False
        assert bool((out[rest] == 0).all())
    finally:
        x = x_out = out = rest = None
        torch.cuda.empty_cache()
