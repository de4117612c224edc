"""The 8-bit integer (W8A8) linears against 64-bit math: product, residual + norm and SiLU in front of it, the expert layer.

Tolerances: one rounding to the output's type (half a step), and in front of it 32-bit steps on the finished integer sum: its conversion,
two factors and the bias, each 2^-24, together below 2^-21 of product and bias.  A norm's rows carry the 32-bit sum of squares as well:
chains of up to 600 additions, half of whose relative error comes through the square root, below 2^-15."""
import pytest
import torch

import int8_reference as R

pytestmark = pytest.mark.gpu

PLAIN, NORM, SILU = 2.0 ** -21, 2.0 ** -15, 2.0 ** -19
# v / m of a norm's or a SiLU's row: sums, factors, an exponential and a quotient of 32 bits each in v and in m, below 2^-19 of a code
LOOSE = 2.0 ** -19


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


def _case(M, K, N, dt, seed, bias):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * (1 + 7 * (torch.rand(K, generator=g) < 0.02))).to(dt)
    w, ws = R.codes_like_weights(g, N, K), R.scales(g, N)
    b = torch.randn(N, generator=g).to(dt) if bias else None
    return g, x, w, ws, b


def _check(got, q, s, near, w, ws, b, dt, rel):
    ref, slack = R.product(q, s, near, w, ws)
    parts = ref.abs()
    if b is not None:
        ref, parts = ref + b.double(), parts + b.double().abs()
    ok, worst = R.within(got.cpu(), ref, slack, dt, rel, parts)
    assert ok, f"{worst:.2f} of the tolerance"


def _to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


# every place where the choice of kernel, tile, staging or slices changes, odd sizes, rows that end inside a piece of 128, one column
SIZES = [(1, 16, 1), (1, 512, 40), (1, 4096, 257), (2, 2048, 1000), (3, 1040, 130), (4, 4096, 512), (5, 528, 77), (7, 8192, 96), (8, 4096, 1024),
         (9, 144, 300), (16, 2048, 129), (17, 1024, 515), (24, 16384, 64), (31, 5120, 136), (32, 4096, 2048), (33, 2064, 200), (48, 512, 1003), (64, 5120, 640),
         (65, 4096, 96), (100, 11008, 64), (127, 48, 257), (128, 1024, 4096), (129, 1040, 129), (200, 2048, 1001), (255, 128, 640), (256, 4096, 256), (257, 640, 2049),
         (520, 1168, 520), (1, 14336, 160), (2, 20480, 72), (6, 32768, 40), (40, 40000, 24), (1, 131056, 9), (70, 131056, 5), (1030, 256, 1100), (2049, 64, 300)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_product(v, dev, M, K, N, dt):
    g, x, w, ws, b = _case(M, K, N, dt, M + K + N, bias=N % 2 == 1)
    xd, wd, wsd, bd = _to(dev, x, w, ws, b)
    out = torch.full((M, N), float("nan"), dtype=dt, device=dev)
    assert v.gemm_int8(xd, None, wd, wsd, bd, out) is out
    q, s, near = R.quantise(x.double())
    _check(out, q, s, near, w, ws, b, dt, PLAIN)
    codes, cs = R.codes_like_weights(g, M, K), 0.01 + 0.05 * torch.rand(M, generator=g)
    codes[0, 0] = -128                                   # a code that quantising never gives
    out.fill_(float("nan"))
    v.gemm_int8(codes.to(dev), cs.to(dev), wd, wsd, bd, out)
    _check(out, codes.double(), cs.double(), torch.zeros_like(codes, dtype=torch.bool), w, ws, b, dt, PLAIN)


# large and small tiles by what a round of the CUs costs with them, rows of outputs that start on 16 bytes and anywhere
TILES = [(1500, 656, 8200), (1030, 656, 12289), (517, 656, 14336), (517, 672, 12289), (400, 656, 14336), (400, 672, 12289), (400, 656, 8200),
         (260, 656, 12289), (201, 656, 8200), (129, 656, 12289), (77, 4112, 8200), (77, 4112, 9001), (30, 2064, 8200), (30, 2064, 9001),
         (49, 2064, 4008), (49, 2064, 2049), (30, 272, 4008), (30, 656, 6008), (49, 656, 2049), (77, 656, 8200), (77, 656, 9001), (17, 14352, 6144),
         (31, 14352, 6007)]


@pytest.mark.parametrize("M,K,N", TILES)
def test_product_of_tiles(v, dev, M, K, N):
    test_product(v, dev, M, K, N, torch.bfloat16 if K % 32 else torch.float16)


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_silu_and_norm_in_front(v, dev, M, K, N, dt):
    g, x, w, ws, b = _case(M, K, N, dt, M * 3 + K + N, bias=N % 2 == 0)
    up = torch.randn(M, K, generator=g).to(dt)
    wd, wsd, bd = _to(dev, w, ws, b)
    out = torch.full((M, N), float("nan"), dtype=dt, device=dev)
    gate_up = torch.cat([x, up], 1)
    assert v.silu_mul_gemm_int8(gate_up.to(dev), wd, wsd, bd, out) is out
    _check(out, *R.quantise(R.silu_mul(gate_up.double()), LOOSE), w, ws, b, dt, SILU)
    nw = (1 + 0.1 * torch.randn(K, generator=g)).to(dt)
    a, rows = R.norm(x, up, nw, 1e-6)
    for in_place in (False, True):
        res = up.to(dev)
        res_out = res if in_place else torch.full_like(res, float("nan"))
        out.fill_(float("nan"))
        assert v.resadd_norm_gemm_int8(x.to(dev), res, res_out, nw.to(dev), wd, wsd, bd, out, 1e-6) is out
        assert torch.equal(res_out.cpu(), (x.float() + up.float()).to(dt))
        assert in_place or torch.equal(res.cpu(), up)
        _check(out, *R.quantise(rows, LOOSE), w, ws, b, dt, NORM)


def test_codes_are_determined(v, dev):
    """Ties (an entry of half the largest is 63.5 steps) and their neighbours, over every fp16 and bf16 spacing: the identity as weights
    returns the codes."""
    K = 256
    eye, one = torch.eye(K, dtype=torch.int8, device=dev), torch.ones(K, device=dev)
    for dt in (torch.float16, torch.bfloat16):
        g = torch.Generator().manual_seed(3)
        m = (torch.rand(2000, 1, generator=g) + 0.5).to(dt)
        steps = torch.randint(-253, 254, (2000, K), generator=g)
        x = (m.double() * steps / 254).to(dt)
        nudge = torch.randint(-1, 2, x.shape, generator=g).to(torch.int16)
        x = (x.view(torch.int16) + torch.where(x == 0, 0, nudge).to(torch.int16)).view(dt)
        x = torch.where(x.abs() > m, m, x)
        x[:, :1] = m
        x[1] = x[1] * 2.0 ** -14                         # small numbers, fp16 subnormals among them
        x[2] = 0
        q, s, _ = R.quantise(x.double())
        # a code is at most 127: exact in 16 bits where the scale is a power of two, so the row's scale is taken out in 64 bits
        out = torch.empty(2000, K, dtype=dt, device=dev)
        v.gemm_int8(x.to(dev), None, eye, one, None, out)
        got = torch.round(out.cpu().double() / s[:, None])
        assert torch.equal(got, q)


def test_extreme_rows(v, dev):
    """Infinities and NaN: their own row is NaN, the others are untouched.  Zero rows, rows of the largest and of the smallest numbers."""
    for dt in (torch.float16, torch.bfloat16):
        for M in (1, 6, 70):
            g, x, w, ws, b = _case(M, 512, 72, dt, 5, bias=True)
            big, small = torch.finfo(dt).max, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
            kinds = [0.0, big, small, float("inf"), float("nan"), -float("inf")]
            kinds = kinds[:M] if M > 1 else kinds[4:5]
            for i, kind in enumerate(kinds):
                if kind == 0.0 or kind == big or kind == small:
                    x[i] = kind
                else:
                    x[i, 77] = kind
            xd, wd, wsd, bd = _to(dev, x, w, ws * 1e-3, b)
            out = torch.zeros(M, 72, dtype=dt, device=dev)
            v.gemm_int8(xd, None, wd, wsd, bd, out)
            bad = ~torch.isfinite(x).all(1)
            assert bool(out.cpu()[bad].isnan().all())
            q, s, near = R.quantise(x[~bad].double())
            _check(out[~bad.to(dev)], q, s, near, w, ws * 1e-3, b, dt, PLAIN)
            up = torch.ones_like(x)
            v.silu_mul_gemm_int8(torch.cat([xd, up.to(dev)], 1), wd, wsd, bd, out)
            # SiLU(-inf) is -inf / inf
            assert bool(out.cpu()[bad].isnan().all()) and bool(torch.isfinite(out.cpu()[~bad]).all())


def test_a_row_depends_on_itself_alone(v, dev):
    """Integer sums: a row's bits are the same whatever rows stand beside it, whichever kernel takes the call."""
    g, x, w, ws, b = _case(300, 2064, 200, torch.bfloat16, 9, bias=True)
    xd, wd, wsd, bd = _to(dev, x, w, ws, b)
    whole = torch.empty(300, 200, dtype=torch.bfloat16, device=dev)
    v.gemm_int8(xd, None, wd, wsd, bd, whole)
    for lo, hi in ((0, 1), (1, 3), (3, 8), (8, 30), (30, 94), (94, 300)):
        part = torch.empty(hi - lo, 200, dtype=torch.bfloat16, device=dev)
        v.gemm_int8(xd[lo:hi], None, wd, wsd, bd, part)
        assert torch.equal(part, whole[lo:hi])


@pytest.mark.parametrize("M", [1, 3, 20, 65, 300])
def test_nothing_outside_the_output_is_written(v, dev, M):
    """Outputs inside a larger buffer, starting off every wide boundary; views of x that start at a later row."""
    for N in (1, 37, 128, 203):
        g, x, w, ws, b = _case(M + 2, 272, N, torch.float16, N, bias=True)
        xd, wd, wsd, bd = _to(dev, x, w, ws, b)
        for lead in (1, 3, 8):
            buf = torch.full((lead + M * N + 64,), 7.0, dtype=torch.float16, device=dev)
            out = buf[lead:lead + M * N].view(M, N)
            v.gemm_int8(xd[2:], None, wd, wsd, bd, out)
            _check(out, *R.quantise(x[2:].double()), w, ws, b, torch.float16, PLAIN)
            assert bool((buf[:lead] == 7).all()) and bool((buf[lead + M * N:] == 7).all())


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_operands_on_odd_addresses(v, dev, M):
    """Scales, bias and row scales start on their element's boundary alone; the results are those of aligned ones."""
    K, N = 512, 203
    g, x, w, ws, b = _case(M, K, N, torch.float16, 22, bias=True)
    xd, wd, wsd, bd = _to(dev, x, w, ws, b)
    cs = (0.01 + 0.05 * torch.rand(M, generator=g)).to(dev)
    codes = R.codes_like_weights(g, M, K).to(dev)
    late = lambda t: torch.cat([t.new_zeros(1), t])[1:]
    new = lambda: torch.full((M, N), float("nan"), dtype=torch.float16, device=dev)
    want, got = [new(), new()], [new(), late(new().view(-1)).view(M, N)]
    for (a, s, r), out in zip(((wsd, bd, cs), (late(wsd), late(bd), late(cs))), (want, got)):
        v.gemm_int8(xd, None, wd, a, s, out[0])
        v.gemm_int8(codes, r, wd, a, s, out[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("M", [1, 4, 40, 130])
def test_weights_past_32_bit_offsets(v, dev, M):
    N, K = 36000, 65536                                   # 2.4 GB
    g = torch.Generator(device=dev).manual_seed(1)
    w = torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8)
    ws = torch.rand(N, generator=g, device=dev) * 1e-3
    x = torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=dev)
    v.gemm_int8(x, None, w, ws, None, out)
    pick = torch.tensor([0, 1, 16, 32766, 32767, 32768, 32769, 35983, 35999], device=dev)
    _check(out[:, pick], *R.quantise(x.cpu().double()), w[pick].cpu(), ws[pick].cpu(), None, torch.bfloat16, PLAIN)
    assert bool(torch.isfinite(out).all())


def test_outputs_past_32_bit_offsets(v, dev):
    M, N, K = 70000, 32776, 16                            # 4.6 GB of outputs
    g = torch.Generator(device=dev).manual_seed(2)
    x, w = (torch.randint(-127, 128, (n, K), generator=g, device=dev, dtype=torch.int8) for n in (M, N))
    xs, ws = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=dev)
    v.gemm_int8(x, xs, w, ws, None, out)
    rows = torch.tensor([0, 1, 32767, 65518, 65519, 65535, 65536, 69999], device=dev)
    none = torch.zeros(len(rows), K, dtype=torch.bool)
    _check(out[rows], x[rows].cpu().double(), xs[rows].cpu().double(), none, w.cpu(), ws.cpu(), None, torch.bfloat16, PLAIN)
    assert bool(torch.isfinite(out).all())


def test_no_rows_and_no_columns(v, dev):
    w, ws = torch.zeros(8, 32, dtype=torch.int8, device=dev), torch.ones(8, device=dev)
    x, out = torch.empty(0, 32, dtype=torch.float16, device=dev), torch.empty(0, 8, dtype=torch.float16, device=dev)
    assert v.gemm_int8(x, None, w, ws, None, out) is out
    assert v.silu_mul_gemm_int8(torch.empty(0, 64, dtype=torch.float16, device=dev), w, ws, None, out) is out
    x, res = torch.ones(2, 32, dtype=torch.float16, device=dev), torch.ones(2, 32, dtype=torch.float16, device=dev)
    res_out = torch.zeros_like(res)
    v.resadd_norm_gemm_int8(x, res, res_out, x[0], w[:0], ws[:0], None, torch.empty(2, 0, dtype=torch.float16, device=dev), 1e-6)
    assert bool((res_out == 2).all())


def test_refusals(v, dev):
    x = torch.ones(2, 32, dtype=torch.float16, device=dev)
    w, ws, out = torch.ones(8, 32, dtype=torch.int8, device=dev), torch.ones(8, device=dev), torch.empty(2, 8, dtype=torch.float16, device=dev)
    xs, nw = torch.ones(2, device=dev), torch.ones(32, dtype=torch.float16, device=dev)
    wide = torch.ones(2, 64, dtype=torch.int8, device=dev)
    both = torch.ones(4, 32, dtype=torch.float16, device=dev)
    odd = torch.ones(8 * 32 + 1, dtype=torch.int8, device=dev)
    bad = [(lambda: v.gemm_int8(x.float(), None, w, ws, None, out), "fp16 or bf16"),
           (lambda: v.gemm_int8(x, None, w, ws, None, out.bfloat16()), "like the output"),
           (lambda: v.gemm_int8(x, xs, w, ws, None, out), "must be int8"),
           (lambda: v.gemm_int8(x.to(torch.int8), None, w, ws, None, out), "fp16 or bf16"),
           (lambda: v.gemm_int8(x.to(torch.int8), xs[:1], w, ws, None, out), "x_scale must be fp32 with M=2"),
           (lambda: v.gemm_int8(x.to(torch.int8), xs.double(), w, ws, None, out), "x_scale must be fp32"),
           (lambda: v.gemm_int8(x, None, w.to(torch.uint8), ws, None, out), "weight must be int8"),
           (lambda: v.gemm_int8(x, None, w.view(-1), ws, None, out), "weight must be int8"),
           (lambda: v.gemm_int8(x, None, w[:, :24].contiguous(), ws, None, out), "multiple of 16"),
           (lambda: v.gemm_int8(x, None, w.t(), ws, None, out), "weight must be contiguous"),
           (lambda: v.gemm_int8(x.t(), None, w, ws, None, out), "input must be contiguous"),
           (lambda: v.gemm_int8(x[:, :16].contiguous(), None, w, ws, None, out), "rows must have 32"),
           (lambda: v.gemm_int8(x, None, w, ws.half(), None, out), "weight_scale must be fp32"),
           (lambda: v.gemm_int8(x, None, w, ws[:7], None, out), "weight_scale must be fp32 with N=8"),
           (lambda: v.gemm_int8(x, None, w, ws, ws, out), "bias must have N=8"),
           (lambda: v.gemm_int8(x, None, w, ws, nw[:7], out), "bias must have N=8"),
           (lambda: v.gemm_int8(x, None, w, ws, None, out[:1]), "expected M\\*N=16"),
           (lambda: v.gemm_int8(x, None, w, ws, None, x.view(-1)[:16].view(2, 8)), "must not overlap the input"),
           (lambda: v.gemm_int8(x, None, odd[1:].view(8, 32), ws, None, out), "16-byte boundary"),
           (lambda: v.gemm_int8(x, None, w.cpu(), ws, None, out), "same ROCm device"),
           (lambda: v.gemm_int8(x, None, w, ws, nw[:8].cpu(), out), "same ROCm device"),
           (lambda: v.gemm_int8(x, None, torch.ones(1, 131072, dtype=torch.int8, device=dev), ws[:1], None, out[:, :1].contiguous()), "below 131072"),
           (lambda: v.silu_mul_gemm_int8(x, w, ws, None, out), "rows must have 64"),
           (lambda: v.silu_mul_gemm_int8(wide, w, ws, None, out), "fp16 or bf16"),
           (lambda: v.resadd_norm_gemm_int8(x, x, both[1:3], nw, w, ws, None, out, 1e-6), None),
           (lambda: v.resadd_norm_gemm_int8(both[:2], both[2:], both[1:3], nw, w, ws, None, out, 1e-6), "must not overlap hidden_states"),
           (lambda: v.resadd_norm_gemm_int8(x, both[:2], both[1:3], nw, w, ws, None, out, 1e-6), "residual_out must be residual"),
           (lambda: v.resadd_norm_gemm_int8(x, both[:2], x, nw, w, ws, None, out, 1e-6), "must not overlap hidden_states"),
           (lambda: v.resadd_norm_gemm_int8(x, x.bfloat16(), both[:2], nw, w, ws, None, out, 1e-6), "must have the input's type"),
           (lambda: v.resadd_norm_gemm_int8(x, x, both[:3], nw, w, ws, None, out, 1e-6), "input's size"),
           (lambda: v.resadd_norm_gemm_int8(x, x, both[:2], nw[:16], w, ws, None, out, 1e-6), "norm_weight must have K=32")]
    for call, why in bad:
        if why is None:
            call()                                        # x as hidden_states and residual: read twice, allowed
            continue
        with pytest.raises(RuntimeError, match=why):
            call()


@pytest.mark.parametrize("M,K,N", [(1, 4096, 512), (16, 2048, 512), (64, 8192, 256), (300, 8192, 256)])
def test_graph_and_streams(v, dev, M, K, N):
    """Captured calls of two graphs, replayed with eager calls of other sizes between them and on two streams at a time: every result
    is the eager one."""
    from test_gpu_graph import _check_graph
    dt = torch.bfloat16
    g, x, w, ws, b = _case(M, K, N, dt, 21, bias=True)
    xd, wd, wsd, bd = _to(dev, x, w, ws, b)
    nw, up = torch.ones(K, dtype=dt, device=dev), torch.randn(M, K, generator=g).to(dt).to(dev)
    gate_up = torch.cat([xd, up], 1)
    outs = [torch.empty(M, N, dtype=dt, device=dev) for _ in range(3)]
    res_out = torch.empty_like(up)

    def run():
        v.gemm_int8(xd, None, wd, wsd, bd, outs[0])
        v.silu_mul_gemm_int8(gate_up, wd, wsd, None, outs[1])
        v.resadd_norm_gemm_int8(xd, up, res_out, nw, wd, wsd, bd, outs[2], 1e-6)
    _check_graph(dev, run, outs + [res_out])
    want = [o.clone() for o in outs]
    graphs, streams, sets = [], [torch.cuda.Stream(), torch.cuda.Stream()], []
    for st in streams:
        mine = [torch.empty_like(o) for o in outs]
        sets.append(mine)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            v.gemm_int8(xd, None, wd, wsd, bd, mine[0])
            v.silu_mul_gemm_int8(gate_up, wd, wsd, None, mine[1])
        graphs.append(graph)
    for _ in range(5):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        eager = torch.empty_like(outs[0])
        v.gemm_int8(xd, None, wd, wsd, bd, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for mine in sets:
            assert torch.equal(mine[0], want[0]) and torch.equal(mine[1], want[1])


# ------------------------------------------------------------------------------------------------ expert layer
def _moe(T, E, k, H, I, dt, seed, shared, ties=False):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=torch.randn(T, H, generator=g).to(dt), logits=torch.randn(T, E, generator=g).to(dt), w13=R.codes_like_weights(g, E, 2 * I, H),
             s13=R.scales(g, E, 2 * I), w2=R.codes_like_weights(g, E, H, I), s2=R.scales(g, E, H))
    if ties:
        c["logits"] = c["logits"].round()
    c.update(sw13=R.codes_like_weights(g, 2 * I, H), ss13=R.scales(g, 2 * I), sw2=R.codes_like_weights(g, H, I), ss2=R.scales(g, H),
             gw=(torch.randn(1, H, generator=g) * 0.05).to(dt)) if shared else c.update(sw13=None, ss13=None, sw2=None, ss2=None, gw=None)
    return c


def _moe_run(dev, c, k):
    d = {n: None if t is None else t.to(dev) for n, t in c.items()}
    out = torch.full_like(d["x"], float("nan"))
    r = torch.ops.moe_ops.moe_forward_full_int8(d["x"], d["logits"], out, d["w13"], d["s13"], d["sw13"], d["ss13"], d["w2"], d["s2"], d["sw2"],
                                                d["ss2"], d["gw"], k, 0 if c["gw"] is None else 1, d["w13"].shape[0])
    assert r is out
    return out.cpu()


def _moe_reference(dev, c, k):
    """(out, slack, sum of the summands' sizes); routing weights and gates are those of the framework's own selection.  An expert's row
    may pass from the down product to the weighted sum as 16-bit integers with a scale per 32 to 128 of its columns: off by half of
    1 / 32767 of their largest value, which is at most the row's (and that of its own error)."""
    from mi355x_qlinear import ops
    T, H = c["x"].shape
    E, dt = c["w13"].shape[0], c["x"].dtype
    tw, ids = torch.empty(T, k, dtype=dt, device=dev), torch.empty(T, k, dtype=torch.int32, device=dev)
    gate = torch.zeros(T, device=dev)
    ops.esimd_moe_topk(c["logits"].to(dev), tw, ids, T, gate=None if c["gw"] is None else (c["x"].to(dev), c["gw"].to(dev), gate))
    top = torch.argsort(c["logits"].double(), dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(ids.cpu().long(), top)
    tw, gate = tw.cpu().double(), gate.cpu().double()
    q, s, near = R.quantise(c["x"].double())

    def expert(rows, w13, s13, w2, s2):
        gu, _ = R.product(q[rows], s[rows], near[rows], w13, s13)
        y, sl = R.product(*R.quantise(R.silu_mul(gu), LOOSE), w2, s2)
        return y, sl + (y.abs() + sl).amax(1, keepdim=True) * (0.5 / 32767 * (1 + 2.0 ** -10))
    out, slack, parts = (torch.zeros(T, H, dtype=torch.float64) for _ in range(3))
    for e in range(E):
        rows, j = (top == e).nonzero(as_tuple=True)
        if rows.numel():
            y, sl = expert(rows, c["w13"][e], c["s13"][e], c["w2"][e], c["s2"][e])
            f = tw[rows, j][:, None]
            out[rows] += f * y
            slack[rows] += f * sl
            parts[rows] += f * y.abs()
    if c["gw"] is not None:
        y, sl = expert(torch.arange(T), c["sw13"], c["ss13"], c["sw2"], c["ss2"])
        out += gate[:, None] * y
        slack += gate[:, None] * sl
        parts += gate[:, None] * y.abs()
    return out, slack, parts


# one token, few, a row or none per expert, every route the same expert's neighbours, tiles that end inside an expert, sizes off every power of two
MOE = [(1, 1, 1, 16, 16), (1, 8, 2, 256, 128), (1, 32, 8, 2048, 768), (2, 5, 5, 272, 48), (3, 130, 8, 1040, 96), (4, 16, 4, 512, 256), (6, 64, 64, 128, 32),
       (8, 8, 8, 2048, 64), (12, 40, 8, 528, 208), (17, 300, 6, 640, 16), (33, 4, 2, 1024, 512), (64, 16, 8, 512, 112), (130, 3, 1, 400, 80),
       (200, 32, 4, 256, 256), (515, 8, 2, 144, 144), (1100, 6, 3, 96, 64), (5, 1024, 10, 64, 16), (1, 4, 2, 8192, 256), (2, 4, 4, 256, 4096), (100, 2, 2, 336, 80), (750, 3, 1, 208, 112),
       (4200, 8, 2, 64, 48), (480, 3, 1, 144, 160), (640, 3, 1, 160, 144), (1050, 3, 1, 208, 112)]


@pytest.mark.parametrize("T,E,k,H,I", MOE)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shared", [False, True])
def test_expert_layer(dev, T, E, k, H, I, dt, shared):
    import custom_esimd_kernels_vllm  # noqa: F401
    c = _moe(T, E, k, H, I, dt, T + E + H, shared, ties=T % 2 == 1)
    out, slack, parts = _moe_reference(dev, c, k)
    ok, worst = R.within(_moe_run(dev, c, k), out, slack, dt, SILU, parts)
    assert ok, f"{worst:.2f} of the tolerance"


def test_expert_layer_one_token_of_nan(dev):
    """A NaN in one token's row leaves the others as they were."""
    import custom_esimd_kernels_vllm  # noqa: F401
    for T in (2, 9, 150):
        c = _moe(T, 16, 4, 256, 64, torch.bfloat16, 4, True)
        want = _moe_run(dev, c, 4)
        c["x"][1, 5] = float("nan")
        got = _moe_run(dev, c, 4)
        others = torch.arange(T) != 1
        assert bool(got[1].isnan().all()) and torch.equal(got[others], want[others])


@pytest.mark.parametrize("T", [1, 5, 40, 200])
def test_expert_layer_graph(dev, T):
    import custom_esimd_kernels_vllm  # noqa: F401
    from test_gpu_graph import _check_graph
    c = {n: t.to(dev) for n, t in _moe(T, 24, 4, 512, 128, torch.float16, 6, True).items()}
    out = torch.empty_like(c["x"])
    _check_graph(dev, lambda: torch.ops.moe_ops.moe_forward_full_int8(c["x"], c["logits"], out, c["w13"], c["s13"], c["sw13"], c["ss13"], c["w2"], c["s2"],
                                                                      c["sw2"], c["ss2"], c["gw"], 4, 1, 24), [out])


@pytest.mark.parametrize("T", [1, 20, 40, 300, 5000])
def test_expert_layer_on_two_streams(dev, T):
    """Two captured calls of their own inputs replayed side by side, with an eager call of another size between."""
    import custom_esimd_kernels_vllm  # noqa: F401
    streams, sets = [torch.cuda.Stream(), torch.cuda.Stream()], []
    names = ("w13", "s13", "sw13", "ss13", "w2", "s2", "sw2", "ss2", "gw")

    def call(c, out):
        torch.ops.moe_ops.moe_forward_full_int8(c["x"], c["logits"], out, *[c[n] for n in names], 4, 1, 24)
    other = {n: t.to(dev) for n, t in _moe(33, 24, 4, 256, 128, torch.bfloat16, 40, True).items()}
    other_want, other_out = torch.empty_like(other["x"]), torch.empty_like(other["x"])
    call(other, other_want)
    for i in range(2):
        c = {n: t.to(dev) for n, t in _moe(T, 24, 4, 256, 128, torch.bfloat16, 30 + i, True).items()}
        want, out = torch.empty_like(c["x"]), torch.empty_like(c["x"])
        call(c, want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(c, out)
        sets.append((c, want, out, graph))
    for _ in range(5):
        for st, (c, want, out, graph) in zip(streams, sets):
            out.fill_(float("nan"))
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        other_out.fill_(float("nan"))
        call(other, other_out)
        torch.cuda.synchronize()
        assert torch.equal(other_out, other_want)
        for _, want, out, _ in sets:
            assert torch.equal(out, want)


@pytest.mark.parametrize("T", [1, 40, 700])
def test_expert_layer_on_odd_addresses(dev, T):
    import custom_esimd_kernels_vllm  # noqa: F401
    c = {n: t.to(dev) for n, t in _moe(T, 6, 2, 256, 80, torch.bfloat16, 13, True).items()}
    want = _moe_run(dev, c, 2)
    for n in ("logits", "s13", "s2", "ss13", "ss2"):
        c[n] = torch.cat([c[n].new_zeros(1), c[n].reshape(-1)])[1:].view(c[n].shape)
        assert c[n].data_ptr() % 16
    assert torch.equal(_moe_run(dev, c, 2), want)


def test_expert_layer_masked_and_bad_logits(dev):
    """Experts at -inf are taken last and weigh nothing; the token of a NaN logit is NaN, the others are as they were."""
    import custom_esimd_kernels_vllm  # noqa: F401
    for T in (1, 7, 150):
        c = _moe(T, 16, 4, 256, 64, torch.float16, 8, False)
        c["logits"][:, ::2] = float("-inf")
        c["logits"][0, 5:] = float("-inf")                # two experts left for four places
        out, slack, parts = _moe_reference(dev, c, 4)
        want = _moe_run(dev, c, 4)
        ok, worst = R.within(want, out, slack, torch.float16, SILU, parts)
        assert ok, f"{worst:.2f} of the tolerance"
        if T > 1:
            c["logits"][1, 3] = float("nan")
            got = _moe_run(dev, c, 4)
            others = torch.arange(T) != 1
            assert bool(got[1].isnan().all()) and torch.equal(got[others], want[others])


def test_expert_layer_nan_weight_scale(dev):
    """A NaN among the down product's scales reaches its own column and at most the 128 that share its tile, of the expert's tokens alone."""
    import custom_esimd_kernels_vllm  # noqa: F401
    for T in (1, 60, 300, 900):
        c = _moe(T, 4, 1, 512, 64, torch.bfloat16, 12, False)
        want = _moe_run(dev, c, 1)
        c["s2"][2, 200] = float("nan")
        got = _moe_run(dev, c, 1)
        hit = c["logits"].double().argmax(1) == 2
        assert bool(got[hit, 200].isnan().all()) and torch.equal(got[~hit], want[~hit])
        assert torch.equal(got[hit][:, :72], want[hit][:, :72]) and torch.equal(got[hit][:, 328:], want[hit][:, 328:])


@pytest.mark.parametrize("T", [3, 90, 900, 10000])
def test_expert_layer_all_to_one_expert(dev, T):
    """Every token takes the same two of many experts: one expert fills tile after tile, the others have no row."""
    import custom_esimd_kernels_vllm  # noqa: F401
    c = _moe(T, 200, 2, 64, 48, torch.bfloat16, 9, True)
    c["logits"][:, 199] += 20
    c["logits"][:, 70] += 20
    out, slack, parts = _moe_reference(dev, c, 2)
    ok, worst = R.within(_moe_run(dev, c, 2), out, slack, torch.bfloat16, SILU, parts)
    assert ok, f"{worst:.2f} of the tolerance"


@pytest.mark.parametrize("T", [1, 40, 700])
def test_expert_weights_past_32_bit_offsets(dev, T):
    """72 experts of 67 + 34 MB; the four that are taken lie at both ends and past 2^31 and 2^32 bytes."""
    import custom_esimd_kernels_vllm  # noqa: F401
    E, k, H, I, taken = 72, 2, 4096, 8192, [0, 33, 70, 71]
    c = _moe(T, 4, k, H, I, torch.bfloat16, 10, False)
    ops_in = {n: torch.zeros(E, *c[n].shape[1:], dtype=c[n].dtype, device=dev) for n in ("w13", "s13", "w2", "s2")}
    for n, t in ops_in.items():
        t[taken] = c[n].to(dev)
    logits = torch.full((T, E), float("-inf"), dtype=torch.bfloat16)
    logits[:, taken] = c["logits"]
    x = c["x"].to(dev)
    out = torch.full_like(x, float("nan"))
    torch.ops.moe_ops.moe_forward_full_int8(x, logits.to(dev), out, ops_in["w13"], ops_in["s13"], None, None, ops_in["w2"], ops_in["s2"], None, None,
                                            None, k, 0, E)
    few = torch.arange(T)[:: max(1, T // 8)]
    ref, slack, parts = _moe_reference(dev, {**c, "x": c["x"][few], "logits": c["logits"][few]}, k)
    ok, worst = R.within(out.cpu()[few], ref, slack, torch.bfloat16, SILU, parts)
    assert ok and bool(torch.isfinite(out).all()), f"{worst:.2f} of the tolerance"


def test_expert_results_past_32_bit_offsets(dev):
    """560000 routes of 4096 columns: more than 2^31 results between the down product and the sum."""
    import custom_esimd_kernels_vllm  # noqa: F401
    T, E, k, H, I = 70000, 8, 8, 4096, 16
    c = _moe(T, E, k, H, I, torch.bfloat16, 11, False)
    got = _moe_run(dev, c, k)
    few = torch.tensor([0, 1, 32767, 32768, 65535, 65536, 69998, 69999])
    ref, slack, parts = _moe_reference(dev, {**c, "x": c["x"][few], "logits": c["logits"][few]}, k)
    ok, worst = R.within(got[few], ref, slack, torch.bfloat16, SILU, parts)
    assert ok and bool(torch.isfinite(got).all()), f"{worst:.2f} of the tolerance"


def test_expert_layer_refusals(dev):
    import custom_esimd_kernels_vllm  # noqa: F401
    c = {n: t.to(dev) for n, t in _moe(2, 4, 2, 64, 32, torch.float16, 7, True).items()}
    names = ("x", "logits", "out", "w13", "s13", "sw13", "ss13", "w2", "s2", "sw2", "ss2", "gw")

    def call(k=2, shared=1, E=4, **kw):
        d = {**c, "out": torch.empty_like(c["x"]), **kw}
        return torch.ops.moe_ops.moe_forward_full_int8(*[d[n] for n in names], k, shared, E)
    call()
    for kw, why in (({"k": 5}, "top_k=5 of 4"), ({"k": 0}, "top_k=0"), ({"E": 3}, "must be"), ({"shared": 2}, "0 or 1"),
                    ({"shared": 0}, "given without a shared expert"), ({"gw": None}, "shared_expert_gate_weight is missing"),
                    ({"sw2": None}, "shared_down_weight is missing"), ({"logits": c["logits"].float()}, "logits must be"),
                    ({"w13": c["w13"].to(torch.uint8)}, "gate_up_weight must be"), ({"w2": c["w2"][:, :, :16]}, "down_weight must be"),
                    ({"w2": c["w2"].transpose(1, 2).contiguous().transpose(1, 2)}, "down_weight must be contiguous"),
                    ({"s13": c["s13"].half()}, "gate_up_scale must be"), ({"s2": c["s2"].cpu()}, "same ROCm device"),
                    ({"out": c["x"]}, "must not overlap x"), ({"x": c["x"].t().contiguous().t()}, "x must be contiguous"),
                    ({"out": torch.empty(2, 64, dtype=torch.bfloat16, device=dev)}, "output must be")):
        with pytest.raises(RuntimeError, match=why):
            call(**kw)


def test_a_layer_of_these_linears(v, dev):
    """Norm + projection, output projection, norm + gate and up, SiLU + down, as a decoder layer calls them, prompt and single tokens:
    every step against 64-bit math on what the step before left."""
    dt, H, F = torch.bfloat16, 512, 1360
    g = torch.Generator().manual_seed(12)
    w = {n: (R.codes_like_weights(g, o, i), R.scales(g, o)) for n, (o, i) in dict(qkv=(768, H), o=(H, 512), gu=(2 * F, H), down=(H, F)).items()}
    d = {n: (a.to(dev), b.to(dev)) for n, (a, b) in w.items()}
    nw = (1 + 0.1 * torch.randn(H, generator=g)).to(dt)
    for M in (1, 2, 37, 150):
        hidden, residual = torch.randn(M, H, generator=g).to(dt), torch.randn(M, H, generator=g).to(dt)
        hd, rd, nd = _to(dev, hidden, residual, nw)
        new = lambda n: torch.full((M, n), float("nan"), dtype=dt, device=dev)
        r1, qkv, o, r2, gu, y = new(H), new(768), new(H), new(H), new(2 * F), new(H)
        v.resadd_norm_gemm_int8(hd, rd, r1, nd, *d["qkv"], None, qkv, 1e-6)
        attn = qkv[:, :512].contiguous()
        v.gemm_int8(attn, None, *d["o"], None, o)
        v.resadd_norm_gemm_int8(o, r1, r2, nd, *d["gu"], None, gu, 1e-6)
        v.silu_mul_gemm_int8(gu, *d["down"], None, y)
        _check(qkv, *R.quantise(R.norm(hidden, residual, nw, 1e-6)[1], LOOSE), *w["qkv"], None, dt, NORM)
        _check(o, *R.quantise(attn.cpu().double()), *w["o"], None, dt, PLAIN)
        _check(gu, *R.quantise(R.norm(o.cpu(), r1.cpu(), nw, 1e-6)[1], LOOSE), *w["gu"], None, dt, NORM)
        _check(y, *R.quantise(R.silu_mul(gu.cpu().double()), LOOSE), *w["down"], None, dt, SILU)
