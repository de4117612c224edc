"""Windows that leave few keys of long contexts, whatever length the call is told: chunks by a workgroup per tile, single tokens and few ones in parts of what
they see."""
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def v(dev):
    import custom_esimd_kernels_vllm as v
    return v


@pytest.mark.parametrize("lens,news", [([9000], [1]), ([9000, 300], [40, 40]), ([9000], [300]), ([700], [700]), ([9000, 4000, 500], [300, 1, 20])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (130, 4), (1000, 0), (3000, 70)])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 12), (256, 32)])
def test_small_windows_over_long_contexts(v, dev, lens, news, window, sinks, D, page):
    case = R.make(dev, window + D, lens, news, 8, 2, D, page, torch.bfloat16)
    q, kc, vc, table, seq, cu, _ = case
    ref, tol = R.attention(q, kc, vc, table, lens, news, D ** -0.5, window, sinks)
    for told in (max(lens), 131072, window + 1):
        out = v.paged_attention(q, kc, vc, table, seq, cu, torch.full_like(q, float("nan")), D ** -0.5, window, sinks, max(news), told)
        worst = ((out.double() - ref).abs() / tol.clamp_min(1e-300)).max().item()
        assert not out.isnan().any() and worst <= 1.0, f"told {told}: {worst:.2f} of the tolerance"


def test_the_larger_workspace_serves_any_window(dev):
    """A workspace of the size that a call without a window needs, filled with NaN; and one of the size that the window needs, with nothing behind it touched."""
    import ctypes
    from mi355x_qlinear import capi
    lib, LL, P = capi.lib(), ctypes.c_longlong, ctypes.c_void_p

    class Cache(ctypes.Structure):
        _fields_ = [("key", P), ("value", P), ("page_stride", LL), ("token_stride", LL), ("head_stride", LL), ("pages", ctypes.c_int), ("page_size", ctypes.c_int)]
    D, Hq, Hkv = 128, 8, 2
    for lens, news, window in (([5000], [1], 300), ([5000, 700], [40, 9], 2500), ([5000], [40], 100)):
        q, kc, vc, table, seq, cu, _ = R.make(dev, window, lens, news, Hq, Hkv, D, 16, torch.bfloat16)
        ref, tol = R.attention(q, kc, vc, table, lens, news, D ** -0.5, window, 4)
        T, B = q.shape[0], len(lens)
        most, exact = LL(-1), LL(-1)
        assert lib.mi_paged_attention_workspace(T, B, Hq, Hkv, D, max(news), 5000, ctypes.byref(most)) == 0
        assert lib.mi_paged_attention_window_workspace(T, B, Hq, Hkv, D, window, 4, max(news), 5000, ctypes.byref(exact)) == 0
        assert 0 <= exact.value <= most.value
        cache = Cache(kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), kc.shape[0], kc.shape[1])
        for size in (most.value, exact.value):
            ws = torch.full((size // 4 + 1024,), float("nan"), device=dev)
            out = torch.full_like(q, float("nan"))
            torch.cuda.synchronize()
            assert lib.mi_paged_attention_ws(P(q.data_ptr()), q.stride(0), q.stride(1), ctypes.byref(cache), P(table.data_ptr()), table.shape[1],
                                             P(seq.data_ptr()), P(cu.data_ptr()), P(out.data_ptr()), P(ws.data_ptr()), size, T, B, Hq, Hkv, D, D ** -0.5,
                                             window, 4, max(news), 5000, 1, None) == 0
            torch.cuda.synchronize()
            assert not out.isnan().any() and ((out.double() - ref).abs() <= tol).all()
            assert ws[size // 4:].isnan().all()
