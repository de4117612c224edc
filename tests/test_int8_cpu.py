"""Host-side answers of the 8-bit integer entries: sizes, arguments, workspaces.  Nothing here reaches a launch."""
import ctypes

import pytest
import torch

from mi355x_qlinear import capi

OK = ctypes.c_void_p(256)


def _ws(*a):
    n = ctypes.c_longlong(-1)
    return capi.lib().mi_gemm_int8_workspace(*a, ctypes.byref(n)), n.value


def test_workspace_of_the_linears():
    codes, act, norm, in_place, silu = range(5)
    for rows in (act, norm, in_place, silu):
        rc, n = _ws(rows, 100, 64, 4096)
        assert rc == 0 and n >= 100 * 4096 + 400
    assert _ws(codes, 100, 64, 4096) == (0, 0) and _ws(act, 0, 64, 4096)[0] == 0
    # one launch: none, unless the new residual is written over the old one
    assert _ws(act, 1, 64, 4096) == _ws(norm, 1, 64, 4096) == _ws(silu, 1, 64, 4096) == (0, 0) and _ws(in_place, 1, 64, 4096)[1] > 0
    assert _ws(act, 16, 64, 4096)[1] > 0 and _ws(act, 17, 64, 64)[1] > 0 and _ws(norm, 1, 0, 4096)[1] > 0
    for bad in ((-1, 64, 4096), (1, -1, 64), (1, 1, 0), (1, 1, 24), (1, 1, 131072)):
        assert _ws(act, *bad)[0] == -2
    assert _ws(5, 1, 1, 16)[0] == _ws(-1, 1, 1, 16)[0] == capi.lib().mi_gemm_int8_workspace(act, 1, 1, 16, None) == -1


def test_sizes_past_a_grid_are_refused():
    # a grid holds less than 2^32 threads, and an answer comes before the first launch (the residual is not written yet)
    for rows_from in range(5):
        assert _ws(rows_from, (1 << 24) - 1, 16, 16)[0] == _ws(rows_from, 1, (1 << 24) - 1, 16)[0] == _ws(rows_from, 1 << 20, 4096, 4096)[0] == 0
        for bad in ((1 << 24, 16, 16), (1, 1 << 24, 16), ((1 << 24) - 1, (1 << 24) - 1, 16), (2**31 - 1, 2**31 - 1, 16)):
            assert _ws(rows_from, *bad)[0] == -2, bad
    n = ctypes.c_longlong()
    size = capi.lib().mi_moe_forward_full_int8_workspace
    assert size(1 << 22, 2, 8, 256, 64, 1, ctypes.byref(n)) == 0 and size(1 << 23, 1, 8, 16, 16, 1, ctypes.byref(n)) == -2


def test_linears_answer_bad_arguments_before_a_launch():
    lib = capi.lib()
    f = ctypes.c_float(1e-6)

    def plain(x=OK, xs=None, w=OK, ws=OK, out=OK, buf=OK, n=1 << 40, M=20, N=8, K=32, dt=0):
        return lib.mi_gemm_int8_ws(x, xs, w, ws, None, out, buf, ctypes.c_longlong(n), M, N, K, dt, None)
    assert plain(M=0) == 0 and plain(M=0, x=None) == 0
    assert plain(dt=2) == -1 and plain(x=None) == -1 and plain(w=None) == -1 and plain(ws=None) == -1 and plain(out=None) == -1
    assert plain(buf=None) == -1 and plain(n=8) == -1
    assert plain(x=ctypes.c_void_p(264)) == -1 and plain(w=ctypes.c_void_p(257)) == -1 and plain(buf=ctypes.c_void_p(264)) == -1
    assert plain(K=24) == -2 and plain(K=131072) == -2 and plain(M=-1) == -2 and plain(N=-1) == -2 and plain(K=0) == -2

    def norm(x=OK, res=OK, ro=OK, nw=OK, M=20):
        return lib.mi_resadd_norm_gemm_int8_ws(x, res, ro, nw, f, OK, OK, None, OK, None, ctypes.c_longlong(0), M, 8, 32, 0, None)
    assert norm(M=0) == 0 and norm(res=None) == -1 and norm(ro=None) == -1 and norm(nw=None) == -1 and norm(x=None) == -1
    assert norm(res=ctypes.c_void_p(264)) == -1
    assert lib.mi_silu_mul_gemm_int8_ws(None, OK, OK, None, OK, OK, ctypes.c_longlong(1 << 40), 2, 8, 32, 0, None) == -1


def test_expert_layer_answers_bad_arguments_before_a_launch():
    lib = capi.lib()
    n = ctypes.c_longlong(-1)

    def size(T=4, k=2, E=8, H=64, I=32, shared=1):
        return lib.mi_moe_forward_full_int8_workspace(T, k, E, H, I, shared, ctypes.byref(n))
    assert size() == 0 and n.value > 0
    one = n.value
    assert size(shared=0) == 0 and n.value < one
    for bad in (dict(T=-1), dict(k=0), dict(k=9), dict(k=65, E=100), dict(E=0), dict(E=1025), dict(H=24), dict(I=24), dict(H=131072), dict(H=0),
                dict(H=65536, I=65536), dict(T=1 << 30, H=64)):
        assert size(**bad) == -2, bad

    def run(T=4, dt=1, nbytes=1 << 40, **kw):
        p = dict(x=OK, logits=OK, out=OK, w13=OK, s13=OK, sw13=OK, ss13=OK, w2=OK, s2=OK, sw2=OK, ss2=OK, gw=OK, buf=OK)
        p.update(kw)
        return lib.mi_moe_forward_full_int8_ws(*p.values(), ctypes.c_longlong(nbytes), T, 2, 8, 64, 32, dt, None)
    assert run(T=0) == 0 and run(dt=3) == -1 and run(T=-1) == -2 and run(nbytes=16) == -1
    for name in ("x", "logits", "out", "w13", "s13", "w2", "s2", "sw13", "ss13", "sw2", "ss2", "gw", "buf"):
        assert run(**{name: None}) == -1, name
    for name in ("x", "out", "w13", "w2", "sw13", "sw2", "gw", "buf"):
        assert run(**{name: ctypes.c_void_p(264)}) == -1, name


def test_host_tensors_have_no_kernel():
    import custom_esimd_kernels_vllm as v
    x, w = torch.zeros(1, 32, dtype=torch.float16), torch.zeros(8, 32, dtype=torch.int8)
    with pytest.raises(NotImplementedError):
        v.gemm_int8(x, None, w, torch.zeros(8), None, torch.zeros(1, 8, dtype=torch.float16))


def test_fake_tensors_trace():
    import custom_esimd_kernels_vllm as v
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(3, 32, dtype=torch.float16, device="cuda"), torch.empty(8, 32, dtype=torch.int8, device="cuda")
        out = torch.empty(3, 8, dtype=torch.float16, device="cuda")
        assert v.gemm_int8(x, None, w, torch.empty(8, device="cuda"), None, out).shape == (3, 8)
