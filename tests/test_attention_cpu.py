"""Host-side answers of the attention entries: sizes, arguments, workspaces.  Nothing here reaches a launch."""
import ctypes

import pytest
import torch

from mi355x_qlinear import capi

OK = ctypes.c_void_p(256)
LL = ctypes.c_longlong


class Cache(ctypes.Structure):
    _fields_ = [("key", ctypes.c_void_p), ("value", ctypes.c_void_p), ("page_stride", LL), ("token_stride", LL), ("head_stride", LL),
                ("pages", ctypes.c_int), ("page_size", ctypes.c_int)]


def _cache(key=256, value=256, page_stride=2048, token_stride=128, head_stride=64, pages=10, page_size=16):
    return ctypes.byref(Cache(key, value, page_stride, token_stride, head_stride, pages, page_size))


def _size(T=4, B=2, Hq=8, Hkv=2, D=64, mq=2, mk=100):
    n = LL(-1)
    return capi.lib().mi_paged_attention_workspace(T, B, Hq, Hkv, D, mq, mk, ctypes.byref(n)), n.value


def test_workspace():
    assert _size()[0] == 0 and _size()[1] > 0
    assert _size(T=0) == _size(B=0) == (0, 0)
    one, many = _size(T=1, B=1, mq=1, mk=64)[1], _size(T=1, B=1, mq=1, mk=100000)[1]
    assert 0 < one < many                                               # no more parts than blocks of keys
    assert _size(T=200000, B=1, mq=200000, mk=200000) == (0, 0)         # a prompt of many tiles is not cut along its keys
    assert _size(T=200, B=1, mq=200, mk=200000)[1] >= 2 * 200 * 8 * 66 * 4
    for bad in (dict(D=32), dict(D=96), dict(D=512), dict(Hq=0), dict(Hkv=0), dict(Hq=7), dict(T=-1), dict(B=-1), dict(mq=-1), dict(mk=-1),
                dict(T=1 << 25), dict(B=1 << 24), dict(Hq=1 << 17), dict(T=2**31 - 1, Hq=65536, Hkv=1)):
        assert _size(**bad)[0] == -2, bad
    assert capi.lib().mi_paged_attention_workspace(1, 1, 1, 1, 64, 1, 1, None) == -1
    assert _size(T=2**31 - 1, B=1, Hq=1, Hkv=1)[0] == -2 and _size(T=(1 << 28) - 1, B=1, Hq=1, Hkv=1, mq=2**31 - 1, mk=2**31 - 1)[0] == 0
    # a grid holds less than 2^32 threads: a workgroup per tile and kv head, 512 threads each (256 with heads of 256), and a tile or more per sequence
    for D, most in ((64, 1 << 23), (128, 1 << 23), (256, 1 << 24)):
        many = dict(T=most // 8, Hq=8, Hkv=8, D=D, mq=100)
        assert _size(B=most // 8 - most // 64, **many)[0] == 0 and _size(B=most // 8, **many)[0] == -2
        assert _size(**dict(many, B=most // 8, mq=1))[0] == 0           # single tokens: a fixed number of workgroups


@pytest.mark.parametrize("tree", [False, True])
def test_attention_answers_bad_arguments_before_a_launch(tree):
    def call(q=OK, tok=512, head=64, cache=_cache(), table=OK, width=8, seq=OK, cu=OK, mask=OK, words=1, out=OK, ws=OK, n=1 << 40, T=4, B=2, Hq=8,
             Hkv=2, D=64, scale=0.1, window=-1, sinks=0, mq=2, mk=100, dt=0):
        a = [q, LL(tok), LL(head), cache, table, width, seq, cu]
        b = [out, ws, LL(n), T, B, Hq, Hkv, D, ctypes.c_float(scale)]
        if tree:
            return capi.lib().mi_tree_attention_ws(*a, mask, words, *b, mq, mk, dt, None)
        return capi.lib().mi_paged_attention_ws(*a, *b, window, sinks, mq, mk, dt, None)
    assert call(T=0) == call(B=0) == call(T=0, q=None, cache=None) == 0
    for name in ("q", "cache", "table", "seq", "cu", "out", "ws") + (("mask",) if tree else ()):
        assert call(**{name: None}) == -1, name
    for name in ("q", "out", "ws"):
        assert call(**{name: ctypes.c_void_p(264)}) == -1, name
    assert call(cache=_cache(key=264)) == call(cache=_cache(value=8)) == call(cache=_cache(key=None)) == call(cache=_cache(value=None)) == -1
    assert call(n=16) == -1 and call(dt=2) == -1 and call(dt=-1) == -1
    assert call(scale=0.0) == call(scale=-1.0) == call(scale=float("nan")) == call(scale=float("inf")) == -1
    assert call(cache=_cache(pages=0)) == call(cache=_cache(page_size=0)) == call(width=-1) == -1
    assert call(D=96) == call(Hq=7) == call(tok=4) == call(head=9) == call(mq=-1) == call(mk=-1) == -2
    assert call(cache=_cache(page_stride=2050)) == call(cache=_cache(token_stride=4)) == call(cache=_cache(head_stride=-64)) == -2
    assert call(width=1 << 27) == call(cache=_cache(page_size=1 << 28)) == -2
    assert call(cache=_cache(pages=2**31 - 1, page_stride=2048)) == -2                    # past 64 GiB
    if tree:
        assert call(words=0) == call(words=-1) == call(words=(1 << 20) + 1) == -2
    else:
        assert call(window=0) == call(window=-2) == call(sinks=-1) == -2


def test_rope_answers_bad_arguments_before_a_launch():
    def call(x=OK, xs=768, qw=OK, kw=OK, table=OK, pos=OK, q=OK, qt=512, qh=64, k=OK, kt=128, kh=64, cache=_cache(), slots=OK, T=4, Hq=8, Hkv=2, D=64,
             rot=64, places=10, dt=1):
        return capi.lib().mi_qk_norm_rope(x, LL(xs), qw, kw, table, 0, pos, q, LL(qt), LL(qh), k, LL(kt), LL(kh), cache, slots, T, Hq, Hkv, D, rot,
                                          places, ctypes.c_float(1e-6), 0, dt, None)
    assert call(T=0) == call(T=0, x=None) == 0
    for kw in (dict(x=None), dict(q=None), dict(table=None), dict(pos=None), dict(places=0), dict(k=None, cache=None, slots=None), dict(cache=None),
               dict(slots=None), dict(cache=_cache(key=None)), dict(cache=_cache(value=264)), dict(dt=2)):
        assert call(**kw) == -1, kw
    for name in ("x", "qw", "kw", "table", "q", "k"):
        assert call(**{name: ctypes.c_void_p(260)}) == -1, name
    for kw in (dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=96), dict(rot=8), dict(rot=80), dict(rot=-16), dict(places=-1), dict(xs=12), dict(qt=4), dict(qh=1),
               dict(kt=2), dict(kh=3), dict(cache=_cache(pages=0)), dict(cache=_cache(page_size=0)), dict(cache=_cache(head_stride=4)),
               dict(T=2**31 - 1), dict(T=1 << 26)):
        assert call(**kw) == -2, kw


def test_host_tensors_have_no_kernel():
    import custom_esimd_kernels_vllm as v
    q, kc = torch.zeros(1, 2, 64, dtype=torch.float16), torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    one = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        v.paged_attention(q, kc, kc.clone(), one, one[0], torch.zeros(2, dtype=torch.int32), q.clone(), 0.1, -1, 0, 1, 1)
    with pytest.raises(NotImplementedError):
        v.tree_attention(q, kc, kc.clone(), one, one[0], torch.zeros(2, dtype=torch.int32), one.long(), q.clone(), 0.1, 1, 1)
    with pytest.raises(NotImplementedError):
        v.qk_norm_rope(torch.zeros(1, 256, dtype=torch.float16), None, None, torch.zeros(4, 64), torch.zeros(1).long(), q, q[:, :1].clone(), None, None, None,
                       1e-6)


def test_fake_tensors_trace():
    import custom_esimd_kernels_vllm as v
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        new = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="cuda")
        q, kc, vc = new(3, 4, 64), new(5, 16, 2, 64), new(5, 16, 2, 64)
        i = lambda *s: new(*s, dtype=torch.int32)
        assert v.paged_attention(q, kc, vc, i(2, 4), i(2), i(3), new(3, 4, 64), 0.1, -1, 0, 2, 9).shape == (3, 4, 64)
        assert v.tree_attention(q, kc, vc, i(2, 4), i(2), i(3), new(3, 1, dtype=torch.int64), new(3, 4, 64), 0.1, 2, 9).shape == (3, 4, 64)
        x, where = new(3, 512), new(3, dtype=torch.int64)
        assert v.qk_norm_rope(x, None, None, new(9, 64), where, q, None, kc, vc, where, 1e-6).shape == (3, 4, 64)
