"""Which way the attention over a paged cache takes, as its workspace tells: parts of tiles that are cut along their keys, or none."""
import ctypes

import pytest

from mi355x_qlinear import capi


def _size(T, B, Hq, Hkv, D, mq, mk, window=None, sinks=0):
    n = ctypes.c_longlong(-1)
    if window is None:
        rc = capi.lib().mi_paged_attention_workspace(T, B, Hq, Hkv, D, mq, mk, ctypes.byref(n))
    else:
        rc = capi.lib().mi_paged_attention_window_workspace(T, B, Hq, Hkv, D, window, sinks, mq, mk, ctypes.byref(n))
    return n.value if rc == 0 else rc


# chunks and prompts in a window: a workgroup per tile sees the window, an equal share all that any token of the call sees
@pytest.mark.parametrize("T,Hq,Hkv,D,L,window", [(8192, 64, 8, 64, 131072, 1024), (2048, 64, 8, 128, 65536, 1024), (2048, 64, 8, 256, 65536, 1024),
                                                 (6000, 8, 1, 64, 6000, 512), (6000, 8, 1, 128, 6000, 512), (512, 16, 2, 128, 16384, 512)])
def test_long_calls_in_a_window_have_a_workgroup_per_tile(T, Hq, Hkv, D, L, window):
    assert _size(T, 1, Hq, Hkv, D, T, L, window) == 0


def test_few_tokens_in_a_wide_window_are_cut_along_their_keys():
    assert _size(40, 1, 32, 8, 128, 40, 131072, 100000) > 0
    assert _size(160, 4, 32, 8, 128, 40, 32768, 4096, 4) > 0
    assert _size(40, 1, 32, 8, 128, 40, 131072, 100) == 0              # a hundred keys are not worth it


def test_single_tokens_have_parts_for_what_they_see():
    """As many as if the sequence were no longer than the window."""
    for D in (64, 128, 256):
        for window, sinks in ((1, 0), (128, 4), (1024, 64)):
            for B in (1, 3):
                full, told = _size(B, B, 64, 8, D, 1, 131072), _size(B, B, 64, 8, D, 1, window + sinks + 32)
                assert _size(B, B, 64, 8, D, 1, 131072, window, sinks) == told <= full
                assert _size(B, B, 64, 8, D, 1, 100, 1000, sinks) == _size(B, B, 64, 8, D, 1, 100)     # a window longer than the sequence


def test_a_window_never_needs_more():
    """The workspace that the call without one needs is enough, whatever the window."""
    for D in (64, 128, 256):
        for T, B, mq in ((1, 1, 1), (64, 64, 1), (300, 5, 100), (4000, 2, 2000), (4000, 4000, 1), (9000, 30, 4000), (40, 1, 40), (20000, 1, 20000)):
            for Hq, Hkv in ((8, 8), (32, 8), (16, 1)):
                for mk in (0, 1, 500, 3000, 40000, 2 ** 31 - 1):
                    most = _size(T, B, Hq, Hkv, D, mq, mk)
                    for window in (1, 31, 700, 1900, 30000, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, -1):
                        for sinks in (0, 4, 5000, 2 ** 31 - 1):
                            n = _size(T, B, Hq, Hkv, D, mq, mk, window, sinks)
                            assert 0 <= n <= most, (T, B, Hq, Hkv, D, mq, mk, window, sinks)
                            if window in (-1, 2 ** 30, 2 ** 31 - 1):
                                assert n == most


def test_refusals():
    good = dict(T=4, B=2, Hq=8, Hkv=2, D=64, mq=2, mk=100, window=10, sinks=0)
    assert _size(**good) > 0
    for bad in (dict(window=0), dict(window=-2), dict(sinks=-1), dict(D=96), dict(Hq=7), dict(T=-1), dict(B=1 << 24), dict(mq=-1), dict(mk=-1)):
        assert _size(**dict(good, **bad)) == -2, bad
    assert capi.lib().mi_paged_attention_window_workspace(1, 1, 1, 1, 64, -1, 0, 1, 1, None) == -1
