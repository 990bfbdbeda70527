"""CPU: what the 4-bit cache's entry points refuse, before any GPU work."""
from __future__ import annotations

import ctypes

import pytest

import transfer_station_b200 as ts

P = 1 << 20  # a non-null, aligned address: never read, every check is on the host
BAD_POOL = [dict(ps=0), dict(ps=24), dict(ps=192), dict(ps=-16), dict(npages=0), dict(maxp=0), dict(D=32), dict(D=96),
            dict(D=256), dict(B=-1), dict(Hkv=0), dict(kc=0), dict(ks=0), dict(vc=0), dict(vs=0), dict(bt=0),
            dict(scratch=0)]


def produce(**kw):
    a = dict(qkv=P, pos=P, cs=P, max_pos=64, qw=P, kw=P, eps=1e-6, B=2, S=3, Hq=8, Hkv=2, D=64, rot=64, style=1, Q=P, kc=P,
             ks=P, vc=P, vs=P, bt=P, ps=16, npages=4, maxp=2, scratch=P)
    a.update(kw)
    return ts.load_library().attn_qkv_rope_kv4_stream(
        a["qkv"], a["pos"], a["cs"], a["max_pos"], a["qw"], a["kw"], a["eps"], a["B"], a["S"], a["Hq"], a["Hkv"], a["D"],
        a["rot"], a["style"], a["Q"], a["kc"], a["ks"], a["vc"], a["vs"], a["bt"], a["ps"], a["npages"], a["maxp"],
        a["scratch"], None)


def unpack(**kw):
    a = dict(kc=P, ks=P, vc=P, vs=P, bt=P, pos=P, K=P, V=P, B=2, S=3, Hkv=2, D=64, ps=16, npages=4, maxp=2, scratch=P)
    a.update(kw)
    return ts.load_library().attn_kv4_unpack_stream(
        a["kc"], a["ks"], a["vc"], a["vs"], a["bt"], a["pos"], a["K"], a["V"], a["B"], a["S"], a["Hkv"], a["D"], a["ps"],
        a["npages"], a["maxp"], a["scratch"], None)


def attend(m=None, **kw):
    a = dict(Q=P, kc=P, ks=P, vc=P, vs=P, bt=P, sl=P, O=P, out=0, B=2, Hq=8, Hkv=2, Sq=1, D=64, ps=16, npages=4, maxp=2,
             scratch=P)
    a.update(kw)
    return ts.load_library().attn_flash_kv4_stream(
        a["Q"], a["kc"], a["ks"], a["vc"], a["vs"], a["bt"], a["sl"], a["O"], a["out"], a["B"], a["Hq"], a["Hkv"], a["Sq"],
        a["D"], None if m is None else ctypes.byref(m), a["ps"], a["npages"], a["maxp"], a["scratch"], None)


@pytest.mark.parametrize("bad", BAD_POOL + [dict(qkv=0), dict(pos=0), dict(Q=0), dict(S=-1), dict(Hq=0), dict(rot=3),
                                            dict(rot=80), dict(rot=-16), dict(max_pos=0), dict(cs=0), dict(style=9),
                                            dict(eps=-1.0), dict(B=1 << 20, S=1 << 12)])
def test_producer_arguments(built_lib, bad):
    assert produce(**bad) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("bad", BAD_POOL + [dict(pos=0), dict(K=0), dict(V=0), dict(S=-1), dict(B=1 << 20, S=1 << 12)])
def test_unpack_arguments(built_lib, bad):
    assert unpack(**bad) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("bad", BAD_POOL + [dict(Q=0), dict(O=0), dict(sl=0), dict(out=2), dict(out=-1), dict(Hq=6, Hkv=4),
                                            dict(B=0), dict(Sq=0), dict(ps=1 << 20, maxp=1 << 11), dict(B=1 << 29)])
def test_attention_arguments(built_lib, bad):
    assert attend(**bad) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("cap", [-1.0, 1e-4, 2e6, float("inf"), float("nan")])
def test_cap_out_of_bounds(built_lib, cap):
    assert attend(ts.attn_mod(softcap=cap)) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("name", ["kc", "ks", "vc", "vs", "Q"])
def test_misaligned(built_lib, name):
    assert attend(**{name: P + 8}) == ts.ATTN_ERR_ALIGN
    assert produce(**{name: P + 8}) == ts.ATTN_ERR_ALIGN
    if name != "Q":
        assert unpack(**{name: P + 8}) == ts.ATTN_ERR_ALIGN


def test_no_b200_is_reported(built_lib):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses are not memory")
    assert attend() == ts.ATTN_ERR_NOT_SM100
    assert produce() == ts.ATTN_ERR_NOT_SM100
    assert unpack() == ts.ATTN_ERR_NOT_SM100
