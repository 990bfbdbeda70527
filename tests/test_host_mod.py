"""CPU: what attn_flash_mod_* and attn_mask_ranges_stream refuse, before any GPU work."""
from __future__ import annotations

import ctypes

import pytest

import transfer_station_b200 as ts

P = 1 << 20  # a non-null, aligned address: never read, every check is on the host


def mod(**kw):
    m = ts.attn_mod(softcap=kw.pop("softcap", 0.0), causal=kw.pop("causal", 0))
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def contiguous(m, **kw):
    a = dict(Q=P, K=P, V=P, O=P, out=0, B=2, Hq=8, Hkv=2, Sq=4, Sk=16, D=64, scratch=P)
    a.update(kw)
    return ts.load_library().attn_flash_mod_stream(a["Q"], a["K"], a["V"], a["O"], a["out"], a["B"], a["Hq"], a["Hkv"],
                                                   a["Sq"], a["Sk"], a["D"], None if m is None else ctypes.byref(m),
                                                   a["scratch"], None)


def paged(m, **kw):
    a = dict(Q=P, K=P, V=P, bt=P, sl=P, O=P, out=0, B=2, Hq=8, Hkv=2, Sq=1, D=64, ps=16, npages=4, maxp=2, scratch=P)
    a.update(kw)
    return ts.load_library().attn_flash_mod_paged_stream(
        a["Q"], a["K"], a["V"], a["bt"], a["sl"], a["O"], a["out"], a["B"], a["Hq"], a["Hkv"], a["Sq"], a["D"],
        None if m is None else ctypes.byref(m), a["ps"], a["npages"], a["maxp"], a["scratch"], None)


@pytest.mark.parametrize("bad", [dict(Q=0), dict(K=0), dict(V=0), dict(O=0), dict(scratch=0), dict(out=2), dict(out=-1),
                                 dict(B=0), dict(Hq=6, Hkv=4), dict(Hkv=0), dict(Sq=0), dict(Sk=0), dict(D=0),
                                 dict(D=257), dict(B=1 << 28), dict(B=1 << 16, Sk=1 << 15)])
def test_contiguous_arguments(built_lib, bad):
    assert contiguous(mod(softcap=30.0), **bad) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("bad", [dict(bt=0), dict(sl=0), dict(O=0), dict(out=5), dict(ps=24), dict(D=36), dict(D=136),
                                 dict(npages=0), dict(maxp=0), dict(B=0), dict(Hq=6, Hkv=4)])
def test_paged_arguments(built_lib, bad):
    assert paged(mod(softcap=30.0), **bad) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("cap", [-1.0, 1e-4, 2e6, float("inf"), float("nan")])
def test_cap_out_of_bounds(built_lib, cap):
    assert contiguous(mod(softcap=cap)) == ts.ATTN_ERR_ARGS
    assert paged(mod(softcap=cap)) == ts.ATTN_ERR_ARGS


@pytest.mark.parametrize("field", ["slopes", "key_begin", "key_end"])
def test_misaligned_arrays(built_lib, field):
    if ts.load_library().attn_mask_ranges_stream(P, None, 1, 8, 1, 0, P, P + 2, None) != ts.ATTN_ERR_ALIGN:
        pytest.fail("attn_mask_ranges_stream took a misaligned array")
    assert contiguous(mod(**{field: P + 2})) == ts.ATTN_ERR_ALIGN
    assert paged(mod(**{field: P + 2})) == ts.ATTN_ERR_ALIGN


@pytest.mark.parametrize("bad", [dict(cu=0), dict(begin=0), dict(end=0), dict(n=0), dict(S=0), dict(window=-1),
                                 dict(prefix=P, window=4)])
def test_mask_ranges_arguments(built_lib, bad):
    a = dict(cu=P, prefix=None, n=2, S=8, causal=1, window=0, begin=P, end=P)
    a.update(bad)
    rc = ts.load_library().attn_mask_ranges_stream(a["cu"], a["prefix"], a["n"], a["S"], a["causal"], a["window"],
                                                   a["begin"], a["end"], None)
    assert rc == ts.ATTN_ERR_ARGS


def test_no_b200_is_reported(built_lib):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert contiguous(mod(softcap=30.0)) == ts.ATTN_ERR_NOT_SM100
    assert contiguous(None) == ts.ATTN_ERR_NOT_SM100
    assert paged(mod(causal=1)) == ts.ATTN_ERR_NOT_SM100


def test_more_kv_heads_than_heads(built_lib):
    """Refused before the product of batch and kv heads is formed."""
    assert contiguous(mod(softcap=30.0), B=1 << 20, Hq=8, Hkv=1 << 20) == ts.ATTN_ERR_ARGS
