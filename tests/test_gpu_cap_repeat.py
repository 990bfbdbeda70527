"""GPU: capped scores of few rows over small pages give the same bits whatever an earlier call left in shared memory: the
slots of a tile whose page is not loaded, next to the sequence's last keys."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.test_gpu_kv4 import pools
from tests.test_gpu_kv4 import cache
from tests.test_gpu_kv4 import run as run_kv4
from tests.test_gpu_mod import inputs, paged, scratch

pytestmark = pytest.mark.gpu

LENS = [37, 5, 100, 133, 161, 300, 70, 19] * 20


@pytest.mark.parametrize("P", [8, 16, 32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (32, 2)])
def test_4_bit_cache(cuda_dev, P, D, Hq, Hkv):
    dev, B = cuda_dev, len(LENS)
    pl, table, total, _, _ = cache(B, Hkv, D, LENS, P, dev, P + D)
    g = torch.Generator(device=dev)
    g.manual_seed(P)
    q = torch.randn(B, Hq, 1, D, generator=g, device=dev).bfloat16()
    mod = ts.attn_mod(softcap=50.0)
    got = []
    for code, scale in ((0x88, 0x00), (0xFF, 0x7E)):  # zeros, and keys of 7 * 448
        other = pools(64, Hkv, 128, D, dev, code)
        other[1].fill_(scale), other[3].fill_(scale)
        t = torch.arange(64, dtype=torch.int32, device=dev).expand(64, 64).contiguous()
        run_kv4(torch.ones(64, Hq, 1, D, device=dev).bfloat16(), other, t, 64, [8192] * 64, 128, None, torch.float32, dev)
        o, scr = run_kv4(q, pl, table, total, LENS, P, mod, torch.float32, dev)
        assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
        got.append(o)
    assert torch.equal(*got)


@pytest.mark.parametrize("P", [8, 16, 32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (32, 2)])
def test_bf16_pages(cuda_dev, P, D, Hq, Hkv):
    dev, B = cuda_dev, len(LENS)
    q, k, v = inputs(B, Hq, Hkv, 1, max(LENS), D, dev, P)
    kp, vp, table, total, per = paged(k, v, LENS, P, dev, 3)
    n = torch.tensor(LENS, dtype=torch.int32, device=dev)
    mod, scr = ts.attn_mod(softcap=50.0), scratch(D, dev)
    got = []
    for size in (0.0, 1e4):
        ones = torch.full((64, Hkv, 4096, D), size, device=dev).bfloat16()
        junk = torch.empty(64, Hq, 1, D, device=dev)
        o = torch.empty(B, Hq, 1, D, device=dev)
        rc = ts.attn_flash_mod_stream(torch.ones_like(junk).bfloat16(), ones, ones, junk, ts.ATTN_OUT_F32, 64, Hq, Hkv, 1, 4096,
                                      D, ts.attn_mod(softcap=50.0), scr)
        assert rc == ts.ATTN_OK
        rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, n, o, ts.ATTN_OUT_F32, B, Hq, Hkv, 1, D, mod, P, total, per, scr)
        assert rc == ts.ATTN_OK and ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
        got.append(o)
    assert torch.equal(*got)
