"""GPU: a page id outside the pool, found while earlier key blocks of a unit are still in the softmax, ends a call
of the prompt form with modified scores with an error, at once and with nothing left behind."""
from __future__ import annotations

import time

import pytest
import torch

import transfer_station_b200 as ts
from tests.test_gpu_mod import inputs, paged, scratch, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hq,Hkv,Sq,D,cap,bias", [
    (40, 24, 4, 4, 64, 0.0, 0),     # 24 rows of a kv head, the ranges read by the kernel itself
    (20, 8, 2, 40, 64, 0.0, 0),     # two row tiles, bounds and order
    (20, 8, 2, 40, 128, 30.0, 0),
    (20, 8, 2, 40, 64, 0.0, 1),     # the walk goes back from the query's position
    (40, 24, 4, 4, 64, 30.0, 1),
    (1, 24, 4, 4, 64, 0.0, 0),      # keys in pieces
])
def test_bad_page_under_ranges_with_gaps(cuda_dev, B, Hq, Hkv, Sq, D, cap, bias):
    P, Sk = 8, 2048 + 1500  # the producer holds 256 page ids at a time: the second lot begins at key 2048
    lens = [Sk] * B
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, B + Sq)
    kp, vp, table, total, per = paged(k, v, lens, P, cuda_dev, 3)
    i = torch.arange(Sq, device=cuda_dev, dtype=torch.int32)
    begin = (i * Sk // Sq).expand(B, Sq).contiguous()          # one row after another along the keys,
    end = (begin + Sk // Sq - 70).contiguous()                 # with slots between that none of them sees
    mod = ts.attn_mod(softcap=cap, slopes=slopes_of(Hq, cuda_dev) if bias else None, key_begin=begin, key_end=end)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    o, scr = torch.empty(B, Hq, Sq, D, device=cuda_dev), scratch(D, cuda_dev)

    def go():
        rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, n, o, ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, D, mod, P, total,
                                            per, scr)
        assert rc == ts.ATTN_OK, ts.strerror(rc)
        return ts.attn_flash_status(scr)

    assert go() == (ts.ATTN_OK, 0)
    want = o.clone()
    for page in (255, 256, 300, 40):
        for seq in {0, B // 2, B - 1}:
            good = table[seq, page].item()
            table[seq, page] = total
            start = time.monotonic()
            # the one report, and no wait that ran out (two seconds each)
            assert go() == (ts.ATTN_ERR_DEVICE, ts.ATTN_DEV_BAD_PAGE)
            assert time.monotonic() - start < 1.5
            table[seq, page] = good
            assert go() == (ts.ATTN_OK, 0) and torch.equal(o, want)
    table[:, 256:] = -1  # every unit at once
    assert go() == (ts.ATTN_ERR_DEVICE, ts.ATTN_DEV_BAD_PAGE)
