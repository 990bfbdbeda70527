"""GPU: which entries of a block table attention with key ranges reads: none before the first key that a query of the
sequence sees, none behind the last (rounded to 128 keys in the form for prompts)."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible
from tests.test_gpu_kv4 import cache
from tests.test_gpu_kv4 import run as run_kv4
from tests.test_gpu_mod import check, inputs, paged, scratch, slopes_of

pytestmark = pytest.mark.gpu


def window(table, lens, P, lo, hi, total):
    """The table with no page in the entries wholly outside keys [lo, hi) of each sequence."""
    t = table.clone()
    for b, n in enumerate(lens):
        t[b, : lo[b] // P] = total
        t[b, (min(hi[b], n) + P - 1) // P:] = -1
    return t


def blind(begin, end, lens):
    """Queries that see nothing, their empty ranges at either end and outside."""
    for b, n in enumerate(lens):
        if begin.shape[1] > 2:
            begin[b, 0], end[b, 0] = ((0, 0), (-9, -3), (n, n))[b]
            begin[b, 1], end[b, 1] = ((n + 4, n + 8), (5, 5), (2 ** 31 - 1, -2 ** 31))[b]


@pytest.mark.parametrize("P", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(8, 2, 1), (8, 2, 3), (24, 2, 3), (4, 2, 40), (8, 2, 200)])
@pytest.mark.parametrize("cap,bias", [(0.0, 0), (30.0, 0), (0.0, 1), (20.0, 1)])
def test_bf16_pages_outside_the_ranges(cuda_dev, P, Hq, Hkv, Sq, cap, bias):
    dev, D, lens = cuda_dev, 64, [5000, 3071, 900]
    B, Sk = len(lens), max(lens)
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, dev, P + Sq)
    kp, vp, table, total, per = paged(k, v, lens, P, dev, 3)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    i = torch.arange(Sq, dtype=torch.int32, device=dev)
    sl = slopes_of(Hq, dev) if bias else None
    # a window that ends at the query's own position, and a range in the sequence's middle
    for begin, end in ((n.view(B, 1) - Sq + i - 300, n.view(B, 1) - Sq + i + 1),
                       (n.view(B, 1) // 2 - 200 + i, n.view(B, 1) // 2 + 77 + 0 * i)):
        begin, end = begin.contiguous(), end.contiguous()
        blind(begin, end, lens)
        seen = visible(B, Sq, lens, 0, begin, end, Sk, dev)
        some = [seen[b].any(0).nonzero() for b in range(B)]
        lo = [int(x.min()) // 128 * 128 for x in some]
        hi = [(int(x.max()) + 128) // 128 * 128 for x in some]
        t = window(table, lens, P, lo, hi, total)
        mod = ts.attn_mod(softcap=cap, slopes=sl, key_begin=begin, key_end=end)
        o, scr = torch.full((B, Hq, Sq, D), float("nan"), device=dev), scratch(D, dev)
        rc = ts.attn_flash_mod_paged_stream(q, kp, vp, t, n, o, ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, D, mod, P, total, per, scr)
        assert rc == ts.ATTN_OK, ts.strerror(rc)
        assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
        ref, tol = attend(q, k, v, seen, lens, cap, sl)
        check(o, ref, tol)


@pytest.mark.parametrize("P", [8, 32, 64, 256])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(8, 2, 1), (24, 2, 3), (4, 2, 16)])
def test_4_bit_pages_outside_the_ranges(cuda_dev, P, D, Hq, Hkv, Sq):
    dev, lens = cuda_dev, [5000, 3071, 900]
    B = len(lens)
    pl, table, total, k, v = cache(B, Hkv, D, lens, P, dev, P + Sq)
    g = torch.Generator(device=dev)
    g.manual_seed(P)
    q = torch.randn(B, Hq, Sq, D, generator=g, device=dev).bfloat16()
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    i = torch.arange(Sq, dtype=torch.int32, device=dev)
    for begin, end in ((n.view(B, 1) - Sq + i - 300, n.view(B, 1) - Sq + i + 1),
                       (n.view(B, 1) // 2 - 200 + i, n.view(B, 1) // 2 + 77 + 0 * i)):
        begin, end = begin.contiguous(), end.contiguous()
        blind(begin, end, lens)
        seen = visible(B, Sq, lens, 0, begin, end, k.shape[2], dev)
        some = [seen[b].any(0).nonzero() for b in range(B)]
        t = window(table, lens, P, [int(x.min()) for x in some], [int(x.max()) + 1 for x in some], total)
        o, scr = run_kv4(q, pl, t, total, lens, P, ts.attn_mod(key_begin=begin, key_end=end), torch.float32, dev)
        assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
        ref, tol = attend(q, k, v, seen, lens, p_half=2.0 ** -10, p_abs=2.0 ** -26)
        check(o, ref, tol)
