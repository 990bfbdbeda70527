"""GPU: the paged call with modified scores where nothing modifies them: rows of a page behind the sequence's end are no
numbers there either."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible
from tests.test_gpu_mod import check, inputs, paged, scratch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,Sq,D,P", [
    ([184], 32, 8, 17, 128, 16),                  # one row tile
    ([405, 1, 129, 0], 4, 2, 1, 64, 16),          # single tokens
    ([579, 104, 386], 8, 8, 8, 72, 64),
    ([3], 2, 2, 9, 120, 256),                     # a page longer than the sequence
    ([135, 300, 71, 0, 43], 56, 8, 60, 64, 8),    # two row tiles, more units than SMs
    ([3000], 24, 2, 3, 128, 128),                 # keys in pieces
])
@pytest.mark.parametrize("causal", [None, 0, 1])  # None: no struct at all
def test_no_modifier_over_pages(cuda_dev, lens, Hq, Hkv, Sq, D, P, causal, out, fill):
    B, Sk, dev = len(lens), max(lens), cuda_dev
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, dev, sum(lens) + D)
    kp, vp, table, total, per = paged(k, v, lens, P, dev, 3, fill=fill)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    o, scr = torch.full((B, Hq, Sq, D), float("nan"), dtype=out, device=dev), scratch(D, dev)
    mod = None if causal is None else ts.attn_mod(causal=causal)
    rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, n, o, ts.ATTN_OUT_BF16 if out == torch.bfloat16 else ts.ATTN_OUT_F32,
                                        B, Hq, Hkv, Sq, D, mod, P, total, per, scr)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    seen = visible(B, Sq, lens, causal, Sk=Sk, dev=dev)
    ref, tol = attend(q, k, v, seen, lens, out=out)
    check(o, ref, tol)
    assert (o.transpose(1, 2)[~seen.any(2)] == 0).all()
