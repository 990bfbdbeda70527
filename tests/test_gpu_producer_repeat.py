"""GPU: the QKV producer's bytes repeat. The kernel streams its input through a ring of shared-memory stages while its
stores fill the memory pipe; a stage that is refilled before it has been read shows as one call in a few hundred whose
rows hold another chunk's bytes."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.test_gpu_kv4 import rot_table, scratch, table_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,style,norm,paged", [
    (2, 1479, 63, 9, 128, 32, ts.ATTN_ROPE_GPTJ, 0, 1),
    (2, 1479, 63, 9, 128, 128, ts.ATTN_ROPE_NEOX, 1, 1),
    (1, 2048, 32, 8, 128, 128, ts.ATTN_ROPE_NEOX, 1, 0),
    (1, 3001, 32, 8, 64, 64, ts.ATTN_ROPE_NEOX, 0, 0),
    (3, 999, 35, 5, 64, 16, ts.ATTN_ROPE_GPTJ, 0, 1),
    (1, 1500, 16, 2, 256, 64, ts.ATTN_ROPE_NEOX, 0, 0),
])
def test_producer_repeats(cuda_dev, B, S, Hq, Hkv, D, rot, style, norm, paged):
    dev, P, past, reps = cuda_dev, 16, 333, 800
    g = torch.Generator(device=dev)
    g.manual_seed(S + D)
    x = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=g, device=dev).bfloat16()
    w = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).bfloat16() if norm else None
    pos = (torch.arange(S, dtype=torch.int32, device=dev) + past).repeat(B)
    rt, scr = rot_table(past + S, rot, dev), scratch(D, dev)
    per = (past + S + P - 1) // P
    table, total = table_for(B, per, dev, 1)

    def outputs():
        q = torch.full((B * Hq, S, D), 77.0, dtype=torch.bfloat16, device=dev)
        k, v = (torch.full((total, Hkv, P, D) if paged else (B * Hkv, past + S, D), 77.0, dtype=torch.bfloat16, device=dev)
                for _ in range(2))
        return q, k, v

    def go(q, k, v):
        a = (x, pos, rt, past + S, w, w, 1e-6, B, S, Hq, Hkv, D, rot, style, q, k, v)
        rc = (ts.attn_qkv_rope_paged_stream(*a, table, P, total, per, scr) if paged else
              ts.attn_qkv_rope_stream(*a, past + S, scr))
        assert rc == ts.ATTN_OK, ts.strerror(rc)

    first, again = outputs(), outputs()
    go(*first)
    # value heads are copied: the first call against its input
    vh = x.view(B, S, Hq + 2 * Hkv, D)[:, :, Hq + Hkv:]
    if paged:
        b = torch.arange(B, device=dev).repeat_interleave(S)
        got = first[2][table.long()[b, pos.long() // P], :, pos.long() % P].view(B, S, Hkv, D)
    else:
        got = first[2].view(B, Hkv, past + S, D)[:, :, past:].transpose(1, 2)
    assert torch.equal(got.view(torch.int16), vh.view(torch.int16))
    differ = torch.zeros((), dtype=torch.int64, device=dev)
    for _ in range(reps):
        go(*again)
        for s, t in zip(first, again):
            differ += (s.view(torch.int64) != t.view(torch.int64)).any()
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    assert differ.item() == 0
