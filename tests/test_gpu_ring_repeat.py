"""GPU: attention of few rows, over bf16 keys and over the 4-bit cache, repeats bit for bit while another stream's stores
fill the memory pipes of the same SMs: a ring stage is read before the copy that refills it."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.test_gpu_kv4 import pools, run as run_kv4
from tests.test_gpu_mod import call, inputs, scratch

pytestmark = pytest.mark.gpu


def repeats(go, first, dev, reps=150):
    src = torch.zeros(96 << 20, dtype=torch.uint8, device=dev)
    dst = torch.empty_like(src)
    side, differ = torch.cuda.Stream(), torch.zeros((), dtype=torch.int64, device=dev)
    for _ in range(reps):
        with torch.cuda.stream(side):
            dst.copy_(src)
            src.add_(1)
        differ += (go() != first).any()
    torch.cuda.synchronize()
    assert differ.item() == 0


@pytest.mark.parametrize("D,Sq", [(64, 1), (128, 1), (128, 4)])
def test_bf16(cuda_dev, D, Sq):
    B, Hq, Hkv, Sk = 16, 16, 4, 4096
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, D)
    mod, scr, o = ts.attn_mod(softcap=50.0), scratch(D, cuda_dev), torch.empty(B, Hq, Sq, D, device=cuda_dev)
    first = call(q, k, v, mod)

    def go():
        assert ts.attn_flash_mod_stream(q, k, v, o, ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, Sk, D, mod, scr) == ts.ATTN_OK
        return o

    repeats(go, first, cuda_dev)


@pytest.mark.parametrize("D,Sq,P", [(64, 1, 64), (128, 1, 128), (128, 4, 64), (128, 1, 16)])
def test_4_bits(cuda_dev, D, Sq, P):
    dev, B, Hq, Hkv, L = cuda_dev, 16, 16, 4, 8192
    g = torch.Generator(device=dev)
    g.manual_seed(P + D)
    total = B * L // P
    pl = pools(total, Hkv, P, D, dev)
    for t in pl[0::2]:
        t.random_(0, 256, generator=g)
    for t in pl[1::2]:
        t.random_(0x20, 0x38, generator=g)
    table = torch.randperm(total, generator=g, device=dev).int().view(B, L // P).contiguous()
    lens = torch.full((B,), L, dtype=torch.int32, device=dev)
    q = torch.randn(B, Hq, Sq, D, generator=g, device=dev).bfloat16()
    first, scr = run_kv4(q, pl, table, total, lens, P, None, torch.float32, dev)
    assert torch.isfinite(first).all()
    o = torch.empty_like(first)
    repeats(lambda: run_kv4(q, pl, table, total, lens, P, None, torch.float32, dev, scr, o)[0], first, dev)
