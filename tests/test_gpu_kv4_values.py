"""GPU: the values of the 4-bit cache in the attention over it, at every scale and every size of weight. The bounds are
relative to sum_j p_j |v_j|: they shrink with the values."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend
from tests.test_gpu_kv4 import cache, check, decode, run, table_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_every_value_of_every_scale(cuda_dev, D):
    """One key a sequence: the output is the value itself, each product exact.

    The bound: the key's score less its reference (itself less 12) is rounded twice at that size, 2^-21 each, its
    exponential and 1 / l are good to 2^-22, the last product to 2^-24: below 2^-19 in all. (The weight in fp16 is
    then 2^12 to the last bit.)"""
    dev, P, Hkv, B = cuda_dev, 8, 1, 126
    pl = [torch.full((B, Hkv, P, n), 0x7F, dtype=torch.uint8, device=dev) for n in (D // 2, D // 32, D // 2, D // 32)]
    g = torch.Generator(device=dev)
    g.manual_seed(D)
    pl[0][:, :, 0], pl[1][:, :, 0] = 0x88, 0x38
    n = torch.stack([torch.arange(D, device=dev).roll(b) for b in range(B)]) % 16  # every code in every place
    pl[2][:, 0, 0] = (n[:, 0::2] | (n[:, 1::2] << 4)).to(torch.uint8)
    pl[3][:, 0, 0] = torch.arange(1, 127, device=dev, dtype=torch.uint8)[:, None]   # all scales but zero
    table = torch.arange(B, dtype=torch.int32, device=dev).view(B, 1)
    q = torch.randn(B, 4, 1, D, generator=g, device=dev).bfloat16()
    o, scr = run(q, pl, table, B, [1] * B, P, None, torch.float32, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    want = decode(pl[2][:, 0, 0], pl[3][:, 0, 0])[:, None, None].expand_as(o)
    assert ((o.double() - want).abs() <= 2.0 ** -19 * want.abs()).all()


@pytest.mark.parametrize("scale", [0x20, 0x10, 0x08, 0x01])  # 2^-3, 2^-5, 2^-6 and the smallest, 2^-9
@pytest.mark.parametrize("D,Hkv,Hq", [(128, 1, 8), (64, 1, 16), (128, 2, 4)])
@pytest.mark.parametrize("equal", [True, False])
def test_small_values_behind_one_heavy_key(cuda_dev, scale, D, Hkv, Hq, equal):
    """Contexts whose first key holds most of the weight and stands for zeros, the others' values small: the output is
    made of weights 2^13 to 2^22 times below the largest. More sequences than CTAs (they share the pages), so that a
    warp meets the heavy key and a fourth of the others under one reference.

    The bound: a weight is rounded to fp16 once, 2^-11 of itself; below 2^-14 by half of the smallest step, 2^-25.
    The largest weight is at least 2^12 and l no less, so that is 2^-37 |v| for each key. The rest as in attend()."""
    dev, B, L, P = cuda_dev, 900, 16384, 128
    per = L // P
    table, total = table_for(1, per, dev, D + scale)
    g = torch.Generator(device=dev)
    g.manual_seed(scale + D)
    rnd = lambda n: torch.randint(0, 256, (1, L, Hkv, n), generator=g, device=dev, dtype=torch.uint8)  # noqa: E731
    kc, vc = rnd(D // 2), rnd(D // 2)
    ks = torch.full((1, L, Hkv, D // 32), 0x00 if equal else 0x08, dtype=torch.uint8, device=dev)
    vs = torch.full((1, L, Hkv, D // 32), scale, dtype=torch.uint8, device=dev)
    kc[:, 0], ks[:, 0], vs[:, 0] = 0xFF, 0x24, 0  # 7 * 0.1875 in every element
    # q: its sum gives the heavy key 13 to 22 log2 units (9 to 15.2 nats)
    nats = torch.linspace(9.0, 15.2, Hq, device=dev)
    q = (nats * D ** 0.5 / (D * 7 * 0.1875)).view(1, Hq, 1, 1).expand(1, Hq, 1, D).bfloat16().contiguous()
    pl = [torch.zeros(total, Hkv, P, n, dtype=torch.uint8, device=dev) for n in (D // 2, D // 32, D // 2, D // 32)]
    t = torch.arange(L, device=dev)
    pg, row = table[0].long()[t // P], t % P
    for pool, x in zip(pl, (kc, ks, vc, vs)):
        pool[pg, :, row] = x[0]
    o, scr = run(q.expand(B, -1, -1, -1).contiguous(), pl, table.expand(B, -1).contiguous(), total, [L] * B, P, None,
                 torch.float32, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    k, v = decode(kc, ks).transpose(1, 2), decode(vc, vs).transpose(1, 2)
    ref, tol = attend(q, k, v, torch.ones(1, 1, L, dtype=torch.bool, device=dev), [L], p_half=2.0 ** -11)
    tol += 2.0 ** -37 * v.abs().sum(2, keepdim=True).repeat_interleave(Hq // Hkv, 1)
    check(o, ref, tol)


@pytest.mark.parametrize("e", [90, 104, 110, 118, 125])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_queries_near_the_largest_number(cuda_dev, e, D, cap):
    """Query rows up to 2^127: their largest score takes all the weight, or under a cap every positive one has the same.

    The bound: weights are 2^12 times one or nothing (under a cap e^60 apart), so what remains is 1 / l, and the sum of
    up to 333 values in 32 bits: 2^-14 of it."""
    dev, L, Hq, Hkv, P = cuda_dev, 333, 8, 2, 32
    pl, table, total, k, v = cache(1, Hkv, D, [L], P, dev, e)
    g = torch.Generator(device=dev)
    g.manual_seed(e + D)
    q = (torch.randn(1, Hq, 1, D, generator=g, device=dev).clamp(-3.5, 3.5).double() * 2.0 ** e).bfloat16()
    assert torch.isfinite(q).all()
    o, scr = run(q, pl, table, total, [L], P, ts.attn_mod(softcap=cap), torch.float32, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    kk, vv = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = q.double() @ kk.transpose(-1, -2)  # [1][Hq][1][L]
    w = (s > 0).double() if cap else (s == s.amax(-1, keepdim=True)).double()
    w = w / w.sum(-1, keepdim=True)
    err = (o.double() - w @ vv).abs()
    assert (err <= 2.0 ** -14 * (w @ vv.abs())).all()
