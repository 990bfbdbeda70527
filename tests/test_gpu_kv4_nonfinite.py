"""GPU: infinities, NaN and values past the largest scale on their way into the 4-bit cache, next to ordinary ones."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.test_gpu_kv4 import encode, pools, produce, rot_table, table_for

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv", [1, 3, 8])
def test_extreme_groups_beside_ordinary_ones(cuda_dev, D, Hkv):
    """Groups with a NaN, an infinity or a saturated scale in any place of a warp's pass: each has one scale, taken over
    both of its halves, and its neighbours are as if they were alone."""
    dev, B, S, P = cuda_dev, 1, 333, 16
    g = torch.Generator(device=dev)
    g.manual_seed(D + Hkv)
    x = torch.randn(S, 1 + 2 * Hkv, D // 32, 32, generator=g, device=dev)
    odd = torch.rand(x.shape[:3], generator=g, device=dev) < 0.4
    for n, value in enumerate((NAN, INF, -INF, 4000.0, 1e30)):
        at = torch.randint(0, 32, x.shape[:3], generator=g, device=dev)  # in either half of the group
        here = odd & (torch.rand(x.shape[:3], generator=g, device=dev) < 0.4)
        x = torch.where(here[..., None] & (torch.arange(32, device=dev) == at[..., None]), torch.full_like(x, value), x)
    x = x.flatten(2).bfloat16()
    pos = torch.arange(S, dtype=torch.int32, device=dev)
    table, total = table_for(B, (S + P - 1) // P, dev, 2)
    pl = pools(total, Hkv, P, D, dev)
    _, scr = produce(x.flatten(1).contiguous(), pos, None, 0, None, None, B, S, 1, Hkv, D, 0, ts.ATTN_ROPE_NEOX, table, P,
                     total, pl, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    pg, row = table[0].long()[pos.long() // P], pos.long() % P
    for codes, scales, src in ((pl[0], pl[1], x[:, 1:1 + Hkv]), (pl[2], pl[3], x[:, 1 + Hkv:])):
        wc, ws = encode(src)
        assert torch.equal(scales[pg, :, row], ws) and torch.equal(codes[pg, :, row], wc)


@pytest.mark.parametrize("D,rot,style", [(64, 64, ts.ATTN_ROPE_NEOX), (128, 64, ts.ATTN_ROPE_NEOX),
                                         (128, 128, ts.ATTN_ROPE_GPTJ), (64, 0, ts.ATTN_ROPE_NEOX)])
def test_nonfinite_keys_under_the_norm(cuda_dev, D, rot, style):
    """A key head with an infinity or a NaN is stored as the bf16 producer's row is (its root is zero or a NaN); the other
    heads' codes do not change."""
    dev, B, S, Hq, Hkv, P = cuda_dev, 1, 150, 2, 5, 16
    g = torch.Generator(device=dev)
    g.manual_seed(D + rot)
    x = torch.randn(S, Hq + 2 * Hkv, D, generator=g, device=dev).bfloat16()
    clean = x.clone()
    keys = x[:, Hq:Hq + Hkv]
    hit = torch.rand(S, Hkv, generator=g, device=dev) < 0.4
    for value in (INF, -INF, NAN):
        here = hit & (torch.rand(S, Hkv, generator=g, device=dev) < 0.5)
        at = torch.randint(0, D, (S, Hkv), generator=g, device=dev)
        keys[here[..., None] & (torch.arange(D, device=dev) == at[..., None])] = value
    hit = ~torch.isfinite(keys).all(-1)
    assert hit.any() and not hit.all()
    kw = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).bfloat16()
    pos = torch.arange(S, dtype=torch.int32, device=dev)
    table, total = table_for(B, (S + P - 1) // P, dev, 2)
    rt = rot_table(S, rot, dev) if rot else None
    got = []
    for src in (x, clean):
        pl = pools(total, Hkv, P, D, dev)
        _, scr = produce(src.flatten(1).contiguous(), pos, rt, S, kw, kw, B, S, Hq, Hkv, D, rot, style, table, P, total, pl,
                         dev)
        assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
        got.append(pl)
    q16 = torch.empty(B * Hq, S, D, dtype=torch.bfloat16, device=dev)
    k16, v16 = (torch.full((total, Hkv, P, D), NAN, dtype=torch.bfloat16, device=dev) for _ in range(2))
    rc = ts.attn_qkv_rope_paged_stream(x.flatten(1).contiguous(), pos, rt, S, kw, kw, 1e-6, B, S, Hq, Hkv, D, rot, style,
                                       q16, k16, v16, table, P, total, table.shape[1], scr)
    assert rc == ts.ATTN_OK
    pg, row = table[0].long()[pos.long() // P], pos.long() % P
    wc, ws = encode(k16[pg, :, row])
    codes, scales = got[0][0][pg, :, row], got[0][1][pg, :, row]
    assert torch.equal(scales[hit], ws[hit]) and torch.equal(codes[hit], wc[hit])
    for a, b in zip(got[0][:2], got[1][:2]):
        assert torch.equal(a[pg, :, row][~hit], b[pg, :, row][~hit])
