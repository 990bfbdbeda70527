"""GPU: the softmax of the prompt form with modified scores where its paths meet."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible
from tests.test_gpu_mod import call, check, inputs, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Sq", [30, 300])  # one row tile a unit, two
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [0, 1])
@pytest.mark.parametrize("step", [6.0, 9.0])
def test_maximum_moves_at_every_block(cuda_dev, Sq, D, bias, step):
    """Each block's scores lie `step` above those of the block before (8.7 and 13 in log2 units, past what the
    speculation takes), so every block's weights are stored twice; the last block's make up the result."""
    B, Hq, Hkv, Sk = 2, 6, 2, 1280
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 31 + Sq + D)
    q[..., 0] = 1.0
    k[..., 0] = step * D ** 0.5 * (torch.arange(Sk, device=cuda_dev) // 128)
    lo = torch.zeros(B, Sq, dtype=torch.int32, device=cuda_dev)
    sl = slopes_of(Hq, cuda_dev, 0.01) if bias else None
    mod = ts.attn_mod(slopes=sl, key_begin=lo)
    o = call(q, k, v, mod)
    seen = visible(B, Sq, [Sk] * B, 0, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, [Sk] * B, 0.0, sl)
    check(o, ref, tol)
    for _ in range(5):
        assert torch.equal(call(q, k, v, mod), o)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,causal,cap,signs", [
    (1, 4, 2, 300, 1500, 128, 1, 50.0, "-"),   # 216 log2 units of bias over the keys
    (1, 4, 2, 300, 1500, 64, 0, 30.0, "-"),    # keys ahead of the query too
    (2, 4, 1, 60, 1100, 128, 1, 20.0, "+-"),   # heads of either sign share a unit, and a warp
    (1, 6, 2, 10, 3000, 64, 1, 50.0, "+-"),    # one row tile, keys in pieces
    (1, 4, 2, 130, 1200, 64, 1, 200.0, "-"),   # a cap past the fixed reference
    (1, 4, 2, 3, 1500, 128, 1, 50.0, "-"),     # the form for few rows
    (1, 4, 2, 20, 1500, 36, 1, 50.0, "-"),     # the general form
])
def test_capped_scores_with_a_rising_bias(cuda_dev, B, Hq, Hkv, Sq, Sk, D, causal, cap, signs):
    """Negative slopes: scores grow with the distance, past the cap and any fixed reference."""
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, Sq + D, 2.0)
    sl = torch.full((Hq,), -0.1, device=cuda_dev)
    if signs == "+-":
        sl[::2] = 0.07
    mod = ts.attn_mod(softcap=cap, causal=causal, slopes=sl)
    o = call(q, k, v, mod)
    seen = visible(B, Sq, [Sk] * B, causal, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, [Sk] * B, cap, sl)
    check(o, ref, tol)
    assert torch.equal(call(q, k, v, mod), o)


@pytest.mark.parametrize("cap", [5.0, 15.0, 30.0, 37.0, 50.0, 52.0, 80.0])
@pytest.mark.parametrize("size", [60, -20])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("bias", [0, 1])
def test_values_of_any_size_under_a_cap(cuda_dev, cap, size, sign, bias):
    """The documented range of values, where every score of a row lies near the cap (sign 1) or near its negative:
    neither overflow nor what lies below fp32's normal numbers reaches the result."""
    B, Hq, Hkv, Sq, Sk, D = 1, 4, 2, 200, 700, 64
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 7)
    v = (v.float() * 2.0 ** size).bfloat16()
    q[..., 0], k[..., 0] = 32.0 * sign, 40.0  # raw scores of 160
    sl = slopes_of(Hq, cuda_dev, 0.1) if bias else None
    o = call(q, k, v, ts.attn_mod(softcap=cap, causal=1, slopes=sl))
    seen = visible(B, Sq, [Sk], 1, Sk=Sk, dev=cuda_dev)
    # (the bound with the values at one, scaled back: its smallest term is absolute)
    ref, tol = attend(q, k, v.double() * 2.0 ** -size, seen, [Sk], cap, sl)
    check(o.double() * 2.0 ** -size, ref, tol)
