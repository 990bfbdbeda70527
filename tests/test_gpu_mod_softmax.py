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
