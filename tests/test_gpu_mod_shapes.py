"""GPU: modified scores where the kernel's form or order of work depends on the shape: up to 16 query rows of
a kv head (keys as the matrix rows), and more units than the GPU runs at once (sorted by length)."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible
from tests.test_gpu_mod import call, check, inputs, paged, scratch, slopes_of

pytestmark = pytest.mark.gpu


def ranges(B, Sq, Sk, dev, seed):
    """Key ranges of every kind: anywhere, of any length, some empty, some past the ends."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    a = torch.randint(-5, Sk + 3, (B, Sq), generator=g, device=dev, dtype=torch.int32)
    e = a + torch.randint(-9, max(2, Sk // 2) + 9, (B, Sq), generator=g, device=dev, dtype=torch.int32)
    return a, e


def spoil(k, v, seen):
    """NaN and infinities where no row sees a key."""
    unused = ~seen.any(1)
    k.transpose(1, 2)[unused] = float("nan")
    v.transpose(1, 2)[unused] = float("inf")
    v.transpose(1, 2)[unused & (torch.arange(k.shape[2], device=k.device) % 2 == 0)] = float("nan")


def run(B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, ranged, out, dev, seed):
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, dev, seed, 2.0)
    a, e = ranges(B, Sq, Sk, dev, seed) if ranged else (None, None)
    seen = visible(B, Sq, [Sk] * B, causal, a, e, Sk, dev)
    spoil(k, v, seen)
    sl = slopes_of(Hq, dev) if bias else None
    mod = ts.attn_mod(softcap=cap, causal=causal, slopes=sl, key_begin=a, key_end=e)
    o = call(q, k, v, mod, out)
    ref, tol = attend(q, k, v, seen, [Sk] * B, cap, sl, out=out)
    check(o, ref, tol, str((B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, ranged)))
    assert (o.view(B, Hq, Sq, D).transpose(1, 2)[~seen.any(2)] == 0).all()
    assert torch.equal(o, call(q, k, v, mod, out)), "two runs differ"


@pytest.mark.parametrize("Hq,Hkv,Sq", [(1, 1, 1), (3, 1, 1), (8, 1, 1), (9, 1, 1), (16, 1, 1), (17, 1, 1), (4, 2, 5),
                                       (2, 2, 16), (2, 2, 17), (6, 2, 3)])
@pytest.mark.parametrize("Sk,D", [(1, 64), (63, 128), (64, 8), (65, 72), (200, 40), (4097, 128), (1000, 64)])
def test_rows(cuda_dev, Hq, Hkv, Sq, Sk, D):
    n = Hq * 7 + Sq + Sk
    cap, bias = ((30.0, 0), (0.0, 1), (8.0, 1), (0.0, 0))[n % 4]
    run(2, Hq, Hkv, Sq, Sk, D, n % 3 == 0, cap, bias, cap == 0.0 and not bias or n % 5 < 3,
        torch.bfloat16 if n % 2 else torch.float32, cuda_dev, n)


def test_many_ragged_sequences(cuda_dev):
    """Lengths from none to all of a padded batch's keys; what lies past a length is no number."""
    B, Hq, Hkv, Sk, D = 70, 32, 8, 500, 64
    q, k, v = inputs(B, Hq, Hkv, 1, Sk, D, cuda_dev, 9)
    n = (torch.arange(B, device=cuda_dev, dtype=torch.int32) * 37 % (Sk + 40)).view(B, 1)
    seen = visible(B, 1, [Sk] * B, 0, None, n, Sk, cuda_dev)
    spoil(k, v, seen)
    o = call(q, k, v, ts.attn_mod(softcap=50.0, key_end=n), torch.bfloat16)
    ref, tol = attend(q, k, v, seen, [Sk] * B, 50.0, None, out=torch.bfloat16)
    check(o, ref, tol)
    assert (o.view(B, Hq, D)[n.view(-1) == 0] == 0).all()


@pytest.mark.parametrize("P", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("D", [40, 128])
def test_paged_rows(cuda_dev, P, D):
    lens, Hq, Hkv, Sq = [0, 1, 513, 64, 900, 5], 8, 4, 3
    B, Sk = len(lens), max(lens)
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, P + D, 2.0)
    kp, vp, table, total, per = paged(k, v, lens, P, cuda_dev, 3)
    sl = slopes_of(Hq, cuda_dev)
    o = torch.full((B, Hq, Sq, D), float("nan"), device=cuda_dev)
    scr = scratch(D, cuda_dev)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)

    def go():
        rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, n, o, ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, D,
                                            ts.attn_mod(softcap=20.0, causal=1, slopes=sl), P, total, per, scr)
        assert rc == ts.ATTN_OK, ts.strerror(rc)
        return ts.attn_flash_status(scr)

    assert go() == (ts.ATTN_OK, 0)
    seen = visible(B, Sq, lens, 1, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, lens, 20.0, sl)
    check(o, ref, tol)
    good = table[2, 0].item()
    for bad in (total, -1):  # reported; the other sequences keep their bits, and the next call is clean
        table[2, 0] = bad
        before = o.clone()
        rc, code = go()
        assert rc != ts.ATTN_OK and code != 0
        keep = [b for b in range(B) if b != 2]
        assert torch.equal(o[keep], before[keep])
        table[2, 0] = good
        assert go() == (ts.ATTN_OK, 0) and torch.equal(o, before)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,causal,cap,bias,ranged", [
    (2, 16, 16, 1300, 1300, 64, 0, 0.0, 0, 1),    # random ranges: gaps, holes between heads, empty units
    (2, 16, 4, 1300, 1300, 128, 1, 0.0, 1, 0),    # causal, units straddle heads
    (1, 24, 2, 1601, 1777, 64, 1, 30.0, 0, 1),
    (3, 16, 8, 900, 1000, 128, 1, 30.0, 1, 1),
    (5, 20, 20, 300, 640, 128, 0, 0.0, 1, 1),
    (1100, 1, 1, 20, 90, 64, 0, 0.0, 0, 1),       # more sequences than are ranked one against all
])
def test_sorted_units(cuda_dev, B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, ranged):
    run(B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, ranged, torch.bfloat16, cuda_dev, Sq)


def test_sorted_windows_and_documents(cuda_dev):
    """Contiguous visibility (windows, documents with prefixes) over more units than SMs, and a captured run."""
    Hq, Hkv, S, D = 32, 8, 1531, 128
    q, k, v = inputs(1, Hq, Hkv, S, S, D, cuda_dev, 4, 2.0)
    cu = torch.tensor([3, 4, 500, 500, 1101, 1490], dtype=torch.int32, device=cuda_dev)
    prefix = torch.tensor([1, 200, 0, 90, 389], dtype=torch.int32, device=cuda_dev)
    a, e = (torch.empty(1, S, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    scr = scratch(D, cuda_dev)
    for pre, window in ((prefix, 0), (None, 130)):
        o = torch.empty(1, Hq, S, D, dtype=torch.bfloat16, device=cuda_dev)

        def go():
            assert ts.attn_mask_ranges_stream(cu, pre, 5, S, 1, window, a, e) == ts.ATTN_OK
            call(q, k, v, ts.attn_mod(key_begin=a, key_end=e), torch.bfloat16, scr, o=o)

        go()
        seen = visible(1, S, [S], 0, a, e, S, cuda_dev)
        ref, tol = attend(q, k, v, seen, [S], out=torch.bfloat16)
        check(o, ref, tol)
        want = o.clone()
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=s):
            go()
        for _ in range(3):
            o.zero_(), a.zero_(), e.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


def test_sorted_paged_batch(cuda_dev):
    """A ragged batch of prompts over a paged cache, one sequence without keys, one shorter than its queries."""
    lens, Hq, Hkv, Sq, D, P = [777, 0, 130, 51, 1200, 64, 300, 901] * 3, 16, 8, 120, 128, 32
    B, Sk = len(lens), max(lens)
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 6, 2.0)
    kp, vp, table, total, per = paged(k, v, lens, P, cuda_dev, 3)
    o = torch.full((B, Hq, Sq, D), float("nan"), device=cuda_dev)
    scr = scratch(D, cuda_dev)
    sl = slopes_of(Hq, cuda_dev)
    rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), o,
                                        ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, D, ts.attn_mod(causal=1, slopes=sl), P, total, per,
                                        scr)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    seen = visible(B, Sq, lens, 1, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, lens, 0.0, sl)
    check(o, ref, tol)


def test_what_a_fresh_scratch_block_holds(cuda_dev):
    """Small numbers in a scratch block's first words are no report of a call, whichever call it is."""
    B, Hq, Hkv, Sk, D = 1, 4, 1, 40, 64
    q, k, v = inputs(B, Hq, Hkv, 1, Sk, D, cuda_dev, 2)
    mod = ts.attn_mod(softcap=30.0)
    scr = scratch(D, cuda_dev)
    words = scr[:256].view(torch.int32)
    want = call(q, k, v, mod, scr=scr)
    for gen in range(1, 400):  # (calls of one process are numbered: words that run ahead of them by any amount)
        words.copy_(torch.arange(64, dtype=torch.int32, device=cuda_dev) * 0 + 4)
        words[3] = gen * 2
        assert torch.equal(call(q, k, v, mod, scr=scr), want)
