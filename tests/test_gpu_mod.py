"""GPU: attention with modified scores (attn_flash_mod_stream, attn_flash_mod_paged_stream,
attn_mask_ranges_stream) against a 64-bit restatement; every bound is the sum of the kernel's own
roundings (tests/mod_util.py)."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible

pytestmark = pytest.mark.gpu


def scratch(D, dev):
    return torch.empty(ts.attn_flash_scratch_bytes(max(D, 1), 128), dtype=torch.uint8, device=dev)


def inputs(B, Hq, Hkv, Sq, Sk, D, dev, seed, spread=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=g, device=dev)  # noqa: E731
    return ((r(B, Hq, Sq, D) * spread).bfloat16(), r(B, Hkv, Sk, D).bfloat16(), r(B, Hkv, Sk, D).bfloat16())


def slopes_of(Hq, dev, sign=1.0):
    return torch.tensor([sign * 2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=dev)


def call(q, k, v, mod, out=torch.float32, scr=None, stream=None, o=None):
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    if o is None:
        o = torch.full((B, Hq, Sq, D), float("nan"), dtype=out, device=q.device)
    scr = scratch(D, q.device) if scr is None else scr
    rc = ts.attn_flash_mod_stream(q, k, v, o, ts.ATTN_OUT_BF16 if out == torch.bfloat16 else ts.ATTN_OUT_F32, B, Hq,
                                  Hkv, Sq, Sk, D, mod, scr, stream)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    if not torch.cuda.is_current_stream_capturing():
        assert ts.attn_flash_status(scr, stream) == (ts.ATTN_OK, 0)
    return o


def check(o, ref, tol, what=""):
    err = (o.double() - ref).abs()
    assert not torch.isnan(o).any(), f"{what}: NaN in the output"
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound (error {err.max().item():.3g})"


CASES = [
    # B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, spread, out
    (1, 8, 2, 300, 300, 128, 1, 30.0, 0, 4.0, torch.bfloat16),    # capped prompt, units straddle heads
    (1, 4, 4, 512, 512, 64, 1, 50.0, 0, 2.0, torch.float32),      # whole units per head
    (2, 8, 2, 257, 391, 128, 1, 5.0, 0, 8.0, torch.bfloat16),     # arguments of tanh far above 1
    (1, 2, 1, 130, 515, 80, 0, 20.0, 0, 3.0, torch.float32),      # bidirectional, head width padded
    (2, 6, 2, 200, 200, 64, 1, 0.0, 1, 1.0, torch.bfloat16),      # distance bias
    (1, 8, 8, 321, 321, 128, 0, 0.0, 1, 1.0, torch.float32),      # bias on both sides of the query
    (1, 4, 1, 140, 1000, 128, 1, 15.0, 1, 2.0, torch.bfloat16),   # both
    (1, 4, 2, 300, 128, 64, 1, 0.0, 1, 1.0, torch.float32),       # rows before the first key: empty
    (3, 16, 2, 1, 2500, 128, 1, 30.0, 1, 2.0, torch.float32),     # single tokens, split keys
    (1, 8, 1, 1, 20001, 64, 0, 50.0, 0, 2.0, torch.bfloat16),     # long context, many pieces
    (1, 1, 1, 1, 1, 128, 1, 50.0, 1, 1.0, torch.float32),         # one key
    (2, 4, 2, 3, 5, 8, 1, 2.0, 0, 4.0, torch.float32),            # narrow heads
    (1, 4, 2, 37, 61, 36, 1, 30.0, 1, 2.0, torch.bfloat16),       # general path: D % 8 != 0
    (1, 2, 1, 20, 333, 256, 1, 30.0, 0, 2.0, torch.float32),      # general path: wide heads
    (4, 4, 2, 64, 64, 128, 1, 1000.0, 0, 30.0, torch.float32),    # a wide cap, large scores
]


@pytest.mark.parametrize("case", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_cap_and_bias(cuda_dev, case):
    B, Hq, Hkv, Sq, Sk, D, causal, cap, bias, spread, out = case
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 17 + Sq + Sk, spread)
    sl = slopes_of(Hq, cuda_dev) if bias else None
    o = call(q, k, v, ts.attn_mod(softcap=cap, causal=causal, slopes=sl), out)
    seen = visible(B, Sq, [Sk] * B, causal, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, [Sk] * B, cap, sl, out=out)
    check(o, ref, tol, str(case))
    assert (o.view(B, Hq, Sq, D).transpose(1, 2)[~seen.any(2)] == 0).all()


@pytest.mark.parametrize("Sq,Sk,D,cap,bias", [(200, 333, 128, 0.0, 0), (64, 700, 64, 30.0, 0), (5, 900, 128, 0.0, 1),
                                              (1, 3000, 128, 50.0, 1), (700, 700, 128, 0.0, 0), (33, 50, 20, 9.0, 1),
                                              (300, 2000, 64, 0.0, 1)])
@pytest.mark.parametrize("causal", [0, 1])
def test_key_ranges(cuda_dev, Sq, Sk, D, cap, bias, causal):
    """Random ranges, some empty, some reaching outside [0, Sk); NaN and infinities in every key and value
    that no query of the sequence sees."""
    B, Hq, Hkv = 2, 8, 2
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 5 + Sq, 2.0)
    g = torch.Generator(device=cuda_dev)
    g.manual_seed(Sq * 7 + Sk)
    a = torch.randint(Sk // 5, max(Sk // 5 + 1, Sk // 2), (B, Sq), generator=g, device=cuda_dev, dtype=torch.int32)
    e = a + torch.randint(-3, Sk // 3 + 2, (B, Sq), generator=g, device=cuda_dev, dtype=torch.int32)
    if Sq > 3:
        a[0, 1], e[0, 1] = -2 ** 31, Sk // 4
        a[0, 2], e[0, 2] = 2 ** 31 - 1, -2 ** 31
    seen = visible(B, Sq, [Sk] * B, causal, a, e, Sk, cuda_dev)
    unused = ~seen.any(1)
    for t, bad in ((k, float("nan")), (v, float("inf"))):
        t.transpose(1, 2)[unused] = bad
    v.transpose(1, 2)[unused & (torch.arange(Sk, device=cuda_dev) % 3 == 0)] = float("nan")
    sl = slopes_of(Hq, cuda_dev, -0.01 if causal else 1.0) if bias else None
    o = call(q, k, v, ts.attn_mod(softcap=cap, causal=causal, slopes=sl, key_begin=a, key_end=e), torch.bfloat16)
    ref, tol = attend(q, k, v, seen, [Sk] * B, cap, sl, out=torch.bfloat16)
    check(o, ref, tol)
    assert (o.transpose(1, 2)[~seen.any(2)] == 0).all()


@pytest.mark.parametrize("which", ["begin", "end"])
def test_one_sided_ranges(cuda_dev, which):
    B, Hq, Hkv, Sq, Sk, D = 3, 4, 2, 1, 700, 128
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 3)
    r = torch.tensor([[0], [129], [700]], dtype=torch.int32, device=cuda_dev)
    kw = {"key_" + which: r}
    o = call(q, k, v, ts.attn_mod(**kw))
    seen = visible(B, Sq, [Sk] * B, 0, Sk=Sk, dev=cuda_dev, **{which: r})
    ref, tol = attend(q, k, v, seen, [Sk] * B)
    check(o, ref, tol)


@pytest.mark.parametrize("causal,window,with_prefix", [(1, 0, True), (1, 0, False), (0, 0, False), (1, 9, False),
                                                       (0, 5, False)])
@pytest.mark.parametrize("cu", [[0, 5, 5, 140, 300], [3, 4, 260], [0, 0]])
def test_mask_ranges(cuda_dev, cu, causal, window, with_prefix):
    S, n = 303, len(cu) - 1
    pre = [2 * d + 1 if d % 2 == 0 else 1000 for d in range(n)]
    begin, end = (torch.full((S + 2,), -7, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    cut = torch.tensor(cu, dtype=torch.int32, device=cuda_dev)
    pt = torch.tensor(pre, dtype=torch.int32, device=cuda_dev) if with_prefix else None
    assert ts.attn_mask_ranges_stream(cut, pt, n, S, causal, window, begin, end) == ts.ATTN_OK
    got_b, got_e = begin.tolist(), end.tolist()
    assert got_b[S:] == [-7, -7] and got_e[S:] == [-7, -7]
    for i in range(S):
        want = set()
        for d in range(n):
            s, e = cu[d], cu[d + 1]
            if s <= i < e:
                for j in range(s, e):
                    ok = not causal or j <= i or (with_prefix and j < s + pre[d])
                    if window and j <= i - window:
                        ok = False
                    if ok:
                        want.add(j)
        assert set(range(got_b[i], got_e[i])) == want, i


@pytest.mark.parametrize("with_prefix", [False, True])
def test_documents_end_to_end(cuda_dev, with_prefix):
    """Ranges built and used on one stream: each document's rows equal attention over the document alone."""
    Hq, Hkv, S, D = 8, 2, 900, 128
    cu = [0, 130, 131, 512, 880]
    pre = [10, 0, 200, 3]
    q, k, v = inputs(1, Hq, Hkv, S, S, D, cuda_dev, 8)
    v[:, :, 880:] = float("nan")
    cut = torch.tensor(cu, dtype=torch.int32, device=cuda_dev)
    pt = torch.tensor(pre, dtype=torch.int32, device=cuda_dev) if with_prefix else None
    begin, end = (torch.empty(S, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    assert ts.attn_mask_ranges_stream(cut, pt, 4, S, 1, 0, begin, end) == ts.ATTN_OK
    o = call(q, k, v, ts.attn_mod(key_begin=begin, key_end=end))
    for d, (a, b) in enumerate(zip(cu, cu[1:])):
        n = b - a
        seen = torch.ones(n, n, dtype=torch.bool, device=cuda_dev).tril()
        if with_prefix:
            seen[:, : pre[d]] = True
        ref, tol = attend(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], seen[None], [n])
        check(o[:, :, a:b], ref, tol, f"document {d}")
    assert (o[:, :, 880:] == 0).all()


def test_no_modifier_is_the_plain_call(cuda_dev):
    """Without modifiers the plain kernels run: the same bits as attn_flash_stream_out."""
    for (B, Hq, Hkv, Sq, Sk, D, causal) in [(2, 8, 2, 200, 300, 128, 1), (1, 16, 2, 1, 4000, 64, 0)]:
        q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 2)
        scr = scratch(D, cuda_dev)
        want = torch.empty(B, Hq, Sq, D, dtype=torch.bfloat16, device=cuda_dev)
        rc = ts.attn_flash_stream_out(q, k, v, want, ts.ATTN_OUT_BF16, B * Hq, B * Hkv, Sq, Sk, D, causal, 128, scr)
        assert rc == ts.ATTN_OK
        assert torch.equal(call(q, k, v, ts.attn_mod(causal=causal), torch.bfloat16), want)
        if not causal:
            assert torch.equal(call(q, k, v, None, torch.bfloat16), want)


def test_far_keys_keep_their_bits(cuda_dev):
    """A row that sees only keys far from its position: the bias of the nearest cancels in the softmax."""
    B, Hq, Hkv, Sq, Sk, D = 1, 4, 2, 2, 60000, 64
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 4)
    end = torch.tensor([[500, 701]], dtype=torch.int32, device=cuda_dev)
    sl = torch.tensor([0.5, 0.3, 1e-3, 2.0], device=cuda_dev)
    o = call(q, k, v, ts.attn_mod(slopes=sl, key_end=end))
    seen = visible(B, Sq, [Sk], 0, end=end, Sk=Sk, dev=cuda_dev)
    ref, tol = attend(q, k, v, seen, [Sk], 0.0, sl)
    check(o, ref, tol)


def test_nan_and_inf_scores_stay_in_their_row(cuda_dev):
    B, Hq, Hkv, Sq, Sk, D = 1, 2, 1, 150, 150, 64
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 6)
    clean = call(q, k, v, ts.attn_mod(softcap=30.0, causal=1))
    q[0, 0, 40] = float("nan")
    o = call(q, k, v, ts.attn_mod(softcap=30.0, causal=1))
    assert torch.isnan(o[0, 0, 40]).all()
    keep = torch.ones(Hq, Sq, dtype=torch.bool, device=cuda_dev)
    keep[0, 40] = False
    assert torch.equal(o[0][keep], clean[0][keep])


def paged(k, v, lens, P, dev, seed, spare=2, fill=float("nan")):
    B, Hkv, _, D = k.shape
    per = max(1, max((n + P - 1) // P for n in lens))
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    total = B * per + spare
    table = torch.randperm(total, generator=g)[: B * per].view(B, per).int()
    kp, vp = (torch.full((total, Hkv, P, D), fill, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for b, n in enumerate(lens):
        for j in range(0, n, P):
            m = min(P, n - j)
            kp[table[b, j // P], :, :m] = k[b, :, j:j + m]
            vp[table[b, j // P], :, :m] = v[b, :, j:j + m]
        table[b, (n + P - 1) // P:] = -5  # never read
    return kp, vp, table.to(dev), total, per


@pytest.mark.parametrize("lens,Hq,Hkv,Sq,D,P,causal,cap,bias,ranges", [
    ([1000, 1, 777], 16, 4, 1, 128, 16, 1, 30.0, 0, 0),
    ([130, 0, 2049], 8, 2, 1, 64, 64, 0, 0.0, 1, 0),
    ([700, 4, 1500], 16, 2, 4, 128, 32, 1, 20.0, 1, 0),
    ([300, 513], 8, 1, 2, 128, 256, 1, 0.0, 0, 1),
    ([400, 250], 4, 2, 200, 64, 8, 1, 0.0, 0, 1),
    ([640, 1111], 8, 2, 130, 128, 128, 1, 50.0, 0, 0),
])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_paged(cuda_dev, lens, Hq, Hkv, Sq, D, P, causal, cap, bias, ranges, out):
    """Rows of a page past the sequence's end hold NaN; table entries past it hold no page."""
    B, Sk = len(lens), max(lens)
    q, k, v = inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, sum(lens), 2.0)
    kp, vp, table, total, per = paged(k, v, lens, P, cuda_dev, 3)
    sl = slopes_of(Hq, cuda_dev) if bias else None
    begin = end = None
    if ranges:
        i = torch.arange(Sq, dtype=torch.int32, device=cuda_dev)
        n = torch.tensor(lens, dtype=torch.int32, device=cuda_dev).view(B, 1)
        begin = (n - Sq + i - 99).contiguous()
        end = (n - Sq + i + 1 - (i % 5)).contiguous()
    mod = ts.attn_mod(softcap=cap, causal=causal, slopes=sl, key_begin=begin, key_end=end)
    o = torch.full((B, Hq, Sq, D), float("nan"), dtype=out, device=cuda_dev)
    scr = scratch(D, cuda_dev)
    rc = ts.attn_flash_mod_paged_stream(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), o,
                                        ts.ATTN_OUT_BF16 if out == torch.bfloat16 else ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, D,
                                        mod, P, total, per, scr)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    seen = visible(B, Sq, lens, causal, begin, end, Sk, cuda_dev)
    ref, tol = attend(q, k, v, seen, lens, cap, sl, out=out)
    check(o, ref, tol)


def test_graphs_and_streams(cuda_dev):
    """A captured call replays with new inputs; two streams with a scratch block each give the bits of one."""
    B, Hq, Hkv, Sq, Sk, D = 2, 8, 2, 160, 160, 128
    mod = ts.attn_mod(softcap=30.0, causal=1, key_end=torch.full((B, Sq), 150, dtype=torch.int32, device=cuda_dev))
    sets = [inputs(B, Hq, Hkv, Sq, Sk, D, cuda_dev, 60 + n) for n in range(3)]
    want = [call(*s, mod) for s in sets]
    q, k, v = (t.clone() for t in sets[0])
    o = torch.empty_like(want[0])
    scr = scratch(D, cuda_dev)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        call(q, k, v, mod, scr=scr, o=o)
    for n, st in enumerate(sets):
        for dst, src in zip((q, k, v), st):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[n]) and ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs, scrs = [torch.empty_like(want[0]) for _ in sets], [scratch(D, cuda_dev) for _ in sets]
    torch.cuda.synchronize()
    for n, st in enumerate(sets):
        rc = ts.attn_flash_mod_stream(*st, outs[n], ts.ATTN_OUT_F32, B, Hq, Hkv, Sq, Sk, D, mod, scrs[n], streams[n])
        assert rc == ts.ATTN_OK
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
