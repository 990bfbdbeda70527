"""GPU: the 4-bit paged key cache -- the producer (attn_qkv_rope_kv4_stream), its tokens back
(attn_kv4_unpack_stream) and the attention over it (attn_flash_kv4_stream).

The stored codes and scales are compared exactly with a plain encoder run on the bf16 rows that
attn_qkv_rope_paged_stream writes (its own tests hold it to the oracle); the attention with a 64-bit
restatement on the values the cache stands for, within the sum of its roundings (tests/mod_util.py)."""
from __future__ import annotations

import pytest
import torch

import transfer_station_b200 as ts
from tests.mod_util import attend, visible

pytestmark = pytest.mark.gpu
G = 32


def scratch(D, dev):
    return torch.empty(ts.attn_flash_scratch_bytes(D, 128), dtype=torch.uint8, device=dev)


def encode(x):
    """bf16 [..., D] -> codes uint8 [..., D/2], scales uint8 [..., D/32], from the definition in 64 bits."""
    g = x.double().unflatten(-1, (-1, G))
    g = torch.where(torch.isnan(g), torch.zeros_like(g), g)
    s8 = (g.abs().amax(-1) / 7).clamp(max=448.0).float().to(torch.float8_e4m3fn)
    s = s8.double().unsqueeze(-1)
    q = torch.where(s > 0, (g / torch.where(s > 0, s, torch.ones_like(s))).round().clamp(-8, 7), torch.zeros_like(g))
    n = (q.flatten(-2) + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), s8.view(torch.uint8)


def decode(codes, scales):
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    return (n.unflatten(-1, (-1, G)) * scales.view(torch.float8_e4m3fn).double().unsqueeze(-1)).flatten(-2)


def pools(total, Hkv, P, D, dev, byte=0x7F):
    """Pools whose every byte is `byte` (0x7F: NaN scales)."""
    return [torch.full((total, Hkv, P, n), byte, dtype=torch.uint8, device=dev) for n in (D // 2, D // G, D // 2, D // G)]


def table_for(B, per, dev, seed, spare=2):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    total = B * per + spare
    return torch.randperm(total, generator=g)[: B * per].view(B, per).int().to(dev), total


def rot_table(n, rot, dev):
    t = torch.empty(n, rot, dtype=torch.float32, device=dev)
    assert ts.attn_rope_table_stream(t, n, rot, 1e6) == ts.ATTN_OK
    return t


def produce(qkv, pos, rt, maxpos, qw, kw, B, S, Hq, Hkv, D, rot, style, table, P, total, pl, dev, scr=None):
    q = torch.full((B * Hq, S, D), float("nan"), dtype=torch.bfloat16, device=dev)
    scr = scratch(D, dev) if scr is None else scr
    rc = ts.attn_qkv_rope_kv4_stream(qkv, pos, rt, maxpos, qw, kw, 1e-6, B, S, Hq, Hkv, D, rot, style, q, *pl, table, P,
                                     total, table.shape[1], scr)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    return q, scr


PRODUCE = [
    # B, S, Hq, Hkv, D, rot, style, norm, P, past
    (2, 70, 8, 2, 128, 128, ts.ATTN_ROPE_NEOX, 1, 16, 0),
    (3, 33, 4, 4, 64, 64, ts.ATTN_ROPE_NEOX, 1, 8, 5),
    (1, 200, 16, 2, 128, 16, ts.ATTN_ROPE_NEOX, 0, 64, 100),
    (2, 41, 4, 2, 64, 32, ts.ATTN_ROPE_GPTJ, 1, 32, 3),
    (5, 1, 8, 1, 128, 96, ts.ATTN_ROPE_NEOX, 1, 128, 300),
    (1, 129, 2, 1, 128, 128, ts.ATTN_ROPE_GPTJ, 0, 256, 0),
    (2, 19, 6, 3, 64, 0, ts.ATTN_ROPE_NEOX, 1, 16, 0),
    (1, 1, 1, 1, 64, 48, ts.ATTN_ROPE_NEOX, 0, 8, 0),
]


@pytest.mark.parametrize("case", PRODUCE, ids=[str(i) for i in range(len(PRODUCE))])
def test_producer_and_unpack(cuda_dev, case):
    B, S, Hq, Hkv, D, rot, style, norm, P, past = case
    dev = cuda_dev
    g = torch.Generator(device=dev)
    g.manual_seed(S + D)
    qkv = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=g, device=dev)
    qkv[:, ::37] *= 20.0
    qkv = qkv.bfloat16()
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)).bfloat16() if norm else None for _ in range(2))
    pos = (torch.arange(S, dtype=torch.int32, device=dev) + past).repeat(B)
    per = (past + S + P - 1) // P
    table, total = table_for(B, per, dev, 1)
    rt = rot_table(past + S, rot, dev) if rot else None
    pl = pools(total, Hkv, P, D, dev, 0xA5)
    q, scr = produce(qkv, pos, rt, past + S, qw, kw, B, S, Hq, Hkv, D, rot, style, table, P, total, pl, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    # the bf16 producer on the same input
    q16 = torch.empty_like(q)
    k16, v16 = (torch.full((total, Hkv, P, D), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    rc = ts.attn_qkv_rope_paged_stream(qkv, pos, rt, past + S, qw, kw, 1e-6, B, S, Hq, Hkv, D, rot, style, q16, k16, v16,
                                       table, P, total, per, scr)
    assert rc == ts.ATTN_OK
    assert torch.equal(q.view(torch.int16), q16.view(torch.int16))
    b = torch.arange(B, device=dev).repeat_interleave(S)
    pg, row = table.long()[b, pos.long() // P], pos.long() % P
    for (codes, scales), x in (((pl[0], pl[1]), k16[pg, :, row]), ((pl[2], pl[3]), v16[pg, :, row])):
        wc, ws = encode(x)
        gc, gs = codes[pg, :, row], scales[pg, :, row]
        if x is not None and norm and codes is pl[0]:
            # the double-precision root may differ from the bf16 call's in its last bit and move a bf16
            # value by one step (2^-8): a code by at most one, a scale by at most one E4M3 step
            step = (gs.int() - ws.int()).abs()
            assert step.max() <= 1 and (step > 0).float().mean() < 0.01
            same = (step == 0).repeat_interleave(G // 2, -1)
            for sh in (0, 4):
                d = ((gc.int() >> sh) & 15) - ((wc.int() >> sh) & 15)
                assert d[same].abs().max() <= 1 and (d[same] != 0).float().mean() < 0.01
        else:
            assert torch.equal(gs, ws) and torch.equal(gc, wc)
    # nothing else was written
    used = torch.zeros(total, P, dtype=torch.bool, device=dev)
    used[pg, row] = True
    for t in pl:
        assert (t.transpose(1, 2)[~used] == 0xA5).all()
    # and back
    k, v = (torch.full((B * Hkv, S, D), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    rc = ts.attn_kv4_unpack_stream(*pl, table, pos, k, v, B, S, Hkv, D, P, total, per, scr)
    assert rc == ts.ATTN_OK and ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    for got, codes, scales in ((k, pl[0], pl[1]), (v, pl[2], pl[3])):
        want = decode(codes[pg, :, row], scales[pg, :, row]).view(B, S, Hkv, D).transpose(1, 2).reshape(B * Hkv, S, D)
        assert torch.equal(got.double(), want)


def test_norm_of_keys_is_rounded_once(cuda_dev):
    """With the norm, codes equal the encoder's on keys whose root was taken in 64 bits and rounded once."""
    dev, B, S, Hq, Hkv, D, P = cuda_dev, 1, 2000, 1, 2, 128, 64
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    qkv = torch.randn(S, (Hq + 2 * Hkv) * D, generator=g, device=dev).bfloat16()
    kw = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).bfloat16()
    pos = torch.arange(S, dtype=torch.int32, device=dev)
    per = (S + P - 1) // P
    table, total = table_for(B, per, dev, 2)
    pl = pools(total, Hkv, P, D, dev)
    rt = rot_table(S, D, dev)
    produce(qkv, pos, rt, S, None, kw, B, S, Hq, Hkv, D, D, ts.ATTN_ROPE_NEOX, table, P, total, pl, dev)
    x = qkv.view(S, -1, D)[:, Hq:Hq + Hkv].float()
    eps = torch.tensor(1e-6, dtype=torch.float32).double().item()
    x = x * (x.double().square().mean(-1, keepdim=True) + eps).rsqrt().float() * kw.float()
    c, s = rt[:, None, : D // 2], rt[:, None, D // 2:]
    a, b = x[..., : D // 2], x[..., D // 2:]
    wc, ws = encode(torch.cat((a * c - b * s, b * c + a * s), -1).bfloat16())
    pg, row = table[0].long()[pos.long() // P], pos.long() % P
    assert torch.equal(pl[1][pg, :, row], ws) and torch.equal(pl[0][pg, :, row], wc)


def test_encoder_edges(cuda_dev):
    """Zeros, the smallest and largest scales, ties, infinities and NaN."""
    dev, D, P = cuda_dev, 64, 8
    v = torch.zeros(11, D)
    v[1, :] = 2.0 ** -14                      # a / 7 rounds to zero: the group stands for zeros
    v[2, :32] = 7 * 2.0 ** -9                 # the smallest scale
    v[2, 1], v[2, 2], v[2, 3] = 0.5 * 2.0 ** -9, 1.5 * 2.0 ** -9, -2.5 * 2.0 ** -9
    v[3, 0], v[3, 1] = 3e38, 5000.0           # beyond 448 * 7: clamped
    v[4, 0], v[4, 1:9] = 7.0, torch.arange(8) - 3.5   # scale 1: ties to even
    v[5, 0], v[5, 1] = float("inf"), 100.0
    v[6, 0], v[6, 1], v[6, 2] = float("nan"), 7.0, -3.0
    v[7, :] = float("nan")
    v[8, 0], v[8, 1:5] = 21.0, torch.tensor([4.5, -4.5, 7.5, 10.5])  # scale 3: ties off powers of two
    v[9, 0] = 7 * 17 / 16.0                   # a / 7 between two E4M3 values
    v[10, 0], v[10, 1] = -float("inf"), float("nan")
    v = v.bfloat16().to(dev)
    S = v.shape[0]
    qkv = torch.cat((v, v, v), 1).contiguous()
    pos = torch.arange(S, dtype=torch.int32, device=dev)
    table, total = table_for(1, 2, dev, 3)
    pl = pools(total, 1, P, D, dev)
    _, scr = produce(qkv, pos, None, 0, None, None, 1, S, 1, 1, D, 0, ts.ATTN_ROPE_NEOX, table, P, total, pl, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    wc, ws = encode(v)
    pg, row = table[0].long()[pos.long() // P], pos.long() % P
    for codes, scales in ((pl[0], pl[1]), (pl[2], pl[3])):
        assert torch.equal(scales[pg, 0, row], ws)
        assert torch.equal(codes[pg, 0, row], wc)


def test_producer_and_unpack_report_bad_slots(cuda_dev):
    dev, B, S, Hq, Hkv, D, P = cuda_dev, 2, 4, 2, 1, 64, 8
    qkv = torch.ones(B * S, (Hq + 2 * Hkv) * D, device=dev).bfloat16()
    table = torch.tensor([[1, 0], [2, 99]], dtype=torch.int32, device=dev)
    pos = torch.tensor([0, 15, 16, -1, 1, 9, 2, 3], dtype=torch.int32, device=dev)  # past, before, bad page
    pl = pools(3, Hkv, P, D, dev, 0x11)
    q, scr = produce(qkv, pos, None, 0, None, None, B, S, Hq, Hkv, D, 0, ts.ATTN_ROPE_NEOX, table, P, 3, pl, dev)
    rc, code = ts.attn_flash_status(scr)
    assert rc == ts.ATTN_ERR_DEVICE and code == (ts.ATTN_DEV_BAD_PAGE | ts.ATTN_DEV_BAD_POS)
    written = {(1, 0), (0, 7), (2, 1), (2, 2), (2, 3)}
    for page in range(3):
        for r in range(P):
            assert ((pl[0][page, 0, r] != 0x11).all().item()) == ((page, r) in written)
    k, v = (torch.full((B * Hkv, S, D), 5.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    assert ts.attn_kv4_unpack_stream(*pl, table, pos, k, v, B, S, Hkv, D, P, 3, 2, scr) == ts.ATTN_OK
    rc, code = ts.attn_flash_status(scr)
    assert rc == ts.ATTN_ERR_DEVICE and code == (ts.ATTN_DEV_BAD_PAGE | ts.ATTN_DEV_BAD_POS)
    assert (k[0, 2:] == 5).all() and (k[1, 1] == 5).all() and (k[0, :2] != 5).all() and (k[1, 2:] != 5).all()


def cache(B, Hkv, D, lens, P, dev, seed, junk=0x7F):
    """A filled cache: pools (bytes of unwritten slots: NaN scales), table (entries past a sequence's pages hold
    no page), and the values [B][Hkv][Sk][D] it stands for."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    Sk = max(max(lens), 1)
    per = (Sk + P - 1) // P
    table, total = table_for(B, per, dev, seed)
    pl = pools(total, Hkv, P, D, dev, junk)
    vals = []
    for n in range(2):
        x = torch.randn(B, Sk, Hkv, D, generator=g, device=dev)
        x[..., 5] *= 8.0
        c, s = encode(x.bfloat16())
        vals.append(decode(c, s).transpose(1, 2))
        for b, m in enumerate(lens):
            t = torch.arange(m, device=dev)
            pg, row = table[b].long()[t // P], t % P
            pl[2 * n][pg, :, row], pl[2 * n + 1][pg, :, row] = c[b, :m], s[b, :m]
    for b, m in enumerate(lens):
        table[b, (m + P - 1) // P:] = -7
    return pl, table, total, vals[0], vals[1]


def run(q, pl, table, total, lens, P, mod, out, dev, scr=None, o=None, stream=None):
    B, Hq, Sq, D = q.shape
    o = torch.full((B, Hq, Sq, D), float("nan"), dtype=out, device=dev) if o is None else o
    scr = scratch(D, dev) if scr is None else scr
    ln = lens if torch.is_tensor(lens) else torch.tensor(lens, dtype=torch.int32, device=dev)
    rc = ts.attn_flash_kv4_stream(q, *pl, table, ln, o, ts.ATTN_OUT_BF16 if out == torch.bfloat16 else ts.ATTN_OUT_F32, B,
                                  Hq, pl[0].shape[1], Sq, D, mod, P, total, table.shape[1], scr, stream)
    assert rc == ts.ATTN_OK, ts.strerror(rc)
    return o, scr


def check(o, ref, tol, what=""):
    err = (o.double() - ref).abs()
    assert not torch.isnan(o).any(), f"{what}: NaN in the output"
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound (error {err.max().item():.3g})"


ATTEND = [
    # lens, Hq, Hkv, Sq, D, P, causal, cap, bias, out
    ([1], 1, 1, 1, 64, 8, 0, 0.0, 0, torch.float32),
    ([37, 1, 64, 65], 8, 2, 1, 128, 16, 0, 0.0, 0, torch.float32),
    ([1000, 0, 129], 8, 1, 1, 64, 64, 1, 0.0, 0, torch.bfloat16),
    ([3000, 777], 16, 2, 1, 128, 128, 1, 30.0, 0, torch.float32),
    ([700, 4, 1500], 16, 4, 4, 64, 32, 1, 50.0, 0, torch.bfloat16),      # 16 rows of a kv head
    ([513, 200], 10, 2, 1, 128, 256, 1, 0.0, 1, torch.float32),          # 5 rows
    ([300], 12, 1, 5, 128, 8, 1, 10.0, 1, torch.float32),                # 60 rows: four row blocks
    ([2, 3], 4, 4, 6, 64, 16, 1, 0.0, 0, torch.float32),                 # rows before the first key: empty
    ([40000], 8, 1, 1, 128, 64, 1, 0.0, 0, torch.float32),               # one unit over every CTA
    ([90, 20000, 5, 64, 128, 333], 8, 8, 1, 64, 16, 0, 0.0, 1, torch.bfloat16),
    ([256] * 70, 4, 4, 1, 128, 128, 1, 0.0, 0, torch.float32),
]


@pytest.mark.parametrize("case", ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attention(cuda_dev, case):
    lens, Hq, Hkv, Sq, D, P, causal, cap, bias, out = case
    dev, B = cuda_dev, len(lens)
    pl, table, total, k, v = cache(B, Hkv, D, lens, P, dev, sum(lens) % 1000 + P)
    g = torch.Generator(device=dev)
    g.manual_seed(D + Sq)
    q = (torch.randn(B, Hq, Sq, D, generator=g, device=dev) * 1.5).bfloat16()
    sl = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=dev) if bias else None
    o, scr = run(q, pl, table, total, lens, P, ts.attn_mod(softcap=cap, causal=causal, slopes=sl), out, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    seen = visible(B, Sq, lens, causal, Sk=k.shape[2], dev=dev)
    ref, tol = attend(q, k, v, seen, lens, cap, sl, p_half=2.0 ** -10, p_abs=2.0 ** -26, out=out)
    check(o, ref, tol, str(case))
    assert (o.transpose(1, 2)[~seen.any(2)] == 0).all()


@pytest.mark.parametrize("Sq", [1, 3, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_key_ranges(cuda_dev, Sq, D):
    """Windows and ends per row, some empty or outside the sequence; slots that no row sees hold NaN scales."""
    dev, lens, Hq, Hkv, P = cuda_dev, [900, 130, 64], 4, 2, 16
    B = len(lens)
    pl, table, total, k, v = cache(B, Hkv, D, lens, P, dev, Sq)
    begin = torch.tensor([[200 + 3 * i for i in range(Sq)], [-5] * Sq, [64] * Sq], dtype=torch.int32, device=dev)
    end = torch.tensor([[700 - i for i in range(Sq)], [100] * Sq, [2 ** 31 - 1] * Sq], dtype=torch.int32, device=dev)
    if Sq > 1:
        begin[0, 1], end[0, 1] = 2 ** 31 - 1, -2 ** 31
    seen = visible(B, Sq, lens, 1, begin, end, k.shape[2], dev)
    if Sq <= 16:
        for b, n in enumerate(lens):
            t = torch.arange(n, device=dev)
            lo, hi = int(begin[b].clamp(min=0).min()), int(end[b].max())
            gone = (t < lo) | (t >= hi)
            pg, row = table[b].long().clamp(min=0)[t // P][gone], (t % P)[gone]
            pl[1][pg, :, row] = 0x7F
            pl[3][pg, :, row] = 0xFF
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    q = torch.randn(B, Hq, Sq, D, generator=g, device=dev).bfloat16()
    o, scr = run(q, pl, table, total, lens, P, ts.attn_mod(causal=1, key_begin=begin, key_end=end), torch.float32, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    ref, tol = attend(q, k, v, seen, lens, p_half=2.0 ** -10, p_abs=2.0 ** -26)
    check(o, ref, tol)
    assert (o.transpose(1, 2)[~seen.any(2)] == 0).all()


def test_rows_of_any_size(cuda_dev):
    """Query rows from 2^-100 to 2^100 keep 8 significant bits: each row has its own power of two."""
    dev, lens, Hq, Hkv, D, P = cuda_dev, [333], 8, 1, 128, 32
    pl, table, total, k, v = cache(1, Hkv, D, lens, P, dev, 4)
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    q = torch.randn(1, Hq, 1, D, generator=g, device=dev)
    f = torch.tensor([2.0 ** e for e in (-100, -20, -3, 0, 1, -126, 2, 0)], device=dev).view(1, Hq, 1, 1)
    q = (q * f).bfloat16()
    q[0, 7] = 0
    o, _ = run(q, pl, table, total, lens, P, None, torch.float32, dev)
    seen = visible(1, 1, lens, 0, Sk=k.shape[2], dev=dev)
    ref, tol = attend(q, k, v, seen, lens, p_half=2.0 ** -10, p_abs=2.0 ** -26)
    check(o, ref, tol)
    q[0, 2, 0, 7] = float("nan")
    o2, _ = run(q, pl, table, total, lens, P, None, torch.float32, dev)
    assert torch.isnan(o2[0, 2]).all() and torch.equal(o2[0, 3:], o[0, 3:]) and torch.equal(o2[0, :2], o[0, :2])


def test_bad_page_is_reported_and_later_calls_are_clean(cuda_dev):
    dev, lens, Hq, Hkv, D, P = cuda_dev, [600, 300], 8, 2, 128, 64
    pl, table, total, k, v = cache(2, Hkv, D, lens, P, dev, 6)
    q = torch.randn(2, Hq, 1, D, device=dev).bfloat16()
    bad = table.clone()
    bad[0, 3] = total + 3
    scr = scratch(D, dev)
    o, _ = run(q, pl, bad, total, lens, P, None, torch.float32, dev, scr)
    rc, code = ts.attn_flash_status(scr)
    assert rc == ts.ATTN_ERR_DEVICE and code == ts.ATTN_DEV_BAD_PAGE
    seen = visible(2, 1, lens, 0, Sk=k.shape[2], dev=dev)
    ref, tol = attend(q, k, v, seen, lens, p_half=2.0 ** -10, p_abs=2.0 ** -26)
    check(o[1], ref[1], tol[1], "the other sequence")
    o, _ = run(q, pl, table, total, lens, P, None, torch.float32, dev, scr)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    check(o, ref, tol)


def test_repeats_are_bit_identical(cuda_dev):
    dev, lens, Hq, Hkv, D, P = cuda_dev, [5000, 77, 1234], 32, 8, 128, 16
    pl, table, total, k, v = cache(3, Hkv, D, lens, P, dev, 7)
    q = torch.randn(3, Hq, 1, D, device=dev).bfloat16()
    first, scr = run(q, pl, table, total, lens, P, None, torch.bfloat16, dev)
    for _ in range(5):
        o, _ = run(q, pl, table, total, lens, P, None, torch.bfloat16, dev, scr)
        assert torch.equal(o, first)


def test_decode_steps_in_a_graph(cuda_dev):
    """Decode as it is used: append one token a sequence and attend, captured once and replayed while the lengths
    grow; each step equals the calls made one by one, and the values attention over the unpacked cache."""
    dev, B, Hq, Hkv, D, P, steps = cuda_dev, 3, 8, 2, 128, 16, 5
    start = [30, 47, 1]
    lens = torch.tensor(start, dtype=torch.int32, device=dev)
    pl, table, total, _, _ = cache(B, Hkv, D, [n + 16 for n in start], P, dev, 11)
    per = table.shape[1]
    rt = rot_table(per * P, D, dev)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    tokens = torch.randn(steps, B, (Hq + 2 * Hkv) * D, generator=g, device=dev).bfloat16()
    w = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).bfloat16()
    mod = ts.attn_mod(softcap=30.0, causal=1)

    def step(qkv, ln, pool, q, o, scr_a, scr_b):
        rc = ts.attn_qkv_rope_kv4_stream(qkv, ln, rt, per * P, w, w, 1e-6, B, 1, Hq, Hkv, D, D, ts.ATTN_ROPE_NEOX, q, *pool,
                                         table, P, total, per, scr_a)
        assert rc == ts.ATTN_OK
        ln.add_(1)
        rc = ts.attn_flash_kv4_stream(q, *pool, table, ln, o, ts.ATTN_OUT_F32, B, Hq, Hkv, 1, D, mod, P, total, per, scr_b)
        assert rc == ts.ATTN_OK

    new = lambda: (torch.empty(B * Hq, 1, D, dtype=torch.bfloat16, device=dev),  # noqa: E731
                   torch.empty(B, Hq, 1, D, device=dev), scratch(D, dev), scratch(D, dev))
    plain_pool, plain_len, bufs = [t.clone() for t in pl], lens.clone(), new()
    want = []
    for s in range(steps):
        step(tokens[s], plain_len, plain_pool, *bufs)
        want.append(bufs[1].clone())
        assert ts.attn_flash_status(bufs[2]) == (ts.ATTN_OK, 0) and ts.attn_flash_status(bufs[3]) == (ts.ATTN_OK, 0)
    graph_pool, graph_len, gb = [t.clone() for t in pl], lens.clone(), new()
    qkv = tokens[0].clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        step(qkv, graph_len, graph_pool, *gb)
    for s in range(steps):
        qkv.copy_(tokens[s])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gb[1], want[s]), s
        assert ts.attn_flash_status(gb[3]) == (ts.ATTN_OK, 0)
    assert all(torch.equal(a, b) for a, b in zip(graph_pool, plain_pool))
    # the last step against the unpacked cache through the bf16 kernels' 64-bit restatement
    n = [x + steps for x in start]
    Sk = max(n)
    pos = torch.arange(Sk, dtype=torch.int32, device=dev).repeat(B)
    k, v = (torch.empty(B * Hkv, Sk, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    flat = table.clone()
    flat[flat < 0] = 0
    rc = ts.attn_kv4_unpack_stream(*graph_pool, flat, pos, k, v, B, Sk, Hkv, D, P, total, per, gb[2])
    assert rc == ts.ATTN_OK
    q = gb[0].view(B, Hq, 1, D)
    k, v = k.view(B, Hkv, Sk, D), v.view(B, Hkv, Sk, D)
    seen = visible(B, 1, n, 1, Sk=Sk, dev=dev)
    ref, tol = attend(q, torch.nan_to_num(k), torch.nan_to_num(v), seen, n, 30.0, p_half=2.0 ** -10, p_abs=2.0 ** -26)
    check(gb[1], ref, tol)


def test_streams_with_their_own_scratch(cuda_dev):
    dev, lens, Hq, Hkv, D, P = cuda_dev, [3000, 500], 16, 2, 64, 16
    pl, table, total, k, v = cache(2, Hkv, D, lens, P, dev, 12)
    qs = [torch.randn(2, Hq, 1, D, device=dev).bfloat16() for _ in range(3)]
    want = [run(q, pl, table, total, lens, P, None, torch.float32, dev)[0] for q in qs]
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    st = [torch.cuda.Stream() for _ in qs]
    outs, scrs = [torch.empty_like(w) for w in want], [scratch(D, dev) for _ in qs]
    torch.cuda.synchronize()
    for _ in range(4):
        for n, q in enumerate(qs):
            run(q, pl, table, total, ln, P, None, torch.float32, dev, scrs[n], outs[n], st[n])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("Hq,Sq", [(4, 3), (16, 2), (8, 20), (2, 40)])
@pytest.mark.parametrize("D", [64, 128])
def test_unseen_slots_between_ranges(cuda_dev, Hq, Sq, D):
    """Rows that see ranges far apart: the slots between, before and behind them hold NaN scales and any code."""
    dev, lens, Hkv, P = cuda_dev, [1200, 700], 2, 32
    B = len(lens)
    pl, table, total, k, v = cache(B, Hkv, D, lens, P, dev, Sq)
    i = torch.arange(Sq, dtype=torch.int32, device=dev)
    begin = torch.stack([101 + 190 * (i % 5), 333 - 7 * (i % 3)]).contiguous()
    end = begin + torch.stack([13 + i % 9, 2 + 0 * i])
    seen = visible(B, Sq, lens, 0, begin, end, k.shape[2], dev)
    for b, n in enumerate(lens):
        t = torch.arange(n, device=dev)
        gone = ~seen[b, :, :n].any(0)
        pg, row = table[b].long().clamp(min=0)[t // P][gone], (t % P)[gone]
        pl[1][pg, :, row] = 0x7F
        pl[3][pg, :, row] = 0xFF
    g = torch.Generator(device=dev)
    g.manual_seed(8)
    q = torch.randn(B, Hq, Sq, D, generator=g, device=dev).bfloat16()
    o, scr = run(q, pl, table, total, lens, P, ts.attn_mod(key_begin=begin, key_end=end), torch.float32, dev)
    assert ts.attn_flash_status(scr) == (ts.ATTN_OK, 0)
    ref, tol = attend(q, k, v, seen, lens, p_half=2.0 ** -10, p_abs=2.0 ** -26)
    check(o, ref, tol)
