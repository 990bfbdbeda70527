"""The operators of a decoder whose attention is modified and whose key cache is held in 4 bits, as a
user's program calls them:

  mod     attention whose scores are capped by a tanh, get a bias by distance, or see per-row key
          ranges (documents packed into one sequence with visible prefixes, padded batches):
          attn_flash_mod_stream, attn_mask_ranges_stream
  append  split, norm and rotate a fused QKV projection and append its keys and values to a 4-bit
          paged cache, then read the appended tokens back: attn_qkv_rope_kv4_stream,
          attn_kv4_unpack_stream
  unpack  tokens of a 4-bit paged cache as contiguous bf16 keys and values: attn_kv4_unpack_stream
  kv4     attention over the 4-bit paged cache: attn_flash_kv4_stream

The 4-bit cache: per token and kv head, groups of 32 consecutive elements share one E4M3 scale s; an
element is stored as the nibble q + 8, q in [-8, 7], and stands for q * s. s is the group's largest
magnitude over 7, rounded to E4M3; q is the element over s, rounded to the nearest (ties to even).

`own` False: plain torch in 32 bits (64 where a rounding border has to be met exactly). `own` True: the
framework's calls.
"""
import math
import random

import torch

own = False

GROUP = 32
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a prompt of a model that caps its scores (the framework's prefill shape, causal)
        dict(name="cap_prefill_s4096", op="mod", B=1, Hq=32, Hkv=8, Sq=4096, Sk=4096, D=128, causal=True, cap=30.0,
             alibi=False, mask="none"),
        # a batch of prompts of a model that biases by distance; one kv head per query head, small heads, odd length
        dict(name="alibi_prefill_s2041_d64", op="mod", B=2, Hq=16, Hkv=16, Sq=2041, Sk=2041, D=64, causal=True, cap=0.0,
             alibi=True, mask="none"),
        # documents packed into one row with visible prefixes and padding behind the last document
        dict(name="documents_s6007", op="mod", B=1, Hq=32, Hkv=8, Sq=6007, Sk=6007, D=128, causal=True, cap=0.0,
             alibi=False, mask="docs", docs=9),
        # single tokens of a padded batch, scores capped
        dict(name="cap_decode_b16_s8192", op="mod", B=16, Hq=32, Hkv=8, Sq=1, Sk=8192, D=128, causal=False, cap=50.0,
             alibi=False, mask="lens"),
        # the smallest call: one token early in a conversation
        dict(name="alibi_decode_b1_s129", op="mod", B=1, Hq=8, Hkv=2, Sq=1, Sk=129, D=64, causal=False, cap=0.0,
             alibi=True, mask="none"),
        # serving a full batch from the 4-bit cache (the framework's batched decode shape)
        dict(name="kv4_decode_b64_s8192", op="kv4", B=64, Hq=32, Hkv=8, Sq=1, L=8192, D=128, page=64, ragged=False,
             cap=0.0, alibi=False),
        # few long conversations (the framework's long-context decode shape)
        dict(name="kv4_decode_b4_s131072", op="kv4", B=4, Hq=64, Hkv=8, Sq=1, L=131072, D=128, page=128, ragged=False,
             cap=0.0, alibi=False),
        # checking four drafted tokens of a ragged batch, scores capped, small heads
        dict(name="kv4_verify4_b24_d64", op="kv4", B=24, Hq=16, Hkv=4, Sq=4, L=3001, D=64, page=16, ragged=True,
             cap=50.0, alibi=False),
        # the smallest call: one short conversation
        dict(name="kv4_decode_b1_s37", op="kv4", B=1, Hq=8, Hkv=2, Sq=1, L=37, D=128, page=16, ragged=False,
             cap=0.0, alibi=False),
        # a long prompt into the cache, with q/k norm and rotate-half pairs
        dict(name="append_prompt_s16384", op="append", B=1, S=16384, Hq=32, Hkv=8, D=128, rot=128, neox=True,
             norm=True, page=64, past=0),
        # one new token for each sequence of a batch; interleaved pairs on half of each head, no norm
        dict(name="append_decode_b61_d64", op="append", B=61, S=1, Hq=16, Hkv=4, D=64, rot=32, neox=False, norm=False,
             page=16, past=700),
        # the cached part of four conversations read back for the next chunk of their prompts
        dict(name="unpack_b4_s8192", op="unpack", B=4, S=8192, Hkv=8, D=128, page=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["mod", "mod", "kv4", "kv4", "append", "unpack"])
    D = rng.choice([64, 128])
    if op == "mod":
        D = rng.choice([64, 80, 128])
        Hkv = rng.choice([1, 2, 8])
        Hq = Hkv * rng.choice([1, 4, 7] if Hkv > 1 else [1, 4, 16])
        kind = rng.choice(["prompt", "docs", "decode"])
        cap = rng.choice([0.0, 20.0, 50.0])
        alibi = cap == 0.0 and kind != "docs" or rng.random() < 0.3
        if kind == "decode":
            B = _log(rng, 1, 32)
            Sk = _log(rng, 1, min(32768, 16 * 8192 // B))
            return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Sq=1, Sk=Sk, D=D, causal=False, cap=cap, alibi=alibi, mask="lens")
        B = 1 if kind == "docs" else rng.choice([1, 2, 3])
        S = _log(rng, 5, 4001 if B == 1 else 1501)
        if kind == "docs":
            return dict(op=op, B=1, Hq=Hq, Hkv=Hkv, Sq=S, Sk=S, D=D, causal=rng.random() < 0.8, cap=cap, alibi=alibi,
                        mask="docs", docs=rng.randint(1, 12))
        Sk = S + rng.choice([0, 0, 1, 77, 500])
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Sq=S, Sk=Sk, D=D, causal=rng.random() < 0.8, cap=cap, alibi=alibi,
                    mask="none")
    page = rng.choice([8, 16, 32, 64, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "kv4":
        B = _log(rng, 1, 64)
        L = _log(rng, 1, min(131072, 64 * 8192 // B))
        cap = rng.choice([0.0, 0.0, 20.0, 50.0])
        return dict(op=op, B=B, Hq=Hkv * rng.choice([1, 4, 5, 8, 12]), Hkv=Hkv, Sq=rng.choice([1, 1, 1, 2, 5]), L=L, D=D,
                    page=page, ragged=rng.random() < 0.5, cap=cap, alibi=rng.random() < 0.3)
    if op == "append":
        B = _log(rng, 1, 64)
        S = _log(rng, 1, max(1, 8192 // B))
        return dict(op=op, B=B, S=S, Hq=Hkv * rng.choice([1, 4, 6]), Hkv=Hkv, D=D, rot=rng.choice([16, D // 2, D]),
                    neox=rng.random() < 0.6, norm=rng.random() < 0.6, page=page, past=rng.choice([0, 5, 333]))
    B = _log(rng, 1, 16)
    return dict(op=op, B=B, S=_log(rng, 1, 4 * 8192 // B), Hkv=Hkv, D=D, page=page)


def _lens(case):
    """Each sequence's length: a case's own, not the seed's, so that the work of a case is known."""
    n, B = case.get("Sk", case.get("L")), case["B"]
    if not (case.get("mask") == "lens" or case.get("ragged")):
        return [n] * B
    r = random.Random(n * 131 + B)
    return [n] + [max(1, int(n * r.uniform(0.2, 1.0))) for _ in range(B - 1)]


def _documents(case):
    """Document borders (rising, the last one short of the row's end where there is room for padding) and prefix lengths."""
    S, n = case["Sq"], case["docs"]
    r = random.Random(S * 17 + n)
    end = S - S // 50
    cuts = sorted(r.randint(0, end) for _ in range(n - 1))
    cu = [0] + cuts + [end]
    prefix = [int((b - a) * r.choice([0.0, 0.1, 0.3])) for a, b in zip(cu, cu[1:])]
    return cu, prefix


def work(case):
    B, D, Hkv = case["B"], case["D"], case["Hkv"]
    if case["op"] == "mod":
        Hq, Sq, Sk = case["Hq"], case["Sq"], case["Sk"]
        if case["mask"] == "docs":
            cu, pre = _documents(case)
            pairs = sum((n * (n + 1) // 2 + p * (p - 1) // 2) if case["causal"] else n * n
                        for n, p in ((b - a, p) for a, b, p in zip(cu, cu[1:], pre)))
        elif case["mask"] == "lens":
            pairs = sum(_lens(case)) * Sq
        else:
            pairs = B * (Sq * (Sk - Sq) + Sq * (Sq + 1) // 2 if case["causal"] else Sq * Sk)
        keys = sum(_lens(case)) if case["mask"] == "lens" else B * Sk
        return {"bytes": 4 * B * Hq * Sq * D + 4 * keys * Hkv * D, "flops": 4 * Hq * pairs * D}
    row = D // 2 + D // GROUP  # bytes of one key (or value) of one head
    if case["op"] == "kv4":
        Hq, Sq, lens = case["Hq"], case["Sq"], _lens(case)
        pairs = sum(sum(min(n, max(0, n - Sq + i + 1)) for i in range(Sq)) for n in lens)
        return {"bytes": 4 * B * Hq * Sq * D + 2 * sum(lens) * Hkv * row, "flops": 4 * Hq * pairs * D}
    S = case["S"]
    if case["op"] == "append":
        Hq = case["Hq"]
        # read the projection, write q and the 4-bit rows, then read those and write bf16 keys and values
        return {"bytes": B * S * (2 * (Hq + 2 * Hkv) * D + 2 * Hq * D + 4 * Hkv * row + 4 * Hkv * D),
                "flops": 10 * B * S * (Hq + 2 * Hkv) * D}
    return {"bytes": B * S * Hkv * (2 * row + 4 * D), "flops": 2 * B * S * Hkv * D}


# ------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _encode(x):
    """bf16 [..., D] -> nibble pairs uint8 [..., D/2] and E4M3 scales as uint8 [..., D/32]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    s = (g.abs().amax(-1) / torch.full((), 7.0, device=x.device)).clamp(max=448.0).to(torch.float8_e4m3fn)
    f = s.float().unsqueeze(-1)
    q = torch.where(f > 0, torch.round(g / f.clamp(min=2.0 ** -9)), torch.zeros_like(g)).clamp(-8, 7)
    n = (q + 8).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), s.view(torch.uint8)


def _decode(codes, scales):
    """The values, in 32 bits, that nibble pairs and scales stand for."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (n.unflatten(-1, (-1, GROUP)) * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _slopes(Hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], dtype=torch.float32, device=DEV)


def _cache(case, tokens, g):
    """A shuffled block table for `tokens` tokens a sequence, and the pools, filled with what other tokens left there."""
    B, Hkv, D, P = case["B"], case["Hkv"], case["D"], case["page"]
    per = (tokens + P - 1) // P
    total = B * per + 3
    table = torch.randperm(total, generator=g, device=DEV)[: B * per].to(torch.int32).view(B, per).contiguous()
    pools = []
    for _ in range(2):
        pools.append(torch.randint(0, 256, (total, Hkv, P, D // 2), generator=g, device=DEV, dtype=torch.uint8))
        # scales between 2^-2 and 2, as a cache of normed keys has them
        pools.append(torch.randint(0x28, 0x40, (total, Hkv, P, D // GROUP), generator=g, device=DEV, dtype=torch.uint8))
    return table, total, per, pools


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *n: torch.randn(*n, generator=g, device=DEV, dtype=torch.float32)  # noqa: E731
    B, D, Hkv = case["B"], case["D"], case["Hkv"]
    st = {"case": case, "scratch": torch.empty(40 << 20, dtype=torch.uint8, device=DEV)}
    if case["op"] == "mod":
        Hq, Sq, Sk = case["Hq"], case["Sq"], case["Sk"]
        st["q"] = (rand(B * Hq, Sq, D) * 2.0).bfloat16()  # scores a few units wide, so that a cap bends them
        st["k"], st["v"] = rand(B * Hkv, Sk, D).bfloat16(), rand(B * Hkv, Sk, D).bfloat16()
        st["o"] = torch.empty(B * Hq, Sq, D, dtype=torch.bfloat16, device=DEV)
        st["slopes"] = _slopes(Hq) if case["alibi"] else None
        if case["mask"] == "docs":
            cu, pre = _documents(case)
            st["cu"], st["prefix"] = _ints(cu), _ints(pre)
            st["begin"], st["end"] = torch.empty(Sq, dtype=torch.int32, device=DEV), torch.empty(Sq, dtype=torch.int32, device=DEV)
        if case["mask"] == "lens":
            st["begin"], st["end"] = None, _ints(_lens(case)).view(B, 1).expand(B, Sq).contiguous()
        return st
    P = case["page"]
    if case["op"] == "kv4":
        Hq, Sq, L = case["Hq"], case["Sq"], case["L"]
        st["table"], st["pages"], st["per"], st["pools"] = _cache(case, L, g)
        st["lens"] = _ints(_lens(case))
        st["q"] = rand(B * Hq, Sq, D).bfloat16()
        st["o"] = torch.empty(B * Hq, Sq, D, dtype=torch.bfloat16, device=DEV)
        st["slopes"] = _slopes(Hq) if case["alibi"] else None
        return st
    S = case["S"]
    if case["op"] == "append":
        Hq, past, rot = case["Hq"], case["past"], case["rot"]
        st["table"], st["pages"], st["per"], st["pools"] = _cache(case, past + S, g)
        st["pos"] = (torch.arange(S, device=DEV, dtype=torch.int32) + past).repeat(B)
        # a few channels of the keys far larger than the others, as projections have them
        x = rand(B * S, Hq + 2 * Hkv, D)
        x[:, :, 3::41] *= 6.0
        st["qkv"] = x.bfloat16()
        angle = torch.arange(past + S, device=DEV, dtype=torch.float64).unsqueeze(1) * (
            1e6 ** (-2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot))
        st["table_rot"] = torch.cat((angle.cos(), angle.sin()), 1).float().contiguous()
        st["qw"] = (1.0 + 0.1 * rand(D)).bfloat16() if case["norm"] else None
        st["kw"] = (1.0 + 0.1 * rand(D)).bfloat16() if case["norm"] else None
        st["q"] = torch.empty(B * Hq, S, D, dtype=torch.bfloat16, device=DEV)
    else:
        st["table"], st["pages"], st["per"], st["pools"] = _cache(case, S, g)
        st["pos"] = torch.arange(S, device=DEV, dtype=torch.int32).repeat(B)
    st["k"] = torch.empty(B * Hkv, S, D, dtype=torch.bfloat16, device=DEV)
    st["v"] = torch.empty(B * Hkv, S, D, dtype=torch.bfloat16, device=DEV)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if own:
        return {"mod": _own_mod, "kv4": _own_kv4, "append": _own_append, "unpack": _own_unpack}[case["op"]](case, st)
    return {"mod": _plain_mod, "kv4": _plain_kv4, "append": _plain_append, "unpack": _plain_unpack}[case["op"]](case, st)


def _ok(rc):
    if rc != 0:
        raise RuntimeError("status %d" % rc)


def _own_mod(c, st):
    import transfer_station_b200 as ts

    begin = end = None
    if c["mask"] == "docs":
        begin, end = st["begin"], st["end"]
        _ok(ts.attn_mask_ranges_stream(st["cu"], st["prefix"], c["docs"], c["Sq"], c["causal"], 0, begin, end))
    elif c["mask"] == "lens":
        end = st["end"]
    mod = ts.attn_mod(softcap=c["cap"], causal=c["causal"] and c["mask"] != "docs", slopes=st["slopes"], key_begin=begin,
                      key_end=end)
    _ok(ts.attn_flash_mod_stream(st["q"], st["k"], st["v"], st["o"], ts.ATTN_OUT_BF16, c["B"], c["Hq"], c["Hkv"], c["Sq"],
                                 c["Sk"], c["D"], mod, st["scratch"]))
    return st["o"]


def _own_kv4(c, st):
    import transfer_station_b200 as ts

    kc, ks, vc, vs = st["pools"]
    mod = ts.attn_mod(softcap=c["cap"], causal=True, slopes=st["slopes"])
    _ok(ts.attn_flash_kv4_stream(st["q"], kc, ks, vc, vs, st["table"], st["lens"], st["o"], ts.ATTN_OUT_BF16, c["B"],
                                 c["Hq"], c["Hkv"], c["Sq"], c["D"], mod, c["page"], st["pages"], st["per"],
                                 st["scratch"]))
    return st["o"]


def _own_append(c, st):
    import transfer_station_b200 as ts

    kc, ks, vc, vs = st["pools"]
    _ok(ts.attn_qkv_rope_kv4_stream(st["qkv"], st["pos"], st["table_rot"], c["past"] + c["S"], st["qw"], st["kw"], 1e-6,
                                    c["B"], c["S"], c["Hq"], c["Hkv"], c["D"], c["rot"],
                                    ts.ATTN_ROPE_NEOX if c["neox"] else ts.ATTN_ROPE_GPTJ, st["q"], kc, ks, vc, vs,
                                    st["table"], c["page"], st["pages"], st["per"], st["scratch"]))
    return (st["q"],) + _own_unpack(c, st)


def _own_unpack(c, st):
    import transfer_station_b200 as ts

    kc, ks, vc, vs = st["pools"]
    _ok(ts.attn_kv4_unpack_stream(kc, ks, vc, vs, st["table"], st["pos"], st["k"], st["v"], c["B"], c["S"], c["Hkv"],
                                  c["D"], c["page"], st["pages"], st["per"], st["scratch"]))
    return st["k"], st["v"]


# ------------------------------------------------------------------ plain forms
def _attend(q, k, v, B, Hq, Hkv, Sq, seen, cap, slopes, dist):
    """softmax(f(q k^T / sqrt(D))) v in 32 bits. q [B*Hq][Sq][D], k and v [B*Hkv][Sk][D]; `seen` truth values and `dist`
    distances, both [B or 1][Sq][Sk]. Rows that see no key are zero."""
    D, Sk = q.shape[-1], k.shape[1]
    s = (q.float().view(B * Hkv, -1, D) @ k.float().transpose(1, 2)).view(B, Hq, Sq, Sk).mul_(1.0 / math.sqrt(D))
    if cap > 0:
        s = s.div_(cap).tanh_().mul_(cap)
    if slopes is not None:
        # distances count from the nearest key that the row sees: softmax does not change, and far rows keep their bits
        near = torch.where(seen, dist, dist.max()).amin(-1, keepdim=True)
        s -= slopes.view(1, Hq, 1, 1) * (dist - near).float().unsqueeze(1)
    s.masked_fill_(~seen.unsqueeze(1), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B * Hkv, -1, Sk) @ v.float()).view(B, Hq, Sq, D)
    return (o / torch.where(total > 0, total, torch.ones_like(total))).view(B * Hq, Sq, D)


def _plain_ranges(c, st):
    """What each query position of packed documents sees: its document up to itself, and its document's prefix."""
    S, cu = c["Sq"], st["cu"].long()
    i = torch.arange(S, device=DEV)
    doc = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    held = doc < c["docs"]
    doc = doc.clamp(max=c["docs"] - 1)
    begin, stop = cu[doc], cu[doc + 1]
    end = torch.maximum(i + 1, torch.minimum(stop, begin + st["prefix"].long()[doc])) if c["causal"] else stop
    return torch.where(held, begin, 0), torch.where(held, end, 0)


def _plain_mod(c, st):
    B, Sq, Sk = c["B"], c["Sq"], c["Sk"]
    j, i = torch.arange(Sk, device=DEV), torch.arange(Sq, device=DEV) + Sk - Sq
    dist = (i.unsqueeze(1) - j).abs().unsqueeze(0)
    if c["mask"] == "docs":
        begin, end = _plain_ranges(c, st)
        seen = ((j >= begin.unsqueeze(1)) & (j < end.unsqueeze(1))).unsqueeze(0)
    elif c["mask"] == "lens":
        seen = j < st["end"].unsqueeze(-1)
    else:
        seen = (j <= (i.unsqueeze(1) if c["causal"] else Sk)).expand(Sq, Sk).unsqueeze(0)
    o = _attend(st["q"], st["k"], st["v"], B, c["Hq"], c["Hkv"], Sq, seen, c["cap"], st["slopes"], dist)
    return o.bfloat16()


def _plain_kv4(c, st):
    B, Hkv, Sq, D = c["B"], c["Hkv"], c["Sq"], c["D"]
    at = st["table"].long()
    kc, ks, vc, vs = st["pools"]
    k = _decode(kc[at], ks[at]).transpose(1, 2).reshape(B * Hkv, -1, D)
    v = _decode(vc[at], vs[at]).transpose(1, 2).reshape(B * Hkv, -1, D)
    j, last = torch.arange(k.shape[1], device=DEV), st["lens"].view(B, 1) - Sq + torch.arange(Sq, device=DEV)
    seen = j <= last.unsqueeze(-1)
    dist = (last.unsqueeze(-1) - j).abs()
    return _attend(st["q"], k, v, B, c["Hq"], Hkv, Sq, seen, c["cap"], st["slopes"], dist).bfloat16()


def _rotated(x, w, pos, table, rot, neox):
    """Heads [tokens][heads][D] normed (the root in 64 bits, rounded once) and rotated in 32 bits, rounded to bf16."""
    if w is not None:
        mean = x.double().square().mean(-1, keepdim=True) + torch.tensor(1e-6, dtype=torch.float32).double().item()
        x = x * mean.rsqrt().float() * w.float()
    cos, sin = table[pos.long()].unsqueeze(1).chunk(2, -1)
    turned, rest = x[..., :rot], x[..., rot:]
    a, b = (turned[..., : rot // 2], turned[..., rot // 2:]) if neox else (turned[..., 0::2], turned[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((a, b), -1) if neox else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((turned, rest), -1).bfloat16()


def _slots(c, st):
    """Page and row of every token's slot."""
    b = torch.arange(c["B"], device=DEV).repeat_interleave(c["S"])
    pos = st["pos"].long()
    return st["table"].long()[b, pos // c["page"]], pos % c["page"]


def _plain_append(c, st):
    B, S, Hq, Hkv, D = c["B"], c["S"], c["Hq"], c["Hkv"], c["D"]
    x = st["qkv"].float()
    q = _rotated(x[:, :Hq], st["qw"], st["pos"], st["table_rot"], c["rot"], c["neox"])
    k = _rotated(x[:, Hq:Hq + Hkv], st["kw"], st["pos"], st["table_rot"], c["rot"], c["neox"])
    v = st["qkv"][:, Hq + Hkv:]
    page, row = _slots(c, st)
    kc, ks, vc, vs = st["pools"]
    kc[page, :, row], ks[page, :, row] = _encode(k)
    vc[page, :, row], vs[page, :, row] = _encode(v)
    return (q.view(B, S, Hq, D).transpose(1, 2).reshape(B * Hq, S, D),) + _plain_unpack(c, st)


def _plain_unpack(c, st):
    B, S, Hkv, D = c["B"], c["S"], c["Hkv"], c["D"]
    page, row = _slots(c, st)
    kc, ks, vc, vs = st["pools"]
    k, v = _decode(kc[page, :, row], ks[page, :, row]), _decode(vc[page, :, row], vs[page, :, row])
    return tuple(t.bfloat16().view(B, S, Hkv, D).transpose(1, 2).reshape(B * Hkv, S, D) for t in (k, v))


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    st = prepare(case, seed)
    return {"mod": _exact_mod, "kv4": _exact_kv4, "append": _exact_append, "unpack": _exact_unpack}[case["op"]](case, st)


def _value64(codes, scales, e):
    """Element e[...] of rows of nibble pairs, from the bits: (nibble - 8) times a scale of 4 exponent bits and 3 more."""
    byte = codes[..., e // 2].long()
    nibble = torch.where(e % 2 == 0, byte % 16, byte // 16) - 8
    s = scales[..., e // GROUP].long()
    sign, ex, man = 1 - 2 * (s // 128), (s // 8) % 16, s % 8
    low = (man.double() / 8) * 2.0 ** -6
    size = torch.where(ex > 0, (1 + man.double() / 8) * torch.pow(2.0, (ex - 7).double()), low)
    return nibble.double() * sign.double() * size


def _exact_head(q, k, v, allowed, cap, slope, offset):
    """One head in 64 bits: q [Sq][D], k and v [Sk][D]; `offset` is the position of query 0."""
    s = q @ k.T / math.sqrt(q.shape[1])
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    if slope:
        i, j = torch.arange(q.shape[0], device=DEV) + offset, torch.arange(k.shape[0], device=DEV)
        s = s - slope * (i[:, None] - j[None, :]).abs().double()
    p = torch.where(allowed, s, torch.full_like(s, -math.inf))
    empty = ~allowed.any(1)
    p[empty] = 0.0
    o = torch.softmax(p, 1) @ v
    o[empty] = 0.0
    return o


def _exact_mod(c, st):
    B, Hq, Hkv, Sq, Sk = c["B"], c["Hq"], c["Hkv"], c["Sq"], c["Sk"]
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    allowed = torch.ones(B, Sq, Sk, dtype=torch.bool, device=DEV)
    if c["mask"] == "docs":
        allowed.zero_()
        cu, pre = _documents(c)
        for a, b, p in zip(cu, cu[1:], pre):
            block = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV)
            if c["causal"]:
                block = block.tril()
                block[:, :p] = True
            allowed[0, a:b, a:b] = block
    elif c["mask"] == "lens":
        for b, n in enumerate(_lens(c)):
            allowed[b, :, n:] = False
    elif c["causal"]:
        allowed = allowed.tril(Sk - Sq)
    out = torch.empty(B * Hq, Sq, c["D"], dtype=torch.float64, device=DEV)
    for h in range(B * Hq):
        kv = h // (Hq // Hkv)
        slope = 2.0 ** (-8.0 * (h % Hq + 1) / Hq) if c["alibi"] else 0.0
        slope = torch.tensor(slope, dtype=torch.float32).double().item()
        out[h] = _exact_head(q[h], k[kv], v[kv], allowed[h // Hq], c["cap"], slope, Sk - Sq)
    return out


def _exact_kv4(c, st):
    B, Hq, Hkv, Sq, D, P = c["B"], c["Hq"], c["Hkv"], c["Sq"], c["D"], c["page"]
    kc, ks, vc, vs = st["pools"]
    e = torch.arange(D, device=DEV)
    out = torch.empty(B, Hq, Sq, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(c)):
        t = torch.arange(n, device=DEV)
        page, row = st["table"][b].long()[t // P], t % P
        k, v = _value64(kc[page, :, row], ks[page, :, row], e), _value64(vc[page, :, row], vs[page, :, row], e)
        allowed = t[None, :] <= n - Sq + torch.arange(Sq, device=DEV)[:, None]
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            slope = torch.tensor(2.0 ** (-8.0 * (h + 1) / Hq) if c["alibi"] else 0.0, dtype=torch.float32).double().item()
            out[b, h] = _exact_head(st["q"].view(B, Hq, Sq, D)[b, h].double(), k[:, kv], v[:, kv], allowed, c["cap"], slope,
                                    n - Sq)
    return out.view(B * Hq, Sq, D)


def _exact_append(c, st):
    B, S, Hq, Hkv, D, rot = c["B"], c["S"], c["Hq"], c["Hkv"], c["D"], c["rot"]
    x = st["qkv"].double()
    eps = torch.tensor(1e-6, dtype=torch.float32).double()

    def turn(h, w):
        if w is not None:
            h = h / torch.sqrt((h ** 2).sum(-1, keepdim=True) / D + eps) * w.double()
        n = rot // 2
        cs = st["table_rot"].double()[st["pos"].long()]
        y = h.clone()
        for f in range(n):
            a, b = (f, f + n) if c["neox"] else (2 * f, 2 * f + 1)
            cf, sf = cs[:, f, None], cs[:, n + f, None]
            y[..., a], y[..., b] = h[..., a] * cf - h[..., b] * sf, h[..., b] * cf + h[..., a] * sf
        return y

    def stored(h):
        """What the cache stands for: bf16 values, a scale for each group, whole multiples of it."""
        h = h.to(torch.bfloat16).double().view(*h.shape[:-1], D // GROUP, GROUP)
        s = (h.abs().amax(-1, keepdim=True) / 7).clamp(max=448).float().to(torch.float8_e4m3fn).double()
        n = torch.where(s > 0, h / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(h)).round().clamp(-8, 7)
        return (n * s).flatten(-2)

    def whole(h, n):
        return h.view(B, S, n, D).permute(0, 2, 1, 3).reshape(B * n, S, D)

    q, k = turn(x[:, :Hq], st["qw"]), turn(x[:, Hq:Hq + Hkv], st["kw"])
    return whole(q, Hq), whole(stored(k), Hkv), whole(stored(x[:, Hq + Hkv:]), Hkv)


def _exact_unpack(c, st):
    B, S, Hkv, D, P = c["B"], c["S"], c["Hkv"], c["D"], c["page"]
    kc, ks, vc, vs = st["pools"]
    e, t = torch.arange(D, device=DEV), torch.arange(S, device=DEV)
    out = [torch.empty(B, Hkv, S, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    for b in range(B):
        page, row = st["table"][b].long()[t // P], t % P
        for o, codes, scales in ((out[0], kc, ks), (out[1], vc, vs)):
            o[b] = _value64(codes[page, :, row], scales[page, :, row], e).transpose(0, 1)
    return tuple(o.view(B * Hkv, S, D) for o in out)
