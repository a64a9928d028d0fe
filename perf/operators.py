"""Cases that measure the cache-append and 4-bit-cache operators.

Four operators, named by a case's "op":
  append      head norms, rotation and paged append of K and V (kv_append.gqa_append)
  append_kv4  the same into the 4-bit cache, then the new tokens read back
              (kv_append.gqa_append_kv4, kv4_decode.gqa_gather_kv4)
  decode_kv4  attention of one query token per request over the 4-bit cache
              (kv4_decode.gqa_decode_kv4)
  append_mla  latent norm, rotation and append to the latent cache (kv_append.mla_append)

run() computes them with elementary torch operations, or with the framework's
calls when `own` is set.

The 4-bit cache is uint8 [num_blocks, block_size / 16, Hkv, 1024 + 64 * (128 / G)]:
one tile holds 16 tokens of one kv head, G dims share a bf16 scale s and a
bf16 centre c, and code n stands for s * (n - 8) + c.
  K codes: token i at byte 64 i; the word of dims 8w .. 8w + 7 (nibble j = dim
           8w + j) at byte 16 (w % 4) + 4 (w / 4) of it.
  V codes: tokens 2p, 2p + 1 at byte 128 p; the 16 bits of dims 4r .. 4r + 3,
           r = 8y + g, of token 2p + e at byte 16 (g ^ 2 (p % 4)) + 4y + 2e of it.
  then s [16, 128 / G], then c: K [16, 128 / G], V [128 / G, 16].
"""

import math
import os
import sys

import torch

own = False

D = 128
LATENT, ROPE = 512, 64
EPS = 1e-6


# ---- cases --------------------------------------------------------------------


def listed():
    return [
        # one new token of one request: the latency of a decode step's append
        dict(name="append_one_token", op="append", B=1, new=1, ctx_lo=4096, ctx_hi=4096, Hq=32, Hkv=8,
             bs=16, rot=128, interleaved=False, norm=False, packed=True, pad=0),
        # a decode step of a large batch, heads normed, the batch padded to a captured graph's size
        dict(name="append_decode_normed", op="append", B=128, new=1, ctx_lo=64, ctx_hi=2048, Hq=64, Hkv=8,
             bs=64, rot=128, interleaved=False, norm=True, packed=True, pad=9),
        # prompt chunks of uneven lengths, half of each head rotated in adjacent pairs
        dict(name="append_chunks_partial", op="append", B=13, new=631, ctx_lo=1, ctx_hi=4097, Hq=32,
             Hkv=8, bs=16, rot=64, interleaved=True, norm=False, packed=False, pad=0),
        # long prompts: the largest append, bound by memory
        dict(name="append_prefill", op="append", B=4, new=8192, ctx_lo=1, ctx_hi=64, Hq=64, Hkv=8,
             bs=64, rot=128, interleaved=False, norm=True, packed=True, pad=5),
        # a decode step into the 4-bit cache
        dict(name="append_kv4_decode", op="append_kv4", B=32, new=1, ctx_lo=64, ctx_hi=2048, Hq=32, Hkv=8,
             bs=16, rot=128, interleaved=False, norm=False, packed=True, pad=0, group=64),
        # long prompts into the 4-bit cache
        dict(name="append_kv4_prefill", op="append_kv4", B=7, new=2341, ctx_lo=1, ctx_hi=1000, Hq=32,
             Hkv=8, bs=64, rot=128, interleaved=False, norm=True, packed=True, pad=0, group=32),
        # four short requests (uniform in [1, 512]): latency
        dict(name="decode_kv4_small", op="decode_kv4", B=4, lo=1, hi=512, spread="uniform", Hq=32, Hkv=8,
             bs=16, group=64),
        # the representative decode shape
        dict(name="decode_kv4_rep", op="decode_kv4", B=32, lo=8192, hi=8192, spread="uniform", Hq=32,
             Hkv=8, bs=16, group=64),
        # a ragged batch of a wide group, lengths log-uniform, some requests empty
        dict(name="decode_kv4_ragged", op="decode_kv4", B=64, lo=64, hi=16384, spread="log", Hq=64, Hkv=8,
             bs=64, group=32, empty=2),
        # one very long request
        dict(name="decode_kv4_long", op="decode_kv4", B=1, lo=262144, hi=262144, spread="uniform", Hq=32,
             Hkv=8, bs=64, group=128),
        # a decode step of the latent cache with 128 query heads
        dict(name="append_mla_decode", op="append_mla", B=128, new=1, ctx_lo=64, ctx_hi=2048, h=128,
             interleaved=True, norm=True, pad=0),
        # prompts into the latent cache
        dict(name="append_mla_prefill", op="append_mla", B=5, new=1639, ctx_lo=1, ctx_hi=500, h=64,
             interleaved=True, norm=True, pad=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append_kv4", "decode_kv4", "append_mla"])
    if op == "decode_kv4":
        Hkv = rng.choice([1, 2, 4, 8])
        hi = _log(rng, 20, 16384)
        B = max(1, min(_log(rng, 1, 96), 32 * 8192 * 8 // (hi * Hkv)))
        return dict(op=op, B=B, lo=max(1, hi // rng.choice([1, 4, 64])), hi=hi,
                    spread=rng.choice(["uniform", "log"]), Hq=Hkv * rng.choice([1, 3, 4, 7, 8, 16]), Hkv=Hkv,
                    bs=rng.choice([16, 32, 64, 128]), group=rng.choice([32, 64, 128]),
                    empty=rng.randint(0, B // 4))
    if rng.random() < 0.5:
        B, new = _log(rng, 1, 256), 1
    else:
        B = _log(rng, 1, 16)
        new = _log(rng, 2, 16384 // B)
    case = dict(op=op, B=B, new=new, ctx_lo=1, ctx_hi=_log(rng, 2, 2048),
                interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                pad=rng.randint(0, 7) if B > 1 else 0)
    if op == "append_mla":
        return dict(case, h=rng.choice([1, 16, 24, 64, 128]))
    Hkv = rng.choice([1, 2, 4, 8])
    case.update(Hkv=Hkv, Hq=Hkv * rng.choice([1, 3, 4, 7, 8]), rot=rng.choice([16, 32, 64, 96, 128]),
                packed=rng.random() < 0.5)
    if op == "append":
        return dict(case, bs=rng.choice([1, 16, 24, 64, 128]))
    return dict(case, bs=rng.choice([16, 32, 64, 128]), group=rng.choice([32, 64]))


# ---- inputs ---------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _spread(B, gen):
    """B points spread evenly over [0, 1] in a random order: every seed has the same sum."""
    return (torch.randperm(B, generator=gen, device="cuda").double() + 0.5) / B


def _lengths(case, gen):
    """Tokens of every request: uniform or log-uniform in [lo, hi]."""
    u = _spread(case["B"], gen)
    lo, hi = case["lo"], case["hi"]
    if case["spread"] == "log":
        s = torch.exp(math.log(lo) + u * (math.log(hi) - math.log(lo)))
    else:
        s = lo + u * (hi - lo)
    s = s.round().long().clamp(lo, hi)
    if case.get("empty"):
        s[torch.randperm(case["B"], generator=gen, device="cuda")[: case["empty"]]] = 0
    return s


def _pages(lens, bs, gen, tokens):
    """A block table over a permuted pool that holds `tokens` tokens however the requests
    share them: (table [B, max_blocks] int32, blocks in the pool)."""
    n = (lens + bs - 1) // bs
    width, used = max(1, int(n.max())), int(n.sum())
    pool = tokens // bs + len(lens) + 3
    perm = torch.randperm(pool, generator=gen, device="cuda").int()
    col = torch.arange(width, device="cuda")
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[col < n[:, None]] = perm[:used]
    return table, pool


def _table(positions, rot, base=10000.0):
    """Rotation table [positions, rot] fp32: cosines, then sines, the angles in 64 bits."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _bf16(shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).bfloat16()


def _split(case, gen):
    """New tokens of every request: their lengths after the append, the prefix of the
    new tokens' counts (None for one token each), the rows in all, and the most tokens."""
    B, new, pad = case["B"], case["new"], case["pad"]
    lo, hi = math.log(case["ctx_lo"]), math.log(case["ctx_hi"])
    old = torch.exp(lo + _spread(B, gen) * (hi - lo)).round().long()
    most = int(old.sum()) + B * new
    if new == 1:  # a decode step: padding requests have no tokens
        lens = old + 1
        if pad:
            lens[torch.randperm(B, generator=gen, device="cuda")[: min(pad, B - 1)]] = 0
        return lens, None, B, most
    # prompt chunks of uneven lengths, `new` on average; `pad` rows behind the last
    w = torch.rand(B, generator=gen, device="cuda", dtype=torch.float64) + 0.3
    cnt = torch.floor(w / w.sum() * (B * new)).long()
    cnt[0] += B * new - int(cnt.sum())
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    cu[1:] = cnt.cumsum(0)
    return old + cnt, cu, B * new + pad, most


def _pack_tiles(x, group, value):
    """4-bit tiles of x [..., 16, 128] (fp32): uint8 [..., 1024 + 64 * (128 / group)]."""
    n, s, c = _quantise(x, group)
    lead = x.shape[:-2]
    b = n[..., 0::2] | (n[..., 1::2] << 4)  # [..., 16, 64] bytes in the order of the dims
    if value:
        # [pair, token of pair, y, g, byte] -> [pair, g, y, token, byte], g swizzled by the pair
        b = b.view(*lead, 8, 2, 4, 8, 2).movedim(-2, -4).movedim(-3, -2)
        p = torch.arange(8, device=x.device)
        b = b[..., p[:, None], p[None, :] ^ (2 * (p[:, None] % 4)), :, :, :]
        c = c.transpose(-1, -2)
    else:
        b = b.view(*lead, 16, 4, 4, 4).transpose(-2, -3)
    parts = [b.reshape(*lead, 1024), s.contiguous().view(torch.uint8).reshape(*lead, -1),
             c.contiguous().view(torch.uint8).reshape(*lead, -1)]
    return torch.cat(parts, -1)


def _make_kv4(tiles, Hkv, group, gen, value):
    """A filled 4-bit cache of `tiles` tiles per head: normal values under uneven channels."""
    out = torch.empty((tiles, Hkv, 1024 + 64 * (D // group)), dtype=torch.uint8, device="cuda")
    gain = torch.rand((Hkv, 1, D), generator=gen, device="cuda") + 0.5
    step = max(1, 65536 // Hkv)
    for i in range(0, tiles, step):
        m = min(step, tiles - i)
        x = torch.randn((m, Hkv, 16, D), generator=gen, device="cuda") * gain
        out[i:i + m] = _pack_tiles(x, group, value)
    return out


def prepare(case, seed):
    gen = _gen(seed)
    op = case["op"]
    st = dict(case)
    if op == "decode_kv4":
        lens = _lengths(case, gen)
        bs, Hkv, Hq = case["bs"], case["Hkv"], case["Hq"]
        table, pool = _pages(lens, bs, gen, case["B"] * case["hi"])
        for name in ("k_cache", "v_cache"):
            tiles = _make_kv4(pool * (bs // 16), Hkv, case["group"], gen, name == "v_cache")
            st[name] = tiles.view(pool, bs // 16, Hkv, -1)
        st.update(q=_bf16((case["B"], Hq, D), gen), table=table, lens=lens.int(), scale=D ** -0.5)
        return st
    lens, cu, rows, most = _split(case, gen)
    bs = 64 if op == "append_mla" else case["bs"]
    table, pool = _pages(lens, bs, gen, most)
    st.update(table=table, lens=lens.int(), cu=cu, rows=rows)
    if op == "append_mla":
        h = case["h"]
        st.update(kv_c=_bf16((rows, LATENT), gen), k_pe=_bf16((rows, ROPE), gen),
                  q_pe=_bf16((rows, h, 128 + ROPE), gen)[..., 128:], cache=_bf16((pool, 64, 1, LATENT + ROPE), gen),
                  cos_sin=_table(int(lens.max()) + 1, ROPE),
                  weight=_bf16((LATENT,), gen, 0.1) + 1 if case["norm"] else None)
        return st
    Hq, Hkv = case["Hq"], case["Hkv"]
    if case["packed"]:  # slices of one projection's output
        qkv = _bf16((rows, Hq + 2 * Hkv, D), gen)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        q, k, v = (_bf16((rows, n, D), gen) for n in (Hq, Hkv, Hkv))
    st.update(q=q, k=k, v=v, cos_sin=_table(int(lens.max()) + 1, case["rot"]), q_weight=None, k_weight=None)
    if case["norm"]:
        st.update(q_weight=_bf16((D,), gen, 0.1) + 1, k_weight=_bf16((D,), gen, 0.1) + 1)
    if op == "append_kv4":
        for name in ("k_cache", "v_cache"):
            tiles = _make_kv4(pool * (bs // 16), Hkv, case["group"], gen, name == "v_cache")
            st[name] = tiles.view(pool, bs // 16, Hkv, -1)
        if cu is None:  # the rows to read back: each request's last token
            cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda")
            cu[1:] = (lens > 0).cumsum(0)
        st.update(cu_back=cu, rows_back=rows)
    else:
        st.update(k_cache=_bf16((pool, bs, Hkv, D), gen), v_cache=_bf16((pool, bs, Hkv, D), gen))
    return st


# ---- the plain forms ---------------------------------------------------------------


def _norm(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotate(x, cs, interleaved):
    """x [T, H, D] fp32, cs [T, R]: the first R dims of every head rotated."""
    R = cs.shape[1]
    cos, sin = cs[:, None, : R // 2], cs[:, None, R // 2:]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2:R]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., R:]], -1)


def _place(st, cu, rows):
    """Request and position of every row, and whether the row holds a token."""
    lens = st["lens"].long()
    t = torch.arange(rows, device=lens.device)
    if cu is None:
        return t, lens - 1, lens > 0
    cu = cu.long()
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=len(lens) - 1)
    pos = lens[b] - cu[b + 1] + t
    ok = (t < cu[-1]) & (pos >= 0)
    return b, torch.where(ok, pos, 0), ok


def _quantise(x, group):
    """Codes [..., 128] uint8 and the bf16 scales and centres [..., 128 / group] of x (fp32)."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    # the scale is rounded up to bf16, so that 15 steps reach across the group (a tensor
    # divides: division by a number may multiply by its rounded reciprocal)
    s = ((((hi - lo) / torch.full_like(lo, 15)).view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)
    c = (lo + 8 * s).bfloat16()
    n = torch.round((g - c.float()[..., None]) / s[..., None]).nan_to_num(0.0)
    return (n.clamp(-8, 7) + 8).to(torch.uint8).flatten(-2), s.bfloat16(), c


def _unpack(tiles, group, value):
    """What tiles [..., 1024 + 64 * (128 / group)] stand for: fp32 [..., 16, 128]."""
    lead, ng = tiles.shape[:-1], D // group
    b = tiles[..., :1024]
    s = tiles[..., 1024:1024 + 32 * ng].contiguous().view(torch.bfloat16).view(*lead, 16, ng)
    c = tiles[..., 1024 + 32 * ng:].contiguous().view(torch.bfloat16)
    if value:
        p = torch.arange(8, device=tiles.device)
        b = b.reshape(*lead, 8, 8, 4, 2, 2)[..., p[:, None], p[None, :] ^ (2 * (p[:, None] % 4)), :, :, :]
        b = b.movedim(-2, -3).movedim(-4, -2)  # [pair, token, y, g, byte]
        c = c.view(*lead, ng, 16).transpose(-1, -2)
    else:
        b = b.reshape(*lead, 16, 4, 4, 4).transpose(-2, -3)
        c = c.view(*lead, 16, ng)
    b = b.reshape(*lead, 16, 64)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2).float() - 8
    n = n.unflatten(-1, (ng, group))
    return (n * s.float()[..., None] + c.float()[..., None]).flatten(-2)


def _slots(st, b, pos, bs):
    return st["table"].long()[b, pos.clamp(min=0) // bs], pos.clamp(min=0) % bs


def _normed_rotated(st, b, pos):
    cs = st["cos_sin"][pos.clamp(min=0)]
    q = _rotate(_norm(st["q"].float(), st["q_weight"]), cs, st["interleaved"])
    k = _rotate(_norm(st["k"].float(), st["k_weight"]), cs, st["interleaved"])
    return q, k


def _plain_append(st):
    b, pos, ok = _place(st, st["cu"], st["rows"])
    q, k = _normed_rotated(st, b, pos)
    page, slot = _slots(st, b, pos, st["bs"])
    st["k_cache"][page[ok], slot[ok]] = k[ok].bfloat16()
    st["v_cache"][page[ok], slot[ok]] = st["v"][ok]
    return {"q": (q * ok[:, None, None]).bfloat16(), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _byte_offsets(i, ng, value):
    """Bytes of a tile that tokens i [T] own, in the order _token_bytes gives them: [T, 64 + 4 ng]."""
    m = torch.arange(64, device=i.device)
    i = i[:, None]
    if value:
        r = m // 2
        codes = 128 * (i // 2) + 16 * ((r % 8) ^ (2 * (i // 2 % 4))) + 4 * (r // 8) + 2 * (i % 2) + m % 2
    else:
        w = m // 4
        codes = 64 * i + 16 * (w % 4) + 4 * (w // 4) + m % 4
    e = torch.arange(2 * ng, device=i.device)
    s = 1024 + 2 * ng * i + e
    c = 1024 + 32 * ng + (32 * (e // 2) + 2 * i + e % 2 if value else 2 * ng * i + e)
    return torch.cat([codes, s, c], 1)


def _token_bytes(x, group):
    n, s, c = _quantise(x, group)
    return torch.cat([n[..., 0::2] | (n[..., 1::2] << 4), s.view(torch.uint8), c.view(torch.uint8)], -1)


def _plain_append_kv4(st):
    b, pos, ok = _place(st, st["cu"], st["rows"])
    q, k = _normed_rotated(st, b, pos)
    page, slot = _slots(st, b, pos, st["bs"])
    page, slot = page[ok, None, None], slot[ok]
    head = torch.arange(st["Hkv"], device=q.device)[:, None]
    back_b, back_pos, back_ok = _place(st, st["cu_back"], st["rows_back"])
    back_page, back_slot = _slots(st, back_b, back_pos, st["bs"])
    read = []
    for name, x in (("k_cache", k[ok]), ("v_cache", st["v"][ok].float())):
        value = name == "v_cache"
        off = _byte_offsets(slot % 16, D // st["group"], value)
        st[name][page, slot[:, None, None] // 16, head, off[:, None]] = _token_bytes(x, st["group"])
        tiles = st[name][back_page, back_slot // 16]
        y = _unpack(tiles, st["group"], value)[torch.arange(len(tiles), device=q.device), :, back_slot % 16]
        read.append((y * back_ok[:, None, None]).bfloat16())
    return {"q": (q * ok[:, None, None]).bfloat16(), "k": read[0], "v": read[1]}


def _plain_decode_kv4(st):
    B, Hq, Hkv = st["B"], st["Hq"], st["Hkv"]
    table = st["table"].long().clamp(min=0)

    def rows(name):  # [B, Hkv, tokens, 128]
        x = _unpack(st[name][table], st["group"], name == "v_cache")
        return x.movedim(3, 1).reshape(B, Hkv, -1, D)

    q = st["q"].float().view(B, Hkv, Hq // Hkv, D) * st["scale"]
    x = q @ rows("k_cache").transpose(-1, -2)
    hidden = torch.arange(x.shape[-1], device=x.device) >= st["lens"][:, None, None, None]
    x = x.masked_fill(hidden, -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return (p @ rows("v_cache")).view(B, Hq, D).bfloat16()


def _plain_append_mla(st):
    b, pos, ok = _place(st, st["cu"], st["rows"])
    cs = st["cos_sin"][pos.clamp(min=0)]
    latent = _norm(st["kv_c"].float(), st["weight"])
    k = _rotate(st["k_pe"].float()[:, None], cs, st["interleaved"])[:, 0]
    q = _rotate(st["q_pe"].float(), cs, st["interleaved"])
    page, slot = _slots(st, b, pos, 64)
    st["cache"][page[ok], slot[ok], 0] = torch.cat([latent, k], -1)[ok].bfloat16()
    return {"q_pe": (q * ok[:, None, None]).bfloat16(), "cache": st["cache"]}


# ---- the framework's calls ------------------------------------------------------------


def _modules():
    path = os.path.join(os.getcwd(), "mla-decode-kernels_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kv4_decode
    import kv_append

    return kv_append, kv4_decode


def _own(st):
    kv_append, kv4_decode = _modules()
    op = st["op"]
    if op == "decode_kv4":
        return kv4_decode.gqa_decode_kv4(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                                         st["scale"])
    if op == "append_mla":
        q = kv_append.mla_append(st["kv_c"], st["k_pe"], st["cache"], st["table"], st["lens"], st["cos_sin"],
                                 q_pe=st["q_pe"], cu_seqlens=st["cu"], interleaved=st["interleaved"],
                                 kv_weight=st["weight"], eps=EPS)
        return {"q_pe": q, "cache": st["cache"]}
    call = kv_append.gqa_append if op == "append" else kv_append.gqa_append_kv4
    q = call(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["cos_sin"],
             cu_seqlens=st["cu"], interleaved=st["interleaved"], q_weight=st["q_weight"],
             k_weight=st["k_weight"], eps=EPS)
    if op == "append":
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    k, v = kv4_decode.gqa_gather_kv4(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["cu_back"],
                                     st["rows_back"])
    return {"q": q, "k": k, "v": v}


_PLAIN = {"append": _plain_append, "append_kv4": _plain_append_kv4, "decode_kv4": _plain_decode_kv4,
          "append_mla": _plain_append_mla}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


# ---- the work of one pass ----------------------------------------------------------------


def _mean_tokens(case):
    lo, hi = case["lo"], case["hi"]
    mean = (hi - lo) / math.log(hi / lo) if case["spread"] == "log" and hi > lo else (lo + hi) / 2
    return mean * (case["B"] - case.get("empty", 0))


def work(case):
    op = case["op"]
    if op == "decode_kv4":
        tokens = _mean_tokens(case)
        row = 64 + 4 * (D // case["group"])
        return {"bytes": 2 * tokens * case["Hkv"] * row + 4 * case["B"] * case["Hq"] * D,
                "flops": 4 * tokens * case["Hq"] * D}
    T = case["B"] * case["new"] - (min(case["pad"], case["B"] - 1) if case["new"] == 1 else 0)
    if op == "append_mla":
        table = 4 * ROPE
        return {"bytes": T * (4 * (LATENT + ROPE) + 4 * case["h"] * ROPE + table),
                "flops": T * (4 * LATENT * case["norm"] + 3 * ROPE * (1 + case["h"]))}
    Hq, Hkv = case["Hq"], case["Hkv"]
    flops = T * (Hq + Hkv) * (4 * D * case["norm"] + 3 * case["rot"])
    read = T * ((Hq + 2 * Hkv) * 2 * D + 4 * case["rot"])
    if op == "append":
        return {"bytes": read + T * (Hq + 2 * Hkv) * 2 * D, "flops": flops}
    row = 64 + 4 * (D // case["group"])
    # codes and scales written, then read back and written out in bf16
    return {"bytes": read + T * (Hq * 2 * D + 2 * Hkv * (2 * row + 2 * D)), "flops": flops + T * 2 * Hkv * D * 6}


# ---- the definition in 64 bits -------------------------------------------------------------


def _exact_rows(st):
    """(request, position) of every row on the host, None where the row holds no token."""
    lens = st["lens"].tolist()
    if st["cu"] is None:
        return [(b, n - 1) if n > 0 else None for b, n in enumerate(lens)]
    cu = st["cu"].tolist()
    out = [None] * st["rows"]
    for b, n in enumerate(lens):
        for j in range(cu[b], cu[b + 1]):
            pos = n - (cu[b + 1] - j)
            out[j] = (b, pos) if pos >= 0 else None
    return out


def _exact_head(x, weight, angle, interleaved):
    """Norm and rotation of x [T, H, D] in 64 bits; angle = (cos, sin) [T, 1, R / 2]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    cos, sin = angle
    half = cos.shape[-1]
    y = x.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., first] * sin + x[..., second] * cos
    return y


def _exact_tokens(st):
    where = _exact_rows(st)
    live = torch.tensor([j for j, w in enumerate(where) if w is not None], device="cuda")
    b = torch.tensor([w[0] for w in where if w is not None], device="cuda")
    pos = torch.tensor([w[1] for w in where if w is not None], device="cuda")
    cs = st["cos_sin"].double()[pos][:, None]
    half = cs.shape[-1] // 2
    return live, b, pos, (cs[..., :half], cs[..., half:])


def _exact_kv4(x, group):
    """What x [N, 128] stands for after 4-bit storage, by the definition in 64 bits."""
    g = x.double().reshape(-1, group)
    lo, hi = g.min(1, keepdim=True).values, g.max(1, keepdim=True).values
    want = (hi - lo) / 15
    s = want.bfloat16().double()
    # bf16 rounds to nearest: one step further where that fell short
    up = (want.bfloat16().view(torch.int16) + 1).view(torch.bfloat16).double()
    s = torch.where(s < want, up, s)
    c = (lo + 8 * s).bfloat16().double()
    n = torch.where(s > 0, ((g - c) / torch.where(s > 0, s, 1)).round(), 0).clamp(-8, 7)
    return (n * s + c).reshape(x.shape)


def _exact_codes(tile, group, value):
    """A request's tiles [n, Hkv, bytes] as values [Hkv, 16 n, 128] in 64 bits, bit by bit from the layout."""
    ng = D // group
    tok = torch.arange(16, device="cuda")[:, None]
    dim = torch.arange(D, device="cuda")[None, :]
    if value:
        r = dim // 4
        at = 128 * (tok // 2) + 16 * ((r % 8) ^ (2 * (tok // 2 % 4))) + 4 * (r // 8) + 2 * (tok % 2) + dim % 4 // 2
        c_at = 1024 + 32 * ng + 32 * (dim // group) + 2 * tok
    else:
        w = dim // 8
        at = 64 * tok + 16 * (w % 4) + 4 * (w // 4) + dim % 8 // 2
        c_at = 1024 + 32 * ng + 2 * ng * tok + 2 * (dim // group)
    s_at = 1024 + 2 * ng * tok + 2 * (dim // group)

    def half(pos):  # bf16 at a byte offset
        v = tile[..., pos].int() | (tile[..., pos + 1].int() << 8)
        return (v << 16).view(torch.float32).double()

    code = (tile[..., at].int() >> (4 * (dim % 2))) & 15
    x = half(s_at) * (code - 8) + half(c_at)
    return x.transpose(0, 1).reshape(tile.shape[1], -1, D)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "decode_kv4":
        lens, Hkv, G = st["lens"].tolist(), case["Hkv"], case["Hq"] // case["Hkv"]
        out = torch.zeros((case["B"], case["Hq"], D), dtype=torch.float64, device="cuda")
        per = case["bs"] // 16
        for b, n in enumerate(lens):
            if n == 0:
                continue
            q = st["q"][b].double().view(Hkv, G, D)
            top, total, acc = None, None, None
            blocks = (n + case["bs"] - 1) // case["bs"]
            chunk = max(1, 8192 // case["bs"])
            for i in range(0, blocks, chunk):
                ids = st["table"][b, i:min(blocks, i + chunk)].long()
                k = _exact_codes(st["k_cache"][ids].flatten(0, 1), case["group"], False)
                v = _exact_codes(st["v_cache"][ids].flatten(0, 1), case["group"], True)
                keep = min(n - i * case["bs"], len(ids) * per * 16)
                x = torch.einsum("hgd,htd->hgt", q, k[:, :keep]) * st["scale"]
                m = x.max(-1, keepdim=True).values
                if top is not None:
                    m = torch.maximum(m, top)
                e = torch.exp(x - m)
                new_l, new_a = e.sum(-1, keepdim=True), torch.einsum("hgt,htd->hgd", e, v[:, :keep])
                if top is not None:
                    f = torch.exp(top - m)
                    new_l, new_a = new_l + total * f, new_a + acc * f
                top, total, acc = m, new_l, new_a
            out[b] = (acc / total).view(-1, D)
        return out
    live, b, pos, angle = _exact_tokens(st)
    if op == "append_mla":
        q = torch.zeros(st["q_pe"].shape, dtype=torch.float64, device="cuda")
        q[live] = _exact_head(st["q_pe"][live], None, angle, case["interleaved"])
        cache = st["cache"].double()
        at = (st["table"][b, pos // 64].long(), pos % 64, 0)
        latent = st["kv_c"][live].double()
        if st["weight"] is not None:
            latent = latent / torch.sqrt(latent.square().mean(-1, keepdim=True) + EPS) * st["weight"].double()
        cache[at] = torch.cat([latent, _exact_head(st["k_pe"][live][:, None], None, angle, case["interleaved"])[:, 0]], 1)
        return {"q_pe": q, "cache": cache}
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    q[live] = _exact_head(st["q"][live], st["q_weight"], angle, case["interleaved"])
    k = _exact_head(st["k"][live], st["k_weight"], angle, case["interleaved"])
    v = st["v"][live].double()
    if op == "append":
        at = (st["table"][b, pos // case["bs"]].long(), pos % case["bs"])
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        kc[at], vc[at] = k, v
        return {"q": q, "k_cache": kc, "v_cache": vc}
    # read back in the order of the requests: rows without a token are zero
    back = [torch.zeros((st["rows_back"], case["Hkv"], D), dtype=torch.float64, device="cuda") for _ in range(2)]
    for dst, x in zip(back, (k, v)):
        dst[: len(live)] = _exact_kv4(x, case["group"])
    return {"q": q, "k": back[0], "v": back[1]}
