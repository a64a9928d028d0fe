"""The 4-bit cache in plain torch and 64 bits, for the tests: the quantiser and
the tile layout of include/kv4_decode.h written out byte by byte, and the
append's norm and rotation."""

import torch

D, TILE = 128, 16


def tile_bytes(group):
    return 1024 + 64 * (D // group)


def quantise(x, group):
    """x [..., 128] fp32 -> codes [..., 128] int, s and c [..., 128 / group] fp32
    (bf16 values), with the kernel's roundings: one fp32 operation at a time."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    want = (hi - lo) / torch.full_like(lo, 15)
    s = ((want.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)
    c = (lo + 8 * s).bfloat16().float()
    n = torch.round((g - c[..., None]) / s[..., None])
    n = torch.where(s[..., None] == 0, torch.zeros_like(n), n).clamp(-8, 7) + 8
    return n.int().flatten(-2), s, c


def _byte_maps(group, value):
    """Byte positions in a tile: code byte of (token, dim), scale and centre of (token, y)."""
    ng = D // group
    tok = torch.arange(TILE)[:, None]
    dim = torch.arange(D)[None]
    y = torch.arange(ng)[None]
    if value:
        r, p = dim // 4, tok // 2
        code = 128 * p + 16 * ((r % 8) ^ (2 * (p % 4))) + 4 * (r // 8) + 2 * (tok % 2) + dim % 4 // 2
        centre = 1024 + 32 * ng + 2 * (16 * y + tok)
    else:
        w = dim // 8
        code = 64 * tok + 16 * (w % 4) + 4 * (w // 4) + dim % 8 // 2
        centre = 1024 + 32 * ng + 2 * (ng * tok + y)
    scale = 1024 + 2 * (ng * tok + y)
    return code, scale, centre


def pack(x, group, value):
    """x [..., 16, 128] fp32 -> tiles uint8 [..., tile]."""
    n, s, c = quantise(x, group)
    code, scale, centre = _byte_maps(group, value)
    out = torch.zeros(*x.shape[:-2], tile_bytes(group), dtype=torch.uint8)
    out[..., code[:, 0::2]] = (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8)
    for at, t in ((scale, s), (centre, c)):
        b = t.bfloat16().view(torch.uint8).unflatten(-1, (-1, 2))
        out[..., at] = b[..., 0]
        out[..., at + 1] = b[..., 1]
    return out


def unpack(tiles, group, value):
    """tiles uint8 [..., tile] -> (n - 8, s, c), each [..., 16, 128] in 64 bits."""
    code, scale, centre = _byte_maps(group, value)
    n = (tiles[..., code].int() >> (4 * (torch.arange(D) % 2))) & 15

    def half(at):
        v = tiles[..., at].int() | (tiles[..., at + 1].int() << 8)
        return (v << 16).view(torch.float32).double().repeat_interleave(group, -1)

    return (n - 8).double(), half(scale), half(centre)


def norm(x, weight, eps):
    x = x.double()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def rotate(x, cs, interleaved):
    """x [T, H, D], cs [T, R] (cosines, then sines), in x's precision."""
    R = cs.shape[1]
    cos, sin = cs[:, None, : R // 2].to(x.dtype), cs[:, None, R // 2:].to(x.dtype)
    i = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    j = i + 1 if interleaved else i + R // 2
    y = x.clone()
    y[..., i] = x[..., i] * cos - x[..., j] * sin
    y[..., j] = x[..., j] * cos + x[..., i] * sin
    return y


def places(seq_lens, cu, rows):
    """(request, position) of every row, None where it holds no token."""
    out = [None] * rows
    for b, n in enumerate(seq_lens):
        first, last = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
        for t in range(first, last):
            pos = n - (last - t)
            if pos >= 0:
                out[t] = (b, pos)
    return out


def attention(q, k, v, lens, scale):
    """q [B, Hq, 128] and per request k, v = (n - 8, s, c) [tokens, Hkv, 128]:
    (out, bound) in 64 bits; bound = sum of the weighted absolute terms."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    for b, S in enumerate(lens):
        if S == 0:
            continue
        kn, ks, kc = (t[:S] for t in k[b])
        vn, vs, vc = (t[:S] for t in v[b])
        Hkv = kn.shape[1]
        qb = q[b].double().view(Hkv, -1, D)
        x = torch.einsum("hgd,thd->hgt", qb, kn * ks + kc) * scale
        p = torch.softmax(x, -1)
        out[b] = torch.einsum("hgt,thd->hgd", p, vn * vs + vc).reshape(-1, D)
        bound[b] = torch.einsum("hgt,thd->hgd", p, (vn * vs).abs() + vc.abs()).reshape(-1, D)
    return out, bound
