"""4-bit GQA decode where a warp works through many units of one row: the V
sums are folded in mid-row and the softmax reference moves over sums that
already count, neither of which a row cut into short parts reaches.  Each test
first asserts, from the schedule replayed here, that its longest segments pass
the fold; requests share their pages, so that the cache stays small.

Roundings of the kernel, half a step each, relative to what they round: the
output to bf16, 2^-8; the softmax weight that meets V's centre to bf16, 2^-8;
the weight times V's scale to fp16, 2^-11; q - q' / 16 of the q values at dims
2 and 6 of every eight to fp16, 2^-11, and a q below 2^-13 of its head's
largest to a step of 2^-20 of that; the sums of q that meet centres and -8 s to
two bf16 parts, 2^-17; ex2.approx, 2^-22.  Sums are fp32, except that a product
of subnormal codes drops what lies below 2^-15 of a code's step, times the
largest weight and scale of its 16 tokens, from each of 17 terms: with weights
that differ little within a tile only from the running sum, 2^-21 of a tile's
share of the bound, else at most 2^-11 of its largest weight times scale.
"""

import pytest
import torch

import kv4_ref as ref

SCALE = 128 ** -0.5
UNIT, SLACK, FOLD = 4, 6, 8  # tiles of a warp's unit, extra places of a row per warp, units to a fold


def _plan(Hq, Hkv):
    """How q heads map to warps: rows per request, and warps that share a row's units."""
    cols = (Hq // Hkv + 7) // 8
    parts = (cols + 7) // 8
    NT = (cols + parts - 1) // parts
    most, HG, TS = max((d * (8 // (d * NT)), d, 8 // (d * NT)) for d in range(1, Hkv + 1)
                       if Hkv % d == 0 and d * NT <= 8)
    return Hkv // HG * parts, TS


def _segments(tiles, Hq, Hkv, sms):
    """Tiles of every segment of the schedule, and tiles of one chunk (a unit for
    each of a row's warps), for requests of the given numbers of tiles."""
    NHG, TS = _plan(Hq, Hkv)
    rows = [t for t in tiles for _ in range(NHG)]
    spare, total = sms - len(rows), sum(rows)
    if spare > 0:  # a few requests: parts of u tiles, one per CTA
        u = max(UNIT, (total + spare - 1) // spare)
        if u * sms <= total + SLACK * sms:
            return [min(u, t - at) for t in rows for at in range(0, t, u)], UNIT * TS
    pad = SLACK * TS
    T = sum(t + pad for t in rows if t)
    E = max(1, min(sms, T // 2))
    out, first = [], 0
    for t in rows:
        if not t:
            continue
        lo, hi = first + pad, first + pad + t
        for c in range(lo * E // T, min(E, hi * E // T + 1)):
            n = min(hi, (c + 1) * T // E if c + 1 < E else T) - max(lo, c * T // E)
            if n > 0:
                out.append(n)
        first = hi
    return out, UNIT * TS


def _assert_folds(lens, Hq, Hkv):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = [(n + 15) // 16 for n in lens]
    segments, chunk = _segments(tiles, Hq, Hkv, sms)
    assert sum(segments) == sum(tiles) * _plan(Hq, Hkv)[0]
    assert max(segments) > FOLD * chunk, (max(segments), chunk)


def _shared(k, v, B, group, seed):
    """Caches of one request's tokens k and v [S, Hkv, 128] (blocks of 64 in
    random order, what lies behind the last token 0xFF), the table that gives
    them to B requests, and what the codes stand for, [S, Hkv, 128] each."""
    S, Hkv, _ = k.shape
    blocks = (S + 63) // 64
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
    caches, parts = [], []
    for value, x in ((False, k), (True, v)):
        full = torch.zeros(blocks * 64, Hkv, 128)
        full[:S] = x
        tiles = ref.pack(full.view(blocks, 4, 16, Hkv, 128).transpose(2, 3), group, value)
        parts.append(tuple(t.transpose(2, 3).reshape(-1, Hkv, 128)[:S] for t in ref.unpack(tiles, group, value)))
        code, scale, centre = ref._byte_maps(group, value)
        for tok in range(S, blocks * 64):
            t, i = tiles[tok // 64, tok % 64 // 16], tok % 16
            t[:, code[i].unique()] = 0xFF
            for m in (scale, centre):
                t[:, m[i]] = 0xFF
                t[:, m[i] + 1] = 0xFF
        cache = torch.empty_like(tiles)
        cache[order] = tiles
        caches.append(cache.cuda())
    table = order.int()[None].expand(B, -1).contiguous().cuda()
    return caches, table, parts


def _attend(q, parts, lens, scale):
    """Attention in 64 bits on the GPU: the output; the weighted sums of
    |s (n - 8)| + |c|; the root of the summed squares of both, weighted; and
    what the scores' roundings may move the output by."""
    (kn, ks, kc), (vn, vs, vc) = ([t.cuda() for t in p] for p in parts)
    Hkv = kn.shape[1]
    out, bound, rms, moved = ([] for _ in range(4))
    for b, S in enumerate(lens):
        qb = q[b].double().view(Hkv, -1, 128)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", qb, (kn * ks + kc)[:S]) * scale, -1)
        f = (vn * vs)[:S]
        y = torch.einsum("hgt,thd->hgd", p, f + vc[:S])
        out.append(y.flatten(0, 1))
        # a score's error: 2^-11 |q - q' / 16| on the codes of dims 2 and 6 of
        # every eight, 2^-21 of the head's largest |q| (a power of two up) on
        # all, and 2^-16 of |q| (8 s + |c|) for the sums
        a = qb.abs()
        d = torch.zeros_like(a)
        d[..., 2::4] = 2.0 ** -11 * (a[..., 2::4] + a[..., 3::4] / 16)
        d = d + 2.0 ** -20 * a.amax(-1, keepdim=True)
        e = torch.einsum("hgd,thd->hgt", d, (kn * ks)[:S].abs())
        e = p * (e + 2.0 ** -16 * torch.einsum("hgd,thd->hgt", a, (8 * ks + kc.abs())[:S])) * abs(scale)
        moved.append((torch.einsum("hgt,thd->hgd", e, f.abs() + vc[:S].abs()) + e.sum(-1, keepdim=True) * y.abs()).flatten(0, 1))
        bound.append(torch.einsum("hgt,thd->hgd", p, f.abs() + vc[:S].abs()).flatten(0, 1))
        rms.append(torch.einsum("hgt,thd->hgd", p * p, f * f + vc[:S] * vc[:S]).sqrt().flatten(0, 1))
    return [torch.stack(t) for t in (out, bound, rms, moved)]


def _decode(q, caches, table, lens, scale):
    import kv4_decode

    got = kv4_decode.gqa_decode_kv4(q, *caches, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale)
    assert kv4_decode.get_status(True) == 0 and torch.isfinite(got).all()
    return got.double()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,B,S", [(8, 8, 160, 1600), (32, 4, 150, 3000), (8, 1, 160, 9000), (16, 1, 150, 5000),
                                        (128, 1, 160, 1600), (9, 3, 155, 4500)])
def test_the_reference_moves_over_sums_that_count(group, Hq, Hkv, B, S):
    # Plateaus of scores 0, 3.5 and 7 (in powers of two) over 3/4, 3/16 and
    # 1/16 of the tokens: with eight weights of up to 2^9 in a lane's sum, 3.5
    # more pass 2^15 and move the reference, while the first two plateaus keep
    # 7 and 19 % of the weight.  V's mean differs from plateau to plateau, so a
    # sum that is rescaled wrongly, or not at all, shows by far.
    lens = [S - b % 37 for b in range(B)]
    _assert_folds(lens, Hq, Hkv)
    gen = torch.Generator().manual_seed(group + Hq + S)
    edge = [S * 3 // 4, S * 15 // 16]
    level = (torch.arange(S) >= edge[0]).float() + (torch.arange(S) >= edge[1]).float()
    k = 0.1 * torch.randn(S, Hkv, 128, generator=gen)
    k[..., 0] += 3.5 * level[:, None]
    mean = torch.randn(3, Hkv, 128, generator=gen) * 2
    v = torch.randn(S, Hkv, 128, generator=gen) + mean[level.long()]
    caches, table, parts = _shared(k, v, B, group, seed=S)
    q = 0.1 * torch.randn(B, Hq, 128, generator=gen)
    q[..., 0] = 1.0
    q = q.bfloat16().cuda()
    scale = 0.6931471805599453
    got = _decode(q, caches, table, lens, scale)
    want, bound, _, moved = _attend(q, parts, lens, scale)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * bound + moved
    assert torch.all((got - want).abs() <= tol), ((got - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,B,S", [(32, 8, 32, 8192), (8, 1, 32, 40000), (64, 8, 70, 6001)])
def test_long_flat_rows_keep_small_sums(group, Hq, Hkv, B, S):
    # Nearly flat scores: the raw sums of codes grow with the row while what
    # remains of them is one part in about sqrt(S), so a fold that came late or
    # with a wrong factor shows.  V has a mean in some dims, none in others.
    lens = [S - b % 5 for b in range(B)]
    _assert_folds(lens, Hq, Hkv)
    gen = torch.Generator().manual_seed(group + Hq + S)
    k = 0.05 * torch.randn(S, Hkv, 128, generator=gen)
    v = torch.randn(S, Hkv, 128, generator=gen) + (torch.randn(Hkv, 128, generator=gen) * 0.05).clamp(min=0)
    caches, table, parts = _shared(k, v, B, group, seed=S)
    q = torch.randn(B, Hq, 128, generator=gen).bfloat16().cuda()
    got = _decode(q, caches, table, lens, SCALE)
    want, bound, rms, _ = _attend(q, parts, lens, SCALE)
    # Weights are rounded independently of V: each term by up to 2^-8 of itself,
    # evenly, so by 2^-8 / 3^0.5 at one standard deviation, of which six are
    # 2^-8 times 3.5.  A score's error is as independent of V and far below
    # (2^-11 of a few products of 0.05).  fp32: the raw sums of a fold's units
    # reach four times the bound's share of them and lose up to 2^-23 of
    # themselves in each of 32 products: under 2^-16.
    tol = 2.0 ** -8 * want.abs() + 3.5 * 2.0 ** -8 * rms + 2.0 ** -16 * bound
    assert torch.all((got - want).abs() <= tol), ((got - want).abs() / tol).max()


def test_replayed_schedule():
    # 32 requests of 8192 tokens on 148 SMs: shares of 112 places, 28 units of 4 tiles
    segments, chunk = _segments([512] * 32, 32, 8, 148)
    assert chunk == 4 and sum(segments) == 32 * 512 and max(segments) == 112
    # a few requests: parts, one per CTA
    segments, chunk = _segments([20, 0, 7], 32, 8, 148)
    assert segments == [4, 4, 4, 4, 4, 4, 3]
    # one kv head: eight warps share a row; 16 q heads of it: four; three kv heads: eight, a row each
    assert [_plan(*h) for h in ((8, 1), (16, 1), (9, 3), (128, 1), (32, 4))] == [(1, 8), (1, 4), (3, 8), (2, 1), (1, 2)]
