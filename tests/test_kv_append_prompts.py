"""Cache appends and the 4-bit read-back with thousands of rows, as prompts
bring them: one warp then works through all the heads of a token, several
loads at a time and in several rounds, where calls of a few hundred rows give
every half warp one head.  Values are compared on the GPU with the formulas in
64 bits; the 4-bit caches byte for byte with the quantiser written in torch.

Tolerance as in test_kv_append.py: half a bf16 step of the value plus 2^-20 of
the row's largest magnitude for the fp32 operations before the rounding.
"""

import pytest
import torch

import kv4_ref as ref

EPS = 1e-6
# An append gives a token one warp where 148 * 32 rows or more than half of
# them come at once, the read-back where 148 * 64 do.
APPEND_ROWS, GATHER_ROWS = 148 * 32, 148 * 64


def _modules():
    import kv4_decode
    import kv_append

    return kv_append, kv4_decode


def _prompts(gen, rows, bs, extra_pages=3, extra_rows=5, whole=False):
    """Requests with `rows` new tokens in all, some behind a cached prefix
    (whole: none, and full pages), and extra_rows rows behind the last: block
    table, lengths, cu_seqlens and, per new token, its request and position."""
    cnt, left = [], rows
    while left > 0:
        n = min(left, int(torch.randint(1, 1200, (1,), generator=gen)))
        if whole:
            n = min(left, (n + bs - 1) // bs * bs)
        cnt.append(n)
        left -= n
    cnt.insert(1, 0)  # a request that brings nothing
    pre = [0 if whole else int(torch.randint(0, 40, (1,), generator=gen)) for _ in cnt]
    lens = [a + b for a, b in zip(cnt, pre)]
    pages = [(n + bs - 1) // bs for n in lens]
    pool = sum(pages) + extra_pages
    perm = torch.randperm(pool, generator=gen).int()
    table = torch.full((len(cnt), max(pages)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(pages):
        table[b, :m] = perm[at:at + m]
        at += m
    cu = torch.tensor([0] + cnt).cumsum(0)
    req = torch.repeat_interleave(torch.arange(len(cnt)), torch.tensor(cnt))
    pos = torch.arange(rows) - cu[req] + torch.tensor(pre)[req]
    return dict(table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(), cu=cu.int().cuda(), pool=pool,
                req=req.cuda(), pos=pos.cuda(), rows=rows + extra_rows, live=rows, longest=max(lens))


def _angles(gen, positions, rot):
    a = torch.rand(positions, rot // 2, generator=gen) * 6.28
    return torch.cat([a.cos(), a.sin()], 1).cuda()


def _slots(p, bs):
    page = p["table"][p["req"], p["pos"] // bs].long()
    return page * bs + p["pos"] % bs


def _expect(x, w, cs, pos, interleaved):
    x = x.double()
    if w is not None:
        x = ref.norm(x, w, EPS)
    return x if cs is None else _rotate(x, cs.double()[pos], interleaved)


def _rotate(x, cs, interleaved):
    R = cs.shape[1]
    cos, sin = cs[:, None, : R // 2], cs[:, None, R // 2:]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _close(got, want):
    got = got.double()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True)
    bad = (got - want).abs() > tol
    assert not bad.any(), (bad.sum(), (got - want)[bad].abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [APPEND_ROWS // 2 - 300, APPEND_ROWS + 13])
@pytest.mark.parametrize("Hq,Hkv,bs,rot,interleaved,norm,packed", [
    (64, 8, 16, 128, False, True, True),
    (64, 8, 64, 128, True, False, True),
    (32, 8, 16, 64, False, True, False),
    (9, 3, 16, 128, False, False, True),
    (9, 3, 24, 64, True, True, False),
    (7, 1, 16, 128, False, True, True),
    (7, 1, 16, 0, False, False, True),
    (5, 13, 16, 32, False, True, True),
])
def test_append_of_prompts(rows, Hq, Hkv, bs, rot, interleaved, norm, packed):
    kv_append, _ = _modules()
    gen = torch.Generator().manual_seed(rows + Hq + rot)
    p = _prompts(gen, rows, bs)
    n = p["live"]
    qkv = torch.randn(p["rows"], Hq + 2 * Hkv, 128, generator=gen).bfloat16().cuda()
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    w = [(1 + 0.2 * torch.randn(128, generator=gen)).cuda() if norm else None for _ in range(2)]
    cs = _angles(gen, p["longest"], rot) if rot else None
    kc, vc = (torch.full((p["pool"], bs, Hkv, 128), 3.0, device="cuda").bfloat16() for _ in range(2))
    args = dict(cos_sin=cs, cu_seqlens=p["cu"], interleaved=interleaved, q_weight=w[0], k_weight=w[1], eps=EPS)
    got = kv_append.gqa_append(q, k, v, kc, vc, p["table"], p["lens"], **args)
    assert kv_append.get_status(True) == 0
    _close(got[:n], _expect(q[:n], w[0], cs, p["pos"], interleaved))
    assert torch.all(got[n:] == 0)
    at = _slots(p, bs)
    _close(kc.view(-1, Hkv, 128)[at], _expect(k[:n], w[1], cs, p["pos"], interleaved))
    assert torch.equal(vc.view(-1, Hkv, 128)[at], v[:n])
    rest = torch.ones(p["pool"] * bs, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.all(kc.view(-1, Hkv, 128)[rest] == 3) and torch.all(vc.view(-1, Hkv, 128)[rest] == 3)
    # in place: the same values, rows without a token as they were
    behind = q[n:].clone()
    kv_append.gqa_append(q, k, v, kc, vc, p["table"], p["lens"], out=q, **args)
    assert torch.equal(q[:n], got[:n]) and torch.equal(q[n:], behind)
    assert kv_append.get_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,rot,interleaved", [(64, 8, 128, False), (9, 3, 128, True), (7, 1, 64, False),
                                                    (5, 13, 32, False), (8, 8, 0, False)])
def test_append_of_prompts_kv4_bytes_and_read_back(group, Hq, Hkv, rot, interleaved):
    kv_append, kv4_decode = _modules()
    gen = torch.Generator().manual_seed(group + Hq + rot)
    bs = 32
    p = _prompts(gen, (APPEND_ROWS // bs + 2) * bs, bs, whole=True)
    n = p["live"]
    qkv = torch.randn(p["rows"], Hq + 2 * Hkv, 128, generator=gen).bfloat16().cuda()
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    cs = _angles(gen, p["longest"], rot) if rot else None
    kc, vc = kv4_decode.new_cache(p["pool"], bs, Hkv, group)
    kc.fill_(7), vc.fill_(7)
    got = kv_append.gqa_append_kv4(q, k, v, kc, vc, p["table"], p["lens"], cs, p["cu"], interleaved=interleaved)
    assert kv_append.get_status(True) == 0
    _close(got[:n], _expect(q[:n], None, cs, p["pos"], interleaved))
    assert torch.all(got[n:] == 0)
    at = _slots(p, bs).cpu()
    pages = p["table"][p["req"], p["pos"] // bs].unique().long().cpu()
    other = torch.ones(p["pool"], dtype=torch.bool)
    other[pages] = False
    x = k[:n].float()
    if rot:
        # fp32 products and sums one by one, as the kernel rounds them
        x = _rotate(x, cs[p["pos"]], interleaved)
    for cache, rows, value in ((kc, x, False), (vc, v[:n].float(), True)):
        flat = torch.zeros(p["pool"] * bs, Hkv, 128)
        flat[at] = rows.cpu()
        tiles = flat.view(p["pool"], bs // 16, 16, Hkv, 128).transpose(2, 3)[pages]
        assert torch.equal(cache.cpu()[pages], ref.pack(tiles, group, value))
        assert torch.all(cache.cpu()[other] == 7)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hkv", [8, 3, 13])
def test_read_back_of_prompts(group, Hkv):
    _, kv4_decode = _modules()
    gen = torch.Generator().manual_seed(group + Hkv)
    p = _prompts(gen, GATHER_ROWS + 5, 16)
    n = p["live"]
    at = _slots(p, 16).cpu()
    caches, wants = [], []
    for value in (False, True):
        x = torch.randn(p["pool"], 1, Hkv, 16, 128, generator=gen) + torch.randn(Hkv, 1, 128, generator=gen)
        tiles = ref.pack(x, group, value)
        s8, s, c = (t[:, 0].transpose(1, 2).reshape(-1, Hkv, 128) for t in ref.unpack(tiles, group, value))
        caches.append(tiles.cuda())
        wants.append((s8 * s + c)[at].float().bfloat16())
    got = kv4_decode.gqa_gather_kv4(*caches, p["table"], p["lens"], p["cu"], p["rows"])
    assert kv4_decode.get_status(True) == 0
    for g, w in zip(got, wants):
        assert torch.equal(g[:n].cpu(), w) and torch.all(g[n:] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [APPEND_ROWS // 3, APPEND_ROWS + 13])
@pytest.mark.parametrize("h,interleaved,norm", [(128, True, True), (24, False, True), (37, True, False)])
def test_mla_append_of_prompts(rows, h, interleaved, norm):
    kv_append, _ = _modules()
    gen = torch.Generator().manual_seed(rows + h)
    p = _prompts(gen, rows, 64)
    n = p["live"]
    both = torch.randn(p["rows"], 576, generator=gen).bfloat16().cuda()
    q = torch.randn(p["rows"], h, 192, generator=gen).bfloat16().cuda()
    w = (1 + 0.2 * torch.randn(512, generator=gen)).bfloat16().cuda() if norm else None
    cs = _angles(gen, p["longest"], 64)
    cache = torch.full((p["pool"], 64, 1, 576), 3.0, device="cuda").bfloat16()
    args = dict(cu_seqlens=p["cu"], interleaved=interleaved, kv_weight=w, eps=EPS)
    q_pe = q[..., 128:]
    got = kv_append.mla_append(both[:, :512], both[:, 512:], cache, p["table"], p["lens"], cs, q_pe=q_pe, **args)
    assert kv_append.get_status(True) == 0
    _close(got[:n], _expect(q_pe[:n], None, cs, p["pos"], interleaved))
    assert torch.all(got[n:] == 0)
    at = _slots(p, 64)
    rows_of = cache.view(-1, 576)
    _close(rows_of[at, :512], _expect(both[:n, :512], w, None, None, False))
    _close(rows_of[at, 512:], _expect(both[:n, None, 512:], None, cs, p["pos"], interleaved)[:, 0])
    rest = torch.ones(p["pool"] * 64, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.all(rows_of[rest] == 3)
    nope, behind = q[..., :128].clone(), q_pe[n:].clone()
    kv_append.mla_append(both[:, :512], both[:, 512:], cache, p["table"], p["lens"], cs, q_pe=q_pe, out=q_pe, **args)
    assert torch.equal(q_pe[:n], got[:n]) and torch.equal(q_pe[n:], behind) and torch.equal(q[..., :128], nope)
