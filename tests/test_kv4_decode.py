"""GQA decode over the 4-bit cache (kv4_decode.py) against attention in 64 bits
over what the codes stand for.

Caches are random tiles; blocks no request owns, and every byte that belongs to
tokens behind a request's last one, are 0xFF (codes 15, scales and centres
NaN), so any read that reaches the output shows.

Tolerance, per output value: its own rounding to bf16 (2^-8 |out|), the bf16
rounding of the softmax weights times the scales and of the weights that
multiply the centres (2^-8 of the weighted sum of |s (n - 8)| and |c|), and
2^-10 of that sum for the scores' fp32 roundings: a score is off by at most
about 2^-20 of the sum of |q k| scale (under 2^6 here), which moves a weight
by 2^-14, and the exponential by 2^-22.
"""

import ctypes
import math

import pytest
import torch

import kv4_ref as ref

SCALE = 128 ** -0.5


def _modules():
    import kv4_decode
    import kv_append

    return kv_append, kv4_decode


def _case(lens, Hq, Hkv, bs, group, seed, k_scale=1.0):
    """(q, k_cache, v_cache, block_table, per-request k, v parts) on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    n = [(s + bs - 1) // bs for s in lens]
    pool = sum(n) + 2
    perm = torch.randperm(pool, generator=gen).int()
    table = torch.full((len(lens), max(1, max(n))), -1, dtype=torch.int32)
    tiles = {}
    parts = {}
    for value in (False, True):
        x = torch.randn(pool, bs // 16, Hkv, 16, 128, generator=gen) * (0.5 + torch.rand(Hkv, 1, 128, generator=gen))
        x = x + torch.randn(Hkv, 1, 128, generator=gen) * 0.3
        tiles[value] = ref.pack(x if value else x * k_scale, group, value)
    used = torch.zeros(pool, dtype=torch.bool)
    at = 0
    for b, m in enumerate(n):
        table[b, :m] = perm[at:at + m]
        at += m
        used[table[b, :m].long()] = True
    for value in (False, True):
        p = []
        for b, m in enumerate(n):
            t = ref.unpack(tiles[value][table[b, :m].long()], group, value)  # [m, bs/16, Hkv, 16, 128]
            p.append(tuple(z.transpose(2, 3).reshape(-1, Hkv, 128) for z in t))
        parts[value] = p
        code, scale, centre = ref._byte_maps(group, value)
        for b, (m, s) in enumerate(zip(n, lens)):
            for tok in range(s, m * bs):
                t = tiles[value][int(table[b, tok // bs]), tok % bs // 16]
                i = tok % 16
                t[:, code[i].unique()] = 0xFF
                for mp in (scale, centre):
                    t[:, mp[i]] = 0xFF
                    t[:, mp[i] + 1] = 0xFF
        tiles[value][~used] = 0xFF
    q = torch.randn(len(lens), Hq, 128, generator=gen).bfloat16()
    return q, tiles[False], tiles[True], table, parts[False], parts[True]


def _run(c, lens, **kw):
    _, kv4_decode = _modules()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = kv4_decode.gqa_decode_kv4(c[0].cuda(), c[1].cuda(), c[2].cuda(), c[3].cuda(), sl, kw.pop("scale", SCALE), **kw)
    assert kv4_decode.get_status(True) == 0
    return out.cpu()


def _check(c, lens, got, scale=SCALE):
    want, bound = ref.attention(c[0], c[4], c[5], lens, scale)
    err = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * bound
    assert torch.isfinite(got).all()
    assert torch.all(err <= tol), (err / tol.clamp(min=1e-30)).max()
    for b, s in enumerate(lens):
        if s == 0:
            assert torch.all(got[b] == 0)


LENS = [1, 0, 15, 16, 17, 31, 33, 64, 100, 257]


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,bs", [(32, 8, 16), (64, 8, 64), (8, 1, 16), (1, 1, 32), (9, 3, 48),
                                       (28, 4, 16), (18, 2, 16), (16, 1, 128), (40, 5, 16), (12, 12, 16)])
def test_heads_blocks_and_short_lengths(group, Hq, Hkv, bs):
    c = _case(LENS, Hq, Hkv, bs, group, seed=Hq + bs + group)
    _check(c, LENS, _run(c, LENS))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,bs,lens", [(32, 8, 16, [3000, 1, 777]), (8, 2, 64, [5000]), (7, 1, 16, [4099, 64]),
                                            (128, 1, 16, [1500, 3]), (33, 1, 32, [900]), (64, 16, 16, [600, 601])])
def test_rows_cut_between_ctas(group, Hq, Hkv, bs, lens):
    c = _case(lens, Hq, Hkv, bs, group, seed=len(lens) + Hq)
    _check(c, lens, _run(c, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,bs", [(8, 2, 16), (16, 1, 64)])
def test_equal_shares_that_cross_rows(Hq, Hkv, bs):
    # too many rows of too uneven lengths for one part per CTA: shares that end
    # and begin inside rows
    lens = [2500, 3, 1700, 0, 1, 2499, 800] * 6
    c = _case(lens, Hq, Hkv, bs, 64, seed=Hq)
    _check(c, lens, _run(c, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,B", [(8, 8, 160), (4, 2, 160), (1, 1, 600)])
def test_shares_that_end_at_a_row_s_start(Hq, Hkv, B):
    # rows of one tile and rows that are cut, in turn: shares that end inside
    # what a row counts for its start
    gen = torch.Generator().manual_seed(B + Hq)
    lens = [int(2 ** (10.5 * float(x))) - 1 for x in torch.rand(B, generator=gen)]
    c = _case(lens, Hq, Hkv, 16, 128, seed=B)
    _check(c, lens, _run(c, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [147, 512, 513, 700])
def test_many_short_requests(B):
    # several rows per CTA, batches on both sides of the two ways to start the
    # schedule, a third of the requests empty
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(-20, 70, (B,), generator=gen).clamp(min=0).tolist()
    c = _case(lens, 8, 2, 16, 64, seed=B)
    _check(c, lens, _run(c, lens))
    assert torch.equal(_run((c[0] * 0, *c[1:4]), [0] * B), torch.zeros(B, 8, 128, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("k_scale,scale", [(8.0, SCALE), (1.0, 2.0), (0.0, SCALE), (1.0, 0.0), (1.0, -SCALE)])
def test_peaked_and_flat_scores(k_scale, scale):
    # scores that jump by far more than the running maximum's slack, equal
    # scores (scale 0, or K all zero: groups of scale 0), and a negative scale
    lens = [2000, 33, 500]
    c = _case(lens, 16, 4, 16, 64, seed=5, k_scale=k_scale)
    got = _run(c, lens, scale=scale)
    if abs(scale) < 1 and k_scale <= 1:
        _check(c, lens, got, scale)
    else:
        # scores up to 2^10: each is off by up to 2^-20 of the sum of |q k| scale
        # (2^11), so a weight by 2^-9: four times the tolerance covers it
        want, bound = ref.attention(c[0], c[4], c[5], lens, scale)
        assert torch.all((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -6 * bound)


@pytest.mark.gpu
def test_rising_scores_move_the_maximum_often():
    # every token scores more than the one before it, by about one unit: the
    # running maximum moves at every few tiles
    lens = [1600]
    group, Hkv = 128, 2
    x = torch.zeros(100, 1, Hkv, 16, 128)
    x[..., 0] = torch.arange(1600.0).view(100, 1, 16).unsqueeze(2).expand(100, 1, Hkv, 16)
    kt = ref.pack(x, group, False)
    vt = ref.pack(torch.randn(100, 1, Hkv, 16, 128, generator=torch.Generator().manual_seed(1)), group, True)
    table = torch.arange(100, dtype=torch.int32)[None]
    q = torch.zeros(1, 4, 128)
    q[:, :, 0] = torch.tensor([1.0, -1.0, 0.25, 0.0])
    parts = [[tuple(z.transpose(2, 3).reshape(-1, Hkv, 128) for z in ref.unpack(t, group, value))]
             for t, value in ((kt, False), (vt, True))]
    c = (q.bfloat16(), kt, vt, table, parts[0], parts[1])
    got = _run(c, lens, scale=1.0)
    want, bound = ref.attention(c[0], c[4], c[5], lens, 1.0)
    # a score of up to 1600 is a sum of fp32 products: off by at most 2^-12
    assert torch.all((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * bound)


@pytest.mark.gpu
def test_long_context_stays_exact_to_the_tolerance():
    # flat scores over a long context: the sums that fp32 holds are long, the
    # output small beside the single terms
    lens = [40000]
    c = _case(lens, 4, 1, 64, 32, seed=9, k_scale=0.05)
    got = _run(c, lens)
    want, bound = ref.attention(c[0], c[4], c[5], lens, SCALE)
    err = (got.double() - want).abs()
    # random bf16 roundings of 40000 weights: 2^-9 of the terms' root mean
    # square, times 6 standard deviations, over sqrt(40000), and the output's
    rms = bound * 1.3 / 200
    assert torch.all(err <= 2.0 ** -8 * want.abs() + 6 * 2.0 ** -9 * rms + 2.0 ** -16 * bound), err.max()


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_head():
    # a scale that is infinite or NaN spoils the q heads of its request and kv
    # head; the others keep their bits
    lens = [300, 90]
    c = _case(lens, 8, 2, 16, 32, seed=10)
    clean = _run(c, lens)
    k, v = c[1].clone(), c[2].clone()
    scale = ref._byte_maps(32, True)[1]

    def poison(cache, b, tok, head, y, bits):
        tile = cache[int(c[3][b, tok // 16]), 0, head]
        tile[scale[tok % 16, y]], tile[scale[tok % 16, y] + 1] = bits & 255, bits >> 8

    poison(v, 0, 17, 0, 2, 0x7F80)   # infinity: dims 64 .. 95 of request 0, q heads 0 .. 3
    poison(k, 1, 5, 1, 3, 0x7FC0)    # NaN: request 1, q heads 4 .. 7
    got = _run((c[0], k, v, c[3]), lens)
    assert not torch.isfinite(got[0, :4, 64:96]).any() and torch.isnan(got[1, 4:]).all()
    assert torch.equal(got[0, 4:], clean[0, 4:]) and torch.equal(got[1, :4], clean[1, :4])


@pytest.mark.gpu
def test_equal_calls_give_equal_bits_and_out_is_written():
    lens = [3000, 1, 0, 700]
    c = _case(lens, 32, 8, 16, 64, seed=11)
    a = _run(c, lens)
    out = torch.full((4, 32, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    b = _run(c, lens, out=out)
    assert torch.equal(a, b) and torch.equal(out.cpu(), a)


@pytest.mark.gpu
def test_lengths_past_the_table_and_negative_ones_are_clamped():
    lens = [64, 33]
    c = _case(lens, 8, 2, 16, 64, seed=12)
    want = _run(c, lens)
    table = c[3][:, :4].contiguous()
    got = _run((c[0], c[1], c[2], table), [1000, 33])
    assert torch.equal(got, want)
    assert torch.all(_run(c, [-5, 33])[0] == 0)


@pytest.mark.gpu
def test_bad_block_ids_read_block_zero_and_are_reported():
    _, kv4_decode = _modules()
    lens = [200, 64]
    c = _case(lens, 8, 2, 16, 64, seed=13)
    k, v = c[1].clone(), c[2].clone()
    first = c[3][1, 0].long()
    k[0], v[0] = c[1][first], c[2][first]  # block 0 finite
    bad = c[3].clone()
    bad[0, 3], bad[0, 5] = len(k), -7
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = kv4_decode.gqa_decode_kv4(c[0].cuda(), k.cuda(), v.cuda(), bad.cuda(), sl, SCALE)
    assert kv4_decode.get_status(True) == 2 and kv4_decode.get_status() == 0
    bad[0, 3] = bad[0, 5] = 0
    want = kv4_decode.gqa_decode_kv4(c[0].cuda(), k.cuda(), v.cuda(), bad.cuda(), sl, SCALE)
    assert torch.equal(got, want) and torch.isfinite(got).all()


@pytest.mark.gpu
def test_captured_graphs_do_not_share_a_workspace():
    # two graphs replayed at once on two streams, and lengths that change
    # between replays
    _, kv4_decode = _modules()
    lens = [3000, 500, 0, 77]
    cs = [_case(lens, 32, 8, 16, 64, seed=14), _case(lens, 16, 2, 32, 32, seed=15)]
    wants = [_run(c, lens) for c in cs]
    runs = []
    for c in cs:
        args = [t.cuda() for t in c[:4]]
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        kv4_decode.gqa_decode_kv4(*args, sl, SCALE)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kv4_decode.gqa_decode_kv4(*args, sl, SCALE)
        runs.append((g, out, sl, args))
    for g, out, sl, _ in runs:  # other lengths first
        sl.copy_(torch.tensor([10, 0, 0, 70], dtype=torch.int32))
        g.replay()
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (g, _, _, _) in zip(streams, runs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out, _, _), want in zip(runs, wants):
        assert torch.equal(out.cpu(), want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # tiles whose byte offset passes 2^32
    _, kv4_decode = _modules()
    lens = [100, 40]
    c = _case(lens, 32, 8, 64, 64, seed=16)
    block = c[1][0].numel()
    pool = (1 << 32) // block + 10
    k, v = (torch.empty((pool, *c[1].shape[1:]), dtype=torch.uint8, device="cuda") for _ in range(2))
    n = len(c[1])
    k[-n:], v[-n:] = c[1].cuda(), c[2].cuda()
    table = torch.where(c[3] >= 0, c[3] + pool - n, c[3]).cuda()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = kv4_decode.gqa_decode_kv4(c[0].cuda(), k, v, table, sl, SCALE)
    _check(c, lens, got.cpu())
    rk, rv = kv4_decode.gqa_gather_kv4(k, v, table, sl)
    for b, s in enumerate(lens):
        for got_row, parts in ((rk[b], c[4]), (rv[b], c[5])):
            x, sc, ce = (z[s - 1] for z in parts[b])
            assert torch.equal(got_row.cpu(), (x * sc + ce).float().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("Hkv,bs", [(8, 16), (3, 64), (1, 32)])
def test_gather_reads_what_the_codes_stand_for(group, Hkv, bs):
    _, kv4_decode = _modules()
    lens, cu, rows = [5, 0, 33, 64, 100], [2, 7, 7, 8, 40, 140], 143
    c = _case(lens, Hkv, Hkv, bs, group, seed=17)
    k, v = kv4_decode.gqa_gather_kv4(c[1].cuda(), c[2].cuda(), c[3].cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                     torch.tensor(cu, dtype=torch.int32).cuda(), rows)
    assert kv4_decode.get_status(True) == 0
    for t, w in enumerate(ref.places(lens, cu, rows)):
        for got, parts in ((k[t].cpu(), c[4]), (v[t].cpu(), c[5])):
            if w is None:
                assert torch.all(got == 0)
            else:
                x, s, ce = (z[w[1]] for z in parts[w[0]])
                assert torch.equal(got, (x * s + ce).float().bfloat16())


@pytest.mark.gpu
def test_gather_reports_bad_pages_and_positions():
    _, kv4_decode = _modules()
    lens = [20, 40]
    c = _case(lens, 2, 2, 16, 64, seed=18)
    k, v = c[1].cuda(), c[2].cuda()
    sl = torch.tensor([20, 16 * c[3].shape[1] + 1], dtype=torch.int32, device="cuda")
    gk, _ = kv4_decode.gqa_gather_kv4(k, v, c[3].cuda(), sl)
    assert kv4_decode.get_status(True) == 8 and torch.all(gk[1] == 0) and torch.any(gk[0] != 0)
    bad = c[3].clone()
    bad[0, 1] = len(k)
    kv4_decode.gqa_gather_kv4(k, v, bad.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert kv4_decode.get_status(True) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("group", [None, 32, 64, 128])
def test_a_serving_run_prompts_then_steps(group):
    # prompts in uneven chunks, then decode steps with a padded batch, each
    # step appending and attending: against attention in 64 bits over what the
    # cache holds at that step
    kv_append, kv4_decode = _modules()
    import binding

    gen = torch.Generator().manual_seed(20)
    B, Hq, Hkv, bs, total = 4, 16, 4, 16, 120
    w = [(1 + 0.1 * torch.randn(128, generator=gen)).bfloat16().cuda() for _ in range(2)]
    cs = kv_append.rope_cos_sin(total, 128)
    table = torch.randperm(B * 8, generator=gen).int().view(B, 8).cuda()
    if group:
        kc, vc = kv4_decode.new_cache(B * 8, bs, Hkv, group)
        append, decode = kv_append.gqa_append_kv4, kv4_decode.gqa_decode_kv4
    else:
        kc, vc = (torch.full((B * 8, bs, Hkv, 128), float("nan"), device="cuda").bfloat16() for _ in range(2))
        append, decode = kv_append.gqa_append, binding.gqa_decode

    def step(lens, cu, rows):
        qkv = torch.randn(rows, Hq + 2 * Hkv, 128, generator=gen).bfloat16().cuda()
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
        q = append(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], kc, vc, table, sl, cs, cu_seqlens=cu,
                   q_weight=w[0], k_weight=w[1])
        return q, sl

    lens = [0] * B
    for cnt in ([50, 3, 0, 17], [7, 31, 1, 0], [0, 1, 40, 0]):
        lens = [a + b for a, b in zip(lens, cnt)]
        step(lens, [0] + torch.tensor(cnt).cumsum(0).tolist(), sum(cnt) + 2)
    live = [True, True, True, True]
    for i in range(6):
        live[2] = i != 3  # one request sits out a step
        lens = [n + 1 if on else n for n, on in zip(lens, live)]
        now = [n if on else 0 for n, on in zip(lens, live)]
        q, sl = step(now, None, B)
        got = decode(q, kc, vc, table, sl, SCALE).cpu()
        for b, n in enumerate(now):
            if n == 0:
                assert torch.all(got[b] == 0)
                continue
            blocks = table[b, : (n + bs - 1) // bs].cpu().long()
            if group:
                k, v = ([z.transpose(2, 3).reshape(-1, Hkv, 128)[:n] for z in ref.unpack(c.cpu()[blocks], group, value)]
                        for c, value in ((kc, False), (vc, True)))
            else:
                k, v = ([c.cpu()[blocks].double().reshape(-1, Hkv, 128)[:n], torch.ones(1), torch.zeros(1, 1, 1)]
                        for c in (kc, vc))
            want, bound = ref.attention(q[b:b + 1].cpu(), [k], [v], [n], SCALE)
            tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * bound
            assert torch.all((got[b:b + 1].double() - want).abs() <= tol)
    assert kv_append.get_status(True) == 0 and kv4_decode.get_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv4", [False, True])
def test_a_step_captured_with_copies_and_a_fork(kv4):
    # kernels that may be launched early behind a copy, a memset and a join of
    # two streams, all in one graph, replayed with other tokens each time
    kv_append, kv4_decode = _modules()
    import binding

    gen = torch.Generator().manual_seed(22)
    B, Hq, Hkv, bs = 40, 16, 4, 16
    lens = torch.randint(1, 400, (B,), generator=gen).int()
    table = torch.randperm(B * 26, generator=gen).int().view(B, 26).cuda()
    cs = kv_append.rope_cos_sin(401, 128)

    def caches():
        g = torch.Generator().manual_seed(23)
        if not kv4:
            return [torch.randn(B * 26, bs, Hkv, 128, generator=g).bfloat16().cuda() for _ in range(2)]
        c = kv4_decode.new_cache(B * 26, bs, Hkv)
        rows = [torch.randn(B * 400, Hkv, 128, generator=g).bfloat16().cuda() for _ in range(2)]
        kv_append.gqa_append_kv4(None, *rows, *c, table, torch.full((B,), 400, dtype=torch.int32, device="cuda"),
                                 cu_seqlens=torch.arange(0, B * 400 + 1, 400, dtype=torch.int32, device="cuda"))
        return c

    append = kv_append.gqa_append_kv4 if kv4 else kv_append.gqa_append
    decode = kv4_decode.gqa_decode_kv4 if kv4 else binding.gqa_decode
    sl = torch.zeros(B, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(B, Hq + 2 * Hkv, 128, device="cuda").bfloat16()
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    mine = caches()
    src, host_lens = torch.zeros_like(qkv), lens.cuda()
    side = torch.cuda.Stream()

    def step():
        sl.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sl.add_(host_lens)
        qkv.copy_(src)
        torch.cuda.current_stream().wait_stream(side)
        qo = append(q, k, v, *mine, table, sl, cs)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one = decode(qo, *mine, table, sl, SCALE)
        if not kv4:  # binding.gqa_decode's calls share a workspace
            torch.cuda.current_stream().wait_stream(side)
        two = decode(qo, *mine, table, sl, -SCALE)
        torch.cuda.current_stream().wait_stream(side)
        return one, two

    step()
    torch.cuda.synchronize()
    mine = [t.copy_(c) for t, c in zip(mine, caches())]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    plain = caches()
    for _ in range(4):
        rows = torch.randn(qkv.shape, generator=gen).bfloat16().cuda()
        src.copy_(rows)
        host_lens.copy_(lens)
        g.replay()
        torch.cuda.synchronize()
        qo = append(*rows.split([Hq, Hkv, Hkv], 1), *plain, table, lens.cuda(), cs)
        torch.cuda.synchronize()
        for o, s in zip(got, (SCALE, -SCALE)):
            assert torch.equal(o, decode(qo, *plain, table, lens.cuda(), s))
        lens = lens % 400 + 1


@pytest.mark.gpu
def test_a_latent_step_appends_and_attends():
    kv_append, _ = _modules()
    import mla_decode

    gen = torch.Generator().manual_seed(21)
    B, h = 3, 16
    cs = kv_append.rope_cos_sin(200, 64)
    cache = torch.full((6, 64, 1, 576), float("nan"), device="cuda").bfloat16()
    table = torch.randperm(6, generator=gen).int().view(3, 2).cuda()
    weight = torch.ones(512, device="cuda").bfloat16()

    def step(lens, cu, rows):
        q = torch.randn(rows, h, 576, generator=gen).bfloat16().cuda()
        kv = torch.randn(rows, 576, generator=gen).bfloat16().cuda()
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
        kv_append.mla_append(kv[:, :512], kv[:, 512:], cache, table, sl, cs, q_pe=q[..., 512:], cu_seqlens=cu,
                             kv_weight=weight, out=q[..., 512:])
        return q, sl

    lens = [100, 1, 63]
    step(lens, [0, 100, 101, 164], 164)
    for _ in range(3):
        lens = [n + 1 for n in lens]
        q, sl = step(lens, None, B)
        out, lse = mla_decode.mla_decode(q[:, None], cache, table, sl, 192 ** -0.5)
        for b, n in enumerate(lens):
            rows = cache[table[b].long()].reshape(-1, 576)[:n].double()
            p = torch.softmax(q[b].double() @ rows.T * 192 ** -0.5, -1)
            torch.testing.assert_close(out[b, 0].double(), p @ rows[:, :512], atol=1e-2, rtol=1e-2)
    assert kv_append.get_status(True) == 0 and mla_decode.get_status(True) == 0


@pytest.mark.gpu
def test_refusals():
    _, kv4_decode = _modules()
    q = torch.zeros(2, 8, 128, device="cuda").bfloat16()
    k, v = kv4_decode.new_cache(3, 16, 2)
    bt = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    sl = torch.ones(2, dtype=torch.int32, device="cuda")
    good = [q, k, v, bt, sl, SCALE]
    kv4_decode.gqa_decode_kv4(*good)
    for match, i, t in [("bf16", 0, q.float()), ("contiguous", 0, q.transpose(0, 1)), ("contiguous", 0, q[..., :64]),
                        ("divisible", 0, q[:, :3].contiguous()), ("at most 128", 0, torch.zeros(2, 258, 128, device="cuda").bfloat16()),
                        ("Byte|uint8", 1, k.float()), ("same shape", 2, v[:2]), ("last dim", 1, k[..., :1024].contiguous()),
                        ("block_table", 3, bt.long()), ("block_table", 3, bt[:1]), ("seq_lens", 4, sl[:1].contiguous()),
                        ("CUDA", 4, sl.cpu()), ("CUDA", 0, q.cpu())]:
        a = list(good)
        a[i] = t
        if match == "last dim":
            a[2] = t.clone()
        with pytest.raises(RuntimeError, match=match):
            kv4_decode.gqa_decode_kv4(*a)
    with pytest.raises(RuntimeError, match="out must be"):
        kv4_decode.gqa_decode_kv4(*good, out=torch.zeros(2, 8, 64, device="cuda").bfloat16())
    with pytest.raises(RuntimeError, match="must not overlap q"):
        kv4_decode.gqa_decode_kv4(*good, out=q)
    with pytest.raises(ValueError, match="rows"):
        kv4_decode.gqa_gather_kv4(k, v, bt, sl, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert kv4_decode.gqa_decode_kv4(q[:0], k, v, bt[:0], sl[:0], SCALE).shape == (0, 8, 128)
    gk, gv = kv4_decode.gqa_gather_kv4(k, v, bt[:0], sl[:0])
    assert gk.shape == gv.shape == (0, 2, 128)


def test_refuses_cpu_tensors():
    _, kv4_decode = _modules()
    k, v = kv4_decode.new_cache(2, 16, 1, device="cpu")
    assert k.shape == (2, 1, 1, 1152) and v.dtype == torch.uint8
    with pytest.raises(RuntimeError, match="k_cache must be a CUDA tensor"):
        kv4_decode.gqa_decode_kv4(torch.zeros(1, 1, 128).bfloat16(), k, v, torch.zeros(1, 1).int(), torch.ones(1).int(), 1.0)


def test_c_entry_points_refuse_before_touching_a_device():
    import binding

    lib = ctypes.CDLL(binding.LIB_PATH)
    P, I, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    lib.kv4_tile_bytes.argtypes, lib.kv4_tile_bytes.restype = [I], Z
    assert [lib.kv4_tile_bytes(g) for g in (32, 64, 128, 16, 0, -1)] == [1280, 1152, 1088, 0, 0, 0]
    f = lib.kv4_decode_launch
    f.argtypes = [P] * 6 + [I] * 7 + [F, P, Z, P]
    ok = 4096
    base = dict(q=ok, k=ok, v=ok, bt=ok, sl=ok, out=ok, B=1, Hq=4, Hkv=2, group=64, bs=16, mb=1, nb=1, scale=1.0,
                ws=ok, wsb=1 << 30, stream=None)
    for kw in [dict(B=-1), dict(Hq=3), dict(Hkv=0), dict(Hq=258), dict(group=48), dict(bs=0), dict(bs=24), dict(mb=0),
               dict(nb=0), dict(q=None), dict(v=None), dict(out=None), dict(sl=None)]:
        assert f(*dict(base, **kw).values()) == 1, kw
    for kw in [dict(q=ok + 2), dict(k=ok + 8), dict(v=ok + 4), dict(out=ok + 8)]:
        assert f(*dict(base, **kw).values()) == 716, kw
    assert f(*dict(base, B=0).values()) == 0
    g = lib.kv4_gather_launch
    g.argtypes = [P] * 7 + [I] * 7 + [P]
    base = dict(k=ok, v=ok, bt=ok, sl=ok, cu=ok, ko=ok, vo=ok, rows=1, B=1, Hkv=1, group=64, bs=16, mb=1, nb=1, stream=None)
    for kw in [dict(rows=-1), dict(B=-1), dict(Hkv=0), dict(group=1), dict(bs=8), dict(mb=0), dict(nb=0), dict(cu=None, B=2),
               dict(k=None), dict(vo=None), dict(bt=None)]:
        assert g(*dict(base, **kw).values()) == 1, kw
    assert g(*dict(base, ko=ok + 2).values()) == 716 and g(*dict(base, rows=0).values()) == 0


def test_every_declared_entry_point_is_exported():
    import os
    import re

    import binding

    lib = ctypes.CDLL(binding.LIB_PATH)
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    names = []
    for h in ("kv_append.h", "kv4_decode.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(inc, h)).read(), flags=re.S)
        names += re.findall(r"\b(kv(?:4|_append)_\w+)\s*\(", text)
    assert len(set(names)) == 9
    for n in names:
        assert hasattr(lib, n), n


def test_oracle_packs_and_unpacks():
    x = torch.randn(2, 3, 16, 128, generator=torch.Generator().manual_seed(0))
    for group in (32, 64, 128):
        n, s, c = ref.quantise(x, group)
        for value in (False, True):
            un, us, uc = ref.unpack(ref.pack(x, group, value), group, value)
            assert torch.equal(un, (n - 8).double())
            assert torch.equal(us, s.double().repeat_interleave(group, -1))
            assert torch.equal(uc, c.double().repeat_interleave(group, -1))
            assert torch.all((un * us + uc - x).abs() <= us / 2 * (1 + 1e-6) + 2.0 ** -8 * uc.abs())
    assert math.isclose(ref.tile_bytes(64), 1152)
