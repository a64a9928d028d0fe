"""Cache appends (kv_append.py): head norm, rotation and the page write against
the formulas in 64 bits, every other byte of the caches unchanged.

Tolerance of a value that the kernel computes in fp32 and rounds once to bf16:
half a bf16 step, 2^-8 |want|, plus the fp32 roundings before it (at most 2^-20
of the row's largest magnitude: a few 2^-24 each for the norm's sum of 128
squares, rsqrt, two products and a sum).  What is only copied is compared bit
for bit.
"""

import ctypes
import math

import pytest
import torch

import kv4_ref as ref

EPS = 1e-6


def _modules():
    import kv4_decode
    import kv_append

    return kv_append, kv4_decode


def _pages(lens, bs, gen, extra=3):
    n = [(s + bs - 1) // bs for s in lens]
    pool = sum(n) + extra
    perm = torch.randperm(pool, generator=gen).int()
    table = torch.full((len(lens), max(1, max(n, default=1))), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(n):
        table[b, :m] = perm[at:at + m]
        at += m
    return table, pool


def _case(lens, cu, rows, Hq, Hkv, bs, rot, seed, norm=False, packed=True, wdtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    table, pool = _pages(lens, bs, gen)
    if packed:
        qkv = torch.randn(rows, Hq + 2 * Hkv, 128, generator=gen).bfloat16()
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        q, k, v = (torch.randn(rows, h, 128, generator=gen).bfloat16() for h in (Hq, Hkv, Hkv))
    w = [(1 + 0.2 * torch.randn(128, generator=gen)).to(wdtype) if norm else None for _ in range(2)]
    cs = None
    if rot:
        ang = torch.rand(max(lens, default=0) + 1, rot // 2, generator=gen) * 2 * math.pi
        cs = torch.cat([ang.cos(), ang.sin()], 1)
    return dict(q=q, k=k, v=v, table=table, pool=pool, lens=lens, cu=cu, rows=rows, bs=bs, w=w, cs=cs,
                gen=gen, Hq=Hq, Hkv=Hkv)


def _cuda_rows(c):
    """q, k, v on the GPU with the strides they have here."""
    base = c["q"]._base
    if base is not None:
        d = base.cuda()
        Hq, Hkv = c["Hq"], c["Hkv"]
        return d[:, :Hq], d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:]
    return c["q"].cuda(), c["k"].cuda(), c["v"].cuda()


def _expected(c, interleaved, positions=None):
    """Normed and rotated q and k in 64 bits, and the rows' places."""
    where = ref.places(c["lens"], c["cu"], c["rows"])
    pos = torch.tensor([w[1] if w else 0 for w in where], dtype=torch.long)
    if positions is not None:
        pos = positions.long()
    out = []
    for x, w in ((c["q"], c["w"][0]), (c["k"], c["w"][1])):
        x = x.double()
        if w is not None:
            x = ref.norm(x, w, EPS)
        if c["cs"] is not None:
            x = ref.rotate(x, c["cs"].double()[pos], interleaved)
        out.append(x)
    return out[0], out[1], where


def _close(got, want):
    got, want = got.double(), want.double()
    top = want.abs().amax(-1, keepdim=True)
    err = (got - want).abs()
    bad = err > 2.0 ** -8 * want.abs() + 2.0 ** -20 * top
    assert not bad.any(), (err[bad].max(), bad.sum())


RAGGED = dict(lens=[5, 0, 17, 64, 100], cu=[0, 5, 5, 6, 30, 99], rows=103)
STEP = dict(lens=[1, 0, 16, 17, 333, 0, 64], cu=None, rows=7)


def _args(c, dev="cuda"):
    return dict(block_table=c["table"].to(dev), seq_lens=torch.tensor(c["lens"], dtype=torch.int32, device=dev),
                cos_sin=None if c["cs"] is None else c["cs"].to(dev),
                cu_seqlens=None if c["cu"] is None else torch.tensor(c["cu"], dtype=torch.int32, device=dev),
                q_weight=None if c["w"][0] is None else c["w"][0].to(dev),
                k_weight=None if c["w"][1] is None else c["w"][1].to(dev), eps=EPS)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [RAGGED, STEP], ids=["ragged", "step"])
@pytest.mark.parametrize("Hq,Hkv,bs,rot,interleaved,norm,packed", [
    (32, 8, 16, 128, False, False, True),
    (32, 8, 16, 128, True, True, True),
    (7, 1, 64, 64, False, True, False),
    (9, 3, 1, 96, False, False, True),
    (64, 8, 24, 16, True, False, False),
    (5, 5, 128, 48, False, True, True),
    (1, 1, 16, 0, False, True, True),
    (16, 2, 16, 0, False, False, False),
])
def test_append(shape, Hq, Hkv, bs, rot, interleaved, norm, packed):
    kv_append, _ = _modules()
    c = _case(**shape, Hq=Hq, Hkv=Hkv, bs=bs, rot=rot, seed=Hq + bs + rot, norm=norm, packed=packed,
              wdtype=torch.float32 if bs == 64 else torch.bfloat16)
    kc0 = torch.randn(c["pool"], bs, Hkv, 128, generator=c["gen"]).bfloat16()
    vc0 = torch.randn(c["pool"], bs, Hkv, 128, generator=c["gen"]).bfloat16()
    kc, vc = kc0.cuda(), vc0.cuda()
    q, k, v = _cuda_rows(c)
    got = kv_append.gqa_append(q, k, v, kc, vc, interleaved=interleaved, **_args(c))
    assert kv_append.get_status(True) == 0
    wq, wk, where = _expected(c, interleaved)
    got, kc, vc = got.cpu(), kc.cpu(), vc.cpu()
    for t, w in enumerate(where):
        if w is None:
            assert torch.all(got[t] == 0)
            continue
        _close(got[t], wq[t])
        page, slot = int(c["table"][w[0], w[1] // bs]), w[1] % bs
        _close(kc[page, slot], wk[t])
        assert torch.equal(vc[page, slot], c["v"][t])
        kc[page, slot], vc[page, slot] = kc0[page, slot], vc0[page, slot]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)  # nothing else was written
    if rot == 0 and not norm:
        live = [t for t, w in enumerate(where) if w]
        assert torch.equal(got[live], c["q"][live])


@pytest.mark.gpu
def test_out_keeps_rows_without_a_token_and_may_be_q():
    kv_append, _ = _modules()
    c = _case(**RAGGED, Hq=8, Hkv=2, bs=16, rot=128, seed=3)
    kc, vc = (torch.zeros(c["pool"], 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = _cuda_rows(c)
    fresh = kv_append.gqa_append(q, k, v, kc, vc, **_args(c))
    out = torch.full((103, 2, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")[:, 1]  # strided
    assert kv_append.gqa_append(q, k, v, kc, vc, out=out, **_args(c)) is not None
    live = torch.tensor([w is not None for w in ref.places(c["lens"], c["cu"], 103)], device="cuda")
    assert torch.equal(out[live], fresh[live]) and torch.all(out[~live] == 7) and torch.all(fresh[~live] == 0)
    before = q.clone()
    kv_append.gqa_append(q, k, v, kc, vc, out=q, **_args(c))
    assert torch.equal(q[live], fresh[live]) and torch.equal(q[~live], before[~live])
    # K and V alone
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    a = _args(c)
    a.pop("q_weight")
    assert kv_append.gqa_append(None, k, v, kc2, vc2, **a) is None
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)


@pytest.mark.gpu
def test_positions_replace_the_cache_positions():
    kv_append, _ = _modules()
    c = _case(**RAGGED, Hq=4, Hkv=4, bs=16, rot=64, seed=4)
    pos = torch.randint(0, 101, (103,), generator=c["gen"]).int()
    kc, vc = (torch.zeros(c["pool"], 16, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = _cuda_rows(c)
    got = kv_append.gqa_append(q, k, v, kc, vc, positions=pos.cuda(), **_args(c))
    wq, wk, where = _expected(c, False, pos)
    for t, w in enumerate(where):
        if w:
            _close(got[t].cpu(), wq[t])
            _close(kc[int(c["table"][w[0], w[1] // 16]), w[1] % 16].cpu(), wk[t])
    assert kv_append.get_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 31, 32, 33, 1000, 1100])
def test_many_requests(B):
    # the row -> request search over batches around its 32-way steps, with
    # requests that have no rows
    kv_append, _ = _modules()
    gen = torch.Generator().manual_seed(B)
    cnt = torch.randint(0, 4, (B,), generator=gen)
    cu = [0] + cnt.cumsum(0).tolist()
    lens = (cnt + torch.randint(0, 20, (B,), generator=gen)).tolist()
    c = _case(lens, cu, cu[-1] + 2, 1, 1, 16, 16, B)
    kc, vc = (torch.zeros(c["pool"], 16, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = _cuda_rows(c)
    kv_append.gqa_append(q, k, v, kc, vc, **_args(c))
    want = torch.zeros(c["pool"], 16, 1, 128, dtype=torch.bfloat16)
    for t, w in enumerate(ref.places(lens, cu, c["rows"])):
        if w:
            want[int(c["table"][w[0], w[1] // 16]), w[1] % 16] = c["v"][t]
    assert torch.equal(vc.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [RAGGED, STEP], ids=["ragged", "step"])
@pytest.mark.parametrize("Hq,Hkv,bs,rot,interleaved", [(32, 8, 16, 128, False), (3, 3, 64, 64, True),
                                                      (4, 1, 32, 96, False), (7, 7, 16, 0, False)])
def test_append_kv4_bytes(group, shape, Hq, Hkv, bs, rot, interleaved):
    # without a norm every fp32 operation before the codes is one the host can
    # repeat: every byte of the caches is the oracle's
    kv_append, kv4_decode = _modules()
    c = _case(**shape, Hq=Hq, Hkv=Hkv, bs=bs, rot=rot, seed=group + Hq)
    c["v"][0] = 1.5  # a constant row: scale 0
    kc, vc = kv4_decode.new_cache(c["pool"], bs, Hkv, group)
    kc.random_(generator=torch.Generator("cuda").manual_seed(1))
    vc.random_(generator=torch.Generator("cuda").manual_seed(2))
    want = [kc.cpu(), vc.cpu()]
    q, k, v = _cuda_rows(c)
    got = kv_append.gqa_append_kv4(q, k, v, kc, vc, interleaved=interleaved, **_args(c))
    assert kv_append.get_status(True) == 0
    wq, _, where = _expected(c, interleaved)
    pos = torch.tensor([w[1] if w else 0 for w in where])
    x = [c["k"].float(), c["v"].float()]
    if rot:
        x[0] = ref.rotate(x[0], c["cs"][pos], interleaved)
    maps = [ref._byte_maps(group, value) for value in (False, True)]
    for t, w in enumerate(where):
        if w is None:
            assert torch.all(got[t] == 0)
            continue
        _close(got[t].cpu(), wq[t])
        page, slot = int(c["table"][w[0], w[1] // bs]), w[1] % bs
        for i in range(2):
            one = torch.zeros(Hkv, 16, 128)
            one[:, slot % 16] = x[i][t]
            tile = ref.pack(one, group, i == 1)
            for m in maps[i]:
                at = m[slot % 16].unique()
                at = torch.cat([at, at + 1]) if m is not maps[i][0] else at
                want[i][page, slot // 16][:, at] = tile[:, at]
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_append_kv4_normed_and_read_back(group):
    # after the norm a value may land on either side of a code's border: what is
    # read back is within half a step of the formula's, plus the roundings of
    # the centre and of the bf16 output (half a step of bf16 each)
    kv_append, kv4_decode = _modules()
    c = _case(**RAGGED, Hq=8, Hkv=4, bs=32, rot=128, seed=group, norm=True)
    kc, vc = kv4_decode.new_cache(c["pool"], 32, 4, group)
    q, k, v = _cuda_rows(c)
    kv_append.gqa_append_kv4(q, k, v, kc, vc, **_args(c))
    a = _args(c)
    rk, rv = kv4_decode.gqa_gather_kv4(kc, vc, a["block_table"], a["seq_lens"], a["cu_seqlens"], 103)
    assert kv_append.get_status(True) == 0 and kv4_decode.get_status(True) == 0
    _, wk, where = _expected(c, False)
    live = torch.tensor([w is not None for w in where])
    for got, want in ((rk.cpu(), wk), (rv.cpu(), c["v"].double())):
        g = want.unflatten(-1, (-1, group))
        s = (g.amax(-1) - g.amin(-1)) / 15 * (1 + 2.0 ** -7)  # rounded up to bf16
        half = (s / 2).repeat_interleave(group, -1)
        top = g.abs().amax(-1).repeat_interleave(group, -1)  # bounds |centre| up to a step
        err = (got.double() - want).abs()
        assert torch.all((err <= half * (1 + 2.0 ** -12) + 2.0 ** -7 * (top + 2 * half))[live])
        assert torch.all(got[~live] == 0)


@pytest.mark.gpu
def test_kv4_nan_and_infinity_read_back_as_nan():
    kv_append, kv4_decode = _modules()
    c = _case([1, 1, 1], None, 3, 1, 1, 16, 0, 5)
    c["v"][0, 0, 3] = float("nan")
    c["v"][1, 0, 70] = float("inf")
    c["k"][2, 0, 127] = -float("inf")
    kc, vc = kv4_decode.new_cache(c["pool"], 16, 1, 64)
    q, k, v = _cuda_rows(c)
    kv_append.gqa_append_kv4(q, k, v, kc, vc, **_args(c))
    a = _args(c)
    rk, rv = kv4_decode.gqa_gather_kv4(kc, vc, a["block_table"], a["seq_lens"])
    assert torch.isnan(rv[0, 0, :64]).all() and torch.isfinite(rv[0, 0, 64:]).all()
    assert torch.isnan(rv[1, 0, 64:]).all() and torch.isfinite(rv[1, 0, :64]).all()
    assert torch.isnan(rk[2, 0, 64:]).all() and torch.isfinite(rk[2, 0, :64]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [RAGGED, STEP], ids=["ragged", "step"])
@pytest.mark.parametrize("h,interleaved,norm,rot", [(128, True, True, True), (1, False, False, True),
                                                   (3, True, False, True), (16, False, True, False)])
def test_mla_append(shape, h, interleaved, norm, rot):
    kv_append, _ = _modules()
    gen = torch.Generator().manual_seed(h)
    lens, cu, rows = shape["lens"], shape["cu"], shape["rows"]
    table, pool = _pages(lens, 64, gen)
    kv_c = torch.randn(rows, 512, generator=gen).bfloat16()
    k_pe = torch.randn(rows, 64, generator=gen).bfloat16()
    qf = torch.randn(rows, h, 192, generator=gen).bfloat16()
    w = (1 + 0.2 * torch.randn(512, generator=gen)).bfloat16() if norm else None
    ang = torch.rand(max(lens) + 1, 32, generator=gen) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1) if rot else None
    cache0 = torch.randn(pool, 64, 1, 576, generator=gen).bfloat16()
    cache = cache0.cuda()
    qfull = torch.full((rows, h, 576), 3.0, dtype=torch.bfloat16, device="cuda")
    a = dict(cos_sin=None if cs is None else cs.cuda(),
             cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"),
             interleaved=interleaved, kv_weight=None if w is None else w.cuda(), eps=EPS)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    both = torch.cat([kv_c, k_pe], 1).cuda()  # one projection's output
    args = (both[:, :512], both[:, 512:], cache, table.cuda(), sl)
    got = kv_append.mla_append(*args, q_pe=qf.cuda()[..., 128:], **a)
    kv_append.mla_append(*args, q_pe=qf.cuda()[..., 128:], out=qfull[..., 512:], **a)
    assert kv_append.get_status(True) == 0
    where = ref.places(lens, cu, rows)
    pos = torch.tensor([x[1] if x else 0 for x in where])
    wq, wk = qf[..., 128:].double(), k_pe.double()[:, None]
    if rot:
        wq, wk = ref.rotate(wq, cs.double()[pos], interleaved), ref.rotate(wk, cs.double()[pos], interleaved)
    lat = kv_c.double() if w is None else ref.norm(kv_c, w, EPS)
    cache, got, qfull = cache.cpu(), got.cpu(), qfull.cpu()
    assert torch.all(qfull[..., :512] == 3)
    for t, x in enumerate(where):
        if x is None:
            assert torch.all(got[t] == 0) and torch.all(qfull[t] == 3)
            continue
        _close(got[t], wq[t])
        assert torch.equal(qfull[t, :, 512:], got[t])
        page, slot = int(table[x[0], x[1] // 64]), x[1] % 64
        _close(cache[page, slot, 0, :512], lat[t])
        _close(cache[page, slot, 0, 512:], wk[t, 0])
        cache[page, slot] = cache0[page, slot]
    assert torch.equal(cache, cache0)


@pytest.mark.gpu
def test_bad_pages_and_positions_are_skipped_and_reported():
    kv_append, kv4_decode = _modules()
    c = _case([20, 40, 33, 8], None, 4, 4, 2, 16, 64, 6)
    table = c["table"].clone()
    table[0, 1] = c["pool"]          # past the cache
    table[2, 2] = -1
    q, k, v = _cuda_rows(c)
    a = _args(c)
    a["block_table"] = table.cuda()
    a["seq_lens"] = torch.tensor([20, 16 * table.shape[1] + 1, 33, 8], dtype=torch.int32, device="cuda")
    a["cos_sin"] = torch.cat([a["cos_sin"], a["cos_sin"]])  # positions past the row have a table row
    for kv4 in (False, True):
        if kv4:
            kc, vc = kv4_decode.new_cache(c["pool"], 16, 2)
        else:
            kc, vc = (torch.zeros(c["pool"], 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        call = kv_append.gqa_append_kv4 if kv4 else kv_append.gqa_append
        got = call(q, k, v, kc, vc, **a)
        assert kv_append.get_status(True) == 2 | 8 and kv_append.get_status() == 0
        assert torch.all(got[1] == 0) and torch.any(got[0] != 0) and torch.any(got[2] != 0)
        page = int(c["table"][3, 0])
        used = kc.flatten(1).any(1).nonzero().flatten().tolist()
        assert used == [page]
    short = dict(a, cos_sin=a["cos_sin"][:8].contiguous(), seq_lens=torch.tensor([20, 3, 33, 8], dtype=torch.int32, device="cuda"))
    kc, vc = (torch.zeros(c["pool"], 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    got = kv_append.gqa_append(q, k, v, kc, vc, **short)  # rows 0 and 2 lie past the rotation table
    assert kv_append.get_status(True) == 8
    assert torch.all(got[0] == 0) and torch.all(got[2] == 0) and torch.any(got[3] != 0)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # pages whose byte offset passes 2^32, with a block of 64 tokens and 8 heads (128 KB)
    kv_append, _ = _modules()
    pool = (1 << 32) // (64 * 8 * 128 * 2) + 8
    kc = torch.empty(pool, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty(pool, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    kc[-1], kc[7], vc[-1], vc[7] = 0, 0, 0, 0
    x = torch.randn(1, 8, 128, device="cuda").bfloat16()
    table = torch.tensor([[pool - 1]], dtype=torch.int32, device="cuda")
    sl = torch.tensor([64], dtype=torch.int32, device="cuda")
    kv_append.gqa_append(None, x, 2 * x, kc, vc, table, sl)
    assert torch.equal(kc[-1, 63], x[0]) and torch.equal(vc[-1, 63], 2 * x[0])
    assert torch.all(kc[-1, :63] == 0) and torch.all(kc[7] == 0) and torch.all(vc[7] == 0)
    assert kv_append.get_status(True) == 0


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    kv_append, _ = _modules()
    c = _case(**STEP, Hq=8, Hkv=2, bs=16, rot=128, seed=8, norm=True)
    q, k, v = _cuda_rows(c)
    a = _args(c)
    kc, vc = (torch.zeros(c["pool"], 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    want = kv_append.gqa_append(q, k, v, kc, vc, **a)
    want_k, want_v = kc.clone(), vc.clone()
    side = torch.cuda.Stream()
    kc.zero_(), vc.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv_append.gqa_append(q, k, v, kc, vc, **a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(kc, want_k) and torch.equal(vc, want_v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kv_append.gqa_append(q, k, v, kc, vc, **a)
    kc.zero_(), vc.zero_()
    a["seq_lens"].sub_(1)  # the replay reads the lengths of the time
    g.replay()
    a["seq_lens"].add_(1)
    g.replay()
    assert torch.equal(got, want)
    rest = want_k != 0
    assert torch.equal(kc[rest], want_k[rest]) and torch.equal(vc[rest], want_v[rest])


def test_table_of_rotations():
    kv_append, _ = _modules()
    t = kv_append.rope_cos_sin(1000, 64, base=500.0, device="cpu")
    assert t.shape == (1000, 64) and t.dtype == torch.float32
    p, j = 777, 13
    ang = p * 500.0 ** (-2 * j / 64)
    assert abs(t[p, j].item() - math.cos(ang)) < 1e-6 and abs(t[p, 32 + j].item() - math.sin(ang)) < 1e-6
    # far positions: the angle itself needs 64 bits
    far = kv_append.rope_cos_sin(300000, 16, device="cpu")
    assert abs(far[299999, 0].item() - math.cos(299999.0)) < 1e-6
    lin = kv_append.rope_cos_sin(400, 64, scaling=dict(type="linear", factor=4), device="cpu")
    assert torch.allclose(lin[400 // 4 * 3], kv_append.rope_cos_sin(400, 64, device="cpu")[75], atol=1e-6)
    base = kv_append.rope_cos_sin(400, 64, scaling=dict(type="base", factor=8), device="cpu")
    plain = kv_append.rope_cos_sin(400, 64, device="cpu")
    assert torch.allclose(base[:, 0], plain[:, 0], atol=1e-6)              # the fastest angle is kept
    assert torch.allclose(base[400 - 8 * 40 - 0, 31], plain[10, 31], atol=1e-6)  # the slowest one / 8
    for kind, extra in (("bands", {}), ("yarn", dict(attention=1.0))):
        s = kv_append.rope_cos_sin(400, 64, scaling=dict(type=kind, factor=8, original=2048, **extra), device="cpu")
        assert torch.allclose(s[:, 0], plain[:, 0], atol=1e-6)
        assert torch.allclose(s[80, 31], plain[10, 31], atol=1e-6)
    y = kv_append.rope_cos_sin(4, 64, scaling=dict(type="yarn", factor=8, original=2048), device="cpu")
    assert torch.allclose(y[0, :32], torch.full((32,), 0.1 * math.log(8) + 1))
    for bad in (dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=144), dict(positions=0),
                dict(scaling=dict(type="spline", factor=2)), dict(scaling=dict(type="linear", factor=0.5))):
        with pytest.raises(ValueError):
            kv_append.rope_cos_sin(**dict(dict(positions=4, rotary_dim=64, device="cpu"), **bad))


def _cpu_args():
    q, k = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    return q, k, k.clone(), c, c.clone(), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)


def test_refuses_cpu_tensors():
    kv_append, kv4_decode = _modules()
    with pytest.raises(RuntimeError, match="k_cache must be a CUDA tensor"):
        kv_append.gqa_append(*_cpu_args())
    with pytest.raises(RuntimeError, match="k_cache must be a CUDA tensor"):
        kv_append.gqa_append_kv4(*_cpu_args())
    with pytest.raises(RuntimeError, match="kv_cache must be a CUDA tensor"):
        kv_append.mla_append(torch.zeros(1, 512).bfloat16(), torch.zeros(1, 64).bfloat16(),
                             torch.zeros(2, 64, 1, 576).bfloat16(), torch.zeros(1, 1).int(), torch.ones(1).int())


@pytest.mark.gpu
def test_refusals():
    kv_append, kv4_decode = _modules()
    good = [t.cuda() for t in _cpu_args()]

    def call(i=None, t=None, fn=kv_append.gqa_append, **kw):
        a = list(good)
        if i is not None:
            a[i] = t
        return fn(*a, **kw)

    q, k, v, kc, vc, bt, sl = good
    table = torch.zeros(4, 128, device="cuda")
    call(cos_sin=table)
    for match, kw in [
        ("bf16", dict(i=0, t=q.float())), ("bf16", dict(i=1, t=k.half())),
        ("last of size 128", dict(i=1, t=k[..., :64])), (r"\[rows, Hkv, 128\]", dict(i=2, t=v[:, :1])),
        ("same rows", dict(i=0, t=q[:1])), ("contiguous", dict(i=0, t=q.transpose(1, 2).contiguous().transpose(1, 2))),
        ("multiples of 8", dict(i=0, t=torch.zeros(2, 4, 132, device="cuda").bfloat16()[..., :128])),
        ("16-byte aligned", dict(i=0, t=torch.zeros(2 * 4 * 128 + 8, device="cuda").bfloat16()[4:-4].view(2, 4, 128))),
        ("k_cache must be", dict(i=3, t=kc.float())), ("same shape", dict(i=4, t=vc[:2])),
        ("block_table", dict(i=5, t=bt.long())), ("block_table", dict(i=5, t=bt[:1])),
        ("seq_lens", dict(i=6, t=sl.float())), ("block_table", dict(i=6, t=sl[:1].contiguous())),
        ("one row per request", dict(i=0, t=None, fn=lambda q, k, v, *r, **kw: kv_append.gqa_append(q, k[:1], v[:1], *r))),
        ("cu_seqlens", dict(cu_seqlens=torch.zeros(2, dtype=torch.int32, device="cuda"))),
        ("positions", dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda"))),
        ("positions", dict(positions=torch.zeros(2, dtype=torch.int64, device="cuda"))),
        ("rotary_dim", dict(cos_sin=torch.zeros(4, 24, device="cuda"))),
        ("rotary_dim", dict(cos_sin=torch.zeros(4, 144, device="cuda"))),
        ("cos_sin", dict(cos_sin=table.double())), ("cos_sin", dict(cos_sin=table.cpu())),
        ("q_weight", dict(q_weight=torch.ones(64, device="cuda"))),
        ("k_weight", dict(k_weight=torch.ones(128, device="cuda").half())),
        ("eps", dict(k_weight=torch.ones(128, device="cuda"), eps=-1.0)),
        ("out must have", dict(out=torch.zeros(2, 3, 128, device="cuda").bfloat16())),
        ("share memory", dict(out=torch.zeros(1, 4, 128, device="cuda").bfloat16().expand(2, 4, 128))),
        ("out and q_weight need q", dict(i=0, t=None, out=q)),
        ("k_cache must be", dict(fn=kv_append.gqa_append_kv4)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    buf = torch.zeros(6 * 4 * 128, device="cuda").bfloat16()
    out, behind = buf[:1024].view(2, 4, 128), buf[512:1024].view(2, 2, 128)
    for match, kw in [("overlap k", dict(i=1, t=behind, out=out)), ("overlap v", dict(i=2, t=behind, out=out)),
                      ("overlap q", dict(i=0, t=buf[512:1536].view(2, 4, 128), out=out)),
                      ("another view", dict(i=0, t=buf.view(6, 4, 128)[::3], out=out))]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    row = torch.zeros(1, 4, 128, device="cuda").bfloat16()  # the stride of a single row says nothing
    kv_append.gqa_append(row.as_strided((1, 4, 128), (8, 128, 1)), k[:1], v[:1], kc, vc, bt[:1], sl[:1], out=row)
    wrong = torch.zeros(3, 1, 2, 1200, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="last dim of a 4-bit cache"):
        kv_append.gqa_append_kv4(q, k, v, wrong, wrong.clone(), bt, sl)
    for bad in (dict(group=16), dict(block_size=24)):
        with pytest.raises(ValueError):
            kv4_decode.new_cache(**dict(dict(num_blocks=2, block_size=16, num_kv_heads=1), **bad))
    # no rows: nothing to do
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert kv_append.gqa_append(q[:0], k[:0], v[:0], kc, vc, bt[:0], empty).shape == (0, 4, 128)


class _Tokens(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("block_table", "seq_lens", "cu_seqlens", "positions")] + \
               [(n, ctypes.c_int) for n in ("rows", "batch", "max_blocks", "num_blocks", "block_size")]


class _Rope(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p)] + [(n, ctypes.c_int) for n in ("rotary_dim", "max_positions", "interleaved")]


class _Heads(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong)]


class _Norm(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("is_fp32", ctypes.c_int), ("eps", ctypes.c_float)]


def test_c_entry_points_refuse_before_touching_a_device():
    import binding

    lib = ctypes.CDLL(binding.LIB_PATH)
    P, L, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int
    f = lib.kv_append_gqa_kv4_launch
    f.argtypes = [P, P, _Heads, _Heads, _Heads, _Norm, _Norm, P, L, L, I, P, P, I, I, I, P]
    ok = 4096  # an aligned address that is never read

    def call(tok=None, rope=None, q=None, k=None, qw=None, out=ok, ot=512, kc=ok, Hq=4, Hkv=2, group=64):
        t = _Tokens(**dict(dict(block_table=ok, seq_lens=ok, rows=1, batch=1, max_blocks=1, num_blocks=1,
                                block_size=16), **(tok or {})))
        r = _Rope(**dict(dict(table=ok, rotary_dim=64, max_positions=8), **(rope or {})))
        h = dict(data=ok, token_stride=1024, head_stride=128)
        return f(ctypes.byref(t), ctypes.byref(r), _Heads(**dict(h, **(q or {}))), _Heads(**dict(h, **(k or {}))),
                 _Heads(**h), _Norm(qw, 0, 1e-6), _Norm(None, 0, 0.0), out, ot, 128, 0, kc, ok, Hq, Hkv, group, None)

    INVALID, MISALIGNED = 1, 716  # cudaError_t
    invalid = [dict(tok=dict(rows=-1)), dict(tok=dict(batch=2)), dict(tok=dict(max_blocks=0)),
               dict(tok=dict(num_blocks=0)), dict(tok=dict(block_size=24)), dict(tok=dict(block_table=None)),
               dict(rope=dict(rotary_dim=24)), dict(rope=dict(rotary_dim=144)), dict(rope=dict(max_positions=0)),
               dict(rope=dict(table=ok + 4)), dict(k=dict(data=None)), dict(out=None), dict(kc=None),
               dict(Hkv=0), dict(Hq=-1), dict(group=16), dict(group=0)]
    for kw in invalid:
        assert call(**kw) == INVALID, kw
    for kw in [dict(q=dict(data=ok + 2)), dict(q=dict(token_stride=4)), dict(k=dict(head_stride=132)),
               dict(qw=ok + 2), dict(out=ok + 8), dict(ot=4), dict(kc=ok + 8)]:
        assert call(**kw) == MISALIGNED, kw
    assert call(tok=dict(rows=0, batch=0)) == 0
