"""The 4-bit cache at the ends of its number formats, and calls that must not
pass: against the formulas in 64 bits, or bit for bit."""

import pytest
import torch

import kv4_ref as ref


def _modules():
    import kv4_decode
    import kv_append

    return kv_append, kv4_decode


@pytest.mark.gpu
def test_codes_of_zero_cancel_for_q_values_that_fp16_rounds():
    # K is 0 wherever q is not (codes 8, centre 0; the groups' outliers meet a
    # zero of q), so every score is 0 whatever the scale, and with V = +1 and
    # -1 in turn every output is 0.  q holds values far below its head's
    # largest, which lose bits where the kernel takes q, q / 16 and q - q' / 16
    # to fp16: what is taken off for the codes' offset has to be the sum of the
    # rounded values, or a scale of 2^15 shows the difference as a score of up
    # to 1/2.
    _, kv4_decode = _modules()
    S, Hkv, group = 208, 1, 32
    k, v = torch.zeros(S, Hkv, 128), torch.ones(S, Hkv, 128)
    k[0::2, :, 16], k[0::2, :, 24] = -8.0 * 2 ** 15, 7.0 * 2 ** 15
    k[1::2, :, 16], k[1::2, :, 24] = -8.0, 7.0
    v[1::2] = -1.0
    q = torch.zeros(1, 4, 128)
    q[..., 127] = 1.0
    low = torch.tensor([2.0 ** -14 + 2.0 ** -21, 2.0 ** -14 + 2.0 ** -21, 2.0 ** -18 + 2.0 ** -25, 2.0 ** -18 + 2.0 ** -25])
    for h, dims in enumerate(([1, 5], [3, 7], [0, 4], [2, 6])):
        for o in (0, 8):
            q[0, h, [d + o for d in dims]] = low[h]
    assert torch.equal(q.bfloat16().float(), q)
    caches = [ref.pack(x.view(S // 16, 1, 16, Hkv, 128).transpose(2, 3), group, value)
              for x, value in ((k, False), (v, True))]
    kn, ks, kc = (t.transpose(2, 3).reshape(S, Hkv, 128) for t in ref.unpack(caches[0], group, False))
    assert torch.equal(kn * ks + kc, k.double())
    table = torch.arange(S // 16, dtype=torch.int32, device="cuda")[None]
    sl = torch.tensor([S], dtype=torch.int32, device="cuda")
    got = kv4_decode.gqa_decode_kv4(q.bfloat16().cuda(), *(c.cuda() for c in caches), table, sl, 1.0)
    assert kv4_decode.get_status(True) == 0
    # equal scores: equal weights, whose sum over +1 and -1 is exact
    assert got.abs().max() <= 2.0 ** -20, got.abs().amax(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_codes_of_the_smallest_and_largest_values(group):
    # groups whose scale is subnormal, just above, and near the top of the
    # range: every byte is the quantiser's, and what is read back is within half
    # a step (and c's and the output's bf16 roundings)
    kv_append, kv4_decode = _modules()
    gen = torch.Generator().manual_seed(group)
    exps = [-136, -133, -130, -127, -125, -122, -118, -110, -102, -98, -60, 0, 60, 100, 122]
    rows, Hkv = len(exps) * 16, 3
    x = torch.randn(2, len(exps), 16, Hkv, 128, generator=gen) + torch.randn(2, 1, 1, Hkv, 128, generator=gen)
    # (two factors: 2^-136 is none of fp32's normal numbers)
    half = torch.tensor([2.0 ** (e // 2) for e in exps]).view(-1, 1, 1, 1)
    rest = torch.tensor([2.0 ** (e - e // 2) for e in exps]).view(-1, 1, 1, 1)
    x = (x * half * rest).bfloat16()
    k, v = (t.reshape(rows, Hkv, 128).cuda() for t in x)
    caches = kv4_decode.new_cache(len(exps), 16, Hkv, group)
    table = torch.arange(len(exps), dtype=torch.int32, device="cuda")[None]
    sl = torch.tensor([rows], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    kv_append.gqa_append_kv4(None, k, v, *caches, table, sl, cu_seqlens=cu)
    back = kv4_decode.gqa_gather_kv4(*caches, table, sl, cu, rows)
    assert kv_append.get_status(True) == 0 and kv4_decode.get_status(True) == 0
    for cache, t, got, value in ((caches[0], x[0], back[0], False), (caches[1], x[1], back[1], True)):
        tiles = ref.pack(t.float().transpose(1, 2)[:, None], group, value)
        for i, e in enumerate(exps):
            assert torch.equal(cache[i].cpu(), tiles[i]), (value, e)
        want = t.reshape(rows, Hkv, 128).double()
        g = want.unflatten(-1, (-1, group))
        s = (g.amax(-1) - g.amin(-1)) / 15 * (1 + 2.0 ** -7) + 2.0 ** -133
        top = g.abs().amax(-1) + 2.0 ** -133
        tol = (s / 2 + 2.0 ** -7 * (top + s) + 2.0 ** -133).repeat_interleave(group, -1)
        assert torch.all((got.cpu().double() - want).abs() <= tol)


def _c_append():
    """kv_append_gqa_launch and _kv4_launch as functions of the caches' addresses
    (one row and head, 3 pages of 16 tokens); nothing is read before the refusal."""
    import ctypes

    import binding
    import test_kv_append as t

    lib = ctypes.CDLL(binding.LIB_PATH)
    P, L, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int
    head = [P, P, t._Heads, t._Heads, t._Heads, t._Norm, t._Norm, P, L, L, I, P, P, I, I]
    lib.kv_append_gqa_launch.argtypes = head + [P]
    lib.kv_append_gqa_kv4_launch.argtypes = head + [I, P]
    ok = 4096
    tok = t._Tokens(block_table=ok, seq_lens=ok, rows=1, batch=1, max_blocks=1, num_blocks=3, block_size=16)
    rope = t._Rope(table=None)
    row = t._Heads(data=ok, token_stride=128, head_stride=128)
    args = [ctypes.byref(tok), ctypes.byref(rope), t._Heads(None, 0, 0), row, row, t._Norm(None, 0, 0.0),
            t._Norm(None, 0, 0.0), None, 0, 0, 0]
    return (lambda k, v: lib.kv_append_gqa_launch(*args, k, v, 0, 1, None),
            lambda k, v: lib.kv_append_gqa_kv4_launch(*args, k, v, 0, 1, 64, None))


def test_c_appends_refuse_caches_that_overlap():
    bf16, kv4 = _c_append()
    at = 1 << 20
    for call, size in ((bf16, 3 * 16 * 256), (kv4, 3 * 1152)):
        for k, v in ((at, at), (at, at + 16), (at + size - 16, at), (at, at + size - 16)):
            assert call(k, v) == 1, (k, v)  # cudaErrorInvalidValue


@pytest.mark.gpu
def test_caches_and_outputs_that_overlap_are_refused():
    kv_append, kv4_decode = _modules()
    pages = torch.zeros(6, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    tiles = torch.zeros(6, 1, 2, 1152, dtype=torch.uint8, device="cuda")
    x = torch.ones(2, 2, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    sl = torch.ones(2, dtype=torch.int32, device="cuda")
    for call, c in ((kv_append.gqa_append, pages), (kv_append.gqa_append_kv4, tiles)):
        for k, v in ((c, c), (c[:4], c[2:]), (c[3:], c[1:4])):
            with pytest.raises(RuntimeError, match="k_cache must not overlap v_cache"):
                call(None, x, x, k, v, table, sl)
        call(None, x, x, c[:3], c[3:], table, sl)  # neighbours in one buffer
        assert torch.any(c[0] != 0) and torch.any(c[3] != 0)
    assert torch.equal(pages[0, 0], x[0]) and torch.equal(pages[4, 0], x[1])
    assert not pages[2].any() and not pages[5].any() and not tiles[2].any() and not tiles[5].any()
    inside = pages.view(-1, 2, 128)[:2]
    with pytest.raises(RuntimeError, match="out must not overlap k_cache"):
        kv_append.gqa_append(x, x, x, pages[:3], pages[3:], table, sl, out=inside)
    with pytest.raises(RuntimeError, match="out must not overlap v_cache"):
        kv_append.gqa_append(x, x, x, pages[3:], pages[:3], table, sl, out=inside)
    inside = tiles.view(torch.bfloat16).flatten()[:512].view(2, 2, 128)
    for k, v, name in ((tiles[:3], tiles[3:], "k_cache"), (tiles[3:], tiles[:3], "v_cache")):
        with pytest.raises(RuntimeError, match="out must not overlap " + name):
            kv4_decode.gqa_decode_kv4(x, k, v, table, sl, 1.0, out=inside)
    latent = torch.zeros(2, 64, 1, 576, dtype=torch.bfloat16, device="cuda")
    q = torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="out must not overlap kv_cache"):
        kv_append.mla_append(torch.ones(2, 512, device="cuda").bfloat16(), q[:, 0], latent, table, sl, q_pe=q,
                             out=latent.flatten()[:256].view(2, 2, 64))
    assert kv_append.get_status(True) == 0 and kv4_decode.get_status(True) == 0


def test_read_back_refuses_rows_that_it_would_not_return():
    _, kv4_decode = _modules()
    k, v = kv4_decode.new_cache(2, 16, 1, device="cpu")
    table, sl = torch.zeros(2, 1).int(), torch.ones(2).int()
    with pytest.raises(ValueError, match="one row per request"):
        kv4_decode.gqa_gather_kv4(k, v, table, sl, rows=3)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):  # the right number passes on
        kv4_decode.gqa_gather_kv4(k, v, table, sl, rows=2)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(65, 1), (100, 1), (146, 2), (127, 1)])
def test_groups_of_q_heads_cut_into_unequal_parts(Hq, Hkv):
    # more than 64 q heads per kv head are two rows of the schedule, the second
    # with fewer heads, down to warps that have none
    import test_kv4_decode as t

    for lens in ([1, 0, 40, 300], [900, 17] * 80):
        c = t._case(lens, Hq, Hkv, 16, 64, seed=Hq + len(lens))
        t._check(c, lens, t._run(c, lens))


@pytest.mark.gpu
def test_outputs_that_overlap_between_strides_are_refused():
    # slices of one projection whose bounds interleave: refused where heads
    # share memory, taken where they only lie between one another
    kv_append, _ = _modules()
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda")
    sl = torch.ones(3, dtype=torch.int32, device="cuda")
    kc, vc = torch.zeros(2, 3, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    cs = kv_append.rope_cos_sin(4, 128)
    qkv = torch.randn(3, 16, 128, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:8]

    def call(out, q=q):
        return kv_append.gqa_append(q, k, v, kc, vc, table, sl, cs, out=out)

    for out, what in ((qkv[:, 1:5], "q"), (qkv[:, 5:9], "k"), (qkv[:, 7:11], "v"),
                      (qkv.flatten()[4 * 128 - 8:].as_strided((3, 4, 128), (2048, 128, 1)), "q"),
                      (qkv.as_strided((3, 4, 128), (2048, 64, 1), 8 * 128), "memory"),
                      (qkv.as_strided((3, 4, 128), (384, 128, 1), 8 * 128), "memory"),
                      (qkv.as_strided((3, 4, 128), (8, 512, 1), 8 * 128), "memory")):
        before = qkv.clone()
        with pytest.raises(RuntimeError, match="overlap " + what if what != "memory" else "share memory"):
            call(out)
        assert torch.equal(qkv, before)
    want = call(None)
    row = torch.zeros(3, 5, 128, dtype=torch.bfloat16, device="cuda")
    for out in (qkv[:, 8:12], qkv[:, 8:16:2], row[:, 1:], torch.zeros(4, 3, 128, device="cuda").bfloat16().transpose(0, 1),
                torch.zeros(3000, device="cuda").bfloat16().as_strided((3, 4, 128), (640, 256, 1))):
        assert torch.equal(call(out), want)
    assert torch.equal(call(q.clone()), want)
    assert torch.equal(call(q), want)  # in place, last: q is rotated now
    latent = torch.zeros(3, 64, 1, 576, dtype=torch.bfloat16, device="cuda")
    full = torch.randn(3, 2, 192, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    args = (torch.ones(3, 512, device="cuda").bfloat16(), torch.ones(3, 64, device="cuda").bfloat16(), latent, table, sl)
    with pytest.raises(RuntimeError, match="overlap q"):
        kv_append.mla_append(*args, q_pe=full[..., 64:128], out=full[..., 72:136])
    kv_append.mla_append(*args, q_pe=full[..., 64:128], out=full[..., 128:])
    assert torch.equal(full[..., 128:], full[..., 64:128])  # no table: a copy
    assert kv_append.get_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_a_heavy_token_of_zeros_costs_little_of_the_others(group):
    # One token takes nearly all the weight and its V is 0 (codes 8, centre 0,
    # scale 1): 8 p s comes and goes in the sums, from which each product may
    # drop 2^-15 of its tile's largest p s per term, 17 terms.  The other tokens
    # of V's output, far smaller, are right to that.
    _, kv4_decode = _modules()
    S, Hkv, heavy = 176, 2, 70
    gen = torch.Generator().manual_seed(group)
    k = 0.1 * torch.randn(S, Hkv, 128, generator=gen)
    k[heavy, :, 0] = 8.0
    v = torch.randn(S, Hkv, 128, generator=gen)
    v[heavy] = 0.0
    v[heavy, :, 0::group], v[heavy, :, 1::group] = -8.0, 7.0
    caches = [ref.pack(x.view(S // 16, 1, 16, Hkv, 128).transpose(2, 3), group, value)
              for x, value in ((k, False), (v, True))]
    (kn, ks, kc), (vn, vs, vc) = ([t.transpose(2, 3).reshape(S, Hkv, 128) for t in ref.unpack(c, group, value)]
                                  for c, value in zip(caches, (False, True)))
    q = 0.05 * torch.randn(1, 8, 128, generator=gen)
    q[..., 0] = 1.0
    q = q.bfloat16()
    table = torch.arange(S // 16, dtype=torch.int32, device="cuda")[None]
    sl = torch.tensor([S], dtype=torch.int32, device="cuda")
    got = kv4_decode.gqa_decode_kv4(q.cuda(), *(c.cuda() for c in caches), table, sl, 1.0).cpu().double()[0]
    assert kv4_decode.get_status(True) == 0
    a = q.double().view(Hkv, 4, 128)
    p = torch.softmax(torch.einsum("hgd,thd->hgt", a, kn * ks + kc), -1)
    assert p[..., heavy].min() > 0.9
    want = torch.einsum("hgt,thd->hgd", p, vn * vs + vc).reshape(8, 128)
    bound = torch.einsum("hgt,thd->hgd", p, (vn * vs).abs() + vc.abs()).reshape(8, 128)
    # a score's error: 2^-11 of the q that meet dims 2 and 6 of eight, 2^-11 of
    # the largest q per product of 16 dims, eight of them, and 2^-16 for the sums
    d = torch.zeros_like(a)
    d[..., 2::4] = 2.0 ** -11 * (a[..., 2::4].abs() + a[..., 3::4].abs() / 16)
    e = torch.einsum("hgd,thd->hgt", d, (kn * ks).abs()) + 2.0 ** -8 * a.abs().amax(-1, keepdim=True) * ks.amax(-1).T[:, None]
    e = p * (e + 2.0 ** -16 * torch.einsum("hgd,thd->hgt", a.abs(), 8 * ks + kc.abs()))
    moved = torch.einsum("hgt,thd->hgd", e, (vn * vs).abs() + vc.abs()).reshape(8, 128) + e.sum(-1).reshape(8, 1) * want.abs()
    drop = (p[:, :, None] * vs.permute(1, 2, 0)[:, None]).unflatten(-1, (-1, 16)).amax(-1).sum(-1).reshape(8, 128)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * bound + moved + 2.0 ** -11 * drop
    assert torch.all((got - want).abs() <= tol), ((got - want).abs() / tol).max()
