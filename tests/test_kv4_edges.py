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
