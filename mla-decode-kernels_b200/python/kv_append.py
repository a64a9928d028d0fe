"""Filling the paged caches on B200: the step before every decode.

    q = gqa_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin)
    out = binding.gqa_decode(q, k_cache, v_cache, block_table, seq_lens, scale)

One kernel norms every q and k head (optional), rotates it by its token's
position (optional) and writes K and V to the pages of block_table:
gqa_append for K1's bf16 caches, gqa_append_kv4 for the 4-bit caches of
kv4_decode.py, mla_append for the latent cache of mla_decode.py.

Tokens.  Rows of q, k and v are tokens.  Without cu_seqlens row b is the one
new token of request b (a decode step); with cu_seqlens [B + 1] int32 request
b's new tokens are the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (prompts,
chunks, several tokens per step).  seq_lens [B] int32 counts each request's
tokens after the append, the value the decode takes, so request b's last row
goes to position seq_lens[b] - 1.  Rows behind the last request and rows at
negative positions (padding: seq_lens[b] == 0) hold no token: the caches are
left alone, their rows of a new output are zero, those of an `out` that was
passed in stay as they were.  No two rows of a call may go to the same slot.

Rotation.  cos_sin [positions, rotary_dim] fp32 (rope_cos_sin) rotates the
first rotary_dim dims of every head, in the pairs (j, j + rotary_dim / 2) or,
interleaved, (2 j, 2 j + 1); positions [rows] int32 replaces the cache
positions as its index.  None: no rotation.

q, k and v may be strided views (slices of one projection's output): last dim
contiguous, other strides multiples of 8 elements, 16-byte aligned.  Launches
go to the current stream without a synchronisation and can be captured.
The reference has no counterpart (its benchmarks fill the caches with random
data, bench/common.py:16-46).
"""

import math

import torch

from binding import _ext


def rope_cos_sin(positions, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """Rotation table [positions, rotary_dim] fp32: row p holds the cosines, then
    the sines, of p * f_j, j < rotary_dim / 2, f_j = base^(-2 j / rotary_dim),
    the angles taken in 64 bits.

    scaling stretches the table for contexts longer than trained for, a dict
    with "type" and "factor" (how many times longer):
      "linear"  f_j / factor
      "base"    base grown by factor^(rotary_dim / (rotary_dim - 2)), so that
                the slowest angle is divided by factor and the fastest kept
      "bands"   angles with a wavelength under original / high are kept, over
                original / low divided by factor, linear in between; keys
                original (trained positions), low (1.0), high (4.0)
      "yarn"    f_j up to the angle that makes fast (32.0) turns in `original`
                positions, f_j / factor from the one that makes slow (1.0), and
                linear in j between those two (rounded down and up, as trained
                models' tables are); cosines and sines are multiplied by
                attention (0.1 ln(factor) + 1).  The method is Peng et al.,
                "YaRN: Efficient Context Window Extension of Large Language
                Models", 2023
    """
    if rotary_dim < 16 or rotary_dim > 128 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16 up to 128")
    if positions < 1:
        raise ValueError("the table needs a position")
    j = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    gain = 1.0
    kind = scaling["type"] if scaling else None
    factor = float(scaling["factor"]) if scaling else 1.0
    if factor < 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(base) ** (-j / rotary_dim)
    if kind == "linear":
        f = f / factor
    elif kind == "bands":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not high > low:
            raise ValueError("bands needs high > low")
        turns = scaling["original"] * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    elif kind == "yarn":
        slow, fast = float(scaling.get("slow", 1.0)), float(scaling.get("fast", 32.0))
        if not fast > slow:
            raise ValueError("yarn needs fast > slow")
        # the (fractional) index of the angle that makes n turns
        at = [rotary_dim * math.log(scaling["original"] / (n * 2 * math.pi)) / (2 * math.log(base))
              for n in (fast, slow)]
        first = max(math.floor(at[0]), 0)
        last = min(math.ceil(at[1]), rotary_dim - 1)
        ramp = ((j / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
        f = f * (1 - ramp + ramp / factor)
        gain = float(scaling.get("attention", 0.1 * math.log(factor) + 1.0))
    elif kind not in (None, "base"):
        raise ValueError(f"unknown scaling type {kind!r}")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return (torch.cat([angle.cos(), angle.sin()], 1) * gain).float()


def gqa_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin=None, cu_seqlens=None,
               positions=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6, out=None):
    """Norm, rotate and append to bf16 caches; returns the normed and rotated q.

    q [rows, Hq, 128] (None: only K and V are handled, None is returned), k and
    v [rows, Hkv, 128] bf16, caches [num_blocks, block_size, Hkv, 128] bf16;
    q_weight and k_weight [128] bf16 or fp32 (None: no norm): y = x *
    rsqrt(mean(x^2) + eps) * weight over each head.  out may be q itself, and
    else must not overlap q, k, v or the caches, nor k_cache v_cache."""
    return _ext.gqa_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin, cu_seqlens,
                           positions, interleaved, q_weight, k_weight, eps, out, False)


def gqa_append_kv4(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin=None,
                   cu_seqlens=None, positions=None, interleaved=False, q_weight=None,
                   k_weight=None, eps=1e-6, out=None):
    """gqa_append into 4-bit caches (kv4_decode.new_cache): K, after norm and
    rotation, and V are quantised per token, head and group of dims."""
    return _ext.gqa_append(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin, cu_seqlens,
                           positions, interleaved, q_weight, k_weight, eps, out, True)


def mla_append(kv_c, k_pe, kv_cache, block_table, seq_lens, cos_sin=None, q_pe=None,
               cu_seqlens=None, positions=None, interleaved=True, kv_weight=None, eps=1e-6,
               out=None):
    """Norm the latent, rotate the position dims and append to the latent cache.

    kv_c [rows, 512] (normed with kv_weight [512]) and k_pe [rows, 64] (rotated)
    -> kv_cache [num_blocks, 64, 1, 576]; q_pe [rows, h_q, 64] -> its rotation,
    returned, written to out where given, e.g. the last 64 dims of the decode's
    q: mla_append(..., q_pe=q_pe, out=q.view(-1, h_q, 576)[..., 512:])."""
    return _ext.mla_append(kv_c, k_pe, kv_cache, block_table, seq_lens, cos_sin, q_pe, cu_seqlens,
                           positions, interleaved, kv_weight, eps, out)


get_status = _ext.kv_append_get_status
