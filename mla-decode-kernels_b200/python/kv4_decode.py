"""GQA decode over a paged cache held in 4 bits, on B200.

    k_cache, v_cache = new_cache(num_blocks, block_size, Hkv)
    q = kv_append.gqa_append_kv4(q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin)
    out = gqa_decode_kv4(q, k_cache, v_cache, block_table, seq_lens, scale)

The operator is binding.gqa_decode's over caches of 0.5 + 4 / group bytes per
value instead of 2: `group` (32, 64 or 128) dims of one token and kv head
share a bf16 scale s and centre c, and a code n in 0 .. 15 stands for
s * (n - 8) + c.  include/kv4_decode.h has the quantiser and the byte layout
(16-token tiles, so block_size is a multiple of 16).  The reference has no
counterpart.  Every call allocates its own workspace from torch's allocator,
so calls on different streams and captured graphs do not share one.
"""

import torch

from binding import _ext

TILE = 16


def new_cache(num_blocks, block_size, num_kv_heads, group=64, device="cuda"):
    """(k_cache, v_cache): uint8 [num_blocks, block_size / 16, num_kv_heads, tile]."""
    tile = _ext.kv4_tile_bytes(int(group))
    if tile == 0:
        raise ValueError("group must be 32, 64 or 128")
    if block_size <= 0 or block_size % TILE:
        raise ValueError("block_size must be a multiple of 16")
    shape = (num_blocks, block_size // TILE, num_kv_heads, tile)
    return tuple(torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))


def gqa_decode_kv4(q, k_cache, v_cache, block_table, seq_lens, scale, out=None):
    """out [B, Hq, 128] bf16: softmax_t(q . K[t] * scale) @ V[t] over each
    request's first seq_lens[b] tokens (at most the block table's row), 0 for a
    request without tokens; q contiguous.  Block ids outside the cache set bit 1
    of get_status() and read block 0.  A group of the cache that holds a NaN or
    an infinity spoils all dims of its request's q heads of that kv head."""
    return _ext.gqa_decode_kv4(q, k_cache, v_cache, block_table, seq_lens, scale, out)


def gqa_gather_kv4(k_cache, v_cache, block_table, seq_lens, cu_seqlens=None, rows=None):
    """(k, v) bf16 [rows, Hkv, 128]: what the caches hold, e.g. for a prompt's
    attention over a cached prefix.  The last cu_seqlens[b + 1] - cu_seqlens[b]
    of request b's seq_lens[b] tokens go to the rows from cu_seqlens[b] on, as
    gqa_append_kv4 takes them; rows without a token are zero.  rows is the
    output's size (without cu_seqlens: one row per request, its last token)."""
    if cu_seqlens is None:
        if rows not in (None, seq_lens.shape[0]):
            raise ValueError("without cu_seqlens there is one row per request")
        rows = seq_lens.shape[0]
    elif rows is None:
        raise ValueError("rows is needed with cu_seqlens")
    return _ext.gqa_gather_kv4(k_cache, v_cache, block_table, seq_lens, cu_seqlens, rows)


get_status = _ext.kv4_get_status
