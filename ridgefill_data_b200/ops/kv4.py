"""A paged K/V cache held in 4 bits (csrc/kv4.cu, csrc/kv4_attention.cu): append, read back, decode attention.

pool(...)       the storage: uint8 [pages, kv_heads, page_size / 16, 20 head_dim + 32], 16 rows of one KV head a block
                (csrc/kv4.cuh describes the bytes). A cached row of one head takes 1.25 head_dim + 2 bytes for K and V
                together; bf16 takes 4 head_dim. Per 32 values: 16 steps between their smallest and largest.
append(...)     projected rows -> q / k head norm and RoPE, q rows out, K and V rows quantised into their pages
read(...)       cached rows as bf16 K / V
attention(...)  one query row of every sequence over its cached rows

A sequence is its page table: an int32 vector of page ids, cache row r being row r % page_size of page
pages[r // page_size]. `pages` is one such tensor per sequence in a list. Tables, first rows and positions live on the
device and are read by the kernels, so a CUDA graph of these calls replays at new positions; a page id outside the pool
or a row past the table records error code 7 (ops/_ext.py check_errors): append writes nothing there, read gives
zeros, attention leaves the page's rows out (a position past the table: a zero row).

Rows are independent: appending a row again overwrites it, rows not appended keep their bytes; those of a new pool are zero
rows, to read and to attention alike. A row's values are kept up to 2^56 (beyond that, or not finite, the whole row is NaN).
Outputs given to a call must share no element. Two sequences may share pages that both only read; rows that one call, or
two calls at once, append must be different rows of the pool. A sequence holds up to 2^30 rows. Head dims 64, 128 and 256.

A call works on the current stream and allocates what it needs for itself, so calls on several streams and captured graphs
share nothing but the pool.
"""
from __future__ import annotations

import torch

from ._ext import ext

BLOCK = 16       # rows of a block


def block_bytes(head_dim):
    return 20 * head_dim + 32


def supported(head_dim, hq, hkv, rot):
    """Head shapes of append and attention: head_dim 64 / 128 / 256, 1 to 8 query heads per KV head, rotary dims a
    multiple of head_dim / 16."""
    return (head_dim in (64, 128, 256) and hkv > 0 and hq % hkv == 0 and 1 <= hq // hkv <= 8 and 0 <= rot <= head_dim
            and rot % (head_dim // 16) == 0)


def pool(pages, n_kv, page_size, head_dim, device="cuda"):
    """Zeroed storage of `pages` pages of page_size rows (a multiple of 16)."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"4-bit K/V: head_dim 64, 128 or 256, not {head_dim}")
    if page_size <= 0 or page_size % BLOCK:
        raise ValueError(f"4-bit K/V: page_size {page_size}: a multiple of {BLOCK}")
    return torch.zeros(int(pages), n_kv, page_size // BLOCK, block_bytes(head_dim), dtype=torch.uint8, device=device)


def _tables(pages):
    return [pages] if torch.is_tensor(pages) else pages


def _row0(row0):
    """(device rows, host row): a tensor of first rows, or one host integer."""
    return (row0, 0) if torch.is_tensor(row0) else (None, int(row0))


def append(src, pool, pages, row0, q_heads=0, gated=False, q_norm=None, k_norm=None, norm_mode=-1, eps=1e-6,
           tables=None, rot=0, pos=None, pos_offset=-1, q_out=None):
    """Append T rows to each of R sequences: src [R * T, *] bf16 projected rows, sequence after sequence: q_heads q heads
    (each [q | gate] when gated; none when 0), then the KV heads' k, then their v. Row t of sequence r becomes cache row
    row0[r] + t (row0: int32 [R] on the device, a negative entry skips its sequence; or an int for a single sequence).
    Head norm of q and k (norm_mode -1 none, 0 plain, 1 zero-centred; weights q_norm / k_norm [head_dim]) and RoPE on
    the first rot dims at positions pos (int32 [R * T]), pos_offset + t (one sequence), or the cache row; tables (cos,
    sin) bf16 [positions, rot / 2]. Roundings as the bf16 model's; the norm's sum and root in 64 bits.
    Returns the rotated q rows [R * T, q_heads, head_dim] (q_out when given, with any row and head pitch), or None."""
    cos, sin = tables if tables is not None and rot else (None, None)
    dev, host = _row0(row0)
    return ext().kv4_append(src, pool, _tables(pages), dev, host, q_heads, gated, q_norm, k_norm, norm_mode, eps, cos, sin,
                            rot, pos, pos_offset, q_out)


def read(pool, pages, n, row0=0, out=None):
    """(k, v) bf16 [R, kv_heads, n, head_dim]: cache rows row0[r] .. row0[r] + n of every sequence (row0 as in append; a
    skipped sequence reads zeros); without the first dim when `pages` is one table instead of a list. out: (k, v) to
    write into, of equal strides."""
    k, v = out if out is not None else (None, None)
    dev, host = _row0(row0)
    return ext().kv4_read(pool, _tables(pages), dev, host, n, torch.is_tensor(pages), k, v)


def attention(q, pool, pages, pos, scale, out=None, gate=None, gate_head=0):
    """Decode attention: q [R, q_heads, head_dim] bf16, one rotated query row per sequence, over cache rows 0 .. pos[r]
    of its pages (pos int32 [R] on the device; negative: no rows, the output is zero). gate: a [R, *] view whose head h
    starts at column h * gate_head (o * sigmoid(gate)). Returns out [R, q_heads * head_dim] bf16. The keys are split
    by pos alone: a sequence gets the same bits alone or batched, whatever pages hold it."""
    return ext().kv4_attention(q, pool, _tables(pages), pos, scale, gate, gate_head, out)
