"""The 4-bit K/V cache on the CPU: the stored layout, the rounding error of a cached value, and the calls that the entry
points refuse (every check but the last, for a CUDA device, holds on any device)."""
import math

import pytest
import torch

from ridgefill_data_b200.ops import kv4
from ridgefill_data_b200.ops import oracle as ops


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_every_byte_of_a_block_belongs_to_one_row(hd):
    steps, halves = [], []
    for row in range(16):
        k, v, at, ke, ve = ops.kv4_places(hd, row)
        steps += k + v
        halves += [b for part in at.values() for b in part]
        halves_end = [ke, ve]
        steps += [2 * b + j for b in halves_end for j in (0, 1)]
    steps += [2 * b + j for b in halves for j in range(4)]
    assert sorted(steps) == list(range(2 * kv4.block_bytes(hd)))
    # the parts in their order, scales on 2-byte and whole blocks on 16-byte borders
    assert all(b % 2 == 0 for b in halves) and kv4.block_bytes(hd) % 32 == 0


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_fragment_loads_touch_every_bank_once(hd):
    """The attention's shared-memory loads: a K lane (g, t) reads the words of row g, a V lane chunk g of row 2t + i.
    Each phase of 32 lanes x 4 bytes, 16 x 8 or 8 x 16 covers the 32 banks once."""
    def phases(first_bytes, size):
        lanes = 128 // size
        for lo in range(0, 32, lanes):
            banks = [(b // 4 + j) % 32 for b in first_bytes[lo:lo + lanes] for j in range(size // 4)]
            assert sorted(banks) == list(range(32))
    words = hd // 32
    for half in range(max(1, words // 4)):
        for r8 in (0, 8):
            first = [min(ops.kv4_places(hd, lane // 4 + r8)[0][32 * (i + 4 * half) + 8 * (lane % 4)] // 2
                         for i in range(min(4, words))) for lane in range(32)]
            phases(first, 4 * min(4, words))
    for i in (0, 1, 8, 9):
        first = [ops.kv4_places(hd, 2 * (lane % 4) + i)[1][4 * (lane // 4)] // 2 - 8 * hd for lane in range(32)]
        phases(first, hd // 16)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_put_then_get_stands_for_the_quantised_rows(hd):
    g = torch.Generator().manual_seed(hd)
    k, v = (torch.randn(16, hd, generator=g).bfloat16() for _ in range(2))
    k[3, 5], v[4, 1] = math.inf, math.nan
    k[5], v[6] = 0.0, 3.0
    k[7] *= 1e-20
    block = torch.randint(0, 256, (kv4.block_bytes(hd),), dtype=torch.uint8, generator=g)
    for row in range(16):
        ops.kv4_put(block, row, k[row], v[row])
    gk, gv = ops.kv4_get(block[None], hd)
    for got, y in ((gk[0], k), (gv[0], v)):
        want = ops.kv4_values(*ops.kv4_quantise(y))
        assert torch.equal(got.nan_to_num(nan=7e7), want.nan_to_num(nan=7e7))
    assert gk[0, 3].isnan().all() and gv[0, 4].isnan().all()
    assert gk[0, 5].eq(0).all() and gv[0, 6].eq(3.0).all()


def test_a_cached_value_is_within_half_a_step():
    """|value - y| <= s / 2 plus fp16's roundings of m and s: m is off by at most 2^-11 |m| <= 2^-10 in z (|z| < 2), s by
    2^-11 s, over 15 steps, and 2^-25 each where they are subnormal."""
    g = torch.Generator().manual_seed(0)
    y = (torch.randn(200, 128, generator=g) * torch.exp(2 * torch.randn(200, 1, generator=g))).bfloat16()
    byte, s, m, c = ops.kv4_quantise(y)
    size = torch.pow(2.0, byte.double() - 127)[:, None, None]
    err = (ops.kv4_values(byte, s, m, c) - y.double()).abs().unflatten(-1, (-1, 32))
    bound = s.double()[..., None] * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -10 + 16 * 2.0 ** -25
    assert (err <= size * bound).all()


def _args(hd=128, hkv=2, hq=4, pages=4, page=32, T=3):
    pool = kv4.pool(pages, hkv, page, hd, "cpu")
    src = torch.zeros(T, (hq + 2 * hkv) * hd, dtype=torch.bfloat16)
    return pool, src, torch.arange(2, dtype=torch.int32)


def test_storage_is_checked():
    with pytest.raises(ValueError):
        kv4.pool(4, 2, 100, 128, "cpu")
    with pytest.raises(ValueError):
        kv4.pool(4, 2, 128, 96, "cpu")
    assert kv4.pool(3, 2, 128, 64, "cpu").shape == (3, 2, 8, 20 * 64 + 32)
    assert kv4.supported(256, 24, 4, 64) and kv4.supported(128, 32, 8, 128) and kv4.supported(64, 3, 1, 0)
    assert not kv4.supported(96, 8, 2, 0) and not kv4.supported(128, 18, 2, 0) and not kv4.supported(128, 5, 2, 0)
    assert not kv4.supported(256, 24, 4, 24) and not kv4.supported(128, 8, 2, 256)


APPEND_REFUSED = {
    "row past the table": (dict(row0=62), "rows 62"),
    "negative host row": (dict(row0=-1), "rows -1"),
    "row0 count": (dict(row0=torch.zeros(2, dtype=torch.int32)), "one row0 per sequence"),
    "row0 type": (dict(row0=torch.zeros(1, dtype=torch.int64)), "expected Int"),
    "narrow rows": (dict(q_heads=5), "k heads"),
    "norm mode": (dict(norm_mode=2), "norm_mode"),
    "norm weight missing": (dict(norm_mode=0), "norm weights"),
    "norm weight size": (dict(norm_mode=0, k_norm=torch.zeros(64).bfloat16(), q_norm=torch.zeros(128).bfloat16()),
                         "norm weights"),
    "norm eps": (dict(norm_mode=0, eps=0.0, k_norm=torch.zeros(128).bfloat16(), q_norm=torch.zeros(128).bfloat16()), "eps"),
    "rotary dims": (dict(rot=12), "rotary dims"),
    "rotary dims wide": (dict(rot=136), "rotary dims"),
    "no tables": (dict(rot=64), "RoPE tables"),
    "table width": (dict(rot=64, tables=(torch.zeros(99, 16).bfloat16(),) * 2), "RoPE tables"),
    "table type": (dict(rot=64, tables=(torch.zeros(99, 32),) * 2), "RoPE table has dtype"),
    "tables unlike": (dict(rot=64, tables=(torch.zeros(99, 32).bfloat16(), torch.zeros(98, 32).bfloat16())),
                      "RoPE tables"),
    "positions past the tables": (dict(rot=64, pos_offset=97, tables=(torch.zeros(99, 32).bfloat16(),) * 2),
                                  "positions past"),
    "pos count": (dict(pos=torch.zeros(2, dtype=torch.int32)), "one position a row"),
    "pos type": (dict(pos=torch.zeros(3, dtype=torch.int64)), "pos has dtype"),
    "q_out shape": (dict(q_out=torch.zeros(3, 4, 64).bfloat16()), "q_out"),
    "q_out pitch": (dict(q_out=torch.zeros(3, 4, 132).bfloat16()[..., :128]), "q_out"),
}


@pytest.mark.parametrize("name", APPEND_REFUSED)
def test_append_refuses(name):
    over, message = APPEND_REFUSED[name]
    pool, src, table = _args()
    kw = dict(row0=1, q_heads=4)
    kw.update(over)
    with pytest.raises((RuntimeError, ValueError), match=message):
        kv4.append(src, pool, [table], **kw)


def test_append_refuses_layouts():
    pool, src, table = _args()
    ok = dict(row0=0, q_heads=4)
    for bad, message in ((src.float(), "src has dtype"), (src[0], "rows"), (src.t().contiguous().t(), "rows"),
                         (src.repeat(1, 2)[:, 4:4 + src.shape[1]], "16-byte")):
        with pytest.raises(RuntimeError, match=message):
            kv4.append(bad, pool, [table], **ok)
    for bad, message in ((pool.float(), "uint8"), (pool[:, :, ::2], "contiguous"), (pool[..., :-1], "contiguous"),
                         (pool[0], "contiguous"), (torch.zeros(2, 2, 2, 20 * 96 + 32, dtype=torch.uint8), "head_dim"),
                         (torch.zeros(0, 2, 2, 20 * 128 + 32, dtype=torch.uint8), "empty")):
        with pytest.raises(RuntimeError, match=message):
            kv4.append(src, bad, [table], q_out=torch.zeros(3, 4, 128).bfloat16(), **ok)
    for bad, message in ((table.long(), "pages has dtype"), (table[None], "page table"),
                         (torch.zeros(4, dtype=torch.int32)[::2], "page table")):
        with pytest.raises(RuntimeError, match=message):
            kv4.append(src, pool, [bad], **ok)
    with pytest.raises(RuntimeError, match="the same number of rows"):
        kv4.append(src, pool, [table, table], torch.zeros(2, dtype=torch.int32), q_heads=4)
    with pytest.raises(RuntimeError, match="serves one sequence"):
        kv4.append(src[:2], pool, [table, table], 0, q_heads=4)
    with pytest.raises(RuntimeError, match="the same number of rows"):
        kv4.append(src, pool, [], 0, q_heads=4)
    with pytest.raises(RuntimeError, match="CUDA device"):       # everything in order but the device
        kv4.append(src, pool, [table], **ok)


def test_read_refuses():
    pool, _, table = _args()
    for n, row0, message in ((65, 0, "rows 0 .. 65"), (1, 64, "rows 64"), (1, -1, "rows -1")):
        with pytest.raises(RuntimeError, match=message):
            kv4.read(pool, table, n, row0)
    k = torch.zeros(2, 3, 128).bfloat16()
    for out in ((k, k[:, :2]), (k, k.float()), (k, torch.zeros(2, 3, 136).bfloat16()[..., :128]),
                (k, torch.zeros(3, 2, 128).bfloat16().transpose(0, 1)), (k[:, :, :64],) * 2):
        with pytest.raises(RuntimeError, match="k and v|k / v"):
            kv4.read(pool, table, 3, 0, out=out)
    with pytest.raises(RuntimeError, match="serves one sequence"):
        kv4.read(pool, [table, table], 3, 0)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv4.read(pool, table, 3, 0)


def test_refuses_numbers_at_their_ends_and_outputs_on_themselves():
    """Host numbers whose sum passes 64 bits, more heads than a launch has rows of blocks, outputs whose rows lie on each
    other."""
    pool, src, table = _args()
    last = 2 ** 63 - 1
    with pytest.raises(RuntimeError, match="rows 9223372036854775807"):
        kv4.append(src, pool, [table], last, q_heads=4)
    with pytest.raises(RuntimeError, match="rows 9223372036854775807"):
        kv4.read(pool, table, 3, last)
    with pytest.raises(RuntimeError, match="pos_offset"):
        kv4.append(src, pool, [table], 0, q_heads=4, pos_offset=last)
    with pytest.raises(RuntimeError, match="65535"):
        kv4.append(torch.empty(1, 65535 * 64).bfloat16(), torch.zeros(1, 2, 1, 20 * 64 + 32, dtype=torch.uint8),
                   [table], 0, q_heads=65532)
    one = torch.zeros(1, 4, 128).bfloat16()
    with pytest.raises(RuntimeError, match="memory location"):
        kv4.append(src, pool, [table], 0, q_heads=4, q_out=one.expand(3, 4, 128))
    with pytest.raises(RuntimeError, match="memory location"):
        kv4.read(pool, table, 3, 0, out=(torch.zeros(1, 3, 128).bfloat16().expand(2, 3, 128),) * 2)
    with pytest.raises(RuntimeError, match="memory location"):
        kv4.attention(one.expand(2, 4, 128), pool, [table, table], torch.zeros(2, dtype=torch.int32), 0.1,
                      out=torch.zeros(1, 512).bfloat16().expand(2, 512))


def test_attention_refuses():
    pool, _, table = _args()
    q, pos = torch.zeros(1, 4, 128).bfloat16(), torch.zeros(1, dtype=torch.int32)
    gate = torch.zeros(1, 4 * 256).bfloat16()
    for kw, message in ((dict(q=q.float()), "q has dtype"), (dict(q=torch.zeros(2, 4, 128).bfloat16()), "q \\[seq"),
                        (dict(q=torch.zeros(1, 4, 64).bfloat16()), "q \\[seq"),
                        (dict(q=torch.zeros(1, 3, 128).bfloat16()), "query heads"),
                        (dict(q=torch.zeros(1, 18, 128).bfloat16()), "query heads"),
                        (dict(pos=pos.long()), "pos has dtype"), (dict(pos=torch.zeros(2, dtype=torch.int32)), "position"),
                        (dict(out=torch.zeros(1, 256).bfloat16()), "out"), (dict(out=torch.zeros(1, 512)), "out"),
                        (dict(gate=gate.float()), "gate"), (dict(gate=gate, gate_head=300), "gate"),
                        (dict(gate=gate, gate_head=4), "gate"), (dict(gate=gate[:, 3:], gate_head=256), "gate")):
        args = dict(q=q, pos=pos, out=None, gate=None, gate_head=0)
        args.update(kw)
        with pytest.raises(RuntimeError, match=message):
            kv4.attention(args["q"], pool, [table], args["pos"], 0.1, out=args["out"], gate=args["gate"],
                          gate_head=args["gate_head"])
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv4.attention(q, pool, [table], pos, 0.1, gate=gate[:, 128:], gate_head=256)


def test_4_bit_pool_on_the_cpu():
    """Page bookkeeping and refusals of a pool of 4-bit pages."""
    from types import SimpleNamespace

    from ridgefill_data_b200.models.kvpool import KVPool, PoolExhausted
    model = SimpleNamespace(head_dim=128, n_kv=2, n_heads=8, layer_types=["gdn", "attn", "attn"], cfg=SimpleNamespace(rot_dim=64),
                            device=torch.device("cpu"), dtype=torch.bfloat16)
    pool = KVPool(model, pages=6, page_size=128, bits=4)
    assert pool.k is None and pool.v is None and pool.kv[1].shape == (6, 2, 8, kv4.block_bytes(128))
    assert pool.bytes() == 2 * 6 * 2 * 8 * kv4.block_bytes(128)
    entry = {}
    pool.grow(2, entry, 129, "cpu")
    assert len(entry["pages"]) == 2 and pool.free_pages(2) == 4
    with pytest.raises(PoolExhausted):
        pool.grow(2, {}, 700, "cpu")
    pool.release([{}, {}, entry])
    assert pool.free_pages(2) == 6
    for over in (dict(head_dim=96), dict(n_heads=18), dict(n_heads=7), dict(cfg=SimpleNamespace(rot_dim=20))):
        with pytest.raises(ValueError):
            KVPool(SimpleNamespace(**{**vars(model), **over}), pages=2, bits=4)
    for kw in (dict(bits=8), dict(bits=4, page_size=64), dict(bits=4, page_size=0)):
        with pytest.raises(ValueError):
            KVPool(model, pages=2, **kw)


def test_server_flag_needs_a_pool():
    from ridgefill_data_b200.serve.__main__ import main
    with pytest.raises(SystemExit):
        main(["--kv-bits", "4"])
