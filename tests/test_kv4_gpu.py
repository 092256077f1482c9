"""The 4-bit K/V cache's kernels against the fp64 oracle (ops/oracle.py): append byte for byte, read bit for bit,
attention within the arithmetic's error bound; and how they are called: ragged batches, shuffled pages, bad page ids,
captured graphs, other streams, pools past 4 GiB, stale bytes behind a sequence's end."""
import math

import pytest
import torch

from ridgefill_data_b200.ops import kernels as K
from ridgefill_data_b200.ops import kv4
from ridgefill_data_b200.ops import oracle as ops
from ridgefill_data_b200.ops._ext import check_errors, ext

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    torch.cuda.synchronize()
    check_errors()


def _error():
    """The error code the kernels recorded, cleared."""
    torch.cuda.synchronize()
    w = ext().error_word(torch.cuda.current_device())
    code = int(w.item())
    w.zero_()
    return code


def _pages(lens, page, extra=2, seed=0):
    held = [-(-n // page) for n in lens]
    total = sum(held) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return [t.to(DEV) for t in order[:sum(held)].split(held)], total


def _random_pool(total, hkv, page, hd, seed=1):
    """A pool of arbitrary bytes: what other requests left."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, 256, (total, hkv, page // 16, kv4.block_bytes(hd)), dtype=torch.uint8, device=DEV,
                         generator=g)


def _tables(n, rot, theta=1e4):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return tuple(t.bfloat16().to(DEV) for t in (ang.cos(), ang.sin()))


APPEND = [
    # hd, hkv, G, gated, norm, rot, page, row0 of each sequence, rows
    (128, 2, 4, False, 0, 128, 128, [0], 1),
    (128, 1, 1, False, -1, 0, 16, [15], 1),
    (256, 2, 6, True, 1, 64, 128, [37, 0, 255, 127], 3),
    (256, 1, 3, False, -1, 256, 32, [31], 66),
    (64, 3, 5, False, 0, 32, 48, [7, 40], 45),
    (64, 2, 4, True, 1, 64, 64, [0], 16),
    (128, 3, 0, False, 1, 64, 256, [100], 33),
    (128, 3, 5, True, 1, 64, 48, [5, 90], 70),
    (256, 3, 2, False, 0, 64, 128, [200], 80),
    (64, 5, 1, False, 1, 16, 32, [3], 100),
    (128, 2, 2, False, -1, 0, 128, [0], 64),
    # 256 rows and more
    (128, 3, 5, True, 1, 64, 48, [5, 90], 140),
    (256, 3, 2, False, 0, 64, 128, [200], 300),
    (64, 5, 1, False, 1, 32, 32, [3], 261),
    (64, 2, 8, False, 0, 64, 80, [16, 0, 9], 99),
    (128, 2, 2, False, -1, 0, 128, [0], 256),
    (256, 1, 3, False, -1, 256, 32, [31], 266),
    (256, 2, 6, True, 1, 64, 128, [130], 257),
    (128, 1, 8, False, 0, 128, 64, list(range(0, 60, 3)), 16),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append_writes_the_oracles_bytes_and_no_others(case):
    hd, hkv, G, gated, norm, rot, page, row0, T = case
    R, hq = len(row0), hkv * G
    pages, total = _pages([r + T for r in row0], page)
    pool = _random_pool(total, hkv, page, hd)
    g = torch.Generator().manual_seed(2)
    qw = hq * hd * (2 if gated else 1)
    src = (torch.randn(R * T, qw + 2 * hkv * hd + 8, generator=g) *
           torch.exp(1.5 * torch.randn(1, qw + 2 * hkv * hd + 8, generator=g))).bfloat16()
    norms = [(0.3 * torch.randn(hd, generator=g) + (norm == 0)).bfloat16() for _ in range(2)] if norm >= 0 else [None] * 2
    tables = _tables(600, rot) if rot else None
    before = pool.cpu()
    q = kv4.append(src.to(DEV), pool, pages, torch.tensor(row0, dtype=torch.int32, device=DEV), q_heads=hq, gated=gated,
                   q_norm=None if norm < 0 else norms[0].to(DEV), k_norm=None if norm < 0 else norms[1].to(DEV),
                   norm_mode=norm, eps=1e-6, tables=tables, rot=rot)
    rows = (torch.tensor(row0)[:, None] + torch.arange(T)).reshape(-1)
    cos, sin = (t.cpu()[rows][:, None] for t in tables) if rot else (None, None)
    k = src[:, qw:qw + hkv * hd].reshape(R * T, hkv, hd)
    v = src[:, qw + hkv * hd:qw + 2 * hkv * hd].reshape(R * T, hkv, hd)
    k = ops.kv4_head_row(k, norms[1], norm, 1e-6, cos, sin)
    want = before.clone()
    for n in range(R * T):
        row = int(rows[n])
        p = int(pages[n // T][row // page])
        for h in range(hkv):
            ops.kv4_put(want[p, h, row % page // 16], row % 16, k[n, h].float(), v[n, h])
    assert torch.equal(pool.cpu(), want)
    if hq:
        want_q = torch.empty(R * T, hq, hd, dtype=torch.bfloat16, device=DEV)     # the bf16 path's query rows, bit for bit
        K.head_norm_rope(src.to(DEV), hq, hd, 2 * hd if gated else hd, want_q, hd, hq * hd,
                         norm_w=None if norm < 0 else norms[0].to(DEV), norm_mode=norm, eps=1e-6, tables=tables, rot=rot,
                         pos=rows.to(DEV, torch.int32))
        assert torch.equal(q, want_q)
    else:
        assert q is None


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_of_many_extreme_rows(hd):
    """The same rows through the kernel for many rows: every block as the one that the kernel for few rows writes."""
    y = torch.randn(16, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    y[0], y[1], y[2] = 0.0, -0.0, -7.25
    y[3], y[3, 9] = 0.0, -5.0
    y[4, 0], y[5, hd - 1], y[6, 40] = math.inf, -math.inf, math.nan
    y[7] *= 2.0 ** 54
    y[8, 3] = -(2.0 ** 56)
    y[9] *= 1e-38
    y[10] *= 2.0 ** -41
    y[11, 5] = 2.0 ** 55.9
    y[12] = 1e-40
    y[13, 32:64] = 3.0
    y[14, 33], y[14, 34] = -math.nan, math.inf
    heads = [y.roll(i, 0) for i in range(6)]                       # 3 KV heads of K, then of V
    src = torch.cat(heads, 1).to(DEV)
    few, many = _random_pool(1, 3, 16, hd), _random_pool(17, 3, 16, hd)
    kv4.append(src, few, torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    want = torch.zeros(3, kv4.block_bytes(hd), dtype=torch.uint8)
    for h in range(3):
        for r in range(16):
            ops.kv4_put(want[h], r, heads[h][r], heads[3 + h][r])
    assert torch.equal(few.cpu()[0, :, 0], want)
    kv4.append(src.repeat(17, 1), many, torch.arange(17, dtype=torch.int32, device=DEV), 0)
    assert torch.equal(many, few.expand(17, -1, -1, -1))


def test_append_extreme_rows():
    """Zeros, constants, one value, infinities, NaN, the largest and the smallest magnitudes, both signs of zero."""
    hd = 128
    y = torch.randn(16, hd, generator=torch.Generator().manual_seed(3)).bfloat16()
    y[0], y[1], y[2] = 0.0, -0.0, 7.25
    y[3], y[3, 9] = 0.0, 5.0
    y[4, 0], y[5, 127], y[6, 64] = math.inf, -math.inf, math.nan
    y[7] *= 2.0 ** 54
    y[8, 3] = 2.0 ** 56
    y[9] *= 1e-38
    y[10] *= 2.0 ** -41
    y[11, 5] = 2.0 ** 55.9
    y[12] = 1e-40
    y[13, 32:64] = 3.0
    src = torch.cat((y, y.flip(0)), 1).to(DEV)
    pool = _random_pool(1, 1, 16, hd)
    kv4.append(src, pool, [torch.zeros(1, dtype=torch.int32, device=DEV)], 0)
    want = torch.zeros(kv4.block_bytes(hd), dtype=torch.uint8)
    for r in range(16):
        ops.kv4_put(want, r, y[r], y[15 - r])
    assert torch.equal(pool.cpu().flatten(), want)
    k, v = kv4.read(pool, torch.zeros(1, dtype=torch.int32, device=DEV), 16)
    for got, ref in ((k[0].cpu(), y), (v[0].cpu(), y.flip(0))):
        assert torch.equal(got.isnan().all(-1), (ref.float().abs().amax(-1) < 2.0 ** 56).logical_not())
        assert torch.equal(got.isnan().any(-1), got.isnan().all(-1))


def test_append_skips_and_refuses_rows_on_the_device():
    hd, hkv, page, T = 128, 2, 32, 4
    pages, total = _pages([32, 32, 64, 32], page)
    pool = _random_pool(total, hkv, page, hd)
    src = torch.randn(4 * T, 3 * hkv * hd, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    before = pool.clone()
    # sequence 0 skipped, 1 with two rows past its table, 2 on a page id outside the pool from row 32 on, 3 in order
    pages[2][1] = total
    row0 = torch.tensor([-1, 30, 30, 0], dtype=torch.int32, device=DEV)
    q = kv4.append(src, pool, pages, row0, q_heads=hkv)
    assert _error() == 7
    assert q[:T].eq(0).all() and q[T + 2:2 * T].eq(0).all() and torch.equal(q[3 * T:], src[3 * T:, :hkv * hd].unflatten(1, (hkv, hd)))
    changed = (pool != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted(int(pages[s][0]) for s in (1, 2, 3))
    pages[2][1] = -5
    pool.copy_(before)
    kv4.append(src, pool, pages, row0, q_heads=hkv)
    assert _error() == 7
    pages[2][1] = 0 if int(pages[2][0]) else 1
    # rotary positions past the tables: the row is left out
    pool.copy_(before)
    tables = _tables(8, hd)
    kv4.append(src, pool, pages[3:], 0, q_heads=hkv, rot=hd, tables=tables,
               pos=torch.arange(4 * T, dtype=torch.int32, device=DEV) - 4)
    assert _error() == 7
    k, _ = kv4.read(pool, pages[3], 4 * T)
    old, _ = kv4.read(before, pages[3], 4 * T)
    same = (k.view(torch.int16) == old.view(torch.int16)).all(-1).all(0)
    assert same[:4].all() and same[12:].all() and not same[4:12].any()


def test_append_of_many_rows_skips_and_refuses_on_the_device():
    """The kernel for many rows: a skipped sequence, one past its table, a page id outside the pool, one in order; pages of
    three blocks."""
    hd, hkv, page, T = 128, 3, 48, 70
    pages, total = _pages([96, 96, 96, 96], page)
    pool = _random_pool(total, hkv, page, hd)
    src = torch.randn(4 * T, 3 * hkv * hd, generator=torch.Generator().manual_seed(0)).bfloat16()
    before = pool.cpu()
    pages[2][1] = total
    row0 = torch.tensor([-1, 50, 1, 7], dtype=torch.int32, device=DEV)
    q = kv4.append(src.to(DEV), pool, pages, row0, q_heads=hkv)
    assert _error() == 7
    want = before.clone()
    for s, r0 in enumerate((-1, 50, 1, 7)):
        for t in range(T):
            row = r0 + t
            if r0 < 0 or row >= 96 or (s == 2 and row >= 48):
                continue
            n = s * T + t
            for h in range(hkv):
                ops.kv4_put(want[int(pages[s][row // page]), h, row % page // 16], row % 16,
                            src[n, (hkv + h) * hd:(hkv + h + 1) * hd], src[n, (2 * hkv + h) * hd:(2 * hkv + h + 1) * hd])
    assert torch.equal(pool.cpu(), want)
    rows = src[:, :hkv * hd].to(DEV).view(4, T, hkv, hd)
    got = q.view(4, T, hkv, hd)
    assert got[0].eq(0).all() and got[1, 46:].eq(0).all() and torch.equal(got[1, :46], rows[1, :46])
    assert torch.equal(got[3], rows[3])


@pytest.mark.parametrize("T", [100, 300])
def test_append_of_many_rows_replayed_from_a_graph(T):
    """Captured once, replayed with other rows at another first row and on other pages."""
    hd, hkv = 64, 2
    pages, total = _pages([500, 500], 64)
    pool, table = kv4.pool(total, hkv, 64, hd), pages[0].clone()
    src = torch.randn(2, T, 3 * hkv * hd, device=DEV).bfloat16()
    rows, row0 = src[0].clone(), torch.tensor([0], dtype=torch.int32, device=DEV)
    kv4.append(rows, pool, [table], row0, q_heads=hkv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = kv4.append(rows, pool, [table], row0, q_heads=hkv)
    for i, r0 in ((1, 150), (0, 33)):
        pool.zero_()
        rows.copy_(src[i])
        row0.fill_(r0)
        table.copy_(pages[i])
        graph.replay()
        want = kv4.pool(total, hkv, 64, hd)
        want_q = kv4.append(src[i], want, pages[i], r0, q_heads=hkv)
        assert torch.equal(pool, want) and torch.equal(q, want_q)
    del graph


def test_append_positions_apart_from_rows():
    """Rotary positions from a vector, an offset, or the cache row."""
    hd, T = 64, 9
    src = torch.randn(T, 3 * hd, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    tables = _tables(64, hd)
    table = torch.zeros(1, dtype=torch.int32, device=DEV)
    outs = []
    for row0, kw in ((20, dict()), (0, dict(pos_offset=20)), (3, dict(pos=torch.arange(20, 29, dtype=torch.int32, device=DEV)))):
        pool = kv4.pool(1, 1, 64, hd)
        q = torch.empty(1, T, hd, dtype=torch.bfloat16, device=DEV)
        assert kv4.append(src, pool, table, row0, q_heads=1, rot=hd, tables=tables, q_out=q.transpose(0, 1), **kw) is not None
        outs.append((q, *kv4.read(pool, table, T, row0)))
    for a in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(a, outs[0]))


@pytest.mark.parametrize("hd,hkv,page,lens,n", [(64, 3, 48, [100, 7], 7), (128, 2, 128, [1000], 1000),
                                                (256, 1, 16, [33, 64, 50], 33), (256, 4, 256, [513], 1)])
def test_read_gives_the_stored_values(hd, hkv, page, lens, n):
    pages, total = _pages(lens, page)
    pool = _random_pool(total, hkv, page, hd)
    pool[..., 20 * hd:] = pool[..., 20 * hd:] % 81 + 87                      # exponent bytes that append can write
    half = pool[..., 16 * hd:20 * hd]
    half[..., 1::2] &= 0xBB                                                  # finite scales and minima
    row0 = [x - n for x in lens]
    k, v = kv4.read(pool, pages, n, torch.tensor(row0, dtype=torch.int32, device=DEV))
    for s, r0 in enumerate(row0):
        rows = torch.arange(r0, r0 + n, device=DEV)
        blocks = pool[pages[s].long()[rows // page], :, rows % page // 16]   # [n, hkv, bytes]
        got = ops.kv4_get(blocks.flatten(0, 1), hd)
        pick = (rows % 16).repeat_interleave(hkv)
        for out, ref in ((k[s], got[0]), (v[s], got[1])):
            ref = ref[torch.arange(n * hkv, device=DEV), pick].view(n, hkv, hd).transpose(0, 1)
            assert torch.equal(out, ref.float().bfloat16())
    one, _ = kv4.read(pool, pages[0], n, row0[0])
    assert torch.equal(one, k[0])
    big = torch.full((hkv, n + 5, hd), 9.0, dtype=torch.bfloat16, device=DEV), torch.zeros(hkv, n + 5, hd, dtype=torch.bfloat16, device=DEV)
    kv4.read(pool, pages[0], n, row0[0], out=tuple(t[:, 2:2 + n] for t in big))
    assert torch.equal(big[0][:, 2:2 + n], k[0]) and torch.equal(big[1][:, 2:2 + n], v[0]) and big[0][:, :2].eq(9).all()
    assert kv4.read(pool, pages[0], 0, 0)[0].shape == (hkv, 0, hd)


def test_read_skips_and_refuses_rows_on_the_device():
    pages, total = _pages([32, 32, 32], 16)
    pool = _random_pool(total, 2, 16, 64) & 0x3B
    pages[2][1] = total + 7
    k, v = kv4.read(pool, pages, 20, torch.tensor([-3, 20, 0], dtype=torch.int32, device=DEV))
    assert _error() == 7
    assert k[0].eq(0).all() and v[0].eq(0).all() and k[1, :, 12:].eq(0).all() and v[2, :, 16:].eq(0).all()


def _filled(lens, hkv, page, hd, seed=0, stale=True, vscale=1.0):
    """Sequences whose pages hold lens rows that append wrote, in a pool of other requests' bytes."""
    pages, total = _pages(lens, page, seed=seed)
    pool = _random_pool(total, hkv, page, hd) if stale else kv4.pool(total, hkv, page, hd)
    g = torch.Generator(device=DEV).manual_seed(seed + 10)
    for s, n in enumerate(lens):
        if n:
            src = torch.randn(n, 2 * hkv * hd, device=DEV, generator=g)
            src = src * torch.exp(0.5 * torch.randn(1, 2 * hkv * hd, device=DEV, generator=g))
            src[:, hkv * hd:] *= vscale
            kv4.append(src.bfloat16(), pool, [pages[s]], 0)
    return pool, pages


def _reference(q, pool, pages, pos, scale, gate=None, gate_head=0):
    """(out, error bound) [R, hq * hd] in fp64. A value is V = M + C, M = 2^e m its group's minimum and C = 2^e s c the
    steps above it. Per output of head h, with P the softmax, the bound counts
      the final rounding to bf16: 2^-8 |out|
      P rounded to 11 bits, a factor of the whole value: 2^-11 sum_j P_j |V_j|
      P s rounded to 11 bits, a factor of the steps alone: 2^-11 sum_j P_j C_j; both absolute where they fall below
      2^-14: P is held so that the largest is between 2^6 and 2^14, so below 2^-30 of sum_j C_j over n keys
      the scores, 32-bit sums of exact products over hd dims (2^-24 each) with the query's group sums held to 22 bits:
      below 2^-18 of max_j sum_d |q_d| (|M_jd| + C_jd) scale, which moves the weighted mean by twice that."""
    hkv, hd, page = pool.shape[1], q.shape[2], pool.shape[2] * 16
    R, hq = q.shape[:2]
    G = hq // hkv
    out = torch.zeros(R, hq, hd, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    for s in range(R):
        n = int(pos[s]) + 1
        if n <= 0:
            continue
        blocks = pool[pages[s].long()[:-(-n // page)]].transpose(0, 1).reshape(-1, pool.shape[3])
        k, v = (t.view(hkv, -1, hd)[:, :n] for t in ops.kv4_get(blocks, hd))
        kc, vc = (t.view(hkv, -1, hd)[:, :n] for t in ops.kv4_get(blocks, hd, steps_only=True))
        for h in range(hq):
            qq = q[s, h].double()
            x = (k[h // G] @ qq) * scale
            p = torch.softmax(x, 0)
            out[s, h] = p @ v[h // G]
            spread = 2.0 ** -18 * (((k - kc).abs() + kc)[h // G] @ qq.abs()).max() * abs(scale)
            A, C = p @ v[h // G].abs(), p @ vc[h // G]
            bound[s, h] = (2.0 ** -8 * out[s, h].abs() + (2.0 ** -11 + 2 * spread) * A + (2.0 ** -11 + n * 2.0 ** -30) * C)
    if gate is not None:
        sg = torch.sigmoid(torch.stack([gate[:, h * gate_head:h * gate_head + hd] for h in range(hq)], 1).double())
        out, bound = out * sg, bound * sg + 2.0 ** -18 * (out * sg).abs()
    return out.flatten(1), bound.flatten(1) + 1e-30


def _check(out, ref):
    want, bound = ref
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), (off / bound).max().item()


ATTEND = [(hd, hkv, G, page, lens) for hd, hkv, G, page, lens in [
    (128, 2, 4, 128, [1]), (128, 2, 4, 128, [2, 15, 16, 17, 63, 64, 65]),
    (128, 1, 8, 16, [255, 256, 257, 511, 513]), (256, 4, 6, 128, [1, 300, 1025]),
    (256, 2, 8, 256, [4097]), (64, 3, 5, 48, [31, 1000, 48]), (64, 1, 1, 64, [777]), (128, 3, 7, 32, [129]),
    (256, 1, 3, 32, [20, 33]), (128, 2, 2, 128, [16385]), (256, 1, 1, 128, [16384, 16383])]]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attention_matches_the_oracle(case):
    hd, hkv, G, page, lens = case
    pool, pages = _filled(lens, hkv, page, hd)
    g = torch.Generator(device=DEV).manual_seed(5)
    hq = hkv * G
    q = (1.5 * torch.randn(len(lens), hq, hd, device=DEV, generator=g)).bfloat16()
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    _check(kv4.attention(q, pool, pages, pos, hd ** -0.5), _reference(q, pool, pages, pos, hd ** -0.5))
    gate = torch.randn(len(lens), 2 * hq * hd, device=DEV, generator=g).bfloat16()[:, hd:]
    out = torch.full((len(lens), hq * hd + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    kv4.attention(q, pool, pages, pos, hd ** -0.5, gate=gate, gate_head=2 * hd, out=out[:, 8:-8])
    _check(out[:, 8:-8], _reference(q, pool, pages, pos, hd ** -0.5, gate, 2 * hd))
    assert out[:, :8].eq(3).all() and out[:, -8:].eq(3).all()


@pytest.mark.parametrize("vscale", [1e-30, 1e-6, 3e4, 1e12])
def test_attention_over_values_of_any_size(vscale):
    """V rows of very small and very large values, K and q stretched so that the softmax is one-sided."""
    pool, pages = _filled([300], 1, 128, 128, vscale=vscale)
    q = (20 * torch.randn(1, 4, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))).bfloat16()
    pos = torch.tensor([299], dtype=torch.int32, device=DEV)
    _check(kv4.attention(q, pool, pages, pos, 0.2), _reference(q, pool, pages, pos, 0.2))


def test_attention_over_rows_of_mixed_sizes():
    """Rows of one cache whose values differ by 2^40 and more, zero rows among them: a zero V row still takes its weight."""
    hd, n = 64, 90
    g = torch.Generator(device=DEV).manual_seed(0)
    src = torch.randn(n, 2 * hd, device=DEV, generator=g)
    src[:, hd:] *= torch.exp2(40 * torch.rand(n, 1, device=DEV, generator=g) - 30)
    src[10:40, hd:] = 0.0
    src[50:55] = 0.0
    pool = kv4.pool(1, 1, 96, hd)
    table = torch.zeros(1, dtype=torch.int32, device=DEV)
    kv4.append(src.bfloat16(), pool, table, 0)
    q = torch.randn(1, 8, hd, device=DEV, generator=g).bfloat16()
    for p in (5, 39, 40, 89):
        pos = torch.tensor([p], dtype=torch.int32, device=DEV)
        _check(kv4.attention(q, pool, table, pos, 0.125), _reference(q, pool, [table], pos, 0.125))


@pytest.mark.parametrize("size", [1e-20, 1e-3, 1e4, 1e20])
def test_attention_with_queries_of_any_size(size):
    pool, pages = _filled([200], 2, 64, 128)
    q = (size * torch.randn(1, 6, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))).bfloat16()
    pos = torch.tensor([199], dtype=torch.int32, device=DEV)
    scale = 0.1 / size
    _check(kv4.attention(q, pool, pages, pos, scale), _reference(q, pool, pages, pos, scale))


def test_attention_zero_query_is_the_mean():
    pool, pages = _filled([100], 1, 128, 128)
    q = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device=DEV)
    pos = torch.tensor([99], dtype=torch.int32, device=DEV)
    _check(kv4.attention(q, pool, pages, pos, 0.1), _reference(q, pool, pages, pos, 0.1))


def test_non_finite_rows_reach_only_who_sees_them():
    """A NaN or infinite K or V row is NaN for queries that see it and nothing for the others; a NaN query head is NaN
    alone."""
    hd, hkv, lens = 128, 2, [40, 40, 40]
    pool, pages = _filled(lens, hkv, 64, hd)
    src = torch.randn(1, 2 * hkv * hd, device=DEV).bfloat16()
    bad_k, bad_v = src.clone(), src.clone()
    bad_k[0, 3], bad_v[0, 2 * hd + 7] = math.inf, math.nan
    kv4.append(bad_k, pool, pages[:1], 30)
    kv4.append(bad_v, pool, pages[1:2], 30)
    q = torch.randn(3, 4, hd, device=DEV).bfloat16()
    q[2, 1, 5] = math.nan
    full = torch.tensor([39, 39, 39], dtype=torch.int32, device=DEV)
    out = kv4.attention(q, pool, pages, full, 0.1).view(3, 4, hd)
    assert out[0, :2].isnan().all() and torch.isfinite(out[0, 2:]).all()
    assert out[1, :2].isnan().all() and torch.isfinite(out[1, 2:]).all()
    assert out[2, 1].isnan().all() and torch.isfinite(out[2, [0, 2, 3]]).all()
    short = torch.tensor([29, 29, 39], dtype=torch.int32, device=DEV)
    q[2, 1, 5] = 0.0
    _check(kv4.attention(q, pool, pages, short, 0.1), _reference(q, pool, pages, short, 0.1))


def test_bytes_behind_the_end_do_not_matter():
    """Unwritten rows of the last block and page hold 0xFF (NaN scales, marked exponents) or anything else."""
    for fill in (0xFF, 0x7C, 0x00):
        lens = [1, 17, 130, 256]
        pages, total = _pages(lens, 128)
        pool = torch.full((total, 2, 8, kv4.block_bytes(128)), fill, dtype=torch.uint8, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(9)
        for s, n in enumerate(lens):
            kv4.append(torch.randn(n, 4 * 128, device=DEV, generator=g).bfloat16(), pool, [pages[s]], 0)
        q = torch.randn(4, 8, 128, device=DEV, generator=g).bfloat16()
        pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
        out = kv4.attention(q, pool, pages, pos, 0.1)
        _check(out, _reference(q, pool, pages, pos, 0.1))
        if fill == 0xFF:
            first = out
        assert torch.equal(out, first)


def test_attention_skips_and_refuses_on_the_device():
    lens = [50, 50, 50, 50]
    pool, pages = _filled(lens, 2, 32, 128)
    q = torch.randn(4, 4, 128, device=DEV).bfloat16()
    pos = torch.tensor([-1, 49, -7, 49], dtype=torch.int32, device=DEV)
    out = kv4.attention(q, pool, pages, pos, 0.1)
    assert out[0].eq(0).all() and out[2].eq(0).all()
    _check(out, _reference(q, pool, pages, pos, 0.1))
    check_errors()
    pos[3] = 64                                          # the table holds 64 rows
    assert kv4.attention(q, pool, pages, pos, 0.1)[3].eq(0).all() and _error() == 7
    pos[3] = 49
    keep = int(pages[1][1])
    pages[1][1] = pool.shape[0]                          # rows 32 .. are left out
    out = kv4.attention(q, pool, pages, pos, 0.1)
    assert _error() == 7
    short = torch.tensor([-1, 31, -7, 49], dtype=torch.int32, device=DEV)
    _check(out, _reference(q, pool, pages, short, 0.1))
    pages[1][0], pages[1][1] = -1, -1
    out = kv4.attention(q, pool, pages, pos, 0.1)
    assert out[1].eq(0).all() and _error() == 7
    pages[1][0] = keep


def test_the_same_bits_alone_batched_and_on_other_pages():
    hd, hkv, lens = 256, 2, [1, 700, 3000, 16500]
    pool, pages = _filled(lens, hkv, 128, hd, stale=False)
    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn(4, 12, hd, device=DEV, generator=g).bfloat16()
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    out = kv4.attention(q, pool, pages, pos, 0.0625)
    for s in range(4):
        assert torch.equal(kv4.attention(q[s:s + 1], pool, pages[s:s + 1], pos[s:s + 1], 0.0625), out[s:s + 1])
    perm = torch.randperm(pool.shape[0], device=DEV)
    moved = torch.empty_like(pool)
    moved[perm] = pool
    tables = [torch.cat((perm[t.long()].int(), torch.zeros(3, dtype=torch.int32, device=DEV))) for t in pages]
    assert torch.equal(kv4.attention(q, moved, tables, pos, 0.0625), out)
    many = 70                                            # more sequences than one launch takes, tables shared
    pick = [i % 4 for i in range(many)]
    big = kv4.attention(q[pick], pool, [pages[i] for i in pick], pos[pick], 0.0625)
    assert torch.equal(big, out[pick])
    k, _ = kv4.read(pool, [pages[3]] * many, 5, torch.full((many,), 11, dtype=torch.int32, device=DEV))
    assert torch.equal(k, k[:1].expand_as(k))


@pytest.mark.parametrize("lens", [[120, 5, 254], [1500, 5, 500]], ids=str)
@pytest.mark.parametrize("hd", [128, 256])
def test_decode_loop_replayed_from_a_graph_on_another_stream(hd, lens):
    """append + attention (of one split and of several) captured once; the replays at new positions equal the eager calls
    bit for bit."""
    hkv, G, R, steps = 2, 4, 3, 20
    hq = hkv * G
    tables = _tables(1600, 64)
    g = torch.Generator(device=DEV).manual_seed(4)
    rows = [torch.randn(R, (2 * hq + 2 * hkv) * hd, device=DEV, generator=g).bfloat16() for _ in range(steps)]
    w = torch.randn(2, hd, device=DEV, generator=g).bfloat16()

    def step(src, pool, pages, pos):
        q = kv4.append(src, pool, pages, pos, q_heads=hq, gated=True, q_norm=w[0], k_norm=w[1], norm_mode=1, rot=64,
                       tables=tables)
        return kv4.attention(q, pool, pages, pos, 0.1, gate=src[:, hd:], gate_head=2 * hd)

    pages, total = _pages([n + steps for n in lens], 128)
    pools = [kv4.pool(total, hkv, 128, hd) for _ in range(2)]
    for p in pools:
        for s, n in enumerate(lens):
            kv4.append(torch.ones(n, 2 * hkv * hd, device=DEV).cumsum(0).sin().bfloat16(), p, [pages[s]], 0)
    want = [step(rows[i], pools[0], pages, torch.tensor([n + i for n in lens], dtype=torch.int32, device=DEV))
            for i in range(steps)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        src, pos = rows[0].clone(), torch.tensor(lens, dtype=torch.int32, device=DEV)
        step(src, pools[1], pages, pos)                  # the same row again: appended twice, the same bytes
        graphs, outs = [], []
        for _ in range(2):                               # two graphs of the same step, replayed in turn
            graphs.append(torch.cuda.CUDAGraph())
            side.synchronize()
            with torch.cuda.graph(graphs[-1], stream=side, capture_error_mode="thread_local"):
                outs.append(step(src, pools[1], pages, pos))
        for i in range(steps):
            src.copy_(rows[i])
            pos.copy_(torch.tensor([n + i for n in lens], dtype=torch.int32))
            graphs[i % 2].replay()
            assert torch.equal(outs[i % 2], want[i])
    torch.cuda.current_stream().wait_stream(side)
    for s, n in enumerate(lens):
        for a, b in zip(kv4.read(pools[0], pages[s], n + steps), kv4.read(pools[1], pages[s], n + steps)):
            assert torch.equal(a, b)


def test_steps_enqueued_without_a_pause():
    """Append, attention and its join start before their predecessors end; a chain of dependent steps (each row made of the
    last step's output, positions advanced on the device) enqueued at once equals the same steps with a pause after each."""
    hd, hkv, R = 128, 2, 3
    lens = [700, 40, 1300]
    g = torch.Generator(device=DEV).manual_seed(8)
    pages, total = _pages([n + 40 for n in lens], 128)
    base = kv4.pool(total, hkv, 128, hd)
    for s, n in enumerate(lens):
        kv4.append(torch.randn(n, 2 * hkv * hd, device=DEV, generator=g).bfloat16(), base, [pages[s]], 0)
    first = torch.randn(R, 4 * hd, device=DEV, generator=g).bfloat16()

    def chain(pause):
        pool, x, outs = base.clone(), first, []
        pos = torch.tensor(lens, dtype=torch.int32, device=DEV)
        for _ in range(40):
            q = kv4.append(torch.cat((x, x, x), 1)[:, :8 * hd], pool, pages, pos, q_heads=4)
            x = kv4.attention(q, pool, pages, pos, 0.1)
            outs.append(x)
            x = (x + first).contiguous()
            pos = pos + 1
            if pause:
                torch.cuda.synchronize()
        return torch.stack(outs)
    a, b = chain(False), chain(True)
    assert torch.isfinite(a).all() and torch.equal(a, b)


def test_inputs_written_just_before():
    """attention starts while the kernel before it ends: queries, positions and page tables that this kernel writes."""
    pool, pages = _filled([700, 700], 2, 128, 128)
    q = torch.randn(2, 8, 128, device=DEV).bfloat16()
    table, other = pages
    at = [torch.tensor([n], dtype=torch.int32, device=DEV) for n in (20, 699)]
    want = {(i, j): kv4.attention(q[i:i + 1], pool, [pages[i]], at[j], 0.1) for i in range(2) for j in range(2)}
    pos, now, mine = at[0].clone(), q[:1].clone(), table.clone()
    for step in range(60):
        i, j = step % 2, step // 2 % 2
        now.copy_(q[i:i + 1]), mine.copy_(pages[i]), pos.copy_(at[j])
        last = (lambda: pos.mul_(1), lambda: mine.mul_(1), lambda: now.mul_(1))[step % 3]
        last()
        assert torch.equal(kv4.attention(now, pool, [mine], pos, 0.1), want[i, j])
    pos.fill_(0)
    got = []
    for n in range(0, 640, 20):
        got.append(kv4.attention(now, pool, [mine], pos, 0.1))
        pos.add_(20)
    for n, o in zip(range(0, 640, 20), got):
        assert torch.equal(o, kv4.attention(now, pool, [mine], torch.tensor([n], dtype=torch.int32, device=DEV), 0.1))


def test_more_sequences_than_one_launch_takes():
    """150 sequences of one page each: appended, attended and read in several launches, as each alone."""
    hd, hkv, R = 64, 2, 150
    pages = list(torch.randperm(R, generator=torch.Generator().manual_seed(1)).to(DEV, torch.int32).split(1))
    pool = kv4.pool(R, hkv, 16, hd)
    src = torch.randn(3 * R, 3 * hkv * hd, device=DEV).bfloat16()
    row0 = (torch.arange(R, device=DEV) % 13).int()
    q = kv4.append(src, pool, pages, row0, q_heads=hkv)
    out = kv4.attention(q[2::3], pool, pages, row0 + 2, 0.2)
    k, _ = kv4.read(pool, pages, 3, row0)
    alone = kv4.pool(R, hkv, 16, hd)
    for s in range(R):
        one = kv4.append(src[3 * s:3 * s + 3], alone, pages[s], s % 13, q_heads=hkv)
        assert torch.equal(q[3 * s:3 * s + 3], one)
        assert torch.equal(out[s:s + 1], kv4.attention(one[2:], alone, [pages[s]], row0[s:s + 1] + 2, 0.2))
        assert torch.equal(k[s], kv4.read(alone, pages[s], 3, s % 13)[0])
    assert torch.equal(pool, alone)


def test_two_streams_at_once():
    """The same sequences attended from two streams at once: workspaces are each call's own."""
    pool, pages = _filled([3000, 2000], 2, 128, 128)
    pos = torch.tensor([2999, 1999], dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 8, 128, device=DEV).bfloat16() for _ in range(2)]
    want = [kv4.attention(q, pool, pages, pos, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv4.attention(qs[i], pool, pages, pos, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_pool_past_4_gib():
    """Offsets past 32 bits: a sequence on the last pages of a large pool equals the same sequence in a small one."""
    hd, hkv, page = 256, 8, 128
    small, pages = _filled([300], hkv, page, hd, stale=False)
    slab = small[0].numel()
    n_pages = (1 << 32) // slab + 300
    big = torch.empty(n_pages, hkv, page // 16, kv4.block_bytes(hd), dtype=torch.uint8, device=DEV)
    table = torch.tensor([n_pages - 1, n_pages - 250, n_pages - 120], dtype=torch.int32, device=DEV)
    k, v = kv4.read(small, pages[0], 300)
    kv4.append(torch.cat((k.transpose(0, 1).reshape(300, -1), v.transpose(0, 1).reshape(300, -1)), 1), big, table, 0)
    kv4.append(torch.cat((k.transpose(0, 1).reshape(300, -1), v.transpose(0, 1).reshape(300, -1)), 1), small, pages, 0)
    for a, b in zip(kv4.read(big, table, 300), kv4.read(small, pages[0], 300)):
        assert torch.equal(a, b)
    q = torch.randn(1, 8 * hkv, hd, device=DEV).bfloat16()
    pos = torch.tensor([299], dtype=torch.int32, device=DEV)
    assert torch.equal(kv4.attention(q, big, table, pos, 0.06), kv4.attention(q, small, pages, pos, 0.06))


def test_inputs_keep_their_strides():
    """Rows of a wider buffer, query rows and outputs of other pitches."""
    hd, hkv, G = 128, 2, 3
    pool, pages = _filled([70, 20], hkv, 64, hd)
    q = torch.randn(2, hkv * G, hd, device=DEV).bfloat16()
    pos = torch.tensor([69, 19], dtype=torch.int32, device=DEV)
    want = kv4.attention(q, pool, pages, pos, 0.1)
    wide = torch.zeros(hkv * G, 2, hd + 8, dtype=torch.bfloat16, device=DEV)
    wide[..., :hd] = q.transpose(0, 1)
    assert torch.equal(kv4.attention(wide[..., :hd].transpose(0, 1), pool, pages, pos, 0.1), want)


def test_sequences_of_no_rows_and_no_sequences():
    pool = kv4.pool(2, 1, 16, 64)
    table = torch.zeros(1, dtype=torch.int32, device=DEV)
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    src = torch.zeros(0, 3 * 64, dtype=torch.bfloat16, device=DEV)
    assert kv4.append(src, pool, table, 3, q_heads=1).shape == (0, 1, 64)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.tensor([-1], dtype=torch.int32, device=DEV)
    assert kv4.attention(q, pool, [empty], none, 0.1).eq(0).all()
    assert kv4.attention(q[:0], pool, [], none[:0], 0.1).shape == (0, 128)
    assert kv4.read(pool, [], 4, none[:0])[0].shape == (0, 1, 4, 64)
    k, _ = kv4.read(pool, [empty], 4, none)
    assert k.eq(0).all()
