"""Decode attention over the 4-bit cache at the ends of the values that it holds: finite V rows up to 2^56, zero V rows beside
small ones, rows that were never appended."""
import pytest
import torch

from ridgefill_data_b200.ops import kv4
from ridgefill_data_b200.ops._ext import check_errors

from test_kv4_gpu import DEV, _check, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    torch.cuda.synchronize()
    check_errors()


def _cache(k, v, page=48):
    """One sequence of rows k, v [n, kv heads, hd] on shuffled pages -> (pool, page table)."""
    n, hkv, hd = k.shape
    held = -(-n // page)
    table = torch.randperm(held, generator=torch.Generator().manual_seed(3)).to(DEV, torch.int32)
    pool = kv4.pool(held, hkv, page, hd)
    kv4.append(torch.cat((k.flatten(1), v.flatten(1)), 1).bfloat16(), pool, table, 0)
    return pool, table


def _rows(*shape, seed):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [40, 42, 44, 50, 53])
def test_large_value_rows(hd, size):
    """V rows of 2^size (their largest values near 2^(size + 2)), alone, many, and beside rows of size 1. Keys that grow along
    the sequence raise the largest score in small steps, so probabilities reach the top of their range."""
    n = 150
    k, v = _rows(n, 2, hd, seed=1), _rows(n, 2, hd, seed=2).clamp(-6, 6)
    v *= 2.0 ** size
    v[70:90] *= 2.0 ** -size                                          # rows of size 1 among them
    q = _rows(1, 6, hd, seed=3).bfloat16()
    k += q.float().view(2, 3, hd).mean(1) * torch.linspace(0, 2, n, device=DEV)[:, None, None]
    pool, table = _cache(k, v)
    for last in (0, 1, 16, 75, n - 1):
        pos = torch.tensor([last], dtype=torch.int32, device=DEV)
        _check(kv4.attention(q, pool, table, pos, 0.1), _reference(q, pool, [table], pos, 0.1))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_largest_value_rows(hd):
    """The largest finite row, both signs in one group (the largest step), under a query that sees it alone or among others."""
    top = 2.0 ** 56 * (1 - 2.0 ** -8)
    v = _rows(20, 1, hd, seed=4)
    v[0], v[7] = top, -top
    v[0, :, ::2] = -top
    v[7, :, 5::7] = top
    k = _rows(20, 1, hd, seed=5)
    pool, table = _cache(k, v)
    got = kv4.read(pool, table, 20)[1]
    assert torch.isfinite(got).all() and got[0, 0].abs().max() == top
    q = _rows(1, 4, hd, seed=6).bfloat16()
    for last in (0, 6, 7, 19):
        pos = torch.tensor([last], dtype=torch.int32, device=DEV)
        _check(kv4.attention(q, pool, table, pos, 0.1), _reference(q, pool, [table], pos, 0.1))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [-10, -22, -28, -34, -38])
@pytest.mark.parametrize("zeros", [[0], [99], list(range(20, 50))], ids=["first", "last", "many"])
def test_zero_value_rows_beside_small_ones(hd, size, zeros):
    """V rows of zeros take their weight and nothing else: what rows of any size add keeps its bits. First among rows of
    similar scores, then with 2^13 times the weight of the others."""
    n = 100
    k, v = _rows(n, 2, hd, seed=7), _rows(n, 2, hd, seed=8) * 2.0 ** size
    v[zeros] = 0.0
    q = _rows(1, 4, hd, seed=9).bfloat16()
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    for lead in (0.0, 13 * 0.6931):
        k[zeros] = 0.0
        if lead:                               # the zero rows' keys along the first query of each KV head: score + lead
            q[0, 1::2] = q[0, ::2]
            w = q[0, ::2].float()
            k[zeros] = w / w.square().sum(-1, keepdim=True) * lead / 0.1
        pool, table = _cache(k, v)
        _check(kv4.attention(q, pool, table, pos, 0.1), _reference(q, pool, [table], pos, 0.1))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_never_appended_are_zero_rows(hd):
    """A pool starts zeroed: a visible row that nothing was appended to reads as zeros and counts as a row of zeros."""
    pool, table = _cache(_rows(60, 2, hd, seed=1), _rows(60, 2, hd, seed=2) * 2.0 ** -20, page=96)
    q = _rows(1, 6, hd, seed=3).bfloat16()
    for last in (60, 95):
        pos = torch.tensor([last], dtype=torch.int32, device=DEV)
        _check(kv4.attention(q, pool, table, pos, 0.1), _reference(q, pool, [table], pos, 0.1))
    empty = kv4.pool(8, 2, 96, hd)
    table = torch.arange(8, dtype=torch.int32, device=DEV)
    for last in (0, 95, 700):
        pos = torch.tensor([last], dtype=torch.int32, device=DEV)
        assert kv4.attention(q, empty, table, pos, 0.1).eq(0).all()
