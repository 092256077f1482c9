"""Appends of many rows whose rotary dims are not a multiple of 32: whole against pieces of at most 100 rows, which
test_kv4_gpu.py holds to the oracle byte for byte."""
import pytest
import torch

from ridgefill_data_b200.ops import kv4
from ridgefill_data_b200.ops._ext import check_errors

from test_kv4_gpu import DEV, _pages, _random_pool, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,rot,norm", [(64, 16, -1), (64, 48, 1), (128, 16, 0), (256, 16, 1)])
def test_many_rows_equal_their_pieces(hd, rot, norm):
    hkv, G, n, first = 2, 3, 4097, 37
    pages, total = _pages([n + first], 128)
    whole = _random_pool(total, hkv, 128, hd)
    pieces = whole.clone()
    g = torch.Generator(device=DEV).manual_seed(0)
    src = torch.randn(n, (hkv * G + 2 * hkv) * hd, device=DEV, generator=g).bfloat16()
    w = [torch.randn(hd, device=DEV, generator=g).bfloat16() for _ in range(2)] if norm >= 0 else [None, None]
    kw = dict(q_heads=hkv * G, q_norm=w[0], k_norm=w[1], norm_mode=norm, tables=_tables(n + first, rot), rot=rot)
    q = kv4.append(src, whole, pages, first, **kw)
    for lo in range(0, n, 100):
        part = kv4.append(src[lo:lo + 100], pieces, pages, first + lo, **kw)
        assert torch.equal(part, q[lo:lo + 100])
    assert torch.equal(whole, pieces)
    torch.cuda.synchronize()
    check_errors()
