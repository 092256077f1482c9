"""Attention behind a kernel that lets it start early and then writes what it reads."""
import pytest
import torch

from ridgefill_data_b200.ops import kv4
from ridgefill_data_b200.ops._ext import check_errors

from test_kv4_gpu import DEV, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 300])
def test_positions_and_tables_written_by_an_append(rows):
    """append allows its successor to start and stores its query rows at its end. Without norm and rotation they are its
    input's bits, so here they are int32 positions and page tables in a buffer that attention reads: every step changes them,
    old and new ones alike are valid. (rows 300: through the kernel for many rows.)"""
    pool, pages = _filled([700, 700], 2, 128, 128)
    scratch = kv4.pool(3, 1, 128, 64)                      # where the append's own K / V rows go
    own = torch.arange(3, dtype=torch.int32, device=DEV)
    q = torch.randn(1, 8, 128, device=DEV).bfloat16()
    plans = []                                             # 32 int32: position, 3 unused, a page table, unused
    for table in pages:
        for last in (20, 555, 699):
            plan = torch.zeros(32, dtype=torch.int32, device=DEV)
            plan[0], plan[4:4 + len(table)] = last, table
            plans.append(plan)
    src = [torch.cat((p.view(torch.bfloat16).expand(rows, 64), torch.ones(rows, 128, device=DEV).bfloat16()), 1).contiguous()
           for p in plans]
    buffer = torch.zeros(rows, 1, 64, dtype=torch.bfloat16, device=DEV)
    last_row = buffer[rows - 1, 0].view(torch.int32)
    pos, table = last_row[:1], last_row[4:4 + len(pages[0])]
    want = [kv4.attention(q, pool, [p[4:4 + len(pages[0])]], p[:1], 0.1) for p in plans]
    torch.cuda.synchronize()
    got = []
    for step in range(60):
        kv4.append(src[step % 6], scratch, own, 0, q_heads=1, q_out=buffer)
        got.append(kv4.attention(q, pool, [table], pos, 0.1))
    torch.cuda.synchronize()
    check_errors()
    for step, out in enumerate(got):
        assert torch.equal(out, want[step % 6]), step
