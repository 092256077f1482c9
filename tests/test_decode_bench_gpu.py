"""bench.py --decode: every number of sequences is timed at the context that its line reports, on bf16 caches and on a pool of
4-bit pages."""
import importlib.util
import json
import os
from types import SimpleNamespace

import pytest

from ridgefill_data_b200.engine import decode_graph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 16])
def test_every_entry_starts_at_its_context(bits, monkeypatch, capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")
    spec = importlib.util.spec_from_file_location("bench_under_test", path)
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    starts, make = [], decode_graph.DecodeGraph.__init__

    def noted(self, model, caches, *args, **kw):
        make(self, model, caches, *args, **kw)
        starts.append(list(self.lengths))
    monkeypatch.setattr(decode_graph.DecodeGraph, "__init__", noted)
    # 120 rows and 64 steps: two pages a sequence; two entries one after another would need three
    bench.decode_bench(SimpleNamespace(model="tiny-llama", decode="1,2,3", kv_bits=bits, decode_context=120, steps=64))
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines() if x.startswith("{")]
    assert [x["sequences"] for x in lines] == [1, 2, 3] and all(x["config"]["context"] == 120 for x in lines)
    assert starts == [[120], [120] * 2, [120] * 3]
