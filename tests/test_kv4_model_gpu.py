"""Models serving from a pool of 4-bit K/V pages (models/kvpool.py bits=4): prefill, exact rows, continued prompts and decode
steps against the same model on bf16 caches whose rows are replaced by the values their 4-bit form stands for; decode steps
alone, batched and replayed from a graph give the same bits; the scheduler serves requests from such a pool."""
import threading

import pytest
import torch

from ridgefill_data_b200.engine.decode import step
from ridgefill_data_b200.engine.decode_graph import DecodeGraph
from ridgefill_data_b200.engine.prefill import finish, run_lower
from ridgefill_data_b200.models.base import from_config
from ridgefill_data_b200.models.kvpool import KVPool, PoolExhausted
from ridgefill_data_b200.ops import oracle as ops
from ridgefill_data_b200.ops._ext import check_errors

from test_b200_model_gpu import HYB, LLAMA, QWEN3
from test_paged_kv_gpu import _arm

pytestmark = pytest.mark.gpu
CFGS = [HYB, QWEN3, LLAMA]


def _model(cfg, bits, pages=64):
    m = from_config(cfg, seed=0, device="cuda", std=0.05, backend="b200")
    if bits == 4:
        m.kv_pool = KVPool(m, pages, 128, bits=4)
        return m
    # bf16 caches that hold what 4 bits keep of every row
    write, decode_ok = m._write_kv, m._attn_decode_ok
    m._attn_decode_ok = lambda: False

    def rounded(i, src, pos, c):
        n0 = write(i, src, pos, c)
        for name in ("kbuf", "vbuf"):
            rows = c[name][:, n0:c["n"]]
            rows.copy_(ops.kv4_values(*ops.kv4_quantise(rows)).float())
        return n0
    m._write_kv = rounded
    assert decode_ok() or cfg is LLAMA
    return m


def _close(a, b):
    """The two sides do the same products on the same values but for bf16 roundings (2^-8 each) of a layer's attention
    output and a cached value; a rounding reaches a logit through at most 3 products a layer and 4 to 8 layers whose
    residual sums keep their size, 24 roundings of independent sign: sqrt(24) 2^-8 = 0.02 of the largest logit, and the
    3e-2 of the bf16 decode kernels against their per-sequence path covers it."""
    assert torch.isfinite(a).all()
    return (a.float() - b.float()).abs().max().item() / b.float().abs().max().item() < 3e-2


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
@pytest.mark.parametrize("rows", [None, [5, 40, 200]])
def test_prefill_and_decode_match_rounded_bf16_caches(cfg, rows):
    arm = _arm(cfg, cfg.n_layers // 2)
    ids = torch.randint(0, cfg.vocab, (333,), generator=torch.Generator().manual_seed(2)).cuda()
    runs = []
    with torch.no_grad():
        for bits in (4, 16):
            m = _model(cfg, bits)
            hs, lower = run_lower(m, ids, [arm.split])
            logits, cache, _ = finish(m, ids, hs[arm.split], lower, arm, 2, exact_rows=rows)
            outs = [logits]
            for s in range(3):                         # the same tokens on both sides
                outs.append(step(m, 11 + s, ids.shape[0] + s, cache, arm))
            runs.append(outs)
            if bits == 4:
                att = m.kv_pool.layers[0]
                assert m.kv_pool.free_pages(att) == 64 - 3
                m.kv_pool.release(cache)
                assert m.kv_pool.free_pages(att) == 64
    check_errors()
    for a, b in zip(*runs):
        assert _close(a, b)


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_a_prompt_in_pieces_gives_the_whole_prompts_logits(cfg):
    """A second piece appended behind the first one (its rows start inside a 16-row block) reads the first one's quantised
    rows, as the whole prompt's own later rows do: the same logits within bf16 rounding."""
    ids = torch.randint(0, cfg.vocab, (300,), generator=torch.Generator().manual_seed(3)).cuda()
    m = _model(cfg, 4)
    logits, caches = [], []
    with torch.no_grad():
        for cuts in ([300], [101, 199]):
            cache, lo = m.new_cache(), 0
            for n in cuts:
                pos = torch.arange(lo, lo + n, device="cuda")
                h = m.embed(ids[lo:lo + n])
                for i in range(m.n_layers):
                    h = m.layer(i, h, pos, cache)
                lo += n
            logits.append(m.logits(h[-1:]))
            caches.append(cache)
    check_errors()
    assert _close(logits[1], logits[0])
    assert caches[0][m.kv_pool.layers[0]]["n"] == 300


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_decode_alone_batched_and_graphed_give_the_same_bits(cfg):
    lens = [130, 257, 64]
    runs = {}
    for mode in ("alone", "batch", "graph"):
        m = _model(cfg, 4)
        caches, toks = [], []
        g = torch.Generator().manual_seed(7)
        with torch.no_grad():
            for n in lens:
                ids = torch.randint(0, cfg.vocab, (n,), generator=g).cuda()
                caches.append(run_lower(m, ids, [m.n_layers], reserve=64)[1])
                toks.append(int(ids[-1]))
            pos, out = list(lens), []
            dg = DecodeGraph(m, caches, headroom=8) if mode == "graph" else None
            for _ in range(5):
                if mode == "alone":
                    lg = torch.cat([m.decode_batch([t], [p], [c]) for t, p, c in zip(toks, pos, caches)])
                else:
                    lg = dg.step(toks) if dg is not None else m.decode_batch(toks, pos, caches)
                out.append(lg.clone())
                toks = [int(t) for t in lg.argmax(-1)]
                pos = [p + 1 for p in pos]
        torch.cuda.synchronize()
        check_errors()
        runs[mode] = torch.stack(out)
        del dg, m
    assert torch.equal(runs["alone"], runs["batch"]) and torch.equal(runs["batch"], runs["graph"])


def test_pool_bytes_and_exhaustion():
    m = _model(HYB, 4, pages=8)
    full = KVPool(m, 8, 128)
    assert m.kv_pool.bytes() == 8 * 8 * (20 * 256 + 32) * len(m.kv_pool.layers)
    assert full.bytes() / m.kv_pool.bytes() > 3.1
    ids = torch.randint(0, HYB.vocab, (1100,), generator=torch.Generator().manual_seed(6)).cuda()
    with torch.no_grad(), pytest.raises(PoolExhausted):
        run_lower(m, ids, [m.n_layers])


def test_scheduler_serves_from_a_4_bit_pool():
    pytest.importorskip("fastapi")
    from ridgefill_data_b200.serve.engine import Request, Scheduler
    m = _model(HYB, 4, pages=12)
    arm = _arm(HYB, HYB.n_layers // 2)
    sched = Scheduler(m, interleave=1).start()
    tokens = {}
    try:
        dones = []
        for seed, n in ((7, 300), (8, 260), (9, 420)):
            ev = threading.Event()

            def emit(e, ev=ev, seed=seed):
                tokens.setdefault(seed, []).append(e)
                if e.get("stop"):
                    ev.set()
            ids = torch.randint(0, HYB.vocab, (n,), generator=torch.Generator().manual_seed(seed))
            sched.submit(Request(ids=ids, n_predict=6, arm=arm, emit=emit, ignore_eos=True))
            dones.append(ev)
        assert all(ev.wait(120) for ev in dones)
    finally:
        sched.stop()
    check_errors()
    assert sched.stats["errors"] == 0 and sched.stats["completed"] == 3
    assert m.kv_pool.free_pages() == 12
