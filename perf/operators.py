"""The 4-bit K/V cache: rows appended with head norm and rotation, decode attention over it, and rows read back.

Three kinds of pass:
  append  projected rows of R sequences, T each: q and k head norm, rotary positions, q out, K / V into the cache's
          4-bit pages; the rows just written are read back as bf16 (as a prefill does before its attention)
  attend  one query row of each of R sequences over its pages
  read    n rows of one sequence as bf16 K / V

The cache: uint8 [pages, kv heads, page_size / 16, 20 hd + 32], blocks of 16 rows. A row of hd values y is kept as an
exponent e (max|y| in [2^e, 2^(e+1)), e in -40 .. 40; byte e + 127; byte 255 marks a row with a non-finite value, or one
of 2^56 and more, whose values are NaN) and, per 32 dims, fp16 m = min z and s = (max z - min z) / 15 of z = y 2^-e and
codes c = rint((z - m) / s) in 0 .. 15; the value is 2^e (m + s c). A block holds, in this order: K codes (8 hd bytes),
V codes (8 hd), K scales [16][hd / 32], K minima [16][hd / 32], V scales [hd / 32][16], V minima [hd / 32][16], 16 K
exponents, 16 V exponents. code_places() and row_places() give the order inside those parts."""
import math

import torch

own = False

GROUP = 32
LIMIT = 40
MARK = 255

# head shapes of the models that the repository configures: KV heads, query heads per KV head, head dim, rotary dims,
# head norm (-1 none, 0 plain, 1 zero-centred), gated output
SHAPES = {"hybrid-256": (4, 6, 256, 64, 1, True), "hybrid-moe-256": (2, 8, 256, 64, 1, True),
          "dense-128": (8, 4, 128, 128, -1, False), "dense-norm-128": (8, 4, 128, 128, 0, False),
          "small-64": (2, 4, 64, 64, -1, False)}


def _case(name, kind, shape, R, rows, ctx, page=128, ragged=False, **kw):
    hkv, G, hd, rot, norm, gated = SHAPES[shape] if isinstance(shape, str) else shape
    return dict(name=name, kind=kind, R=R, rows=rows, ctx=ctx, page=page, ragged=ragged, hkv=hkv, G=G, hd=hd, rot=rot,
                norm=norm, gated=gated, **kw)


def listed():
    return [
        # one stream's decode row of a dense model: latency alone
        _case("append-token", "append", "dense-norm-128", 1, 1, 700),
        # a decode round of 16 streams at different lengths
        _case("append-round", "append", "hybrid-256", 16, 1, 16384, ragged=True),
        # an odd piece of a prompt behind an odd number of rows, starting and ending inside 16-row blocks
        _case("append-odd", "append", (2, 5, 64, 32, 0, False), 1, 1021, 1058, page=256),
        # the exact tail of a 16K prompt behind its filled prefix
        _case("append-tail", "append", "hybrid-256", 1, 4096, 16384),
        # a whole 16K prompt of a dense model
        _case("append-prompt", "append", "dense-128", 1, 16384, 16384),
        # a short cache read for a follow-up turn, odd length
        _case("read-odd", "read", "small-64", 1, 1001, 1001, page=256),
        # a 16K prompt's cache read before the tail's attention
        _case("read-prompt", "read", "hybrid-256", 1, 16384, 16384),
        # a chat's first tokens: a cache of one or two pages
        _case("attend-short", "attend", "dense-norm-128", 1, 1, 130),
        # odd head counts, ragged odd lengths from one row on
        _case("attend-odd", "attend", (3, 5, 64, 64, -1, False), 5, 1, 4099, page=256, ragged=True),
        # one stream behind a 16K prompt
        _case("attend-one", "attend", "hybrid-256", 1, 1, 16384),
        # a decode round of 8 streams behind prompts up to 32K
        _case("attend-round", "attend", "hybrid-256", 8, 1, 32768, ragged=True),
        # four streams behind 128K prompts of a dense model
        _case("attend-long", "attend", "dense-128", 4, 1, 131072),
    ]


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "read"])
    hd = rng.choice([64, 128, 256])
    rot = rng.choice([0, hd // 4, hd])
    if rot % (hd // 16):
        rot = 0
    norm, gated = rng.choice([-1, 0, 1]), rng.random() < 0.5
    hkv, G = rng.randint(1, 8), rng.randint(1, 8)
    page = rng.choice([128, 256, 512])
    most = 5.3e8                                        # cache values of the largest listed case, K alone

    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))
    if kind == "attend":
        R = spread(1, 32)
        ctx = spread(1, 131072)
        ctx = max(1, min(ctx, int(most / (R * hkv * hd))))
        return _case(None, kind, (hkv, G, hd, rot, norm, gated), R, 1, ctx, page=page, ragged=rng.random() < 0.7)
    if kind == "read":
        rows = min(spread(1, 65536), int(most / 4 / (hkv * hd)))
        return _case(None, kind, (hkv, G, hd, rot, norm, gated), 1, rows, rows + rng.randint(0, 300), page=page)
    if rng.random() < 0.5:
        R, rows = spread(1, 32), 1
    else:
        R, rows = rng.choice([1, 1, 2, 3]), spread(1, 16384)
        rows = max(1, min(rows, int(8e7 / (R * hkv * (G + 2) * hd))))
    return _case(None, kind, (hkv, G, hd, rot, norm, gated), R, rows, rows + spread(1, 8192), page=page,
                 ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------- the cache's layout
def code_places(hd, device):
    """Place, in 4-bit steps from the start of its part, of the code of (row of the block, dim): K's and V's, each
    [16, hd]."""
    k = torch.arange(16, device=device)[:, None]
    d = torch.arange(hd, device=device)[None, :]
    group = d // GROUP
    t, nib = d % GROUP // 8, d % 8
    word = (group // 4 ^ (k & 1)) * 16 + t * 4 + group % 4 if hd == 256 else t * (hd // GROUP) + group
    kp = k * hd + word * 8 + nib
    g, j = d % GROUP // 4, d % 4
    unit = 256 // hd                                   # rows in 128 bytes
    flip = {256: 2 * (k // 2 % 4), 128: 4 * (k // 2 % 4), 64: 8 * (k // 4 % 2)}[hd]
    chunk = (g + 8 * (k % unit)) ^ flip
    vp = (k // unit) * 256 + chunk * (hd // 8) + group * 4 + j
    return kp, vp


def row_places(device):
    """Place of a block's row among the 16 entries of a V scale or minimum."""
    k = torch.arange(16, device=device)
    return 4 * (k % 8 // 2) + 2 * (k // 8) + k % 2


def pack(kz, vz, hd):
    """(exponent byte, s, m, codes) of K and V rows in blocks [..., 16, *] -> the blocks' bytes [..., 20 hd + 32]."""
    (ke, ks, km, kc), (ve, vs, vm, vc) = kz, vz
    lead, dev = ke.shape[:-1], ke.device
    kp, vp = code_places(hd, dev)

    def nibbles(c, place):
        flat = torch.zeros(*lead, 16 * hd, dtype=torch.uint8, device=dev)
        flat[..., place.reshape(-1)] = c.to(torch.uint8).reshape(*lead, 16 * hd)
        return flat[..., 0::2] | (flat[..., 1::2] << 4)

    def halves(x):
        return x.half().contiguous().reshape(*lead, -1).view(torch.uint8)

    def turned(x):
        y = torch.empty(*lead, hd // GROUP, 16, dtype=torch.half, device=dev)
        y[..., row_places(dev)] = x.half().transpose(-1, -2)
        return halves(y)
    return torch.cat((nibbles(kc, kp), nibbles(vc, vp), halves(ks), halves(km), turned(vs), turned(vm),
                      ke.to(torch.uint8), ve.to(torch.uint8)), -1)


def unpack(blocks, hd):
    """The K and V values [..., 16, hd] (fp32) of blocks [..., 20 hd + 32]."""
    lead, dev = blocks.shape[:-1], blocks.device
    kp, vp = code_places(hd, dev)
    n = 16 * (hd // GROUP)

    def codes(part, place):
        nib = torch.stack((part & 15, part >> 4), -1).reshape(*lead, 16 * hd)
        return nib[..., place.reshape(-1)].reshape(*lead, 16, hd // GROUP, GROUP).float()

    def halves(i):
        return blocks[..., 16 * hd + 2 * n * i:16 * hd + 2 * n * (i + 1)].contiguous().view(torch.half).float()

    def values(c, s, m, byte):
        e = torch.where(byte == MARK, math.nan, (byte.int() - 127).float())[..., None]
        return (torch.exp2(e)[..., None] * (m[..., None] + s[..., None] * c)).reshape(*lead, 16, hd)
    ks, km = (halves(i).reshape(*lead, 16, -1) for i in (0, 1))
    vs, vm = (halves(i).reshape(*lead, -1, 16)[..., row_places(dev)].transpose(-1, -2) for i in (2, 3))
    return (values(codes(blocks[..., :8 * hd], kp), ks, km, blocks[..., 20 * hd:20 * hd + 16]),
            values(codes(blocks[..., 8 * hd:16 * hd], vp), vs, vm, blocks[..., 20 * hd + 16:]))


def quantise(y):
    """(exponent byte [...], s, m [..., hd / 32], codes [..., hd / 32, 32]) of rows y [..., hd] (values of bf16)."""
    a = y.abs().amax(-1)
    bad = ~(a < 2.0 ** 56)
    y = torch.where(bad[..., None], 0.0, y)
    e = torch.frexp(torch.where(bad | (a == 0), 1.0, a))[1] - 1
    e = e.clamp(-LIMIT, LIMIT)
    z = (y * torch.exp2(-e.float())[..., None]).unflatten(-1, (-1, GROUP))
    lo, hi = z.amin(-1), z.amax(-1)
    m = lo.half().float()
    s = ((hi - lo) / 15).half().float()
    c = torch.round((z - m[..., None]) / torch.where(s == 0, 1.0, s)[..., None]).clamp(0, 15)
    c = torch.where(s[..., None] == 0, 0.0, c)
    return torch.where(bad, MARK, e + 127), s, m, c


# ------------------------------------------------------------------------------------------------- inputs
def _lengths(c, g):
    """Rows each sequence's cache holds after the pass (appended or the query's own row among them)."""
    if not c["ragged"]:
        return [c["ctx"]] * c["R"]
    low = c["rows"]
    u = torch.rand(c["R"], generator=g, dtype=torch.float64).tolist()
    return [c["ctx"]] + [low + int((c["ctx"] - low) * x) for x in u[1:]]


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    hkv, hd, page, R, T = c["hkv"], c["hd"], c["page"], c["R"], c["rows"]
    hq = hkv * c["G"]
    lens = _lengths(c, host)
    held = [-(-n // page) for n in lens]
    total = sum(held) + 3
    order = torch.randperm(total, generator=host).to(torch.int32)
    pages = [p.to(dev) for p in order[:sum(held)].split(held)]
    pool = torch.zeros(total, hkv, page // 16, 20 * hd + 32, dtype=torch.uint8, device=dev)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=dev)
    # keys: a few strong channels, rows of different size; values: milder; both as the bf16 rows that a projection gives
    kbig = torch.exp(0.8 * rnd(hkv, 1, 1, hd))
    if c["kind"] != "append":
        for lo in range(0, total, 256):                # filled by pieces: the rows a long prompt left
            n = min(256, total - lo)
            k = (rnd(n, hkv, page // 16, 16, hd) * kbig * torch.exp(0.2 * rnd(n, hkv, page // 16, 16, 1))).bfloat16()
            v = (0.5 * rnd(n, hkv, page // 16, 16, hd)).bfloat16()
            pool[lo:lo + n] = pack(quantise(k.float()), quantise(v.float()), hd)
    st = dict(case=c, pool=pool, pages=pages, lens=lens)
    if c["kind"] == "read":
        st["row0"] = c["ctx"] - c["rows"]
        return st
    qw = hq * hd * (2 if c["gated"] else 1)
    if c["kind"] == "attend":
        st["q"] = rnd(R, hq, hd).bfloat16()                         # a normed, rotated query: logits a few units wide
        st["pos"] = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=dev)
        st["gate"] = rnd(R, qw).bfloat16() if c["gated"] else None
        st["scale"] = hd ** -0.5
        return st
    st["qkv"] = rnd(R * T, qw + 2 * hkv * hd).bfloat16()
    kc = st["qkv"][:, qw:qw + hkv * hd]
    kc.copy_(kc * kbig.reshape(-1))
    st["qw"] = qw
    st["row0"] = torch.tensor([n - T for n in lens], dtype=torch.int32, device=dev)
    st["norms"] = (None, None)
    if c["norm"] >= 0:
        st["norms"] = tuple((0.2 * rnd(hd) + (1.0 if c["norm"] == 0 else 0.0)).bfloat16() for _ in range(2))
    st["tables"] = None
    if c["rot"]:
        inv = 1e6 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
        ang = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None] * inv
        st["tables"] = (ang.cos().bfloat16(), ang.sin().bfloat16())
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _blocks_of(pool, pages):
    """Blocks [R, kv heads, blocks, bytes] of each sequence's pages (short tables repeat page 0 behind their end)."""
    table = torch.nn.utils.rnn.pad_sequence([p.long() for p in pages], batch_first=True)
    got = pool[table]                                               # [R, pages, heads, blocks, bytes]
    return got.transpose(1, 2).flatten(2, 3)


def _rounded(x):
    return x.float().bfloat16().float()


def _norm_rope(x, w, norm, cos, sin):
    """Head norm and rotation of rows x [N, heads, hd], rounded to bf16 where the bf16 model rounds."""
    if norm >= 0:
        xd, wd = x.double(), w.double()
        f = xd * (xd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        x = _rounded(_rounded(f) * w.float()) if norm == 0 else _rounded(f * (1.0 + wd))
    if cos is None:
        return x
    h = cos.shape[-1]
    a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    c, s = cos[:, None].float(), sin[:, None].float()
    return torch.cat((_rounded(_rounded(a * c) - _rounded(b * s)), _rounded(_rounded(b * c) + _rounded(a * s)), rest), -1)


def _append(st):
    c = st["case"]
    hkv, hd, page, R, T = c["hkv"], c["hd"], c["page"], c["R"], c["rows"]
    hq, qw, pool = hkv * c["G"], st["qw"], st["pool"]
    rows = st["row0"][:, None].long() + torch.arange(T, device=pool.device)          # [R, T]
    cos = sin = None
    if st["tables"] is not None:
        cos, sin = (t[rows.reshape(-1)] for t in st["tables"])
    x = st["qkv"].float()
    q = x[:, :qw].unflatten(-1, (hq, -1))[..., :hd]
    k = x[:, qw:qw + hkv * hd].unflatten(-1, (hkv, hd))
    v = x[:, qw + hkv * hd:].unflatten(-1, (hkv, hd))
    q = _norm_rope(q, st["norms"][0], c["norm"], cos, sin)
    k = _norm_rope(k, st["norms"][1], c["norm"], cos, sin)
    table = torch.nn.utils.rnn.pad_sequence([p.long() for p in st["pages"]], batch_first=True)
    at = table.gather(1, rows // page).reshape(-1)                                   # page of every row
    block, r = (rows % page // 16).reshape(-1), (rows % 16).reshape(-1)
    kp, vp = code_places(hd, pool.device)
    head = torch.arange(hkv, device=pool.device)[None, :]
    n, ng = R * T, hd // GROUP
    dest = ((at[:, None] * hkv + head) * (page // 16) + block[:, None]) * (20 * hd + 32)   # [N, heads] first byte
    flat = pool.view(-1)

    def put(quant, first, place, scales, per_row):
        byte, s, m, codes = quant
        codes = codes.reshape(n, hkv, hd).to(torch.uint8)
        spot = place[r]                                                              # [N, hd], in 4-bit steps
        order = spot.argsort(-1)
        spot, codes = spot.gather(-1, order), codes.gather(-1, order[:, None].expand(n, hkv, hd))
        both = codes[..., 0::2] | (codes[..., 1::2] << 4)
        flat[dest[..., None] + first + (spot[:, None, 0::2] >> 1)] = both
        unit = torch.arange(ng, device=flat.device)
        slot = r[:, None] * ng + unit if per_row else unit * 16 + row_places(flat.device)[r][:, None]
        for_s = dest[..., None] + scales + 2 * slot[:, None]
        halves = torch.stack((s, m), 2).half().reshape(n, hkv, 2, ng, 1).view(torch.uint8)
        where = torch.stack((for_s, for_s + 32 * ng), 2)[..., None] + torch.arange(2, device=flat.device)
        flat[where] = halves
        flat[dest + (20 * hd if per_row else 20 * hd + 16) + r[:, None]] = byte.to(torch.uint8)
    put(quantise(k), 0, kp, 16 * hd, True)
    put(quantise(v), 8 * hd, vp, 18 * hd, False)
    return q.bfloat16(), *_read(pool, st["pages"], rows)


def _read(pool, pages, rows):
    """bf16 K and V [R, kv heads, n, hd] of the sequences' cache rows [R, n]."""
    hkv, hd = pool.shape[1], (pool.shape[3] - 32) // 20
    table = torch.nn.utils.rnn.pad_sequence([p.long() for p in pages], batch_first=True)
    page = pool.shape[2] * 16
    lo, hi = rows[:, :1] // 16, rows[:, -1:] // 16
    span = int((rows.shape[1] + 30) // 16)                                           # blocks that n rows can touch
    blk = torch.minimum(lo + torch.arange(span, device=rows.device), hi)
    got = pool[table.gather(1, blk * 16 // page), :, blk % (page // 16)]             # [R, span, heads, bytes]
    k, v = unpack(got, hd)
    back = rows - lo * 16
    out = []
    for x in (k, v):
        x = x.transpose(1, 2).flatten(2, 3)                                          # [R, heads, span * 16, hd]
        out.append(x.gather(2, back[:, None, :, None].expand(-1, hkv, -1, hd)).bfloat16())
    return out


def _attend(st):
    c = st["case"]
    hkv, G, hd = c["hkv"], c["G"], c["hd"]
    k, v = unpack(_blocks_of(st["pool"], st["pages"]), hd)
    k, v = k.flatten(2, 3), v.flatten(2, 3)                                          # [R, heads, n, hd]
    q = st["q"].float().unflatten(1, (hkv, G))
    s = torch.matmul(q, k.transpose(-1, -2)) * st["scale"]
    dead = torch.arange(k.shape[2], device=k.device) > st["pos"][:, None]            # [R, n]
    s = s.masked_fill(dead[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.masked_fill(dead[:, None, :, None], 0.0)).flatten(1, 2)
    if c["gated"]:
        o = o / (1.0 + torch.exp(-st["gate"].float().unflatten(1, (hkv * G, 2, hd))[:, :, 1]))
    return o.flatten(1, 2).bfloat16()


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    st, c = state, state["case"]
    if own:
        return _run_own(st, c)
    if c["kind"] == "attend":
        return _attend(st)
    if c["kind"] == "append":
        return _append(st)
    rows = st["row0"] + torch.arange(c["rows"], device=st["pool"].device)
    k, v = _read(st["pool"], st["pages"], rows[None])
    return k[0], v[0]


def _run_own(st, c):
    from ridgefill_data_b200.ops import kv4
    hkv, hd = c["hkv"], c["hd"]
    if c["kind"] == "read":
        return kv4.read(st["pool"], st["pages"][0], c["rows"], st["row0"])
    if c["kind"] == "attend":
        gate = st["gate"][:, hd:] if c["gated"] else None
        return kv4.attention(st["q"], st["pool"], st["pages"], st["pos"], st["scale"], gate=gate, gate_head=2 * hd)
    q = kv4.append(st["qkv"], st["pool"], st["pages"], st["row0"], q_heads=hkv * c["G"], gated=c["gated"],
                   q_norm=st["norms"][0], k_norm=st["norms"][1], norm_mode=c["norm"], eps=1e-6, tables=st["tables"],
                   rot=c["rot"])
    return q, *kv4.read(st["pool"], st["pages"], c["rows"], st["row0"])


def work(case):
    c = case
    hkv, hd, R, T = c["hkv"], c["hd"], c["R"], c["rows"]
    hq = hkv * c["G"]
    row = hkv * (1.25 * hd + 2)                                    # a cache row's bytes, K and V
    if c["kind"] == "read":
        return {"bytes": T * (row + 4 * hkv * hd), "flops": T * 4 * hkv * hd}
    if c["kind"] == "append":                                      # rows in, q out, cache rows written, then read back
        n = R * T
        return {"bytes": n * (2 * (2 * hq + 2 * hkv) * hd + 2 * row + 4 * hkv * hd),
                "flops": n * hd * (10 * hq + 30 * hkv)}
    keys = (R + 1) * c["ctx"] // 2 if c["ragged"] else R * c["ctx"]     # ragged: one full cache, the others half on average
    return {"bytes": keys * row + R * hq * hd * (6 if c["gated"] else 4), "flops": 4 * keys * hq * hd}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _cached(pool, page_ids, rows, head, which):
    """Values [rows, hd] in 64 bits of one sequence's K (which 0) or V (1) at a KV head, read byte by byte from the
    layout's definition."""
    hd = (pool.shape[3] - 32) // 20
    page, ng, dev = pool.shape[2] * 16, hd // 32, pool.device
    page_ids = page_ids.long()
    b = pool[page_ids[rows // page], head, rows % page // 16]                        # [n, bytes]
    r = (rows % 16)[:, None]
    d = torch.arange(hd, device=dev)[None, :]
    i = d // 32                                                                      # the dim's group
    if which == 0:
        if hd == 256:
            byte = r * 128 + 64 * ((i >= 4).long() ^ (r % 2)) + 16 * (d % 32 // 8) + 4 * (i % 4) + d % 8 // 2
        else:
            byte = r * (hd // 2) + (d % 32 // 8) * (hd // 8) + 4 * i + d % 8 // 2
        sb = 16 * hd + 2 * (r * ng + i)
        mb, eb = sb + 32 * ng, 20 * hd + r
    else:
        piece = d % 32 // 4
        if hd == 256:
            byte = r * 128 + 16 * (piece ^ (2 * (r // 2 % 4)))
        elif hd == 128:
            byte = r // 2 * 128 + 8 * ((piece + 8 * (r % 2)) ^ (4 * (r // 2 % 4)))
        else:
            byte = r // 4 * 128 + 4 * ((piece + 8 * (r % 4)) ^ (8 * (r // 4 % 2)))
        byte = 8 * hd + byte + 2 * i + d % 4 // 2
        slot = 4 * (r % 8 // 2) + 2 * (r // 8) + r % 2
        sb = 18 * hd + 2 * (16 * i + slot)
        mb, eb = sb + 32 * ng, 20 * hd + 16 + r
    code = b.gather(1, byte) >> (4 * (d % 2)).to(torch.uint8) & 15

    def half(at):                                       # a 16-bit float from its two bytes
        bits = b.gather(1, at).long() | b.gather(1, at + 1).long() << 8
        sign, ex, frac = 1.0 - 2.0 * (bits >> 15).double(), bits >> 10 & 31, (bits & 1023).double()
        return sign * torch.where(ex == 0, torch.ldexp(frac, torch.tensor(-24, device=dev)),
                                  torch.ldexp(1024 + frac, ex - 25))
    e = b.gather(1, eb.expand(-1, 1)).long()
    value = torch.ldexp(half(mb) + half(sb) * code.double(), e - 127)
    return torch.where(e == 255, math.nan, value)


def _same(x):
    return x


def _to_bf16(x):
    return x.float().bfloat16().double()


def _turn(x, w, c, tables, rows, to=_same):
    """Norm and rotation of rows x [N, heads, hd] in 64 bits; `to` rounds where the bf16 model does."""
    if c["norm"] >= 0:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["hd"] + 1e-6)
        x = to(to(x) * w.double()) if c["norm"] == 0 else to(x * (1.0 + w.double()))
    h = c["rot"] // 2
    if not h:
        return x
    cos, sin = (t.double()[rows][:, None] for t in tables)
    left, right = x[..., :h], x[..., h:2 * h]
    return torch.cat((to(to(left * cos) + to(-right * sin)), to(to(left * sin) + to(right * cos)), x[..., 2 * h:]), -1)


def _kept(y):
    """The values in 64 bits that the cache keeps of rows y [..., hd]."""
    top = y.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top == 0, 1.0, top))).clamp(-LIMIT, LIMIT)
    z = (y / 2.0 ** e).reshape(*y.shape[:-1], -1, GROUP)
    low = z.amin(-1, keepdim=True).half().double()
    step = ((z.amax(-1, keepdim=True) - z.amin(-1, keepdim=True)) / 15).half().double()
    code = torch.where(step > 0, torch.clamp(torch.round((z - low) / step), 0, 15), 0.0)
    return (low + step * code).reshape(y.shape) * 2.0 ** e


def exact(case, seed):
    c = case
    hkv, G, hd, R, T = c["hkv"], c["G"], c["hd"], c["R"], c["rows"]
    st = prepare(case, seed)
    dev = st["pool"].device
    if c["kind"] == "read":
        rows = torch.arange(st["row0"], st["row0"] + T, device=dev)
        return tuple(torch.stack([_cached(st["pool"], st["pages"][0], rows, h, w) for h in range(hkv)]) for w in (0, 1))
    if c["kind"] == "attend":
        out = torch.empty(R, hkv * G, hd, dtype=torch.float64, device=dev)
        for s, n in enumerate(st["lens"]):
            rows = torch.arange(n, device=dev)
            for h in range(hkv):
                x = _cached(st["pool"], st["pages"][s], rows, h, 0) @ st["q"][s, h * G:(h + 1) * G].double().T
                p = torch.softmax(x * st["scale"], 0)
                out[s, h * G:(h + 1) * G] = p.T @ _cached(st["pool"], st["pages"][s], rows, h, 1)
        if c["gated"]:
            out = out * torch.sigmoid(st["gate"].double().reshape(R, hkv * G, 2 * hd)[..., hd:])
        return out.reshape(R, -1)
    # append: q by the formula alone; K with the roundings that the cached row is defined by, V as it is
    rows = (st["row0"].long()[:, None] + torch.arange(T, device=dev)).reshape(-1)
    x = st["qkv"].double()
    q, k, v = x[:, :st["qw"]].reshape(R * T, hkv * G, -1)[..., :hd], x[:, st["qw"]:-hkv * hd], x[:, -hkv * hd:]
    k, v = (y.reshape(R * T, hkv, hd) for y in (k, v))
    k = _turn(k, st["norms"][1], c, st["tables"], rows, _to_bf16)
    return (_turn(q, st["norms"][0], c, st["tables"], rows),
            *(_kept(y).reshape(R, T, hkv, hd).transpose(1, 2) for y in (k, v)))
