"""Measured cases of the operators for serving many sequences and beams: rotary positions, attention over a paged
key-value cache, the pages' own operations, and beam selection.

`run` computes each in plain torch operations, or, where `own` is true, calls the framework's C entry points. A case
is made by `prepare`; lengths, page fills and parents follow from the case alone, data and page placement from the seed.
"""
import ctypes
import math
import random

import torch

own = False

DEVICE = "cuda"
PAD = 2                            # the one token that a finished beam goes on with
ATTN_WORKSPACE = 32 << 20          # tl_paged_attn_workspace never asks for more

# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one new token of one sequence, 32 heads of 128: queries and keys rotated, stored in the cache's page
        dict(name="append_one_token", op="append", tokens=1, prompt=0, heads=32, kv_heads=32, dim=128, rot=128, half=False,
             scaling="none", page=16, hnd=False, top=2048, lens_seed=1),
        # a decode step of 192 sequences with shared heads, half layout, part of the head rotated, some rows padding
        dict(name="append_batch_part", op="append", tokens=192, prompt=0, heads=32, kv_heads=8, dim=128, rot=64, half=True,
             scaling="parts", page=16, hnd=False, top=60000, lens_seed=2),
        # a long prompt rotated in place, positions beyond the trained length
        dict(name="rotary_prompt_16k", op="rotary", tokens=16384, heads=40, dim=128, rot=128, half=False, scaling="ramp",
             top=500000, inverse=False),
        # one sequence of a few hundred tokens, a head of its own for every query head: latency
        dict(name="attn_one_short", op="attn", batch=1, low=333, high=333, heads=32, kv_heads=32, dim=128, page=16, hnd=False,
             empty=0, lens_seed=3),
        # an ordinary batch with shared heads and ragged lengths
        dict(name="attn_batch_ragged", op="attn", batch=48, low=200, high=6000, heads=32, kv_heads=8, dim=128, page=16, hnd=False,
             empty=1, lens_seed=4),
        # four long contexts
        dict(name="attn_long_context", op="attn", batch=4, low=100000, high=131072, heads=32, kv_heads=8, dim=128, page=64,
             hnd=False, empty=0, lens_seed=5),
        # odd sizes: heads of 80, groups of five, pages of 24 laid out by head, empty rows
        dict(name="attn_odd", op="attn", batch=37, low=1, high=2300, heads=15, kv_heads=3, dim=80, page=24, hnd=True, empty=3,
             lens_seed=6),
        # samples branch off shared prompts and get room for their next token: free, fork, reserve with copied last pages
        dict(name="fork_samples", op="fork", parents=16, children=128, layers=8, low=100, high=4000, kv_heads=8, dim=128, page=16,
             lens_seed=7),
        # a fragmented pool of 32 layers moved together
        dict(name="compact_pool", op="compact", pages=2048, live=900, layers=32, kv_heads=8, dim=128, page=16, rows=64,
             lens_seed=8),
        # four beams of one sequence: latency
        dict(name="select_one", op="select", batch=1, beams=4, vocab=32000, k=8, finished=0, dead=0),
        # sixty-four sequences of eight beams, some finished, some dead
        dict(name="select_batch", op="select", batch=64, beams=8, vocab=32000, k=16, finished=20, dead=10),
        # contiguous caches of the beams follow their parents
        dict(name="reorder_caches", op="reorder", outer=16, rows=32, used=700 * 1024, pitch=1024 * 1024, lens_seed=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "attn", "attn", "attn", "fork", "compact", "select", "select", "reorder"])
    seed = rng.randrange(1 << 30)
    dim = rng.choice([32, 48, 64, 64, 72, 80, 96, 112, 128, 128, 128, 160, 192, 256])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
    page = rng.choice([1, 8, 16, 16, 16, 24, 32, 64, 100, 128])
    while kv * group > 64:
        group = max(1, group // 2)
    if op == "rotary":
        heads = kv * group
        tokens = _log(rng, 1, max(1, min(16384, 16384 * 40 * 128 // (heads * dim))))
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, 8 * max(1, dim // 32)]),
                    half=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "parts", "ramp"]),
                    top=max(tokens, _log(rng, 64, 1 << 20)), inverse=rng.random() < 0.3)
    if op == "append":
        prompt = rng.choice([0, 0, 1])
        tokens = _log(rng, 1, 6000 if prompt else 512)
        return dict(op=op, tokens=tokens, prompt=prompt, heads=kv * group, kv_heads=kv, dim=dim, rot=rng.choice([dim, dim // 2, 0]),
                    half=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "parts", "ramp"]), page=page,
                    hnd=rng.random() < 0.3, top=max(2 * tokens, _log(rng, 64, 100000)), lens_seed=seed)
    if op == "attn":
        most = 4 * 115000 * 8 * 128               # cached values of the largest listed case
        high = _log(rng, 1, 131072)
        batch = _log(rng, 1, max(1, min(256, most // (high * kv * dim))))
        high = max(1, min(high, most // (batch * kv * dim)))
        return dict(op=op, batch=batch, low=max(1, high // rng.choice([1, 2, 10])), high=high, heads=kv * group, kv_heads=kv, dim=dim,
                    page=page, hnd=rng.random() < 0.3, empty=rng.choice([0, 0, 1]) if batch > 1 else 0, lens_seed=seed)
    if op == "fork":
        parents = _log(rng, 1, 32)
        high = _log(rng, 4, 6000)
        return dict(op=op, parents=parents, children=parents * rng.choice([1, 2, 4, 5, 8]), layers=rng.randint(1, 8), low=max(1, high // 8),
                    high=high, kv_heads=min(kv, 8), dim=dim, page=rng.choice([8, 16, 16, 24, 32]), lens_seed=seed)
    if op == "compact":
        pages = _log(rng, 16, 2048)
        return dict(op=op, pages=pages, live=max(1, int(pages * rng.uniform(0.2, 0.8))), layers=rng.randint(1, 32), kv_heads=min(kv, 8),
                    dim=min(dim, 128), page=rng.choice([8, 16, 16]), rows=rng.randint(1, 64), lens_seed=seed)
    if op == "select":
        beams = _log(rng, 1, 16)
        vocab = _log(rng, 500, 130000)
        batch = _log(rng, 1, max(1, min(64, 64 * 8 * 32000 // (beams * vocab))))
        k = min(beams * rng.choice([1, 2]), 32)
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, k=k, finished=rng.randint(0, batch * beams // 8),
                    dead=rng.randint(0, batch * beams // 8))
    rows = _log(rng, 2, 64)
    outer = rng.randint(1, 16)
    pitch = 8 * _log(rng, 64, 16 * 32 * 1024 * 1024 // (rows * outer * 8))
    return dict(op="reorder", outer=outer, rows=rows, used=max(1, int(pitch * rng.uniform(0.1, 1.0))), pitch=pitch, lens_seed=seed)


def _lengths(c):
    r = random.Random(c["lens_seed"])
    n = [r.randint(c["low"], c["high"]) for _ in range(c["batch"])]
    for i in r.sample(range(c["batch"]), c["empty"]):
        n[i] = 0
    return n


def _fork_plan(c):
    """Lengths of the parents, and the parent of each child."""
    r = random.Random(c["lens_seed"])
    return [r.randint(c["low"], c["high"]) for _ in range(c["parents"])], [r.randrange(c["parents"]) for _ in range(c["children"])]


def _append_plan(c):
    """(row, position) of every token; position -1 is padding. Rows: one a sequence."""
    r = random.Random(c["lens_seed"])
    if c["prompt"]:                       # one sequence continued by `tokens` tokens, a few padding ones behind
        start, pad = r.randint(0, c["top"] - c["tokens"]), c["tokens"] // 20
        pos = [start + i if i < c["tokens"] - pad else -1 for i in range(c["tokens"])]
        return [0] * c["tokens"], pos, 1
    pos = [r.randrange(c["top"]) for _ in range(c["tokens"])]
    for i in range(0, c["tokens"], 17):
        if i:
            pos[i] = -1
    return list(range(c["tokens"])), pos, c["tokens"]


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------


def _freqs(rot, scaling):
    """(radians a position for each pair, magnitude): the scaled forms for long contexts, base 10000."""
    n, base, factor, orig = rot // 2, 10000.0, 8.0, 4096.0
    if scaling == "base":
        base *= factor ** (rot / max(1, rot - 2))
    f = [base ** (-2.0 * i / rot) for i in range(n)]
    mag = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "parts":              # by wavelength: kept below orig / 4, divided above orig, blended between
        g = []
        for x in f:
            turns = orig * x / (2 * math.pi)
            s = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            g.append((1 - s) * x / factor + s * x)
        f = g
    elif scaling == "ramp":               # by index: the pairs that turn 32 to 1 times over the trained length
        lo = rot * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(base))
        hi = rot * math.log(orig / (1 * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        s = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(n)]
        f = [(1 - a) * x + a * x / factor for a, x in zip(s, f)]
        mag = 0.1 * math.log(factor) + 1.0
    return f, mag


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, dtype=torch.float16, device=DEVICE).normal_(0.0, std, generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _pool(g, layers, pages, page, kv_heads, dim, hnd):
    """A pool of pages as [layers, pages, page, kv_heads, dim], stored by token or by head."""
    if hnd:
        return _normal(g, layers, pages, kv_heads, page, dim).transpose(2, 3)
    return _normal(g, layers, pages, page, kv_heads, dim)


def _table(counts, pages, width, g, start=0):
    """Page table [rows, width] with counts[r] pages of the pool in random order, -1 behind them."""
    order = torch.randperm(pages, generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)
    first = torch.tensor([0] + counts, dtype=torch.int64, device=DEVICE).cumsum(0)[:-1] + start
    n = torch.tensor(counts, dtype=torch.int64, device=DEVICE)
    at = torch.arange(width, device=DEVICE)
    valid = at[None, :] < n[:, None]
    idx = (first[:, None] + at[None, :]).clamp(max=pages - 1)
    return torch.where(valid, order[idx], torch.full_like(order[idx], -1)).contiguous()


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = {"case": c}
    op = c["op"]
    if op == "rotary":
        f, s["mag"] = _freqs(c["rot"], c["scaling"])
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device=DEVICE)
        s["x"] = _normal(g, c["tokens"], c["heads"], c["dim"])
        s["out"] = torch.empty_like(s["x"])
        start = c["top"] - c["tokens"]
        s["pos"] = _ints(list(range(start, start + c["tokens"])))
    elif op == "append":
        rows, pos, n_rows = _append_plan(c)
        p = c["page"]
        # every row owns just the page that a token goes to, except a prompt's, which owns them all
        width = -(-c["top"] // p)
        if c["prompt"]:
            pages = width
            table = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)[None, :].contiguous()
        else:
            pages = n_rows
            order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
            table = torch.full((n_rows, width), -1, dtype=torch.int32, device=DEVICE)
            table[torch.arange(n_rows, device=DEVICE), torch.tensor(pos, device=DEVICE).clamp(min=0) // p] = order
        f, s["mag"] = _freqs(c["rot"], c["scaling"]) if c["rot"] else ([0.0], 1.0)
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device=DEVICE)
        s["rows"], s["pos"], s["table"] = _ints(rows), _ints(pos), table
        s["qkv"] = _normal(g, c["tokens"], c["heads"] + 2 * c["kv_heads"], c["dim"])      # one fused projection
        s["q_out"] = torch.zeros(c["tokens"], c["heads"], c["dim"], dtype=torch.float16, device=DEVICE)
        s["k"] = _pool(g, 1, pages + 1, p, c["kv_heads"], c["dim"], c["hnd"])       # the last page takes the plain form's padding
        s["v"] = _pool(g, 1, pages + 1, p, c["kv_heads"], c["dim"], c["hnd"])
        s["pages"] = pages
    elif op == "attn":
        n = _lengths(c)
        counts = [-(-x // c["page"]) for x in n]
        width, pages = max(1, max(counts)), sum(counts) + 3
        s["lengths"], s["table"], s["pages"] = _ints(n), _table(counts, pages, width, g), pages
        s["k"] = _pool(g, 1, pages, c["page"], c["kv_heads"], c["dim"], c["hnd"])
        s["v"] = _pool(g, 1, pages, c["page"], c["kv_heads"], c["dim"], c["hnd"])
        # what lies behind a row's last token was never written: it may hold anything
        some = [(i, (x - 1) // c["page"], (x - 1) % c["page"]) for i, x in enumerate(n) if x]
        row, last, slot = (torch.tensor(v, device=DEVICE) for v in zip(*some))
        pg = s["table"][row, last].long()
        bad = (torch.arange(c["page"], device=DEVICE)[None, :] > slot[:, None])[:, :, None, None]
        s["k"][0, pg] = s["k"][0, pg].masked_fill(bad, float("nan"))
        s["v"][0, pg] = s["v"][0, pg].masked_fill(bad, float("nan"))
        s["q"] = _normal(g, c["batch"], c["heads"], c["dim"], std=1.5)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["batch"], c["heads"], dtype=torch.float32, device=DEVICE)
        s["work"] = torch.zeros(ATTN_WORKSPACE, dtype=torch.uint8, device=DEVICE)
    elif op == "fork":
        n, par = _fork_plan(c)
        counts = [-(-x // c["page"]) for x in n]
        rows = c["parents"] + c["children"]
        width, pages = max(counts) + 1, sum(counts) + 2 * c["children"]
        table = torch.full((rows, width), -1, dtype=torch.int32, device=DEVICE)
        table[: c["parents"]] = _table(counts, pages, width, g)
        ref = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
        used = table[: c["parents"]].reshape(-1)
        ref.index_add_(0, used.clamp(min=0).long(), (used >= 0).to(torch.int32))
        s["table"], s["ref"], s["pages"] = table, ref, pages
        s["lengths"] = _ints(n + [0] * c["children"])
        s["drop"] = _ints(list(range(c["parents"])) + [-1] * c["children"])
        s["fork"] = _ints(list(range(c["parents"])) + par)
        s["new"] = _ints([0] * c["parents"] + [1] * c["children"])
        s["k"] = _pool(g, c["layers"], pages + 1, c["page"], c["kv_heads"], c["dim"], False)    # the last page: the plain form's spare
        s["v"] = _pool(g, c["layers"], pages + 1, c["page"], c["kv_heads"], c["dim"], False)
        s["result"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        s["work"] = torch.zeros(65536 + 16 * (rows + pages), dtype=torch.uint8, device=DEVICE)
    elif op == "compact":
        rows = min(c["rows"], c["live"])
        counts = [c["live"] // rows + (i < c["live"] % rows) for i in range(rows)]
        s["table0"] = _table(counts, c["pages"], max(counts), g)
        s["table"] = s["table0"].clone()
        ref = torch.zeros(c["pages"], dtype=torch.int32, device=DEVICE)
        used = s["table0"].reshape(-1)
        ref.index_add_(0, used.clamp(min=0).long(), (used >= 0).to(torch.int32))
        s["ref0"], s["ref"], s["pages"] = ref, ref.clone(), c["pages"]
        s["lengths"] = _ints([x * c["page"] for x in counts])
        s["k"] = _pool(g, c["layers"], c["pages"], c["page"], c["kv_heads"], c["dim"], False)
        s["v"] = _pool(g, c["layers"], c["pages"], c["page"], c["kv_heads"], c["dim"], False)
        s["moved"] = torch.empty(c["pages"], dtype=torch.int32, device=DEVICE)
        s["result"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        s["work"] = torch.zeros(65536 + 16 * (rows + c["pages"]), dtype=torch.uint8, device=DEVICE)
    elif op == "select":
        rows = c["batch"] * c["beams"]
        s["logits"] = _normal(g, rows, c["vocab"], std=2.5)
        s["scores"] = torch.empty(rows, dtype=torch.float32, device=DEVICE).uniform_(-12.0, -8.0, generator=g)
        order = torch.randperm(rows, generator=g, device=DEVICE)
        s["scores"][order[: c["dead"]]] = -math.inf
        s["finished"] = torch.zeros(rows, dtype=torch.uint8, device=DEVICE)
        s["finished"][order[c["dead"]: c["dead"] + c["finished"]]] = 1
        s["values"] = torch.empty(c["batch"], c["k"], dtype=torch.float32, device=DEVICE)
        s["parents"] = torch.empty(c["batch"], c["k"], dtype=torch.int32, device=DEVICE)
        s["tokens"] = torch.empty(c["batch"], c["k"], dtype=torch.int32, device=DEVICE)
        s["work"] = torch.zeros(65536 + 8 * c["batch"] + 64 * rows * (8 * c["k"] + 32), dtype=torch.uint8, device=DEVICE)
    else:
        r = random.Random(c["lens_seed"])
        s["src"] = _normal(g, c["outer"], c["rows"], c["pitch"])
        s["dst"] = torch.zeros_like(s["src"])
        s["parents"] = _ints([r.randrange(c["rows"]) for _ in range(c["rows"])])
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass: plain torch operations
# ---------------------------------------------------------------------------------------------------------------


def _rotated(x, pos, freqs, mag, rot, half, inverse=False):
    """x [tokens, heads, dim] turned by its position, in 32 bits; the angles of far positions in 64."""
    angle = pos.double()[:, None] * freqs[None, :]
    if inverse:
        angle = -angle
    cos, sin = (angle.cos() * mag).float()[:, None, :], (angle.sin() * mag).float()[:, None, :]
    y = x.float()
    part = y[..., :rot]
    if half:
        a, b = part[..., : rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).half()


def _plain_rotary(s):
    c = s["case"]
    s["out"].copy_(_rotated(s["x"], s["pos"], s["freqs"], s["mag"], c["rot"], c["half"], c["inverse"]))
    return [s["out"]]


def _plain_append(s):
    c = s["case"]
    h, kv, p = c["heads"], c["kv_heads"], c["page"]
    q, k, v = s["qkv"][:, :h], s["qkv"][:, h:h + kv], s["qkv"][:, h + kv:]
    live = s["pos"] >= 0
    pos = s["pos"].clamp(min=0)
    if c["rot"]:
        q, k = (_rotated(x, pos, s["freqs"], s["mag"], c["rot"], c["half"]) for x in (q, k))
    page = s["table"][s["rows"].long(), (pos // p).long()]
    page = torch.where(live, page, torch.full_like(page, s["pages"])).long()
    s["k"][0, page, (pos % p).long()] = k
    s["v"][0, page, (pos % p).long()] = v
    s["q_out"].copy_(torch.where(live[:, None, None], q, s["q_out"]))
    return [s["q_out"], s["k"][0, : s["pages"]], s["v"][0, : s["pages"]]]


def _plain_attn(s):
    c = s["case"]
    b, h, kv, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    table = s["table"].clamp(min=0).long()
    seen = torch.arange(table.shape[1] * c["page"], device=DEVICE)[None, :] < s["lengths"][:, None]
    k = s["k"][0][table].reshape(b, -1, kv, d).float()
    q = s["q"].float().reshape(b, kv, h // kv, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    del k
    x = torch.where(seen[:, None, None, :], x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    v = s["v"][0][table].reshape(b, -1, kv, d).float()
    v = torch.where(seen[:, :, None, None], v, torch.zeros_like(v))
    o = torch.matmul(e, v.permute(0, 2, 1, 3)) / torch.where(total == 0, torch.ones_like(total), total)
    lse = top + torch.log(total)
    return [o.reshape(b, h, d).half(), lse.reshape(b, h)]


def _plain_fork_rows(s, parents):
    """Row r becomes a copy of row parents[r] by reference; -1 empties it."""
    old = s["table"]
    take = parents.clamp(min=0).long()
    new = torch.where((parents >= 0)[:, None], old[take], torch.full_like(old, -1))
    n = torch.where(parents >= 0, s["lengths"][take], torch.zeros_like(s["lengths"]))
    flat_old, flat_new = old.reshape(-1), new.reshape(-1)
    s["ref"].index_add_(0, flat_new.clamp(min=0).long(), (flat_new >= 0).to(torch.int32))
    s["ref"].index_add_(0, flat_old.clamp(min=0).long(), -(flat_old >= 0).to(torch.int32))
    s["table"].copy_(new)
    s["lengths"].copy_(n)


def _plain_reserve(s):
    """Room for s["new"] (0 or 1) more tokens of each row: a shared last page is copied, a full one followed by a new one."""
    p = s["case"]["page"]
    n, add, table, ref = s["lengths"].long(), s["new"].long(), s["table"], s["ref"]
    rows = torch.arange(n.shape[0], device=DEVICE)
    fill = n % p
    at = n // p                                                        # the page that the next token goes to
    page = table.gather(1, at[:, None])[:, 0].long()
    writes = (add > 0) & (fill > 0)                                    # into a page that is there already
    where = page.clamp(min=0)
    writers = torch.zeros_like(ref).index_add_(0, where, writes.to(torch.int32))
    keeper = torch.full_like(ref, -1).long().scatter_reduce_(0, where, torch.where(writes, rows, torch.full_like(rows, -1)), "amax")
    keeps = writes & (writers[where] == ref[where]) & (keeper[where] == rows)
    copies = writes & ~keeps
    needs = copies | ((add > 0) & (fill == 0))
    free = torch.argsort((ref > 0).to(torch.int32), stable=True)       # the free pages first, ascending
    got = free[(needs.long().cumsum(0) - 1).clamp(min=0)]
    ref.index_add_(0, where, -copies.to(torch.int32))
    ref.index_add_(0, got, needs.to(torch.int32))
    table.scatter_(1, at[:, None], torch.where(needs, got, page).to(torch.int32)[:, None])
    # copied pages: the filled tokens only; the other rows turn to the spare page
    spare = torch.full_like(where, s["pages"])
    src, dst = torch.where(copies, where, spare), torch.where(copies, got, spare)
    filled = (torch.arange(p, device=DEVICE)[None, :] < fill[:, None])[None, :, :, None, None]
    s["k"][:, dst] = torch.where(filled, s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(filled, s["v"][:, src], s["v"][:, dst])
    s["lengths"].add_(s["new"])


def _fork_out(s):
    return [s["table"], s["lengths"], s["ref"], s["result"], s["k"][:, : s["pages"]], s["v"][:, : s["pages"]]]


def _plain_fork(s):
    _plain_fork_rows(s, s["drop"])
    _plain_fork_rows(s, s["fork"])
    _plain_reserve(s)
    return _fork_out(s)


def _compact_out(s):
    return [s["table"], s["ref"], s["moved"], s["result"], s["k"], s["v"]]


def _plain_compact(s):
    s["table"].copy_(s["table0"])                                      # the fragmented pool again
    s["ref"].copy_(s["ref0"])
    ref, pages = s["ref"], s["pages"]
    ids = torch.arange(pages, device=DEVICE)
    live = ref > 0
    total = live.sum()
    moves = live & (ids >= total)                                      # the highest live page goes to the lowest free one
    slots = torch.argsort((~(~live & (ids < total))).to(torch.int32), stable=True)
    rank = (moves.long().flip(0).cumsum(0).flip(0) - 1).clamp(min=0)
    to = torch.where(moves, slots[rank], ids)
    s["moved"].copy_(torch.where(live, to, torch.full_like(to, -1)))
    # no more pages can move than are live, or than are free; the places behind the last move hold pages that stay
    most = min(s["case"]["live"], pages - s["case"]["live"])
    down = torch.argsort(torch.where(moves, -ids, torch.ones_like(ids)), stable=True)
    dst = slots[:most]
    src = torch.where(torch.arange(most, device=DEVICE) < moves.sum(), down[:most], dst)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    new = torch.zeros_like(ref).index_add_(0, torch.where(live, to, ids), torch.where(live, ref, torch.zeros_like(ref)))
    ref.copy_(new)
    t = s["table"]
    t.copy_(torch.where(t >= 0, to[t.clamp(min=0).long()].to(torch.int32), t))
    s["result"].copy_(total.to(torch.int32)[None])
    return _compact_out(s)


def _plain_select(s):
    c = s["case"]
    b, w, n = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()
    x = x - torch.logsumexp(x, -1, keepdim=True) + s["scores"].double()[:, None]      # 64 bits: values next to one another
    done = s["finished"].bool()[:, None]
    pad = torch.zeros(n, dtype=torch.bool, device=DEVICE)
    pad[PAD] = True
    only = torch.where(pad[None, :], s["scores"].double()[:, None], torch.full_like(x, -math.inf))
    x = torch.where(done, only, x).reshape(b, w * n)
    v, at = torch.sort(x, dim=-1, descending=True, stable=True)
    v, at = v[:, : c["k"]], at[:, : c["k"]]
    first = (torch.arange(b, device=DEVICE) * w)[:, None]
    return [v.float(), (first + at // n).to(torch.int32), (at % n).to(torch.int32)]


def _plain_reorder(s):
    u = s["case"]["used"]
    s["dst"][:, :, :u] = s["src"][:, s["parents"].long(), :u]
    return [s["dst"]]


# ---------------------------------------------------------------------------------------------------------------
# one pass: the framework's calls
# ---------------------------------------------------------------------------------------------------------------


def _own(s):
    """The library, initialised, and the cache's handle: made at a state's first pass and kept, as a server keeps them."""
    import tensorlib_b200 as tl
    lib = tl.load()
    tl.check(lib.tl_init(torch.cuda.current_device()), "tl_init")
    s["lib"], s["check"] = lib, tl.check
    if "k" in s:
        k, c = s["k"], s["case"]
        ref = s["ref"].data_ptr() if "ref" in s else None
        lengths = s["lengths"].data_ptr() if "lengths" in s else None
        cache = tl.tl_paged_cache(k.data_ptr(), s["v"].data_ptr(), k.stride(0), k.stride(1), k.stride(2), k.stride(3), k.shape[0],
                                  s["pages"], c["page"], c["kv_heads"], c["dim"], s["table"].shape[0], s["table"].shape[1],
                                  s["table"].data_ptr(), lengths, ref)
        s["cache"] = ctypes.byref(cache)
    return lib


def _own_pass(s):
    c, lib = s["case"], s.get("lib") or _own(s)
    op, stream, check = c["op"], torch.cuda.current_stream().cuda_stream, s["check"]
    if op == "rotary":
        x, o = s["x"], s["out"]
        check(lib.tl_rotary_f16(x.data_ptr(), o.data_ptr(), s["pos"].data_ptr(), s["freqs"].data_ptr(), s["mag"], c["tokens"], c["heads"],
                                c["dim"], c["rot"], int(c["half"]), int(c["inverse"]), x.stride(0), x.stride(1), o.stride(0), o.stride(1),
                                stream), "tl_rotary_f16")
        return [o]
    if op == "append":
        q = s["qkv"].data_ptr()
        k = q + 2 * c["heads"] * c["dim"]
        v = k + 2 * c["kv_heads"] * c["dim"]
        w = s["qkv"].stride(0)
        check(lib.tl_rotary_append_f16(s["cache"], 0, q, s["q_out"].data_ptr(), k, v, s["rows"].data_ptr(), s["pos"].data_ptr(),
                                       s["freqs"].data_ptr(), s["mag"], c["tokens"], c["heads"], c["rot"], int(c["half"]), w,
                                       s["q_out"].stride(0), w, stream), "tl_rotary_append_f16")
        return [s["q_out"], s["k"][0, : s["pages"]], s["v"][0, : s["pages"]]]
    if op == "attn":
        check(lib.tl_paged_attn_decode_f16(s["cache"], 0, s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), None, c["batch"],
                                           c["heads"], 1.0 / math.sqrt(c["dim"]), s["q"].stride(0), s["out"].stride(0),
                                           s["work"].data_ptr(), s["work"].numel(), stream), "tl_paged_attn_decode_f16")
        return [s["out"], s["lse"]]
    if op == "fork":
        check(lib.tl_paged_fork(s["cache"], s["drop"].data_ptr(), stream), "tl_paged_fork")
        check(lib.tl_paged_fork(s["cache"], s["fork"].data_ptr(), stream), "tl_paged_fork")
        check(lib.tl_paged_reserve_f16(s["cache"], s["new"].data_ptr(), s["result"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                                       stream), "tl_paged_reserve_f16")
        return _fork_out(s)
    if op == "compact":
        s["table"].copy_(s["table0"])
        s["ref"].copy_(s["ref0"])
        check(lib.tl_paged_compact_f16(s["cache"], s["moved"].data_ptr(), s["result"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                                       stream), "tl_paged_compact_f16")
        return _compact_out(s)
    if op == "select":
        check(lib.tl_beam_select_f16(s["logits"].data_ptr(), s["logits"].stride(0), s["scores"].data_ptr(), s["finished"].data_ptr(), PAD,
                                     c["batch"], c["beams"], c["vocab"], c["k"], s["values"].data_ptr(), s["parents"].data_ptr(),
                                     s["tokens"].data_ptr(), s["work"].data_ptr(), s["work"].numel(), stream), "tl_beam_select_f16")
        return [s["values"], s["parents"], s["tokens"]]
    a, d = s["src"], s["dst"]
    check(lib.tl_beam_reorder_f16(a.data_ptr(), d.data_ptr(), s["parents"].data_ptr(), c["outer"], c["rows"], c["used"], a.stride(0),
                                  a.stride(1), d.stride(0), d.stride(1), stream), "tl_beam_reorder_f16")
    return [d]


_PLAIN = dict(rotary=_plain_rotary, append=_plain_append, attn=_plain_attn, fork=_plain_fork, compact=_plain_compact,
              select=_plain_select, reorder=_plain_reorder)


def run(state):
    if own:
        return _own_pass(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its exact results
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    op = c["op"]
    if op == "rotary":
        n = c["tokens"] * c["heads"]
        return {"bytes": 4 * n * c["dim"] + 4 * c["tokens"] + 4 * c["rot"], "flops": 3 * n * c["rot"]}
    if op == "append":
        _, pos, _ = _append_plan(c)
        n = sum(x >= 0 for x in pos)
        return {"bytes": 4 * n * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] + 12 * len(pos) + 4 * c["rot"],
                "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if op == "attn":
        n = _lengths(c)
        return {"bytes": 4 * sum(n) * c["kv_heads"] * c["dim"] + 4 * c["batch"] * c["heads"] * (c["dim"] + 1)
                + 4 * sum(-(-x // c["page"]) for x in n) + 4 * c["batch"], "flops": 4 * sum(n) * c["heads"] * c["dim"]}
    if op == "fork":
        n, par = _fork_plan(c)
        # each child's filled part of its last page is read and written once for K and V of every layer; its table row is
        # written three times over the pass (dropped, forked, extended)
        copied = sum(n[p] % c["page"] for p in par)
        entries = sum(-(-n[p] // c["page"]) for p in par)
        return {"bytes": 8 * copied * c["layers"] * c["kv_heads"] * c["dim"] + 12 * entries + 16 * (len(n) + len(par)), "flops": 0}
    if op == "compact":
        # the number of moves is the number of live pages above the live count: its mean over placements
        moves = c["live"] * (c["pages"] - c["live"]) // c["pages"]
        return {"bytes": 8 * moves * c["layers"] * c["page"] * c["kv_heads"] * c["dim"] + 24 * c["pages"] + 16 * c["live"], "flops": 0}
    if op == "select":
        rows = c["batch"] * c["beams"]
        return {"bytes": 2 * (rows - c["finished"] - c["dead"]) * c["vocab"] + 5 * rows + 12 * c["batch"] * c["k"], "flops": 4 * rows * c["vocab"]}
    r = random.Random(c["lens_seed"])
    read = len({r.randrange(c["rows"]) for _ in range(c["rows"])})
    return {"bytes": 2 * c["outer"] * c["used"] * (read + c["rows"]) + 4 * c["rows"], "flops": 0}


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    op = c["op"]

    def turn(x, pos):
        """[tokens, heads, dim] in 64 bits as complex numbers times exp(i angle)."""
        rot = c["rot"]
        y = x.double().clone()
        if not rot:
            return y
        angle = torch.outer(pos.double(), s["freqs"]) * (-1.0 if c.get("inverse") else 1.0)
        phase = torch.polar(torch.full_like(angle, s["mag"]), angle)[:, None, :]
        i = torch.arange(rot // 2, device=DEVICE)
        re, im = (i, i + rot // 2) if c["half"] else (2 * i, 2 * i + 1)
        z = torch.complex(y[..., re], y[..., im]) * phase
        y[..., re], y[..., im] = z.real, z.imag
        return y

    if op == "rotary":
        return [turn(s["x"], s["pos"])]
    if op == "append":
        rows, pos, _ = _append_plan(c)
        h, kv, p = c["heads"], c["kv_heads"], c["page"]
        q, k, v = turn(s["qkv"][:, :h], s["pos"]), turn(s["qkv"][:, h:h + kv], s["pos"]), s["qkv"][:, h + kv:].double()
        out = [s["q_out"].double(), s["k"][0, : s["pages"]].double(), s["v"][0, : s["pages"]].double()]
        table = s["table"].cpu()
        live = [i for i, x in enumerate(pos) if x >= 0]
        page = torch.tensor([int(table[rows[i], pos[i] // p]) for i in live], device=DEVICE)
        slot = torch.tensor([pos[i] % p for i in live], device=DEVICE)
        at = torch.tensor(live, device=DEVICE)
        out[0][at], out[1][page, slot], out[2][page, slot] = q[at], k[at], v[at]
        return out
    if op == "attn":
        n, d, h, kv, p = _lengths(c), c["dim"], c["heads"], c["kv_heads"], c["page"]
        out = torch.zeros(c["batch"], h, d, dtype=torch.float64, device=DEVICE)
        lse = torch.full((c["batch"], h), -math.inf, dtype=torch.float64, device=DEVICE)
        for b in range(c["batch"]):
            if n[b] == 0:
                continue
            pages = s["table"][b, : -(-n[b] // p)].long()
            for j in range(kv):
                k = s["k"][0, pages, :, j].reshape(-1, d)[: n[b]].double()
                v = s["v"][0, pages, :, j].reshape(-1, d)[: n[b]].double()
                hs = slice(j * (h // kv), (j + 1) * (h // kv))
                x = s["q"][b, hs].double() @ k.T / math.sqrt(d)
                lse[b, hs] = torch.logsumexp(x, -1)
                out[b, hs] = torch.softmax(x, -1) @ v
        return [out, lse]
    if op == "fork":
        n, par = _fork_plan(c)
        p, base = c["page"], c["parents"]
        table, ref, lengths = s["table"].cpu().tolist(), s["ref"].cpu().tolist(), n + [n[j] for j in par]
        for i, j in enumerate(par):
            table[base + i] = list(table[j])
            for e in table[j]:
                if e >= 0:
                    ref[e] += 1
        copies, free = [], [e for e, r in enumerate(ref) if r == 0]
        for r in range(base, base + len(par)):
            m = lengths[r]
            e = table[r][m // p]
            if m % p == 0 or ref[e] > 1:
                new = free.pop(0)
                if m % p:
                    copies.append((e, new, m % p))
                    ref[e] -= 1
                table[r][m // p], ref[new] = new, 1
            lengths[r] += 1
        for e, new, m in copies:
            for t in (s["k"], s["v"]):
                t[:, new, :m] = t[:, e, :m]
        return [_ints(table), _ints(lengths), _ints(ref), s["result"], s["k"][:, : s["pages"]], s["v"][:, : s["pages"]]]
    if op == "compact":
        table, ref = s["table"].cpu().tolist(), s["ref"].cpu().tolist()
        to = [i if r else -1 for i, r in enumerate(ref)]
        lo, hi = 0, len(ref) - 1
        while True:
            while lo < hi and ref[lo]:
                lo += 1
            while lo < hi and not ref[hi]:
                hi -= 1
            if lo >= hi:
                break
            to[hi], ref[lo], ref[hi] = lo, ref[hi], 0
            s["k"][:, lo], s["v"][:, lo] = s["k"][:, hi], s["v"][:, hi]
        table = [[to[e] if e >= 0 else e for e in row] for row in table]
        return [_ints(table), _ints(ref), _ints(to), _ints([sum(r > 0 for r in ref)]), s["k"], s["v"]]
    if op == "select":
        b, w, n, k = c["batch"], c["beams"], c["vocab"], c["k"]
        out = [torch.empty(b, k, dtype=torch.float64), torch.empty(b, k, dtype=torch.int32), torch.empty(b, k, dtype=torch.int32)]
        score, done = s["scores"].cpu().double(), s["finished"].cpu()
        for i in range(b):
            found = []
            for j in range(i * w, (i + 1) * w):
                x = s["logits"][j].cpu().double().numpy()
                top = x.max()
                v = x + (float(score[j]) - (top + math.log(math.fsum(math.e ** (x - top)))))
                if done[j]:
                    v[:] = -math.inf
                    v[PAD] = float(score[j])
                best = (-v).argsort(kind="stable")[:k]
                found += [(-v[t], j, int(t)) for t in best]
            for t, (v, j, a) in enumerate(sorted(found)[:k]):
                out[0][i, t], out[1][i, t], out[2][i, t] = -v, j, a
        return out
    r = random.Random(c["lens_seed"])
    for i in range(c["rows"]):
        s["dst"][:, i, : c["used"]] = s["src"][:, r.randrange(c["rows"]), : c["used"]]
    return [s["dst"]]
