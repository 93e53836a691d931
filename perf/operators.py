"""What the 8-bit KV cache, the drafted-tree attention and the logit rules are measured on.

A case names one operator and its sizes; `prepare` makes what a serving program holds before the
call (projections, cache pool, page table, histories), `run` makes the call, either in the plain
form (`own` false: elementary torch operations) or through libhobbygpu.so (`own` true).

The cache pool's layout (include/hobbygpu.h): page p, kv head h is a block of 32 * hd + 128 bytes at
p * page_stride + h * block: K codes of the page's 16 slots in 8-slot x 16-byte tiles
[slot / 8][dim / 16][slot % 8][dim % 16], V codes transposed [dim][slot], 16 f32 K scales, 16 f32 V
scales.
"""
import ctypes
import math
import random

import torch

own = False

PAGE = 16  # slots of a page
EPS = 1e-5
DEV = "cuda"

# (q heads, kv heads, head dim) of the synthetic presets and of the small test model
HEADS = {"130M": (8, 2, 64), "500M": (12, 3, 128), "1B": (16, 8, 128), "tiny": (4, 1, 64)}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _heads(nh, nkv, hd):
    return {"nh": nh, "nkv": nkv, "hd": hd}


def listed():
    p500, p130, p1b = (_heads(*HEADS[k]) for k in ("500M", "130M", "1B"))
    return [
        # one chat sequence decoding one token: latency only
        {"name": "write one token", "op": "write", **p500, "seqs": 1, "start": 2048, "start_hi": 2048, "rows": 1,
         "rows_hi": 1, "tree": False, "lens": 1},
        # a decode step of the benchmark's batch: 256 sequences of mixed lengths, one token each
        {"name": "write 256 sequences", "op": "write", **p500, "seqs": 256, "start": 1024, "start_hi": 8192, "rows": 1,
         "rows_hi": 1, "tree": False, "lens": 2},
        # prompts of mixed lengths entering the cache after whatever their sequences hold already
        {"name": "write prompts", "op": "write", **p1b, "seqs": 13, "start": 0, "start_hi": 777, "rows": 130,
         "rows_hi": 2500, "tree": False, "lens": 3},
        # one sequence handed back as f32 rows (moving it to the f32 pool)
        {"name": "read one sequence", "op": "read", **p130, "seqs": 1, "start": 0, "start_hi": 0, "rows": 601,
         "rows_hi": 601, "tree": False, "lens": 4},
        # sequences of a batch handed back, each from where its shared prompt ends
        {"name": "read 64 sequences", "op": "read", **p500, "seqs": 64, "start": 0, "start_hi": 500, "rows": 12,
         "rows_hi": 4096, "tree": False, "lens": 5},
        # single-token decode of one sequence after a 2048-token prompt: latency
        {"name": "attend one token", "op": "attend", **p500, "seqs": 1, "start": 2100, "start_hi": 2100, "rows": 1,
         "rows_hi": 1, "tree": False, "lens": 6},
        # single-token decode of the benchmark's batch: bound by the cache's bytes
        {"name": "attend 256 sequences", "op": "attend", **p500, "seqs": 256, "start": 1024, "start_hi": 8192,
         "rows": 1, "rows_hi": 1, "tree": False, "lens": 7},
        # a few drafted tokens per sequence, ragged trees, small heads
        {"name": "attend small trees", "op": "attend", **p130, "seqs": 48, "start": 1, "start_hi": 4001, "rows": 1,
         "rows_hi": 12, "tree": True, "lens": 8},
        # wide draft trees of 64 nodes: the most arithmetic per byte of cache
        {"name": "attend wide trees", "op": "attend", **p500, "seqs": 32, "start": 900, "start_hi": 7000, "rows": 64,
         "rows_hi": 64, "tree": True, "lens": 9},
        # the logits of one sequence's step
        {"name": "rules one row", "op": "rules", "vocab": 50304, "valid": 50257, "seqs": 1, "rows": 1, "rows_hi": 1,
         "tree": False, "hist": 700, "hist_hi": 700, "bias": 20, "bias_hi": 20, "masks": 1, "lens": 10},
        # a batch's step: histories of mixed lengths, biases, no grammar
        {"name": "rules 256 rows", "op": "rules", "vocab": 50304, "valid": 50257, "seqs": 256, "rows": 1, "rows_hi": 1,
         "tree": False, "hist": 0, "hist_hi": 2000, "bias": 0, "bias_hi": 300, "masks": 0, "lens": 11},
        # every node of the drafted trees under a grammar, an odd vocabulary
        {"name": "rules tree nodes", "op": "rules", "vocab": 128259, "valid": 128259, "seqs": 24, "rows": 1,
         "rows_hi": 16, "tree": True, "hist": 0, "hist_hi": 1500, "bias": 0, "bias_hi": 40, "masks": 40, "lens": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "rules"])
    lens = rng.randrange(1 << 30)
    if op == "rules":
        tree = rng.random() < 0.5
        rows_hi = rng.randint(2, 16) if tree else 1
        vocab = 50304 if rng.random() < 0.4 else _log_int(rng, 100, 130000)
        seqs = _log_int(rng, 1, max(1, min(256, 12_000_000 // (vocab * rows_hi))))
        return {"op": op, "vocab": vocab, "valid": vocab if rng.random() < 0.5 else vocab - vocab // 100, "seqs": seqs,
                "rows": 1, "rows_hi": rows_hi, "tree": tree, "hist": 0, "hist_hi": _log_int(rng, 1, 4000),
                "bias": 0, "bias_hi": _log_int(rng, 1, 300), "masks": rng.choice([0, 1, 7, seqs]), "lens": lens}
    nh, nkv, hd = rng.choice(list(HEADS.values()) + [(12, 12, 64), (12, 2, 128), (7, 1, 128), (10, 2, 64)])
    case = {"op": op, **_heads(nh, nkv, hd)}
    if op == "attend":
        tree = rng.random() < 0.6
        rows_hi = _log_int(rng, 1, 64) if tree else rng.choice([1, 1, 1, 3, 17])
        ctx = _log_int(rng, 1, 16000)
        most = min(1_000_000 * 6 // (2 * nkv * hd // 128), 120_000 * 12 * 64 // (nh * rows_hi))
        seqs = _log_int(rng, 1, max(1, min(256, most // (ctx + rows_hi))))
        return {**case, "seqs": seqs, "start": rng.randint(0, ctx), "start_hi": ctx, "rows": rng.randint(0, 1),
                "rows_hi": rows_hi, "tree": tree, "lens": lens}
    seqs = _log_int(rng, 1, 256)
    most = 16_000 * 32 * 128 // ((nh + 2 * nkv) * hd) if op == "write" else 120_000 * 3 * 128 // (nkv * hd)
    rows_hi = _log_int(rng, 1, max(1, most // seqs))
    tree = op == "write" and rows_hi <= 64 and rng.random() < 0.5
    return {**case, "seqs": seqs, "start": 0, "start_hi": _log_int(rng, 1, 9000 if seqs < 64 else 1500),
            "rows": rng.randint(0, min(rows_hi, 4)), "rows_hi": rows_hi, "tree": tree, "lens": lens}


def _lengths(case):
    """The sequences' lengths: part of the case, not of the seed."""
    r = random.Random(case["lens"])
    starts = [r.randint(min(case["start"], case["start_hi"]), case["start_hi"]) for _ in range(case["seqs"])]
    rows = [r.randint(min(case["rows"], case["rows_hi"]), case["rows_hi"]) for _ in range(case["seqs"])]
    if not sum(rows):
        rows[0] = 1
    return starts, rows


def _list_lengths(case):
    r = random.Random(case["lens"])
    rows = [r.randint(case["rows"], case["rows_hi"]) for _ in range(case["seqs"])]
    hist = [r.randint(case["hist"], case["hist_hi"]) for _ in range(case["seqs"])]
    bias = [min(case["vocab"], r.randint(case["bias"], case["bias_hi"])) for _ in range(case["seqs"])]
    return rows, hist, bias


def work(case):
    if case["op"] == "rules":
        rows, hist, bias = _list_lengths(case)
        n, v = sum(rows), case["vocab"]
        return {"bytes": n * v * 8 + min(n, case["masks"]) * v // 8 + 4 * sum(hist) + 8 * sum(bias) + 12 * n, "flops": 0}
    starts, rows = _lengths(case)
    nh, nkv, hd, n = case["nh"], case["nkv"], case["hd"], sum(rows)
    cached = 2 * nkv * (hd + 4)  # bytes of one slot in the cache
    if case["op"] == "write":  # projections in, q out, codes and scales in and back out as f32
        return {"bytes": n * ((nh + 2 * nkv) * hd * 4 + nh * hd * 4 + 2 * cached + 2 * nkv * hd * 4), "flops": 0}
    if case["op"] == "read":
        return {"bytes": n * (cached + 2 * nkv * hd * 4), "flops": 0}
    slots = sum(s + r for s, r in zip(starts, rows) if r)
    pairs = sum(r * s + r * (r + 1) // 2 for s, r in zip(starts, rows))
    return {"bytes": slots * cached + n * nh * hd * 8, "flops": 4 * nh * hd * pairs}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int32, device=DEV)


def _trees(rows, tree, rnd):
    """A parent per row, local to its sequence: -1 under the context, -2 a padding row; None: chains."""
    if not tree:
        return None
    p = []
    for n in rows:
        for j in range(n):
            p.append(-1 if j == 0 else -2 if rnd.random() < 0.04 else rnd.randint(max(-1, j - 9), j - 1))
    return torch.tensor(p, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + case["lens"] % 100003)
    rnd = random.Random(seed)
    if case["op"] == "rules":
        return _prepare_rules(case, gen, rnd)
    starts, rows = _lengths(case)
    nh, nkv, hd, n, s = case["nh"], case["nkv"], case["hd"], sum(rows), case["seqs"]
    pages = [(a + b + PAGE - 1) // PAGE for a, b in zip(starts, rows)]
    bt_stride, n_pages = max(pages) + 1, sum(pages) + 3
    block = 32 * hd + 128
    perm = torch.randperm(n_pages, generator=gen, device=DEV, dtype=torch.int32)
    off = _offsets(pages).long()
    at = off[:-1, None] + torch.arange(bt_stride, device=DEV)[None]
    # entries past a sequence's last page are never read: a server leaves there what was there
    table = torch.where(at < off[1:, None], perm[at.clamp(max=n_pages - 1)], 1 << 30).to(torch.int32)
    st = {"case": case, "n": n, "row_off": _offsets(rows), "start": torch.tensor(starts, dtype=torch.int32, device=DEV),
          "parent": _trees(rows, case["tree"], rnd), "max_rows": max(rows), "table": table.contiguous(),
          "max_len": max(a + b for a, b in zip(starts, rows)), "n_pages": n_pages, "block": block}
    if case["op"] == "write":
        st["pool"] = torch.zeros(n_pages, nkv, block, dtype=torch.uint8, device=DEV)
        heads = nh + 2 * nkv
        size = 0.5 + 2.0 * torch.rand(1, heads, 1, generator=gen, device=DEV)
        st["qkv"] = (torch.randn(n, heads, hd, generator=gen, device=DEV) * size).reshape(n, heads * hd)
        st["q_norm"] = 1.0 + 0.2 * torch.randn(hd, generator=gen, device=DEV)
        st["k_norm"] = 1.0 + 0.2 * torch.randn(hd, generator=gen, device=DEV)
        pos = torch.arange(st["max_len"] + 1, device=DEV, dtype=torch.float64)[:, None]
        ang = pos * 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)[None]
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["q"] = torch.empty(n, nh * hd, device=DEV)
        st["k"], st["v"] = (torch.empty(n, nkv * hd, device=DEV) for _ in range(2))
        return st
    pool = torch.empty(n_pages, nkv, block, dtype=torch.uint8, device=DEV)
    # codes of rows with a largest value near three deviations; k rows have the norm's length
    codes = torch.randn(n_pages, nkv, 32 * hd, generator=gen, device=DEV).mul_(42).round_().clamp_(-127, 127)
    pool[..., :32 * hd] = codes.to(torch.int8).view(torch.uint8)
    del codes
    scale = (0.02 + 0.012 * torch.rand(n_pages, nkv, 32, generator=gen, device=DEV))
    pool[..., 32 * hd:] = scale.view(torch.uint8)
    st["pool"] = pool
    if case["op"] == "attend":
        st["q"] = torch.randn(n, nh * hd, generator=gen, device=DEV)
        st["out"] = torch.empty(n, nh * hd, device=DEV)
    else:
        st["k"], st["v"] = (torch.empty(n, nkv * hd, device=DEV) for _ in range(2))
    return st


def _prepare_rules(case, gen, rnd):
    rows, hist, bias = _list_lengths(case)
    v, n, s = case["vocab"], sum(rows), case["seqs"]

    def ids(count):  # frequent tokens are frequent: a log-uniform rank, spread over the ids
        rank = torch.exp(torch.rand(count, generator=gen, device=DEV) * math.log(v)).long().clamp(max=v) - 1
        return ((rank * 7919 + 13) % v).to(torch.int32)

    words = (v + 31) // 32
    masks = case["masks"]
    allowed = torch.rand(max(masks, 1), words * 32, generator=gen, device=DEV) < 0.3
    bits = (allowed.view(-1, words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    mask_row = torch.randint(-1, max(masks, 1), (n,), generator=gen, device=DEV, dtype=torch.int32)
    return {"case": case, "n": n, "row_off": _offsets(rows), "parent": _trees(rows, case["tree"], rnd),
            "max_rows": max(rows), "logits": torch.randn(n, v, generator=gen, device=DEV) * 3.0,
            "token": ids(n) if case["tree"] else None, "hist_off": _offsets(hist), "hist": ids(max(1, sum(hist))),
            "rep": 1.0 + 0.15 * torch.rand(s, generator=gen, device=DEV),
            "freq": 0.3 * torch.rand(s, generator=gen, device=DEV),
            "pres": 0.5 * torch.rand(s, generator=gen, device=DEV), "bias_off": _offsets(bias),
            "bias_id": torch.cat([torch.randperm(v, generator=gen, device=DEV)[:b] for b in bias] + [ids(1)]).to(torch.int32),
            "bias": torch.randn(max(1, sum(bias)), generator=gen, device=DEV) * 2.0,
            "mask": bits.contiguous() if masks else None, "mask_row": mask_row if masks else None, "words": words,
            "out": torch.empty(n, v, device=DEV), "next": torch.empty(n, dtype=torch.int32, device=DEV)}


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _rows_of(st):
    """Each row's sequence and its index there."""
    row = torch.arange(st["n"], device=DEV)
    seq = torch.searchsorted(st["row_off"][1:].contiguous(), row.to(torch.int32), right=True)
    return seq, row - st["row_off"][seq]


def _path(st, seq, j):
    """[n][max_rows] truth values: the rows of its sequence that a row sees (itself and its ancestors,
    or all before it in a chain); none for a padding row."""
    m, cols = st["max_rows"], torch.arange(st["max_rows"], device=DEV)
    if st["parent"] is None:
        return cols[None] <= j[:, None]
    row = torch.arange(st["n"], device=DEV)
    live = st["parent"] > -2
    up = torch.where(st["parent"] >= 0, st["row_off"][seq] + st["parent"], row)  # roots point at themselves
    up = torch.where(live[up], up, row)  # nothing is seen through a padding row
    see = (cols[None] == j[:, None]) & live[:, None]
    for _ in range(max(1, (m - 1).bit_length())):  # ancestors up to 2^k levels away
        see = see | see[up]
        up = up[up]
    return see


def _write_plain(st):
    c, n = st["case"], st["n"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    seq, j = _rows_of(st)
    see = _path(st, seq, j) if st["parent"] is not None else None
    depth = j if see is None else (see.sum(1) - 1).clamp(min=0)
    live = torch.ones(n, 1, 1, device=DEV) if see is None else (st["parent"] > -2).float()[:, None, None]
    pos = st["start"][seq] + depth
    x = st["qkv"].view(n, nh + 2 * nkv, hd)
    qk = x[:, :nh + nkv].double()
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    gain = torch.cat([st["q_norm"].expand(nh, hd), st["k_norm"].expand(nkv, hd)]).double()
    qk = qk * gain
    cos, sin = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
    a, b = qk[..., :hd // 2], qk[..., hd // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def kept(y):  # the values that the 8-bit rows stand for
        scale = (y.abs().amax(-1, keepdim=True) / 127.0).float()
        inv = torch.where(scale > 0, 1.0 / scale.double(), 0.0)
        code = torch.round(y * inv).clamp(-127, 127)
        return (code.float() * scale * live).reshape(n, -1)

    return {"q": (qk[:, :nh].float() * live).reshape(n, -1), "k": kept(qk[:, nh:]),
            "v": kept(x[:, nh + nkv:].double())}


def _pool_rows(st):
    """K and V of every page as f32 [page][slot][kv head][dim]."""
    c = st["case"]
    nkv, hd, pages = c["nkv"], c["hd"], st["n_pages"]
    codes = st["pool"][..., :32 * hd].view(torch.int8)
    scales = st["pool"][..., 32 * hd:].contiguous().view(torch.float32).view(pages, nkv, 2, PAGE)
    k = codes[..., :16 * hd].reshape(pages, nkv, 2, hd // 16, 8, 16).permute(0, 2, 4, 1, 3, 5)
    v = codes[..., 16 * hd:].reshape(pages, nkv, hd, PAGE).permute(0, 3, 1, 2)
    ks, vs = (scales[:, :, i].permute(0, 2, 1)[..., None] for i in range(2))
    return (k.reshape(pages, PAGE, nkv, hd).float() * ks, v.float() * vs)


def _read_plain(st):
    seq, j = _rows_of(st)
    slot = st["start"][seq].long() + j
    page = st["table"][seq, slot // PAGE].long()
    k, v = _pool_rows(st)
    return {"k": k[page, slot % PAGE].reshape(st["n"], -1), "v": v[page, slot % PAGE].reshape(st["n"], -1)}


def _attend_plain(st):
    c, n, m = st["case"], st["n"], st["max_rows"]
    nh, nkv, hd, s = c["nh"], c["nkv"], c["hd"], c["seqs"]
    g = nh // nkv
    seq, j = _rows_of(st)
    length = -(-st["max_len"] // PAGE) * PAGE
    table = st["table"][:, :length // PAGE].long().clamp(max=st["n_pages"] - 1)
    k, v = _pool_rows(st)
    k = k[table].reshape(s, length, nkv, hd).permute(0, 2, 1, 3)  # [seq][kv head][slot][dim]
    q = torch.zeros(s, m, nkv, g, hd, device=DEV)
    q[seq, j] = st["q"].view(n, nkv, g, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(s, nkv, m * g, hd)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    del k
    slot = torch.arange(length, device=DEV)
    rel = slot[None] - st["start"][:, None]  # [seq][slot]: index among the sequence's rows
    see = torch.zeros(s, m, m, dtype=torch.bool, device=DEV)
    see[seq, j] = _path(st, seq, j)
    live = torch.zeros(s, m, dtype=torch.bool, device=DEV)
    live[seq, j] = True if st["parent"] is None else st["parent"] > -2
    rel_in = rel.clamp(0, m - 1)[:, None].expand(s, m, length)
    seen = torch.where(rel[:, None] < 0, live[:, :, None], see.gather(2, rel_in) & (rel < m)[:, None])
    seen = seen[:, None, :, None].expand(s, nkv, m, g, length).reshape(s, nkv, m * g, length)
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    v = v[table].reshape(s, length, nkv, hd).permute(0, 2, 1, 3)
    v = v.masked_fill((rel >= m)[:, None, :, None], 0.0)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.view(s, nkv, m, g, hd).permute(0, 2, 1, 3, 4)
    return out[seq, j].reshape(n, nh * hd)


def _counts(st):
    """[n][vocab]: how often each id stands in a row's history and drafted path."""
    n, v = st["n"], st["case"]["vocab"]
    seq, j = _rows_of(st)
    s = st["case"]["seqs"]
    total = st["hist"][:int(st["hist"].numel())]
    at = torch.arange(total.numel(), device=DEV)
    owner = torch.searchsorted(st["hist_off"][1:].contiguous(), at.to(torch.int32), right=True)
    table = torch.zeros(s + 1, v, dtype=torch.int32, device=DEV)
    table.view(-1).index_add_(0, owner * v + total, torch.ones_like(total))
    counts = table[seq]
    if st["token"] is not None:
        see = _path(st, seq, j)  # the drafted tokens on the row's path, its own among them
        row, col = see.nonzero(as_tuple=True)
        tok = st["token"][st["row_off"][seq[row]] + col]
        counts.view(-1).index_add_(0, row * v + tok, torch.ones_like(tok))
    return seq, counts


def _rules_plain(st):
    c, n = st["case"], st["n"]
    v, valid = c["vocab"], c["valid"]
    seq, counts = _counts(st)
    count = counts.double()
    x = st["logits"].double()
    rep, freq, pres = (st[k].double()[seq][:, None] for k in ("rep", "freq", "pres"))
    x = torch.where(x > 0, x * rep ** -count, x * rep ** count)  # once for each occurrence
    x = x - freq * count - pres * (count > 0)
    at = torch.arange(int(st["bias"].numel()), device=DEV)
    owner = torch.searchsorted(st["bias_off"][1:].contiguous(), at.to(torch.int32), right=True)
    bias = torch.zeros(c["seqs"] + 1, v, dtype=torch.float64, device=DEV)
    ids = st["bias_id"][:at.numel()]
    bias.view(-1).index_add_(0, owner[:ids.numel()] * v + ids, st["bias"][:ids.numel()].double())
    x = x + bias[seq]
    barred = (torch.arange(v, device=DEV) >= valid)[None].expand(n, v)
    if st["mask"] is not None:
        bit = (st["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        allow = bit.reshape(-1, st["words"] * 32)[:, :v].bool()
        allow = allow[st["mask_row"].long().clamp(min=0)] | (st["mask_row"] < 0)[:, None]
        barred = barred | ~allow
    out = x.masked_fill(barred, -math.inf).float()
    best = torch.where(out.amax(1) > -math.inf, out.argmax(1), -1)
    if st["parent"] is not None:  # padding rows stay as they were
        pad = st["parent"] == -2
        out = torch.where(pad[:, None], 0.0, out)
        best = torch.where(pad, -1, best)
    return {"logits": out, "next": best.to(torch.int32)}


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _bind(st):
    """The argument structs over the state's buffers, as a serving loop keeps them."""
    from hobbylm_b200 import _native as N

    c, lib = st["case"], N.lib()
    rows = N.Rows(n_seqs=c["seqs"], n_rows=st["n"], max_rows=st["max_rows"], row_off=_ptr(st["row_off"]),
                  start=_ptr(st.get("start")), parent=_ptr(st["parent"]))
    st["keep"] = keep = {"rows": rows}
    by = ctypes.byref
    if c["op"] == "rules":
        if st["parent"] is not None:
            st["out"].zero_()  # rows that the call leaves alone
        a = keep["args"] = N.LogitsRules(
            vocab=c["vocab"], valid=c["valid"], logits=_ptr(st["logits"]), out=_ptr(st["out"]),
            next_ids=_ptr(st["next"]), token=_ptr(st["token"]), hist_off=_ptr(st["hist_off"]), hist=_ptr(st["hist"]),
            rep_penalty=_ptr(st["rep"]), freq_penalty=_ptr(st["freq"]), pres_penalty=_ptr(st["pres"]),
            bias_off=_ptr(st["bias_off"]), bias_id=_ptr(st["bias_id"]), bias=_ptr(st["bias"]), mask=_ptr(st["mask"]),
            mask_row=_ptr(st["mask_row"]), mask_words=st["words"])
        result = {"logits": st["out"], "next": st["next"]}
        return lambda stream: (N.check(lib.hg_op_logits_rules(by(rows), by(a), stream)), result)[1]
    cache = keep["cache"] = N.Kv8Cache(n_kv_heads=c["nkv"], head_dim=c["hd"], n_pages=st["n_pages"],
                                       bt_stride=st["table"].shape[1], block_table=_ptr(st["table"]),
                                       pool=_ptr(st["pool"]), page_stride=c["nkv"] * st["block"])
    if c["op"] == "attend":
        size = lib.hg_op_kv8_attn_scratch_bytes(by(cache), by(rows), c["nh"])
        scratch = keep["scratch"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        args = (by(cache), by(rows), c["nh"], _ptr(st["q"]), _ptr(st["out"]), _ptr(scratch))
        return lambda stream: (N.check(lib.hg_op_kv8_attn(*args, stream)), st["out"])[1]
    read = (by(cache), by(rows), _ptr(st["k"]), _ptr(st["v"]))
    if c["op"] == "read":
        result = {"k": st["k"], "v": st["v"]}
        return lambda stream: (N.check(lib.hg_op_kv8_read(*read, stream)), result)[1]
    a = keep["args"] = N.Kv8Append(n_heads=c["nh"], max_pos=st["cos"].shape[0], eps=EPS, qkv=_ptr(st["qkv"]),
                                   q_norm=_ptr(st["q_norm"]), k_norm=_ptr(st["k_norm"]), rope_cos=_ptr(st["cos"]),
                                   rope_sin=_ptr(st["sin"]), q_out=_ptr(st["q"]))
    result = {"q": st["q"], "k": st["k"], "v": st["v"]}
    # written, then read back as the f32 rows that the codes stand for
    return lambda stream: (N.check(lib.hg_op_kv8_append(by(cache), by(rows), by(a), stream)),
                           N.check(lib.hg_op_kv8_read(*read, stream)), result)[2]


def run(state):
    if own:
        call = state.get("call")
        if call is None:
            call = state["call"] = _bind(state)
        return call(torch.cuda.current_stream().cuda_stream)
    return {"write": _write_plain, "read": _read_plain, "attend": _attend_plain,
            "rules": _rules_plain}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------
def _chains(st):
    """Per row: the rows (global) it sees, walked up one by one."""
    off = st["row_off"].tolist()
    par = None if st["parent"] is None else st["parent"].tolist()
    paths = []
    for s in range(len(off) - 1):
        for j in range(off[s + 1] - off[s]):
            if par is None:
                paths.append(list(range(off[s], off[s] + j + 1)))
                continue
            path, at = [], j
            while at >= 0 and par[off[s] + at] > -2:
                path.append(off[s] + at)
                at = par[off[s] + at]
            paths.append(path)
    return off, paths


def _decode_slots(st, seq, lo, hi):
    """K and V of slots lo..hi-1 of a sequence: [slot][kv head][dim] in 64 bits."""
    c = st["case"]
    hd = c["hd"]
    slot = torch.arange(lo, hi, device=DEV)
    pages = st["table"][seq].long()[slot // PAGE]
    raw = st["pool"][pages]  # [slot][kv head][block]
    i, w = torch.arange(hd, device=DEV), slot % PAGE
    k_at = (w // 8)[:, None] * (8 * hd) + (i // 16)[None] * 128 + (w % 8)[:, None] * 16 + (i % 16)[None]
    v_at = 16 * hd + i[None] * PAGE + w[:, None]

    def values(at, scale_at):
        code = raw.view(torch.int8).gather(2, at[:, None].expand(-1, c["nkv"], -1)).double()
        word = (scale_at + 4 * w)[:, None] + torch.arange(4, device=DEV)[None]
        scale = raw.gather(2, word[:, None].expand(-1, c["nkv"], -1)).contiguous().view(torch.float32)
        return code * scale.double()

    return values(k_at, 32 * hd), values(v_at, 32 * hd + 64)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rules":
        return _exact_rules(st)
    nh, nkv, hd, n = case["nh"], case["nkv"], case["hd"], st["n"]
    start = st["start"].tolist()
    if case["op"] == "write":
        off = st["row_off"].tolist()
        owner = [s for s in range(case["seqs"]) for _ in range(off[s + 1] - off[s])]
        if st["parent"] is None:
            deep = [j for s in range(case["seqs"]) for j in range(off[s + 1] - off[s])]
            live = torch.ones(n, device=DEV, dtype=torch.float64)
        else:
            paths = _chains(st)[1]
            deep = [max(0, len(p) - 1) for p in paths]
            live = torch.tensor([float(bool(p)) for p in paths], device=DEV, dtype=torch.float64)
        pos = torch.tensor([start[s] + d for s, d in zip(owner, deep)], device=DEV)
        turn = torch.complex(st["cos"].double(), st["sin"].double())[pos]
        x = st["qkv"].double().view(n, -1, hd)

        def turned(y, gain):
            y = y / (torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / hd + EPS).sqrt() * gain.double()
            z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        def kept(y):
            scale = (y.abs().max(-1, keepdim=True).values / 127).float().double()
            code = torch.where(scale > 0, (y / torch.where(scale > 0, scale, 1.0)).round().clamp(-127, 127), 0.0)
            return (code * scale * live[:, None, None]).reshape(n, -1)

        q = turned(x[:, :nh], st["q_norm"]) * live[:, None, None]
        return {"q": q.reshape(n, -1), "k": kept(turned(x[:, nh:nh + nkv], st["k_norm"])),
                "v": kept(x[:, nh + nkv:])}
    off = st["row_off"].tolist()
    if case["op"] == "read":
        got = [_decode_slots(st, s, start[s], start[s] + off[s + 1] - off[s]) for s in range(case["seqs"])]
        return {k: torch.cat([g[i].reshape(-1, nkv * hd) for g in got]) for i, k in enumerate(("k", "v"))}
    paths = _chains(st)[1]
    out = torch.zeros(n, nkv, nh // nkv, hd, device=DEV, dtype=torch.float64)
    for s in range(case["seqs"]):
        r = off[s + 1] - off[s]
        if not r:
            continue
        k, v = _decode_slots(st, s, 0, start[s] + r)
        q = st["q"][off[s]:off[s + 1]].double().view(r, nkv, nh // nkv, hd)
        bar = torch.zeros(r, start[s] + r)
        bar[:, start[s]:] = -math.inf
        for j in range(r):
            bar[j, [start[s] + x - off[s] for x in paths[off[s] + j]]] = 0.0
        score = torch.einsum("rhgd,lhd->rhgl", q, k) / math.sqrt(hd) + bar.to(DEV).double()[:, None, None]
        got = torch.einsum("rhgl,lhd->rhgd", torch.softmax(score, -1), v)
        blank = [j for j in range(r) if not paths[off[s] + j]]
        got[blank] = 0.0
        out[off[s]:off[s + 1]] = got
    return out.reshape(n, nh * hd)


def _exact_rules(st):
    c = st["case"]
    v = c["vocab"]
    off, paths = _chains(st)
    h_off, b_off = st["hist_off"].tolist(), st["bias_off"].tolist()
    out = torch.zeros(st["n"], v, dtype=torch.float64, device=DEV)
    best = torch.full((st["n"],), -1, dtype=torch.int32, device=DEV)
    which = None if st["mask"] is None else st["mask_row"].tolist()
    for s in range(c["seqs"]):
        told = torch.bincount(st["hist"][h_off[s]:h_off[s + 1]].long(), minlength=v).double()
        add = torch.zeros(v, dtype=torch.float64, device=DEV)
        mine = slice(b_off[s], b_off[s + 1])
        add[st["bias_id"][mine].long()] = st["bias"][mine].double()  # a list's ids are distinct here
        rep, freq, pres = (st[k][s].double() for k in ("rep", "freq", "pres"))
        for row in range(off[s], off[s + 1]):
            if not paths[row]:
                continue
            count = told
            if st["token"] is not None:
                count = told + torch.bincount(st["token"][paths[row]].long(), minlength=v)
            x = st["logits"][row].double()
            x = x * torch.exp(torch.where(x > 0, -count, count) * rep.log())
            x = x - freq * count - pres * count.clamp(max=1) + add
            x[c["valid"]:] = -math.inf
            if which is not None and which[row] >= 0:
                bit = st["mask"][which[row]].repeat_interleave(32) >> torch.arange(32, device=DEV).repeat(st["words"])
                x[(bit[:v] & 1) == 0] = -math.inf
            out[row] = x
            if bool(x.max() > -math.inf):
                best[row] = int(x.argmax())
    return {"logits": out, "next": best}
