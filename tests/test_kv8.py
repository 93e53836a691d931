"""The 8-bit KV cache, drafted-tree attention and logit rules against plain 64-bit implementations.

Tolerances count roundings: u = 2^-24 is half a step of f32. The codes of the cache are exact (the
kernel rounds f64 values), the rules are compared bit for bit with f32 arithmetic and to the 64-bit
definition within one u per operation.
"""
import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24
PAGE = 16
INVALID, CONTEXT = -1, -7


# ---------------------------------------------------------------------------------------------
# refusals: nothing of these calls reaches a GPU
# ---------------------------------------------------------------------------------------------
P = 1 << 20  # an aligned address that is never used


def _good(native):
    c = native.Kv8Cache(n_kv_heads=3, head_dim=128, n_pages=4, bt_stride=2, block_table=P, pool=P, page_stride=3 * 4224)
    r = native.Rows(n_seqs=1, n_rows=1, max_rows=1, row_off=P, start=P)
    a = native.Kv8Append(n_heads=12, max_pos=32, eps=1e-5, qkv=P, q_norm=P, k_norm=P, rope_cos=P, rope_sin=P, q_out=P)
    lr = native.LogitsRules(vocab=100, valid=100, logits=P, out=P, next_ids=P)
    return c, r, a, lr


CACHE_BAD = [dict(n_kv_heads=0), dict(n_kv_heads=2000), dict(head_dim=96), dict(n_pages=0), dict(bt_stride=0),
             dict(bt_stride=1 << 28), dict(block_table=None), dict(block_table=P + 2), dict(pool=None),
             dict(pool=P + 8), dict(page_stride=3 * 4224 - 16), dict(page_stride=3 * 4224 + 8)]
ROWS_BAD = [dict(n_seqs=-1), dict(n_seqs=1025), dict(n_rows=-1), dict(max_rows=0), dict(row_off=None),
            dict(row_off=P + 1), dict(start=P + 2), dict(parent=P + 3), dict(err=P + 1), dict(n_rows=1 << 30)]
APPEND_BAD = [dict(n_heads=0), dict(n_heads=13), dict(max_pos=0), dict(qkv=None), dict(qkv=P + 4), dict(q_norm=None),
              dict(k_norm=None), dict(rope_cos=None), dict(rope_sin=P + 1), dict(q_out=P + 8)]
RULES_BAD = [dict(vocab=0), dict(ld=99), dict(ld_out=50), dict(logits=None), dict(out=None), dict(ld=128),
             dict(hist_off=P), dict(bias_off=P), dict(bias_off=P, bias_id=P), dict(mask=P, mask_words=3),
             dict(logits=P + 2), dict(token=P + 1), dict(mask=P + 2, mask_words=4)]


def _set(struct, fields):
    for k, v in fields.items():
        setattr(struct, k, v)


@pytest.mark.parametrize("where,bad", [("c", b) for b in CACHE_BAD] + [("r", b) for b in ROWS_BAD] +
                         [("a", b) for b in APPEND_BAD])
def test_kv8_refusals(native, where, bad):
    c, r, a, _ = _good(native)
    _set({"c": c, "r": r, "a": a}[where], bad)
    L, by = native.lib(), C.byref
    assert L.hg_op_kv8_append(by(c), by(r), by(a), None) == INVALID
    if where != "a":
        r_only_start = where == "r" and set(bad) == {"start"}
        assert L.hg_op_kv8_read(by(c), by(r), P, P, None) == INVALID, r_only_start
        assert L.hg_op_kv8_attn(by(c), by(r), 12, P, P, P, None) == INVALID
        assert L.hg_op_kv8_attn_scratch_bytes(by(c), by(r), 12) == 0


def test_kv8_refuses_bad_buffers_and_heads(native):
    c, r, a, _ = _good(native)
    L, by = native.lib(), C.byref
    for k, v in ((None, None), (P + 4, P), (P, P + 8)):
        assert L.hg_op_kv8_read(by(c), by(r), k, v, None) == INVALID
    for nh, q, out, scratch in ((0, P, P, P), (13, P, P, P), (3 * 33, P, P, P), (12, None, P, P), (12, P, None, P),
                                (12, P, P, None), (12, P + 4, P, P), (12, P, P + 4, P), (12, P, P, P + 8)):
        assert L.hg_op_kv8_attn(by(c), by(r), nh, q, out, scratch, None) == INVALID
    for x in (None,):
        assert L.hg_op_kv8_append(x, by(r), by(a), None) == INVALID
        assert L.hg_op_kv8_append(by(c), x, by(a), None) == INVALID
        assert L.hg_op_kv8_append(by(c), by(r), x, None) == INVALID
    assert L.hg_kv8_block_bytes(64) == 2176 and L.hg_kv8_block_bytes(128) == 4224 and L.hg_kv8_block_bytes(96) == 0
    assert "null argument" in L.hg_last_error().decode()


@pytest.mark.parametrize("bad", RULES_BAD)
def test_rules_refusals(native, bad):
    _, r, _, a = _good(native)
    _set(a, bad)
    assert native.lib().hg_op_logits_rules(C.byref(r), C.byref(a), None) == INVALID
    assert native.lib().hg_op_logits_rules(C.byref(r), None, None) == INVALID


def test_no_rows_is_no_work(native):
    """An empty batch launches nothing and needs no GPU."""
    c, r, a, lr = _good(native)
    L, by = native.lib(), C.byref
    for n_seqs, n_rows in ((0, 0), (1, 0), (0, 1)):
        r.n_seqs, r.n_rows = n_seqs, n_rows
        assert L.hg_op_kv8_append(by(c), by(r), by(a), None) == 0
        assert L.hg_op_kv8_read(by(c), by(r), P, None, None) == 0
        assert L.hg_op_kv8_attn(by(c), by(r), 12, P, P, P, None) == 0
        assert L.hg_op_logits_rules(by(r), by(lr), None) == 0


# ---------------------------------------------------------------------------------------------
# 64-bit forms
# ---------------------------------------------------------------------------------------------
def offsets(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def path_of(parent, r0, j):
    """Rows (local) that row j sees, itself first; empty for padding."""
    if parent is None:
        return list(range(j, -1, -1))
    path = []
    while j >= 0 and parent[r0 + j] != -2:
        path.append(j)
        j = int(parent[r0 + j]) if parent[r0 + j] < j else -1
    return path


def norm_rope(x, gain, eps, cos, sin):
    x = x.astype(np.float64)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    h = x.shape[-1] // 2
    a, b = n[..., :h], n[..., h:]
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.tile(np.abs(a) + np.abs(b), 2)


def quantised(y):
    """(codes, f32 scale) of rows, along the last axis."""
    y = y.astype(np.float64)
    sc = (np.abs(y).max(-1, keepdims=True) / 127.0).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(sc > 0, np.clip(np.round(y / sc.astype(np.float64)), -127, 127), 0)
    return code.astype(np.int8), sc[..., 0]


def block_index(hd):
    """Byte offsets [16][hd] of the K and the V codes of a page's block."""
    w, i = np.arange(PAGE)[:, None], np.arange(hd)[None]
    return (w // 8) * 8 * hd + (i // 16) * 128 + (w % 8) * 16 + i % 16, 16 * hd + i * 16 + w


def unpack(pool, hd):
    """K codes, V codes [page][head][16][hd] and scales [page][head][2][16] of a pool array."""
    k_at, v_at = block_index(hd)
    codes = pool.view(np.int8)
    return codes[..., k_at], codes[..., v_at], np.ascontiguousarray(pool[..., 32 * hd:32 * hd + 128]).view(
        np.float32).reshape(*pool.shape[:2], 2, PAGE)


def attend_ref(q, kc, vc, ks, vs, table, starts, row_off, parent, nkv):
    """[n][nh][hd] attention in 64 bits and a bound on the kernel's error, row by row."""
    n, nh, hd = q.shape
    g = nh // nkv
    out, tol = np.zeros((n, nh, hd)), np.zeros((n, nh, 1))
    n_pages = kc.shape[0]
    for s in range(len(starts)):
        for r in range(row_off[s], row_off[s + 1]):
            j = r - row_off[s]
            path = path_of(parent, row_off[s], j)
            if not path:
                continue
            slots = np.concatenate([np.arange(starts[s]), starts[s] + np.array(path)]).astype(np.int64)
            slots = slots[slots // PAGE < table.shape[1]]
            pages = table[s, slots // PAGE]
            ok = (pages >= 0) & (pages < n_pages)
            slots, pages = slots[ok], pages[ok]
            if not len(slots):
                continue
            w = slots % PAGE
            k = kc[pages, :, w].astype(np.float64) * ks[pages, :, w][..., None].astype(np.float64)  # [l][nkv][hd]
            v = vc[pages, :, w].astype(np.float64) * vs[pages, :, w][..., None].astype(np.float64)
            for h in range(nh):
                qq, kk, vv = q[r, h].astype(np.float64), k[:, h // g], v[:, h // g]
                sc = kk @ qq / np.sqrt(hd)
                p = np.exp(sc - sc.max())
                out[r, h] = p @ vv / p.sum()
                # a score: q rounded to 2^-23 of its greatest, sums in at most hd roundings of the terms
                ds = (np.abs(kk).sum(1).max() * np.abs(qq).max() * 2 + (np.abs(kk) @ np.abs(qq)).max() * 12) * U / np.sqrt(hd)
                ds += (np.abs(sc).max() + 1) * 8 * U
                # a probability: e^ds, exp's 2 ulp, 2^-23 of the greatest each; the sums' roundings
                tol[r, h] = np.abs(vv).max() * (2 * ds + 24 * U + 2 * len(slots) * U / p.sum() + len(slots) / 64 * U)
    return out, tol


def rules_ref(logits, row_off, parent, token, hists, rep, freq, pres, biases, valid, allow, exact):
    """The rules in f32, rounding after every operation (exact: in 64 bits), and the picks."""
    n, v = logits.shape
    out = logits.astype(np.float64 if exact else np.float32)
    f = out.dtype.type
    nxt = np.full(n, -1, np.int32)
    ops = np.zeros((n, v))  # roundings of a value, times its greatest intermediate
    with np.errstate(all="ignore"):
        for s in range(len(row_off) - 1):
            for r in range(row_off[s], row_off[s + 1]):
                path = path_of(parent, row_off[s], r - row_off[s])
                if not path:
                    continue
                ids = list(hists[s]) + ([] if token is None else [int(token[row_off[s] + j]) for j in path])
                count = np.bincount([i for i in ids if 0 <= i < v], minlength=v)
                x = out[r].copy()
                for i in np.nonzero(count)[0]:
                    big = abs(x[i])
                    for _ in range(count[i]):
                        if rep[s] != 1:
                            x[i] = f(x[i] / f(rep[s])) if x[i] > 0 else f(x[i] * f(rep[s]))
                            big = max(big, abs(x[i]))
                    t = f(f(freq[s]) * f(count[i]))
                    x[i] = f(f(x[i] - t) - f(pres[s]))
                    ops[r, i] = (count[i] + 3) * max(big, abs(t) + abs(f(pres[s])) + big)
                total, size = {}, {}
                for i, b in biases[s]:
                    total[i] = f(total.get(i, f(0)) + f(b))
                    size[i] = size.get(i, 0) + abs(f(b))
                for i, b in total.items():
                    if 0 <= i < v:
                        x[i] = f(x[i] + b)
                        ops[r, i] += len(biases[s]) * size[i] + abs(x[i])
                x[valid:] = -np.inf
                if allow[r] is not None:
                    x[~allow[r]] = -np.inf
                out[r] = x
                y = np.where(np.isnan(x), -np.inf, x)
                if y.max() > -np.inf:
                    nxt[r] = int(np.argmax(y))
    return out, nxt, ops


# ---------------------------------------------------------------------------------------------
# GPU harness
# ---------------------------------------------------------------------------------------------
def dev(a):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


class Batch:
    """A cache pool on the GPU with a shuffled page table, and the rows of one call."""

    def __init__(self, native, rng, heads, starts, rows, parent=None, spare=0, extra_cols=1, stride_pad=0):
        import torch

        self.native, self.heads = native, heads
        self.nh, self.nkv, self.hd = heads
        self.starts, self.rows = np.asarray(starts, np.int32), list(rows)
        self.row_off, self.n = offsets(rows), int(np.sum(rows))
        self.parent = None if parent is None else np.asarray(parent, np.int32)
        pages = [max(1, -(-(int(a) + b) // PAGE)) for a, b in zip(starts, rows)]
        self.n_pages, cols = sum(pages) + 2, max(pages) + extra_cols
        perm, at = rng.permutation(self.n_pages), 0
        self.table = np.full((len(starts), cols), 0x7fffffff, np.int32)
        for s, p in enumerate(pages):
            self.table[s, :p] = perm[at:at + p]
            at += p
        self.block = 32 * self.hd + 128
        self.stride = self.nkv * self.block + stride_pad
        self.spare = spare  # rows behind the last sequence
        self.pool = torch.zeros(self.n_pages * self.stride, dtype=torch.uint8, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.t = {k: dev(v) for k, v in (("table", self.table), ("row_off", self.row_off), ("start", self.starts),
                                         ("parent", self.parent))}
        self.cache = native.Kv8Cache(n_kv_heads=self.nkv, head_dim=self.hd, n_pages=self.n_pages, bt_stride=cols,
                                     block_table=ptr(self.t["table"]), pool=ptr(self.pool), page_stride=self.stride)
        self.r = native.Rows(n_seqs=len(self.rows), n_rows=self.n + spare, max_rows=max(max(self.rows), 1),
                             row_off=ptr(self.t["row_off"]), start=ptr(self.t["start"]), parent=ptr(self.t["parent"]),
                             err=ptr(self.err))

    def pool_np(self):
        return self.pool.cpu().numpy().reshape(self.n_pages, self.stride)[:, :self.nkv * self.block].reshape(
            self.n_pages, self.nkv, self.block)

    def fill(self, rng):
        """Random codes and scales in every block."""
        p = np.zeros((self.n_pages, self.stride), np.uint8)
        b = p[:, :self.nkv * self.block].reshape(self.n_pages, self.nkv, self.block)
        b = np.zeros((self.n_pages, self.nkv, self.block), np.uint8)
        b[..., :32 * self.hd] = np.clip(np.round(rng.standard_normal((self.n_pages, self.nkv, 32 * self.hd)) * 42), -127,
                                        127).astype(np.int8).view(np.uint8)
        sc = (0.02 + 0.02 * rng.random((self.n_pages, self.nkv, 32))).astype(np.float32)
        b[..., 32 * self.hd:] = sc.view(np.uint8)
        p[:, :self.nkv * self.block] = b.reshape(self.n_pages, -1)
        self.pool.copy_(dev(p.reshape(-1)))
        return b

    def append(self, qkv, gains, rope, eps=1e-5, max_pos=None, stream=None, q=True):
        import torch

        self.a_t = [dev(x) for x in (qkv, gains[0], gains[1], rope[0], rope[1])]
        out = torch.full((self.n + self.spare, self.nh * self.hd), 7.0, dtype=torch.float32, device="cuda") if q else None
        a = self.native.Kv8Append(n_heads=self.nh, max_pos=max_pos or len(rope[0]), eps=eps, qkv=ptr(self.a_t[0]),
                                  q_norm=ptr(self.a_t[1]), k_norm=ptr(self.a_t[2]), rope_cos=ptr(self.a_t[3]),
                                  rope_sin=ptr(self.a_t[4]), q_out=ptr(out))
        self.native.check(self.native.lib().hg_op_kv8_append(C.byref(self.cache), C.byref(self.r), C.byref(a), stream))
        return out

    def read(self, stream=None):
        import torch

        k, v = (torch.full((self.n + self.spare, self.nkv * self.hd), 7.0, device="cuda") for _ in range(2))
        self.native.check(self.native.lib().hg_op_kv8_read(C.byref(self.cache), C.byref(self.r), ptr(k), ptr(v), stream))
        return k, v

    def attn(self, q, stream=None, scratch=None, out=None):
        import torch

        L = self.native.lib()
        size = L.hg_op_kv8_attn_scratch_bytes(C.byref(self.cache), C.byref(self.r), self.nh)
        assert size > 0
        self.scratch = torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda") if scratch is None else scratch
        out = torch.full((self.n + self.spare, self.nh * self.hd), 7.0, device="cuda") if out is None else out
        self.q_t = q if hasattr(q, "data_ptr") else dev(q)
        self.native.check(L.hg_op_kv8_attn(C.byref(self.cache), C.byref(self.r), self.nh, ptr(self.q_t), ptr(out),
                                           ptr(self.scratch), stream))
        return out

    def err_code(self):
        return int(self.err.cpu()[0])


def rope_tables(hd, n):
    ang = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def random_tree(rng, rows, pad=0.1):
    p = []
    for n in rows:
        for j in range(n):
            p.append(-2 if rng.random() < pad else -1 if j == 0 else int(rng.integers(max(-1, j - 6), j)))
    return p


HEADS = [(12, 3, 128), (8, 2, 64), (4, 1, 64), (16, 8, 128), (3, 3, 64), (10, 2, 128), (32, 1, 64)]
# (starts, rows): single tokens at page borders, chains, ragged with empty sequences, long appends
ROWS = [([0], [1]), ([15, 16, 17, 31], [1, 1, 1, 1]), ([0, 5, 100], [3, 0, 20]), ([7, 0, 250, 16], [40, 16, 1, 33]),
        ([3], [130])]


# ---------------------------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("case", range(len(ROWS)))
@pytest.mark.parametrize("tree", [False, True])
def test_append_and_read(native, heads, case, tree):
    nh, nkv, hd = heads
    starts, rows = ROWS[case]
    rng = np.random.default_rng(100 * case + nh + hd)
    parent = random_tree(rng, rows) if tree else None
    b = Batch(native, rng, heads, starts, rows, parent, spare=2, stride_pad=48)
    before = b.fill(rng)
    qkv = (rng.standard_normal((b.n + 2, nh + 2 * nkv, hd)) * rng.uniform(0.1, 5, (b.n + 2, nh + 2 * nkv, 1))).astype(np.float32)
    qkv[0, nh, :] = 0.0          # a zero K row
    qkv[b.n // 2, nh + nkv] = 0  # and a zero V row: scale 0
    gains = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    rope = rope_tables(hd, 512)
    q = b.append(qkv, gains, rope).cpu().numpy().reshape(-1, nh, hd)
    k, v = (t.cpu().numpy().reshape(-1, nkv, hd) for t in b.read())
    after = b.pool_np()
    kc, vc, sc = unpack(after, hd)
    touched = np.zeros((b.n_pages, PAGE), bool)
    for s in range(len(rows)):
        for j in range(rows[s]):
            r, slot = b.row_off[s] + j, starts[s] + j
            page, w = b.table[s, slot // PAGE], slot % PAGE
            path = path_of(b.parent, b.row_off[s], j)
            if path:
                pos = starts[s] + len(path) - 1
                qr, amp = norm_rope(qkv[r, :nh], gains[0], 1e-5, rope[0][pos], rope[1][pos])
                # f32: sum of squares, root, two products, rotation: fewer than 24 roundings of |a| + |b|
                assert (np.abs(q[r] - qr) <= 24 * U * amp + 1e-30).all()
                kr, _ = norm_rope(qkv[r, nh:nh + nkv], gains[1], 1e-5, rope[0][pos], rope[1][pos])
                for got, gs, want in ((kc[page, :, w], sc[page, :, 0, w], kr), (vc[page, :, w], sc[page, :, 1, w], qkv[r, nh + nkv:])):
                    code, scale = quantised(want)
                    assert np.array_equal(got, code)
                    assert np.array_equal(gs.view(np.int32), scale.view(np.int32))
                touched[page, w] = True
            else:
                assert (q[r] == 0).all()
            for got, codes, i in ((k, kc, 0), (v, vc, 1)):
                want = codes[page, :, w].astype(np.float32) * sc[page, :, i, w][:, None]
                assert np.array_equal(got[r], want)
    for t in (q, k, v):
        assert (t[b.n:] == 7.0).all()  # rows behind the last sequence
    kb, vb, sb = unpack(before, hd)
    for a0, a1 in ((kb, kc), (vb, vc)):
        keep = np.broadcast_to(~touched[:, None, :, None], a0.shape)
        assert np.array_equal(a0[keep], a1[keep])
    keep = np.broadcast_to(~touched[:, None, None, :], sb.shape)
    assert np.array_equal(sb[keep], sc[keep])
    assert b.err_code() == 0


@pytest.mark.gpu
def test_append_nonfinite_rows_have_nan_scale(native):
    rng = np.random.default_rng(5)
    b = Batch(native, rng, (4, 2, 64), [0], [6])
    qkv = rng.standard_normal((6, 8, 64)).astype(np.float32)
    qkv[1, 4, 3] = np.nan
    qkv[2, 5, 60] = np.inf
    qkv[3, 6, 0] = -np.inf
    qkv[4, 7, 17] = np.nan
    qkv[5, 7] = 1e-44  # below what a scale can hold: reads back as zero
    one = np.ones(64, np.float32)
    b.append(qkv, (one, one), rope_tables(64, 16))
    k, v = (t.cpu().numpy().reshape(6, 2, 64) for t in b.read())
    assert np.isnan(k[1, 0]).all() and np.isfinite(k[1, 1]).all() and np.isnan(k[2, 1]).all()
    assert np.isnan(v[3, 0]).all() and np.isnan(v[4, 1]).all() and np.isfinite(v[4, 0]).all() and (v[5, 1] == 0).all()
    assert np.isfinite(k[[0, 3, 4, 5]]).all() and np.isfinite(v[[0, 1, 2]]).all()


@pytest.mark.gpu
def test_bad_tables_positions_and_offsets_are_left_out(native):
    """What device arrays get wrong is skipped and reported, and nothing else is written."""
    import torch

    rng = np.random.default_rng(6)
    heads, hd, nkv = (4, 1, 64), 64, 1
    one, rope = np.ones(hd, np.float32), rope_tables(hd, 64)
    qkv = rng.standard_normal((20, 6, hd)).astype(np.float32)
    # a table entry outside the pool: its rows are not cached, read as zeros, not attended
    b = Batch(native, rng, heads, [10], [20])
    b.fill(rng)
    for bad in (-1, b.n_pages, 0x7fffffff):
        b.err.zero_()
        table = b.table.copy()
        table[0, 1] = bad
        b.t["table"].copy_(dev(table))
        before = b.pool_np().copy()
        q = b.append(qkv, (one, one), rope).cpu().numpy()
        assert b.err_code() == CONTEXT
        assert (q[6:20] == 0).all() and (q[:6] != 0).any()
        changed = np.nonzero((before != b.pool_np()).reshape(b.n_pages, -1).any(1))[0]
        assert set(changed) <= {b.table[0, 0]}
        k, _ = b.read()
        assert (k.cpu().numpy()[6:20] == 0).all() and b.err_code() == CONTEXT
        kc, vc, sc = unpack(b.pool_np(), hd)
        qq = rng.standard_normal((20, 4, hd)).astype(np.float32)
        out = b.attn(qq).cpu().numpy().reshape(20, 4, hd)
        want, tol = attend_ref(qq, kc, vc, sc[:, :, 0], sc[:, :, 1], table, b.starts, b.row_off, None, nkv)
        assert (np.abs(out - want) <= tol).all()
    # positions past the RoPE table
    b = Batch(native, rng, heads, [10], [20])
    q = b.append(qkv, (one, one), rope, max_pos=15).cpu().numpy()
    assert b.err_code() == CONTEXT and (q[5:] == 0).all() and (q[:5] != 0).any()
    # more slots than the table holds; a negative start; more rows than max_rows; descending offsets
    for change, code in ((dict(starts=[2 * PAGE * 9]), CONTEXT), (dict(starts=[2 ** 31 - 5]), CONTEXT), (dict(starts=[-3]), INVALID),
                         (dict(max_rows=4), INVALID), (dict(row_off=[0, 40]), INVALID), (dict(row_off=[9, 3]), INVALID),
                         (dict(row_off=[-4, 3]), INVALID)):
        b = Batch(native, rng, heads, [10], [20])
        if "starts" in change:
            b.t["start"].copy_(dev(np.array(change["starts"], np.int32)))
        if "row_off" in change:
            b.t["row_off"].copy_(dev(np.array(change["row_off"], np.int32)))
        b.r.max_rows = change.get("max_rows", b.r.max_rows)
        b.append(qkv, (one, one), rope)
        assert b.err_code() == code, change
        b.err.zero_()
        b.read()
        b.attn(rng.standard_normal((20, 4, hd)).astype(np.float32))
        torch.cuda.synchronize()
        assert b.err_code() == code, change


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def _check_attn(b, rng, q=None, seqs=None):
    pool = b.fill(rng)
    q = rng.standard_normal((b.n + b.spare, b.nh, b.hd)).astype(np.float32) if q is None else q
    out = b.attn(q).cpu().numpy().reshape(-1, b.nh, b.hd)
    kc, vc, sc = unpack(pool, b.hd)
    want, tol = attend_ref(q[:b.n], kc, vc, sc[:, :, 0], sc[:, :, 1], b.table, b.starts, b.row_off, b.parent, b.nkv)
    bad = np.abs(out[:b.n] - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(out[:b.n] - want).max(), tol.max())
    assert (out[b.n:] == 7.0).all()
    assert b.err_code() == 0
    return out, want


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("starts,rows", [([0], [1]), ([1], [1]), ([127, 128, 129, 0], [1, 1, 1, 1]),
                                         ([5, 300, 0, 77], [2, 1, 5, 0]), ([1000], [1])])
def test_attn_decode_and_chains(native, heads, starts, rows):
    rng = np.random.default_rng(sum(starts) + heads[0])
    _check_attn(Batch(native, rng, heads, starts, rows, spare=1, stride_pad=16), rng)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("starts,rows", [([0, 3], [1, 9]), ([120, 0, 130], [12, 7, 20]), ([513], [64]), ([40], [150])])
def test_attn_trees(native, heads, starts, rows):
    rng = np.random.default_rng(sum(rows) + heads[0] + 1)
    b = Batch(native, rng, heads, starts, rows, random_tree(rng, rows), spare=3)
    out, _ = _check_attn(b, rng)
    pad = b.parent == -2
    assert (out[:b.n][pad] == 0).all()


@pytest.mark.gpu
def test_attn_many_sequences_and_long_context(native):
    """More sequences than SMs with uneven lengths, and one context of many splits."""
    rng = np.random.default_rng(9)
    heads = (4, 1, 64)
    starts, rows = rng.integers(0, 400, 300), rng.integers(0, 4, 300)
    _check_attn(Batch(native, rng, heads, starts, rows, random_tree(rng, rows, 0.2)), rng)
    _check_attn(Batch(native, rng, (12, 3, 128), [20000, 3], [2, 1]), rng)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-3, 30.0, 3e4])
def test_attn_score_ranges(native, scale):
    """Flat, peaked and one-hot probabilities."""
    rng = np.random.default_rng(10)
    b = Batch(native, rng, (4, 2, 128), [333, 20], [3, 5], spare=0)
    q = (rng.standard_normal((b.n, 4, 128)) * scale).astype(np.float32)
    q[1, 2] = 0.0
    _check_attn(b, rng, q)


@pytest.mark.gpu
def test_attn_nan_goes_where_it_is_seen(native):
    """A poisoned slot reaches exactly the rows that see it; stale blocks behind the length reach none."""
    rng = np.random.default_rng(11)
    nh, nkv, hd = heads = (4, 2, 64)
    b = Batch(native, rng, heads, [20, 20], [4, 2], [-1, 0, 0, -2, -1, 0])
    pool = b.fill(rng)
    sc = np.ascontiguousarray(pool[..., 32 * hd:]).view(np.float32)  # [page][head][32]
    last = b.table[0, 1], b.table[1, 1]
    sc[last[0], :, 8:16] = np.nan    # slots 24.. of sequence 0: behind its rows (K scales)
    sc[last[0], :, 24:32] = np.inf   # (V scales)
    sc[last[0], 1, 5] = np.nan       # slot 21: row 1's K, kv head 1
    sc[last[0], :, 7] = np.nan       # slot 23: the padding row
    sc[b.table[1, 0], 0, 16 + 3] = np.nan  # slot 3 of sequence 1: a V scale, kv head 0
    pool[..., 32 * hd:] = sc.view(np.uint8)
    b.pool.copy_(dev(pool.reshape(-1)))
    q = rng.standard_normal((6, nh, hd)).astype(np.float32)
    q[5, 3, 7] = np.nan
    out = b.attn(q).cpu().numpy().reshape(6, nh, hd)
    nan = np.isnan(out).all(-1)
    assert np.array_equal(nan, np.isnan(out).any(-1))
    want = np.zeros((6, nh), bool)
    want[1, 2:] = True   # row 1 sees itself
    want[4:, :2] = True  # sequence 1's rows see slot 3
    want[5, 3] = True    # a NaN query
    assert np.array_equal(nan, want)
    assert (out[3] == 0).all()


@pytest.mark.gpu
def test_attn_64_bit_offsets(native):
    """Pages behind 4 GiB of pool."""
    import torch

    rng = np.random.default_rng(12)
    b = Batch(native, rng, (4, 1, 64), [50], [2])
    pool = b.fill(rng)
    far = (5 << 30) // b.stride
    big = torch.zeros((far + b.n_pages) * b.stride, dtype=torch.uint8, device="cuda")
    big[far * b.stride:] = b.pool
    b.t["table"].copy_(dev(np.where(b.table < b.n_pages, b.table + far, b.table).astype(np.int32)))
    b.cache.pool, b.cache.n_pages = ptr(big), far + b.n_pages
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    out = b.attn(q).cpu().numpy().reshape(2, 4, 64)
    kc, vc, sc = unpack(pool, 64)
    want, tol = attend_ref(q, kc, vc, sc[:, :, 0], sc[:, :, 1], b.table, b.starts, b.row_off, None, 1)
    assert (np.abs(out - want) <= tol).all()
    k, _ = b.read()
    w = (50 + np.arange(2)) % PAGE
    page = b.table[0, (50 + np.arange(2)) // PAGE]
    assert np.array_equal(k.cpu().numpy(), kc[page, 0, w].astype(np.float32) * sc[page, 0, 0, w][:, None])


# ---------------------------------------------------------------------------------------------
# rules
# ---------------------------------------------------------------------------------------------
def _rules(native, logits, rows, parent=None, token=None, hists=None, rep=None, freq=None, pres=None, biases=None,
           valid=0, masks=None, mask_row=None, in_place=False, ld=None, spare=0, want_next=True, stream=None):
    import torch

    n, v = logits.shape
    ld = ld or v
    buf = np.full((n, ld), 5.0, np.float32)
    buf[:, :v] = logits
    t = {"logits": dev(buf), "row_off": dev(offsets(rows)), "parent": dev(None if parent is None else np.asarray(parent, np.int32)),
         "token": dev(None if token is None else np.asarray(token, np.int32)), "mask_row": dev(None if mask_row is None else np.asarray(mask_row, np.int32))}
    t["out"] = t["logits"] if in_place else torch.full((n, ld), 9.0, device="cuda")
    t["next"] = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    f = {}
    if hists is not None:
        t["hist_off"] = dev(offsets([len(h) for h in hists]))
        t["hist"] = dev(np.array([i for h in hists for i in h] + [0], np.int32))
    for k, x in (("rep_penalty", rep), ("freq_penalty", freq), ("pres_penalty", pres)):
        t[k] = dev(None if x is None else np.asarray(x, np.float32))
    if biases is not None:
        t["bias_off"] = dev(offsets([len(b) for b in biases]))
        t["bias_id"] = dev(np.array([i for b in biases for i, _ in b] + [0], np.int32))
        t["bias"] = dev(np.array([x for b in biases for _, x in b] + [0], np.float32))
    if masks is not None:
        bits = np.zeros((len(masks), (v + 31) // 32 * 32), bool)
        bits[:, :v] = masks
        t["mask"] = dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
        f["mask_words"] = bits.shape[1] // 32
    a = native.LogitsRules(vocab=v, valid=valid, ld=ld, ld_out=ld, **f)
    for k in ("logits", "out", "token", "hist_off", "hist", "rep_penalty", "freq_penalty", "pres_penalty", "bias_off", "bias_id", "bias", "mask", "mask_row"):
        setattr(a, k, ptr(t.get(k)))
    a.next_ids = ptr(t["next"]) if want_next else None
    r = native.Rows(n_seqs=len(rows), n_rows=n, max_rows=max(rows), row_off=ptr(t["row_off"]), parent=ptr(t["parent"]))
    native.check(native.lib().hg_op_logits_rules(C.byref(r), C.byref(a), stream))
    torch.cuda.synchronize()
    return t["out"].cpu().numpy(), t["next"].cpu().numpy()


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 31, 1000, 50257, 50304, 131073])
@pytest.mark.parametrize("n_seqs,tree", [(1, False), (5, True), (70, True)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules(native, vocab, n_seqs, tree, in_place):
    rng = np.random.default_rng(vocab + n_seqs)
    rows = [int(x) for x in (rng.integers(0, 4, n_seqs) if tree else np.ones(n_seqs, int))]
    rows[0] = max(rows[0], 1)
    n = sum(rows) + 1  # one row behind the last sequence
    parent = random_tree(rng, rows + [1]) if tree else None
    logits = (rng.standard_normal((n, vocab)) * 4).astype(np.float32)
    pick = lambda k: (vocab * rng.random(k) ** 3).astype(int).tolist()  # noqa: E731
    hists = [pick(int(rng.integers(0, 300))) + [-1, vocab, 2 ** 31 - 1] for _ in rows]
    biases = [[(i, float(np.float32(rng.standard_normal()))) for i in pick(int(rng.integers(0, 70))) + [-5, vocab]] for _ in rows]
    rep, freq, pres = 1 + 0.4 * rng.random(n_seqs), rng.random(n_seqs) * 0.3, rng.random(n_seqs)
    rep, freq, pres = (x.astype(np.float32) for x in (rep, freq, pres))
    rep[0] = 1.0
    token = pick(n) if tree else None
    masks = rng.random((3, vocab)) < 0.4
    mask_row = rng.integers(-1, 3, n)
    allow = [None if m < 0 else masks[m] for m in mask_row]
    valid = max(1, vocab - 47) if vocab > 100 else 0
    out, nxt = _rules(native, logits, rows, parent, token, hists, rep, freq, pres, biases, valid, masks, mask_row, in_place, ld=vocab + 4 * (vocab % 2))
    off = offsets(rows)
    args = (off, parent, token, hists, rep, freq, pres, biases, valid or vocab, allow)
    want, ids, _ = rules_ref(logits, *args, exact=False)
    m = sum(rows)
    pad = np.zeros(n, bool) if parent is None else np.array(parent) == -2
    pad[m:] = True
    assert _same(out[~pad][:, :vocab], want[~pad])
    assert np.array_equal(nxt[:m], ids[:m]) and nxt[m] == -9
    stay = logits if in_place else np.full_like(logits, 9.0)
    assert np.array_equal(out[pad][:, :vocab], stay[pad])
    assert (out[:, vocab:] == (5.0 if in_place else 9.0)).all()
    exact, _, ops = rules_ref(logits, *args, exact=True)
    fin = np.isfinite(exact) & ~pad[:, None]
    assert (np.abs(out[:, :vocab].astype(np.float64) - exact)[fin] <= (ops * U)[fin] + U * np.abs(exact)[fin]).all()


@pytest.mark.gpu
def test_rules_special_values(native):
    """NaN never wins, infinities and barred NaNs, ties to the first, rows with nothing left, the same id
    many times in the biases and the history."""
    v = 9000
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, v)).astype(np.float32)
    x[0, 17] = np.nan
    x[0, 40] = x[0, 8990] = 50.0       # a tie
    x[1, :] = -np.inf
    x[2, 5] = np.inf
    x[3, 100:200] = np.nan             # barred by the mask
    x[4, :] = np.nan
    x[5, 8999] = 1e30
    masks = np.ones((6, v), bool)
    masks[3, 100:200] = False
    masks[5] = False
    hists = [[40] * 3, [], [5] * 200, [7] * 1500, [1], []]
    biases = [[(40, 1e8), (3, 1.0), (40, 1.0), (40, -1e8)] + [(8, 0.1)] * 100, [(9, np.inf)], [], [(7, -1.0)] * 64, [], []]
    rep = np.array([1.0, 2.0, 1.5, 1.01, 3.0, 1.0], np.float32)
    zero = np.zeros(6, np.float32)
    out, nxt = _rules(native, x, [1] * 6, hists=hists, rep=rep, biases=biases, masks=masks)
    want, ids, _ = rules_ref(x, offsets([1] * 6), None, None, hists, rep, zero, zero, biases, v, list(masks), exact=False)
    assert _same(out, want) and np.array_equal(nxt, ids)
    assert nxt.tolist()[1:] == [-1, 5, ids[3], -1, -1] and np.isnan(out[1, 9])
    out, nxt = _rules(native, x, [1] * 6)  # no rules at all: a copy and the picks
    assert _same(out, x) and nxt.tolist()[:3] == [40, -1, 5] and nxt[5] == 8999


@pytest.mark.gpu
def test_rules_equal_engine_penalty(native):
    """The pick under a repetition penalty is the one that the host sampler makes of the same logits."""
    rng = np.random.default_rng(8)
    v, p = 50304, np.float32(1.3)
    logits = (rng.standard_normal((4, v)) * 2).astype(np.float32)
    hists = [np.argsort(-logits[i])[:40].repeat(i + 1).tolist() for i in range(4)]
    out, nxt = _rules(native, logits, [1] * 4, hists=hists, rep=[p] * 4, valid=50257)
    for i in range(4):
        x = logits[i].copy()
        for t in hists[i]:
            x[t] = x[t] / p if x[t] > 0 else x[t] * p
        x[50257:] = -np.inf
        got, state = C.c_uint32(), C.c_uint64(1)
        native.check(native.lib().hg_host_sample(x.ctypes.data, v, 0.0, 0.95, C.byref(state), C.byref(got)))
        assert np.array_equal(out[i], x) and nxt[i] == got.value


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_drafted_step_end_to_end(native):
    """Prompt in, a tree drafted behind it, its rows attended, ruled and the accepted path appended again
    as a chain: a row of the tree gives what decoding its path one token at a time gives, bit for bit."""
    import torch

    rng = np.random.default_rng(21)
    nh, nkv, hd = heads = (8, 2, 64)
    one, rope = np.ones(hd, np.float32), rope_tables(hd, 256)
    ctx, rows = [37, 5, 0], [6, 4, 3]
    parent = [-1, 0, 0, 1, -2, 3, -1, -1, 1, 2, -1, 0, 1]
    prompt = rng.standard_normal((sum(ctx), nh + 2 * nkv, hd)).astype(np.float32)
    tree = rng.standard_normal((sum(rows), nh + 2 * nkv, hd)).astype(np.float32)
    b = Batch(native, rng, heads, ctx, rows, parent)
    fresh = Batch(native, rng, heads, [0, 0, 0], ctx)
    for name in ("cache", "pool", "table", "n_pages"):
        setattr(fresh, name, getattr(b, name))
    fresh.append(prompt, (one, one), rope)
    q = b.append(tree, (one, one), rope)
    out = b.attn(q).cpu().numpy()
    want_pool = b.pool_np()
    kc, vc, sc = unpack(want_pool, hd)
    qn = q.cpu().numpy().reshape(-1, nh, hd)
    ref, tol = attend_ref(qn, kc, vc, sc[:, :, 0], sc[:, :, 1], b.table, b.starts, b.row_off, b.parent, nkv)
    assert (np.abs(out.reshape(ref.shape) - ref) <= tol).all()
    # logits of the rows, ruled along their paths
    proj = torch.from_numpy(rng.standard_normal((nh * hd, 500)).astype(np.float32)).cuda()
    logits = (torch.from_numpy(out).cuda() @ proj).cpu().numpy()
    token = rng.integers(0, 500, sum(rows)).tolist()
    hists = [rng.integers(0, 500, c).tolist() for c in ctx]
    rep = np.array([1.2, 1.0, 1.5], np.float32)
    ruled, nxt = _rules(native, logits, rows, parent, token, hists, rep)
    zero = np.zeros(3, np.float32)
    want, ids, _ = rules_ref(logits, b.row_off, b.parent, token, hists, rep, zero, zero, [[]] * 3, 500, [None] * sum(rows), exact=False)
    live = np.array(parent) != -2
    assert _same(ruled[live], want[live]) and np.array_equal(nxt, ids)
    # accept row 5's path of sequence 0, row 3's of sequence 1, row 2's of sequence 2: appended as chains
    paths = [path_of(np.array(parent), int(b.row_off[s]), j)[::-1] for s, j in ((0, 5), (1, 3), (2, 2))]
    chain = Batch(native, rng, heads, ctx, [len(p) for p in paths])
    for name in ("cache", "pool", "table", "n_pages"):
        setattr(chain, name, getattr(b, name))
    picked = np.concatenate([tree[b.row_off[s] + np.array(p)] for s, p in enumerate(paths)])
    q2 = chain.append(picked, (one, one), rope)
    rows_of = np.concatenate([b.row_off[s] + np.array(p) for s, p in enumerate(paths)])
    assert np.array_equal(q2.cpu().numpy(), q.cpu().numpy()[rows_of])  # same positions, same q
    out2 = chain.attn(q2).cpu().numpy().reshape(-1, nh, hd)
    ref2, tol2 = ref.reshape(-1, nh, hd)[rows_of], tol[rows_of]
    assert (np.abs(out2 - ref2) <= tol2).all()
    assert b.err_code() == chain.err_code() == fresh.err_code() == 0


@pytest.mark.gpu
def test_graphs_and_streams(native):
    """Captured once, replayed with new lengths on another stream; two graphs that share a scratch buffer
    one after the other; results equal the eager calls bit for bit."""
    import torch

    rng = np.random.default_rng(22)
    heads = (12, 3, 128)
    b = Batch(native, rng, heads, [700, 90], [2, 3], extra_cols=4)
    b.fill(rng)
    q = dev(rng.standard_normal((5, 12, 128)).astype(np.float32))
    eager = b.attn(q).clone()
    scratch, st = b.scratch, torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    outs, graphs = [torch.zeros_like(eager) for _ in range(2)], []
    with torch.cuda.stream(st):
        for o in outs:
            b.attn(q, st.cuda_stream, scratch, o)  # first use outside a capture
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                b.attn(q, st.cuda_stream, scratch, o)
                b.attn(q, st.cuda_stream, scratch, o)
            graphs.append(g)
        for o in outs:
            o.zero_()
        for _ in range(3):
            for g in graphs:
                g.replay()
    st.synchronize()
    assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
    b.t["start"].copy_(dev(np.array([311, 64], np.int32)))  # shorter contexts, the same graph
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graphs[0].replay()
    st.synchronize()
    assert torch.equal(outs[0], b.attn(q)) and not torch.equal(outs[0], eager)


# ---------------------------------------------------------------------------------------------
# the variants and their borders
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [1, 2, 3, 4, 7, 8, 9, 16, 33])
@pytest.mark.parametrize("extra_cols", [1, 40, 900])
def test_attn_every_block_size(native, hd, nodes, extra_cols):
    """Uniform trees that fill blocks of 4, 8, 16 and 32 rows exactly, or leave some of one, under tables
    so short that a unit has its own CTA, longer (its own cluster) and long (a share of the line)."""
    rng = np.random.default_rng(nodes + hd)
    rows = [nodes] * 3
    b = Batch(native, rng, (8, 2, hd), [0, 250, 285], rows, random_tree(rng, rows, 0.05), spare=1, extra_cols=extra_cols)
    _check_attn(b, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(12, 3, 128), (8, 2, 64), (16, 8, 128)])
def test_attn_clusters_of_every_size(native, heads):
    """One sequence under tables from one tile to more than the largest cluster takes; the context leaves
    some CTAs of a cluster without a tile."""
    rng = np.random.default_rng(41)
    for cols in (8, 16, 17, 40, 100, 200, 383, 384, 385, 500):
        for start in (0, 3, min(cols * PAGE - 2, 700)):
            b = Batch(native, rng, heads, [start], [2], extra_cols=1)
            table = np.full((1, cols), 0x7fffffff, np.int32)
            table[:, :b.table.shape[1]] = b.table[:, :cols]
            b.table, b.t["table"] = table, dev(table)
            b.cache.block_table, b.cache.bt_stride = ptr(b.t["table"]), cols
            _check_attn(b, rng)


@pytest.mark.gpu
def test_parents_that_break_the_rule(native):
    """A parent that is not below its row counts as none, -7 as padding; both are the same to every call."""
    import torch

    rng = np.random.default_rng(31)
    bad = [-1, 5, 1, -7, 4, 3, -2, 2]      # rows 1 and 4 point at or above themselves, row 5 at padding
    good = [-1, -1, 1, -2, -1, -1, -2, 2]
    outs = []
    for parent in (bad, good):
        rng = np.random.default_rng(32)
        b = Batch(native, rng, (4, 1, 64), [21], [8], parent)
        qkv = rng.standard_normal((8, 6, 64)).astype(np.float32)
        q = b.append(qkv, [np.ones(64, np.float32)] * 2, rope_tables(64, 64))
        out = b.attn(q)
        torch.cuda.synchronize()
        assert b.err_code() == (INVALID if parent is bad else 0)
        logits = rng.standard_normal((8, 300)).astype(np.float32)
        token = rng.integers(0, 300, 8).tolist()
        ruled, nxt = _rules(native, logits, [8], parent, token, [[1, 2]], np.array([1.5], np.float32))
        outs.append((q.cpu().numpy(), out.cpu().numpy(), b.pool_np(), ruled, nxt))
    for x, y in zip(*outs):
        assert np.array_equal(x, y)


@pytest.mark.gpu
def test_append_takes_gains_at_any_float(native):
    """Gains and RoPE tables need only be aligned to a float."""
    import torch

    rng = np.random.default_rng(33)
    for heads in ((4, 2, 128), (4, 2, 64)):
        b = Batch(native, rng, heads, [3], [20])
        hd = heads[2]
        qkv = rng.standard_normal((20, 8, hd)).astype(np.float32)
        gains = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        rope = rope_tables(hd, 64)
        want, pool = b.append(qkv, gains, rope).cpu().numpy(), b.pool_np()
        b.pool.zero_()
        shifted = [torch.cat([torch.zeros(1, device="cuda"), t.reshape(-1)]) for t in (dev(gains[0]), dev(gains[1]), dev(rope[0]), dev(rope[1]))]
        out = torch.empty((20, 4 * hd), device="cuda")
        ptrs = [t.data_ptr() + 4 for t in shifted]
        a = native.Kv8Append(n_heads=4, max_pos=64, eps=1e-5, qkv=ptr(b.a_t[0]), q_norm=ptrs[0], k_norm=ptrs[1],
                             rope_cos=ptrs[2], rope_sin=ptrs[3], q_out=ptr(out))
        native.check(native.lib().hg_op_kv8_append(C.byref(b.cache), C.byref(b.r), C.byref(a), None))
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(b.pool_np(), pool)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,hist,ids", [(1000, 9000, 3), (1000, 3000, 1000), (60000, 20000, 2), (250003, 900, 250003), (250003, 12000, 40)])
def test_rules_long_lists_and_chunks(native, vocab, hist, ids):
    """Counts that 13 bits do not hold, more listed ids than a work list, rows of several chunks."""
    rng = np.random.default_rng(hist + ids)
    logits = (rng.standard_normal((3, vocab)) * 5).astype(np.float32)
    hists = [rng.integers(0, ids, n).tolist() for n in (hist, 0, hist // 2)]
    biases = [[(int(i), 0.25) for i in rng.integers(0, vocab, n)] for n in (5, 1500, 0)]
    rep, freq, pres = (np.array(x, np.float32) for x in ([1.0005, 1.0, 0.999], [0.0, 0.5, 0.001], [0.1, 0.0, 0.0]))
    masks = rng.random((2, vocab)) < 0.5
    out, nxt = _rules(native, logits, [1] * 3, None, None, hists, rep, freq, pres, biases, 0, masks, [0, -1, 1])
    want, got, _ = rules_ref(logits, offsets([1] * 3), None, None, hists, rep, freq, pres, biases, vocab,
                             [masks[0], None, masks[1]], exact=False)
    assert _same(out, want) and np.array_equal(nxt, got)


@pytest.mark.gpu
def test_rules_long_path(native):
    """A drafted path of more tokens than are in hand at a time, as a tree and as a chain."""
    rng = np.random.default_rng(35)
    n, v = 601, 700
    logits = rng.standard_normal((n, v)).astype(np.float32)
    token = rng.integers(0, 50, n).tolist()
    rep, zero = np.array([1.1], np.float32), np.zeros(1, np.float32)
    chain = [j - 1 for j in range(n)]
    outs = [_rules(native, logits, [n], parent, token, [[3]], rep) for parent in (chain, None)]
    want, ids, _ = rules_ref(logits, offsets([n]), None, token, [[3]], rep, zero, zero, [[]], v, [None] * n, exact=False)
    for out, nxt in outs:
        assert _same(out, want) and np.array_equal(nxt, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [(0, 0), (1, 1), (2, 2), (3, 3), (1, 2)])
def test_rules_any_alignment(native, shift):
    """Rows that start anywhere in a 16-byte line, alike and not alike in logits and out."""
    import torch

    rng = np.random.default_rng(36)
    v, n = 5003, 4
    x = rng.standard_normal((n, v)).astype(np.float32)
    src, dst = (torch.full((n * v + 8,), 4.0, device="cuda") for _ in range(2))
    src[shift[0]:shift[0] + n * v] = dev(x).reshape(-1)
    row_off, nxt = dev(offsets([1] * n)), torch.full((n,), -9, dtype=torch.int32, device="cuda")
    a = native.LogitsRules(vocab=v, valid=v - 3, logits=ptr(src) + 4 * shift[0], out=ptr(dst) + 4 * shift[1], next_ids=ptr(nxt))
    r = native.Rows(n_seqs=n, n_rows=n, max_rows=1, row_off=ptr(row_off))
    native.check(native.lib().hg_op_logits_rules(C.byref(r), C.byref(a), None))
    got = dst.cpu().numpy()
    want = x.copy()
    want[:, v - 3:] = -np.inf
    assert np.array_equal(got[shift[1]:shift[1] + n * v].reshape(n, v), want)
    assert (got[:shift[1]] == 4.0).all() and (got[shift[1] + n * v:] == 4.0).all()
    assert nxt.cpu().numpy().tolist() == want.argmax(1).tolist()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(native):
    """Each with its own scratch and outputs: the same bits as one after the other."""
    import torch

    rng = np.random.default_rng(37)
    bs = [Batch(native, rng, (12, 3, 128), rng.integers(100, 3000, 40), [1] * 40),
          Batch(native, rng, (8, 2, 64), rng.integers(1, 900, 30), [9] * 30)]
    qs, want, streams = [], [], [torch.cuda.Stream() for _ in bs]
    for b in bs:
        b.fill(rng)
        qs.append(dev(rng.standard_normal((b.n, b.nh, b.hd)).astype(np.float32)))
        want.append(b.attn(qs[-1]).clone())
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for b, q, o, st in zip(bs, qs, outs, streams):
            b.attn(q, st.cuda_stream, b.scratch, o)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


FIRST_CAPTURE = """
import sys
sys.path[:0] = ["tests", "."]
import numpy as np, torch, ctypes as C
import test_kv8 as t
from hobbylm_b200 import _native as N
rng = np.random.default_rng(1)
b = t.Batch(N, rng, (12, 3, 128), [40, 7], [2, 3])
qkv = rng.standard_normal((5, 18, 128)).astype(np.float32)
one, rope = np.ones(128, np.float32), t.rope_tables(128, 64)
args = [t.dev(x) for x in (qkv, one, one, *rope)]
q, out, ids = torch.zeros(5, 1536, device="cuda"), torch.zeros(5, 1536, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
a = N.Kv8Append(n_heads=12, max_pos=64, eps=1e-5, qkv=t.ptr(args[0]), q_norm=t.ptr(args[1]), k_norm=t.ptr(args[2]),
                rope_cos=t.ptr(args[3]), rope_sin=t.ptr(args[4]), q_out=t.ptr(q))
lr = N.LogitsRules(vocab=1536, logits=t.ptr(out), out=t.ptr(out), next_ids=t.ptr(ids))
L, by = N.lib(), C.byref
scratch = torch.empty(L.hg_op_kv8_attn_scratch_bytes(by(b.cache), by(b.r), 12), dtype=torch.uint8, device="cuda")
g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
st.wait_stream(torch.cuda.current_stream())
with torch.cuda.graph(g, stream=st):  # the process's first use of each kernel
    s = st.cuda_stream
    N.check(L.hg_op_kv8_append(by(b.cache), by(b.r), by(a), s))
    N.check(L.hg_op_kv8_attn(by(b.cache), by(b.r), 12, t.ptr(q), t.ptr(out), t.ptr(scratch), s))
    N.check(L.hg_op_logits_rules(by(b.r), by(lr), s))
g.replay()
torch.cuda.synchronize()
got = out.clone(), ids.clone()
b2 = b.append(qkv, (one, one), rope)
want = b.attn(b2)
assert torch.equal(got[0], want) and torch.equal(got[1].long(), want.argmax(1)), "replay differs"
print("first capture ok")
"""


@pytest.mark.gpu
def test_first_use_inside_a_capture():
    """A process whose first call of each kernel is recorded into a graph."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CAPTURE], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "first capture ok" in r.stdout, r.stdout[-500:] + r.stderr[-1500:]
