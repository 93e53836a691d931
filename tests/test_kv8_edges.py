"""Edges of the 8-bit KV cache, the tree attention and the logit rules, against plain 64-bit forms:
pages of mostly padding rows, scales of any spread, ties, chains given by their parents.

Tolerances count roundings: u = 2^-24 is half a step of f32 (relative).
"""
import ctypes as C

import numpy as np
import pytest

import test_kv8 as kv

U, PAGE, INVALID, CONTEXT = kv.U, kv.PAGE, kv.INVALID, kv.CONTEXT
EPS = float(np.float32(1e-5))  # as the calls take it


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(16, 8, 128), (12, 3, 128), (8, 2, 64)])
def test_append_between_padding_rows(native, heads):
    """Pages of 5 to 15 rows, half of them padding or past the RoPE table, in any order, from a buffer
    larger than the L2 cache: a live row's q, codes and scales come from its own projections alone."""
    import torch

    nh, nkv, hd = heads
    rng = np.random.default_rng(nh)
    n_seqs = min(1024, 160 * 2 ** 20 // (10 * (nh + 2 * nkv) * hd * 4))  # about 160 MB
    rows = rng.integers(5, 16, n_seqs)
    starts = rng.choice([0, 16, 32, 48, 52], n_seqs)  # from 48 + max. depth on: past the table
    parent = []
    for n in rows:
        live = [j for j in range(n) if rng.random() < 0.5]
        parent += [-2 if j not in live else int(rng.integers(-1, j)) if j else -1 for j in range(n)]
    b = kv.Batch(native, rng, heads, starts, rows, parent)
    size = rng.uniform(0.1, 5, (b.n, nh + 2 * nkv, 1))
    qkv = (rng.standard_normal((b.n, nh + 2 * nkv, hd), np.float32) * size).astype(np.float32)
    gains = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    rope, max_pos = kv.rope_tables(hd, 64), 55
    path = [kv.path_of(b.parent, b.row_off[s], j) for s in range(n_seqs) for j in range(rows[s])]
    seq = np.repeat(np.arange(n_seqs), rows)
    slot = b.starts[seq] + np.arange(b.n) - b.row_off[seq]
    pos = b.starts[seq] + np.array([len(p) for p in path]) - 1
    live = np.array([bool(p) for p in path]) & (pos < max_pos)
    assert 0.3 < live.mean() < 0.6 and (pos >= max_pos).any()
    at, page, w = pos[live], b.table[seq[live], slot[live] // PAGE], slot[live] % PAGE
    cos, sin = rope[0][at][:, None], rope[1][at][:, None]
    qr, amp = kv.norm_rope(qkv[live, :nh], gains[0], EPS, cos, sin)
    kr, _ = kv.norm_rope(qkv[live, nh:nh + nkv], gains[1], EPS, cos, sin)
    want = [kv.quantised(kr), kv.quantised(qkv[live, nh + nkv:])]
    a_t = None
    for _ in range(4):
        b.pool.zero_()
        if a_t is None:
            q = b.append(qkv, gains, rope, max_pos=max_pos)
            a_t = b.a_t
        else:  # the same inputs again
            a = native.Kv8Append(n_heads=nh, max_pos=max_pos, eps=1e-5, qkv=kv.ptr(a_t[0]), q_norm=kv.ptr(a_t[1]),
                                 k_norm=kv.ptr(a_t[2]), rope_cos=kv.ptr(a_t[3]), rope_sin=kv.ptr(a_t[4]), q_out=kv.ptr(q))
            q.fill_(7.0)
            native.check(native.lib().hg_op_kv8_append(C.byref(b.cache), C.byref(b.r), C.byref(a), None))
        torch.cuda.synchronize()
        got = q.cpu().numpy().reshape(-1, nh, hd)
        assert (np.abs(got[live] - qr) <= 24 * U * amp + 1e-30).all()
        assert (got[~live] == 0).all()
        codes = kv.unpack(b.pool_np(), hd)
        for i in range(2):
            wc, ws = np.zeros_like(codes[i]), np.zeros((b.n_pages, nkv, PAGE), np.float32)
            wc[page, :, w], ws[page, :, w] = want[i]
            assert np.array_equal(codes[i], wc)
            assert np.array_equal(codes[2][:, :, i].view(np.int32), ws.view(np.int32))
    assert b.err_code() == CONTEXT


# ---------------------------------------------------------------------------------------------
# attention at any spread of scales
# ---------------------------------------------------------------------------------------------
def _attend(q, kc, vc, ks, vs, b, f32=False):
    """Attention in 64 bits with a bound on the kernel's error, and (f32) the plain 32-bit form beside it.

    The bound, from what the kernel rounds, for a row that sees n slots in T tiles, with x its scores:
    * the joined sums, K scale, q scale, and the sum with the V scale's exponent: 5 roundings of |x|, 3 of
      the exponent in log2 units (its rounding, the difference to the maximum, that maximum in the join);
      exp2: 2 ulp. A row's maximum changes at most T + 2 times (its tiles, the join), each an exp2.
    * q: fixed point, off by 2^-30 of its greatest value at most, each dim's with a sign of its own: eight
      of the greatest deviations over dims and slots (Hoeffding: 1e-13).
    * a product p v_scale: half a unit, 2^-22 / (1 - 2^-7) of the greatest; the roundings of n slots have
      independent signs (the codes' are random): eight of the greatest deviations.
    * f32 sums: four roundings a tile, and 40 for the warps' and the shares' sums and the quotients."""
    n, nh, hd = q.shape
    g = nh // b.nkv
    out, tol, plain = np.zeros((n, nh, hd)), np.zeros((n, nh, hd)), np.zeros((n, nh, hd), np.float32)
    for s in range(len(b.starts)):
        for r in range(b.row_off[s], b.row_off[s + 1]):
            path = kv.path_of(b.parent, b.row_off[s], r - b.row_off[s])
            slots = np.concatenate([np.arange(b.starts[s]), b.starts[s] + np.array(path)]).astype(np.int64)
            if not path:
                continue
            page, w = b.table[s, slots // PAGE], slots % PAGE
            tiles = int(slots.max()) // 128 + 1
            for h in range(nh):
                i = h // g
                kk, vv = (c[page, i, w].astype(np.float64) * sc[page, i, w][:, None].astype(np.float64) for c, sc in ((kc, ks), (vc, vs)))
                qq = q[r, h].astype(np.float64)
                x = kk @ qq / np.sqrt(hd)
                p = np.exp(x - x.max())
                out[r, h] = p @ vv / p.sum()
                scale = vs[page, i, w].astype(np.float64)
                e = np.maximum(np.floor(np.log2(np.maximum(scale, 1e-300))), -60)
                top = np.abs(x).max()
                rel = U * (5 * top + 3 * (1.45 * top + np.abs(e).max() + 1) + 5) + 5 * U * (tiles + 2)
                step = 2.0 ** -30 * np.abs(qq).max() / np.sqrt(hd)  # of q, as a score takes it
                pk = p * np.sqrt((kk * kk).sum(1))
                q_off = 8 * step * (np.sqrt(pk ** 2 @ vv ** 2) + np.sqrt((pk ** 2).sum()) * np.abs(out[r, h]))
                size = p @ np.abs(vv)
                most = (p * np.maximum(scale, 2.0 ** -60)).max()
                codes = np.sqrt((vc[page, i, w].astype(np.float64) ** 2).sum(0))
                unit = most * 2.0 ** -22 / (1 - 2.0 ** -7)
                tol[r, h] = (size * (2 * rel + (4 * tiles + 40) * U) + 8 * codes * unit / 2 + q_off) / p.sum()
                if f32:
                    x4 = (kk.astype(np.float32) @ q[r, h]) * np.float32(1 / np.sqrt(hd))
                    p4 = np.exp(x4 - x4.max())
                    plain[r, h] = p4 @ vv.astype(np.float32) / p4.sum()
    return (out, tol, plain) if f32 else (out, tol)


def _scaled_pool(b, rng, change):
    """Random codes, scales changed by change(scales [page][head][32], K codes, V codes), uploaded."""
    b.fill(rng)
    pool = b.pool_np().copy()
    k_at, v_at = kv.block_index(b.hd)
    kc, vc = (np.ascontiguousarray(pool.view(np.int8)[..., at]) for at in (k_at, v_at))
    sc = np.ascontiguousarray(pool[..., 32 * b.hd:]).view(np.float32).copy()
    change(sc, kc, vc)
    pool.view(np.int8)[..., k_at], pool.view(np.int8)[..., v_at] = kc, vc
    pool[..., 32 * b.hd:] = sc.view(np.uint8)
    full = np.zeros((b.n_pages, b.stride), np.uint8)
    full[:, :b.nkv * b.block] = pool.reshape(b.n_pages, -1)
    b.pool.copy_(kv.dev(full.reshape(-1)))
    return kc, vc, sc[..., :16], sc[..., 16:]


def _check_scales(b, rng, change, q=None):
    kc, vc, ks, vs = _scaled_pool(b, rng, change)
    q = rng.standard_normal((b.n, b.nh, b.hd)).astype(np.float32) if q is None else q
    out = b.attn(q).cpu().numpy().reshape(-1, b.nh, b.hd)
    want, tol, plain = _attend(q, kc, vc, ks, vs, b, True)
    size = np.sqrt((want ** 2).mean(-1, keepdims=True)) + 1e-300
    live = (want != 0).any((1, 2))
    rms = [np.sqrt((((y - want) / size)[live] ** 2).mean()) for y in (out, plain)]
    print(f"relative error, root mean square: kernel {rms[0]:.1e}, plain f32 {rms[1]:.1e}")
    bad = ~(np.abs(out - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], rms)
    assert (out[~live] == 0).all() and b.err_code() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("factor", [30.0, 300.0, 5000.0])
def test_attn_channels_of_unequal_size(native, hd, factor):
    """K's great channels stand where q is small, q's where K is: neither takes the others' accuracy."""
    rng = np.random.default_rng(55)
    b = kv.Batch(native, rng, (4, 1, hd), [900], [3])
    q = rng.standard_normal((b.n, 4, hd)).astype(np.float32)
    q[..., 5] *= np.float32(factor)
    q[..., 20] /= np.float32(factor)

    def change(sc, kc, vc):
        kc[..., 5] = 0
        kc[..., 20] = np.where(rng.random(kc[..., 20].shape) < 0.5, 127, -127)

    _check_scales(b, rng, change, q)


SPREADS = {
    "sigma 1": lambda sc, rng: np.exp(rng.standard_normal(sc.shape)) * 0.02,
    "sigma 3": lambda sc, rng: np.where(np.arange(32) < 16, sc, np.exp(3 * rng.standard_normal(sc.shape)) * 0.02),
    "tiny": lambda sc, rng: np.where(np.arange(32) < 16, sc, sc * 1e-13),
    "below 2^-60": lambda sc, rng: np.where(np.arange(32) < 16, sc, sc * 1e-22),
    "huge": lambda sc, rng: np.where(np.arange(32) < 16, sc, sc * 1e13),
    "1 in 100 is 100 times the rest": lambda sc, rng: np.where((np.arange(32) >= 16) & (rng.random(sc.shape) < 0.01), sc * 100, sc),
    "1 in 100 is 1000 times the rest": lambda sc, rng: np.where((np.arange(32) >= 16) & (rng.random(sc.shape) < 0.01), sc * 1000, sc),
}


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(12, 3, 128), (4, 1, 64), (32, 1, 64)])
@pytest.mark.parametrize("spread", SPREADS)
@pytest.mark.parametrize("peak", [1.0, 3.0])
def test_attn_spread_of_scales(native, heads, spread, peak):
    rng = np.random.default_rng(51)
    rows = [1, 9, 3]
    b = kv.Batch(native, rng, heads, [2500, 700, 90], rows, kv.random_tree(rng, rows))

    def change(sc, kc, vc):
        sc[:] = SPREADS[spread](sc, rng)

    q = (rng.standard_normal((b.n, b.nh, b.hd)) * peak).astype(np.float32)
    _check_scales(b, rng, change, q)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("factor", [1e3, 1e6, 1e9, 1e30])
def test_attn_large_scales_that_a_row_does_not_see(native, hd, factor):
    """Values of a sibling, of padding and of what lies behind the rows count nowhere, however large."""
    rng = np.random.default_rng(52)
    parent = [-1, 0, 0, -2, 1, 2, 0, 4]
    b = kv.Batch(native, rng, (8, 2, hd), [150], [8], parent)
    big = [150 + 2, 150 + 3, 150 + 9]  # row 2 (seen by rows 2 and 5), the padding row, behind the rows

    def change(sc, kc, vc):
        for slot in big:
            sc[b.table[0, slot // PAGE], :, 16 + slot % PAGE] *= factor

    _check_scales(b, rng, change)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("factor", [1e2, 1e4, 1e8])
def test_attn_large_scales_that_hardly_count(native, hd, factor):
    """A slot that is seen with next to no probability and a large V scale takes no accuracy from the others."""
    rng = np.random.default_rng(53)
    b = kv.Batch(native, rng, (4, 1, hd), [1200, 40], [1, 2])
    q = np.abs(rng.standard_normal((b.n, 4, hd))).astype(np.float32) + np.float32(0.5)

    def change(sc, kc, vc):
        for s, slot in ((0, 300), (0, 1100), (1, 7)):
            page, w = b.table[s, slot // PAGE], slot % PAGE
            kc[page, 0, w] = -np.abs(kc[page, 0, w])
            sc[page, 0, w] *= 4
            sc[page, 0, 16 + w] *= factor

    _check_scales(b, rng, change, q)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_attn_zero_value_rows(native, hd):
    """A zero V row (scale 0) takes its probability and adds nothing, the row's only slot or its greatest too."""
    rng = np.random.default_rng(54)
    b = kv.Batch(native, rng, (8, 2, hd), [600, 0, 130], [2, 1, 3])
    zero = [(0, slot) for slot in range(0, 600, 3)] + [(1, 0), (2, 5), (2, 130)]
    q = rng.standard_normal((b.n, 8, hd)).astype(np.float32)

    def change(sc, kc, vc):
        for s, slot in zero:
            page, w = b.table[s, slot // PAGE], slot % PAGE
            sc[page, :, 16 + w] = 0.0
            vc[page, :, w] = 0
        page = b.table[2, 0]  # slot 5 of sequence 2: the greatest score of head 0's rows
        kc[page, 0, 5] = np.clip(np.round(q[3:, :4].mean((0, 1)) * 200), -127, 127)

    _check_scales(b, rng, change, q)


@pytest.mark.gpu
def test_attn_scales_that_no_append_writes(native):
    """A row that sees an infinite or NaN scale, or a V scale below zero, gets NaN; the others do not."""
    rng = np.random.default_rng(56)
    b = kv.Batch(native, rng, (4, 1, 64), [140], [6], [-1, 0, 0, 0, 0, 0])
    values = [(0, np.inf), (16, np.inf), (16, -1.0), (0, np.nan)]

    def change(sc, kc, vc):
        for j, (at, x) in enumerate(values):
            slot = 141 + j
            sc[b.table[0, slot // PAGE], :, at + slot % PAGE] = x

    _scaled_pool(b, rng, change)
    out = b.attn(rng.standard_normal((6, 4, 64)).astype(np.float32)).cpu().numpy().reshape(6, -1)
    nan = np.isnan(out)
    assert nan[1:5].all() and not nan[[0, 5]].any()


# ---------------------------------------------------------------------------------------------
# codes at a rounding border
# ---------------------------------------------------------------------------------------------
def tie_rows(hd):
    """V rows whose values lie half-way between two codes of their scale: (k + 1/2) scale and the greatest,
    127 scale, with scales for which x * (1 / scale) in f64 is off the border on either side."""
    rows = []
    for scale in (49.0, 98.0 * 2.0 ** -9, 103.0, 107.0, 161.0 * 2.0 ** 4, 187.0, 65521.0, 1.0, 0.75):
        x = (np.arange(hd) % 127 + 0.5) * scale * np.where(np.arange(hd) % 3, 1, -1)
        x[hd // 2] = 127 * scale
        assert (x == x.astype(np.float32)).all()
        rows.append(x)
    return np.array(rows, np.float32)


def test_tie_rows_tell_a_product_from_a_quotient():
    x = tie_rows(128).astype(np.float64)
    scale = np.abs(x).max(-1, keepdims=True) / 127
    assert (np.round(x * (1 / scale)) != np.round(x / scale)).sum() > 50


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_codes_half_way_between_two_go_to_the_even_one(native, hd):
    x = tie_rows(hd)
    rng = np.random.default_rng(57)
    b = kv.Batch(native, rng, (1, 1, hd), [3], [len(x)])
    qkv = rng.standard_normal((len(x), 3, hd)).astype(np.float32)
    qkv[:, 2] = x
    one = np.ones(hd, np.float32)
    b.append(qkv, (one, one), kv.rope_tables(hd, 32))
    _, vc, sc = kv.unpack(b.pool_np(), hd)
    slot = 3 + np.arange(len(x))
    page, w = b.table[0, slot // PAGE], slot % PAGE
    code, scale = kv.quantised(x)
    assert np.array_equal(sc[page, 0, 1, w], scale) and np.array_equal(vc[page, 0, w], code)


# ---------------------------------------------------------------------------------------------
# logit rules: zeros of both signs
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 5003, 50304])
def test_rules_minus_zero_equals_zero(native, vocab):
    """The first of the greatest wins where -0.0 and +0.0 are the greatest: in different threads and CTAs,
    in the stream or listed, a zero that a penalty made among them."""
    rng = np.random.default_rng(58)
    pairs = [(0, vocab - 1), (3, 4), (5, 6 + vocab // 2), (vocab // 2, vocab // 2 + 9)]
    for first, second in pairs:
        for listed in ([], [first], [second], [first, second]):
            x = -1 - np.abs(rng.standard_normal((3, vocab))).astype(np.float32)
            x[0, first], x[0, second] = -0.0, 0.0
            x[1, first], x[1, second] = 0.0, -0.0
            x[2, first], x[2, second] = -1e-45, 0.0  # listed: halved to -0.0
            hists = [listed] * 3
            rep = np.full(3, 0.5, np.float32)
            out, nxt = kv._rules(native, x, [1] * 3, hists=hists, rep=rep)
            zero = np.zeros(3, np.float32)
            want, ids, _ = kv.rules_ref(x, kv.offsets([1] * 3), None, None, hists, rep, zero, zero, [[]] * 3, vocab, [None] * 3, exact=False)
            assert np.array_equal(out, want) and np.array_equal(nxt, ids), (first, second, listed)
            assert nxt.tolist()[:2] == [first, first]


# ---------------------------------------------------------------------------------------------
# long paths given by parents
# ---------------------------------------------------------------------------------------------
def deep_tree(rng, n, kind):
    if kind == "chain":
        return [j - 1 for j in range(n)]
    if kind == "two chains":  # every other row
        return [j - 2 if j > 1 else -1 for j in range(n)]
    if kind == "chain and trees":  # a prompt, drafts behind it
        return [j - 1 for j in range(n - 40)] + [int(rng.integers(n - 41, n - 40 + j)) for j in range(40)]
    p = []  # runs with jumps, padding rows, roots
    for j in range(n):
        x = rng.random()
        p.append(j - 1 if x < 0.95 else -2 if x < 0.96 else int(rng.integers(max(-1, j - 70), j)) if j else -1)
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(12, 3, 128), (4, 4, 64), (32, 1, 64)])
@pytest.mark.parametrize("kind", ["chain", "two chains", "chain and trees", "runs"])
def test_long_paths(native, heads, kind):
    """Appended and attended: positions by the number of ancestors, visibility by the path, over many tiles."""
    nh, nkv, hd = heads
    rng = np.random.default_rng(61)
    starts, rows = [77, 0, 300], [333, 150, 1]
    parent = sum((deep_tree(rng, n, kind) if n > 100 else [-1] for n in rows), [])
    b = kv.Batch(native, rng, heads, starts, rows, parent)
    qkv = rng.standard_normal((b.n, nh + 2 * nkv, hd)).astype(np.float32)
    one, rope = np.ones(hd, np.float32), kv.rope_tables(hd, 512)
    q = b.append(qkv, (one, one), rope).cpu().numpy().reshape(-1, nh, hd)
    depth = np.array([len(kv.path_of(b.parent, b.row_off[s], j)) - 1 for s in range(3) for j in range(rows[s])])
    live = depth >= 0
    pos = (b.starts[np.repeat(np.arange(3), rows)] + depth)[live]
    want, amp = kv.norm_rope(qkv[live, :nh], one, EPS, rope[0][pos][:, None], rope[1][pos][:, None])
    assert (np.abs(q[live] - want) <= 24 * U * amp + 1e-30).all() and (q[~live] == 0).all()
    kv._check_attn(b, rng)


@pytest.mark.gpu
def test_a_chain_of_parents_is_the_chain(native):
    """The same bits as parent = NULL, and in the same order of time."""
    import torch

    rng = np.random.default_rng(62)
    heads, n = (8, 2, 64), 2500
    q = kv.dev(rng.standard_normal((n, 8, 64)).astype(np.float32))
    qkv = rng.standard_normal((n, 12, 64)).astype(np.float32)
    one, rope = np.ones(64, np.float32), kv.rope_tables(64, 2600)
    got, ms = [], []
    for parent in (None, [j - 1 for j in range(n)]):
        b = kv.Batch(native, np.random.default_rng(63), heads, [50], [n], parent)
        b.fill(np.random.default_rng(64))
        qs = b.append(qkv, (one, one), rope)
        out = b.attn(q).clone()
        scratch, best = b.scratch, 1e9
        for _ in range(3):
            a, e = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            b.attn(q, None, scratch, out)
            e.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(e))
        got.append((qs, b.pool.clone(), out.clone()))
        ms.append(best)
        assert b.err_code() == 0
    for x, y in zip(*got):
        assert torch.equal(x, y)
    print(f"chain {ms[0]:.3f} ms, by parents {ms[1]:.3f} ms")
    # a row block walks its rows' paths once, at most 2500 rows at 16 a load (157 loads), beside up to 20 tiles
    # of a dozen dependent steps each; a walk of every path for every tile took 46 times the chain's time
    assert ms[1] <= 8 * ms[0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "two chains", "runs"])
def test_rules_long_paths(native, kind):
    rng = np.random.default_rng(65)
    n, v = 700, 300
    parent = deep_tree(rng, n, kind)
    logits = rng.standard_normal((n, v)).astype(np.float32)
    token = rng.integers(0, v, n).tolist()
    rep, freq, zero = np.array([1.1], np.float32), np.array([0.25], np.float32), np.zeros(1, np.float32)
    out, nxt = kv._rules(native, logits, [n], parent, token, [[3]], rep, freq)
    want, ids, _ = kv.rules_ref(logits, kv.offsets([n]), np.array(parent), token, [[3]], rep, freq, zero, [[]], v, [None] * n, exact=False)
    live = np.array(parent) != -2
    assert np.array_equal(out[live], want[live]) and np.array_equal(nxt, ids)


@pytest.mark.gpu
def test_rules_list_offsets_out_of_order(native):
    """Offsets below zero and descending ones: no entries for that sequence, reported; the others as ever."""
    import torch

    rng = np.random.default_rng(59)
    v, n = 500, 4
    x = rng.standard_normal((n, v)).astype(np.float32)
    hist, bias_id = rng.integers(0, v, 30), rng.integers(0, v, 30)
    t = {k: kv.dev(a) for k, a in (("logits", x), ("hist", hist.astype(np.int32)), ("bias_id", bias_id.astype(np.int32)),
                                   ("bias", np.ones(30, np.float32)), ("rep_penalty", np.full(n, 1.5, np.float32)))}
    row_off, err = kv.dev(kv.offsets([1] * n)), torch.zeros(1, dtype=torch.int32, device="cuda")
    r = native.Rows(n_seqs=n, n_rows=n, max_rows=1, row_off=kv.ptr(row_off), err=kv.ptr(err))
    good, cases = [0, 10, 10, 20, 30], ([0, 10, 10, 20, 30], [-5, 10, 10, 20, 30], [0, 10, 20, 15, 30], [-9, -4, 10, 20, 30])
    for which in ("hist_off", "bias_off"):
        for off in cases:
            used = {k: kv.dev(np.array(off if k == which else good, np.int32)) for k in ("hist_off", "bias_off")}
            out = torch.zeros((n, v), device="cuda")
            err.zero_()
            a = native.LogitsRules(vocab=v, out=kv.ptr(out), **{k: kv.ptr(b) for k, b in {**t, **used}.items()})
            native.check(native.lib().hg_op_logits_rules(C.byref(r), C.byref(a), None))
            lists = [[slice(o[s], o[s + 1]) if 0 <= o[s] <= o[s + 1] else slice(0, 0) for s in range(n)]
                     for o in ((off, good) if which == "hist_off" else (good, off))]
            hists = [hist[c].tolist() for c in lists[0]]
            biases = [[(int(i), 1.0) for i in bias_id[c]] for c in lists[1]]
            zero = np.zeros(n, np.float32)
            want, _, _ = kv.rules_ref(x, kv.offsets([1] * n), None, None, hists, np.full(n, 1.5, np.float32), zero, zero, biases, v, [None] * n, exact=False)
            assert np.array_equal(out.cpu().numpy(), want)
            assert int(err.cpu()[0]) == (0 if off == good else INVALID)
