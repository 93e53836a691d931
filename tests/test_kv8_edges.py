"""Edges of the 8-bit KV cache, the tree attention and the logit rules, against plain 64-bit forms:
pages of mostly padding rows, scales of any spread, ties, chains given by their parents.

Tolerances count roundings: u = 2^-24 is half a step of f32 (relative).
"""
import ctypes as C

import numpy as np
import pytest

import test_kv8 as kv

U, PAGE, INVALID, CONTEXT = kv.U, kv.PAGE, kv.INVALID, kv.CONTEXT


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
    qr, amp = kv.norm_rope(qkv[live, :nh], gains[0], 1e-5, cos, sin)
    kr, _ = kv.norm_rope(qkv[live, nh:nh + nkv], gains[1], 1e-5, cos, sin)
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
