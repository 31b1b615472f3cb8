"""Packed attention, rotary positions and the gated norm without a GPU: the plans' tables against a plain count, and every refusal."""
import numpy as np
import pytest
import torch

from crog_amd import _lib
from crog_amd import functional as Fn
from crog_amd.packed import KEY_TILE, OPERANDS, SHARE_MIN, SLOTS, SPLIT_MIN, TILE, PackedRows, RotaryAxes


def tables(p):
    t = p._table.numpy()
    n = p.seqs + 1
    cu_q, cu_k, rest = t[:n], t[n:2 * n], t[2 * n:]
    return cu_q, cu_k, rest[:2 * p.n_row_tiles].reshape(-1, 2), rest[2 * p.n_row_tiles:2 * (p.n_row_tiles + p.n_key_tiles)].reshape(-1, 2)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("group", [1, 3])
def test_plan_covers_every_row_and_key_once(causal, group):
    lq, lk = [5, 0, 1, 300, 43], [5, 7, 0, 129, 4000]
    p = PackedRows(lq, lk, group=group, causal=causal, device="cpu")
    cu_q, cu_k, rt, kt = tables(p)
    assert cu_q.tolist() == [0] + np.cumsum(lq).tolist() and cu_k.tolist() == [0] + np.cumsum(lk).tolist()
    assert (p.rows_q, p.rows_k, p.max_k) == (sum(lq), sum(lk), 4000)
    want_r = {(s, t) for s, n in enumerate(lq) for t in range(-(-n * group // TILE))}
    want_k = {(s, t) for s, n in enumerate(lk) for t in range(-(-n // KEY_TILE))}
    assert len(rt) == len(want_r) and {tuple(r) for r in rt.tolist()} == want_r
    assert len(kt) == len(want_k) and {tuple(r) for r in kt.tolist()} == want_k
    # the costliest block first: the keys a row tile sees do not grow along the list
    cost = [min(lk[s], max(0, (min(t * TILE + TILE, lq[s] * group) - 1) // group + 1 + lk[s] - lq[s])) if causal else lk[s] for s, t in rt.tolist()]
    assert cost == sorted(cost, reverse=True)
    assert p.cu_k_ptr - p.cu_q_ptr == 4 * len(cu_q) and p.key_tiles_ptr - p.row_tiles_ptr == 8 * len(rt)


def test_plan_of_nothing():
    for lens in ([], [0], [0, 0]):
        p = PackedRows(lens, device="cpu")
        assert (p.rows_q, p.n_row_tiles, p.n_key_tiles) == (0, 0, 0) and p.splits(8, 2)[0] == 1 and p.share(8, 64, 2) == (0, 0)


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("seqs,keys,kv", [(1, 8192, 1), (1, 8192, 8), (16, 777, 8), (3, 65, 2), (600, 5000, 1), (1, 100000, 1)])
def test_splits_cover_the_keys(seqs, keys, kv, size):
    p = PackedRows([1] * seqs, [keys] * seqs, device="cpu")
    n, piece = p.splits(kv, size)
    if n == 1:
        assert seqs * kv >= 512 or keys < 2 * SPLIT_MIN[size]
    else:
        assert piece % 64 == 0 and n * piece >= keys > (n - 1) * piece and piece >= SPLIT_MIN[size] // 2


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("lq,lk,group,kv,causal", [([5000, 300], None, 4, 4, True), ([4096], None, 8, 1, True), ([16384], [20], 1, 8, False), ([20] * 32, None, 1, 8, True),
                                                   ([3000], [100], 2, 1, True)])
def test_shares_cover_the_steps(lq, lk, group, kv, causal, size):
    p = PackedRows(lq, lk, group=group, causal=causal, device="cpu")
    # a tile's steps - 32 queries of one head - and OPERANDS units more, in the list's order
    pairs, sums = tables(p)[3], p._table.numpy()[-p.n_key_tiles - 1:]
    assert p.key_units_ptr == p.key_tiles_ptr + 8 * p.n_key_tiles
    lks = lk or lq
    want = []
    for s, t in pairs.tolist():
        first = min(max(t * KEY_TILE - (lks[s] - lq[s]), 0), lq[s]) if causal else 0
        want.append((-(-lq[s] // 32) - first // 32) * group + OPERANDS)
    assert sums[0] == 0 and np.diff(sums).tolist() == want and (p.key_units, p.key_most) == (sum(want), max(want))
    for dim in (32, 64, 128):
        share, blocks = p.share(kv, dim, size)
        if share:
            assert share >= SHARE_MIN[size] and share * blocks >= p.key_units * kv > share * (blocks - 1)
            assert blocks <= SLOTS[dim // 32]
        else:
            assert blocks == p.n_key_tiles * kv


@pytest.mark.parametrize("make,error", [
    (lambda: PackedRows([3, -1], device="cpu"), ValueError),
    (lambda: PackedRows([3], [3, 4], device="cpu"), ValueError),
    (lambda: PackedRows([3], group=0, device="cpu"), ValueError),
    (lambda: PackedRows([2.5], device="cpu"), TypeError),
    (lambda: PackedRows([1 << 31], device="cpu"), ValueError),
    (lambda: PackedRows([1 << 30], group=4, device="cpu"), ValueError),
    (lambda: RotaryAxes([], device="cpu"), ValueError),
    (lambda: RotaryAxes([4, 0], device="cpu"), ValueError),
    (lambda: RotaryAxes([100, 29], device="cpu"), ValueError),
    (lambda: RotaryAxes([4], theta=0, device="cpu"), ValueError),
])
def test_plans_refuse(make, error):
    with pytest.raises(error):
        make()


def attn(q=(6, 4, 64), k=(6, 2, 64), v=None, dtype=torch.bfloat16, k_dtype=None, lens=(2, 4), group=2, scale=None):
    q, k_, v = torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=k_dtype or dtype), torch.zeros(v or k, dtype=dtype)
    return Fn.packed_attention(q, k_, v, PackedRows(lens, group=group, device="cpu"), scale)


@pytest.mark.parametrize("kw,error", [
    (dict(q=(6, 256)), ValueError),
    (dict(dtype=torch.float16), TypeError),
    (dict(k_dtype=torch.float32), TypeError),
    (dict(q=(6, 3, 64)), ValueError),
    (dict(group=4), ValueError),
    (dict(v=(6, 2, 32)), ValueError),
    (dict(q=(6, 4, 60), k=(6, 2, 60)), ValueError),
    (dict(q=(6, 4, 136), k=(6, 2, 136)), ValueError),
    (dict(q=(5, 4, 64)), ValueError),
    (dict(k=(5, 2, 64)), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(), RuntimeError),      # (all well: but there is no CPU path)
])
def test_packed_attention_refuses(kw, error):
    with pytest.raises(error):
        attn(**kw)


def rot(q=(6, 4, 64), k=(6, 2, 64), pos=(6, 2), axes=(8, 8), dtype=torch.bfloat16, pos_dtype=torch.int32):
    return Fn.rotary(torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=dtype), torch.zeros(pos, dtype=pos_dtype), RotaryAxes(axes, device="cpu"))


@pytest.mark.parametrize("kw,error", [
    (dict(q=(6, 64)), ValueError), (dict(k=(5, 2, 64)), ValueError), (dict(k=(6, 2, 32)), ValueError), (dict(dtype=torch.float16), TypeError),
    (dict(pos_dtype=torch.float32), TypeError), (dict(pos=(6, 3)), ValueError), (dict(pos=(5, 2)), ValueError), (dict(axes=(30, 8)), ValueError),
    (dict(), RuntimeError),
])
def test_rotary_refuses(kw, error):
    with pytest.raises(error):
        rot(**kw)


class Ref:
    """Stands for a WRef of n values."""

    def __init__(self, n):
        self.rows, self.cols, self.P, self.param = n, 1, torch.zeros(n), torch.nn.Parameter(torch.zeros(n))


@pytest.mark.parametrize("kw,error", [
    (dict(y=torch.zeros(4, 9)), ValueError),
    (dict(y=torch.zeros(4, 8, dtype=torch.bfloat16)), ValueError),
    (dict(x=torch.zeros(4, 8, dtype=torch.float16), y=torch.zeros(4, 8, dtype=torch.float16)), TypeError),
    (dict(x=torch.zeros(1, 8200), y=torch.zeros(1, 8200)), ValueError),
    (dict(gate=Ref(9)), ValueError),
    (dict(pre=(Ref(8), Ref(7))), ValueError),
    (dict(pre=(Ref(8),)), ValueError),
    (dict(post=(Ref(8), Ref(8)), rms=True), ValueError),
    (dict(eps=-1e-5), ValueError),
    (dict(res_scale=float("inf")), ValueError),
    (dict(), RuntimeError),
])
def test_gated_norm_refuses(kw, error):
    args = dict(x=torch.zeros(4, 8), y=torch.zeros(4, 8))
    args.update(kw)
    with pytest.raises(error):
        Fn.gated_norm(args.pop("x"), args.pop("y"), **args)


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    buf = torch.zeros(4096)
    p = (buf.data_ptr() + 15) // 16 * 16

    def fwd(dtype=1, head_dim=64, ld=64, hs=64, ptr=p, cu=p, splits=1, piece=0, ws=None, rows=8, group=1):
        return lib.crog_packed_attn_fwd(dtype, ptr, ld, hs, ptr, ld, hs, ptr, ld, hs, ptr, ld, hs, None, cu, cu, cu, 1, 1, rows, 8, 1, group, head_dim, 1.0, 0,
                                        splits, piece, ws, None)
    bad = [dict(dtype=3), dict(head_dim=60), dict(head_dim=136), dict(head_dim=0), dict(ld=60), dict(hs=4), dict(ptr=p + 2), dict(ptr=None), dict(cu=None),
           dict(splits=2), dict(splits=2, piece=100, ws=p), dict(splits=0), dict(rows=0), dict(rows=1 << 30, group=8)]
    for kw in bad:
        assert fwd(**kw) == -1, kw
        assert b"packed_attn_fwd" in lib.crog_last_error()
    args = [1] + [p, 64, 64] * 5 + [p, p] + [p, 64, 64] * 3 + [p, p, p, 1, p, 1, 1, 8, 8, 1, 1, 64, 1.0, 0, 1, 0, None, 0, 0, None, None]
    for at, v in ((0, 2), (1, None), (13, p + 8), (16, None), (17, None), (20, 4), (27, None), (38, 60), (41, 2), (41, 0), (45, -1), (45, 5), (2, 1 << 40), (5, 1 << 30)):
        assert lib.crog_packed_attn_bwd(*args[:at], v, *args[at + 1:]) == -1, at
    r = [1, p, 64, 64, p, 64, 64, p, 64, 64, p, 64, 64, p, 1, 4, p, p, 8, 1, 1, 64, 32, 1, 0, 0, None]
    for at, v in ((0, 2), (1, None), (13, None), (14, 0), (15, 2), (16, None), (18, -1), (22, 33), (22, 0), (23, 0)):
        assert lib.crog_rotary(*r[:at], v, *r[at + 1:]) == -1, at
    g = [1, p, 64, p, 64, None, None, None, None, None, 0, 1, 0, 1.0, 1e-5, 4, 64, p, 64, p, 64, None, None]
    for at, v in ((0, 2), (1, None), (2, 63), (15, -1), (16, 0), (16, 8193), (17, None), (19, None), (21, p + 4)):
        assert lib.crog_gated_norm_fwd(*g[:at], v, *g[at + 1:]) == -1, at
    b = [1, p, 64, p, 64, p, 64, p, 64, None, None, None, None, 0, 1, 0, 1.0, 4, 64, p, p, 64, p, 64, None, None]
    for at, v in ((0, 2), (1, None), (17, -1), (18, 8193), (19, None), (19, p + 4), (21, 63)):
        assert lib.crog_gated_norm_bwd(*b[:at], v, *b[at + 1:]) == -1, at
    c = [p, 4, 64, None, None, None, 0, p, None, None, None, None, None]
    for at, v in ((0, None), (1, -1), (2, 0), (2, 8193)):
        assert lib.crog_gated_norm_sums(*c[:at], v, *c[at + 1:]) == -1, at
    assert lib.crog_gated_norm_slab_floats(0, 64) == 0 and lib.crog_gated_norm_slab_floats(10 ** 6, 64) == 512 * 4 * 64
