"""Plans of a transformer block on packed rows: what a program builds once for a batch (PackedRows) or once for a model (RotaryAxes) and hands to
crog_amd.functional.packed_attention / rotary.

A packed tensor holds the rows of all sequences of a batch one behind the other, [rows, heads, dim], with no padding between them: captions of
different lengths, images of different sizes, documents.  Nothing here launches a kernel; a plan is two or three small tables on the device.
A plan is made outside a captured graph, and outlives every graph that was captured with it (its replays read the tables; eager launches keep them
themselves until they are through).
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence

import numpy as np
import torch

TILE = 128      # rows (query rows x heads of a group) of a forward / dQ block of csrc/packed_attn.hip
KEY_TILE = 128  # keys of a dK / dV block
# Long chains of work are cut where there are too few blocks to fill the device (256 CUs, two blocks each) or where it would wait for the longest: the
# keys that a block of the forward or dQ pass walks over in equal pieces, the steps of the dK / dV pass in equal shares of all of them.  The pieces meet
# in a second launch, which costs 4 to 25 us, so a piece has at least SPLIT_MIN keys or SHARE_MIN units (by the bytes of an element; fp32 products take
# eight times as long).  100 keys over 4000 queries of 8 heads, bf16: dK / dV 27 us uncut, 16 + 4 cut; one token over 8192 keys, 8 key heads: 85 us in
# one piece, 11 + 6 in 32; two, four and eight times as many pieces were no faster or slower.
FILL_BLOCKS = 512
SPLIT_MIN = {2: 256, 4: 128}
# dK / dV: blocks that the device holds, by head_dim / 32 (bf16; fp32: one a CU); queries of a step; units of a tile's operands and results; units of a
# share at least.
SLOTS, SLOTS_FP32 = {1: 1024, 2: 768, 3: 512, 4: 512}, 256
STEP, OPERANDS, SHARE_MIN = 32, 2, {2: 8, 4: 4}


def _stream_of(table: torch.Tensor):
    """Raw handle of the stream whose allocations the table belongs to."""
    return torch.cuda.current_stream(table.device).cuda_stream if table.is_cuda else None


def _lengths(name: str, lengths: Sequence[int]) -> np.ndarray:
    if isinstance(lengths, torch.Tensor):
        if lengths.is_cuda:
            raise TypeError(f"PackedRows: {name} are host numbers (a list, or a CPU tensor): the launch grid depends on them")
        lengths = lengths.tolist()
    out = [operator.index(n) for n in lengths]
    if min(out, default=0) < 0:
        raise ValueError(f"PackedRows: {name} must not be negative")
    if sum(out) > 0x7fffff00:
        raise ValueError(f"PackedRows: {sum(out)} rows are too many")
    return np.asarray(out, dtype=np.int64)


def _tiles(rows: np.ndarray, size: int, cost, together: bool = False):
    """Sequences, numbers and costs of all tiles of `size` rows, the costliest first (a late long one would leave the device waiting for a
    single block); together: a sequence's tiles one behind the other, the sequence with the costliest first."""
    n = (rows + size - 1) // size
    ends = n.cumsum()
    seq = np.arange(len(rows)).repeat(n)
    tile = np.arange(len(seq)) - (ends - n).repeat(n)
    c = cost(seq, tile)
    order = (-(cost(seq, 0) if together else c)).argsort(kind="stable")
    return seq[order], tile[order], c[order]


class PackedRows:
    """The sequences of a packed batch, for attention.

    lengths: query rows of each sequence; key_lengths: its key rows where they are others (cross-attention, or new tokens over what a
    sequence has behind it), by default the same rows.  group: query heads per key head.  causal: query i of a sequence with Lq queries and
    Lk keys sees keys j <= i + Lk - Lq, i.e. the last query sees them all; a query that sees none gets zeros.  A length may be zero.
    device: where the tensors will live.  One plan serves every layer of a batch; it has to outlive the graphs captured with it."""

    def __init__(self, lengths: Sequence[int], key_lengths: Optional[Sequence[int]] = None, *, group: int = 1, causal: bool = False, device="cuda"):
        lq = _lengths("lengths", lengths)
        lk = lq if key_lengths is None else _lengths("key_lengths", key_lengths)
        if len(lk) != len(lq):
            raise ValueError(f"PackedRows: {len(lq)} lengths and {len(lk)} key_lengths")
        self.group = operator.index(group)
        if self.group < 1:
            raise ValueError("PackedRows: group must be at least 1")
        self.causal = bool(causal)
        self.seqs = len(lq)
        self.rows_q, self.rows_k = int(lq.sum()), int(lk.sum())
        self.max_k = int(lk.max()) if self.seqs else 0
        if self.rows_q * self.group > 0x7fffff00:
            raise ValueError("PackedRows: too many rows for a group")
        g, c = self.group, self.causal

        def row_cost(s, t):      # keys of the tile's last row
            if not c:
                return lk[s]
            last = np.minimum(t * TILE + TILE - 1, lq[s] * g - 1) // g
            return np.minimum(np.maximum(last + 1 + lk[s] - lq[s], 0), lk[s])

        def key_cost(s, t):      # steps of the tile (32 queries of one head each, from the block that first sees its first key to the last), and its operands
            lqs = lq[s]
            steps = (lqs + STEP - 1) // STEP
            if c:
                steps = steps - np.minimum(np.maximum(t * KEY_TILE - (lk[s] - lqs), 0), lqs) // STEP
            return steps * g + OPERANDS

        rs, rt, _ = _tiles(lq * g, TILE, row_cost)
        ks, kt, kc = _tiles(lk, KEY_TILE, key_cost, together=True)
        self.n_row_tiles, self.n_key_tiles = nr, nk = len(rt), len(kt)
        units = kc.cumsum()
        self.key_units, self.key_most = (int(units[-1]), int(kc.max())) if nk else (0, 0)
        # the tables one behind the other, in one copy: the sequences' ends on both sides, (sequence, tile) of the row tiles and the key tiles, the
        # units before each key tile and of all
        n = self.seqs + 1
        at = np.array([0, n, 2 * n, 2 * (n + nr), 2 * (n + nr + nk)])
        table = np.zeros(at[-1] + nk + 1, dtype=np.int32)
        table[1:n], table[n + 1:2 * n] = lq.cumsum(), lk.cumsum()
        table[at[2]:at[3]:2], table[at[2] + 1:at[3]:2], table[at[3]:at[4]:2], table[at[3] + 1:at[4]:2] = rs, rt, ks, kt
        if self.key_units < 1 << 31:
            table[at[4] + 1:] = units
        self._table = torch.from_numpy(table).to(device)
        self.device, self.made_on = self._table.device, _stream_of(self._table)
        self.cu_q_ptr, self.cu_k_ptr, self.row_tiles_ptr, self.key_tiles_ptr, self.key_units_ptr = (self._table.data_ptr() + 4 * at).tolist()

    def splits(self, kv_heads: int, size: int):
        """(pieces, keys of a piece) of the forward and dQ passes' key axis; size: bytes of an element.  A single query over 8192 keys of 8 heads
        would be 8 blocks on 256 CUs; in pieces of 256 keys it is 256.  Enough blocks, or short keys: one piece, no second launch.  All
        sequences are cut by the longest one's keys, and a tile counts as a block whatever its keys: one long sequence among many short ones is
        walked by its own blocks alone."""
        blocks = max(self.n_row_tiles * kv_heads, 1)
        n = min(-(-FILL_BLOCKS // blocks), self.max_k // SPLIT_MIN[size])
        if n <= 1:
            return 1, 0
        piece = -(-self.max_k // n)
        piece = -(-piece // 64) * 64
        return -(-self.max_k // piece), piece

    def share(self, kv_heads: int, dim: int, size: int):
        """(units of a block, blocks) of the dK / dV pass: a block walks over every query that sees its keys - 16384 queries of 8 heads are 4096
        steps -, so the steps of all tiles are dealt out evenly where the device would wait for the longest.  (0, blocks): a block a tile."""
        slots = SLOTS[-(-dim // 32)] if size == 2 else SLOTS_FP32
        n, work = self.n_key_tiles * kv_heads, self.key_units * kv_heads
        even = max(-(-work // slots), SHARE_MIN[size])
        # uncut: as long as the longest tile; with more tiles than places, half of it beyond an even share, or so many rounds of them
        whole = max(self.key_most, min(even + self.key_most // 2, -(-n // slots) * self.key_most))
        if whole <= even + SHARE_MIN[size] or self.key_units >= 1 << 31:
            return 0, n
        return even, -(-work // even)


class RotaryAxes:
    """Rotary positions of heads whose first 2 * sum(pairs) columns are pairs.

    pairs: how many pairs turn with each axis of the positions - (32,) for text, (16, 24, 24) for time, height and width.  Pair i of an axis
    with n pairs turns by position * theta^(-i / n).  interleaved: a pair is two neighbouring columns (2 i, 2 i + 1); otherwise column i and
    column sum(pairs) + i.  One plan serves a model; it has to outlive the graphs captured with it."""

    def __init__(self, pairs: Sequence[int], *, theta: float = 10000.0, interleaved: bool = False, device="cuda"):
        sizes = [operator.index(n) for n in pairs]
        if not sizes or any(n < 1 for n in sizes):
            raise ValueError("RotaryAxes: every axis needs at least one pair")
        if sum(sizes) > 128:
            raise ValueError(f"RotaryAxes: {sum(sizes)} pairs, at most 128 (a head of 256 columns)")
        if not (theta > 0):
            raise ValueError("RotaryAxes: theta must be positive")
        self.axes, self.pairs, self.interleaved, self.theta = len(sizes), sum(sizes), bool(interleaved), float(theta)
        with np.errstate(over="ignore"):
            revs = np.concatenate([float(theta) ** (-np.arange(n, dtype=np.float64) / n) for n in sizes]) / (2 * np.pi)
        if not np.isfinite(revs).all():
            raise ValueError(f"RotaryAxes: theta {theta} gives angles beyond 64 bits")
        axis = np.repeat(np.arange(len(sizes), dtype=np.int64), sizes).astype(np.int32)
        raw = np.concatenate([revs.view(np.uint8), axis.view(np.uint8)])      # (the doubles first: aligned)
        self._table = torch.from_numpy(raw).to(device)
        self.device, self.made_on = self._table.device, _stream_of(self._table)
        self.revs_ptr, self.axis_ptr = self._table.data_ptr(), self._table.data_ptr() + 8 * self.pairs
