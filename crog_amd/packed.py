"""Plans of a transformer block on packed rows: what a program builds once for a batch (PackedRows) or once for a model (RotaryAxes) and hands to
crog_amd.functional.packed_attention / rotary.

A packed tensor holds the rows of all sequences of a batch one behind the other, [rows, heads, dim], with no padding between them: captions of
different lengths, images of different sizes, documents.  Nothing here launches a kernel; a plan is two or three small tables on the device.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence

import numpy as np
import torch

TILE = 128      # rows (query rows x heads of a group) or keys of a block of csrc/packed_attn.hip
# Key splits of the forward pass: with fewer blocks than this, a long key axis is cut into pieces so that every CU has work (256 CUs, two blocks
# each); a piece is at least SPLIT_MIN keys.
FILL_BLOCKS = 512
SPLIT_MIN = 256


def _lengths(name: str, lengths: Sequence[int]) -> np.ndarray:
    if isinstance(lengths, torch.Tensor):
        if lengths.is_cuda:
            raise TypeError(f"PackedRows: {name} are host numbers (a list, or a CPU tensor): the launch grid depends on them")
        lengths = lengths.tolist()
    out = [operator.index(n) for n in lengths]
    if any(n < 0 for n in out):
        raise ValueError(f"PackedRows: {name} must not be negative")
    if sum(out) > 0x7fffff00:
        raise ValueError(f"PackedRows: {sum(out)} rows are too many")
    return np.asarray(out, dtype=np.int64)


def _tiles(rows: np.ndarray, cost) -> np.ndarray:
    """[(sequence, tile)] of all 128-row tiles, the costliest first (a late long one would leave the device waiting for a single block)."""
    n = (rows + TILE - 1) // TILE
    seq = np.repeat(np.arange(len(rows)), n)
    tile = np.arange(len(seq)) - np.repeat(np.cumsum(n) - n, n)
    order = np.argsort(-cost(seq, tile), kind="stable")
    return np.stack([seq[order], tile[order]], 1)


class PackedRows:
    """The sequences of a packed batch, for attention.

    lengths: query rows of each sequence; key_lengths: its key rows where they are others (cross-attention, or new tokens over what a
    sequence has behind it), by default the same rows.  group: query heads per key head.  causal: query i of a sequence with Lq queries and
    Lk keys sees keys j <= i + Lk - Lq, i.e. the last query sees them all; a query that sees none gets zeros.  A length may be zero.
    device: where the tensors will live.  One plan serves every layer of a batch."""

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
            last = np.minimum(t * TILE + TILE - 1, lq[s] * g - 1) // g
            return np.clip(last + 1 + lk[s] - lq[s], 0, lk[s]) if c else lk[s]

        def key_cost(s, t):      # rows that see the tile's first key
            return (lq[s] - np.clip(t * TILE - (lk[s] - lq[s]), 0, lq[s])) * g if c else lq[s] * g

        rt, kt = _tiles(lq * g, row_cost), _tiles(lk, key_cost)
        self.n_row_tiles, self.n_key_tiles = len(rt), len(kt)
        zero = np.zeros(1, dtype=np.int64)
        parts = [np.concatenate([zero, np.cumsum(lq)]), np.concatenate([zero, np.cumsum(lk)]), rt.reshape(-1), kt.reshape(-1)]
        table = torch.from_numpy(np.concatenate(parts).astype(np.int32))
        self._table = table.to(device)      # one copy; the tables lie in it one behind the other
        self.device = self._table.device
        at, addr = 0, []
        for p in parts:
            addr.append(self._table.data_ptr() + 4 * at)
            at += len(p)
        self.cu_q_ptr, self.cu_k_ptr, self.row_tiles_ptr, self.key_tiles_ptr = addr

    def splits(self, kv_heads: int):
        """(pieces, keys of a piece) of the forward pass's key axis.  A single query over 8192 keys of 8 heads would be 8 blocks on 256 CUs;
        in pieces of 256 keys it is 256.  Enough blocks, or short keys: one piece, no second launch."""
        blocks = max(self.n_row_tiles * kv_heads, 1)
        n = min(-(-FILL_BLOCKS // blocks), -(-self.max_k // SPLIT_MIN))
        if n <= 1:
            return 1, 0
        piece = -(-self.max_k // n)
        piece = -(-piece // 64) * 64
        return -(-self.max_k // piece), piece


class RotaryAxes:
    """Rotary positions of heads whose first 2 * sum(pairs) columns are pairs.

    pairs: how many pairs turn with each axis of the positions - (32,) for text, (16, 24, 24) for time, height and width.  Pair i of an axis
    with n pairs turns by position * theta^(-i / n).  interleaved: a pair is two neighbouring columns (2 i, 2 i + 1); otherwise column i and
    column sum(pairs) + i.  One plan serves a model."""

    def __init__(self, pairs: Sequence[int], *, theta: float = 10000.0, interleaved: bool = False, device="cuda"):
        sizes = [operator.index(n) for n in pairs]
        if not sizes or any(n < 1 for n in sizes):
            raise ValueError("RotaryAxes: every axis needs at least one pair")
        if sum(sizes) > 128:
            raise ValueError(f"RotaryAxes: {sum(sizes)} pairs, at most 128 (a head of 256 columns)")
        if not (theta > 0):
            raise ValueError("RotaryAxes: theta must be positive")
        self.axes, self.pairs, self.interleaved, self.theta = len(sizes), sum(sizes), bool(interleaved), float(theta)
        revs = np.concatenate([float(theta) ** (-np.arange(n, dtype=np.float64) / n) for n in sizes]) / (2 * np.pi)
        axis = np.repeat(np.arange(len(sizes), dtype=np.int64), sizes).astype(np.int32)
        raw = np.concatenate([revs.view(np.uint8), axis.view(np.uint8)])      # (the doubles first: aligned)
        self._table = torch.from_numpy(raw).to(device)
        self.device = self._table.device
        self.revs_ptr, self.axis_ptr = self._table.data_ptr(), self._table.data_ptr() + 8 * self.pairs
