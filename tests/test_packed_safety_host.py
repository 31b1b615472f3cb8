"""What keeps the packed operators inside their memory and their promises, without a GPU: the shares of the dK / dV pass compiled for the host."""
import contextlib
import os
import random
import re
import subprocess
import types

import pytest
import torch

from crog_amd import _lib
from crog_amd.packed import KEY_TILE, PackedRows

WALK = r'''
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "packed_share.h"
// the walk of packed_bwd_dkdv_kernel over the shares and of packed_meet_kernel over the tiles: prints what every block and tile does
int main() {
  int n, total, kv, share, blocks;
  while (scanf("%d %d %d %d %d", &n, &total, &kv, &share, &blocks) == 5) {
    std::vector<int> units(n + 1), steps(n);
    for (int& u : units) if (scanf("%d", &u) != 1) return 1;
    for (int& s : steps) if (scanf("%d", &s) != 1) return 1;
    printf("case\n");
    const int grid = (blocks + 7) / 8 * 8;
    for (int b = 0; b < grid; b++) {
      const Place p = place_of(units.data(), n, total, kv, share, b);
      if (p.pos >= p.end) continue;
      long pos = p.pos;
      int kh = p.kh, ti = p.ti, rounds = 0;
      while (pos < p.end) {
        if (kh < 0 || kh >= kv || ti < 0 || ti >= n) { printf("outside\n"); return 0; }
        const Segment s = segment_of(pos, p.end, b, (long)kh * units[n] + units[ti], units_of(units.data(), ti), steps[ti]);
        printf("walk %d %d %d %d %d %d\n", b, kh, ti, s.first, s.last, s.slot);
        if (s.next <= pos || ++rounds > share) { printf("endless\n"); return 0; }
        pos = s.next;
        if (++ti == n) { ti = 0; kh = kh + 1 < kv ? kh + 1 : kv - 1; }
      }
    }
    for (int kh = 0; kh < kv; kh++)
      for (int t = 0; t < n; t++) {
        const Meeting m = meeting_of((long)kh * total + units[t], units_of(units.data(), t), share, blocks);
        if (m.first < m.last) printf("meet %d %d %d %d\n", kh, t, m.first, m.last);
      }
  }
}
'''


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("share")
    (d / "walk.cpp").write_text(WALK)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", _lib.CSRC, str(d / "walk.cpp"), "-o", str(d / "walk")])

    def run(n, total, kv, share, blocks, units, steps):
        text = " ".join(map(str, [n, total, kv, share, blocks, *units, *steps]))
        out = subprocess.run([str(d / "walk")], input=text, capture_output=True, text=True, timeout=60)
        assert out.returncode == 0, out.stderr
        assert "outside" not in out.stdout and "endless" not in out.stdout
        rows = [line.split() for line in out.stdout.splitlines()[1:]]
        return [tuple(map(int, r[1:])) for r in rows if r[0] == "walk"], [tuple(map(int, r[1:])) for r in rows if r[0] == "meet"]
    return run


def plan(lq, lk, group, causal):
    p = PackedRows(lq, lk, group=group, causal=causal, device="cpu")
    t = p._table.numpy()
    pairs = t[2 * (p.seqs + 1) + 2 * p.n_row_tiles:][:2 * p.n_key_tiles].reshape(-1, 2)
    lk = lk or lq
    first = [min(max(k * KEY_TILE - (lk[s] - lq[s]), 0), lq[s]) if causal else 0 for s, k in pairs.tolist()]
    steps = [(-(-lq[s] // 32) - f // 32) * group for (s, _), f in zip(pairs.tolist(), first)]
    return p, t[-p.n_key_tiles - 1:].tolist(), steps


PLANS = [([5000, 300], None, 4, 4, True), ([4096], None, 8, 1, True), ([400, 0, 5, 900], [400, 300, 5, 901], 2, 3, False), ([3000], [100], 2, 1, True),
         ([700, 260], [130, 500], 1, 5, True)]


@pytest.mark.parametrize("lq,lk,group,kv,causal", PLANS)
def test_shares_walk_every_step_once_and_meet_where_they_left_sums(walk, lq, lk, group, kv, causal):
    p, units, steps = plan(lq, lk, group, causal)
    for share in (1, 3, 8, 50, 1000):
        blocks = -(-p.key_units * kv // share)
        walks, meets = walk(p.n_key_tiles, p.key_units, kv, share, blocks, units, steps)
        seen, slots = {}, {}
        for b, kh, t, first, last, slot in walks:
            seen.setdefault((kh, t), []).append((first, last))
            if slot >= 0:
                assert 0 <= slot < 2 * blocks and slot not in slots
                slots[slot] = (kh, t)
        assert set(seen) == {(kh, t) for kh in range(kv) for t in range(p.n_key_tiles)}
        for (kh, t), parts in seen.items():
            assert parts[0][0] == 0 and parts[-1][1] == steps[t] and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        met = {2 * b + (b == first): (kh, t) for kh, t, first, last in meets for b in range(first, last + 1)}
        assert met == slots


@pytest.mark.parametrize("lq,lk,group,kv,causal", PLANS)
def test_shares_stay_in_their_workspace_whatever_the_table_holds(walk, lq, lk, group, kv, causal):
    """A table whose memory was given away (a plan dropped while a graph that was captured with it is still replayed): too many units, none at all,
    anything."""
    p, units, steps = plan(lq, lk, group, causal)
    n, total = p.n_key_tiles, p.key_units
    rng = random.Random(1)
    wrong = [units[:-1] + [units[-1] + 1000 * kv], [0] * (n + 1), [u + 7 for u in units], units[::-1], [0x7fffffff] * (n + 1), [-0x80000000, 0x7fffffff] * n,
             *[[rng.randrange(-(1 << 31), 1 << 31) for _ in range(n + 1)] for _ in range(5)], *[[rng.randrange(0, 2 * total) for _ in range(n + 1)] for _ in range(5)]]
    for table in wrong:
        for share in (3, 50, total):
            blocks = -(-total * kv // share)
            walks, meets = walk(n, total, kv, share, blocks, (table + table)[:n + 1], steps)
            for b, kh, t, first, last, slot in walks:
                assert -1 <= slot < 2 * blocks and 0 <= first <= last <= steps[t], (table, share)
            for kh, t, first, last in meets:
                assert 0 <= first and last < blocks


def test_requests_into_lds_hold_their_wait_states(tmp_path):
    """A request into LDS as inline assembly: the hardware wants one wait state between the write of M0 and a load that goes to LDS by it, and five between a
    vector instruction's write of a scalar register (readfirstlane, readlane) and a load that reads it.  The compiler puts both in front of its own
    instructions, but not into a text of ours."""
    found = 0
    for name in sorted(os.listdir(_lib.CSRC)):
        if not name.endswith((".hip", ".h")):
            continue
        for text in re.findall(r'asm volatile\("((?:[^"\\]|\\.)*)"', open(os.path.join(_lib.CSRC, name)).read()):
            lines = text.replace("\\t", "").split("\\n")
            for before, line in zip([""] + lines, lines):
                if line.startswith("buffer_load") and line.endswith(" lds"):
                    found += 1
                    assert before.startswith("s_nop"), (name, text)
    assert found >= 3

    out = tmp_path / "packed_attn.s"
    flags = [f for f in _lib.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.check_call(["hipcc"] + flags + ["-S", "--cuda-device-only", os.path.join(_lib.CSRC, "packed_attn.hip"), "-o", str(out)], stderr=subprocess.DEVNULL)
    lines = [line.split(";")[0].strip() for line in out.read_text().splitlines()]
    lines = [line for line in lines if line and line[0] not in ".#"]

    def scalars(text):
        got = set()
        for lo, hi, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
            got |= set(range(int(lo), int(hi) + 1)) if lo else {int(one)}
        return got
    requests = 0
    for i, line in enumerate(lines):
        if not (line.startswith("buffer_load") and line.endswith(" lds")):
            continue
        requests += 1
        need, waits, moved = scalars(line), 0, 0
        for before in reversed(lines[max(i - 8, 0):i]):
            if before.endswith(":"):
                continue
            if re.match(r"s_\w+ m0,", before):
                moved = waits
                assert moved >= 1, (i, before, line)
            if before.startswith("v_") and waits < 5:
                first = before.split(None, 1)[1].split(",")[0] if " " in before else ""
                assert not scalars(first) & need, (i, before, line)
            waits += int(before.split()[1]) + 1 if before.startswith("s_nop") else 1
        assert moved
    assert requests > 500


class Streams:
    """Streams without a device: each knows which launches it comes behind."""

    class One:
        def __init__(self, handle, capturing=False):
            self.cuda_stream, self.seen, self.capturing = handle, set(), capturing

        def wait_stream(self, other):
            assert self.capturing == other.capturing or not self.capturing, "a captured stream waits for work outside its capture"
            self.seen |= other.seen

    def __init__(self, monkeypatch, rt, defer=""):
        from crog_amd import kernels as K
        self.main, self.wgrad = self.One(1), self.One(99)
        self.now, self.launched, self.callbacks, self.kept = self.main, [], [], []
        self.all = {1: self.main, 99: self.wgrad}

        @contextlib.contextmanager
        def on(s):
            old, self.now = self.now, s
            yield
            self.now = old
        self.on = on
        monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: self.now)
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.now.capturing)
        monkeypatch.setattr(torch.autograd.Variable, "_execution_engine", types.SimpleNamespace(queue_callback=self.callbacks.append))
        monkeypatch.setattr(K, "stream", lambda: K._STREAM_OVERRIDE if K._STREAM_OVERRIDE is not None else self.now.cuda_stream)
        monkeypatch.setattr(K, "gated_norm_bwd", lambda *a: self.slab())
        monkeypatch.setattr(K, "gated_norm_sums", lambda slab, *a: self.launch(slab))
        for name, value in (("_wgrad_stream", [self.wgrad]), ("_streams_ready", True), ("streams", [self.wgrad]), ("text_stream", None), ("aux_stream", None),
                            ("_join_armed", False), ("_direct", None), ("defer_wgrad", defer), ("overlap_wgrad", True), ("deterministic", False)):
            monkeypatch.setattr(rt, name, value, raising=False)
        self.K = K

    def user(self, handle, capturing=False):
        return self.all.setdefault(handle, self.One(handle, capturing))

    def slab(self):
        slab = types.SimpleNamespace(record_stream=lambda s: None)
        self.all[self.K.stream()].seen.add(id(slab))
        self.kept.append(slab)
        return slab

    def launch(self, slab=None):
        s = self.all[self.K.stream()]
        assert slab is None or id(slab) in s.seen, "the sums are read before they are there"
        for before in self.launched:
            assert before in s.seen, "two kernels add onto one gradient, neither behind the other"
        s.seen.add(len(self.launched))
        self.launched.append(len(self.launched))

    def end_of_backward(self, nodes_streams):
        """backward() returns: its stream waits for the nodes whose gradients went on, and the queued callbacks run on it."""
        for s in nodes_streams:
            if s is not self.main:
                self.main.wait_stream(s)
        calls, self.callbacks[:] = list(self.callbacks), []
        for c in calls:
            c()
        assert set(self.launched) <= self.main.seen, "backward() has returned, and its stream is not behind a weight's gradient"


@pytest.mark.parametrize("defer", ["", "all"])
@pytest.mark.parametrize("seed", range(40))
def test_gradients_of_a_shared_weight_are_added_one_after_the_other(monkeypatch, seed, defer):
    """Gated norms and LayerNorms that share a weight, their forward passes (so their backward nodes) on several streams of the user's: every addition onto the
    weight's gradient is ordered against every other, and the stream that called backward() is behind them all."""
    from crog_amd.functional import RT, GatedNormFn, WRef
    from crog_amd.runtime import ParamStore
    m = torch.nn.Module()
    m.w = torch.nn.Parameter(torch.ones(8))
    w = WRef(ParamStore(m, torch.device("cpu")), m.w, cols=1)
    fake = Streams(monkeypatch, RT, defer)
    rng = random.Random(seed)
    x = torch.zeros(4, 8)
    if rng.random() < 0.3:      # (the device's first stream may have been somebody else's before)
        with fake.on(fake.user(7)):
            GatedNormFn.backward(types.SimpleNamespace(cfg=(w, None, None, 1.0, False), saved_tensors=(x, x, x), needs_input_grad=(True, True)), x, None)
        fake.end_of_backward([fake.user(7)])
    for _ in range(3):
        joined = []
        for _ in range(rng.randrange(1, 6)):
            s = rng.choice([fake.main, fake.main, fake.user(2), fake.user(3)])
            with fake.on(s):
                kind = rng.choice(["gated", "gated", "gated", "alone", "layer"])
                if kind == "layer":
                    RT.on_wgrad_stream(fake.launch, tag="ln")
                else:
                    needs = (False, False) if kind == "alone" else (True, rng.random() < 0.5)      # alone: only its weights take a gradient
                    GatedNormFn.backward(types.SimpleNamespace(cfg=(w, None, None, 1.0, False), saved_tensors=(x, x, x), needs_input_grad=needs), x, None)
                    if kind == "gated":
                        joined.append(s)
        fake.end_of_backward(joined)
        for s in (fake.user(2), fake.user(3)):      # (the next forward pass on them begins behind the caller's stream)
            s.wait_stream(fake.main)


def test_a_capture_does_not_wait_for_gradients_added_before_it(monkeypatch):
    from crog_amd.functional import RT
    fake = Streams(monkeypatch, RT)
    RT.add_gradients(fake.launch, joined=True)
    captured = fake.user(5, capturing=True)
    captured.seen |= fake.main.seen      # (a capture begins behind what was enqueued)
    with fake.on(captured):
        RT.add_gradients(fake.launch, joined=True)
        fork = fake.user(6, capturing=True)
        fork.wait_stream(captured)
        fake.wgrad.capturing = True
        with fake.on(fork):
            RT.add_gradients(fake.launch, joined=True)
    assert len(fake.launched) == 3 and len(fake.callbacks) == 1


@pytest.mark.parametrize("shape,stride", [((3, 4, 64), (260, 65, 1)), ((1, 1, 64), (260, 65, 1)), ((1, 2, 128), (1 << 24, 128, 1)), ((5, 1, 64), (64, 3, 1)), ((1, 4, 64), (7, 64, 1)),
                                          ((6, 1, 64), (128, 1 << 30, 1))])
def test_heads_of_one_row_or_one_head_have_strides_the_kernels_take(shape, stride):
    """torch leaves a dimension of one element whatever stride a slice gave it, and calls the tensor contiguous."""
    from crog_amd import kernels as K
    rows, heads, dim = shape
    buf = torch.arange(rows * 600 + 600, dtype=torch.float32).bfloat16()
    t = torch.as_strided(buf, shape, tuple(s if n > 1 else s for s, n in zip(stride, shape)))
    got = K.heads16(t)
    at, ld, hs = K._heads(got)
    assert torch.equal(got, t) and at % 16 == 0 and ld % 8 == 0 and hs % 8 == 0 and 0 <= ld * 64 * 2 < 0x7fff0000 and 0 <= hs < 1 << 24
    if rows * heads * dim and (heads == 1 or stride[1] % 8 == 0) and (rows == 1 or stride[0] % 8 == 0) and t.data_ptr() % 16 == 0:
        assert got.data_ptr() == t.data_ptr()      # (nothing to copy)


@pytest.mark.parametrize("shape,stride", [((1, 8), (1, 1)), ((1, 1, 8), (3, 5, 1)), ((4, 1, 8), (16, 2, 1)), ((1, 8), (0, 1)), ((3, 8), (0, 1)), ((2, 3, 8), (0, 8, 1))])
def test_row_matrices_of_one_row_are_taken_whatever_its_stride(shape, stride):
    from crog_amd import kernels as K
    t = torch.as_strided(torch.arange(200.0), shape, stride)
    m = K.as_mat(t)
    rows, cols, ld = K.mat(m)
    assert torch.equal(m, t) and (rows, cols) == (t.numel() // 8, 8) and ld >= 8
    flat = torch.as_strided(m, (rows, cols), (ld, 1), m.storage_offset())
    assert torch.equal(flat, t.reshape(rows, cols))


@pytest.mark.parametrize("rows,axes,stride", [(1, 3, (1, 1)), (1, 1, (0, 1)), (1, 2, (0, 1)), (4, 2, (2, 1)), (4, 2, (7, 1)), (4, 2, (0, 1)), (4, 1, (3, 1)), (4, 1, (3, 5)), (1, 1, (0, 0))])
def test_positions_of_one_row_or_one_axis_are_taken_whatever_their_strides(monkeypatch, rows, axes, stride):
    from crog_amd import functional as Fn
    from crog_amd import kernels as K
    from crog_amd.packed import RotaryAxes
    seen = {}
    monkeypatch.setattr(K, "same_device", lambda *a: None)
    monkeypatch.setattr(K, "plan_used", lambda a: None)
    monkeypatch.setattr(K, "stream", lambda: 0)
    names = _lib.parse_header()["crog_rotary"][2]
    monkeypatch.setattr(K, "lib", lambda: types.SimpleNamespace(crog_rotary=lambda *a: seen.update(zip(names, a)) or 0))
    pos = torch.as_strided(torch.arange(100), (rows, axes), stride)
    Fn.rotary(torch.zeros(rows, 2, 16), None, pos, RotaryAxes((2,) * axes, device="cpu"))
    assert seen["ldpos"] >= axes and seen["axes"] == axes and seen["rows"] == rows      # (what the C entry asks of them)


@pytest.mark.parametrize("scale", [1e39, -1e39, 2.4e38, -3.4e38, 1e308])
def test_scales_that_float32_does_not_hold_are_refused(scale):
    """The kernels take the scale in float32 and in units of log 2: beyond that range every score would be an infinity or NaN."""
    from crog_amd import functional as Fn
    q = torch.zeros(6, 2, 64)
    rows = PackedRows([6], device="cpu")
    with pytest.raises(ValueError):
        Fn.packed_attention(q, q, q, rows, scale)
    with pytest.raises(RuntimeError):      # (all well: but there is no CPU path)
        Fn.packed_attention(q, q, q, rows, scale / 1e308)
    if abs(scale) > 3.5e38:
        with pytest.raises(ValueError):
            Fn.gated_norm(torch.zeros(4, 8), torch.zeros(4, 8), res_scale=scale)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_c_entries_refuse_scales_that_are_not_finite(value):
    lib = _lib.load()
    buf = torch.zeros(4096)
    p = (buf.data_ptr() + 15) // 16 * 16
    fwd = [1] + [p, 64, 64] * 4 + [None, p, p, p, 1, 1, 8, 8, 1, 1, 64, value, 0, 1, 0, None, None]
    bwd = [1] + [p, 64, 64] * 5 + [p, p] + [p, 64, 64] * 3 + [p, p, p, 1, p, 1, 1, 8, 8, 1, 1, 64, value, 0, 1, 0, None, 0, 0, None, None]
    calls = [(lib.crog_packed_attn_fwd, fwd), (lib.crog_packed_attn_bwd, bwd)]
    if value != 3e38:      # (a float32 like any other where no logarithm is taken)
        calls += [(lib.crog_gated_norm_fwd, [1, p, 64, p, 64, None, None, None, None, None, 0, 1, 0, value, 1e-5, 0, 64, p, 64, p, 64, None, None]),
                  (lib.crog_gated_norm_bwd, [1, p, 64, p, 64, p, 64, p, 64, None, None, None, None, 0, 1, 0, value, 0, 64, p, p, 64, p, 64, None, None])]
    for entry, args in calls:
        assert len(args) == len(entry.argtypes)
        assert entry(*args) == -1 and b"finite" in lib.crog_last_error()


@pytest.mark.parametrize("rows", [(1 << 32) + 5, 1 << 31, 0x7fff0001])
def test_more_rows_than_the_kernels_count_are_refused(rows):
    """Row numbers are 32 bits on the device: 2^32 + 5 rows would be taken for five."""
    from crog_amd import functional as Fn
    from crog_amd.packed import RotaryAxes
    x = torch.zeros(1, 8).expand(rows, 8)
    with pytest.raises(ValueError, match="rows"):
        Fn.gated_norm(x, x)
    with pytest.raises(ValueError, match="rows"):
        Fn.gated_norm(x[None], x[None])
    q, pos = torch.zeros(1, 1, 4).expand(rows, 1, 4), torch.zeros(1, dtype=torch.int32).expand(rows)
    with pytest.raises(ValueError, match="rows"):
        Fn.rotary(q, None, pos, RotaryAxes((2,), device="cpu"))
    lib = _lib.load()
    if rows < 1 << 31:
        buf = torch.zeros(4096)
        p = (buf.data_ptr() + 15) // 16 * 16
        assert lib.crog_rotary(1, p, 64, 64, p, 64, 64, p, 64, 64, p, 64, 64, p, 1, 4, p, p, rows, 1, 1, 64, 32, 1, 0, 0, None) == -1
        assert lib.crog_gated_norm_fwd(1, p, 64, p, 64, None, None, None, None, None, 0, 1, 0, 1.0, 1e-5, rows, 64, p, 64, p, 64, None, None) == -1
        assert lib.crog_gated_norm_bwd(1, p, 64, p, 64, p, 64, p, 64, None, None, None, None, 0, 1, 0, 1.0, rows, 64, p, p, 64, p, 64, None, None) == -1


def test_a_theta_whose_angles_overflow_is_refused():
    """A position of zero times an infinite angle is NaN."""
    from crog_amd.packed import RotaryAxes
    with pytest.raises(ValueError, match="theta"):
        RotaryAxes((128,), theta=5e-324, device="cpu")
    RotaryAxes((128,), theta=1e-300, device="cpu")
