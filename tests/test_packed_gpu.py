"""Packed attention, rotary positions and the gated norm on the GPU against plain float64 implementations.

Every tolerance is an element's own bound, added up from the roundings between the inputs and the output before the first run:
  * a stored value is rounded once, by at most half a step: H = eps(type) / 2 of its size
  * bf16 attention rounds the probabilities (and dS) to bf16 before the second product: H of each term, so H * sum |terms|
  * float32 arithmetic: U = 2^-24 of a term's size for each of its n operations, n counted from the lengths of the sums (worst case, linear)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
H = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def dev(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape) + len(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def within(got, want, bound, what):
    got = got.detach().double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), f"{what}: off by {worst:.3g} times its bound (largest difference {off.max().item():.3g})"


# ---- attention ------------------------------------------------------------------------------------------------------------------------------
def attention_reference(q, k, v, do, lq, lk, causal, scale, few=False):
    """float64 values and the bounds of the float32 / bf16 computation, sequence by sequence and head by head.  few: those of a backward pass of at
    most 64 queries and keys a sequence, where the rest of each rounded operand follows it and D does not come from the stored o."""
    T = q.dtype
    h = H[T]
    hp = h if T == torch.bfloat16 else 0.0      # the rounding of the matrix unit's operand
    D, g = q.shape[2], q.shape[1] // k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    out = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {n: torch.zeros_like(t) for n, t in out.items()}
    q0 = k0 = 0
    for n, m in zip(lq, lk):
        a, b = slice(q0, q0 + n), slice(k0, k0 + m)
        q0, k0 = q0 + n, k0 + m
        if n == 0 or m == 0:
            continue
        ok = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            ok = ok.tril(m - n)
        some = ok.any(1, keepdim=True)
        for hd in range(q.shape[1]):
            e = hd // g
            qq, kk, vv, gg = q[a, hd], k[b, e], v[b, e], do[a, hd]
            s = (qq @ kk.T) * scale
            p = torch.where(some, torch.softmax(s.masked_fill(~ok, -math.inf).masked_fill(~some, 0.0), 1), 0.0) * ok
            o = p @ vv
            # a score: D products and sums, the scale, the base-2 factor, the difference from the maximum; twice (score and maximum / sum)
            smag = abs(scale) * (qq.abs() @ kk.abs().T)
            es = 2 * U * ((D + 4) * smag.amax(1, keepdim=True) + 16)      # relative error of a probability (exp's own few steps in the 16)
            ep = es + U * m                                               # ... and of the sum they are divided by
            pv = p @ vv.abs()
            eo = (hp + ep + U * (m + 4)) * pv
            out["o"][a, hd] = o
            err["o"][a, hd] = h * o.abs() + eo * (1 + h)
            hb = hp * 2.0 ** -8 if few else hp      # (the rest, at most half a step, is rounded by half a step of its own)
            out["dv"][b, e] += p.T @ gg
            err["dv"][b, e] += (hb + U * (n * g + 4)) * (p.T @ gg.abs()) + (p * ep).T @ gg.abs()
            dp = gg @ vv.T
            dd = (gg * o).sum(1, keepdim=True)
            ds = p * (dp - dd) * scale
            # D from the stored o (or, one key tile, from the probabilities: smaller)
            stored = ep * pv if few else h * o.abs() + eo * (1 + h)
            edd = (gg.abs() * stored).sum(1, keepdim=True) + U * (D + m) * ((gg.abs() * o.abs()).sum(1, keepdim=True) + (p * dp.abs()).sum(1, keepdim=True))
            eds = abs(scale) * p * (edd + U * (D + 4) * (gg.abs() @ vv.abs().T)) + ds.abs() * (hb + ep + 4 * U)
            out["dq"][a, hd] = ds @ kk
            err["dq"][a, hd] = h * out["dq"][a, hd].abs() + (eds @ kk.abs()) * (1 + h) + U * m * (ds.abs() @ kk.abs())
            out["dk"][b, e] += ds.T @ qq
            err["dk"][b, e] += (eds.T @ qq.abs()) * (1 + h) + U * n * g * (ds.abs().T @ qq.abs())
    for n in ("dk", "dv"):
        err[n] += h * out[n].abs() + h * err[n]
    return out, {n: t + 1e-30 for n, t in err.items()}


def run_attention(q, k, v, do, rows, scale=None):
    from crog_amd import functional as Fn
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = Fn.packed_attention(q, k, v, rows, scale)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


CASES = [
    # lq, lk (None: the same rows), kv heads, group, dim, causal
    ([1], None, 1, 1, 64, True),
    ([1], [1], 2, 3, 8, False),
    ([7, 0, 20, 1, 13], None, 8, 1, 64, True),
    ([31, 32, 33, 63, 64, 65], None, 2, 1, 64, False),
    ([127, 128, 129, 1], None, 2, 4, 128, True),
    ([257, 3, 190], None, 1, 3, 80, True),
    ([40, 50], [3, 20], 4, 1, 64, False),
    ([1, 1, 1], [700, 1, 1300], 2, 4, 128, True),          # single tokens over long keys: the split form
    ([2, 5, 1], [900, 64, 2049], 1, 1, 32, True),
    ([1, 3], [40000, 6], 1, 2, 64, True),                  # a hundred splits
    ([100, 10, 64], [30, 0, 64], 2, 2, 64, True),          # more queries than keys: rows without a key; no key at all
    ([0, 5], [9, 5], 1, 2, 96, False),
    ([300], [700], 2, 2, 120, True),
    ([676, 676], None, 2, 1, 64, False),
    ([1500, 37], None, 1, 8, 128, True),
    ([400, 0, 5, 900], [400, 300, 5, 901], 3, 2, 32, False),      # dK / dV in shares: over a sequence without queries, from head to head
    ([700, 260], [130, 500], 5, 1, 96, True),
    ([640] * 34, None, 5, 1, 64, False),                          # ... more tiles than the device holds: several tiles in a share
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}x{c[4]}{'c' if c[5] else ''}".replace(" ", ""))
def test_attention_matches_the_formula(case, dtype):
    from crog_amd.packed import PackedRows
    lq, lk, kv, group, dim, causal = case
    rows = PackedRows(lq, lk, group=group, causal=causal)
    lk = lk or lq
    q, do = (dev(sum(lq), kv * group, dim, dtype=dtype, seed=i) for i in (1, 2))
    k, v = (dev(sum(lk), kv, dim, dtype=dtype, seed=i) for i in (3, 4))
    got = run_attention(q, k, v, do, rows)
    want, bound = attention_reference(q, k, v, do, lq, lk, causal, dim ** -0.5)
    for n in got:
        within(got[n], want[n], bound[n], n)
    again = run_attention(q, k, v, do, rows)
    assert all(torch.equal(got[n], again[n]) for n in got)
    from crog_amd import functional as Fn
    with torch.no_grad():
        assert torch.equal(Fn.packed_attention(q, k, v, rows), got["o"])


@pytest.mark.parametrize("lq,lk,kv,group,dim,causal", [([2] * 30, None, 1, 1, 128, True), ([1, 2, 17, 64], [45, 2, 30, 64], 2, 2, 80, False),
                                                       ([64, 5, 33], None, 3, 1, 32, True)])
def test_attention_gradients_of_few_rows_are_rounded_once(lq, lk, kv, group, dim, causal):
    from crog_amd.packed import PackedRows
    rows = PackedRows(lq, lk, group=group, causal=causal)
    lk = lk or lq
    q, do = (dev(sum(lq), kv * group, dim, dtype=torch.bfloat16, seed=i) for i in (1, 2))
    k, v = (dev(sum(lk), kv, dim, dtype=torch.bfloat16, seed=i) for i in (3, 4))
    got = run_attention(q, k, v, do, rows)
    want, bound = attention_reference(q, k, v, do, lq, lk, causal, dim ** -0.5, few=True)
    for n in ("dq", "dk", "dv"):
        within(got[n], want[n], bound[n], n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.7, -0.25, 0.0])
def test_attention_scale_and_sharp_scores(scale, dtype):
    """Scores of hundreds: one key takes everything, and the running maximum jumps by more than its slack again and again; a negative scale; a
    scale of zero, whose probabilities are all the same."""
    from crog_amd.packed import PackedRows
    lq = [300]
    rows = PackedRows(lq, causal=True)
    q, k, v, do = (dev(300, 1, 64, dtype=dtype, seed=i, scale=s) for i, s in ((1, 3.0), (2, 3.0), (3, 1.0), (4, 1.0)))
    k = (k.float() * torch.linspace(0.1, 3, 300, device="cuda")[:, None, None]).to(dtype)
    got = run_attention(q, k, v, do, rows, scale)
    want, bound = attention_reference(q, k, v, do, lq, lq, True, scale)
    for n in got:
        within(got[n], want[n], bound[n], n)


def test_attention_rows_far_apart():
    """Rows 4 MiB apart: offsets beyond 32 bits; and rows further apart than a tile's 32-bit offsets, which are copied first."""
    from crog_amd.packed import PackedRows
    rows = PackedRows([3, 2], [1100, 7], causal=True)
    q, do = dev(5, 2, 64, dtype=torch.bfloat16, seed=1), dev(5, 2, 64, dtype=torch.bfloat16, seed=2)
    k, v = dev(1107, 2, 64, dtype=torch.bfloat16, seed=3), dev(1107, 2, 64, dtype=torch.bfloat16, seed=4)
    want = run_attention(q, k, v, do, rows)
    wide = torch.empty(1107, 1 << 21, device="cuda", dtype=torch.bfloat16)
    far_k, far_v = wide[:, :128].view(1107, 2, 64).copy_(k), wide[:, 128:256].view(1107, 2, 64).copy_(v)
    got = run_attention(q, far_k, far_v, do, rows)
    assert all(torch.equal(got[n], want[n]) for n in got)
    lone = torch.empty(3, 1 << 23, device="cuda", dtype=torch.bfloat16)[:, :128].view(3, 2, 64)
    few = PackedRows([3])
    lone.copy_(k[:3])
    assert torch.equal(run_attention(q[:3], lone, lone, do[:3], few)["o"], run_attention(q[:3], k[:3], k[:3], do[:3], few)["o"])


def test_attention_strides_and_alignment():
    """Slices of one projection buffer, heads in another order of memory, a shared (expanded) key head, a start off 16 bytes."""
    from crog_amd.packed import PackedRows
    lens, kv, g, D = [70, 5, 33], 2, 2, 64
    T = sum(lens)
    rows = PackedRows(lens, group=g, causal=True)
    qkv = dev(T, (kv * g + 2 * kv) * D, dtype=torch.bfloat16, seed=1)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split((kv * g * D, kv * D, kv * D), 1))
    do = dev(kv * g, T, D, dtype=torch.bfloat16, seed=2).transpose(0, 1)
    plain = run_attention(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), rows)
    for a, b, c, d in ((q, k, v, do), (q.transpose(1, 2).contiguous().transpose(1, 2), k, v.transpose(0, 1).contiguous().transpose(0, 1), do)):
        got = run_attention(a, b, c, d, rows)
        assert all(torch.equal(got[n], plain[n]) for n in got)
    odd = torch.empty(T * kv * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(T, kv, D)
    odd.copy_(k)
    got = run_attention(q, odd, v, do, rows)
    assert all(torch.equal(got[n], plain[n]) for n in got)
    one = dev(T, 1, D, dtype=torch.bfloat16, seed=5).expand(T, kv, D)
    a, b = run_attention(q, one, v, do, rows), run_attention(q, one.contiguous(), v, do, rows)
    assert all(torch.equal(a[n], b[n]) for n in a)
    leaf = dev(T, 1, D, dtype=torch.bfloat16, seed=5).requires_grad_()      # the gradient of a broadcast key: the sum over its heads
    from crog_amd import functional as Fn
    d, = torch.autograd.grad(Fn.packed_attention(q, leaf.expand(T, kv, D), v, rows), leaf, do)
    assert torch.equal(d, b["dk"].sum(1, keepdim=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_keeps_sequences_and_the_rows_behind_them_apart(dtype):
    """NaN and infinities in another sequence and behind the last one reach nothing; rows behind the last sequence come out as zeros."""
    from crog_amd.packed import PackedRows
    lens, more = [45, 70, 3], 9
    rows = PackedRows(lens, causal=True)
    T = sum(lens) + more
    q, k, v, do = (dev(T, 2, 64, dtype=dtype, seed=i) for i in range(4))
    clean = run_attention(q, k, v, do, rows)
    assert all((clean[n][-more:] == 0).all() for n in clean)
    for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (do, -math.inf)):
        t[-more:] = bad
    got = run_attention(q, k, v, do, rows)
    assert all(torch.equal(got[n], clean[n]) for n in got)
    for t in (q, k, v):
        t[45:115] = math.nan
    got = run_attention(q, k, v, do, rows)
    for n in got:
        assert torch.equal(got[n][:45], clean[n][:45]) and torch.equal(got[n][115:], clean[n][115:])
        assert torch.isnan(got[n][45:115]).all() if n == "o" else True


def test_attention_of_nothing():
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows
    q, k = torch.zeros(0, 4, 64, device="cuda", requires_grad=True), torch.zeros(0, 2, 64, device="cuda", requires_grad=True)
    assert Fn.packed_attention(q, k, k, PackedRows([0, 0], group=2)).shape == (0, 4, 64)
    q = dev(5, 4, 64).requires_grad_()
    o = Fn.packed_attention(q, k, k, PackedRows([5], [0], group=2, causal=True))
    dq, dk = torch.autograd.grad(o.sum(), (q, k))
    assert (o == 0).all() and (dq == 0).all() and dk.shape == k.shape


def test_attention_gradients_against_differences():
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows
    rows = PackedRows([50, 3, 130], [60, 3, 130], group=2, causal=True)
    q, do, k, v = dev(183, 4, 32, seed=1), dev(183, 4, 32, seed=2), dev(193, 2, 32, seed=3), dev(193, 2, 32, seed=4)
    got = run_attention(q, k, v, do, rows)
    step = 2.0 ** -6
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
        d = dev(*t.shape, seed=9)
        ends = []
        for f in (step, -step):
            args = {"dq": q, "dk": k, "dv": v}
            args[n] = t + f * d
            ends.append((Fn.packed_attention(args["dq"], args["dk"], args["dv"], rows).double() * do.double()).sum())
        slope = ((ends[0] - ends[1]) / (2 * step)).item()
        along = (got[n].double() * d.double()).sum().item()
        # the third derivative of the softmax along a unit-scale direction is of the size of the slope's own terms: step^2 of them
        size = (got[n].double() * d.double()).square().sum().sqrt().item()
        assert abs(slope - along) <= 8 * step * step * size * math.sqrt(8) + 1e-3 * size, (n, slope, along, size)


def test_attention_captured_and_replayed():
    """A captured forward and backward, replayed on new inputs beside eager work; two graphs at once keep their own workspaces."""
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows
    rows = [PackedRows([1, 1], [900, 500], group=4, causal=True), PackedRows([130, 60], group=4, causal=True)]
    graphs = []
    for r in rows:
        q, do = dev(r.rows_q, 8, 64, dtype=torch.bfloat16, seed=1).requires_grad_(), dev(r.rows_q, 8, 64, dtype=torch.bfloat16, seed=2)
        k, v = (dev(r.rows_k, 2, 64, dtype=torch.bfloat16, seed=i).requires_grad_() for i in (3, 4))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(Fn.packed_attention(q, k, v, r), (q, k, v), do)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = Fn.packed_attention(q, k, v, r)
            grads = torch.autograd.grad(o, (q, k, v), do)
        graphs.append((g, r, q, k, v, do, (o, *grads)))
    for turn in range(4):
        for g, r, q, k, v, do, outs in graphs:
            with torch.no_grad():
                for i, t in enumerate((q, k, v, do)):
                    t.copy_(dev(*t.shape, dtype=torch.bfloat16, seed=10 * turn + i))
        for g, *_ in graphs:
            g.replay()
        for g, r, q, k, v, do, outs in graphs:
            want = run_attention(q, k, v, do, r)
            assert all(torch.equal(a, want[n]) for a, n in zip(outs, ("o", "dq", "dk", "dv"))), turn


def test_attention_on_another_stream():
    from crog_amd.packed import PackedRows
    rows = PackedRows([400, 100], causal=True)
    q, k, v, do = (dev(500, 2, 64, dtype=torch.bfloat16, seed=i) for i in range(4))
    want = run_attention(q, k, v, do, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_attention(q, k, v, do, rows)
    rows = None      # (the plan was made on the other stream: its tables' memory goes to no new tensor before the launches have read them)
    filler = [torch.full((64,), 0x7fffffff, device="cuda", dtype=torch.int32) for _ in range(64)]
    side.synchronize()
    del filler
    assert all(torch.equal(got[n], want[n]) for n in got)


# ---- rotary ---------------------------------------------------------------------------------------------------------------------------------
def rotary_reference(x, positions, parts, theta, interleaved, sign):
    n = sum(parts)
    cols = []
    for axis, size in enumerate(parts):
        for i in range(size):
            cols.append(positions[:, axis].double() * theta ** (-i / size))
    angle = sign * torch.stack(cols, 1)[:, None]
    x = x.double()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out, mag = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    mag[..., first] = mag[..., second] = a.abs() + b.abs()
    return out, mag


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,kv,dim,parts,far", [
    (1, 32, 8, 128, (64,), 1000000), (33, 3, 1, 64, (8, 12, 12), 500), (5, 2, 2, 80, (5, 7), 100), (7, 1, 1, 96, (24, 24), 2 ** 31 - 1),
    (130, 4, 4, 64, (16,), 4096), (2, 1, 3, 6, (1, 1, 1), 50), (3, 2, 1, 256, (128,), 70000)])
def test_rotary_matches_the_formula(rows, heads, kv, dim, parts, far, interleaved, dtype):
    from crog_amd import functional as Fn
    from crog_amd.packed import RotaryAxes
    axes = RotaryAxes(parts, interleaved=interleaved)
    q, dq = (dev(rows, heads, dim, dtype=dtype, seed=i).requires_grad_(i == 1) for i in (1, 2))
    k, dk = (dev(rows, kv, dim, dtype=dtype, seed=i).requires_grad_(i == 3) for i in (3, 4))
    pos = torch.randint(-far, far, (rows, len(parts)), generator=torch.Generator().manual_seed(1), dtype=torch.int64).cuda()
    pos[0] = far - 1
    for p in (pos, pos.to(torch.int32), pos.t().contiguous().t()):
        qo, ko = Fn.rotary(q, k, p, axes)
        gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
        for got, x, sign, what in ((qo, q, 1, "q"), (ko, k, 1, "k"), (gq, dq, -1, "dq"), (gk, dk, -1, "dk")):
            want, mag = rotary_reference(x.detach(), pos, parts, 10000.0, interleaved, sign)
            # turns: a product of at most 2^31 turns in 64 bits (2^-53 of it, twice), half a turn rounded to 32 bits (pi 2^-24), sine and
            # cosine within 4 steps, two products and a sum
            within(got, want, H[dtype] * want.abs() + (2 * math.pi * 2.0 ** -20 * 2.0 ** -2 * (far > 2 ** 24) + math.pi * U + 12 * U) * mag, what)
            assert torch.equal(got[..., 2 * sum(parts):], x[..., 2 * sum(parts):])


def test_rotary_strides_one_tensor_and_one_gradient():
    from crog_amd import functional as Fn
    from crog_amd.packed import RotaryAxes
    axes = RotaryAxes((16, 16))
    buf = dev(40, 6, 64, dtype=torch.bfloat16, seed=1)
    pos = torch.randint(0, 99, (40, 2), device="cuda")
    q, k = buf[:, :4], buf[:, 4:]
    a = Fn.rotary(q, k, pos, axes)
    b = Fn.rotary(q.contiguous(), k.contiguous(), pos, axes)
    c = Fn.rotary(q.transpose(1, 2).contiguous().transpose(1, 2), k.clone(), pos, axes)
    odd = torch.empty(buf[:, :4].numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(40, 4, 64).copy_(q)
    d = Fn.rotary(odd, k, pos, axes)
    assert all(torch.equal(x, y) for o in (b, c, d) for x, y in zip(a, o))
    e, none = Fn.rotary(q, None, pos, axes)
    assert none is None and torch.equal(e, a[0])
    ql, kl = q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()
    qo, ko = Fn.rotary(ql, kl, pos, axes)
    g, = torch.autograd.grad(ko, kl, ko.detach())      # (only k's gradient is asked for)
    want, mag = rotary_reference(ko.detach(), pos, (16, 16), 10000.0, False, -1)
    within(g, want, 2.0 ** -8 * want.abs() + 32 * U * mag, "dk")
    assert Fn.rotary(q[:0], k[:0], pos[:0], axes)[0].shape == (0, 4, 64)


# ---- gated norm -----------------------------------------------------------------------------------------------------------------------------
def store_of(C, names, seed):
    from crog_amd.functional import WRef
    from crog_amd.runtime import ParamStore
    m = torch.nn.Module()
    for i, n in enumerate(names):
        m.register_parameter(n, torch.nn.Parameter(dev(C, seed=seed + i) * 0.3 + (1.0 if n.endswith("w") else 0.0)))
    st = ParamStore(m, torch.device("cuda", torch.cuda.current_device()))
    return m, st, {n: WRef(st, p, cols=1) for n, p in m.named_parameters()}


def norm_reference(x, y, du, dh, w, has_post, has_pre, rms, alpha, eps):
    """float64 values, and bounds: an error of a normalised row is the error of its input over its deviation, plus the sums' own steps."""
    T = x.dtype
    h_ = H[T]
    x, y, du, dh = (t.double() for t in (x, y, du, dh))
    w = {n: t.double() for n, t in w.items()}
    C = x.shape[1]
    n = U * (C + 32)      # relative error of a sum over a row (linear bound), with what is around it
    one, nul = torch.ones(C, dtype=torch.float64, device=x.device), torch.zeros(C, dtype=torch.float64, device=x.device)

    def unit(t, et):
        """(normalised, 1 / deviation, error of normalised) of t with error et"""
        c = t if rms else t - t.mean(1, keepdim=True)
        inv = 1 / (c.square().mean(1, keepdim=True) + eps).sqrt()
        top = t.abs().amax(1, keepdim=True)
        e_c = et + (0 if rms else et.mean(1, keepdim=True) + n * top)
        e_inv = inv * ((c.abs() * inv * inv * e_c).mean(1, keepdim=True) + n)      # d(1/dev) = -1/dev^3 mean(c dc)
        return c * inv, inv, e_c * inv + c.abs() * e_inv, e_inv

    def back(d, ed, t, et, inv, einv):
        md, mq = (0.0 if rms else d.mean(1, keepdim=True)), (d * t).mean(1, keepdim=True)
        r = d - md - t * mq
        mag = d.abs() + (0.0 if rms else d.abs().mean(1, keepdim=True)) + t.abs() * (d * t).abs().mean(1, keepdim=True)
        er = ed + (0.0 if rms else ed.mean(1, keepdim=True)) + t.abs() * (ed * t.abs() + d.abs() * et).mean(1, keepdim=True) + et * mq.abs() + n * mag
        return r * inv, er * inv + r.abs() * einv

    gate, pw, pb = w.get("gate", one), w.get("post_w", one), w.get("post_b", nul)
    Y, ey, inv1, einv1 = (y, 0 * y, None, None)
    if has_post:
        Y, inv1, ey, einv1 = unit(y, 0 * y)
    z, ez = (Y * pw + pb, ey * pw.abs() + 4 * U * ((Y * pw).abs() + pb.abs())) if has_post else (y, 0 * y)
    u = alpha * x + gate * z
    eu = gate.abs() * ez + 4 * U * ((alpha * x).abs() + (gate * z).abs())
    out, err = {"u": u}, {"u": h_ * u.abs() + eu * (1 + h_)}
    R = U * (x.shape[0] + 600)      # a sum over the rows
    dU, edU = du, 0 * du
    if has_pre:
        hw, hb = w.get("pre_w", one), w.get("pre_b", nul)
        un, inv2, eun, einv2 = unit(u, eu)
        out["h"] = un * hw + hb
        err["h"] = h_ * out["h"].abs() + (eun * hw.abs() + 4 * U * ((un * hw).abs() + hb.abs())) * (1 + h_)
        d, ed = back(dh * hw, 2 * U * (dh * hw).abs(), un, eun, inv2, einv2)
        dU, edU = du + d, ed + 2 * U * (du.abs() + d.abs())
        out["pre_w"], err["pre_w"] = (dh * un).sum(0), (dh.abs() * eun).sum(0) + R * (dh * un).abs().sum(0)
        out["pre_b"], err["pre_b"] = dh.sum(0), R * dh.abs().sum(0)
    out["dx"] = alpha * dU
    err["dx"] = h_ * out["dx"].abs() + (abs(alpha) * edU + 2 * U * out["dx"].abs()) * (1 + h_)
    sY, sU = (dU * Y).sum(0), dU.sum(0)
    eY, eU = (edU * Y.abs() + dU.abs() * ey).sum(0) + R * (dU * Y).abs().sum(0), edU.sum(0) + R * dU.abs().sum(0)
    out["gate"] = (dU * z).sum(0)
    err["gate"] = (eY * pw.abs() + eU * pb.abs() + 4 * U * ((pw * sY).abs() + (pb * sU).abs())) if has_post else eY
    d, ed = dU * gate, edU * gate.abs() + 2 * U * (dU * gate).abs()
    if has_post:
        out["post_w"], err["post_w"] = gate * sY, gate.abs() * eY + 2 * U * (gate * sY).abs()
        out["post_b"], err["post_b"] = gate * sU, gate.abs() * eU + 2 * U * (gate * sU).abs()
        d, ed = back(d * pw, ed * pw.abs() + 2 * U * (d * pw).abs(), Y, ey, inv1, einv1)
    out["dy"], err["dy"] = d, h_ * d.abs() + ed * (1 + h_)
    return out, {k: v + 1e-30 for k, v in err.items()}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rms", [False, True], ids=["ln", "rms"])
@pytest.mark.parametrize("rows,C,has_post,has_gate,has_pre", [
    (1, 8, True, True, True), (3, 1, False, True, True), (37, 64, True, True, True), (640, 512, False, True, True), (5, 257, True, False, True), (70, 1000, True, True, False),
    (2500, 96, True, True, True), (9, 1024, False, False, True), (33, 1025, True, True, True), (12, 4096, True, True, True), (5, 5000, True, True, True),
    (3, 8192, True, True, True), (8, 333, False, True, False)])
def test_gated_norm_matches_the_formula(rows, C, has_post, has_gate, has_pre, rms, dtype):
    from crog_amd import functional as Fn
    names = (["gate"] if has_gate else []) + (["post_w"] + ([] if rms else ["post_b"]) if has_post else []) + (["pre_w"] + ([] if rms else ["pre_b"]) if has_pre else [])
    m, st, r = store_of(C, names, 20)
    x, y = (dev(rows, C, dtype=dtype, seed=i, scale=1.5).requires_grad_() for i in (1, 2))
    du, dh = (dev(rows, C, dtype=dtype, seed=i) for i in (3, 4))
    kw = dict(post=(r["post_w"], r.get("post_b")) if has_post else None, gate=r.get("gate"), pre=(r["pre_w"], r.get("pre_b")) if has_pre else None,
              res_scale=0.8, eps=1e-3, rms=rms)
    want, bound = norm_reference(x.detach(), y.detach(), du, dh, {n: p.detach() for n, p in m.named_parameters()}, has_post, has_pre, rms, 0.8, 1e-3)
    first = None
    for turn in range(2):
        st.zero_grad()
        u, h = Fn.gated_norm(x, y, **kw)
        assert (h is None) == (not has_pre)
        dx, dy = torch.autograd.grad((u, h) if has_pre else (u,), (x, y), (du, dh) if has_pre else (du,))
        got = {"u": u, "dx": dx, "dy": dy, **{n: ref.grad().clone() for n, ref in r.items()}}
        if has_pre:
            got["h"] = h
        for n in got:
            within(got[n], want[n], bound[n], n)
        first = first or got
        assert all(torch.equal(got[n], first[n]) for n in got)
    with torch.no_grad():
        a, b = Fn.gated_norm(x, y, **kw)
    assert torch.equal(a, u) and (b is None or torch.equal(b, h))


def test_gated_norm_accumulates_views_and_missing_gradients():
    from crog_amd import functional as Fn
    C = 96
    m, st, r = store_of(C, ["gate", "post_w", "post_b", "pre_w", "pre_b"], 5)
    kw = dict(post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["pre_w"], r["pre_b"]), res_scale=0.5, eps=1e-5)
    wide = dev(6, 5, 2 * C + 1, dtype=torch.bfloat16, seed=1)
    x, y = wide[..., 1:C + 1], wide[..., C + 1:]      # rows of odd stride, starts off 16 bytes
    du, dh = dev(6, 5, C, dtype=torch.bfloat16, seed=2), dev(6, 5, C, dtype=torch.bfloat16, seed=3)

    def grads(x, y, du, dh):
        x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
        st.zero_grad()
        u, h = Fn.gated_norm(x, y, **kw)
        outs, gs = zip(*[(o, g) for o, g in ((u, du), (h, dh)) if g is not None])
        return [u.detach(), h.detach(), *torch.autograd.grad(outs, (x, y), gs), *[ref.grad().clone() for ref in r.values()]]
    a, b = grads(x, y, du, dh), grads(x.contiguous(), y.contiguous(), du, dh)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    only_u, zero_h = grads(x, y, du, None), grads(x, y, du, torch.zeros_like(dh))
    assert all(torch.equal(s, t) for s, t in zip(only_u, zero_h))
    only_h, zero_u = grads(x, y, None, dh), grads(x, y, torch.zeros_like(du), dh)
    assert all(torch.equal(s, t) for s, t in zip(only_h, zero_u))
    # one weight in several places: its gradient is the sum over the places
    st.zero_grad()
    xx, yy = (t.detach().requires_grad_() for t in (x, y))
    u, h = Fn.gated_norm(xx, yy, post=(r["post_w"], r["post_b"]), gate=r["post_w"], pre=(r["post_w"], r["post_b"]), res_scale=0.5)
    torch.autograd.grad((u, h), (xx, yy), (du, dh))
    shared = {n: r[n].grad().clone() for n in ("post_w", "post_b")}
    want, bound = norm_reference(x.flatten(0, 1), y.flatten(0, 1), du.flatten(0, 1), dh.flatten(0, 1),
                                 {"gate": m.post_w.detach(), "post_w": m.post_w.detach(), "pre_w": m.post_w.detach(), "post_b": m.post_b.detach(), "pre_b": m.post_b.detach()},
                                 True, True, False, 0.5, 1e-5)
    for n, parts in (("post_w", ("gate", "post_w", "pre_w")), ("post_b", ("post_b", "pre_b"))):
        total = sum(want[p] for p in parts)
        within(shared[n], total, sum(bound[p] for p in parts) + 4 * U * sum(want[p].abs() for p in parts), n)
    # two passes without clearing add up (to one rounding each); a frozen weight is left alone
    st.zero_grad()
    m.post_w.requires_grad_(False)
    for _ in range(2):
        xx = x.detach().requires_grad_()
        u, h = Fn.gated_norm(xx, y, **kw)
        torch.autograd.grad((u, h), (xx,), (du, dh))
    for n, ref, once in zip(r, r.values(), a[4:]):
        assert (ref.grad() == 0).all() if n == "post_w" else torch.equal(ref.grad(), 2 * once)


def test_gated_norm_of_no_rows():
    from crog_amd import functional as Fn
    m, st, r = store_of(64, ["gate", "pre_w", "pre_b"], 3)
    x, y = (torch.zeros(0, 64, device="cuda", requires_grad=True) for _ in range(2))
    st.zero_grad()
    u, h = Fn.gated_norm(x, y, gate=r["gate"], pre=(r["pre_w"], r["pre_b"]))
    dx, dy = torch.autograd.grad((u, h), (x, y), (torch.zeros(0, 64, device="cuda"),) * 2)
    assert u.shape == h.shape == dx.shape == dy.shape == (0, 64) and (st.G == 0).all()


def test_rotary_and_gated_norm_captured_and_replayed():
    """Captured forward and backward passes, replayed on new inputs beside eager work: outputs, gradients and the weights' gradients, added on."""
    from crog_amd import functional as Fn
    from crog_amd.packed import RotaryAxes
    T, C = 300, 192
    axes = RotaryAxes((8, 24))
    _, st, r = store_of(C, ["gate", "post_w", "pre_w", "pre_b"], 2)
    x, y, gu, gh = (dev(T, C, dtype=torch.bfloat16, seed=i) for i in (1, 2, 3, 4))
    pos = torch.arange(2 * T, device="cuda").view(T, 2)
    x.requires_grad_(), y.requires_grad_()

    def step():
        q, _ = Fn.rotary(y.view(T, 3, 64), None, pos, axes)
        u, h = Fn.gated_norm(x, q.reshape(T, C), post=(r["post_w"], None), gate=r["gate"], pre=(r["pre_w"], r["pre_b"]))
        return (u, h, *torch.autograd.grad((u, h), (x, y), (gu, gh)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for turn in range(4):
        with torch.no_grad():
            for i, t in enumerate((x, y, gu, gh)):
                t.copy_(dev(T, C, dtype=torch.bfloat16, seed=10 * turn + i))
            pos.add_(turn)
        st.zero_grad()
        want = step()
        once = st.G.clone()
        st.zero_grad()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(st.G, once), turn
        g.replay()
        assert torch.equal(st.G, once + once), turn


def test_one_block_on_packed_rows_trains():
    """The operators as a block uses them - norm, projections, rotary, packed attention, gated residual - forward and backward, against the same
    block in float64: every gradient within a bf16 step's worth of the largest of its tensor, in float32 within 2^-14."""
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows, RotaryAxes
    lens, E, heads, kv, D = [30, 1, 77, 12], 128, 4, 2, 32
    T = sum(lens)
    rows, axes = PackedRows(lens, group=heads // kv, causal=True), RotaryAxes((8, 8))
    m, st, r = store_of(E, ["gate", "post_w", "post_b", "pre_w", "pre_b"], 3)
    pos = torch.stack([torch.arange(T) % 7, torch.arange(T) // 7], 1).cuda()
    wq = dev(E, (heads + 2 * kv) * D, seed=8, scale=E ** -0.5)
    x0 = dev(T, E, seed=1)
    g_u, g_h = dev(T, E, seed=2), dev(T, E, seed=3)

    def project(x, w):
        q, k, v = (x @ w).split((heads * D, kv * D, kv * D), 1)
        return q.unflatten(1, (heads, D)), k.unflatten(1, (kv, D)), v.unflatten(1, (kv, D))

    x, w = x0.clone().requires_grad_(), wq.clone().requires_grad_()
    st.zero_grad()
    q, k, v = project(x, w)
    q, k = Fn.rotary(q, k, pos, axes)
    o = Fn.packed_attention(q, k, v, rows).reshape(T, E)
    u, h = Fn.gated_norm(x, o, post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["pre_w"], r["pre_b"]), res_scale=0.9)
    dx, dw = torch.autograd.grad((u, h), (x, w), (g_u, g_h))
    got = {"u": u, "h": h, "dx": dx, "dw": dw, **{n: ref.grad() for n, ref in r.items()}}

    x, w = x0.double().requires_grad_(), wq.double().requires_grad_()
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    q, k, v = project(x, w)
    a0, a1 = pos[:, 0].double(), pos[:, 1].double()
    f = 10000.0 ** (-torch.arange(8, device="cuda", dtype=torch.float64) / 8)
    ang = torch.cat([a0[:, None] * f, a1[:, None] * f], 1)[:, None]

    def turn(t):
        a, b = t[..., :16], t[..., 16:]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    q, k = turn(q), turn(k)
    seq = torch.repeat_interleave(torch.arange(4), torch.tensor(lens)).cuda()
    at = torch.arange(T, device="cuda")
    ok = (seq[:, None] == seq[None]) & (at[None] <= at[:, None])
    k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5
    o = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~ok, -math.inf), -1), v).reshape(T, E)
    ln = torch.nn.functional.layer_norm
    u = 0.9 * x + p["gate"] * ln(o, (E,), p["post_w"], p["post_b"], 1e-5)
    h = ln(u, (E,), p["pre_w"], p["pre_b"], 1e-5)
    gs = torch.autograd.grad((u, h), [x, w, *p.values()], (g_u.double(), g_h.double()))
    want = {"u": u, "h": h, "dx": gs[0], "dw": gs[1], **dict(zip(p, gs[2:]))}
    for n in got:
        assert (got[n].double() - want[n]).abs().max() <= 2.0 ** -14 * want[n].abs().max(), n
