"""The packed operators in company: weights shared with the framework's own layers, several streams, captured graphs, plans that are dropped early."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape) + len(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def store_of(seed=0, **shapes):
    from crog_amd.functional import WRef
    from crog_amd.runtime import ParamStore
    m = torch.nn.Module()
    for i, (n, shape) in enumerate(shapes.items()):
        w = dev(*shape, seed=seed + i)
        m.register_parameter(n, torch.nn.Parameter(w * shape[-1] ** -0.5 if len(shape) == 2 else 0.3 * w + n.endswith("w")))
    st = ParamStore(m, torch.device("cuda", torch.cuda.current_device()))
    return m, st, {n: WRef(st, p) if p.dim() == 2 else WRef(st, p, cols=1) for n, p in m.named_parameters()}


@pytest.fixture(params=["as it is", "deferred", "deterministic"])
def mode(request):
    from crog_amd.runtime import RT, set_deterministic
    old = RT.defer_wgrad
    RT.defer_wgrad = "all" if request.param == "deferred" else ""
    if request.param == "deterministic":
        set_deterministic(True)
    yield request.param
    RT.defer_wgrad = old
    if request.param == "deterministic":
        set_deterministic(False)


T, C = 130, 64
WEIGHTS = dict(gate=(C,), post_w=(C,), post_b=(C,), norm_w=(C,), norm_b=(C,), lin_w=(C, C), lin_b=(C,))


def block(r, x, y):
    """Two gated norms, a linear layer and a LayerNorm between them; the three norms share one weight and one bias, the gated norms their gate.  Backward:
    the second gated norm adds first, on its own stream; the layers fork to the weight-gradient stream; the first gated norm follows them there."""
    from crog_amd import functional as Fn
    u, h = Fn.gated_norm(x, y, post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["norm_w"], r["norm_b"]), res_scale=0.9)
    t = Fn.layernorm(Fn.linear(h, r["lin_w"], r["lin_b"]), r["norm_w"], r["norm_b"])
    return Fn.gated_norm(u, t, gate=r["gate"], pre=(r["norm_w"], r["norm_b"]))


def block_reference(m, x, y):
    ln = torch.nn.functional.layer_norm
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    u = 0.9 * x + p["gate"] * ln(y, (C,), p["post_w"], p["post_b"], 1e-5)
    t = ln(ln(u, (C,), p["norm_w"], p["norm_b"], 1e-5) @ p["lin_w"].T + p["lin_b"], (C,), p["norm_w"], p["norm_b"], 1e-5)
    u = u + p["gate"] * t
    return u, ln(u, (C,), p["norm_w"], p["norm_b"], 1e-5), p


def test_gated_norm_beside_the_frameworks_layers(mode):
    """Every gradient within 2^-14 of the largest of its tensor: float32 sums over 130 rows and 64 columns (2^-24 for each of their terms, 2^-16 in all),
    through three norms of rows whose deviation is about one."""
    m, st, r = store_of(**WEIGHTS)
    x, y = (dev(T, C, seed=i).requires_grad_() for i in (1, 2))
    gu, gh = dev(T, C, seed=3), dev(T, C, seed=4)
    x64, y64 = (t.detach().double().requires_grad_() for t in (x, y))
    u, h, p = block_reference(m, x64, y64)
    want = torch.autograd.grad((u, h), [x64, y64, *p.values()], (gu.double(), gh.double()))
    first = None
    for _ in range(3):
        st.zero_grad()
        dx, dy = torch.autograd.grad(block(r, x, y), (x, y), (gu, gh))
        got = [dx, dy, *[ref.grad().view(m.get_parameter(n).shape) for n, ref in r.items()]]
        for n, a, b in zip(["x", "y", *r], got, want):
            assert (a.double() - b).abs().max() <= 2.0 ** -14 * b.abs().max(), n
        got = [t.clone() for t in got]
        first = first or got
        assert all(torch.equal(a, b) for n, a, b in zip(["x", "y", *r], got, first) if not n.startswith("lin"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_gated_norm_adds_the_same_bits_on_either_stream(dtype, mode):
    """Alone (its own stream) and behind a layer whose backward has forked (the weight-gradient stream)."""
    from crog_amd import functional as Fn
    m, st, r = store_of(**WEIGHTS)
    x, y, z = (dev(T, C, dtype=dtype, seed=i).requires_grad_() for i in (1, 2, 5))
    gu, gh = dev(T, C, dtype=dtype, seed=3), dev(T, C, dtype=dtype, seed=4)
    names = ("gate", "post_w", "post_b", "norm_w", "norm_b")

    def gated():
        return Fn.gated_norm(x, y, post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["norm_w"], r["norm_b"]))
    st.zero_grad()
    a = torch.autograd.grad(gated(), (x, y), (gu, gh))
    alone = [r[n].grad().clone() for n in names]
    st.zero_grad()
    outs = gated()
    first = Fn.linear(z, r["lin_w"], r["lin_b"])      # (made last: its backward runs first)
    b = torch.autograd.grad((*outs, first), (x, y, z), (gu, gh, gh))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(t, r[n].grad()) for n, t in zip(names, alone))
    only = Fn.gated_norm(x.detach(), y.detach(), gate=r["gate"])[0]      # nothing but a weight takes a gradient
    st.zero_grad()
    only.backward(gu)
    got = r["gate"].grad().clone()
    st.zero_grad()
    torch.autograd.grad(Fn.gated_norm(x, y.detach(), gate=r["gate"])[0], x, gu)
    assert torch.equal(r["gate"].grad(), got)


def test_gated_norms_on_several_streams_share_weights(mode):
    from crog_amd import functional as Fn
    m, st, r = store_of(**WEIGHTS)
    leaves = [(dev(4000, C, dtype=torch.bfloat16, seed=i).requires_grad_(), dev(4000, C, dtype=torch.bfloat16, seed=i + 10).requires_grad_()) for i in range(4)]
    grads = [dev(4000, C, dtype=torch.bfloat16, seed=20 + i) for i in range(8)]
    main, streams = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(3)]

    def run(where):
        st.zero_grad()
        outs = []
        for (x, y), s in zip(leaves, where):
            s.wait_stream(main)
            with torch.cuda.stream(s):
                outs += Fn.gated_norm(x, y, post=(r["norm_w"], r["norm_b"]), gate=r["norm_w"], pre=(r["norm_w"], r["norm_b"]))
        for s in streams:
            main.wait_stream(s)
        d = torch.autograd.grad(outs, [t for pair in leaves for t in pair], grads)
        return [st.G.clone(), *d]
    want = run([main] * 4)
    assert want[0].abs().sum() > 0
    for where in ([streams[0], streams[1], streams[2], main], [main, streams[0], streams[0], streams[1]], [streams[2]] * 4, [main] * 4):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(run(where), want))


@pytest.mark.parametrize("warm", ["side", "main", "both"])
def test_gated_norm_beside_the_frameworks_layers_captured_and_replayed(warm):
    from crog_amd import functional as Fn
    m, st, r = store_of(**WEIGHTS)
    x, y, gu, gh = (dev(T, C, seed=i) for i in (1, 2, 3, 4))
    x.requires_grad_(), y.requires_grad_()

    def step():
        outs = block(r, x, y)
        return (*outs, *torch.autograd.grad(outs, (x, y), (gu, gh)))
    side = torch.cuda.Stream()
    if warm != "main":
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
    if warm != "side":      # (the last gradients before the capture were added on the device's own stream)
        step()
        torch.autograd.grad(Fn.gated_norm(x, y, gate=r["gate"])[0], x, gu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    norms = [n for n in r if not n.startswith("lin")]
    for turn in range(4):
        with torch.no_grad():
            for i, t in enumerate((x, y, gu, gh)):
                t.copy_(dev(T, C, seed=10 * turn + i))
        st.zero_grad()
        want = step()
        once = {n: r[n].grad().clone() for n in r}
        st.zero_grad()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn
        for n in r:
            assert torch.equal(r[n].grad(), once[n]) if n in norms else (r[n].grad() - once[n]).abs().max() <= 2.0 ** -14 * once[n].abs().max(), (turn, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_one_row_and_one_head_of_any_stride(dtype):
    """Slices of a cache or a projection with an odd or a very long stride along a dimension of one element."""
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows, RotaryAxes

    def odd(t, *strides):      # the same values, with these strides where t has one element
        buf = torch.empty(max(t.numel() * 3, 4096), device="cuda", dtype=t.dtype)
        return torch.as_strided(buf, t.shape, [s if n == 1 else d for n, s, d in zip(t.shape, strides, t.stride())]).copy_(t)
    q, do = (dev(1, 1, 64, dtype=dtype, seed=i) for i in (1, 2))
    k, v = (dev(300, 1, 64, dtype=dtype, seed=i) for i in (3, 4))
    rows = PackedRows([1], [300], causal=True)

    def grads(*ts):
        leaves = [t.detach().requires_grad_() for t in ts[:3]]
        o = Fn.packed_attention(*leaves, rows)
        return [o.detach(), *torch.autograd.grad(o, leaves, ts[3])]
    want = grads(q, k, v, do)
    for s in ((260, 65), (1 << 24, 3), (7, 1 << 30)):
        got = grads(odd(q, s[0], s[1], 1), odd(k, 0, s[1], 1), odd(v, 0, s[1], 1), odd(do, s[0], s[1], 1))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), s
    axes = RotaryAxes((8, 8, 16))
    pos = torch.tensor([[5, 70, 900]], device="cuda")
    a = Fn.rotary(q, k[:1], pos, axes)
    for s in ((1, 1), (0, 1)):
        b = Fn.rotary(odd(q, 65, 3, 1), odd(k[:1], 3, 5, 1), torch.as_strided(torch.cat([pos, pos]), (1, 3), s), axes)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    m, st, r = store_of(**WEIGHTS)
    x, y = dev(1, C, dtype=dtype, seed=5), dev(1, C, dtype=dtype, seed=6)

    def normed(x, y, g):
        x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
        st.zero_grad()
        u, h = Fn.gated_norm(x, y, post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["norm_w"], r["norm_b"]))
        return [u.detach(), h.detach(), *torch.autograd.grad((u, h), (x, y), (g, g)), st.G.clone()]
    want = normed(x, y, x)
    assert all(torch.equal(a, b) for a, b in zip(normed(odd(x, 1, 1), odd(y, 3, 1), odd(x, 0, 1)), want))


def test_a_dropped_plan_keeps_its_memory_until_its_launches_have_read_it():
    """Plans made on one stream, used on another that is still busy, and dropped: their tables' memory goes to no new tensor before the launches on the other
    stream are through."""
    import weakref

    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows, RotaryAxes
    lens = [400, 100]
    q, k, v, do = (dev(500, 2, 64, dtype=torch.bfloat16, seed=i) for i in range(4))
    pos = torch.arange(500, device="cuda")

    def run(rows, axes):
        a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
        o = Fn.packed_attention(*Fn.rotary(a, b, pos, axes), c, rows)
        return [o.detach().clone(), *torch.autograd.grad(o, (a, b, c), do)]

    def plans():
        return PackedRows(lens, causal=True), RotaryAxes((32,))
    want = run(*plans())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*plans())      # (what a first pass allocates on that stream is there)
    torch.cuda.synchronize()
    sizes = [p._table.numel() * p._table.element_size() for p in plans()]

    def fillers():      # (new memory of the tables' size classes, on the stream that the plans were made on; kept, so that each is another)
        return [torch.full((n,), 255, device="cuda", dtype=torch.uint8) for n in sizes for _ in range(40)]
    # without a launch the memory is given away at once: fillers do come to lie where the tables lay
    rows, axes = plans()
    tables = {rows._table.data_ptr(), axes._table.data_ptr()}
    del rows, axes
    assert tables <= {t.data_ptr() for t in fillers()}

    rows, axes = plans()
    tables, alive = {rows._table.data_ptr(), axes._table.data_ptr()}, [weakref.ref(rows), weakref.ref(axes)]
    work = torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(150):      # (a tenth of a second of work ahead of the launches)
            work = torch.mm(work, work) * 1e-2
        got = run(rows, axes)
        done = side.record_event()
    del rows, axes
    dropped = not any(r() for r in alive)
    new = fillers()
    busy = not done.query()
    torch.cuda.synchronize()
    assert dropped
    assert busy, "the other stream was through before the fillers were made: the test shows nothing"
    assert not tables & {t.data_ptr() for t in new}
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item()
    assert (off <= bound).all(), f"{what}: off by {worst:.3g} times its bound"


@pytest.mark.parametrize("n,causal,group,tight", [(65, True, 1, "dq dv"), (100, False, 1, "dq dv"), (128, True, 1, "dq dv"), (128, False, 2, "dv"), (64, False, 2, "dq dv"),
                                                  (129, False, 1, ""), (129, True, 1, "")])
def test_attention_gradients_on_both_sides_of_the_few_row_rule(n, causal, group, tight):
    """Up to 128 rows (dQ: queries times group; dK / dV: queries) the rests of the rounded probabilities and dS follow them.  Bounds, added up from the
    roundings: the output by half a step, a rest by half a step of half a step (2^-16; a rounded value alone 2^-8), D = dO . o from the stored o (half a step of
    o), the probabilities by float32 arithmetic (2^-24 for each of the 64 terms of a score and the n terms of a sum, worst case, as relative error)."""
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows
    D, h, U = 64, 2.0 ** -8, 2.0 ** -24
    lens = [n] * 3
    rows = PackedRows(lens, group=group, causal=causal)
    q, do = (dev(3 * n, group, D, dtype=torch.bfloat16, seed=i).requires_grad_(i == 1) for i in (1, 2))
    k, v = (dev(3 * n, 1, D, dtype=torch.bfloat16, seed=i).requires_grad_() for i in (3, 4))
    dq, dk, dv = torch.autograd.grad(Fn.packed_attention(q, k, v, rows), (q, k, v), do)
    ok = torch.ones(n, n, dtype=torch.bool, device="cuda")
    ok = ok.tril() if causal else ok
    for s in range(3):
        at = slice(s * n, (s + 1) * n)
        kk, vv = k[at, 0].detach().double(), v[at, 0].detach().double()
        want_v = torch.zeros(n, D, dtype=torch.float64, device="cuda")
        err_v = torch.zeros_like(want_v)
        for g in range(group):
            qq, gg = q[at, g].detach().double(), do[at, g].double()
            x = qq @ kk.T / 8
            p = torch.softmax(x.masked_fill(~ok, -float("inf")), 1)
            o, dp = p @ vv, gg @ vv.T
            ep = 2 * U * ((D + 4) * (qq.abs() @ kk.abs().T / 8).amax(1, keepdim=True) + 16) + U * n
            rest = h * h if "dv" in tight else h
            want_v += p.T @ gg
            err_v += (p * (rest + ep)).T @ gg.abs() + U * (n * group + 4) * (p.T @ gg.abs())
            ds = p * (dp - (gg * o).sum(1, keepdim=True)) / 8
            stored = h * o.abs() + (h + ep) * (p @ vv.abs()) * (1 + h)      # (the forward's probabilities are rounded without a rest)
            edd = (gg.abs() * stored).sum(1, keepdim=True) + U * (D + n) * (gg.abs() @ vv.abs().T).amax(1, keepdim=True)
            rest = h * h if "dq" in tight else h
            eds = p / 8 * (edd + U * (D + 4) * (gg.abs() @ vv.abs().T)) + ds.abs() * (rest + ep + 4 * U)
            want_q = ds @ kk
            within(dq[at, g], want_q, (h * want_q.abs() + (eds @ kk.abs() + U * n * (ds.abs() @ kk.abs())) * (1 + h)), f"dq of sequence {s}")
        within(dv[at, 0], want_v, h * want_v.abs() + err_v * (1 + h), f"dv of sequence {s}")


@pytest.mark.parametrize("n,group", [(100, 1), (128, 1), (64, 2), (65, 1)])
def test_dq_of_few_rows_carries_the_rests(n, group):
    """As above, with D from the o that the forward stored where a row sees more than one tile of 64 keys (what the kernel takes), so that its rounding is no
    part of the bound: what is left is the output's half step, the rests' 2^-16 and float32 arithmetic."""
    from crog_amd import functional as Fn
    from crog_amd.packed import PackedRows
    D, h, U = 64, 2.0 ** -8, 2.0 ** -24
    rows = PackedRows([n] * 3, group=group)
    q, do = (dev(3 * n, group, D, dtype=torch.bfloat16, seed=i).requires_grad_(i == 1) for i in (1, 2))
    k, v = (dev(3 * n, 1, D, dtype=torch.bfloat16, seed=i) for i in (3, 4))
    o = Fn.packed_attention(q, k, v, rows)
    dq, = torch.autograd.grad(o, q, do)
    for s in range(3):
        at = slice(s * n, (s + 1) * n)
        kk, vv = k[at, 0].double(), v[at, 0].double()
        for g in range(group):
            qq, gg = q[at, g].detach().double(), do[at, g].double()
            p = torch.softmax(qq @ kk.T / 8, 1)
            ep = 2 * U * ((D + 4) * (qq.abs() @ kk.abs().T / 8).amax(1, keepdim=True) + 16) + U * n
            oo = o[at, g].detach().double() if n > 64 else p @ vv
            dp = gg @ vv.T
            ds = p * (dp - (gg * oo).sum(1, keepdim=True)) / 8
            want = ds @ kk
            edd = U * (D + n) * ((gg.abs() * oo.abs()).sum(1, keepdim=True) + (p * dp.abs()).sum(1, keepdim=True))
            edd = edd + (gg.abs() * ep * (p @ vv.abs())).sum(1, keepdim=True) * (n <= 64)
            eds = p / 8 * (edd + U * (D + 4) * (gg.abs() @ vv.abs().T)) + ds.abs() * (h * h + ep + 4 * U)
            within(dq[at, g], want, h * want.abs() + (eds @ kk.abs() + U * n * (ds.abs() @ kk.abs())) * (1 + h), f"dq of sequence {s}")


def test_gated_norm_captured_on_streams_of_its_own():
    """Two gated norms with one weight, captured alone (nothing else forks) and on two streams of the capture, after eager passes on the device's own stream."""
    from crog_amd import functional as Fn
    m, st, r = store_of(**WEIGHTS)
    x, y, gu, gh = (dev(T, C, dtype=torch.bfloat16, seed=i) for i in (1, 2, 3, 4))
    x.requires_grad_(), y.requires_grad_()

    def one():
        return Fn.gated_norm(x, y, post=(r["post_w"], r["post_b"]), gate=r["gate"], pre=(r["norm_w"], r["norm_b"]))

    def alone():
        return torch.autograd.grad(one(), (x, y), (gu, gh))

    def forked():
        here, other = torch.cuda.current_stream(), streams[0]
        other.wait_stream(here)
        with torch.cuda.stream(other):
            outs = one()
        outs = one() + outs
        here.wait_stream(other)
        return torch.autograd.grad(outs, (x, y), (gu, gh, gu, gh))
    streams = [torch.cuda.Stream()]
    for step in (alone, forked):
        step()
        alone()
        st.zero_grad()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        for turn in range(3):
            with torch.no_grad():
                for i, t in enumerate((x, y, gu, gh)):
                    t.copy_(dev(T, C, dtype=torch.bfloat16, seed=10 * turn + i))
            st.zero_grad()
            want = step()
            once = st.G.clone()
            st.zero_grad()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(st.G, once), (step.__name__, turn)
