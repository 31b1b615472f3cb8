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


def test_gated_norm_beside_the_frameworks_layers_captured_and_replayed():
    m, st, r = store_of(**WEIGHTS)
    x, y, gu, gh = (dev(T, C, seed=i) for i in (1, 2, 3, 4))
    x.requires_grad_(), y.requires_grad_()

    def step():
        outs = block(r, x, y)
        return (*outs, *torch.autograd.grad(outs, (x, y), (gu, gh)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
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
