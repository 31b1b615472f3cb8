"""What the operators of a transformer block on packed rows are measured on: packed attention (captions, image tokens, long prompts, few queries
over many keys), rotary positions with several axes, and the gated residual norm between two blocks - each with its backward pass where it is
trained.  `own` False computes the plain form in float32 torch operations, `own` True calls crog_amd.functional.

A packed tensor holds the rows of all sequences one behind the other, [rows, heads, head dim]; sequence i has the i-th length."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------------------------------
def attention(name, dtype, heads, kv_heads, dim, seqs, shortest, longest, causal, train, keys_shortest=0, keys_longest=0, draw_of_lengths=1):
    """keys_longest 0: the keys are the queries' own rows (self-attention)."""
    case = {"op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs, "shortest": shortest,
            "longest": longest, "causal": causal, "train": train, "keys_shortest": keys_shortest, "keys_longest": keys_longest,
            "draw_of_lengths": draw_of_lengths}
    return dict(case, name=name) if name else case


def rotary(name, dtype, heads, kv_heads, dim, rows, axes, far, interleaved, train):
    """axes: pairs of each axis, as text; far: positions are below it."""
    case = {"op": "rotary", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rows": rows, "axes": axes, "far": far,
            "interleaved": interleaved, "train": train}
    return dict(case, name=name) if name else case


def norm(name, dtype, rows, width, rms, post, train):
    case = {"op": "norm", "dtype": dtype, "rows": rows, "width": width, "rms": rms, "post": post, "train": train}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the text tower's captions without their padding: 32 of at most 20 words, 8 heads of 64 (the smallest training call: latency)
        attention("captions train", "bf16", 8, 8, 64, 32, 3, 20, True, True),
        # the decoder's 26 x 26 image tokens, batch 32, 8 heads of 64
        attention("decoder tokens train", "bf16", 8, 8, 64, 32, 676, 676, False, True),
        # the decoder's image tokens over the words of their captions
        attention("tokens over words train", "bf16", 8, 8, 64, 32, 676, 676, False, True, 3, 20),
        # ViT-B/16 patches of images of different sizes, 12 heads of 64, in the parity type
        attention("patches train fp32", "fp32", 12, 12, 64, 8, 50, 197, False, True),
        # long packed documents with grouped heads, training
        attention("long train", "bf16", 16, 4, 128, 6, 300, 5000, True, True),
        # one whole long prompt, serving: the largest
        attention("long prompt", "bf16", 16, 2, 128, 1, 16384, 16384, True, False),
        # single new tokens over what each sequence has behind it
        attention("single tokens", "bf16", 32, 8, 128, 16, 1, 1, True, False, 200, 8192),
        # one new token's rotary position (the smallest call)
        rotary("rotary one token", "bf16", 32, 8, 128, 1, "64", 100000, False, False),
        # video tokens: time, height and width, q and k of a long pack, training
        rotary("rotary video train", "bf16", 16, 4, 128, 16384, "16,24,24", 4096, False, True),
        # the captions' 640 rows of width 512 through a layer-scaled residual and the next norm, training
        norm("norm captions train", "bf16", 640, 512, False, False, True),
        # norms on both sides of a wide block over a long pack, training
        norm("norm long train", "bf16", 32768, 1024, True, True, True),
        # the same for serving, in an odd number of rows
        norm("norm wide", "bf16", 4099, 4096, True, True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "norm"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8])
    if op == "attention":
        group = rng.choice([1, 1, 2, 3, 4, 8])
        heads = kv_heads * group
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        train = rng.random() < 0.6
        longest = min(_log(rng, 1, 6000 if dtype == "bf16" else 1500), int((4.0e8 / heads) ** 0.5))
        rows = int((1.0e7 if dtype == "bf16" else 5.0e6) / (heads * dim))
        shortest = rng.choice([longest, max(1, longest // 2), 1, 0 if longest > 1 else 1])
        seqs = max(1, min(_log(rng, 1, 64), rows // longest + 1, 12000 // longest, int(3.0e8 // (heads * longest * longest))))
        causal = rng.random() < 0.6
        keys_longest = keys_shortest = 0
        if rng.random() < 0.35:
            keys_longest = min(_log(rng, 1, 6000), int(3.0e8 // (heads * longest * seqs)) + 1, int(4.0e7 // (kv_heads * dim * seqs)) + 1)
            if causal:
                keys_longest = max(keys_longest, longest)      # (a shorter one leaves rows with no key)
            keys_shortest = rng.choice([keys_longest, max(1, keys_longest // 2), 1])
        return attention(None, dtype, heads, kv_heads, dim, seqs, shortest, longest, causal, train, keys_shortest, keys_longest,
                         rng.randrange(1 << 20))
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128])
        pairs = dim // 2 if rng.random() < 0.8 else dim // 4
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        parts = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        return rotary(None, dtype, kv_heads * rng.choice([1, 2, 4]), kv_heads, dim, _log(rng, 1, 16384), ",".join(map(str, parts)),
                      _log(rng, 16, 1000000), rng.random() < 0.4, rng.random() < 0.6)
    width = rng.choice([8 * _log(rng, 8, 512), _log(rng, 8, 4096)])
    return norm(None, dtype, min(_log(rng, 1, 40000), (32000000 if dtype == "bf16" else 16000000) // width), width, rng.random() < 0.5, rng.random() < 0.6, rng.random() < 0.6)


# ---- what the cases are made of -----------------------------------------------------------------------------------------------------------
def lengths(case):
    """Query and key lengths of an attention case (from the case alone: its work is known before its inputs are)."""
    r = random.Random(case["draw_of_lengths"])
    lq = [r.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lq[r.randrange(len(lq))] = case["longest"]
    if not case["keys_longest"]:
        return lq, lq
    lk = [r.randint(case["keys_shortest"], case["keys_longest"]) for _ in range(case["seqs"])]
    lk[r.randrange(len(lk))] = case["keys_longest"]
    return lq, lk


def allowed_pairs(case):
    """Scores that the mask leaves: a causal query sees the keys up to its own place, both ends aligned."""
    n = 0
    for q, k in zip(*lengths(case)):
        if not case["causal"]:
            n += q * k
        elif k >= q:
            n += q * (k - q) + q * (q + 1) // 2
        else:
            n += k * (k + 1) // 2
    return n


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    train = case["train"]
    if case["op"] == "attention":
        lq, lk = lengths(case)
        q = sum(lq) * case["heads"] * case["dim"]
        k = sum(lk) * case["kv_heads"] * case["dim"]
        products = 2 * case["dim"] * case["heads"] * allowed_pairs(case)
        return {"bytes": size * ((2 * q + 2 * k) + (2 * q + 2 * k if train else 0)), "flops": products * (7 if train else 2)}
    if case["op"] == "rotary":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": size * n * (4 if train else 2) + 4 * case["rows"] * (case["axes"].count(",") + 1), "flops": 3 * n * (2 if train else 1)}
    n = case["rows"] * case["width"]
    return {"bytes": size * n * (8 if train else 4), "flops": n * (40 if train else 14)}      # x, y -> u, h;  du, dh -> dx, dy


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    state = {"case": case}
    if case["op"] == "attention":
        lq, lk = lengths(case)
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        state.update(lq=torch.tensor(lq, device="cuda"), lk=torch.tensor(lk, device="cuda"), most_q=max(lq), most_k=max(lk), rows_q=sum(lq),
                     rows_k=sum(lk), q=normal(sum(lq), H, D), k=normal(sum(lk), KV, D), v=normal(sum(lk), KV, D))
        if case["train"]:
            state["do"] = normal(sum(lq), H, D)
        if own:      # the plan that a program makes with a batch and keeps for all its layers
            from crog_amd.packed import PackedRows
            state["rows"] = PackedRows(lq, lk if case["keys_longest"] else None, group=H // KV, causal=case["causal"], device="cuda")
    elif case["op"] == "rotary":
        parts = [int(p) for p in case["axes"].split(",")]
        T, H, KV, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
        state.update(q=normal(T, H, D), k=normal(T, KV, D), parts=parts,
                     positions=torch.randint(0, case["far"], (T, len(parts)), generator=g, device="cuda", dtype=torch.int32))
        if case["train"]:
            state.update(dq=normal(T, H, D), dk=normal(T, KV, D))
        if own:
            from crog_amd.packed import RotaryAxes
            state["axes"] = RotaryAxes(parts, theta=10000.0, interleaved=case["interleaved"], device="cuda")
    else:
        M, C = case["rows"], case["width"]
        state.update(x=normal(M, C, scale=2.0), y=normal(M, C, scale=0.7))
        weights = {}
        if case["post"]:
            weights["post_w"] = 1 + 0.2 * torch.randn(C, generator=g, device="cuda")
            if not case["rms"]:
                weights["post_b"] = 0.2 * torch.randn(C, generator=g, device="cuda")
        weights["gate"] = 0.5 * torch.randn(C, generator=g, device="cuda")
        weights["pre_w"] = 1 + 0.2 * torch.randn(C, generator=g, device="cuda")
        if not case["rms"]:
            weights["pre_b"] = 0.2 * torch.randn(C, generator=g, device="cuda")
        state.update(weights=weights, res_scale=0.9)
        if case["train"]:
            state.update(du=normal(M, C), dh=normal(M, C))
        if own:      # the weights as a model keeps them: parameters in a flat store with its gradient buffer
            from crog_amd.functional import WRef
            from crog_amd.runtime import ParamStore
            module = torch.nn.Module()
            for n, w in weights.items():
                module.register_parameter(n, torch.nn.Parameter(w.clone()))
            store = ParamStore(module, torch.device("cuda", torch.cuda.current_device()))
            state.update(module=module, store=store, refs={n: WRef(store, p, cols=1) for n, p in module.named_parameters()})
    return state


# ---- the calls of a user's program --------------------------------------------------------------------------------------------------------
def run_own(state):
    from crog_amd import functional as Fn
    case = state["case"]
    train = case["train"]
    if case["op"] == "attention":
        if not train:
            with torch.no_grad():
                return {"o": Fn.packed_attention(state["q"], state["k"], state["v"], state["rows"])}
        q, k, v = (state[n].detach().requires_grad_() for n in ("q", "k", "v"))
        o = Fn.packed_attention(q, k, v, state["rows"])
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "rotary":
        if not train:
            with torch.no_grad():
                q, k = Fn.rotary(state["q"], state["k"], state["positions"], state["axes"])
            return {"q": q, "k": k}
        a, b = (state[n].detach().requires_grad_() for n in ("q", "k"))
        q, k = Fn.rotary(a, b, state["positions"], state["axes"])
        da, db = torch.autograd.grad((q, k), (a, b), (state["dq"], state["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": da, "dk": db}
    r = state["refs"]
    post = (r["post_w"], r.get("post_b")) if case["post"] else None
    args = dict(post=post, gate=r["gate"], pre=(r["pre_w"], r.get("pre_b")), res_scale=state["res_scale"], eps=EPS, rms=case["rms"])
    if not train:
        with torch.no_grad():
            u, h = Fn.gated_norm(state["x"], state["y"], **args)
        return {"u": u, "h": h}
    state["store"].zero_grad()
    x, y = (state[n].detach().requires_grad_() for n in ("x", "y"))
    u, h = Fn.gated_norm(x, y, **args)
    dx, dy = torch.autograd.grad((u, h), (x, y), (state["du"], state["dh"]))
    return {"u": u.detach(), "h": h.detach(), "dx": dx, "dy": dy, "weights": {n: ref.grad() for n, ref in r.items()}}


# ---- the plain form -----------------------------------------------------------------------------------------------------------------------
def _padded(x, lens, most):
    """[rows, heads, dim] -> float32 [sequences, heads, most, dim]; places behind a sequence's end hold some row of the pack (masked later)."""
    starts = torch.cumsum(lens, 0) - lens
    at = (starts[:, None] + torch.arange(most, device=x.device)).clamp_(max=max(x.shape[0] - 1, 0))
    return x.float()[at].permute(0, 2, 1, 3).contiguous()


def _packed(x, lens, rows):
    """The inverse, of [sequences, heads, most, dim]."""
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=x.device), lens, output_size=rows)
    place = torch.arange(rows, device=x.device) - (torch.cumsum(lens, 0) - lens)[seq]
    return x[seq, :, place]


def plain_attention(state):
    case = state["case"]
    dt, KV, D = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    group = case["heads"] // KV
    lq, lk, mq, mk = state["lq"], state["lk"], state["most_q"], state["most_k"]
    n = lq.numel()
    scale = D ** -0.5
    # the heads of one group share a key head: their queries stand one behind the other in one product
    q = _padded(state["q"], lq, mq).view(n, KV, group * mq, D)
    k = _padded(state["k"], lk, mk)
    v = _padded(state["v"], lk, mk)
    i = torch.arange(mq, device=q.device)[None, :, None]
    j = torch.arange(mk, device=q.device)[None, None, :]
    allowed = (i < lq[:, None, None]) & (j < lk[:, None, None])
    if case["causal"]:
        allowed = allowed & (j <= i + (lk - lq)[:, None, None])
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(n, KV, group, mq, mk)
    s.masked_fill_(~allowed[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    p = s.div_(torch.where(total == 0, 1.0, total)).view(n, KV, group * mq, mk)
    o = torch.matmul(p, v)
    out = {"o": _packed(o.view(n, KV * group, mq, D), lq, state["rows_q"]).to(dt)}
    if not case["train"]:
        return out
    do = _padded(state["do"], lq, mq).view(n, KV, group * mq, D)
    out["dv"] = _packed(torch.matmul(p.transpose(2, 3).contiguous(), do), lk, state["rows_k"]).to(dt)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    out["dq"] = _packed(torch.matmul(ds, k).view(n, KV * group, mq, D), lq, state["rows_q"]).to(dt)
    out["dk"] = _packed(torch.matmul(ds.transpose(2, 3).contiguous(), q), lk, state["rows_k"]).to(dt)
    return {name: out[name] for name in ("o", "dq", "dk", "dv")}


def _turn(x, cos, sin, interleaved):
    """Rotates the first 2 * pairs columns of each head by the row's angles; the others stay."""
    pairs = cos.shape[-1]
    f = x.float()
    head, rest = f[..., :2 * pairs], f[..., 2 * pairs:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., :pairs], head[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def plain_rotary(state):
    case, parts = state["case"], state["parts"]
    sizes = torch.tensor(parts, device="cuda")
    axis = torch.repeat_interleave(torch.arange(len(parts), device="cuda"), sizes, output_size=sum(parts))
    place = torch.arange(sum(parts), device="cuda") - (torch.cumsum(sizes, 0) - sizes)[axis]
    step = 10000.0 ** (-place.double() / sizes[axis].double())
    angle = state["positions"][:, axis].double() * step      # 64 bits: far positions turn many times
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = {"q": _turn(state["q"], cos, sin, case["interleaved"]), "k": _turn(state["k"], cos, sin, case["interleaved"])}
    if case["train"]:
        out["dq"] = _turn(state["dq"], cos, -sin, case["interleaved"])
        out["dk"] = _turn(state["dk"], cos, -sin, case["interleaved"])
    return out


def _normed(f, rms):
    """(normalised rows, their 1 / deviation)"""
    if not rms:
        f = f - f.mean(-1, keepdim=True)
    inv = (f.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return f * inv, inv


def _normed_back(d, unit, inv, rms):
    d = d - unit * (d * unit).mean(-1, keepdim=True) - (0.0 if rms else d.mean(-1, keepdim=True))
    return d * inv


def plain_norm(state):
    case, w, rms = state["case"], state["weights"], state["case"]["rms"]
    dt, alpha = DTYPES[case["dtype"]], state["res_scale"]
    y = state["y"].float()
    z = y
    if case["post"]:
        y1, inv1 = _normed(y, rms)
        z = y1 * w["post_w"] + w.get("post_b", 0.0)
    u = alpha * state["x"].float() + w["gate"] * z
    u1, inv2 = _normed(u, rms)      # (of the sum itself, before it is rounded to be kept)
    h = (u1 * w["pre_w"] + w.get("pre_b", 0.0)).to(dt)
    out = {"u": u.to(dt), "h": h}
    if not case["train"]:
        return out
    dh = state["dh"].float()
    grads = {"pre_w": (dh * u1).sum(0)}
    if not rms:
        grads["pre_b"] = dh.sum(0)
    du = state["du"].float() + _normed_back(dh * w["pre_w"], u1, inv2, rms)
    grads["gate"] = (du * z).sum(0)
    dy = du * w["gate"]
    if case["post"]:
        grads["post_w"] = (dy * y1).sum(0)
        if not rms:
            grads["post_b"] = dy.sum(0)
        dy = _normed_back(dy * w["post_w"], y1, inv1, rms)
    out.update(dx=(alpha * du).to(dt), dy=dy.to(dt), weights=grads)
    return out


PLAIN = {"attention": plain_attention, "rotary": plain_rotary, "norm": plain_norm}


def run(state):
    return run_own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------------------------
def exact_attention(state):
    """One sequence and one query head at a time."""
    case = state["case"]
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    out = {"o": torch.zeros_like(q)}
    if case["train"]:
        do = state["do"].double()
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    q0 = k0 = 0
    for nq, nk in zip(*lengths(case)):
        a, b = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        if nq == 0 or nk == 0:
            continue
        hidden = torch.ones(nq, nk, dtype=torch.bool, device=q.device).tril(nk - nq).logical_not() if case["causal"] else None
        for h in range(case["heads"]):
            e = h // group
            x = (q[a, h] @ k[b, e].T) * scale
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            p = torch.softmax(x, 1)
            if hidden is not None:
                p = p.masked_fill(hidden, 0.0)      # (a row with nothing left: softmax made it NaN)
            o = p @ v[b, e]
            out["o"][a, h] = o
            if case["train"]:
                g = do[a, h]
                out["dv"][b, e] += p.T @ g
                ds = p * (g @ v[b, e].T - (g * o).sum(1, keepdim=True))
                out["dq"][a, h] = scale * (ds @ k[b, e])
                out["dk"][b, e] += scale * (ds.T @ q[a, h])
    return out


def exact_rotary(state):
    """Each pair as a complex number, multiplied by exp(i angle)."""
    case = state["case"]
    columns, n = [], 0
    for axis, size in enumerate(state["parts"]):
        for i in range(size):
            columns.append(state["positions"][:, axis].double() / 10000.0 ** (i / size))
        n += size
    angle = torch.stack(columns, 1)[:, None]
    unit = torch.polar(torch.ones_like(angle), angle)

    def turned(x, by):
        x = x.double().clone()
        first = slice(0, 2 * n, 2) if case["interleaved"] else slice(0, n)
        second = slice(1, 2 * n, 2) if case["interleaved"] else slice(n, 2 * n)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = {"q": turned(state["q"], unit), "k": turned(state["k"], unit)}
    if case["train"]:
        out.update(dq=turned(state["dq"], unit.conj()), dk=turned(state["dk"], unit.conj()))
    return out


def exact_norm(state):
    """Through autograd in float64."""
    case = state["case"]
    x, y = (state[n].double().requires_grad_() for n in ("x", "y"))
    w = {n: t.double().requires_grad_() for n, t in state["weights"].items()}

    def unit(t):
        if case["rms"]:
            return t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
        return (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + EPS)

    with torch.enable_grad():
        z = unit(y) * w["post_w"] + w.get("post_b", 0.0) if case["post"] else y
        u = state["res_scale"] * x + w["gate"] * z
        h = unit(u) * w["pre_w"] + w.get("pre_b", 0.0)
        out = {"u": u.detach(), "h": h.detach()}
        if case["train"]:
            names = list(w)
            g = torch.autograd.grad((u, h), [x, y] + [w[n] for n in names], (state["du"].double(), state["dh"].double()))
            out.update(dx=g[0], dy=g[1], weights=dict(zip(names, g[2:])))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": exact_attention, "rotary": exact_rotary, "norm": exact_norm}[case["op"]](state)
