"""ops.linear_attention (chunked, forward and backward) and ops.linear_attention_step against the recurrence's definition in 64
bits, with error bounds derived per element.

With u the half step of the tensors' type (0 for fp32), the bf16 kernel rounds as operands of its products: the decayed scores
(u |q.k| w |v|), or for tokens before the chunk the state where a query meets it (u |S|), and every contribution to the state to three
bf16 numbers, u^3 of it.  With M = the same sums over absolute values, o is therefore within (u + u^3 + e) M + (its own rounding) |o|,
a state within (u^3 + e) M.
e counts the fp32 arithmetic: dots of dk products, sums over S tokens (2^-24 each, worst case), a power's 2 units per chunk, and
the argument of a power, whose error 2^-23 |a n| matters only while w^n is not zero in fp32, |a n| < 150."""
import math
import random

import pytest
import torch

from attention_oracle import check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from newsrec_hip import ops as _ops
    _ops.lib()
    return _ops


def form(x, y, z, a, init, rev, amul, imul, umul):
    """one sequence, one head, 64 bits: (o, last), each as (value, sum of absolute values); conventions of the recurrence from
    either end"""
    L = x.shape[0]
    t = torch.arange(L, device=x.device, dtype=torch.float64)
    lag = (t[:, None] - t[None]) * (-1 if rev else 1)
    pw = lambda n: torch.where(n == 0, 1.0, torch.exp(a * n.clamp_min(0)))                 # noqa: E731  (-inf * 0 is not wanted)
    w = torch.where(lag >= 0, pw(lag), 0.0) * amul
    lead = pw(L - 1 - t if rev else t + 1)[:, None] * imul
    rest = pw(t + 1 if rev else L - 1 - t)[:, None] * umul
    whole = pw(torch.tensor(float(L), device=x.device, dtype=torch.float64))
    out = []
    for f in (lambda v: v, torch.abs):
        o = ((f(x) @ f(y).T) * w) @ f(z)
        s = (f(y) * rest).T @ f(z)
        if init is not None:
            o = o + lead * (f(x) @ f(init))
            s = s + whole * f(init)
        out.append((o, s))
    return (out[0][0], out[1][0]), (out[0][1], out[1][1])


def reference(q, k, v, log_decay, lens=None, state=None, scale=None, do=None, dlast=None):
    u = 0.0 if q.dtype == F32 else torch.finfo(q.dtype).eps / 2
    st = torch.finfo(q.dtype).eps / 2
    (N, S, H, dk), dv = q.shape, v.shape[3]
    scale = 1 / math.sqrt(dk) if scale is None else scale
    e = 2.0 ** -24 * (dk + dv + S + S / 8 + 300)
    D = lambda t: None if t is None else t.detach().double()                               # noqa: E731
    q, k, v, state, do, dlast, a = D(q), D(k), D(v), D(state), D(do), D(dlast), D(log_decay)
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)                   # noqa: E731
    got = {n: (z(N, S, H, d), z(N, S, H, d)) for n, d in (("o", dv), ("dq", dk), ("dk", dk), ("dv", dv))}
    got["last"], got["dstate"] = (z(N, H, dk, dv), z(N, H, dk, dv)), (z(N, H, dk, dv), z(N, H, dk, dv))

    def put(name, at, value, magnitude, rounds, own):
        got[name][0][at] = value
        got[name][1][at] = (rounds * u + u ** 3 + e) * magnitude + own * value.abs()

    for n in range(N):
        L = S if lens is None else max(0, min(S, int(lens[n])))
        for h in range(H):
            r, sl = (n, h), (n, slice(0, L), h)
            X, Y, Z = q[sl], k[sl], v[sl]
            s0 = None if state is None else state[r]
            o, last = form(X, Y, Z, a[h], s0, False, scale, scale, 1.0)
            put("o", sl, *o, 1, st)
            put("last", r, *last, 0, 2.0 ** -24)
            if do is None:
                continue
            g, gl = do[sl], None if dlast is None else dlast[r]
            turn = lambda t: None if t is None else t.T                                    # noqa: E731
            put("dq", sl, *form(g, Z, Y, a[h], turn(s0), False, scale, scale, 1.0)[0], 1, st)
            put("dk", sl, *form(Z, g, X, a[h], turn(gl), True, scale, 1.0, scale)[0], 1, st)
            dv_, ds = form(Y, X, g, a[h], gl, True, scale, 1.0, scale)
            put("dv", sl, *dv_, 1, st)
            put("dstate", r, *ds, 0, 2.0 ** -24)
    return got


def make(seed, N, S, H, dk, dv, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)                   # noqa: E731
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")                             # noqa: E731
    return dict(q=r(N, S, H, dk), k=r(N, S, H, dk), v=r(N, S, H, dv), do=r(N, S, H, dv), state=f(N, H, dk, dv), dlast=f(N, H, dk, dv))


def decays(H, kind="mixed"):
    if kind == "mixed":
        return -torch.exp(torch.linspace(math.log(1e-4), math.log(3.0), H, device="cuda")) if H > 1 else torch.tensor([-0.05], device="cuda")
    return torch.full((H,), {"none": 0.0, "fast": -60.0, "nothing kept": -math.inf}[kind], device="cuda")


def run(ops, t, a, lens=None, carried=True, both=True):
    q, k, v = (t[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    s = t["state"].detach().requires_grad_(True) if carried else None
    o, last = ops.linear_attention(q, k, v, a, lens=lens, state=s)
    leaves = (q, k, v) + ((s,) if carried else ())
    grads = torch.autograd.grad((o, last) if both else (o,), leaves, (t["do"], t["dlast"]) if both else (t["do"],))
    return dict(zip(("o", "last", "dq", "dk", "dv", "dstate"), (o, last) + grads))


SIZES = [(1, 1, 1, 1, 1), (2, 2, 3, 5, 7), (2, 31, 2, 16, 16), (1, 33, 3, 25, 25), (2, 63, 2, 32, 64), (2, 64, 2, 64, 32), (1, 65, 2, 64, 64),
         (2, 100, 12, 25, 25), (1, 128, 2, 128, 128), (2, 129, 1, 40, 80), (1, 200, 2, 128, 25), (1, 700, 3, 64, 64), (3, 1100, 2, 25, 128),
         (1, 2000, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("carried", [False, True], ids=["zero", "carried"])
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(ops, size, ragged, carried, dtype):
    N, S, H, dk, dv = size
    t, a = make(sum(size), *size, dtype), decays(H)
    lens = None
    if ragged:
        lens = torch.randint(0, S + 1, (N,), generator=torch.Generator().manual_seed(S)).cuda()
        lens[-1] = 0 if N > 1 else max(1, S - 1)
    want = reference(t["q"], t["k"], t["v"], a, lens, t["state"] if carried else None, do=t["do"], dlast=t["dlast"])
    got = run(ops, t, a, lens, carried)
    for name, x in got.items():
        check(name, x, want[name])
    with torch.no_grad():
        o, last = ops.linear_attention(t["q"], t["k"], t["v"], a, lens=lens, state=t["state"] if carried else None)
        assert torch.equal(o, got["o"]) and torch.equal(last, got["last"])


@pytest.mark.parametrize("seed", range(30))
def test_random_problems(ops, seed):
    """sizes, widths, lengths, type and decays drawn at random"""
    r = random.Random(seed)
    log = lambda hi: int(round(math.exp(r.uniform(0, math.log(hi)))))                      # noqa: E731
    wide = [1, 3, 8, 16, 24, 25, 40, 64, 72, 100, 128]
    size = (log(4), log(1500), log(5), r.choice(wide), r.choice(wide))
    dtype, carried = r.choice([F32, BF16]), r.random() < 0.5
    t = make(seed, *size, dtype)
    a = -torch.exp(torch.randn(size[2], generator=torch.Generator().manual_seed(seed)) * 2 - 2).cuda()
    lens = torch.tensor([r.randint(0, size[1]) for _ in range(size[0])]).cuda() if r.random() < 0.5 else None
    want = reference(t["q"], t["k"], t["v"], a, lens, t["state"] if carried else None, do=t["do"], dlast=t["dlast"])
    for name, x in run(ops, t, a, lens, carried).items():
        check(f"{name} {size} {dtype} carried={carried}", x, want[name])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "fast", "nothing kept"])
@pytest.mark.parametrize("S", [70, 900])
def test_extreme_decays(ops, S, kind, dtype):
    t, a = make(4, 2, S, 2, 32, 48, dtype), decays(2, kind)
    want = reference(t["q"], t["k"], t["v"], a, None, t["state"], do=t["do"], dlast=t["dlast"])
    for name, x in run(ops, t, a).items():
        check(name, x, want[name])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_without_the_last_states_gradient(ops, dtype):
    t, a = make(5, 2, 90, 2, 32, 32, dtype), decays(2)
    want = reference(t["q"], t["k"], t["v"], a, None, t["state"], do=t["do"])
    for name, x in run(ops, t, a, both=False).items():
        check(name, x, want[name])
    # ... and with that gradient alone
    q = t["q"].detach().requires_grad_(True)
    v = t["v"].detach().requires_grad_(True)
    _, last = ops.linear_attention(q, t["k"], v, a)
    dq, dv = torch.autograd.grad(last, (q, v), t["dlast"])
    assert not bool(dq.any())
    check("dv", dv, reference(t["q"], t["k"], t["v"], a, None, None, do=torch.zeros_like(t["do"]), dlast=t["dlast"])["dv"])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("S", [150, 1200])
def test_rows_behind_the_length_may_hold_anything(ops, S, dtype):
    N, H = 3, 2
    t, a = make(6, N, S, H, 32, 32, dtype), decays(H)
    lens = torch.tensor([S // 3, 0, S - 1], device="cuda")
    want = run(ops, t, a, lens)
    away = torch.arange(S, device="cuda")[None] >= lens[:, None]
    bad = dict(t)
    for n in ("q", "k", "v", "do"):
        bad[n] = t[n].clone()
        bad[n][away] = math.nan
    got = run(ops, bad, a, lens)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert not bool(want["o"][away].any()) and not bool(want["dq"][away].any()) and not bool(want["dk"][away].any())
    # a length outside [0, S] is taken into it
    assert torch.equal(run(ops, t, a, lens + torch.tensor([0, -5, S], device="cuda"))["o"], run(ops, t, a, torch.tensor([S // 3, 0, S], device="cuda"))["o"])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("d", [64, 25])
def test_strided_views(ops, d, dtype):
    N, S, H = 2, 140, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(N, S, 3, H, d, generator=g, device="cuda").to(dtype)
    a = decays(H)
    q, k, v = qkv.unbind(2)
    want = ops.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), a)
    turned = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    for args in ((q, k, v), turned):
        got = ops.linear_attention(*args, a)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    leaf = k[:1].detach().requires_grad_(True)               # a key shared by the batch
    (dk,) = torch.autograd.grad(ops.linear_attention(q, leaf.expand(N, S, H, d), v, a)[0].float().sum(), (leaf,))
    t = dict(q=q, k=k[:1].expand(N, S, H, d).contiguous(), v=v, do=torch.ones_like(q), state=None, dlast=None)
    assert torch.equal(dk, run(ops, t, a, carried=False, both=False)["dk"].sum(0, keepdim=True, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("S", [75, 1300])
def test_one_row_for_all_tokens(ops, S, name, dtype):
    """an operand broadcast along the tokens (stride 0), sequences that end inside a tile: the same bits as its copy"""
    N, H, d = 3, 2, 64
    t, a = make(17, N, S, H, d, d, dtype), decays(H)
    lens = torch.tensor([S, S - 9, 33], device="cuda")
    row = t[name][:, :1]

    def both(x):
        ops_in = {n: t[n].detach() for n in ("q", "k", "v")}
        ops_in[name] = x
        leaves = [ops_in[n].requires_grad_(True) for n in ("q", "k", "v")]
        o, last = ops.linear_attention(*leaves, a, lens)
        return (o, last) + torch.autograd.grad((o, last), leaves, (t["do"], torch.ones_like(last)))

    spread = row.detach().expand(N, S, H, d)
    for x, y in zip(both(spread), both(spread.contiguous())):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,H,dk,dv", [(1, 1, 1, 1), (3, 2, 5, 7), (2, 12, 25, 25), (5, 3, 64, 64), (2, 2, 128, 128), (3, 1, 16, 128), (2, 4, 100, 36)])
def test_step(ops, N, H, dk, dv, dtype):
    """one token.  Bound: the new state is one fused product and sum of fp32 operands and a decay known to 2^-22; the output a dot of
    dk terms, then stored."""
    g = torch.Generator(device="cuda").manual_seed(N + dk)
    q, k, v = (torch.randn(N, H, d, generator=g, device="cuda").to(dtype) for d in (dk, dk, dv))
    state = torch.randn(N, H, dk, dv, generator=g, device="cuda")
    a = decays(H)
    new = a.double().exp()[None, :, None, None] * state.double() + k.double()[..., None] * v.double()[..., None, :]
    size = state.double().abs() + (k.double().abs()[..., None] * v.double().abs()[..., None, :])
    scale = 1 / math.sqrt(dk)
    o = scale * (q.double()[..., None, :] @ new).squeeze(-2)
    mag = scale * (q.double().abs()[..., None, :] @ size).squeeze(-2)
    es = 2.0 ** -24 * (8 + 4 * 3.0)
    kept = state.clone()
    other = torch.empty_like(state)
    got = ops.linear_attention_step(q, k, v, a, state, out_state=other)
    assert torch.equal(state, kept)
    check("o", got, (o, (es + 2.0 ** -24 * (dk + 4)) * mag + torch.finfo(dtype).eps / 2 * o.abs()))
    check("state", other, (new, es * size))
    again = ops.linear_attention_step(q, k, v, a, state)              # in place
    assert torch.equal(again, got) and torch.equal(state, other)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("d", [25, 64])
def test_a_history_then_its_clicks(ops, d, dtype):
    """as a user tower has them: attention over the recent clicks and the recurrence over the whole record, whose state then takes
    new clicks one by one; the same outputs as the whole record at once (each side within its own bound of the definition)"""
    N, S, H, more = 3, 300, 4, 5
    t, a = make(8, N, S + more, H, d, d, dtype), decays(H)
    q, k, v = t["q"], t["k"], t["v"]
    want = reference(q, k, v, a)
    old, state = ops.linear_attention(q[:, :S], k[:, :S], v[:, :S], a)
    check("o", old, tuple(x[:, :S] for x in want["o"]))
    lens = torch.full((N,), S, device="cuda")
    padded, same = ops.linear_attention(q, k, v, a, lens=lens)        # the padded batch leaves the same state
    assert torch.equal(same, state) and torch.equal(padded[:, :S], old)
    for i in range(S, S + more):
        o = ops.linear_attention_step(q[:, i], k[:, i], v[:, i], a, state)
        check("step", o, tuple(x[:, i] for x in want["o"]))
    check("last", state, want["last"])
    rest, last = ops.linear_attention(q[:, S:], k[:, S:], v[:, S:], a, state=same)
    check("rest", rest, tuple(x[:, S:] for x in want["o"]))
    check("last", last, want["last"])
    near = ops.attention(q[:, S:], k[:, 150:], v[:, 150:], causal=True)      # the last clicks over a window, beside it
    assert near.shape == rest.shape and bool(torch.isfinite(near.float()).all())
    mix = (near.float() + rest.float()).sum()
    assert bool(torch.isfinite(mix))


@pytest.mark.parametrize("size", [(2, 200, 3, 64, 64), (1, 1500, 2, 32, 64)], ids=lambda s: "x".join(map(str, s)))
def test_captured_and_replayed(ops, size):
    t, a = make(9, *size, BF16), decays(size[2])
    lens = torch.full((size[0],), size[1] // 2, device="cuda")

    def both(t):
        return tuple(x.detach() for x in run(ops, t, a, lens).values())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(t)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(other, both(t)):
        assert torch.equal(x, y)                                      # another stream, and again: the same bits
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(t)
        stepped = ops.linear_attention_step(t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], a, held[1], out_state=torch.empty_like(held[1]))
    for seed in (30, 31, 32):
        new = make(seed, *size, BF16)
        for n in t:
            t[n].copy_(new[n])
        lens.fill_(seed * size[1] // 40)
        want = both(new)
        step = ops.linear_attention_step(new["q"][:, 0], new["k"][:, 0], new["v"][:, 0], a, want[1].clone())
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)
        assert torch.equal(stepped, step)


def test_gradients_against_differences(ops):
    """central differences of the kernel's own forward: o and the last state are linear in each of q, k, v and the starting state, so a
    difference has no truncation error and is off by the two evaluations' own error alone"""
    t, a = make(14, 2, 90, 2, 20, 24, F32), decays(2)
    got = run(ops, t, a)

    def f(**kw):
        x = {**t, **kw}
        o, last = ops.linear_attention(x["q"], x["k"], x["v"], a, state=x["state"])
        return float((o.double() * t["do"].double()).sum() + (last.double() * t["dlast"].double()).sum())

    ref = reference(t["q"], t["k"], t["v"], a, None, t["state"])
    noise = float((ref["o"][1] * t["do"].double().abs()).sum() + (ref["last"][1] * t["dlast"].double().abs()).sum())
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        for n in ("q", "k", "v", "state"):
            r = torch.randn(t[n].shape, generator=g, device="cuda")
            slope = float((got["d" + n].double() * r.double()).sum())
            assert abs((f(**{n: t[n] + r}) - f(**{n: t[n] - r})) / 2 - slope) <= 6 * noise, n


def test_empty_axes(ops):
    a = decays(2)
    for N, S in ((0, 5), (2, 0)):
        t = make(1, N, S, 2, 16, 24, F32)
        got = run(ops, t, a)
        assert got["o"].shape == (N, S, 2, 24)
        assert torch.equal(got["last"], t["state"]) and torch.equal(got["dstate"], t["dlast"])
    assert ops.linear_attention_step(*(torch.zeros(0, 2, d, device="cuda") for d in (16, 16, 24)), a, torch.zeros(0, 2, 16, 24, device="cuda")).shape == (0, 2, 24)


def test_refusals(ops):
    t, a = make(1, 2, 6, 3, 16, 24, F32), decays(3)
    base = dict(q=t["q"], k=t["k"], v=t["v"], log_decay=a)
    lens = torch.tensor([3, 6], device="cuda")
    E = ops.NewsrecError
    for bad in (dict(q=t["q"].half()), dict(k=t["k"].bfloat16()), dict(v=t["v"][:, :5]), dict(k=t["k"][..., :8]), dict(q=t["q"][0]), dict(v=t["v"].cpu()),
                dict(log_decay=a[:2]), dict(log_decay=a.double()), dict(log_decay=a.cpu()), dict(log_decay=a.clone().requires_grad_(True)),
                dict(lens=lens[:1]), dict(lens=lens.float()), dict(lens=lens.cpu()), dict(state=t["state"][:1]), dict(state=t["state"].bfloat16()),
                dict(scale=math.nan), dict(scale=math.inf)):
        with pytest.raises(E):
            ops.linear_attention(**{**base, **bad})
    wide = torch.zeros(1, 2, 3, 129, device="cuda")
    with pytest.raises(E, match="128"):
        ops.linear_attention(wide, wide, wide, a)
    one = dict(q=t["q"][:, 0], k=t["k"][:, 0], v=t["v"][:, 0], log_decay=a, state=t["state"])
    room = torch.zeros(t["state"].numel() + 8, device="cuda")
    for bad in (dict(state=None), dict(state=t["state"][:1]), dict(out_state=t["state"].bfloat16()), dict(out_state=t["state"][:1]), dict(q=t["q"]),
                dict(out_state=t["state"].transpose(2, 3).contiguous().transpose(2, 3)), dict(state=t["state"].transpose(2, 3).contiguous().transpose(2, 3)),
                dict(state=room[:-8].view_as(t["state"]), out_state=room[8:].view_as(t["state"]))):
        with pytest.raises(E):
            ops.linear_attention_step(**{**one, **bad})
    # a state that a graph has saved is not overwritten unnoticed
    s = t["state"].clone().requires_grad_(True)
    q = t["q"].detach().requires_grad_(True)
    o, _ = ops.linear_attention(q, t["k"], t["v"], a, state=s.detach().clone().requires_grad_(True))
    held = t["state"].clone()
    o, _ = ops.linear_attention(q, t["k"], t["v"], a, state=held)
    ops.linear_attention_step(t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], a, held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_step_where_a_gradient_would_be_expected(ops):
    t = make(18, 2, 1, 2, 16, 16, F32)
    q, k, v = (t[n][:, 0] for n in ("q", "k", "v"))
    a, state = decays(2), torch.zeros(2, 2, 16, 16, device="cuda")
    want = ops.linear_attention_step(q, k, v, a, state.clone())
    args = [q, k, v, state]
    for i in range(4):
        leaf = [x.clone().requires_grad_(i == j) for j, x in enumerate(args)]
        with pytest.raises(Exception, match="no gradient"):
            ops.linear_attention_step(*leaf[:3], a, leaf[3])
        assert not bool(leaf[3].any())
        with torch.no_grad():
            assert torch.equal(ops.linear_attention_step(*leaf[:3], a, leaf[3].detach()), want)
