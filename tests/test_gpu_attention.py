"""ops.attention (softmax attention of any length, forward and backward) against the definition in 64 bits, with error bounds
derived per element (attention_oracle.py), and the layers that run on it past 128 positions."""
import math
import random

import pytest
import torch

from attention_oracle import check, reference
from helpers import keep_mask, relerr
from oracle import twotower_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from newsrec_hip import ops as _ops
    _ops.lib()
    return _ops


def make(seed, N, Sq, Sk, H, G, d, dtype, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)     # noqa: E731
    return r(N, Sq, H, d), r(N, Sk, G, d), r(N, Sk, G, d), r(N, Sq, H, d)


def make_mask(kind, seed, N, Sk):
    g = torch.Generator().manual_seed(seed)
    if kind == "none":
        return None
    if kind == "prefix":                        # padded sequences, the first of them empty
        lens = torch.randint(1, Sk + 1, (N,), generator=g)
        lens[0] = 0 if N > 1 else Sk
        m = torch.arange(Sk)[None] < lens[:, None]
    elif kind == "holes":
        m = torch.rand(N, Sk, generator=g) < 0.5
    elif kind == "last":                        # one key, the last
        m = torch.zeros(N, Sk, dtype=torch.bool)
        m[:, -1] = True
    elif kind == "nothing":
        m = torch.zeros(N, Sk, dtype=torch.bool)
    return m.long().cuda()


def run(ops, q, k, v, do, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = ops.attention(q, k, v, **kw)
    return (o,) + torch.autograd.grad(o, (q, k, v), do)


SIZES = [
    # N, Sq, Sk, H, G, d
    (2, 1, 1, 1, 1, 1), (3, 1, 50, 12, 12, 25), (2, 2, 3, 2, 1, 5), (2, 31, 33, 3, 3, 16), (1, 32, 32, 2, 2, 32), (2, 33, 31, 4, 2, 40),
    (1, 64, 64, 2, 2, 64), (2, 65, 63, 2, 1, 64), (1, 128, 128, 1, 1, 128), (2, 129, 127, 3, 1, 80), (2, 200, 200, 12, 12, 25),
    (1, 257, 300, 6, 2, 64), (1, 300, 257, 2, 2, 128), (1, 5, 1300, 6, 2, 64), (1, 1, 2100, 4, 4, 25), (1, 700, 7, 2, 1, 33),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("mask", ["none", "prefix", "holes"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(ops, size, mask, causal, dtype):
    q, k, v, do = make(sum(size), *size, dtype)
    m = make_mask(mask, 3, size[0], size[2])
    want = reference(q, k, v, m, causal, do=do)
    got = run(ops, q, k, v, do, key_mask=m, causal=causal)
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        assert t.dtype == dtype
        check(name, t, want[name])
    with torch.no_grad():                       # without the statistics for a backward: the same bits
        assert torch.equal(ops.attention(q, k, v, key_mask=m, causal=causal), got[0])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["last", "nothing"])
@pytest.mark.parametrize("size", [(2, 40, 130, 2, 2, 25), (2, 3, 900, 4, 2, 64), (1, 300, 300, 1, 1, 64)], ids=lambda s: "x".join(map(str, s)))
def test_one_key_and_no_key(ops, size, kind, dtype):
    q, k, v, do = make(5, *size, dtype)
    m = make_mask(kind, 0, size[0], size[2])
    got = run(ops, q, k, v, do, key_mask=m)
    if kind == "nothing":
        assert all(not bool(t.any()) for t in got)
        return
    want = reference(q, k, v, m, do=do)
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        check(name, t, want[name])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(2, 70, 200, 4, 2, 64), (2, 2, 1500, 4, 2, 25)], ids=lambda s: "x".join(map(str, s)))
def test_masked_rows_may_hold_anything(ops, size, dtype):
    q, k, v, do = make(6, *size, dtype)
    m = make_mask("holes", 1, size[0], size[2])
    want = run(ops, q, k, v, do, key_mask=m)
    k2, v2 = k.clone(), v.clone()
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min], device="cuda", dtype=dtype)
    away = (m == 0)
    k2[away] = bad[torch.randint(0, 5, k2[away].shape, device="cuda")]
    v2[away] = bad[torch.randint(0, 5, v2[away].shape, device="cuda")]
    for a, b in zip(run(ops, q, k2, v2, do, key_mask=m.bool()), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Sq", [3, 70])
@pytest.mark.parametrize("dtype,power", [(F32, 57), (BF16, 13)], ids=["fp32", "bf16"])
def test_scores_far_below_zero(ops, dtype, power, Sq):
    """every score the same and far below zero (fp32: -2^117, bf16: -2^29; powers of two, so exact): every key weighs 1 / Sk"""
    Sk, d = 300, 64
    _, _, v, do = make(15, 2, Sq, Sk, 2, 2, d, dtype)
    q = torch.full((2, Sq, 2, d), 2.0 ** power, device="cuda", dtype=dtype)
    k = torch.full((2, Sk, 2, d), -2.0 ** power, device="cuda", dtype=dtype)
    o, dq, dk, dv = run(ops, q, k, v, do)
    # sums of n terms in fp32 (n 2^-24 of their absolute values), for bf16 the weight as an operand and the result rounded (half a step each)
    u = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    mean = v.double().mean(1, keepdim=True).expand(2, Sq, 2, d)
    off = (o.double() - mean).abs()
    assert bool((off <= (u + (Sk + 8) * 2.0 ** -24) * v.double().abs().mean(1, keepdim=True) + (u + 2.0 ** -24) * mean.abs()).all())
    if dtype == F32:
        want = (do.double().sum(1, keepdim=True) / Sk).expand(2, Sk, 2, d)
        assert bool(((dv.double() - want).abs() <= (Sq + 8) * 2.0 ** -24 * do.double().abs().sum(1, keepdim=True) / Sk + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("d", [64, 25])
def test_strided_views_and_shared_storage(ops, d, dtype):
    """the blocks of one projection, a transposed [N,H,S,d] layout, rows of a larger buffer and an expanded key are read where
    they are: the same bits as from dense copies"""
    N, S, H = 2, 150, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(N, S, 3, H, d, generator=g, device="cuda").to(dtype)
    do = torch.randn(N, S, H, d, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.unbind(2)
    want = run(ops, *(t.contiguous() for t in (q, k, v)), do)
    leaf = qkv.detach().requires_grad_(True)
    o = ops.attention(*leaf.unbind(2))
    (dqkv,) = torch.autograd.grad(o, (leaf,), do)
    assert torch.equal(o, want[0])
    for i in range(3):
        assert torch.equal(dqkv[:, :, i], want[1 + i])
    heads = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    wide = torch.zeros(N, S + 9, H, d + 3, device="cuda", dtype=dtype)
    wide[:, 5:5 + S, :, 1:1 + d] = k
    for a, b in zip(run(ops, heads[0], wide[:, 5:5 + S, :, 1:1 + d], heads[2], do), want):
        assert torch.equal(a, b)
    # a gradient that autograd hands over expanded (the backward of a sum), and a key shared by the batch
    one = k[:1]
    leaf = one.detach().requires_grad_(True)
    (got,) = torch.autograd.grad(ops.attention(q, leaf.expand(N, S, H, d), v).float().sum(), (leaf,))
    full = one.expand(N, S, H, d).contiguous()
    dk = run(ops, q, full, v, torch.ones_like(do))[2]
    assert torch.equal(got, dk.sum(0, keepdim=True, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size,causal", [((2, 40, 70, 2, 2, 25), False), ((1, 130, 131, 4, 2, 64), True), ((1, 3, 700, 2, 1, 64), False)])
def test_dropout(ops, size, causal, dtype):
    N, Sq, Sk, H, G, d = size
    q, k, v, do = make(9, *size, dtype)
    keep = keep_mask((N, H, Sq, Sk), 0.25, 77, 4)
    want = reference(q, k, v, None, causal, do=do, keep=keep, p_drop=0.25)
    got = run(ops, q, k, v, do, causal=causal, p_drop=0.25, seed=77, site=4)
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        check(name, t, want[name])


def test_gradients_against_differences(ops):
    """the directional derivative of sum(o * do) from central differences of the kernel's own forward.  Error: the third
    derivative's share h^2 / 6 * |f'''| (checked by halving h) and the forward's fp32 noise over h."""
    size = (2, 37, 45, 4, 2, 20)
    q, k, v, do = make(11, *size, F32, std=0.5)
    got = run(ops, q, k, v, do)
    f = lambda q, k, v: float((ops.attention(q, k, v).double() * do.double()).sum())     # noqa: E731
    noise = float((reference(q, k, v)["o"][1] * do.double().abs()).sum())
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(3):
        r = torch.randn(got[1 + i].shape, generator=g, device="cuda") * 0.1
        with torch.no_grad():
            ends = {}
            for h in (1.0, 0.5):
                a = [q, k, v]
                lo, hi = list(a), list(a)
                hi[i], lo[i] = a[i] + h * r, a[i] - h * r
                ends[h] = (f(*hi) - f(*lo)) / (2 * h)
        slope = float((got[1 + i].double() * r.double()).sum())
        best = (4 * ends[0.5] - ends[1.0]) / 3                       # the h^2 term cancels
        assert abs(best - slope) <= abs(ends[0.5] - ends[1.0]) / 3 + 4 * noise, (i, best, slope, ends, noise)


@pytest.mark.parametrize("size", [(2, 300, 300, 4, 2, 64), (1, 4, 3000, 8, 2, 64)], ids=lambda s: "x".join(map(str, s)))
def test_same_bits_every_time_and_on_another_stream(ops, size):
    q, k, v, do = make(12, *size, BF16)
    m = make_mask("prefix", 2, size[0], size[2])
    want = run(ops, q, k, v, do, key_mask=m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(ops, q, k, v, do, key_mask=m)
    again = run(ops, q, k, v, do, key_mask=m)
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("size", [(2, 140, 140, 4, 4, 64), (1, 4, 2500, 8, 2, 64)], ids=lambda s: "x".join(map(str, s)))
def test_captured_and_replayed(ops, size):
    """forward and backward in one graph, replayed on new inputs with eager work between the replays"""
    q, k, v, do = make(13, *size, BF16)
    m = make_mask("prefix", 2, size[0], size[2])

    def both(q, k, v, do, m):
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = ops.attention(q, k, v, key_mask=m)
        return (o.detach(),) + torch.autograd.grad(o, (q, k, v), do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(q, k, v, do, m)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(q, k, v, do, m)
    for seed in (20, 21, 22):
        new = make(seed, *size, BF16)
        for a, b in zip((q, k, v, do), new):
            a.copy_(b)
        m.copy_(make_mask("holes", seed, size[0], size[2]))
        want = both(*new, m)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", [0, 1, 2], ids=["q", "k", "v"])
@pytest.mark.parametrize("size", [(2, 75, 75, 2, 2, 64), (2, 3, 1100, 4, 2, 32)], ids=lambda s: "x".join(map(str, s)))
def test_one_row_for_all_positions(ops, size, name, dtype):
    """an operand broadcast along the positions (stride 0), tiles that end inside a sequence: the same bits as its copy"""
    ts = list(make(19, *size, dtype))
    m = make_mask("prefix", 2, size[0], size[2])
    spread = ts[name][:, :1].expand(ts[name].shape)
    got = []
    for x in (spread, spread.contiguous()):
        ts[name] = x
        got.append(run(ops, *ts, key_mask=m, causal=size[1] == size[2]))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_two_graphs_do_not_share_scratch(ops):
    a, b = make(1, 1, 3, 3000, 4, 2, 64, BF16), make(2, 1, 3, 3000, 4, 2, 64, BF16)
    with torch.no_grad():
        want = [ops.attention(*t[:3]) for t in (a, b)]
        graphs, outs = [], []
        for t in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(ops.attention(*t[:3]))
        for _ in range(3):
            streams = [torch.cuda.Stream() for _ in graphs]
            for s, g in zip(streams, graphs):
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("seed", range(40))
def test_random_problems(ops, seed):
    """sizes, head layouts, masks, order, type and dropout drawn at random"""
    r = random.Random(seed)
    log = lambda hi: int(round(math.exp(r.uniform(0, math.log(hi)))))                    # noqa: E731
    G = r.choice([1, 2, 3])
    size = (log(4), log(300), log(600), G * r.choice([1, 2, 5]), G, r.choice([1, 3, 8, 16, 24, 25, 40, 64, 72, 96, 104, 127, 128]))
    dtype, causal, kind, p = r.choice([F32, BF16]), r.random() < 0.4, r.choice(["none", "prefix", "holes", "last"]), r.choice([0.0, 0.0, 0.3])
    q, k, v, do = make(seed, *size, dtype)
    m = make_mask(kind, seed, size[0], size[2])
    scale = r.choice([None, 0.3])
    keep = keep_mask((size[0], size[3], size[1], size[2]), p, seed, 1) if p else None
    want = reference(q, k, v, m, causal, scale=scale, do=do, keep=keep, p_drop=p)
    got = run(ops, q, k, v, do, key_mask=m, causal=causal, scale=scale, p_drop=p, seed=seed, site=1)
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        check(f"{name} {size} {dtype} causal={causal} mask={kind} p={p}", t, want[name])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size,causal", [((2, 3, 20011, 140, 140, 16), False), ((1, 40, 17000, 256, 256, 16), True)])
@pytest.mark.parametrize("kind", ["prefix", "holes"])
def test_masks_longer_than_one_span_of_key_bits(ops, size, causal, kind, dtype):
    """enough heads that the keys are not split: a workgroup walks more keys than it holds presence bits for at a time"""
    q, k, v, do = make(31, *size, dtype)
    m = make_mask(kind, 4, size[0], size[2])
    m[:, 9000:18000] = 0                         # a whole span without a key
    got = run(ops, q, k, v, do, key_mask=m, causal=causal)
    for h in range(0, size[3], 37):
        one = [t[:, :, h:h + 1] for t in (q, k, v, do)]
        want = reference(*one[:3], m, causal, do=one[3])
        for name, t in zip(("o", "dq", "dk", "dv"), got):
            check(name, t[:, :, h:h + 1], want[name])


def test_offsets_past_32_bits(ops):
    """rows of a cache whose offsets pass 2^31 elements"""
    Sk, step = 600, 1 << 22
    room = torch.empty((Sk - 1) * step + 4096, dtype=BF16, device="cuda")
    q, k, v, _ = make(3, 1, 2, Sk, 2, 2, 64, BF16)
    kk = room.as_strided((1, Sk, 2, 64), (0, step, 64, 1), 0)
    vv = room.as_strided((1, Sk, 2, 64), (0, step, 64, 1), 2048)
    kk.copy_(k)
    vv.copy_(v)
    with torch.no_grad():
        assert torch.equal(ops.attention(q, kk, vv), ops.attention(q, k, v))


def test_empty_axes(ops):
    for N, Sq, Sk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, do = make(1, N, Sq, Sk, 2, 2, 16, F32)
        got = run(ops, q, k, v, do)
        assert got[0].shape == (N, Sq, 2, 16) and all(not bool(t.any()) for t in got)


def test_refusals(ops):
    q, k, v, _ = make(1, 2, 4, 6, 4, 2, 16, F32)
    E = ops.NewsrecError
    mask = torch.ones(2, 6, dtype=torch.int64, device="cuda")
    for bad in (dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k.bfloat16()), dict(q=q[0]), dict(k=k[:, :5]), dict(v=v[..., :8]),
                dict(k=k[:1], v=v[:1]), dict(q=q[:, :, :3]), dict(q=q.cpu()), dict(key_mask=mask[:, :5]), dict(key_mask=mask.float()),
                dict(key_mask=mask.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(p_drop=1.0)):
        with pytest.raises(E):
            ops.attention(**{**dict(q=q, k=k, v=v), **bad})
    wide = torch.zeros(1, 2, 1, 129, device="cuda")
    with pytest.raises(E, match="128"):
        ops.attention(wide, wide, wide)
    leaf = q.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.attention(leaf, k, v).square().sum(), (leaf,), create_graph=True)
    with pytest.raises(RuntimeError):            # the backward itself has no derivative: an error, not a silent zero
        torch.autograd.grad(g.sum(), (leaf,))


# ----------------------------------------------------------------------------- the layers past 128 positions
def _mhsa_ref(qkv, mask, N, S, H, dh, keep, p, fill):
    A = H * dh
    q, k, v = [t.reshape(N, S, H, dh).permute(0, 2, 1, 3) for t in qkv.reshape(N, S, 3, A).unbind(2)]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(dh)
    x = x + (1 - mask)[:, None, None, :] * -1e5 if fill else x.masked_fill(mask[:, None, None, :] == 0, -math.inf)
    p_ = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    if keep is not None:
        p_ = p_ * keep.to(p_) / (1 - p)
    return torch.matmul(p_, v).permute(0, 2, 1, 3).reshape(N * S, A)


@pytest.mark.parametrize("N,S,H,dh", [(3, 129, 4, 25), (2, 200, 12, 25), (2, 512, 2, 64), (2, 100, 2, 128), (2, 160, 1, 7)])
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("hf", [False, True], ids=["additive", "excluded"])
def test_mhsa_past_the_short_kernels(ops, N, S, H, dh, p, hf):
    """the layer's attention core at lengths (and head dims) the short-sequence kernels refuse.  Bars: those of the short kernels
    (outputs 1e-5, gradients 2e-5 in the maximum norm).  A fully masked sequence of DIFFERENT tokens is ill-conditioned under the
    additive mask (scores near -1e5 are multiples of 2^-7); one of identical tokens is exactly uniform and held to the bar."""
    g = torch.Generator().manual_seed(8)
    A = H * dh
    qkv = torch.randn(N * S, 3 * A, generator=g)
    lens = torch.randint(1, S + 1, (N,), generator=g)
    mask = (torch.arange(S)[None] < lens[:, None]).long()
    qkv[:S] = qkv[0]
    mask[0] = 0
    dctx = torch.randn(N * S, A, generator=g)
    keep = keep_mask((N, H, S, S), p, 99, 3) if p > 0 else None
    qr = qkv.clone().double().requires_grad_(True)
    ref = _mhsa_ref(qr, mask, N, S, H, dh, keep, p, not hf)
    ref.backward(dctx.double())
    qg = qkv.cuda().requires_grad_(True)
    ctx = ops.mhsa(qg, mask.cuda(), N, S, H, dh, p, 99, 3, hf_mask=hf)
    (dq,) = torch.autograd.grad(ctx, (qg,), dctx.cuda())
    assert relerr(ctx, ref) < 1e-5
    assert relerr(dq[S:], qr.grad[S:]) < 2e-5
    if hf:
        assert not bool(dq[:S].any())
        return
    # the gradients of q and k vanish here (identical keys: the rows of dS sum to zero), so no share of the largest entry measures
    # them: what is left is delta's and dP's fp32 error, at most e * (2 D + 4 B) * scale * |k| per element (attention_oracle.py).
    # All scores of a row carry the same rounded -1e5, so its probabilities are those of the same sequence without a mask.
    q, k, v = (t.reshape(1, S, H, dh) for t in qkv[:S].reshape(S, 3, A).cuda().unbind(1))
    want = reference(q, k, v, do=dctx[:S].reshape(1, S, H, dh).cuda(), keep=None if keep is None else keep[:1], p_drop=p)
    for i, name in enumerate(("dq", "dk", "dv")):
        check(name, dq[:S].reshape(S, 3, A)[:, i].reshape(1, S, H, dh), want[name])


@pytest.mark.parametrize("train", [False, True])
def test_layer_over_long_histories(train):
    """one transformer layer over 200 clicks, forward and every gradient, against the CPU oracle's layer"""
    from models.modules.attention import TFMLayer
    torch.manual_seed(4)
    N, S, D, H = 2, 200, 48, 4
    layer = TFMLayer(D, H, 0.0)
    x = torch.randn(N, S, D)
    mask = torch.ones(N, S, dtype=torch.int64)
    mask[1, 77:] = 0
    P = {k: v.detach().clone().requires_grad_(True) for k, v in layer.state_dict().items()}
    xr = x.clone().requires_grad_(True)
    ref = O.tfm_layer(P, "", xr, mask, H)
    dy = torch.randn(N, S, D)
    ref.backward(dy)
    layer = layer.cuda().train(train)
    xg = x.cuda().requires_grad_(True)
    y = layer(xg, attention_mask=mask.cuda())
    y.backward(dy.cuda())
    assert relerr(y, ref) < 1e-5
    assert relerr(xg.grad, xr.grad) < 5e-5
    for n, p in layer.named_parameters():
        r = P[n].grad
        assert (p.grad.cpu() - r).abs().max().item() <= 5e-5 * r.abs().max().item() + 1e-6, n
