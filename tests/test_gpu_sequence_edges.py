"""ops.attention, ops.linear_attention and ops.linear_attention_step at the edges of what their documentation allows: operands that share
memory between rows, precision that a lost part of an fp32 operand would show, gradients of some of the inputs, dropout beside a mask."""
import math

import pytest
import torch

import attention_oracle
import fp32_oracle
from attention_oracle import check
from helpers import keep_mask, relerr
import test_gpu_attention as A
import test_gpu_linear_attention as L

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from newsrec_hip import ops as _ops
    _ops.lib()
    return _ops


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("name", [0, 1, 2], ids=["q", "k", "v"])
@pytest.mark.parametrize("step", [0, 16], ids=["one row", "overlapping rows"])
@pytest.mark.parametrize("Sq", [75, 5])
def test_shared_rows_under_large_scores(ops, Sq, step, name, causal, dtype):
    """an operand whose rows share memory (position stride 0, or less than the row's width): behind its last row a tile holds more of
    the same memory, and scores past 88 overflow exp() there unless those rows count for nothing.  The same bits as from its copy"""
    N, H, d = 2, 2, 64
    ts = list(A.make(41, N, Sq, 75, H, H, d, dtype))
    ts[0] = (ts[0].float() * 80).to(dtype)               # scores of +-80 and more
    t = ts[name]
    S = t.shape[1]
    room = t.permute(0, 2, 1, 3).reshape(N, H, S * d)[:, :, :S * step + d].contiguous()
    shared = room.as_strided((N, S, H, d), (room.stride(0), step, room.stride(1), 1))
    got = []
    for x in (shared, shared.contiguous()):
        ts[name] = x
        got.append(A.run(ops, *ts, causal=causal))
    if name != 1:                                        # (one key row for all: its scores differ by the query alone)
        assert float((ts[0][0, :, 0].float() @ ts[1][0, :, 0].float().T).max()) / 8 > 89
    for n, a, b in zip(("o", "dq", "dk", "dv"), *got):
        assert bool(torch.isfinite(b.float()).all()), n
        assert torch.equal(a, b), n


def test_a_state_that_belongs_to_a_graph_is_not_written(ops):
    t, a = L.make(49, 2, 40, 2, 16, 24, F32), L.decays(2)
    q = t["q"].detach().requires_grad_(True)
    _, last = ops.linear_attention(q, t["k"], t["v"], a, state=t["state"].clone().requires_grad_(True))
    held = last.detach().clone()
    for out in (last, t["state"].clone().requires_grad_(True)):
        before = out.detach().clone()
        with pytest.raises(ops.NewsrecError, match="out_state.*gradient"):
            ops.linear_attention_step(t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], a, held, out_state=out)
        assert torch.equal(out.detach(), before)


@pytest.mark.parametrize("Sq", [3, 40], ids=["few rows", "rows"])
@pytest.mark.parametrize("d", [1, 2])
@pytest.mark.parametrize("spread", [1.0, 2.0 ** -6], ids=["scores", "weights"])
def test_fp32_operands_keep_all_their_bits(ops, spread, d, Sq):
    """problems so small that the error of fp32 arithmetic is a few units: operands cut to two bf16 parts leave the bounds of
    fp32_oracle.py in every product (test_sequence_edges_cpu.py)"""
    q, k, v, do = fp32_oracle.small_problem(spread, d, Sq, "cuda")
    want = fp32_oracle.reference(q, k, v, do)
    for name, t in zip(("o", "dq", "dk", "dv"), A.run(ops, q, k, v, do)):
        check(name, t, want[name])


@pytest.mark.parametrize("whole", [False, True], ids=["any", "whole numbers"])
@pytest.mark.parametrize("Sq", [3, 40, 200])
def test_a_single_key_is_handed_on(ops, Sq, whole):
    """one key: its probability is 1 and the output its value row, bit for bit; dV is the sum of dO, of which all but one row are zero.  The
    backward forms the score again and in another order: both are within X c(64) + 2^-23 |x| of it (fp32_oracle.py), the probability within
    the sum of that and exp's own 2^-23.  Where q and k are small whole numbers every order gives the same score, and dV is exact."""
    q, k, v, do = A.make(42, 3, Sq, 1, 4, 4, 64, F32)
    do[:, :Sq - 1] = 0
    if whole:
        q, k = (2 * q).round(), (2 * k).round()
    o, _, _, dv = A.run(ops, q, k, v, do)
    assert torch.equal(o, v.expand_as(o))
    if whole:
        assert torch.equal(dv, do[:, Sq - 1:])
        return
    x, X = (((f(q.double()) * f(k.double())).sum(-1, keepdim=True) / 8).abs()[:, Sq - 1:] for f in (lambda t: t, torch.abs))
    check("dv", dv, (do[:, Sq - 1:].double(), (2 * fp32_oracle.c(64) * X + 2.0 ** -22 * x + 2.0 ** -21) * do[:, Sq - 1:].double().abs()))


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("size", [(2, 200, 200, 12, 12, 25), (1, 300, 257, 4, 2, 64), (1, 130, 130, 2, 2, 128), (2, 5, 1500, 4, 2, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_fp32_meets_the_bars_of_the_short_kernels(ops, size, causal):
    """outputs 1e-5 and gradients 2e-5 in the maximum norm, as test_mhsa_past_the_short_kernels asks of the layers"""
    q, k, v, do = A.make(43, *size, F32)
    want = attention_oracle.reference(q, k, v, None, causal, do=do)
    for name, t in zip(("o", "dq", "dk", "dv"), A.run(ops, q, k, v, do, causal=causal)):
        assert relerr(t, want[name][0]) < (1e-5 if name == "o" else 2e-5), name


def steepest(f, noise, x, grad, h):
    """the derivative of f along its own gradient at x: (from the gradient, from central differences over h and h / 2 with the h^2 term
    taken out, how far the two may be apart).  noise: how far one value of f may be off"""
    r = grad / grad.double().norm().item()
    with torch.no_grad():
        far, near = ((f(x + s * r) - f(x - s * r)) / (2 * s) for s in (h, h / 2))
    slope = float((grad.double() * r.double()).sum())
    return slope, (4 * near - far) / 3, abs(near - far) / 3 + 3 * noise / h


@pytest.mark.parametrize("Sq", [3, 37], ids=["few rows", "rows"])
def test_attention_falls_as_its_gradients_say(ops, Sq):
    """central differences of the kernel's own forward along each gradient, where the slope is largest: a gradient 5 % too long or too
    short, or turned by as much as that takes off its length, is outside the tolerance"""
    size = (1, Sq, 9, 2, 1, 8)
    ts = A.make(44, *size, F32)
    got = A.run(ops, *ts)
    noise = float((attention_oracle.reference(*ts[:3])["o"][1] * ts[3].double().abs()).sum())
    for i, name in enumerate("qkv"):
        def f(x, i=i):
            return float((ops.attention(*ts[:i], x, *ts[i + 1:3]).double() * ts[3].double()).sum())
        slope, best, tol = steepest(f, noise, ts[i], got[1 + i], 0.25)
        assert tol < 0.05 * slope, (name, slope, tol)
        assert abs(best - slope) <= tol, (name, slope, best, tol)


@pytest.mark.parametrize("S", [9, 50])
def test_linear_attention_falls_as_its_gradients_say(ops, S):
    """the same of linear attention, whose outputs are linear in each operand: no h^2 term, so a long step"""
    t, a = L.make(45, 1, S, 2, 8, 6, F32), L.decays(2)
    got = L.run(ops, t, a)
    ref = L.reference(t["q"], t["k"], t["v"], a, None, t["state"])
    noise = float((ref["o"][1] * t["do"].double().abs()).sum() + (ref["last"][1] * t["dlast"].double().abs()).sum())
    for n in ("q", "k", "v", "state"):
        def f(x, n=n):
            now = {**t, n: x}
            o, last = ops.linear_attention(now["q"], now["k"], now["v"], a, state=now["state"])
            return float((o.double() * t["do"].double()).sum() + (last.double() * t["dlast"].double()).sum())
        # (at twice the step the sums over absolute values may be a few times larger than at t itself)
        slope, best, tol = steepest(f, 4 * noise, t[n], got["d" + n], 4.0)
        assert tol < 0.05 * slope, (n, slope, tol)
        assert abs(best - slope) <= tol, (n, slope, best, tol)


def subsets(names):
    return [[n for i, n in enumerate(names) if b >> i & 1] for b in range(1, 2 ** len(names) - 1)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_gradients_of_some_inputs(ops, dtype):
    """whichever inputs ask for a gradient, each gets the one it gets when all ask.  (Linear attention on bf16 tensors carries its state
    in three bf16 parts where the state's own gradient is asked for and in two where it is not: each compared with its like.)"""
    t = dict(zip(("q", "k", "v", "do"), A.make(46, 2, 70, 75, 4, 2, 64, dtype)))
    m = A.make_mask("prefix", 3, 2, 75)

    def grads(names):
        x = {n: t[n].detach().requires_grad_(n in names) for n in "qkv"}
        return dict(zip(names, torch.autograd.grad(ops.attention(*x.values(), key_mask=m), [x[n] for n in names], t["do"])))

    want = grads("qkv")
    for names in subsets("qkv"):
        for n, g in grads(names).items():
            assert torch.equal(g, want[n]), (names, n)
    t, a = L.make(47, 2, 90, 2, 32, 48, dtype), L.decays(2)
    lens = torch.tensor([90, 41], device="cuda")

    def grads(names):                                                                      # noqa: F811
        x = {n: t[n].detach().requires_grad_(n in names) for n in ("q", "k", "v", "state")}
        out = ops.linear_attention(x["q"], x["k"], x["v"], a, lens=lens, state=x["state"])
        return dict(zip(names, torch.autograd.grad(out, [x[n] for n in names], (t["do"], t["dlast"]))))

    every = {True: grads(["q", "k", "v", "state"]), False: grads(["q", "k", "v"])}
    for names in subsets(["q", "k", "v", "state"]):
        for n, g in grads(names).items():
            assert torch.equal(g, every["state" in names][n]), (names, n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("mask", ["prefix", "holes"])
@pytest.mark.parametrize("size", [(2, 40, 71, 2, 2, 25), (2, 130, 133, 4, 2, 64), (2, 3, 701, 2, 1, 64), (2, 50, 50, 2, 2, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_dropout_beside_a_mask(ops, size, mask, causal, dtype):
    """rows whose first probability is not the first of four numbers of the stream (Sk % 4 != 0), keys that are not there between them"""
    N, Sq, Sk, H, G, d = size
    q, k, v, do = A.make(48, *size, dtype)
    m = A.make_mask(mask, 5, N, Sk)
    keep = keep_mask((N, H, Sq, Sk), 0.1, 78, 5)
    want = attention_oracle.reference(q, k, v, m, causal, do=do, keep=keep, p_drop=0.1)
    for name, t in zip(("o", "dq", "dk", "dv"), A.run(ops, q, k, v, do, key_mask=m, causal=causal, p_drop=0.1, seed=78, site=5)):
        check(name, t, want[name])


@pytest.mark.parametrize("dh", [33, 40, 64])
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("hf", [False, True], ids=["additive", "excluded"])
def test_mhsa_whose_forward_alone_is_long(ops, dh, p, hf):
    """128 positions of more than 32 columns: too much LDS for the short forward, so the key-tiled one runs and leaves its statistics to the
    short kernels' backward.  Bars of test_mhsa_past_the_short_kernels"""
    N, S, H = 3, 128, 2
    g = torch.Generator().manual_seed(dh)
    qkv, dctx = torch.randn(N * S, 3 * H * dh, generator=g), torch.randn(N * S, H * dh, generator=g)
    mask = (torch.arange(S)[None] < torch.tensor([[S], [70], [0 if hf else 1]])).long()
    keep = keep_mask((N, H, S, S), p, 99, 3) if p else None
    x = qkv.double().requires_grad_(True)
    ref = A._mhsa_ref(x, mask, N, S, H, dh, keep, p, not hf)
    ref.backward(dctx.double())
    leaf = qkv.cuda().requires_grad_(True)
    ctx = ops.mhsa(leaf, mask.cuda(), N, S, H, dh, p, 99, 3, hf_mask=hf)
    (dqkv,) = torch.autograd.grad(ctx, (leaf,), dctx.cuda())
    assert relerr(ctx, ref) < 1e-5
    assert relerr(dqkv, x.grad) < 2e-5


# ----------------------------------------------------------------------------- calls that the documentation allows
@pytest.mark.parametrize("S,step", [(600, 1 << 22), (150, 1 << 24)], ids=["32-bit tiles", "64-bit tiles"])
def test_gradients_of_rows_far_apart(ops, S, step):
    """operands whose offsets pass 2^31 elements, with tiles that a 32-bit offset still spans and with wider ones: the same bits as from
    dense copies, forward and backward, and from linear attention with a length that ends inside"""
    room = torch.empty((S - 1) * step + 4096, dtype=BF16, device="cuda")
    dense = A.make(50, 1, S, S, 2, 2, 64, BF16)
    far = []
    for i, t in enumerate(dense[:3]):
        far.append(room.as_strided((1, S, 2, 64), (0, step, 64, 1), 512 * i))
        far[-1].copy_(t)
    m = A.make_mask("holes", 6, 1, S)
    for a, b in zip(A.run(ops, *far, dense[3], key_mask=m, causal=True), A.run(ops, *dense, key_mask=m, causal=True)):
        assert torch.equal(a, b)
    lens = torch.tensor([S - 7], device="cuda")
    got = []
    for q, k, v in (far, dense[:3]):
        t = dict(q=q, k=k, v=v, do=dense[3], state=None, dlast=None)
        got.append(L.run(ops, t, L.decays(2), lens, carried=False, both=False))
    for n in got[0]:
        assert torch.equal(got[0][n], got[1][n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(2, 5, 3001, 6, 2, 25), (1, 40, 2000, 2, 2, 33), (1, 700, 700, 4, 2, 128), (3, 70, 75, 2, 2, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_nothing_is_read_that_the_call_did_not_write(ops, size, dtype):
    """memory that the allocator hands out again holds NaN: workspaces, statistics and outputs are written before they are read"""
    q, k, v, do = A.make(51, *size, dtype)
    m = A.make_mask("prefix", 7, size[0], size[2])
    m[0] = 0
    want = A.run(ops, q, k, v, do, key_mask=m, causal=True, p_drop=0.1, seed=3)
    t, a = L.make(52, 1, size[2], 2, min(size[5], 64), 40, dtype), L.decays(2)
    lens = torch.tensor([size[2] // 2], device="cuda")
    rec = L.run(ops, t, a, lens)
    for _ in range(2):
        waste = [torch.full((1 << p,), math.nan, device="cuda") for p in range(6, 24) for _ in range(3)]
        del waste
        for x, y in zip(A.run(ops, q, k, v, do, key_mask=m, causal=True, p_drop=0.1, seed=3), want):
            assert torch.equal(x, y)
        waste = [torch.full((1 << p,), math.nan, device="cuda") for p in range(6, 24) for _ in range(3)]
        del waste
        for n, x in L.run(ops, t, a, lens).items():
            assert torch.equal(x, rec[n]), n


@pytest.mark.parametrize("S,dh", [(200, 25), (128, 64)])
def test_layer_core_captured_and_replayed(ops, S, dh):
    """ops.mhsa past the short kernels, forward and backward with dropout in one graph, replayed on new inputs"""
    N, H = 2, 4
    A_ = H * dh
    g = torch.Generator(device="cuda").manual_seed(53)
    draw = lambda: (torch.randn(N * S, 3 * A_, generator=g, device="cuda"), torch.randn(N * S, A_, generator=g, device="cuda"),      # noqa: E731
                    (torch.rand(N, S, generator=g, device="cuda") < 0.7).long())
    held = draw()

    def both(qkv, dctx, mask):
        leaf = qkv.detach().requires_grad_(True)
        ctx = ops.mhsa(leaf, mask, N, S, H, dh, 0.1, 7, 1)
        return (ctx.detach(),) + torch.autograd.grad(ctx, (leaf,), dctx)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*held)
    for _ in range(3):
        new = draw()
        for x, y in zip(held, new):
            x.copy_(y)
        want = both(*new)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_one_tensor_for_everything_and_saved_elsewhere(ops, dtype):
    """q, k and v one leaf, whose gradient is the sum of the three; two backward passes of one graph; and the saved tensors kept on the host"""
    x, _, _, do = A.make(54, 2, 90, 90, 4, 4, 40, dtype)
    parts_ = A.run(ops, x, x, x, do)
    leaf = x.detach().requires_grad_(True)
    o = ops.attention(leaf, leaf, leaf)
    (first,) = torch.autograd.grad(o, leaf, do, retain_graph=True)
    (again,) = torch.autograd.grad(o, leaf, do)
    assert torch.equal(first, again)
    # (autograd adds the three in some order of its own, each addition rounded to the type: two half steps of the absolute values)
    exact = sum(t.double() for t in parts_[1:])
    size = sum(t.double().abs() for t in parts_[1:])
    assert bool(((first.double() - exact).abs() <= 2.02 * torch.finfo(dtype).eps / 2 * size).all())
    with torch.autograd.graph.save_on_cpu():
        o = ops.attention(leaf, leaf, leaf)
        r, last = ops.linear_attention(leaf, leaf.expand(2, 90, 4, 40), leaf, L.decays(4))
    assert torch.equal(torch.autograd.grad(o, leaf, do)[0], first)
    assert bool(torch.isfinite(torch.autograd.grad(r, leaf, do)[0].float()).all())


def test_many_sequences(ops):
    """more workgroups than a 16-bit grid axis, sequences of a few tokens; the step over as many heads"""
    N, H, d = 40000, 2, 8
    q, k, v, do = A.make(55, N, 1, 3, H, H, d, F32)
    m = A.make_mask("prefix", 8, N, 3)
    want = attention_oracle.reference(q, k, v, m, do=do)
    for name, t in zip(("o", "dq", "dk", "dv"), A.run(ops, q, k, v, do, key_mask=m)):
        check(name, t, want[name])
    a, state = L.decays(H), torch.zeros(N, H, d, d, device="cuda")
    outs = [ops.linear_attention_step(k[:, i], k[:, i], v[:, i], a, state) for i in range(3)]
    o, last = ops.linear_attention(k, k, v, a)
    # both are within fp32's few roundings of the definition: dots of 8, sums of 3, a power's 2^-22
    size = (k.double().abs().sum(1).amax(-1) ** 2 * 3).amax() * v.abs().max()
    assert float((torch.stack(outs, 1) - o).abs().max()) <= 2.0 ** -20 * float(size)
    assert float((state - last).abs().max()) <= 2.0 ** -20 * float(size)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_a_long_record(ops, dtype):
    """100 003 tokens of one head in many segments, against the same record walked in four carried pieces and its last 300 tokens against the
    definition with the state that stood before them"""
    S, d = 100003, 32
    t, a = L.make(56, 1, S, 1, d, d, dtype), torch.tensor([-0.01], device="cuda")
    o, last = ops.linear_attention(t["q"], t["k"], t["v"], a)
    state, outs = None, []
    cuts = [0, 30000, 30001, 99703, S]
    for lo, hi in zip(cuts, cuts[1:]):
        before = state
        p, state = ops.linear_attention(t["q"][:, lo:hi], t["k"][:, lo:hi], t["v"][:, lo:hi], a, state=state)
        outs.append(p)
    tail = {n: t[n][:, -300:] for n in ("q", "k", "v")}
    want = L.reference(tail["q"], tail["k"], tail["v"], a, None, before)
    check("o of the pieces", outs[-1], want["o"])
    # the whole walk's state before the tail is another sum of the same tokens: memories of 100 tokens weigh 2^-150 after 10 400, so
    # both are within the bound of a record of that length (e = 2^-24 * 10 400 * 9 / 8 of the absolute values, u^3 of them for bf16)
    mem = L.reference(t["q"][:, -10400:], t["k"][:, -10400:], t["v"][:, -10400:], a)
    for name, x in (("o", o[:, -300:]), ("last", last)):
        value, bound = (y[:, -300:] if name == "o" else y for y in mem[name])
        check(name + " of the whole", x, (value, bound + 1e-30))
    check("last of the pieces", state, mem["last"])


@pytest.mark.parametrize("T", [160, 512])
def test_bert_past_128_positions(ops, T):
    """HipBertModel over long texts, one of them a single token, states and every gradient against the CPU oracle's.  Bars of
    test_layer_over_long_histories"""
    from models.modules.encoder import HipBertModel
    from oracle import twotower_oracle as O
    torch.manual_seed(T)
    plm = HipBertModel(dict(vocab_size=60, hidden_size=64, num_attention_heads=2, num_hidden_layers=2, intermediate_size=256,
                            max_position_embeddings=512, type_vocab_size=2, layer_norm_eps=1e-12, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0,
                            initializer_range=0.2))
    ids, lens = torch.randint(1, 60, (3, T)), torch.tensor([T, 1, T - 31])
    mask = (torch.arange(T)[None] < lens[:, None]).long()
    P = {"newsEncoder.plm." + k: v.detach().clone().double().requires_grad_(True) for k, v in plm.state_dict().items()}
    ref = O.bert_news_encoder(P, ids, mask, 2)[0]
    dy = torch.randn(3, T, 64)
    ref.backward(dy.double())
    plm = plm.cuda().train()
    out = plm(ids.cuda(), mask.cuda())
    out.backward(dy.cuda())
    assert relerr(out, ref) < 1e-5
    for n, p in plm.named_parameters():
        r = P["newsEncoder.plm." + n].grad
        if n.endswith("key.bias"):
            # exactly zero: a constant added to every key moves a row's scores alike.  What is left is the error of sum_j dK_j; that of the
            # weight's gradient, sum_j dK_j x_j, is of the same rows times x_j of mean square 1 (a LayerNorm's), so its size measures both.
            assert r.abs().max().item() < 1e-10
            assert p.grad.abs().max().item() <= 5e-5 * P["newsEncoder.plm." + n[:-4] + "weight"].grad.abs().max().item() + 1e-6, n
            continue
        assert (p.grad.cpu().double() - r).abs().max().item() <= 5e-5 * r.abs().max().item() + 1e-6, n
