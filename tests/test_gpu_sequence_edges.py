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
