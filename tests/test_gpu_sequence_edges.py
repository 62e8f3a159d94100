"""ops.attention, ops.linear_attention and ops.linear_attention_step at the edges of what their documentation allows: operands that share
memory between rows, precision that a lost part of an fp32 operand would show, gradients of some of the inputs, dropout beside a mask."""
import pytest
import torch

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
