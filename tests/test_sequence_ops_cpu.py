"""what can be checked of ops.attention / ops.linear_attention without a GPU: refusals before any device call, the layout of the
problem descriptions that cross the C boundary, and the workspace sizes the library asks for"""
import ctypes as C
import math

import pytest
import torch

from newsrec_hip import _lib, ops
from newsrec_hip._lib import NewsrecError


class CAttention(C.Structure):                                   # nr_attention, include/newsrec_hip.h
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k", "v", "key_mask")] + [(n, C.c_int64) for n in ("N", "Sq", "Sk", "H", "G", "dh")] +
                [(n, C.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride")] +
                [("dtype", C.c_int32), ("causal", C.c_int32), ("scale", C.c_float), ("p_drop", C.c_float), ("seed", C.c_uint64), ("site", C.c_uint32)])


class CLinear(C.Structure):                                      # nr_linear_attention
    _fields_ = ([(n, C.c_void_p) for n in ("q", "k", "v", "log_decay", "lens", "state")] + [(n, C.c_int64) for n in ("N", "S", "H", "dk", "dv")] +
                [(n, C.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride")] + [("dtype", C.c_int32), ("scale", C.c_float)])


ATTN = dict(q=16, k=16, v=16, mask=0, N=2, Sq=5, Sk=7, H=4, G=2, dh=16, strides=(1,) * 9, dtype=0, causal=0, scale=0.25, p_drop=0.0, seed=1, site=2)
LIN = dict(q=16, k=16, v=16, a=16, lens=0, state=0, N=2, S=5, H=4, dk=16, dv=24, strides=(1,) * 9, dtype=0, scale=0.25)


def attn(**kw):
    d = {**ATTN, **kw}
    return _lib.ATTENTION.pack(*(d[n] for n in ("q", "k", "v", "mask", "N", "Sq", "Sk", "H", "G", "dh")), *d["strides"],
                               *(d[n] for n in ("dtype", "causal", "scale", "p_drop", "seed", "site")))


def lin(**kw):
    d = {**LIN, **kw}
    return _lib.LINEAR_ATTENTION.pack(*(d[n] for n in ("q", "k", "v", "a", "lens", "state", "N", "S", "H", "dk", "dv")), *d["strides"], d["dtype"], d["scale"])


def test_packed_descriptions_have_the_header_s_layout():
    assert _lib.ATTENTION.size == C.sizeof(CAttention) and _lib.LINEAR_ATTENTION.size == C.sizeof(CLinear)
    p = CAttention.from_buffer_copy(attn(strides=tuple(range(1, 10)), dtype=1, causal=1, scale=0.5, p_drop=0.25, seed=2 ** 64 - 1, site=2 ** 32 - 1, mask=32))
    assert (p.q, p.key_mask, p.N, p.Sq, p.Sk, p.H, p.G, p.dh) == (16, 32, 2, 5, 7, 4, 2, 16)
    assert (list(p.q_stride), list(p.k_stride), list(p.v_stride)) == ([1, 2, 3], [4, 5, 6], [7, 8, 9])
    assert (p.dtype, p.causal, p.scale, p.p_drop, p.seed, p.site) == (1, 1, 0.5, 0.25, 2 ** 64 - 1, 2 ** 32 - 1)
    p = CLinear.from_buffer_copy(lin(strides=tuple(range(1, 10)), dtype=1, lens=32, state=48))
    assert (p.log_decay, p.lens, p.state, p.N, p.S, p.H, p.dk, p.dv, p.dtype, p.scale) == (16, 32, 48, 2, 5, 4, 16, 24, 1, 0.25)
    assert (list(p.q_stride), list(p.v_stride)) == ([1, 2, 3], [7, 8, 9])


ARG, UNSUPPORTED, WORKSPACE = 1, 2, 4


@pytest.mark.parametrize("kw,status", [(dict(G=3), ARG), (dict(H=0), ARG), (dict(dh=0), ARG), (dict(N=-1), ARG), (dict(dtype=2), ARG), (dict(p_drop=1.0), ARG),
                                       (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=math.nan), ARG), (dict(scale=math.inf), ARG),
                                       (dict(q=0), ARG), (dict(k=0), ARG), (dict(dh=129), UNSUPPORTED), (dict(Sk=1 << 31), UNSUPPORTED),
                                       (dict(Sq=1 << 30), UNSUPPORTED), (dict(N=1, Sk=100000), WORKSPACE)])
def test_attention_refuses_before_any_launch(kw, status):
    L = _lib.load()
    assert L.nr_attention_fwd(attn(**kw), 16, None, None, None, 0, None) == status
    assert b"attention" in L.nr_last_error()
    assert L.nr_attention_bwd(attn(**kw), 16, 16, 16, 16, 16, 16, 16, 16, None, 0, None) == status
    assert L.nr_attention_fwd(None, 16, None, None, None, 0, None) == ARG


def test_attention_refuses_missing_outputs():
    L = _lib.load()
    assert L.nr_attention_fwd(attn(), None, None, None, None, 0, None) == ARG
    assert L.nr_attention_fwd(attn(), 16, 16, None, None, 0, None) == ARG          # one of the two statistics
    assert L.nr_attention_bwd(attn(), 16, 16, 16, 16, None, 16, 16, 16, None, 0, None) == ARG
    assert L.nr_attention_bwd(attn(Sk=0), 16, 16, 16, 16, 16, 16, 16, 16, None, 0, None) == ARG
    assert L.nr_attention_fwd(attn(N=0), None, None, None, None, 0, None) == 0     # nothing to do


@pytest.mark.parametrize("kw,status", [(dict(H=0), ARG), (dict(dk=0), ARG), (dict(dv=0), ARG), (dict(S=-1), ARG), (dict(dtype=3), ARG), (dict(scale=math.nan), ARG),
                                       (dict(a=0), ARG), (dict(v=0), ARG), (dict(dk=129), UNSUPPORTED), (dict(dv=200), UNSUPPORTED), (dict(S=1 << 30), UNSUPPORTED),
                                       (dict(N=1, H=1, S=100000), WORKSPACE)])
def test_linear_attention_refuses_before_any_launch(kw, status):
    L = _lib.load()
    assert L.nr_linear_attention_fwd(lin(**kw), 16, 16, None, 0, None) == status
    assert b"linear_attention" in L.nr_last_error()
    assert L.nr_linear_attention_bwd(lin(**kw), 16, None, 16, 16, 16, None, None, 0, None) == status
    assert L.nr_linear_attention_fwd(lin(), 16, None, None, 0, None) == ARG
    assert L.nr_linear_attention_step(16, 16, 16, 16, None, 1, 1, 16, 16, 0, 1.0, 16, 16, None) == ARG
    assert L.nr_linear_attention_step(16, 16, 16, 16, 16, 1, 1, 129, 16, 0, 1.0, 16, 16, None) == UNSUPPORTED


def test_workspaces():
    """few rows over many keys are split (partial outputs and two statistics per row and split), a full grid is not"""
    L = _lib.load()
    assert L.nr_attention_fwd_ws_bytes(attn(N=32, Sq=512, Sk=512, H=12, G=12, dh=64)) == 0
    few = L.nr_attention_fwd_ws_bytes(attn(N=4, Sq=5, Sk=20011, H=12, G=4, dh=64, dtype=1))
    split = 4 * 4 * 15 * (64 + 2) * 4                                                 # N * G * rows of a key head * floats * bytes
    assert few % split == 0 and few // split in range(2, 79)                          # (down to 256 keys per split)
    assert L.nr_attention_bwd_ws_bytes(attn(N=32, Sq=512, Sk=512, H=12, G=12, dh=64)) == 0
    assert L.nr_attention_bwd_ws_bytes(attn(N=1, Sq=4001, Sk=4001, H=16, G=4, dh=128)) > 0
    assert L.nr_linear_attention_fwd_ws_bytes(lin(N=128, H=12, S=4000)) == 0
    long = L.nr_linear_attention_fwd_ws_bytes(lin(N=1, H=2, S=16384))
    assert long % (2 * 16 * 24 * 4) == 0 and long // (2 * 16 * 24 * 4) == 64          # segments of 256 tokens
    assert L.nr_attention_fwd_ws_bytes(attn(dh=129)) == 0                             # refused by the call itself


def test_ops_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 2, 16)
    with pytest.raises(NewsrecError, match="ROCm"):
        ops.attention(q, q, q)
    with pytest.raises(NewsrecError, match="ROCm"):
        ops.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(NewsrecError, match="ROCm"):
        ops.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 16, 16))
    with pytest.raises(NewsrecError, match="state"):
        ops.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), None)
