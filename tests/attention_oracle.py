"""Softmax attention and its gradients in 64 bits, with the largest error that an implementation of a given precision may have at
every element (test infrastructure of test_gpu_attention.py).

With u the half step of the tensors' type (0 for fp32, whose own roundings are counted in e) and e the fp32 arithmetic's share:
  scores: a dot of dh products in fp32 is off by at most dh * 2^-24 * sum |q||k|, and exp((x - m)) by the error of its argument:
    e = 2^-24 * (2 dh X + 4 X + Sk + 64), X the largest scale * sum |q||k|
  o = sum_j p_j v_j / l:  p rounded to the type as a product's operand (u), o stored (u):  (u + 2 e) sum p|v| + u|o|
  dV: the same with dO
  dS = P (dP - delta):  operand rounding u|dS|;  delta is taken from the stored o, off by the line above times |dO|;  fp32 terms
  dQ, dK: scale * sum of dS's error times |k|, |q|, and the stored result's rounding
"""
import math

import torch


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def reference(q, k, v, mask=None, causal=False, scale=None, do=None, keep=None, p_drop=0.0):
    """q [N,Sq,H,d], k / v [N,Sk,G,d], mask [N,Sk], keep [N,H,Sq,Sk] 0/1 -> {name: (value, bound)} for o (and dq, dk, dv)"""
    u = half_step(q.dtype)
    N, Sq, H, d = q.shape
    Sk, G = k.shape[1:3]
    rep = H // G
    scale = 1 / math.sqrt(d) if scale is None else scale
    store = torch.float32 if q.dtype == torch.float32 else q.dtype
    st = torch.finfo(store).eps / 2 if q.dtype == torch.float32 else u
    out_shape_q, out_shape_k = (N, Sq, H, d), (N, Sk, G, d)
    q, k, v = (t.detach().double().permute(0, 2, 1, 3) for t in (q, k, v))
    ok = torch.ones(N, 1, Sq, Sk, dtype=torch.bool, device=q.device)
    if mask is not None:
        ok = ok & (mask != 0)[:, None, None, :]
        k = torch.where((mask != 0)[:, None, :, None], k, 0.0)
        v = torch.where((mask != 0)[:, None, :, None], v, 0.0)
    if causal:
        ok = ok & (torch.arange(Sk, device=q.device)[None] <= torch.arange(Sq, device=q.device)[:, None] + Sk - Sq)
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    x = scale * q @ k.transpose(-1, -2)
    X = float((scale * q.abs() @ k.abs().transpose(-1, -2)).max()) if x.numel() else 0.0
    e = 2.0 ** -24 * (2 * d * X + 4 * X + Sk + 64)
    x = x.masked_fill(~ok, -math.inf)
    m = x.amax(-1, keepdim=True) if Sk else x.new_zeros(N, H, Sq, 1)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    f = torch.ones_like(p) if keep is None else keep.double().to(p.device) / (1 - p_drop)
    pd = p * f
    o = pd @ v
    A = pd @ v.abs()
    to = lambda t: t.permute(0, 2, 1, 3)                          # noqa: E731
    got = {"o": (to(o), to((u + 2 * e) * A + st * o.abs()))}
    if do is None:
        return got
    g = do.detach().double().permute(0, 2, 1, 3)
    gv = g @ v.transpose(-1, -2)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (f * gv - delta)
    D = (g.abs() * (A + o.abs())).sum(-1, keepdim=True)
    B = p * (f * (g.abs() @ v.abs().transpose(-1, -2)) + D)
    tds = u * ds.abs() + p * (u + 2 * e) * D + 4 * e * B
    group = lambda t: t.view(N, G, rep, Sk, d).sum(2)             # noqa: E731
    dq = scale * ds @ k
    dk = group(scale * ds.transpose(-1, -2) @ q)
    dv = group(pd.transpose(-1, -2) @ g)
    er = e + 2.0 ** -24 * rep * Sq
    got["dq"] = (to(dq), to(scale * tds @ k.abs() + e * scale * ds.abs() @ k.abs() + st * dq.abs()))
    got["dk"] = (to(dk), to(group(scale * tds.transpose(-1, -2) @ q.abs() + er * scale * ds.abs().transpose(-1, -2) @ q.abs()) + st * dk.abs()))
    got["dv"] = (to(dv), to(group((u + 2 * er) * pd.transpose(-1, -2) @ g.abs()) + st * dv.abs()))
    assert got["dq"][0].shape == out_shape_q and got["dk"][0].shape == out_shape_k
    return got


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.detach().double() - value).abs()
    assert bool(torch.isfinite(got.double()).all()), name + ": not finite"
    over = off - bound - 1e-30
    if over.numel() and float(over.max()) > 0:
        at = int(over.argmax())
        raise AssertionError(f"{name}: off by {float(off.reshape(-1)[at]):.3g} at {at} where {float(bound.reshape(-1)[at]):.3g} is allowed "
                             f"(value {float(value.reshape(-1)[at]):.3g}); worst ratio {float((off / (bound + 1e-30)).max()):.3g}")
