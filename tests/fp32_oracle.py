"""fp32 attention over a few keys in 64 bits, with error bounds tight enough to see a part of an operand go missing
(test_gpu_sequence_edges.py, test_sequence_edges_cpu.py).

The kernels multiply fp32 numbers as three bf16 parts each, a = a0 + a1 + a2, cut off (not rounded) after 8 bits, so |a1| < 2^-7 and
|a2| < 2^-15 of a's leading power of two, and leave out a1 b2 + a2 b1 + a2 b2: less than 2^-21 |a b| (1 + 2^-8).  Of what is summed
each addition may cost 2^-23 of the sum of absolute values (a cut-off instead of a rounding inside the matrix unit): with n terms that are
not zero a product is off by

    c(n) = 2^-21 + 2^-29 + (n + 6) 2^-23     of the sum of absolute values

(the six partial products of a term are summed smallest first, so five of their additions are of sums below 2^-6 of it).  Then, with X the
sum scale * |q| |k| of a score and r its error relative to 1 after exp():
    r_j    = X_j c(d) + 2^-23 |x_j| + 3 2^-24 |x_j - m| + 2^-23      score, its scaling, the argument of exp2 (a difference, a constant, a
                                                                     product) and exp2 itself; the maximum m is the same number throughout
    rho_j  = r_j + sum_j p_j r_j + (Sk + 8) 2^-24 + 2^-22            p = exp() / l
    o      : sum p |v| (rho + c(Sk)) + 2^-23 |o|
    dP     : c(d) |dO| |v|          delta: |dO| err(o) + (d + 2) 2^-24 |dO| |o|
    dS     : |dS| (rho + 2^-22) + p (err(dP) + err(delta) + 2^-24 (|dP| + |delta|))
    dV     : sum p |dO| (rho + c(rows)) + 2^-23 |dV|
    dQ, dK : scale * sum (err(dS) + |dS| c(n)) |k|, |q|, and 2^-22 of the result (its scaling and storing)
each 2 % larger for the products of errors."""
import math

import torch


def c(n):
    return 2.0 ** -21 + 2.0 ** -29 + (n + 6) * 2.0 ** -23


def small_problem(spread, d, Sq, device):
    """positive operands (what is cut off then adds up instead of cancelling), two keys of which the second has hardly any value (so dS
    is as large as dP), one row with a gradient.  spread: the size of the queries"""
    g = torch.Generator().manual_seed(int(Sq * 100 + d * 10 + spread))
    r = lambda *s: 1 + torch.rand(*s, generator=g)                                       # noqa: E731
    N, Sk = 64, 2
    q, k, v, do = r(N, Sq, 1, d) * spread, r(N, Sk, 1, d), r(N, Sk, 1, d), torch.zeros(N, Sq, 1, d)
    v[:, 1] *= 2.0 ** -10
    do[:, Sq - 1] = r(N, 1, d)
    return tuple(t.to(device) for t in (q, k, v, do))


def reference(q, k, v, do, product=None):
    """one head, no mask -> {name: (value, bound)}.  product(site, A, B): stands in for A @ B (an implementation to be tried against the
    bounds); its results take the place of the values"""
    d, Sk = q.shape[3], k.shape[1]
    scale = 1 / math.sqrt(d)
    q, k, v, do = (t.detach().double()[:, :, 0] for t in (q, k, v, do))
    kt, vt = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    times = (lambda site, a, b: a @ b) if product is None else product
    rows = int((do != 0).any(-1).sum(1).max())
    x = scale * times("qk", q, kt)
    X = scale * q.abs() @ kt.abs()
    m = x.amax(-1, keepdim=True)
    p = torch.softmax(x, -1)
    r = X * c(d) + 2.0 ** -23 * x.abs() + 3 * 2.0 ** -24 * (x - m).abs() + 2.0 ** -23
    rho = r + (p * r).sum(-1, keepdim=True) + (Sk + 8) * 2.0 ** -24 + 2.0 ** -22
    o = times("pv", p, v)
    eo = (p * (rho + c(Sk))) @ v.abs() + 2.0 ** -23 * o.abs()
    dp, delta = times("dov", do, vt), (do * o).sum(-1, keepdim=True)
    ed = (do.abs() * eo).sum(-1, keepdim=True) + (d + 2) * 2.0 ** -24 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    es = ds.abs() * (rho + 2.0 ** -22) + p * (c(d) * (do.abs() @ vt.abs()) + ed + 2.0 ** -24 * (dp.abs() + delta.abs()))
    pt, st, et = (t.transpose(1, 2).contiguous() for t in (p, ds, es))
    dv, dq, dk = times("pdo", pt, do), scale * times("dsk", ds, k), scale * times("dsq", st, q)
    bounds = dict(o=eo, dv=(pt * (rho.transpose(1, 2) + c(rows))) @ do.abs() + 2.0 ** -23 * dv.abs(),
                  dq=scale * (es + ds.abs() * c(Sk)) @ k.abs() + 2.0 ** -22 * dq.abs(),
                  dk=scale * (et + st.abs() * c(rows)) @ q.abs() + 2.0 ** -22 * dk.abs())
    return {n: (t.unsqueeze(2), 1.02 * bounds[n].unsqueeze(2)) for n, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv))}
