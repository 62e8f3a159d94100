"""what ops.attention, ops.linear_attention and ops.linear_attention_step refuse before any device call, and the arithmetic behind the bounds
of test_gpu_sequence_edges.py"""
import math
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import fp32_oracle
from newsrec_hip import ops
from newsrec_hip._lib import NewsrecError


@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "state", "out_state"])
def test_forward_mode_is_refused(name):
    """a dual tensor has requires_grad == False: a call that looks at no more than that would hand back an output without a tangent"""
    r = lambda *s: torch.ones(*s)                                                          # noqa: E731
    whole = dict(q=r(1, 3, 2, 4), k=r(1, 3, 2, 4), v=r(1, 3, 2, 4))
    rec = dict(whole, log_decay=r(2), state=r(1, 2, 4, 4))
    step = dict({n: t[:, 0] for n, t in whole.items()}, log_decay=r(2), state=r(1, 2, 4, 4), out_state=r(1, 2, 4, 4))
    for op, args in ((ops.attention, whole), (ops.linear_attention, rec), (ops.linear_attention_step, step)):
        if name not in args:
            continue
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(NewsrecError, match="forward-mode"):
                op(**{**args, name: dual})
            with torch.no_grad(), pytest.raises(NewsrecError, match="forward-mode"):
                op(**{**args, name: dual})
        with pytest.raises(NewsrecError, match="forward-mode"):
            torch.func.jvp(lambda t: op(**{**args, name: t}), (args[name],), (torch.ones_like(args[name]),))
        with pytest.raises(NewsrecError, match="ROCm"):           # outside, the next check speaks
            op(**args)


def test_a_state_that_belongs_to_a_graph_is_not_written():
    """torch refuses a tensor that requires a gradient as an out= argument; so does the step, leaf or not"""
    r = lambda *s: torch.ones(*s)                                                          # noqa: E731
    args = dict(q=r(1, 2, 4), k=r(1, 2, 4), v=r(1, 2, 4), log_decay=r(2), state=r(1, 2, 4, 4))
    leaf = r(1, 2, 4, 4).requires_grad_(True)
    for held in (leaf, leaf * 2):
        with pytest.raises(NewsrecError, match="out_state.*gradient"):
            ops.linear_attention_step(**args, out_state=held)
        with torch.no_grad(), pytest.raises(NewsrecError, match="ROCm"):                   # as for out=, no_grad allows it
            ops.linear_attention_step(**args, out_state=held)


@pytest.mark.parametrize("scale", [1e39, 3.5e38, 1e300, math.inf, math.nan])
def test_a_scale_that_fp32_does_not_hold_is_refused(scale):
    x, one = torch.ones(1, 3, 2, 4), torch.ones(1, 2, 4)
    for s in (scale, -scale):
        for call in (lambda: ops.attention(x, x, x, scale=s), lambda: ops.linear_attention(x, x, x, torch.zeros(2), scale=s),
                     lambda: ops.linear_attention_step(one, one, one, torch.zeros(2), torch.zeros(1, 2, 4, 4), scale=s)):
            with pytest.raises(NewsrecError, match="scale"):
                call()
    for s in (0.0, -1.0, 1e-46):                             # (1e-46 is zero in fp32)
        with pytest.raises(NewsrecError, match="scale"):
            ops.attention(x, x, x, scale=s)


def test_a_scale_that_expects_a_gradient_is_refused():
    """float() of it would leave the gradient out"""
    x, one, scale = torch.ones(1, 3, 2, 4), torch.ones(1, 2, 4), torch.tensor(0.5, requires_grad=True)
    for call in (lambda s: ops.attention(x, x, x, scale=s), lambda s: ops.linear_attention(x, x, x, torch.zeros(2), scale=s),
                 lambda s: ops.linear_attention_step(one, one, one, torch.zeros(2), torch.zeros(1, 2, 4, 4), scale=s)):
        with pytest.raises(NewsrecError, match="scale.*no gradient"):
            call(scale)
        with pytest.raises(NewsrecError, match="ROCm"):
            call(scale.detach())


# sizes whose products or fp32-sized integers wrap: each in a process of its own, since what this refuses used to end it
HUGE = [("attention", dict(H=1 << 32, G=1 << 32, Sq=1)), ("attention", dict(H=1 << 62, G=1, Sq=8)), ("attention", dict(N=1 << 62, H=4, G=4)),
        ("attention", dict(N=1 << 40, H=1 << 24, G=1 << 24, Sq=1)), ("linear_attention", dict(N=1 << 62)), ("linear_attention", dict(N=1 << 31, H=4)),
        ("step", dict(N=1 << 62, H=4)), ("mhsa", dict(S=(1 << 32) + 5)), ("mhsa", dict(S=1 << 30)), ("mhsa", dict(H=1 << 32)), ("mhsa", dict(dh=(1 << 32) + 8))]


@pytest.mark.parametrize("what,kw", HUGE, ids=lambda x: x if isinstance(x, str) else "-".join(f"{n}{v}" for n, v in x.items()))
def test_sizes_past_the_kernels_integers_are_refused(what, kw):
    calls = {
        "attention": "L.nr_attention_fwd(d, 16, None, None, None, 0, None), L.nr_attention_bwd(d, 16, 16, 16, 16, 16, 16, 16, 16, None, 0, None), "
                     "2 * (L.nr_attention_fwd_ws_bytes(d) == 0), 2 * (L.nr_attention_bwd_ws_bytes(d) == 0)",
        "linear_attention": "L.nr_linear_attention_fwd(d, 16, 16, None, 0, None), L.nr_linear_attention_bwd(d, 16, None, 16, 16, 16, None, None, 0, None), "
                            "2 * (L.nr_linear_attention_fwd_ws_bytes(d) == 0), 2 * (L.nr_linear_attention_bwd_ws_bytes(d) == 0)",
        "step": "(L.nr_linear_attention_step(16, 16, 16, 16, 16, d['N'], d['H'], 16, 16, 0, 1.0, 16, 16, None),)",
        "mhsa": "L.nr_mhsa_fwd_f32(16, 16, 1, d['S'], d['H'], d['dh'], 0.0, 0, 0, 0, 16, 16, 16, None), "
                "L.nr_mhsa_bwd_f32(16, 16, 16, 16, 16, 16, 1, d['S'], d['H'], d['dh'], 0.0, 0, 0, 0, 16, None)",
    }
    made = {"attention": "t.attn(**kw)", "linear_attention": "t.lin(**kw)", "step": "kw", "mhsa": "{**dict(S=200, H=2, dh=16), **kw}"}
    here = os.path.dirname(os.path.abspath(__file__))
    code = (f"import sys; sys.path[:0] = [{os.path.dirname(here) + '/news-recommendation_amd'!r}, {here!r}]\nfrom newsrec_hip import _lib\n"
            f"import test_sequence_ops_cpu as t\nkw = {kw!r}\nd = {made[what]}\nL = _lib.load()\nprint(*({calls[what]}))")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, (got.returncode, got.stderr[-500:])
    assert set(got.stdout.split()) == {"2"}, got.stdout      # NR_ERR_UNSUPPORTED, and no workspace


# ----------------------------------------------------------------------------- fp32 numbers as bf16 parts
def parts(t, n):
    """what the kernels make of an fp32 number: n bf16 parts, each cut off after 8 bits"""
    rest, out = t.float().clone(), []
    for _ in range(n):
        cut = (rest.contiguous().view(torch.int32) & -65536).view(torch.float32)
        out.append(cut.double())
        rest = rest - cut
    return out


def split_product(a, b, n=3):
    """a @ b (64-bit sums) as the kernels form it: the partial products of the parts whose numbers add up to less than n"""
    x, y = parts(a, n), parts(b, n)
    return sum(x[i] @ y[j] for i in range(n) for j in range(n - i))


def test_what_three_parts_leave_out():
    """below 2^-21 of a product, one-sided, near 2^-24.5 on average"""
    a = torch.tensor([[1 + 2.0 ** -7 - 2.0 ** -23]])
    left = float((a.double() ** 2 - split_product(a, a)) / a.double() ** 2)
    assert 2.0 ** -21.2 < left < 2.0 ** -21                       # near the worst case
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(100000, 1, 1, generator=g) for _ in range(2))
    exact = x.double() @ y.double()
    left = (exact - split_product(x, y)) / exact
    assert bool((left >= 0).all()) and float(left.max()) < 2.0 ** -21
    assert 2.0 ** -25 < float(left.mean()) < 2.0 ** -24


SITES = ("qk", "pv", "dov", "pdo", "dsk", "dsq")


@pytest.mark.parametrize("Sq", [3, 40])
@pytest.mark.parametrize("d", [1, 2])
def test_the_fp32_bounds_see_a_lost_part(d, Sq):
    """operands of three parts stay within fp32_oracle's bounds in every product; cut to two in any one of them they do not"""
    seen = set()
    for spread in (1.0, 2.0 ** -6):
        q, k, v, do = fp32_oracle.small_problem(spread, d, Sq, "cpu")
        want = fp32_oracle.reference(q, k, v, do)
        off = lambda got: max(float(((got[n][0] - want[n][0]).abs() / want[n][1].clamp_min(1e-300)).max()) for n in want)    # noqa: E731
        assert off(fp32_oracle.reference(q, k, v, do, lambda site, a, b: split_product(a, b))) < 0.5
        for site in SITES:
            lost = lambda at, a, b: split_product(a, b, 2 if at == site else 3)           # noqa: E731
            if off(fp32_oracle.reference(q, k, v, do, lost)) > 1.5:
                seen.add(site)
    assert seen == set(SITES), seen
