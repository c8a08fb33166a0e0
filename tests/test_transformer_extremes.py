"""Window attention at the ends of its types' range: values that count although their probability underflows, scores of any size, gradients
that 16 bits hold only scaled. On the host-side emulator and on the GPU."""
import math

import pytest
import torch

from gigagan_pytorch_amd import kernels as K
from gigagan_pytorch_amd import ops
from test_transformer_ops import DT, att_ref, gen, half_step, normal, qkv, seen, within

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)
# queries and keys for the forward kernels: many rows, few rows, few rows with the keys split over workgroups; on the GPU many rows with
# the keys split, and dk / dv in row chunks besides
SHAPES = [(34, 70), (3, 70), (1, 600)]
shapes = pytest.mark.parametrize('where,n,m', [('cpu', *s) for s in SHAPES]
                                 + [pytest.param('cuda', *s, marks=pytest.mark.gpu) for s in SHAPES + [(40, 2000), (300, 300)]])


@shapes
@pytest.mark.parametrize('fill', [math.nan, math.inf])
def test_a_value_of_underflowed_probability_counts(where, n, m, fill):
    """zero times NaN (or infinity) is NaN where the query sees the key, however small its probability; other features and the queries that do
    not see it have their values"""
    g = gen(20, where)
    q, k, v, _ = qkv(1, 2, 1, n, m, 32, 'bf16', g)
    q[..., 0], k[..., 0] = 16.0, 0.0
    at = m - 1 if n == 1 else m - 2                     # seen by the last query, or the last two
    k[0, 0, at] = 0
    k[0, 0, at, 0] = -64.0                              # a score 1024 below the others'
    kw = dict(scale=1.0, window=(None, 0))
    v2 = v.clone()
    v2[0, 0, at, 5] = fill
    got = ops.impl.window_attention(q, k, v2, **kw)
    sees = torch.arange(n) >= n - (m - at)
    assert not torch.isfinite(got[:, :, sees, 5]).any()
    others = [i for i in range(32) if i != 5]
    ref, tol = att_ref(q, k, v, 1.0, seen(1, n, m, (None, 0), 0, None, None, where))[0]
    within(got[..., others], ref[..., others], tol[..., others])
    within(got[:, :, ~sees], ref[:, :, ~sees], tol[:, :, ~sees])


def softmax_grads(q, k, v, do, scale, ok):
    """o, dq, dk, dv in 64 bits by automatic differentiation, masked rows zero"""
    q, k, v = (t.detach().double().requires_grad_() for t in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    x = q @ k.repeat_interleave(grp, 1).mT * scale
    x = x.masked_fill(~ok[:, None], -math.inf)
    some = ok.any(-1)[:, None, :, None]
    p = x.masked_fill(~some, 0.0).softmax(-1) * some
    o = p @ v.repeat_interleave(grp, 1)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), do.double())]


@shapes
@pytest.mark.parametrize('dtype,exponent', [('bf16', 21), ('bf16', 105), ('fp16', 21)])
@pytest.mark.parametrize('sign', [-1, 1])
def test_far_scores(where, n, m, dtype, exponent, sign):
    """scores of 2^21 and 2^105 on either side, far below and above where a running maximum might start: equal ones share the probability
    (exactly: the products are powers of two), one half as large in magnitude takes it all or has none, and so do the gradients"""
    g = gen(21, where)
    q, k, v, do = (t.clone() for t in qkv(1, 2, 1, n, m, 32, dtype, g))
    q.zero_()
    k.zero_()
    q[..., 3] = 2.0 ** (exponent // 2)
    k[..., 3] = sign * 2.0 ** (exponent - exponent // 2)
    k[0, 0, 7, 3] *= 0.5                                # the row's largest score below zero, one that does not count above
    window = (None, 0)
    ok = seen(1, n, m, window, 0, None, None, where)
    # numbers of the gradients' own size: dS k and dS q are up to 2^53 here
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = ops.impl.window_attention(*leaves, scale=1.0, window=window)
    got = [o, *torch.autograd.grad(o, leaves, do)]
    ref = softmax_grads(q, k, v, do, 1.0, ok)
    u = half_step(DT[dtype])
    P = (torch.where(ok[:, None], q.double() @ k.double().mT, torch.full((), -1e300, dtype=torch.float64, device=where))).softmax(-1) * ok[:, None]
    # the row's pass is fp32: 2^-18 covers its sums of up to 600 terms; o's own rounding is kept for D. The results are rounded once.
    e = 2.0 ** -18
    size = P * ((do.abs().double() @ v.abs().double().mT) + (do.abs().double() * (P @ v.abs().double())).sum(-1, keepdim=True))
    tol = [u * ref[0].abs() + e * (P @ v.abs().double()), u * ref[1].abs() + e * (size @ k.abs().double()),
           u * ref[2].abs() + e * (size.mT @ q.abs().double()).sum(1, keepdim=True),
           u * ref[3].abs() + e * (P.mT @ do.abs().double()).sum(1, keepdim=True)]
    # half's numbers below 2^-14 are 2^-24 apart: a result there is rounded by up to 2^-25, which is more than u of it
    step = 2.0 ** -25 if dtype == 'fp16' else 0.0
    for name, a, b, t in zip(('o', 'dq', 'dk', 'dv'), got, ref, tol):
        within(a, b, t + step, name)
    with torch.no_grad():
        assert torch.equal(ops.impl.window_attention(*leaves, scale=1.0, window=window), o)


@shapes
def test_scores_of_minus_infinity_alone(where, n, m):
    """a query whose seen keys all score -inf has 0 / 0 as in any softmax, one that sees no key zeros; a single finite score among them takes all"""
    g = gen(22, where)
    q, k, v, do = (t.clone() for t in qkv(3, 2, 1, n, m, 32, 'bf16', g))
    q[..., 0] = 1.0
    k[..., 0] = -math.inf
    mask = torch.ones((3, m), dtype=torch.bool, device=where)
    mask[1] = False
    k[2, 0, 0] = 0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = ops.impl.window_attention(*leaves, scale=0.5, key_mask=mask)
    assert torch.isnan(o[0]).all() and not o[1].any()
    within(o[2], v[2, :, :1].expand_as(o[2]), 0.0)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    assert torch.isnan(dq[0]).all() and torch.isnan(dk[0]).all() and torch.isnan(dv[0]).all()
    assert not any(t[1].any() for t in (dq, dk, dv))
    within(dv[2, 0, 0], do[2].double().sum((0, 1)), half_step(torch.bfloat16) * do[2].double().sum((0, 1)).abs() + 2.0 ** -18 * do[2].double().abs().sum((0, 1)))


@where
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('exponent', [0, -13, 9])
@pytest.mark.parametrize('shape', [(1, 2, 1, 64, 1024, 32, (None, None)), (1, 1, 1, 130, 130, 64, (None, 0)), (1, 2, 2, 40, 300, 128, (200, 0))])
def test_gradients_of_any_size(where, dtype, exponent, shape):
    """an incoming gradient of 2^-13 gives 2^-13 times the gradients of one, each rounded once to the result's type: nothing on the way is
    lost to half's subnormal numbers, or to its range with 2^9"""
    B, h, hk, n, m, d, window = shape
    dt = DT[dtype]
    q, k, v, do = qkv(B, h, hk, n, m, d, dtype, gen(23, where))
    if dtype == 'fp16' and exponent > 0:
        v = v * 2.0 ** -4                               # (results that half can hold)
        q, k = q * 0.5, k * 0.5
    small = (do * 2.0 ** exponent).to(dt)               # what half keeps of it is the gradient that is meant
    unit = small.double() * 2.0 ** -exponent
    ok = seen(B, n, m, window, 0, None, None, where)
    scale = d ** -0.5
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.impl.window_attention(*leaves, scale=scale, window=window), leaves, small)
    # the tolerance of a gradient of order one, scaled; half: half a subnormal step of the result besides
    step = 2.0 ** -25 if dtype == 'fp16' else 0.0
    for name, got, (ref, tol) in zip(('dq', 'dk', 'dv'), grads, att_ref(q, k, v, scale, ok, unit)[1:]):
        within(got, ref * 2.0 ** exponent, tol * 2.0 ** exponent + step, name)


@where
def test_half_rounds_gradients_once(where):
    """half with gradients of 1e-4 and 1e-3: the error of dq and dk, in relative L2, is at most twice that of the exact result rounded to half
    (P, dP's operands and dS carry relative roundings of their own)"""
    for size in (1e-4, 1e-3):
        q, k, v, do = qkv(1, 1, 1, 64, 1024, 32, 'fp16', gen(24, where))
        do = (do.float() * size).half()
        ref = softmax_grads(q, k, v, do, 32 ** -0.5, torch.ones(1, 64, 1024, dtype=torch.bool, device=where))[1:3]
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        got = torch.autograd.grad(ops.impl.window_attention(*leaves, scale=32 ** -0.5), leaves, do)[:2]
        for a, b in zip(got, ref):
            once = (b.half().double() - b).norm()
            assert (a.double() - b).norm() <= 2 * once + 2.0 ** -10 * b.norm()


@where
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_row_sums_from_the_unrounded_output(where, dtype):
    """D = dO.o is taken from o before its rounding. All scores are zero and 64 keys are seen, so P = 2^-6 is exact; o is near 8 and dP - D of order
    |dO|, and the keys share a mean that only sum_j dS_ij = 0 keeps out of dq: with o rounded in D rows would be twice over the tolerance"""
    g = gen(25, where)
    dt = DT[dtype]
    u, e = half_step(dt), 2.0 ** -24
    n, m, d = 64, 64, 32
    q = torch.zeros((1, 2, n, d), dtype=dt, device=where)
    k = normal((1, 1, m, d), dt, g, shift=64.0)
    v = normal((1, 1, m, d), dt, g, shift=8.0)
    do = normal((1, 2, n, d), dt, g)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    dq, = torch.autograd.grad(ops.impl.window_attention(*leaves, scale=1.0), leaves[:1], do)
    K, V, G = k.double(), v.double(), do.double()
    o = V.mean(2, keepdim=True).expand(1, 2, n, d)
    dP, D = G @ V.mT, (G * o).sum(-1, keepdim=True)
    dS = (dP - D) / m
    ref = dS @ K
    # o in two words is off by u^2 and by fp32's sum of 64 terms; the products' sums are fp32; dS is rounded once
    eD = (G.abs() * o.abs()).sum(-1, keepdim=True) * (u * u + (64 + d + 4) * e)
    eS = u * dS.abs() + (eD + (d + 4) * e * (G.abs() @ V.abs().mT)) / m + 2.0 ** -20 * dS.abs()
    within(dq, ref, eS @ K.abs() + 64 * e * (dS.abs() @ K.abs()) + u * ref.abs())
    rounded = (G * o.to(dt).double()).sum(-1, keepdim=True)
    lost = (rounded - D).abs() * K.mean(2, keepdim=True).abs()
    assert (lost > 2 * (eS @ K.abs())).any()            # what the case would show


@shapes
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_the_output_in_two_words(n, m, where, dtype):
    """o and what its rounding took off add up to o as fp32 had it, near a tie of the rounding too: scores of zero make P a constant and o a mean of
    up to 2000 values"""
    g = gen(26, where)
    dt = DT[dtype]
    q = torch.zeros((1, 2, n, 32), dtype=dt, device=where)
    k, v = normal((1, 1, m, 32), dt, g), normal((1, 1, m, 32), dt, g)
    o, o_lo, _ = K.window_fwd(q, k, v, 1.0, -1, 0, 0, None, None, True)
    seen_keys = torch.arange(m - n + 1, m + 1, device=where, dtype=torch.float64)[:, None]
    V = v.double()[0, 0]
    ref = (V.cumsum(0)[m - n:] / seen_keys).expand(1, 2, n, 32)
    size = (V.abs().cumsum(0)[m - n:] / seen_keys).expand(1, 2, n, 32)
    # the second word is rounded by u of it, which is u of o at most (half: by 2^-25 at least); sums of fp32 in tiles of 64, 1 / l and the product
    u = half_step(dt)
    tol = u * u * ref.abs() + (2.0 ** -25 if dtype == 'fp16' else 0.0) + (64 + m / 64 + 8) * 2.0 ** -24 * size
    within(o.double() + o_lo.transpose(1, 2).double(), ref, tol)
