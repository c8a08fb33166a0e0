"""The transformer operators - layer norm, rotary positions over several axes, attention with a sliding window and sinks - against plain
implementations in 64 bits, on the host-side emulator (small sizes) and on the GPU. Tolerances are counted from the operators' roundings:
u = eps / 2 of the result's type for every rounding to 16 bits (P and dS before their products, the result itself), 2^-24 per fp32
operation on the way, and stated per element."""
import math

import pytest
import torch

from gigagan_pytorch_amd import kernels as K
from gigagan_pytorch_amd import ops

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)
DT = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed, where):
    return torch.Generator(device=where).manual_seed(seed)


def normal(shape, dtype, g, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device=g.device, dtype=torch.float32) * scale + shift).to(dtype)


def within(got, ref, tol, what=''):
    """|got - ref| <= tol per element; NaN and infinities only where the reference has them"""
    got, ref = got.detach().double(), ref.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), (what, 'finite where the reference is not, or the reverse')
    d = torch.where(torch.isfinite(ref), (got - ref).abs(), torch.zeros_like(ref))
    tol = tol.expand_as(d) if torch.is_tensor(tol) else torch.full_like(d, tol)
    over = d > tol
    assert not over.any(), (what, int(over.sum()), float(d[over].max()), float((d / tol.clamp(min=1e-300))[over].max()))


# ---- layer norm -----------------------------------------------------------------------------------------------------

def ln_ref(x, w, b, eps, dy=None):
    """(y, dx, dw, db) in fp64 and the element-wise tolerances that fp32 arithmetic and one final rounding leave"""
    dt = x.dtype
    x, w = x.detach().double(), w.detach().double()
    b = torch.zeros_like(w) if b is None else b.detach().double()
    C = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    y = xh * w + b
    # fp32: a sum of C terms in a tree over chains of at most 32 terms is off by (32 + 14) 2^-24 of the terms' magnitudes; the mean
    # enters xh as it is, the variance halves into rstd; 8 more operations on the way
    e = 2.0 ** -24
    exh = (46 * x.abs().mean(-1, keepdim=True) + x.abs()) * e * rstd + xh.abs() * (46 + 8) * e
    # the mean's error shifts the squared differences' mean by its square only; rstd also takes d(var) / (2 var)
    u = half_step(dt) if dt != torch.float32 else 0.0
    ty = u * y.abs() + exh * w.abs() + 4 * e * (y.abs() + b.abs() + (xh * w).abs())
    out = [(y, ty)]
    if dy is not None:
        g = dy.double()
        gw = g * w
        c1, c2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
        dx = rstd * (gw - c1 - xh * c2)
        ec1 = 50 * e * gw.abs().mean(-1, keepdim=True)
        ec2 = 50 * e * (gw * xh).abs().mean(-1, keepdim=True) + (gw.abs() * exh).mean(-1, keepdim=True)
        tdx = u * dx.abs() + rstd * (ec1 + xh.abs() * ec2 + exh * c2.abs()) + (60 * e) * rstd * (gw.abs() + c1.abs() + (xh * c2).abs())
        f = lambda t: t.reshape(-1, C)
        rows = max(1, f(x).shape[0])
        # sums over the rows: chains of at most rows / (blocks) terms, then a tree; bounded by the number of rows
        n = min(rows, 4096) + 16
        dw, db = f(g * xh).sum(0), f(g).sum(0)
        tdw = n * e * f((g * xh).abs()).sum(0) + f(g.abs() * exh).sum(0)
        tdb = n * e * f(g.abs()).sum(0)
        out += [(dx, tdx), (dw, tdw), (db, tdb)]
    return out


def ln_check(x, w, b, eps, dy):
    x = x.detach().requires_grad_()
    w = w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    y = ops.impl.layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(g.dtype == t.dtype and g.shape == t.shape for g, t in zip(grads, leaves))
    ref = ln_ref(x, w, b, eps, dy)
    for name, got, (r, tol) in zip(('y', 'dx', 'dw', 'db'), (y, *grads), ref):
        within(got, r, tol, name)
    with torch.no_grad():
        assert torch.equal(ops.impl.layer_norm(x, w, b, eps), y)


LN_CPU = [(1, 1), (3, 2), (5, 7), (17, 8), (9, 127), (6, 128), (7, 129), (5, 512), (4, 513), (3, 1001), (3, 2048), (2, 2049), (2, 4097), (2, 8193)]
LN_GPU = LN_CPU + [(1, 16384), (2464, 512), (1031, 96), (70001, 24), (5003, 1001), (2049, 2048), (700, 16383)]


@pytest.mark.parametrize('rows,dim', LN_CPU)
@pytest.mark.parametrize('dtype', DT)
def test_layer_norm_cpu(rows, dim, dtype):
    g = gen(rows * 7 + dim, 'cpu')
    ln_check(normal((rows, dim), DT[dtype], g, 1.5, 0.3), normal(dim, torch.float32, g, 0.2, 1.0), normal(dim, torch.float32, g),
             1e-5, normal((rows, dim), DT[dtype], g))


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim', LN_GPU)
@pytest.mark.parametrize('dtype', DT)
def test_layer_norm_gpu(rows, dim, dtype):
    g = gen(rows * 7 + dim, 'cuda')
    ln_check(normal((rows, dim), DT[dtype], g, 1.5, 0.3), normal(dim, torch.float32, g, 0.2, 1.0), normal(dim, torch.float32, g),
             1e-5, normal((rows, dim), DT[dtype], g))


@where
def test_layer_norm_layouts(where):
    """no bias, weights of other types, a far mean, channel slices of a wider tensor, transposed and broadcast inputs and gradients, a
    view that starts at an odd element"""
    g = gen(1, where)
    w, b = normal(72, torch.float32, g, 0.2, 1.0), normal(72, torch.float32, g)
    dy = normal((2, 5, 72), torch.bfloat16, g)
    ln_check(normal((2, 5, 72), torch.bfloat16, g), w, None, 1e-3, dy)
    ln_check(normal((2, 5, 72), torch.float32, g, 1e-2, 1e2), w, b, 1e-5, dy.float())
    wide = normal((2, 5, 200), torch.bfloat16, g)
    ln_check(wide[..., 8:80], w, b, 1e-5, dy)
    ln_check(wide[..., 7:79], w, b, 1e-5, normal((2, 5, 200), torch.bfloat16, g)[..., 3:75])
    ln_check(normal((5, 2, 72), torch.bfloat16, g).transpose(0, 1), w, b, 1e-5, dy)
    ln_check(normal((2, 72, 5), torch.bfloat16, g).transpose(1, 2), w, b, 1e-5, dy)
    ln_check(normal((1, 1, 72), torch.bfloat16, g).expand(2, 5, 72), w, b, 1e-5, dy[:1, :1].expand(2, 5, 72))
    ln_check(normal((72,), torch.bfloat16, g), w, b, 1e-5, dy[0, 0])
    # 16-bit weights: the same values in fp32 give the same result, the gradients come in the weights' type
    x = normal((4, 72), torch.bfloat16, g).requires_grad_()
    wb = w.to(torch.bfloat16).requires_grad_()
    y = ops.impl.layer_norm(x, wb)
    assert torch.equal(y, ops.impl.layer_norm(x, wb.float()))
    assert torch.autograd.grad(y.float().sum(), wb)[0].dtype == torch.bfloat16


@where
def test_layer_norm_special_rows(where):
    """a constant row has its bias; NaN and infinities stay in their rows; no rows give no output and zero weight gradients"""
    g = gen(2, where)
    x = normal((6, 40), torch.float32, g)
    w, b = normal(40, torch.float32, g), normal(40, torch.float32, g)
    x[1] = 3.0
    clean = ops.impl.layer_norm(x, w, b)
    assert torch.equal(clean[1], b)
    bad = x.clone()
    bad[2, 3], bad[4, 39] = math.nan, math.inf
    y = ops.impl.layer_norm(bad, w, b)
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[2]).any() and not torch.isfinite(y[4]).any()
    x = torch.zeros((0, 40), device=where, requires_grad=True)
    w.requires_grad_()
    y = ops.impl.layer_norm(x, w, b)
    assert y.shape == (0, 40)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros_like(w))


@where
def test_layer_norm_gradient_by_differences(where):
    """dx against central differences of the fp64 definition's loss: the formula itself, not only its evaluation"""
    g = gen(3, where)
    x, w, b = normal((3, 24), torch.float32, g), normal(24, torch.float32, g), normal(24, torch.float32, g)
    dy = normal((3, 24), torch.float32, g)

    def loss(t):
        return (ln_ref(t, w, b, 1e-5)[0][0] * dy.double()).sum()
    xr = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.impl.layer_norm(xr, w, b), xr, dy)
    h = 1e-4
    for i, j in ((0, 0), (1, 11), (2, 23)):
        e = torch.zeros_like(x, dtype=torch.float64)
        e[i, j] = h
        num = (loss(x.double() + e) - loss(x.double() - e)) / (2 * h)
        # the differences' own error is h^2 times a third derivative of order 10; the kernel's 2^-20 of the terms' magnitude
        assert abs(float(num) - float(dx[i, j])) < 1e-6 + 2 ** -20 * float(dy.abs().sum())


# ---- rotary positions -------------------------------------------------------------------------------------------------

def rot_ref(x, positions, spec, inverse=False):
    freq = torch.tensor(spec.freqs, dtype=torch.float64, device=x.device)
    pos = positions if positions.dim() == 3 else positions[None]
    ang = pos.double()[..., spec.axes] * freq
    if inverse:
        ang = -ang
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    p = spec.pairs
    x = x.detach().double()
    y = x.clone()
    ia = torch.arange(p, device=x.device)
    ia, ib = (2 * ia, 2 * ia + 1) if spec.interleaved else (ia, ia + p)
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    size = torch.zeros_like(x)
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def rot_check(q, k, positions, spec):
    """forward and gradient; fp32 sines are off by 2^-23 or so (four units of 2^-24 each with the fraction's rounding: 2 pi 2^-25), the two
    products and their sum by 2^-24 each: 16 x 2^-24 of |a| + |b|, then one rounding to 16 bits"""
    q = q.detach().requires_grad_()
    k = None if k is None else k.detach().requires_grad_()
    out = ops.impl.rotary(q, positions, spec, k=k)
    outs, ins = ([out], [q]) if k is None else (list(out), [q, k])
    u = half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    g = gen(11, q.device.type)
    cot = [normal(o.shape, o.dtype, g) for o in outs]
    grads = torch.autograd.grad(outs, ins, cot)
    for x, o, ct, gr in zip(ins, outs, cot, grads):
        assert o.dtype == x.dtype and o.shape == x.shape and o.transpose(1, 2).is_contiguous()
        for got, src, inv in ((o, x, False), (gr, ct, True)):
            ref, size = rot_ref(src, positions, spec, inv)
            within(got, ref, u * ref.abs() + 16 * 2.0 ** -24 * size)
    return outs


def grid_positions(sizes, dev, dtype=torch.int32):
    axes = torch.meshgrid(*(torch.arange(s, device=dev) for s in sizes), indexing='ij')
    return torch.stack([a.flatten() for a in axes], -1).to(dtype)


@where
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('shared', [False, True])
@pytest.mark.parametrize('case', [(2, 3, 1, (7,), 16, (8,)), (1, 4, 2, (3, 5), 64, (16, 16)), (2, 2, 2, (2, 3, 4), 40, (3, 9, 5)),
                                  (1, 1, 1, (1,), 2, (1,)), (1, 5, 0, (2, 2, 9), 128, (16, 24, 24)), (2, 2, 1, (6,), 30, (11,)),
                                  (1, 3, 1, (4, 2), 20, (0, 10)), (1, 1, 1, (2,), 300, (128,))])
def test_rotary(where, dtype, interleaved, shared, case):
    b, h, hk, sizes, d, sections = case
    g = gen(5, where)
    n = math.prod(sizes)
    spec = ops.RotarySpec(sections, shared=shared, interleaved=interleaved)
    q = normal((b, h, n, d), DT[dtype], g)
    k = normal((b, hk, n, d), DT[dtype], g) if hk else None
    rot_check(q, k, grid_positions(sizes, where), spec)


@where
@pytest.mark.parametrize('pos_dtype', [torch.int32, torch.int64, torch.float32])
def test_rotary_positions_and_layouts(where, pos_dtype):
    """far and negative positions, fractions, positions per batch item, strided views of a fused projection and of the positions, many
    tokens a workgroup and a ragged last one"""
    g = gen(6, where)
    spec = ops.RotarySpec((10, 6), theta=500.0)
    b, n, h, hk, d = 2, 37, 3, 2, 48
    qk = normal((b, n, (h + hk) * d + 8), torch.bfloat16, g)
    q = qk[..., :h * d].unflatten(-1, (h, d)).transpose(1, 2)
    k = qk[..., h * d + 1:(h + hk) * d + 1].unflatten(-1, (hk, d)).transpose(1, 2)          # starts at an odd element
    pos = torch.randint(-5, 1 << 20, (b, n, 2), generator=g, device=where).to(pos_dtype)
    if pos_dtype == torch.float32:
        pos = pos + 0.25
    else:
        pos[0, 0, 0] = (1 << 30) + 1
    rot_check(q, k, pos, spec)
    rot_check(q, k, pos[1], spec)
    rot_check(q, None, pos.transpose(0, 2).contiguous().transpose(0, 2), spec)
    rot_check(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos, spec)
    rot_check(q[:1].expand(2, h, n, d), k, pos, spec)


@where
def test_rotary_properties(where):
    """position zero changes nothing, a turn and its opposite cancel, scores depend on position differences only, and the turn is
    differentiable twice"""
    g = gen(7, where)
    spec = ops.RotarySpec((8, 8))
    q, k = normal((1, 2, 6, 32), torch.float32, g), normal((1, 2, 6, 32), torch.float32, g)
    zero = torch.zeros((6, 2), dtype=torch.int32, device=where)
    assert torch.equal(ops.impl.rotary(q, zero, spec), q)
    pos = grid_positions((2, 3), where)
    y = ops.impl.rotary(q, pos, spec)
    back, _ = K.rotary(y, None, pos, spec, inverse=True)
    within(back, q, 64 * 2.0 ** -24 * q.abs().amax())
    a, b = ops.impl.rotary(q, pos, spec, k=k)
    c, d = ops.impl.rotary(q, pos + 1000, spec, k=k)
    s0, s1 = (x.double() @ z.double().mT for x, z in ((a, b), (c, d)))
    # 32 features of size <= 5: each score's terms are off by 32 x 2^-24 of |q||k|
    within(s1, s0, 64 * 2.0 ** -24 * float((q.abs().double() @ k.abs().double().mT).max()) * 2)
    q.requires_grad_()
    y = ops.impl.rotary(q, pos, spec)
    gr, = torch.autograd.grad((y ** 3).sum(), q, create_graph=True)
    gg, = torch.autograd.grad((gr ** 2).sum(), q)
    qd = q.detach().double().requires_grad_()
    c2, s2 = None, None
    freq = torch.tensor(spec.freqs, dtype=torch.float64, device=where)
    ang = (pos.double()[:, spec.axes] * freq)[None, None]
    yd = torch.cat((qd[..., :16] * ang.cos() - qd[..., 16:] * ang.sin(), qd[..., :16] * ang.sin() + qd[..., 16:] * ang.cos()), -1)
    grd, = torch.autograd.grad((yd ** 3).sum(), qd, create_graph=True)
    ggd, = torch.autograd.grad((grd ** 2).sum(), qd)
    within(gg, ggd, 2.0 ** -17 * float(ggd.abs().max()))        # ~ 60 fp32 operations of the largest magnitude


def test_rotary_spec_copies():
    import copy
    import pickle
    s = ops.RotarySpec((3, 4), theta=100.0, shared=True, interleaved=True)
    for t in (copy.deepcopy(s), pickle.loads(pickle.dumps(s))):
        assert (t.sections, t.theta, t.shared, t.interleaved, t.freqs, t.axes) == (s.sections, 100.0, True, True, s.freqs, s.axes)


# ---- window attention -----------------------------------------------------------------------------------------------

def seen(B, n, m, window, sinks, lengths, key_mask, dev):
    """(B, n, m) bool from the definition"""
    left, right = (m + n if t is None else t for t in window)
    L = torch.full((B,), m, device=dev) if lengths is None else lengths.long().clamp(0, m)
    p = (L[:, None] - n + torch.arange(n, device=dev))[:, :, None]
    j = torch.arange(m, device=dev)[None, None]
    ok = (j < L[:, None, None]) & (j <= p + right) & ((j >= p - left) | (j < sinks)) & (p >= 0)
    return ok if key_mask is None else ok & key_mask[:, None, :]


def att_ref(q, k, v, scale, ok, do=None):
    """(value, tolerance) of o and, with do, of dq, dk, dv: fp64, the tolerance element by element from the roundings"""
    dt = q.dtype
    u, e = half_step(dt), 2.0 ** -24
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0          # half a subnormal step of the rounded P and dS
    q, k, v = (t.detach().double() for t in (q, k, v))
    B, h, n, d = q.shape
    grp = h // k.shape[1]
    kk, vv = (t.repeat_interleave(grp, 1) for t in (k, v))
    see = ok[:, None].expand(B, h, n, -1)
    kk, vv = (torch.where(ok.any(1)[:, None, :, None], t, torch.zeros_like(t)) for t in (kk, vv))      # what nobody sees may be NaN
    x = (q @ kk.mT) * scale
    x = torch.where(see, x, torch.full_like(x, -1e300))
    mx = x.amax(-1, keepdim=True)
    P = torch.where(see, (x - mx).exp(), torch.zeros_like(x))
    z = P.sum(-1, keepdim=True)
    P = P / torch.where(z > 0, z, torch.ones_like(z))
    o = P @ vv
    # a score is off by (d + 4) roundings of its terms' magnitude and by those of its scaling and of the log-sum-exp it is taken
    # relative to; the exponential by 2^-21
    mag = (q.abs() @ kk.abs().mT) * scale
    es = e * ((d + 4) * torch.where(see, mag, torch.zeros_like(mag)) + 8 * torch.where(see, x.abs() + mx.abs(), torch.zeros_like(x))) + 2.0 ** -20
    # the row's own sum of exponentials carries the weighted mean of its entries' errors
    # (fp32 has no normal number below 2^-126: a probability beneath it may be lost)
    ep = P * (es + (P * es).sum(-1, keepdim=True)) + 64 * e * P + 2.0 ** -126 * see
    to = (u * P + ep + tiny) @ vv.abs() + u * o.abs() + tiny
    out = [(o, to)]
    if do is None:
        return out
    do = do.double()
    dP = do @ vv.mT
    D = (do * o).sum(-1, keepdim=True)
    dS = P * (dP - D)
    eD = (do.abs() * to).sum(-1, keepdim=True) + (d + 4) * e * (do * o).abs().sum(-1, keepdim=True)
    edP = (d + 4) * e * (do.abs() @ vv.abs().mT)
    edS = ep * (dP - D).abs() + P * (edP + eD) + u * dS.abs() + tiny * see
    dq, tq = scale * (dS @ kk), scale * (edS @ kk.abs())
    sh = (B, h // grp, grp)
    dk, tk = ((scale * (a.mT @ b)).unflatten(1, sh[1:]).sum(2) for a, b in ((dS, q), (edS, q.abs())))
    dv, tv = ((a.mT @ b).unflatten(1, sh[1:]).sum(2) for a, b in ((P, do), (u * P + ep + tiny * see, do.abs())))
    s32 = 64 * e                       # fp32 accumulation of long sums, relative to the terms (both sides of the chunk split)
    tq = tq + s32 * scale * (dS.abs() @ kk.abs())
    tk = tk + s32 * (scale * (dS.abs().mT @ q.abs())).unflatten(1, sh[1:]).sum(2)
    tv = tv + s32 * (P.mT @ do.abs()).unflatten(1, sh[1:]).sum(2)
    for val, tol in ((dq, tq), (dk, tk), (dv, tv)):
        out.append((val, tol + u * val.abs() + tiny))
    return out


def att_check(q, k, v, do=None, *, window=(None, None), sinks=0, lengths=None, key_mask=None, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ok = seen(q.shape[0], q.shape[2], k.shape[2], window, sinks, lengths, key_mask, q.device)
    kw = dict(scale=scale, window=window, sinks=sinks, lengths=lengths, key_mask=key_mask)
    if do is None:
        o = ops.impl.window_attention(q, k, v, **kw)
        within(o, *att_ref(q, k, v, scale, ok)[0], 'o')
        return o
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = ops.impl.window_attention(q, k, v, **kw)
    assert o.dtype == q.dtype and o.shape == q.shape and o.transpose(1, 2).is_contiguous()
    grads = torch.autograd.grad(o, (q, k, v), do)
    for name, got, (ref, tol) in zip(('o', 'dq', 'dk', 'dv'), (o, *grads), att_ref(q, k, v, scale, ok, do)):
        within(got, ref, tol, name)
    with torch.no_grad():
        assert torch.equal(ops.impl.window_attention(q, k, v, **kw), o)
    return (o, *grads)


def qkv(B, h, hk, n, m, d, dtype, g, scale=1.0):
    dt = DT[dtype]
    return (normal((B, n, h, d), dt, g, scale).transpose(1, 2), normal((B, m, hk, d), dt, g, scale).transpose(1, 2),
            normal((B, m, hk, d), dt, g).transpose(1, 2), normal((B, n, h, d), dt, g).transpose(1, 2))


# (B, h, hk, n, m, d, window, sinks): few rows and many, one token and one key, edges on and off the 32 / 64 / 128 tiles, grouped heads
ATT_CPU = [
    (1, 1, 1, 1, 1, 32, (None, None), 0),
    (1, 2, 1, 1, 77, 64, (None, 0), 0),
    (2, 2, 2, 5, 40, 32, (7, 0), 2),
    (1, 1, 1, 33, 33, 64, (None, 0), 0),
    (1, 3, 1, 50, 70, 32, (10, 3), 4),
    (1, 2, 2, 70, 70, 64, (0, 0), 0),
    (1, 1, 1, 40, 150, 128, (20, 5), 3),
    (1, 1, 1, 130, 64, 32, (None, None), 0),
    (1, 4, 1, 40, 200, 32, (5, 100), 130),
]
ATT_GPU = ATT_CPU + [
    (2, 8, 8, 78, 79, 64, (16, 16), 2),
    (1, 16, 2, 1, 8192, 64, (None, 0), 0),
    (3, 32, 8, 1, 5000, 128, (1023, 0), 4),
    (2, 8, 1, 4, 3001, 128, (500, 0), 1),
    (1, 4, 4, 1024, 1024, 64, (None, None), 0),
    (1, 6, 2, 777, 1291, 32, (100, 7), 3),
    (1, 2, 1, 2048, 2048, 128, (255, 0), 4),
    (1, 2, 1, 40, 8000, 64, (None, 0), 0),
    (1, 8, 8, 300, 4000, 128, (3000, 0), 5),
    (2, 2, 2, 500, 500, 64, (63, 64), 64),
    (1, 1, 1, 1500, 1500, 32, (3, 0), 200),
    (65, 1, 1, 17, 19, 64, (4, 2), 1),
    (128, 2, 2, 33, 130, 128, (70, 30), 2),             # eight waves a workgroup
    (2, 128, 128, 300, 700, 128, (200, 9), 3),
    (1, 64, 32, 1100, 1100, 128, (None, 0), 0),
]


def att_run(where, case, dtype):
    B, h, hk, n, m, d, window, sinks = case
    q, k, v, do = qkv(B, h, hk, n, m, d, dtype, gen(n + 3 * m, where))
    att_check(q, k, v, do, window=window, sinks=sinks)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('case', ATT_CPU)
def test_window_attention_cpu(case, dtype):
    att_run('cpu', case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('case', ATT_GPU)
def test_window_attention_gpu(case, dtype):
    att_run('cuda', case, dtype)


@where
@pytest.mark.parametrize('n', [1, 40])
def test_window_attention_lengths_and_masks(where, n):
    """unequal lengths (zero, shorter than the queries, all of the cache, beyond it), key masks with empty rows, both together; what no
    query sees holds NaN"""
    g = gen(9, where)
    B, h, hk, m, d = 5, 2, 1, 90, 32
    q, k, v, do = qkv(B, h, hk, n, m, d, 'bf16', g)
    lengths = torch.tensor([0, 17, m, 64, m + 5], dtype=torch.int32, device=where)
    mask = torch.rand((B, m), generator=g, device=where) < 0.6
    mask[3] = False
    for kw in (dict(lengths=lengths), dict(key_mask=mask), dict(lengths=lengths.long(), key_mask=mask, window=(6, 2), sinks=3),
               dict(lengths=lengths, window=(9, 0), sinks=1)):
        ok = seen(B, n, m, kw.get('window', (None, None)), kw.get('sinks', 0), kw.get('lengths'), kw.get('key_mask'), where)
        dead = ~ok.any(1)                                     # (B, m)
        for fill in (math.nan, math.inf):
            k2, v2 = (torch.where(dead[:, None, :, None], torch.full_like(t, fill), t) for t in (k, v))
            out = att_check(q, k2, v2, do, **kw)
            empty = ~ok.any(2)                                # (B, n)
            for t in out[:2]:
                assert not t.transpose(1, 2)[empty].any()
            for t in out[2:]:
                assert not t.transpose(1, 2)[dead].any()


@where
def test_window_attention_nan_padding_rows(where):
    """queries of padding (negative positions, items without keys) may hold NaN: their rows are zeros and their keys' gradients clean"""
    g = gen(10, where)
    q, k, v, do = qkv(3, 2, 2, 40, 50, 32, 'bf16', g)
    lengths = torch.tensor([50, 11, 0], dtype=torch.int32, device=where)
    pad = torch.arange(40, device=where)[None] < (40 - lengths[:, None])
    q2, do2 = (torch.where(pad[:, None, :, None], torch.full_like(t, math.nan), t) for t in (q, do))
    got = [t.detach() for t in att_check(q, k, v, do, lengths=lengths)]
    q2, k2, v2 = (t.detach().requires_grad_() for t in (q2, k, v))
    o = ops.impl.window_attention(q2, k2, v2, scale=32 ** -0.5, lengths=lengths)
    for a, b in zip(got, (o, *torch.autograd.grad(o, (q2, k2, v2), do2))):
        assert torch.equal(a, b)


@where
def test_window_attention_layouts(where):
    """one fused projection, head-major and batch-broadcast tensors, views that are not 16-byte aligned, gradients with zero strides: all
    give the bits of the dense layout"""
    g = gen(12, where)
    B, h, hk, n, d = 2, 4, 2, 40, 32
    x = normal((B, n, (h + 2 * hk) * d + 4), torch.bfloat16, g)
    kw = dict(scale=0.2, window=(8, 4), sinks=1)
    for off in (0, 4, 3):
        q, k, v = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in x[..., off:off + (h + 2 * hk) * d].split([h * d, hk * d, hk * d], -1)) \
            if off != 3 else (t.transpose(1, 2).contiguous().transpose(1, 2).transpose(1, 2).contiguous().transpose(1, 2)
                              for t in qkv(B, h, hk, n, n, d, 'bf16', g)[:3])
        do = normal((B, h, 1, 1), torch.bfloat16, g).expand(B, h, n, d)
        a = [t.detach().requires_grad_() for t in (q, k, v)]
        b = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, v)]
        oa, ob = (ops.impl.window_attention(*t, **kw) for t in (a, b))
        assert torch.equal(oa, ob)
        for s, t in zip(torch.autograd.grad(oa, a, do), torch.autograd.grad(ob, b, do.contiguous())):
            assert torch.equal(s, t)
    q, k, v, do = qkv(1, 2, 1, 9, 30, 64, 'bf16', g)
    att_check(q.expand(3, 2, 9, 64), k.expand(3, 1, 30, 64), v.expand(3, 1, 30, 64), do.expand(3, 2, 9, 64), window=(5, 5))


@where
def test_window_attention_large_scores(where):
    """scores of hundreds: probabilities of one and zero, running maxima that move"""
    g = gen(13, where)
    q, k, v, do = qkv(1, 2, 1, 40, 200, 64, 'bf16', g, scale=6.0)
    att_check(q, k, v, do, scale=1.0, window=(150, 0), sinks=2)
    q, k, v, _ = qkv(1, 2, 1, 2, 200, 64, 'bf16', g, scale=6.0)
    att_check(q, k, v, scale=1.0)


@where
def test_window_attention_nan_reaches_only_who_sees_it(where):
    """a NaN or infinite key or value reaches the queries that see it and no other row of the same tile; a NaN query or gradient reaches
    the keys it sees and no other key of the tile"""
    g = gen(14, where)
    for n, h in ((40, 1), (4, 2)):
        q, k, v, do = qkv(1, h, 1, n, 40, 32, 'bf16', g)
        kw = dict(scale=0.2, window=(None, 0))
        clean = [t.detach().requires_grad_() for t in (q, k, v)]
        oc = ops.impl.window_attention(*clean, **kw)
        gc = torch.autograd.grad(oc, clean, do)
        exact = att_ref(q, k, v, 0.2, seen(1, n, 40, (None, 0), 0, None, None, where), do)
        rows = torch.arange(n) < n - 2                          # key 38 is seen by the last two of the queries
        for spoil in ('k', 'v'):
            for fill in (math.nan, math.inf):
                k2, v2 = k.clone(), v.clone()
                (k2 if spoil == 'k' else v2)[0, 0, 38, 5] = fill
                bad = [t.detach().requires_grad_() for t in (q, k2, v2)]
                o = ops.impl.window_attention(*bad, **kw)
                within(o[:, :, rows], exact[0][0][:, :, rows], exact[0][1][:, :, rows], 'o')
                late = o[:, :, ~rows]
                if spoil == 'v':
                    others = [i for i in range(32) if i != 5]
                    assert not torch.isfinite(late[..., 5]).any() and torch.isfinite(late[..., others]).all()
                elif fill != fill:
                    assert not torch.isfinite(late).any()
                else:                                           # a score of +inf spoils its row, one of -inf has probability zero
                    up = (q[:, :, ~rows][..., 5] > 0)[..., None].expand_as(late)
                    assert torch.equal(torch.isfinite(late), ~up)
                dq, dk, dv = torch.autograd.grad(o, bad, do)
                within(dq[:, :, rows], exact[1][0][:, :, rows], exact[1][1][:, :, rows], 'dq')
        # query 1 of n sees keys 0 .. 40 - n + 1
        last = 40 - n + 1
        for spoil in ('q', 'do'):
            q2, do2 = q.clone(), do.clone()
            (q2 if spoil == 'q' else do2)[0, 0, 1, 7] = math.nan
            bad = [t.detach().requires_grad_() for t in (q2, k, v)]
            o = ops.impl.window_attention(*bad, **kw)
            dq, dk, dv = torch.autograd.grad(o, bad, do2)
            for got, (ref, tol) in ((dk, exact[2]), (dv, exact[3])):
                within(got[:, :, last + 1:], ref[:, :, last + 1:], tol[:, :, last + 1:], spoil)
                assert not torch.isfinite(got[:, :, :last + 1, 7]).any()
            others = torch.ones(h, n, dtype=torch.bool)
            others[0, 1] = False
            assert torch.equal(dq[0][others], gc[0][0][others])


# what the key tiles' row chunks can be: only the sinks' tiles are cut (256 key tiles or more, many rows), one and two such tiles, grouped
# heads; every tile is cut; none is
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('case', [(4, 8, 8, 1100, 1100, 32, (40, 0), 3), (10, 4, 4, 1100, 1200, 64, (30, 20), 130),
                                  (8, 8, 4, 1100, 1100, 128, (40, 0), 3), (1, 3, 1, 700, 1500, 128, (600, 0), 2),
                                  (16, 4, 4, 600, 600, 64, (100, 100), 0)])
def test_window_attention_row_chunks(case, dtype):
    att_run('cuda', case, dtype)


@where
@pytest.mark.parametrize('window', [(None, 0), (150, 0)])
def test_window_attention_nan_and_row_chunks(where, window):
    """300 rows, cut into chunks: a NaN query or gradient of a middle chunk reaches the keys that it sees, through the chunks' sum, and no
    other key; bits are the same every time"""
    g = gen(15, where)
    n, at = 300, 200
    q, k, v, do = qkv(1, 2, 1, n, n, 32, 'bf16', g)
    ok = seen(1, n, n, window, 0, None, None, where)
    exact = att_ref(q, k, v, 0.2, ok, do)
    sees = ok[0, at]
    for spoil in ('q', 'do'):
        q2, do2 = q.clone(), do.clone()
        (q2 if spoil == 'q' else do2)[0, 1, at, 7] = math.nan
        runs = []
        for _ in range(2):
            leaves = [t.detach().requires_grad_() for t in (q2, k, v)]
            o = ops.impl.window_attention(*leaves, scale=0.2, window=window)
            runs.append(torch.autograd.grad(o, leaves, do2))
        for got, (ref, tol) in ((runs[0][1], exact[2]), (runs[0][2], exact[3])):
            within(got[:, :, ~sees], ref[:, :, ~sees], tol[:, :, ~sees], spoil)
            assert not torch.isfinite(got[:, :, sees, 7]).any()
        for a, b in zip(*runs):
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@where
def test_window_attention_nothing_to_see(where):
    """no queries, no keys, no batch"""
    for B, n, m in ((2, 0, 5), (2, 3, 0), (0, 3, 5)):
        q = torch.randn(B, 2, n, 32, device=where).to(torch.bfloat16).requires_grad_()
        k, v = (torch.randn(B, 1, m, 32, device=where).to(torch.bfloat16).requires_grad_() for _ in range(2))
        o = ops.impl.window_attention(q, k, v, scale=1.0)
        assert o.shape == q.shape and not o.any()
        for t, s in zip(torch.autograd.grad(o, (q, k, v), torch.ones_like(o)), (q, k, v)):
            assert t.shape == s.shape and not t.any()


# ---- refusals ----------------------------------------------------------------------------------------------------------

def test_refusals():
    x, w = torch.randn(3, 8), torch.ones(8)
    L = ops.impl.layer_norm
    for bad, err in ((lambda: L(x.double(), w), TypeError), (lambda: L(x, torch.ones(7)), ValueError), (lambda: L(x, w, torch.ones(8, 1)), ValueError),
                     (lambda: L(torch.randn(2, 16385), torch.ones(16385)), ValueError), (lambda: L(torch.zeros(()), w), ValueError),
                     (lambda: L(torch.zeros(3, 0), torch.ones(0)), ValueError), (lambda: L(x, None), ValueError),
                     (lambda: L(x, torch.ones(8, dtype=torch.int32)), ValueError)):
        with pytest.raises(err):
            bad()
    for bad in ((0,), (), (-1, 3), (129,), (64, 65)):
        with pytest.raises(ValueError):
            ops.RotarySpec(bad)
    with pytest.raises(ValueError):
        ops.RotarySpec((4,), theta=0.0)
    R, spec = ops.impl.rotary, ops.RotarySpec((2, 2))
    q, pos = torch.randn(1, 2, 5, 8), torch.zeros(5, 2, dtype=torch.int32)
    for bad, err in ((lambda: R(q[0], pos, spec), ValueError), (lambda: R(q, pos, spec, k=q.bfloat16()), TypeError), (lambda: R(q.double(), pos, spec), TypeError),
                     (lambda: R(q, pos[:4], spec), ValueError), (lambda: R(q, pos[:, :1], spec), ValueError), (lambda: R(q, pos.double(), spec), TypeError),
                     (lambda: R(q[..., :7], pos, spec), ValueError), (lambda: R(q, pos, (2, 2)), TypeError), (lambda: R(q, pos, spec, k=q[:, :, :4]), ValueError)):
        with pytest.raises(err):
            bad()
    W = ops.impl.window_attention
    q, k = torch.randn(2, 4, 5, 32).bfloat16(), torch.randn(2, 2, 6, 32).bfloat16()
    ok = dict(scale=1.0)
    for bad, err in ((lambda: W(q.float(), k.float(), k.float(), **ok), TypeError), (lambda: W(q, k, k.half(), **ok), TypeError),
                     (lambda: W(q[:, :3], k, k, **ok), ValueError), (lambda: W(q, k, k[:, :, :5], **ok), ValueError),
                     (lambda: W(q[..., :16], k[..., :16], k[..., :16], **ok), ValueError), (lambda: W(q, k[:1], k[:1], **ok), ValueError),
                     (lambda: W(q, k, k, scale=0.0), ValueError), (lambda: W(q, k, k, scale=math.nan), ValueError), (lambda: W(q, k, k, scale=-1.0), ValueError),
                     (lambda: W(q, k, k, window=(-1, 0), **ok), ValueError), (lambda: W(q, k, k, sinks=-1, **ok), ValueError),
                     (lambda: W(q, k, k, lengths=torch.zeros(3, dtype=torch.int32), **ok), ValueError), (lambda: W(q, k, k, lengths=torch.zeros(2), **ok), ValueError),
                     (lambda: W(q, k, k, key_mask=torch.ones(2, 5, dtype=torch.bool), **ok), ValueError), (lambda: W(q, k, k, key_mask=torch.ones(2, 6), **ok), ValueError),
                     (lambda: W(q[0], k, k, **ok), ValueError)):
        with pytest.raises(err):
            bad()


def test_second_derivatives_are_refused():
    x, w = torch.randn(3, 8, requires_grad=True), torch.ones(8)
    g, = torch.autograd.grad(ops.impl.layer_norm(x, w).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    q = torch.randn(1, 1, 3, 32).bfloat16().requires_grad_()
    g, = torch.autograd.grad(ops.impl.window_attention(q, q, q, scale=1.0).float().pow(2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_c_entry_refusals():
    """the C ABI checks what it is given before it launches anything"""
    import ctypes as C
    from gigagan_pytorch_amd import _C
    L = _C.lib().lib
    t = torch.zeros(4096)
    p = t.data_ptr()
    assert L.gg_layernorm_fwd(None, 8, p, p, p, None, None, 1, 8, 1e-5, 0, None) == -1
    assert L.gg_layernorm_fwd(p, 8, p, p, p, None, None, 1, 16385, 1e-5, 0, None) == -2
    assert L.gg_layernorm_fwd(p, 8, p, p, p, None, None, 1, 8, 1e-5, 3, None) == -3
    assert L.gg_layernorm_fwd(p, 8, p, p, p, p, None, 1, 8, 1e-5, 0, None) == -1
    assert L.gg_layernorm_bwd(p, 8, p, 8, p, p, p, p, None, p, p, 1, 8, 0, None) == -1
    spec = ops.RotarySpec((2, 2))
    d = _C.RotaryDesc(q=p, yq=p, positions=p, freqs=C.addressof(spec._freqs), axes=C.addressof(spec._axes), B=1, n=1, hq=1, d=8, pairs=4, n_axes=1)
    assert L.gg_rotary(C.byref(d), None) == -2          # an axis that is not there
    d.n_axes, d.d = 2, 7
    assert L.gg_rotary(C.byref(d), None) == -2
    d.d, d.hk = 8, 1
    assert L.gg_rotary(C.byref(d), None) == -1
    w = _C.WindowDesc(q=p, k=p, v=p, o=p, B=1, n=1, m=8192, h=1, hk=1, d=64, left=-1, right=-1, scale=1.0)
    assert L.gg_window_workspace_bytes(C.byref(w), 0) > 0
    assert L.gg_window_fwd(C.byref(w), None, 0, None) == -5
    w.d = 48
    assert L.gg_window_fwd(C.byref(w), p, 1 << 20, None) == -2
    w.d, w.scale = 64, 0.0
    assert L.gg_window_fwd(C.byref(w), p, 1 << 20, None) == -3
    w.scale, w.q_strides[2] = 1.0, 12
    assert L.gg_window_fwd(C.byref(w), p, 1 << 20, None) == -4
    w.q_strides[2] = 0
    w.h = 3
    w.hk = 2
    assert L.gg_window_fwd(C.byref(w), p, 1 << 20, None) == -2
    w.hk = 3
    assert L.gg_window_bwd(C.byref(w), None, 0, None) == -1
    assert b'gg_window_bwd' in L.gg_last_error()


def test_launches_of_too_many_threads_are_refused():
    """a launch holds fewer than 2^32 threads: larger calls end in an error, before anything runs"""
    import ctypes as C
    from gigagan_pytorch_amd import _C
    L = _C.lib().lib
    t = torch.zeros(4096)
    p = t.data_ptr()
    assert L.gg_layernorm_fwd(p, 8, p, p, p, None, None, 1 << 31, 8, 1e-5, 0, None) == -2
    assert b'too many rows' in L.gg_last_error()
    spec = ops.RotarySpec((2, 2))
    d = _C.RotaryDesc(q=p, yq=p, positions=p, freqs=C.addressof(spec._freqs), axes=C.addressof(spec._axes), B=1 << 15, n=1 << 15, hq=1024, d=8,
                      pairs=4, n_axes=2)
    assert L.gg_rotary(C.byref(d), None) == -2
    assert b'too many tokens' in L.gg_last_error()
    w = _C.WindowDesc(q=p, k=p, v=p, o=p, o_lo=p, lse=p, d_o=p, dq=p, dk=p, dv=p, dvec=p, B=1 << 12, n=1 << 20, m=128, h=1, hk=1, d=64,
                      left=-1, right=-1, scale=1.0)
    assert L.gg_window_fwd(C.byref(w), None, 0, None) == -2
    assert b'too many rows' in L.gg_last_error()
    assert L.gg_window_bwd(C.byref(w), None, 0, None) == -2
    assert b'too many rows' in L.gg_last_error()
