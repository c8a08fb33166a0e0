"""The transformer operators that are measured: layer norm, rotary positions over several axes, and attention with a
sliding window and sinks. `listed()` and `draw()` name the cases, `prepare()` makes what a program has in hand before the
call, `run()` is one pass: with `own` set through the framework's public entry points, else in elementary torch
operations. `exact()` gives the same outputs from the definitions in 64 bits.

A window-attention case has its queries at the LAST n of a sequence's positions: query i of batch item b sits at position
p = length_b - n + i and sees key j when j < length_b, j <= p + right, and j >= p - left or j < sinks, and the key mask
keeps j. A bound of -1 stands for "no bound".
"""
import math

import numpy as np
import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-5
THETA = 10000.0


# ---- cases --------------------------------------------------------------------------------------------------------

def _ln(rows, dim, dtype, train, bias=True):
    return dict(op='layer_norm', rows=rows, dim=dim, dtype=dtype, train=train, bias=bias)


def _rot(batch, grid, heads, kv_heads, head_dim, sections, dtype, train, start=0, interleaved=False, shared=False):
    return dict(op='rotary', batch=batch, grid=grid, heads=heads, kv_heads=kv_heads, head_dim=head_dim, sections=sections,
                dtype=dtype, train=train, start=start, interleaved=interleaved, shared=shared)


def _att(batch, heads, kv_heads, n, m, head_dim, left, right, sinks, dtype, train, ragged=False, masked=False):
    return dict(op='window_attention', batch=batch, heads=heads, kv_heads=kv_heads, n=n, m=m, head_dim=head_dim, left=left,
                right=right, sinks=sinks, dtype=dtype, train=train, ragged=ragged, masked=masked)


def listed():
    return [
        # the text encoder's norm: 32 captions of 77 tokens behind the learned global token, 512 features; no gradient
        dict(_ln(32 * 78, 512, 'bf16', False), name='norm-text'),
        # a training step of a norm over fp32 features whose width no vector divides
        dict(_ln(5003, 1001, 'fp32', True), name='norm-odd-fp32-train'),
        # a training step of a wide norm over many tokens: the bandwidth-bound end
        dict(_ln(65536, 2048, 'bf16', True), name='norm-wide-train'),
        # the text encoder's queries and keys, one axis: a launch-bound call
        dict(_rot(32, '77', 8, 8, 64, '32', 'bf16', False), name='rotary-text'),
        # the image self-attention of the 32x32 stage, rows and columns as two axes, with its gradient
        dict(_rot(32, '32x32', 8, 8, 64, '16,16', 'bf16', True), name='rotary-image-train'),
        # a long video: time, height and width on one shared frequency ladder, keys of fewer heads, far positions
        dict(_rot(1, '16x45x80', 24, 8, 128, '16,24,24', 'fp16', False, start=100000, shared=True), name='rotary-video'),
        # the text encoder's attention in training: null key and global token as sinks, padded captions
        dict(_att(32, 8, 8, 78, 79, 64, 16, 16, 2, 'bf16', True, masked=True), name='attend-text-train'),
        # one new token on one sequence, everything before it visible: a latency-bound call
        dict(_att(1, 16, 2, 1, 8192, 64, -1, 0, 0, 'bf16', False), name='attend-one-token'),
        # one new token each on 64 sequences of unequal lengths in a padded cache
        dict(_att(64, 32, 8, 1, 16384, 128, 4095, 0, 4, 'bf16', False, ragged=True), name='attend-token-batch'),
        # a long sequence read at once, causal
        dict(_att(1, 32, 8, 32768, 32768, 128, 4095, 0, 4, 'bf16', False), name='attend-long'),
        # training on a 64x64 feature map in raster order, both sides of a pixel visible
        dict(_att(8, 8, 8, 4096, 4096, 64, 512, 512, 0, 'bf16', True), name='attend-map-train'),
        # odd sizes everywhere: grouped heads, unequal lengths, fewer queries than keys, small heads
        dict(_att(3, 6, 2, 777, 1291, 32, 100, 7, 3, 'fp16', True, ragged=True), name='attend-odd-fp16-train'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['layer_norm', 'rotary', 'window_attention', 'window_attention'])
    train = rng.random() < 0.5
    if op == 'layer_norm':
        rows, dim = _log(rng, 1, 65536), _log(rng, 1, 8192)
        if rng.random() < 0.5:
            dim = max(8, dim // 8 * 8)
        rows = max(1, min(rows, 65536 * 2048 // dim))
        return _ln(rows, dim, rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), train, bias=rng.random() < 0.8)
    if op == 'rotary':
        head_dim = rng.choice([32, 64, 64, 128])
        axes = rng.choice([1, 2, 3])
        half = head_dim // 2 if rng.random() < 0.7 else head_dim // 4        # some features left as they are
        cut = sorted(rng.sample(range(1, half), axes - 1))
        sections = [b - a for a, b in zip([0] + cut, cut + [half])]
        tokens = _log(rng, 1, 32768)
        if axes == 1:
            grid = [tokens]
        elif axes == 2:
            w = _log(rng, 1, max(1, int(tokens ** 0.5) * 2))
            grid = [max(1, tokens // w), w]
        else:
            t, w = _log(rng, 1, 16), _log(rng, 1, 90)
            grid = [t, max(1, tokens // (t * w)), w]
        n = math.prod(grid)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3])
        batch = _log(rng, 1, max(1, min(64, 100_000_000 // (n * (heads + kv) * head_dim))))
        return _rot(batch, 'x'.join(map(str, grid)), heads, kv, head_dim, ','.join(map(str, sections)),
                    rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), train, start=rng.choice([0, 0, 7, 100000, 1000000]),
                    interleaved=rng.random() < 0.4, shared=rng.random() < 0.4)
    head_dim = rng.choice([32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    m = _log(rng, 1, 16384)
    shape = rng.random()
    if shape < 0.3:                       # one or a few new tokens
        n, train = min(m, rng.choice([1, 1, 1, 2, 5])), False
    elif shape < 0.5:                     # a chunk of new tokens behind a cache
        n = _log(rng, 1, m)
    else:
        n = m
    left = -1 if rng.random() < 0.2 else _log(rng, 1, 4096) - 1
    right = rng.choice([0, 0, 0, left, left, _log(rng, 1, 256)])
    sinks = rng.choice([0, 0, 1, 4, _log(rng, 1, 100)])
    cap = 2 ** 35 if train else 2 ** 38                              # (query, key) pairs over all heads, times features
    while True:
        cost = n * min(m, (m if left < 0 else left) + (m if right < 0 else right) + 1 + sinks) * heads * head_dim
        if cost <= cap:
            break
        n, m = (n + 1) // 2, max((n + 1) // 2, m // 2)
    batch = max(1, min(_log(rng, 1, 64), cap // cost, 2 ** 29 // ((m * kv + n * heads) * head_dim)))
    masked = rng.random() < 0.3
    return _att(batch, heads, kv, n, m, head_dim, left, right, sinks, rng.choice(['bf16', 'bf16', 'bf16', 'fp16']), train,
                ragged=not masked and rng.random() < 0.4, masked=masked)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _lengths(case):
    """the sequences' lengths: spread evenly between the shortest that holds the queries (or an eighth of the longest) and the longest"""
    b, n, m = case['batch'], case['n'], case['m']
    if not (case['ragged'] or case['masked']):
        return [m] * b
    lo = max(n, m // 8, 1) if case['ragged'] else max(m // 8, 1)
    return [m - (m - lo) * i // max(1, b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    dt = TYPES[case['dtype']]

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device='cuda', dtype=torch.float32) * scale + shift).to(dtype)

    s = dict(case=case)
    train = case['train']
    if case['op'] == 'layer_norm':
        rows, dim = case['rows'], case['dim']
        s['x'] = normal(rows, dim, scale=1.5, shift=0.3).requires_grad_(train)
        s['weight'] = normal(dim, dtype=torch.float32, scale=0.2, shift=1.0).requires_grad_(train)
        s['bias'] = normal(dim, dtype=torch.float32, scale=0.2).requires_grad_(train) if case['bias'] else None
        s['dy'] = normal(rows, dim) if train else None
        return s
    b, h, hk, d = case['batch'], case['heads'], case['kv_heads'], case['head_dim']
    if case['op'] == 'rotary':
        sizes = [int(t) for t in case['grid'].split('x')]
        n = math.prod(sizes)
        # queries and keys as one projection leaves them: features of all heads side by side, token by token
        qk = normal(b, n, (h + hk) * d)
        s['q'] = qk[..., :h * d].unflatten(-1, (h, d)).transpose(1, 2).detach().requires_grad_(train)
        s['k'] = qk[..., h * d:].unflatten(-1, (hk, d)).transpose(1, 2).detach().requires_grad_(train)
        axes = torch.meshgrid(*(torch.arange(t, device='cuda', dtype=torch.int32) for t in sizes), indexing='ij')
        # every batch item has an offset of its own on the first axis: crops and continued sequences
        pos = torch.stack([a.flatten() for a in axes], -1)[None].repeat(b, 1, 1)
        off = torch.randint(0, 64, (b, 1), generator=g, device='cuda', dtype=torch.int32) + case['start']
        pos[:, :, 0] += off
        s['positions'] = pos
        s['dq'] = normal(b, n, h, d).transpose(1, 2) if train else None
        s['dk'] = normal(b, n, hk, d).transpose(1, 2) if train else None
        if own:
            from gigagan_pytorch_amd import ops
            s['spec'] = ops.RotarySpec([int(t) for t in case['sections'].split(',')], theta=THETA, shared=case['shared'],
                                       interleaved=case['interleaved'])
        return s
    n, m = case['n'], case['m']
    if n == m and not case['ragged']:
        # one fused projection: q, k and v of a token side by side
        qkv = normal(b, n, (h + 2 * hk) * d)
        q, k, v = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in qkv.split([h * d, hk * d, hk * d], dim=-1))
    else:
        q = normal(b, n, h, d).transpose(1, 2)
        k, v = normal(b, m, hk, d).transpose(1, 2), normal(b, m, hk, d).transpose(1, 2)
    s['q'], s['k'], s['v'] = (t.detach().requires_grad_(train) for t in (q, k, v))
    s['do'] = normal(b, n, h, d).transpose(1, 2) if train else None
    lens = torch.tensor(_lengths(case), device='cuda', dtype=torch.int32)
    lens = lens[torch.randperm(b, generator=g, device='cuda')]
    s['lengths'] = lens if case['ragged'] else None
    # padded captions: the tokens behind the caption's end carry nothing
    s['key_mask'] = (torch.arange(m, device='cuda')[None] < lens[:, None]) if case['masked'] else None
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------

def _plain_layer_norm(s):
    x, w = s['x'].detach().float(), s['weight'].detach()
    c = x - x.mean(-1, keepdim=True)
    rstd = ((c * c).mean(-1, keepdim=True) + EPS).rsqrt()
    xh = c * rstd
    y = xh * w
    if s['bias'] is not None:
        y = y + s['bias'].detach()
    y = y.to(s['x'].dtype)
    if s['dy'] is None:
        return [y]
    dy = s['dy'].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    out = [y, dx.to(y.dtype), (dy * xh).sum(0)]
    return out if s['bias'] is None else out + [dy.sum(0)]


def _frequencies(case):
    """the angle per position step of every feature pair, and the axis whose position it takes"""
    sections = [int(t) for t in case['sections'].split(',')]
    axis = [a for a, c in enumerate(sections) for _ in range(c)]
    if case['shared']:
        freq = [THETA ** (-i / len(axis)) for i in range(len(axis))]
    else:
        freq = [THETA ** (-i / c) for c in sections for i in range(c)]
    return torch.tensor(freq, dtype=torch.float64), torch.tensor(axis)


def _turn(x, cos, sin, interleaved):
    r = cos.shape[-1]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, x[..., 2 * r:]), -1)


def _plain_rotary(s):
    case = s['case']
    freq, axis = (t.to('cuda') for t in _frequencies(case))
    angle = s['positions'].double()[..., axis] * freq                # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = [_turn(t.detach(), cos, sin, case['interleaved']).to(t.dtype) for t in (s['q'], s['k'])]
    if s['dq'] is not None:
        out += [_turn(t, cos, -sin, case['interleaved']).to(t.dtype) for t in (s['dq'], s['dk'])]
    return out


def _plain_window_attention(s):
    case = s['case']
    q, k, v = (s[t].detach().float() for t in 'qkv')
    b, h, n, d = q.shape
    hk, m = k.shape[1], k.shape[2]
    grp = h // hk
    left = m if case['left'] < 0 else case['left']
    right = m if case['right'] < 0 else case['right']
    scale = d ** -0.5
    dev = q.device
    length = torch.full((b,), m, device=dev) if s['lengths'] is None else s['lengths'].long()
    item = torch.arange(b, device=dev)[:, None]
    k, v = k.transpose(1, 2), v.transpose(1, 2)                      # (b, m, hk, d)
    out = torch.zeros(b, hk, grp, n, d, device=dev)
    do = None
    if s['do'] is not None:
        do = s['do'].float().reshape(b, hk, grp, n, d)
        dq = torch.zeros_like(out)
        dk, dv = torch.zeros(b * m, hk * d, device=dev), torch.zeros(b * m, hk * d, device=dev)
    q = q.reshape(b, hk, grp, n, d)
    rows = max(1, min(n, 2 ** 27 // max(1, b * h * min(m, left + right + 1024)), 1024))
    for t0 in range(0, n, rows):
        t1 = min(n, t0 + rows)
        c = t1 - t0
        p = length[:, None] - n + torch.arange(t0, t1, device=dev)   # (b, c)
        first = (p[:, 0] - left).clamp(min=0)                        # first key that the block's window holds
        span = min(m, left + right + c)
        j = torch.cat((torch.arange(case['sinks'], device=dev).expand(b, -1), first[:, None] + torch.arange(span, device=dev)), 1)
        is_sink = torch.arange(j.shape[1], device=dev) < case['sinks']
        keep = torch.where(is_sink, j < first[:, None], j < length[:, None]) & (j < length[:, None])
        jc = j.clamp(max=m - 1)
        if s['key_mask'] is not None:
            keep = keep & s['key_mask'][item, jc]
        jj, pp = j[:, None, :], p[:, :, None]
        see = keep[:, None, :] & (jj <= pp + right) & ((jj >= pp - left) | (jj < case['sinks'])) & (pp >= 0)
        see = see[:, None, None]                                     # (b, 1, 1, c, keys)
        kb = k[item, jc].transpose(1, 2)                             # (b, hk, keys, d)
        vb = v[item, jc].transpose(1, 2)
        qb = q[:, :, :, t0:t1].reshape(b, hk, grp * c, d)
        x = (qb @ kb.transpose(-1, -2)).view(b, hk, grp, c, -1) * scale
        x = x.masked_fill(~see, -math.inf)
        top = x.amax(-1, keepdim=True)
        e = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
        z = e.sum(-1, keepdim=True)
        pr = e / z.masked_fill(z == 0, 1.0)
        o = (pr.view(b, hk, grp * c, -1) @ vb).view(b, hk, grp, c, d)
        out[:, :, :, t0:t1] = o
        if do is None:
            continue
        g = do[:, :, :, t0:t1]
        gf = g.reshape(b, hk, grp * c, d)
        dp = (gf @ vb.transpose(-1, -2)).view_as(pr)
        ds = (pr * (dp - (g * o).sum(-1, keepdim=True)) * scale).view(b, hk, grp * c, -1)
        dq[:, :, :, t0:t1] = (ds @ kb).view(b, hk, grp, c, d)
        at = (item * m + jc).flatten()
        dk.index_add_(0, at, (ds.transpose(-1, -2) @ qb).transpose(1, 2).reshape(-1, hk * d))
        dv.index_add_(0, at, (pr.view_as(ds).transpose(-1, -2) @ gf).transpose(1, 2).reshape(-1, hk * d))
    dt = s['q'].dtype
    res = [out.view(b, h, n, d).to(dt)]
    if do is not None:
        res += [dq.view(b, h, n, d).to(dt)] + [t.view(b, m, hk, d).transpose(1, 2).to(dt) for t in (dk, dv)]
    return res


def run(state):
    case = state['case']
    if not own:
        with torch.no_grad():
            return globals()['_plain_' + case['op']](state)
    from gigagan_pytorch_amd import ops
    with torch.set_grad_enabled(case['train']):
        if case['op'] == 'layer_norm':
            leaves = [t for t in (state['x'], state['weight'], state['bias']) if t is not None]
            y = ops.impl.layer_norm(state['x'], state['weight'], state['bias'], eps=EPS)
            return [y.detach(), *torch.autograd.grad(y, leaves, state['dy'])] if case['train'] else [y]
        if case['op'] == 'rotary':
            q, k = ops.impl.rotary(state['q'], state['positions'], state['spec'], k=state['k'])
            if not case['train']:
                return [q, k]
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (state['q'], state['k']), (state['dq'], state['dk']))]
        window = tuple(None if t < 0 else t for t in (case['left'], case['right']))
        o = ops.impl.window_attention(state['q'], state['k'], state['v'], scale=case['head_dim'] ** -0.5, window=window,
                                      sinks=case['sinks'], key_mask=state['key_mask'], lengths=state['lengths'])
        if not case['train']:
            return [o]
        return [o.detach(), *torch.autograd.grad(o, (state['q'], state['k'], state['v']), state['do'])]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def _seen(case):
    """(query, key) pairs that see each other, and keys that some query sees, summed over the batch (one head); key masks taken as kept
    up to the spread lengths"""
    n, m, s = case['n'], case['m'], case['sinks']
    left = m if case['left'] < 0 else case['left']
    right = m if case['right'] < 0 else case['right']
    pairs = keys = 0
    for length in _lengths(case):
        end = length if case['ragged'] else m                        # where the queries end; a mask only takes keys away
        p = np.arange(end - n, end, dtype=np.int64)
        p = p[p >= 0]
        hi = np.minimum(p + right, length - 1)
        lo = np.maximum(p - left, 0)
        in_window = np.maximum(hi - lo + 1, 0)
        in_sinks = np.maximum(np.minimum(np.minimum(lo, s) - 1, hi) + 1, 0)
        pairs += int((in_window + in_sinks).sum())
        if len(p):
            a, z = int(lo[0]), int(hi[-1])
            keys += max(0, z - a + 1) + max(0, min(min(a, s) - 1, z) + 1)
    return pairs, keys


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'layer_norm':
        cells = case['rows'] * case['dim']
        if not case['train']:
            return dict(bytes=2 * cells * size + 8 * case['dim'], flops=8 * cells)
        return dict(bytes=4 * cells * size + 16 * case['dim'], flops=22 * cells)
    b, h, hk, d = case['batch'], case['heads'], case['kv_heads'], case['head_dim']
    if case['op'] == 'rotary':
        sizes = [int(t) for t in case['grid'].split('x')]
        cells = b * math.prod(sizes) * (h + hk) * d
        passes = 2 if case['train'] else 1
        return dict(bytes=passes * 2 * cells * size + 4 * b * math.prod(sizes) * len(sizes), flops=passes * 3 * cells)
    pairs, keys = _seen(case)
    rows = b * case['n'] * h
    if not case['train']:
        return dict(bytes=(2 * rows + 2 * keys * hk) * d * size, flops=4 * pairs * h * d)
    # forward: two products; backward: four (the scores could be kept)
    return dict(bytes=(4 * rows + 2 * keys * hk + 2 * b * case['m'] * hk) * d * size, flops=12 * pairs * h * d)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _exact_layer_norm(s):
    train = s['dy'] is not None
    x = s['x'].detach().double().requires_grad_(train)
    w = s['weight'].detach().double().requires_grad_(train)
    leaves, y = [x, w], None
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w
    if s['bias'] is not None:
        leaves.append(s['bias'].detach().double().requires_grad_(train))
        y = y + leaves[-1]
    if not train:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s['dy'].double())]


def _exact_rotary(s):
    case = s['case']
    sections = [int(t) for t in case['sections'].split(',')]
    half = sum(sections)
    factors, base = [], 0
    for a, c in enumerate(sections):
        i = torch.arange(c, device='cuda', dtype=torch.float64)
        power = (base + i) / half if case['shared'] else i / c
        angle = s['positions'][:, None, :, a, None].double() * torch.exp(-math.log(THETA) * power)
        factors.append(torch.polar(torch.ones_like(angle), angle))
        base += c
    factor = torch.cat(factors, -1)

    def turned(x, f):
        y = x.detach().double()
        if case['interleaved']:
            z = torch.view_as_complex(y[..., :2 * half].reshape(*y.shape[:-1], half, 2).contiguous()) * f
            r = torch.view_as_real(z).reshape(*y.shape[:-1], 2 * half)
        else:
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * f
            r = torch.cat((z.real, z.imag), -1)
        return torch.cat((r, y[..., 2 * half:]), -1)
    out = [turned(s['q'], factor), turned(s['k'], factor)]
    if s['dq'] is not None:
        out += [turned(s['dq'], factor.conj()), turned(s['dk'], factor.conj())]
    return out


def _exact_window_attention(s):
    """item by item, block of queries by block of queries: scores of every key from the block's first to its last, softmax as the
    exponential of the score minus the logarithm of the sum; gradients by automatic differentiation"""
    case = s['case']
    train = s['do'] is not None
    b, h, n, d = s['q'].shape
    hk, m = s['k'].shape[1:3]
    lengths = [m] * b if s['lengths'] is None else s['lengths'].tolist()
    outs, grads = [], []
    for i in range(b):
        q = s['q'][i].detach().double().requires_grad_(train)
        k = s['k'][i].detach().double().requires_grad_(train)
        v = s['v'][i].detach().double().requires_grad_(train)
        total = [torch.zeros_like(t) for t in (q, k, v)]
        o_item = torch.zeros_like(q)
        step = 256 if train else 512
        for t0 in range(0, n, step):
            rows = torch.arange(t0, min(n, t0 + step), device='cuda')
            at = rows + (lengths[i] - n)
            lo = 0 if case['left'] < 0 or case['sinks'] > 0 and int(at[0]) - case['left'] <= case['sinks'] else max(0, int(at[0]) - case['left'])
            hi = lengths[i] if case['right'] < 0 else min(lengths[i], int(at[-1]) + case['right'] + 1)
            keys = torch.arange(lo, max(lo, hi), device='cuda')
            if lo > 0 and case['sinks']:
                keys = torch.cat((torch.arange(min(case['sinks'], max(hi, 0)), device='cuda'), keys))
            if len(keys) == 0:
                continue
            ok = torch.ones(len(rows), len(keys), dtype=torch.bool, device='cuda')
            gap = keys[None, :] - at[:, None]
            if case['right'] >= 0:
                ok &= gap <= case['right']
            if case['left'] >= 0:
                ok &= (gap >= -case['left']) | (keys[None, :] < case['sinks'])
            ok &= (at >= 0)[:, None]
            if s['key_mask'] is not None:
                ok &= s['key_mask'][i][keys][None]
            ks, vs = (t[:, keys].repeat_interleave(h // hk, dim=0) for t in (k, v))
            score = torch.matmul(q[:, rows], ks.mT) / math.sqrt(d)
            score = score.masked_fill(~ok, -1e300)
            share = torch.exp(score - torch.logsumexp(score, -1, keepdim=True)) * ok
            o = torch.matmul(share, vs)
            o_item[:, rows] = o.detach()
            if train:
                for acc, g in zip(total, torch.autograd.grad(o, (q, k, v), s['do'][i][:, rows].double())):
                    acc += g
        outs.append(o_item.detach())
        grads.append(total)
    res = [torch.stack(outs)]
    if train:
        res += [torch.stack([g[t] for g in grads]) for t in range(3)]
    return res


def exact(case, seed):
    state = prepare(case, seed)
    with torch.set_grad_enabled(case['train']):
        return globals()['_exact_' + case['op']](state)
