"""ORACLE — test infrastructure only. Not imported by the product path.

A plain fp32 PyTorch restatement of the reference's arithmetic for every op on the GigaGAN G+D hot path
(SURVEY.md §8a), each function citing the reference lines it follows (`gp.py` =
/root/reference/gigagan_pytorch/gigagan_pytorch.py). It exposes the same method set as
`gigagan_pytorch_amd.ops.HipOps`, so tests can (a) compare each HIP kernel against it on the same inputs
and (b) run our Generator/Discriminator on CPU through it and compare with the unmodified reference
(tests/test_reference_parity.py, live when /root/reference exists; tests/golden/*.pt otherwise).

Parity status: pinned against the reference itself — fixtures in tests/golden/ are generated by
tests/golden/make_golden.py, which imports the unmodified reference. The one third-party piece without a
vendored source is kornia's `filter2d` (reflect-padded, abs-sum-normalised depthwise blur, gp.py:255):
its arithmetic is restated in `blur` below and is "parity unpinned" against kornia proper.

`bf16_operands=True` rounds the operands of every contraction to bf16 (fp32 accumulate), which is what
the MFMA kernels compute; this lets GPU tests use a much tighter tolerance than a pure-fp32 comparison.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F


def _r(t, on):
    return t.to(torch.bfloat16).to(torch.float32) if on else t


class OracleOps:
    name = 'oracle'
    act_dtype = torch.float32

    def __init__(self, bf16_operands: bool = False):
        self.bf16 = bf16_operands

    def prepare(self, x):
        return x.float()

    # nn.Conv2d(k, padding=k//2) call sites: gp.py:112-113, :1275-1281, :1454-1470, :1608-1621, :1656
    def conv2d(self, x, weight, bias=None, act=None, stride=1, scale=1.0, residual=None, res_scale=1.0):
        k = weight.shape[-1]
        y = F.conv2d(_r(x.float(), self.bf16), _r(weight.float(), self.bf16), None if bias is None else bias.float(),
                     stride=stride, padding=k // 2 if stride == 1 else 0)          # gp.py:1612 (stride-2 1x1 residual)
        if scale != 1.0:
            y = y * scale
        if act == 'lrelu':
            y = F.leaky_relu(y, 0.2)   # gp.py:109
        if residual is not None:       # the skip connections of gp.py:757-758 folded into the producing conv
            y = y + residual.float() * res_scale
        return y

    # Downsample, gp.py:289-293 ('b c (h s1) (w s2) -> b (c s1 s2) h w' then 1x1 conv) + the merge of gp.py:1826
    def downsample(self, x, weight, bias=None, residual=None, scale=1.0):
        x = x.float()
        b, c, h, w = x.shape
        s2d = x.reshape(b, c, h // 2, 2, w // 2, 2).permute(0, 1, 3, 5, 2, 4).reshape(b, c * 4, h // 2, w // 2)
        y = F.conv2d(_r(s2d, self.bf16), _r(weight.float(), self.bf16), None if bias is None else bias.float()) * scale
        if residual is not None:
            y = y + residual.float()
        return y

    # nn.Linear / EqualLinear: gp.py:302-304, :887, :1121, :1658
    def linear(self, x, weight, bias=None, act=None):
        y = F.linear(_r(x.float(), self.bf16), _r(weight.float(), self.bf16), None if bias is None else bias.float())
        if act == 'lrelu':
            y = F.leaky_relu(y, 0.2)
        return y

    # EqualLinear, gp.py:871-888 (+ the LeakyReLU that follows it in the style network, gp.py:909-914)
    def equal_linear(self, x, weight, bias, lr_mul, act=None):
        return self.linear(x, weight * lr_mul, None if bias is None else bias * lr_mul, act)

    # AdaptiveConv2DMod.forward, gp.py:344-409 (+ Noise gp.py:930-940, LeakyReLU gp.py:109)
    def modconv2d(self, x, weights, mod, kernel_mod=None, demod=True, eps=1e-8, noise=None, noise_weight=None,
                  act=None, in_excite=None):
        x = x.float()
        if in_excite is not None:      # `x * excite` right before the conv (gp.py:1023-1024)
            x = x * in_excite.reshape(x.shape[0], x.shape[1], 1, 1).float()
        b, _, h, w = x.shape
        n, o, i, k, _ = weights.shape
        wts = weights.float()
        if n > 1:
            attn = kernel_mod.float().softmax(dim=-1)                               # gp.py:387
            wts = (wts[None] * attn[:, :, None, None, None, None]).sum(dim=1)     # gp.py:388-390
        else:
            wts = wts[0][None].expand(b, -1, -1, -1, -1)
        wts = wts * (mod.float()[:, None, :, None, None] + 1)                      # gp.py:394-396
        if demod:
            inv = wts.pow(2).sum(dim=(2, 3, 4), keepdim=True).clamp(min=eps).rsqrt()   # gp.py:399
            wts = wts * inv
        y = F.conv2d(_r(x, self.bf16).reshape(1, b * i, h, w), _r(wts, self.bf16).reshape(b * o, i, k, k),
                     padding=k // 2, groups=b).reshape(b, o, h, w)                 # gp.py:402-409
        if noise is not None:
            y = y + noise_weight.float().view(1, o, 1, 1) * noise.float()           # gp.py:940
        if act == 'lrelu':
            y = F.leaky_relu(y, 0.2)
        return y

    # SelfAttention / CrossAttention core, gp.py:573-590, :643-651; q (B,h,n,d), k,v (B,h,m,d)
    def attention(self, q, k, v, *, scale, l2=False, key_mask=None):
        q, k, v = _r(q.float(), self.bf16), _r(k.float(), self.bf16), _r(v.float(), self.bf16)
        if l2:
            qs = (q * q).sum(-1)
            ks = (k * k).sum(-1)
            sim = -(qs[..., :, None] + ks[..., None, :] - 2 * torch.einsum('bhid,bhjd->bhij', q, k))   # gp.py:577-580
        else:
            sim = torch.einsum('bhid,bhjd->bhij', q, k)                                                 # gp.py:574
        sim = sim * scale
        if key_mask is not None:
            sim = sim.masked_fill(~key_mask[:, None, None, :], -torch.finfo(sim.dtype).max)              # gp.py:645-647
        attn = sim.softmax(dim=-1)
        return torch.einsum('bhij,bhjd->bhid', _r(attn, self.bf16), v)                                  # gp.py:590

    # SelfAttention.forward after the q/k/v projections, gp.py:562-592 (heads, null key/value, attention, merge)
    def self_attention(self, q, k, v, null_kv, *, heads, scale, l2):
        # (the oracle's own restatement - nothing from the product package: gp.py:562-566 split heads `b (h d) x y -> b h (x y) d`,
        # :568-571 prepend the learned null key / value, :573-590 similarity -> softmax -> aggregate, :592 merge heads)
        b, _, x, y = q.shape

        def heads_of(t):
            return t.reshape(b, heads, -1, x * y).transpose(2, 3)
        q, k, v = heads_of(q), heads_of(k), heads_of(v)
        nk, nv = (t[None, :, None, :].expand(b, -1, -1, -1).to(q.dtype) for t in null_kv)
        k = torch.cat((nk, k), dim=2)
        v = torch.cat((nv, v), dim=2)
        out = self.attention(q, k, v, scale=scale, l2=l2)
        return out.transpose(2, 3).reshape(b, -1, x, y)

    # ChannelRMSNorm, gp.py:224-232
    def channel_scale(self, x, s):
        """skip-layer excitation multiply `x * excite` (reference gp.py:1023-1024 generator, :1812-1813 discriminator)."""
        return x * s.reshape(x.shape[0], x.shape[1], 1, 1).to(x.dtype)

    # the transformer options that the reference does not have: layer norm, rotary positions, attention with a window and sinks,
    # restated from their definitions (no code shared with the product)
    def layer_norm(self, x, weight, bias=None, eps=1e-5):
        x = x.float()
        c = x - x.mean(-1, keepdim=True)
        y = c / (c.square().mean(-1, keepdim=True) + eps).sqrt() * weight.float()
        return y if bias is None else y + bias.float()

    def rotary(self, q, positions, spec, k=None):
        pos = positions if positions.dim() == 3 else positions[None]
        ang = (pos.double()[..., spec.axes] * torch.tensor(spec.freqs, dtype=torch.float64, device=pos.device))[:, None]
        c, s = ang.cos().float(), ang.sin().float()

        def turn(x):
            x, p = x.float(), spec.pairs
            r, rest = x[..., :2 * p], x[..., 2 * p:]
            a, b = (r[..., 0::2], r[..., 1::2]) if spec.interleaved else (r[..., :p], r[..., p:])
            a, b = a * c - b * s, a * s + b * c
            r = torch.stack((a, b), -1).flatten(-2) if spec.interleaved else torch.cat((a, b), -1)
            return torch.cat((r, rest), -1)
        return turn(q) if k is None else (turn(q), turn(k))

    def window_attention(self, q, k, v, *, scale, window=(None, None), sinks=0, key_mask=None, lengths=None):
        B, h, n, d = q.shape
        m = k.shape[2]
        left, right = (n + m if t is None else t for t in window)
        end = torch.full((B,), m, device=q.device) if lengths is None else lengths.long()
        p = (end[:, None] - n + torch.arange(n, device=q.device))[:, :, None]
        j = torch.arange(m, device=q.device)[None, None]
        ok = (p >= 0) & (j < end[:, None, None]) & (j <= p + right) & ((j >= p - left) | (j < sinks))
        if key_mask is not None:
            ok = ok & key_mask[:, None]
        q, k, v = (_r(t.float(), self.bf16) for t in (q, k, v))
        k, v = (t.repeat_interleave(h // k.shape[1], 1) for t in (k, v))
        sim = (q @ k.transpose(-1, -2) * scale).masked_fill(~ok[:, None], -torch.finfo(torch.float32).max)
        attn = sim.softmax(-1) * ok[:, None]
        return _r(attn, self.bf16) @ v

    # nn.GELU() in FeedForward, gp.py:731 (exact erf form)
    def gelu(self, x):
        return F.gelu(x.float())

    # x[:batch_prev_stage], gp.py:1789
    def scaled_add(self, a, b, c, d=None):
        y = (a + b) * c             # gp.py:1493
        return y if d is None else y + d        # gp.py:1495

    def add_cat(self, x, feats):
        ft = feats if feats.shape[0] == x.shape[0] else feats.repeat(x.shape[0] // feats.shape[0], 1, 1, 1)     # gp.py:1797-1803
        return torch.cat((x + ft, ft), dim=0)

    def take_rows(self, x, n, fork=False):
        return (x[:n], x) if fork else x[:n]

    # SqueezeExcite's Reduce('b c h w -> b c', 'mean'), gp.py:300
    def global_mean(self, x, fork=False):
        m = x.float().mean(dim=(2, 3))
        return (m, x) if fork else m

    # ChannelRMSNorm gp.py:224-232; unet RMSNorm unet.py:224-234 (+ the Block's SiLU, unet.py:268-269)
    def channel_rmsnorm(self, x, gamma, act=None):
        x = x.float()
        y = F.normalize(x, dim=1) * (x.shape[1] ** 0.5) * gamma.float().view(1, -1, 1, 1)
        return F.silu(y) if act == 'silu' else y

    # unet Downsample after its conv, unet.py:134-160: (max-pooled map, high-frequency map x - blur(x))
    def maxpool_highfreq(self, x):
        x = x.float()
        return F.max_pool2d(x, kernel_size=2), x - self.blur(x)

    # LinearAttention core, unet.py:338-348
    def linear_attention(self, q, k, v, *, heads, scale):
        b, c, x, y = q.shape
        q, k, v = (t.float().reshape(b, heads, c // heads, x * y) for t in (q, k, v))
        q = q.softmax(dim=-2) * scale
        k = k.softmax(dim=-1)
        context = torch.einsum('bhdn,bhen->bhde', _r(k, self.bf16), _r(v, self.bf16))
        out = torch.einsum('bhde,bhdn->bhen', _r(context, self.bf16), _r(q, self.bf16))
        return out.reshape(b, c, x, y)

    # Blur, gp.py:246-255: kornia filter2d(normalized=True), border_type='reflect'
    def blur(self, x):
        x = x.float()
        c = x.shape[1]
        f = torch.tensor([1., 2., 1.], device=x.device)
        f = (f[None, :] * f[:, None])
        f = f / f.abs().sum()
        xp = F.pad(x, (1, 1, 1, 1), mode='reflect')
        return F.conv2d(xp, f[None, None].expand(c, 1, 3, 3), groups=c)

    # Upsample, gp.py:257-261
    def upsample_blur(self, x):
        return self.blur(F.interpolate(x.float(), scale_factor=2, mode='bilinear', align_corners=False))

    # Discriminator.resize_image_to, gp.py:1683-1684
    def resize_bilinear(self, x, size):
        size = (size, size) if isinstance(size, int) else tuple(size)
        if tuple(x.shape[-2:]) == size:
            return x
        return F.interpolate(x.float(), size, mode='bilinear')

    # F.interpolate default mode, gp.py:2210, :2623
    def resize_nearest(self, x, size):
        size = (size, size) if isinstance(size, int) else tuple(size)
        if tuple(x.shape[-2:]) == size:
            return x
        return F.interpolate(x.float(), size)
