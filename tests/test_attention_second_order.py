"""Second derivatives through the general fused attention (heads of 64 features): self-attention with a dot product over maps whose
pixels are no multiple of 128, as a gradient penalty differentiates it, and the attention itself, against the fp32 oracle."""
import pytest
import torch

from gigagan_pytorch_amd import ops
from gigagan_pytorch_amd.modules import SelfAttentionBlock
from helpers import rel_err
from oracle.torch_ops import OracleOps

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)
# some twelve roundings to bf16 on the way through a block, each 2^-9 of the value at most (2^-9 / sqrt(3) in the mean square), taken
# four times: forward, backward, and both again
TOL = 48 * 2.0 ** -9 / 3 ** 0.5


@where
@pytest.mark.parametrize('rotary', [False, True])
@pytest.mark.parametrize('announced', [False, True])
def test_penalty_through_dot_product_self_attention(where, rotary, announced):
    """with and without the trainer's announcement that the graph will be differentiated twice"""
    torch.manual_seed(0)
    block = SelfAttentionBlock(32, dim_head=64, heads=1, ff_mult=2, dot_product=True, rotary=rotary).to(where)
    x = torch.randn(2, 32, 4, 4, device=where, requires_grad=True)
    weights = [block.attn.to_q.weight, block.attn.to_k.weight, block.attn.to_v.weight, block.attn.null_kv]

    def penalty():
        y = block(x).float()
        g, = torch.autograd.grad(y.square().mean(), x, create_graph=True)
        return torch.autograd.grad((g.float() * 4).square().sum(), weights)
    with ops.use_impl(OracleOps()):
        ref = penalty()
    ops.second_order = announced
    try:
        got = penalty()
    finally:
        ops.second_order = False
    for a, b in zip(got, ref):
        assert rel_err(a, b) < TOL


@where
@pytest.mark.parametrize('null', [False, True])
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('n,m', [(16, 17), (5, 40), (33, 9)])
def test_fused_attention_differentiated_twice(where, null, masked, n, m):
    """first derivatives under create_graph, and their derivatives by q, k, v, the null token and the incoming gradient"""
    g = torch.Generator().manual_seed(n + m)
    B, h = 2, 2
    rand = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(where)
    leaves = [rand(B, n, h * 64), rand(B, m, h * 64), rand(B, m, h * 64), rand(B, n, h * 64)]
    leaves += [rand(h, 64), rand(h, 64)] if null else []
    bias = None
    if masked:
        bias = torch.zeros(B, m, device=where)
        bias[0, m // 2:] = -1e30
    probe = [torch.randn(t.shape, generator=g).to(where) for t in leaves]

    def second(fn, ts):
        q, k, v, do, *nkv = ts
        o = fn(q, k, v, nkv)
        wrt = [q, k, v, *nkv]
        first = torch.autograd.grad(o, wrt, do, create_graph=True)
        total = sum((a.float() * p).sum() for a, p in zip(first, [*probe[:3], *probe[4:]]))
        return [t.detach() for t in first] + list(torch.autograd.grad(total, ts))

    def fused(q, k, v, nkv):
        return ops.FlashAttnGenFn.apply(q, k, v, *(nkv or (None, None)), bias, h, 0.125)

    def plain(q, k, v, nkv):
        q, k, v = (t.unflatten(-1, (h, 64)).transpose(1, 2) for t in (q, k, v))
        b = torch.zeros(B, m, device=where) if bias is None else bias
        if nkv:
            k, v = (torch.cat((t[None, :, None].expand(B, h, 1, 64), u), 2) for t, u in zip(nkv, (k, v)))
            b = torch.nn.functional.pad(b, (1, 0))
        p = (q @ k.transpose(-1, -2) * 0.125 + b[:, None, None]).softmax(-1)
        return (p @ v).transpose(1, 2).flatten(2)
    got = second(fused, [t.clone().requires_grad_() for t in leaves])
    ref = second(plain, [t.float().requires_grad_() for t in leaves])
    for a, b in zip(got, ref):
        assert rel_err(a, b) < TOL / 2           # one operator: P, dP, dS and the results rounded to bf16, twice


@pytest.mark.gpu
def test_trainer_with_dot_product_attention_on_a_small_map(tmp_path):
    """the captured training step, its gradient penalty through 8 x 8 maps of dot-product attention, eager and as captured graphs"""
    from gigagan_pytorch_amd import GigaGAN
    from gigagan_pytorch_amd.data import SyntheticImages
    from gigagan_pytorch_amd.gigagan import cycle
    losses = []
    for graphs in (False, True):
        torch.manual_seed(0)
        gan = GigaGAN(generator=dict(image_size=32, dim_capacity=8, dim_max=64, style_network=dict(dim=64, depth=2), unconditional=True),
                      discriminator=dict(image_size=32, dim_capacity=8, dim_max=64, attn_resolutions=(8,), attn_heads=2, self_attn_dot_product=True,
                                         self_attn_rotary=True, unconditional=True),
                      amp=True, mixed_precision_type='bf16', apply_gradient_penalty_every=2, use_hip_graphs=graphs, device=torch.device('cuda', 0),
                      model_folder=str(tmp_path / f'm{graphs}'), results_folder=str(tmp_path / f'r{graphs}'))
        assert any(getattr(m, 'dot_product', False) for m in gan.D.modules())
        it = cycle(SyntheticImages(4, 32, device=torch.device('cuda', 0)))
        torch.manual_seed(1)
        runs = []
        for _ in range(6):
            d, g = gan.train_step(it, 4)
            runs.append([float(v) for v in (*d, *g) if v is not None])
        assert all(abs(v) < float('inf') for r in runs for v in r)
        losses.append(runs)
    assert len(losses[0]) == len(losses[1]) and all(len(a) == len(b) for a, b in zip(*losses))
