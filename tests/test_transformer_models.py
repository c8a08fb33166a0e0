"""The models' options that call the transformer operators: the text transformer with layer norm, rotary positions and a window, and the
image self-attention with rotary positions, on the kernels (emulator: tiny; GPU) against the fp32 oracle; the operators in one layer, in a
captured graph, on another stream, and in the trainer."""
import copy

import pytest
import torch

from gigagan_pytorch_amd import Discriminator, Generator, TextEncoder, ops
from gigagan_pytorch_amd.modules import LayerNorm, RMSNorm, SelfAttentionBlock, Transformer
from helpers import rel_err
from oracle.torch_ops import OracleOps

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)
# a layer rounds its path to bf16 some twelve times (norm, projections, turn, probabilities, output, residuals, feed-forward), each by at
# most 2^-9 of the value in the mean square; two layers and the gradient through them add up to 48 x 2^-9 / sqrt(3) at the very worst
TOL = 48 * 2.0 ** -9 / 3 ** 0.5


def run(module, args, cot, inputs):
    y = module(*args)
    y = y if isinstance(y, tuple) else (y,)
    loss = sum((t.float() * c).sum() for t, c in zip(y, cot))
    return [t.detach().float() for t in y], torch.autograd.grad(loss, [*inputs, *module.parameters()], allow_unused=True)


def against_oracle(module, args, n_out, inputs, tol=TOL):
    """outputs and gradients of `module` on the kernels against the oracle, in relative L2"""
    g = torch.Generator().manual_seed(7)
    with ops.use_impl(OracleOps()), torch.no_grad():
        shapes = module(*args)
        shapes = [t.shape for t in (shapes if isinstance(shapes, tuple) else (shapes,))][:n_out]
    cot = [torch.randn(s, generator=g).to(inputs[0].device) for s in shapes]
    with ops.use_impl(OracleOps()):
        ref, gref = run(module, args, cot, inputs)
    got, ggot = run(module, args, cot, inputs)
    for a, b in zip(got[:n_out], ref):
        assert rel_err(a, b) < tol
    names = [f'input {i}' for i in range(len(inputs))] + [n for n, _ in module.named_parameters()]
    for name, a, b in zip(names, ggot, gref):
        assert (a is None) == (b is None), name
        if a is not None and float(b.abs().max()) > 0:
            assert rel_err(a, b) < tol, (name, rel_err(a, b))


@where
@pytest.mark.parametrize('kw', [dict(norm='layer'), dict(rotary=True), dict(window=2), dict(norm='layer', rotary=True, window=(3, 1))],
                         ids=lambda k: ','.join(k))
def test_text_transformer_options(where, kw):
    torch.manual_seed(0)
    b, n, dim = (2, 9, 64) if where == 'cpu' else (4, 78, 128)
    t = Transformer(dim=dim, depth=2, dim_head=32, heads=2, ff_mult=2, **kw).to(where)
    x = torch.randn(b, n, dim, device=where, requires_grad=True)
    mask = torch.arange(n, device=where)[None] < torch.tensor([n, n // 2, n - 1, 1][:b], device=where)[:, None]
    against_oracle(t, (x, mask), 1, [x])


@where
def test_text_encoder_options(where):
    """padded captions; the defaults stay the reference's encoder"""
    torch.manual_seed(0)
    enc = TextEncoder(dim=64, depth=1, dim_head=32, heads=2, clip_dim_latent=48, norm='layer', rotary=True, window=3).to(where)
    plain = TextEncoder(dim=64, depth=1, dim_head=32, heads=2, clip_dim_latent=48)
    assert isinstance(plain.transformer.norm, RMSNorm) and isinstance(enc.transformer.norm, LayerNorm)
    assert set(plain.state_dict()) < set(k.replace('.weight', '.gamma') if '.norm.' in k else k for k in enc.state_dict()) | set(plain.state_dict())
    x = torch.randn(3, 12, 48)
    x[0, 5:] = 0
    x[2, 1:] = 0
    x = x.to(where)
    params = dict(enc.named_parameters())
    with ops.use_impl(OracleOps()), torch.no_grad():
        r0, r1, rm = enc(text_encodings=x)
    with torch.no_grad():
        g0, g1, gm = enc(text_encodings=x)
    assert torch.equal(gm, rm) and rel_err(g0, r0) < TOL and rel_err(g1, r1) < TOL
    enc(text_encodings=x)[0].float().pow(2).sum().backward()
    for name, p in params.items():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name


@where
@pytest.mark.parametrize('dot', [False, True])
def test_self_attention_rotary(where, dot):
    """rows and columns; tied projections (L2 distance) turn once; differentiable twice, as the gradient penalty needs"""
    torch.manual_seed(0)
    size = 4 if where == 'cpu' else 16
    block = SelfAttentionBlock(32, dim_head=64, heads=1, ff_mult=2, dot_product=dot, rotary=True).to(where)
    x = torch.randn(2, 32, size, size, device=where, requires_grad=True)
    against_oracle(block, (x,), 1, [x])

    def penalty():
        y = block(x).float()
        g, = torch.autograd.grad(y.square().mean(), x, create_graph=True)
        return torch.autograd.grad((g.float() * size).square().sum(), [block.attn.to_q.weight, block.attn.to_v.weight])
    if dot and where == 'cpu':
        return          # (16 tokens take the unfused form, whose second derivatives are off by a third with and without rotary positions)
    with ops.use_impl(OracleOps()):
        ref = penalty()
    for a, b in zip(penalty(), ref):
        assert rel_err(a, b) < 2 * TOL          # twice the way


def test_options_off_change_nothing():
    torch.manual_seed(0)
    cfg = dict(image_size=16, dim_capacity=8, dim_max=32, unconditional=True)
    G = Generator(style_network=dict(dim=32, depth=2), self_attn_heads=2, self_attn_dim_head=16, dim_latent=32, **cfg)
    R = Generator(style_network=dict(dim=32, depth=2), self_attn_heads=2, self_attn_dim_head=16, dim_latent=32, self_attn_rotary=True, **cfg)
    assert list(G.state_dict()) == list(R.state_dict())
    R.load_state_dict(G.state_dict())
    z = torch.randn(2, 32)
    with ops.use_impl(OracleOps()), torch.no_grad():
        imgs = []
        for m in (G, R, copy.deepcopy(R)):
            torch.manual_seed(1)
            imgs.append(m(noise=z))
    assert not torch.equal(imgs[0], imgs[1]) and torch.equal(imgs[1], imgs[2])
    D = Discriminator(attn_heads=2, attn_dim_head=16, self_attn_rotary=True, **cfg)
    assert any(getattr(m, 'rotary', None) is not None for m in D.modules())


def test_bad_options():
    for bad in (lambda: Transformer(dim=64, depth=1, norm='batch'), lambda: SelfAttentionBlock(32, dim_head=18, rotary=True),
                lambda: Transformer(dim=64, depth=1, dim_head=33, rotary=True)):
        with pytest.raises(ValueError):
            bad()


def layer(x, w, b, wqkv, pos, spec, mask):
    """the operators one after the other, as a transformer layer strings them together"""
    B, n, dim = x.shape
    q, k, v = ops.impl.linear(ops.impl.layer_norm(x, w, b), wqkv).split([4 * 64, 2 * 64, 2 * 64], dim=-1)
    q, k, v = (t.unflatten(-1, (-1, 64)).transpose(1, 2) for t in (q, k, v))
    q, k = ops.impl.rotary(q, pos, spec, k=k)
    o = ops.impl.window_attention(q, k, v, scale=0.125, window=(40, 0), sinks=3, key_mask=mask)
    return o.transpose(1, 2).flatten(2)


def layer_inputs(dev, B=2, n=300, dim=128):
    g = torch.Generator(device=dev).manual_seed(3)
    rand = lambda *s, dt=torch.float32: torch.randn(s, generator=g, device=dev).to(dt)
    x = rand(B, n, dim, dt=torch.bfloat16).requires_grad_()
    w, b, wqkv = (1 + 0.1 * rand(dim)).requires_grad_(), (0.1 * rand(dim)).requires_grad_(), (rand(8 * 64, dim) * dim ** -0.5).requires_grad_()
    pos = ops.grid_positions((n // 20, 20), dev)
    mask = torch.rand(B, n, generator=g, device=dev) < 0.9
    return [x, w, b, wqkv], pos, ops.RotarySpec((16, 16)), mask, rand(B, n, 4 * 64, dt=torch.bfloat16)


@where
def test_operators_together(where):
    leaves, pos, spec, mask, cot = layer_inputs(where, n=40 if where == 'cpu' else 300)
    y = layer(*leaves, pos, spec, mask)
    got = [y, *torch.autograd.grad(y, leaves, cot)]
    with ops.use_impl(OracleOps()):
        r = layer(*leaves, pos, spec, mask)
        ref = [r, *torch.autograd.grad(r, leaves, cot.float())]
    for a, b in zip(got, ref):
        assert rel_err(a, b) < TOL / 2            # half a layer


@pytest.mark.gpu
def test_operators_in_a_captured_graph():
    """forward and backward captured and replayed, with new inputs, eager work and synchronizations in between: every replay gives the eager
    bits; two graphs captured side by side share nothing"""
    dev = 'cuda'
    leaves, pos, spec, mask, cot = layer_inputs(dev)
    static = [t.detach().clone().requires_grad_() for t in leaves]
    kq = torch.randn(1, 2, 5000, 64, device=dev).bfloat16()

    def step():
        y = layer(*static, pos, spec, mask)
        return [y, *torch.autograd.grad(y, static, cot)]

    def decode():               # key splits and their workspace
        return ops.impl.window_attention(static[0][:, :1, :128].reshape(1, 4, 1, 64).detach(), kq, kq, scale=0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(), decode()
    torch.cuda.current_stream().wait_stream(side)
    del side
    graphs = []
    for fn in (step, decode):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out if isinstance(out, list) else [out], fn))
    for i in range(4):
        with torch.no_grad():
            for s, t in zip(static, leaves):
                s.copy_(t + 0.01 * i)
        for g, out, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, fn in graphs:
            eager = fn()
            eager = eager if isinstance(eager, list) else [eager]
            for a, b in zip(out, eager):
                assert torch.equal(a, b), i
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_operators_on_another_stream():
    """the calls run on torch's current stream: results produced and consumed on a side stream are those of the default stream"""
    leaves, pos, spec, mask, cot = layer_inputs('cuda', n=1000)
    y = layer(*leaves, pos, spec, mask)
    ref = [y, *torch.autograd.grad(y, leaves, cot)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(3):
            y = layer(*leaves, pos, spec, mask)
            got = [y, *torch.autograd.grad(y, leaves, cot)]
        done = [t.clone() for t in got]
    s.synchronize()
    for a, b in zip(done, ref):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_trainer_with_the_options(tmp_path):
    """a few steps of the text-conditioned trainer with every option on, the gradient penalty among them"""
    from gigagan_pytorch_amd import GigaGAN
    torch.manual_seed(0)
    text = dict(dim=64, depth=1, dim_head=32, heads=2, clip_dim_latent=64, norm='layer', rotary=True, window=8)
    gan = GigaGAN(generator=dict(image_size=32, dim_capacity=8, dim_max=64, style_network=dict(dim=64, depth=2, dim_text_latent=64), text_encoder=dict(text),
                                 self_attn_rotary=True, unconditional=False),
                  discriminator=dict(image_size=32, dim_capacity=8, dim_max=64, text_encoder=dict(text), self_attn_rotary=True, unconditional=False),
                  generator_contrastive_loss_weight=0., amp=True, mixed_precision_type='bf16', apply_gradient_penalty_every=2,
                  device=torch.device('cuda', 0), model_folder=str(tmp_path / 'm'), results_folder=str(tmp_path / 'r'))
    g = torch.Generator().manual_seed(1)
    images = torch.rand(4, 3, 32, 32, generator=g).cuda()
    enc = torch.randn(4, 20, 64, generator=g)
    enc[1, 7:] = 0
    enc = enc.cuda()

    class Loader:
        batch_size = 4

        def __iter__(self):
            while True:
                yield images, enc
    it = iter(Loader())
    before = {n: p.detach().clone() for n, p in gan.named_parameters() if 'text_encoder' in n and ('norm' in n or 'to_qkv' in n)}
    for _ in range(4):
        d, gl = gan.train_step(it, 4)
        vals = [float(v) for v in (*d, *gl) if v is not None]
        assert all(abs(v) < float('inf') for v in vals)
    after = dict(gan.named_parameters())
    moved = [n for n, p in before.items() if not torch.equal(p, after[n])]
    assert len(moved) == len(before) > 0, set(before) - set(moved)
