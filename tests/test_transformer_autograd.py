"""The transformer operators as autograd nodes: saved tensors that come back in another layout, forward-mode derivatives, second
derivatives. On the host-side emulator and on the GPU."""
import pytest
import torch

from gigagan_pytorch_amd import ops

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)


def rand(shape, where, seed, dtype=torch.float32):
    g = torch.Generator(device=where).manual_seed(seed)
    return torch.randn(shape, generator=g, device=where).to(dtype)


def operators(where):
    """(name, function of its leaves, leaves): every differentiable operator, small; `x` first"""
    pos = ops.grid_positions((40,), where)
    spec = ops.RotarySpec((16,))
    qkv = [rand((2, h, 40, 32), where, 1 + h, torch.bfloat16) for h in (4, 2, 2)]
    return [('layer_norm', ops.impl.layer_norm, [rand((5, 24), where, 1), rand((24,), where, 2), rand((24,), where, 3)]),
            ('rotary', lambda q, k: torch.cat(ops.impl.rotary(q, pos, spec, k=k), 1), qkv[:2]),
            ('window_attention', lambda q, k, v: ops.impl.window_attention(q, k, v, scale=0.2, window=(9, 3), sinks=1), qkv)]


NAMES = ['layer_norm', 'rotary', 'window_attention']


def operator(name, where):
    return next(o for o in operators(where) if o[0] == name)[1:]


# ---- saved-tensor hooks ----------------------------------------------------------------------------------------------

@where
@pytest.mark.parametrize('name', NAMES)
@pytest.mark.parametrize('hook', ['clone', 'reversed', 'cpu'])
def test_saved_tensors_in_another_layout(where, name, hook):
    """hooks that give the saved tensors back contiguous, with the axes' order in memory turned round, and through host memory: the
    gradients have the same bits"""
    fn, leaves = operator(name, where)
    leaves = [t.requires_grad_() for t in leaves]
    y = fn(*leaves)
    cot = rand(y.shape, where, 9, y.dtype)
    ref = torch.autograd.grad(y, leaves, cot)

    def turned(t):
        if not t.dim():
            return t
        order = list(range(t.dim()))[::-1]
        return t.detach().permute(order).clone(memory_format=torch.contiguous_format).permute(order)
    with {'clone': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), lambda t: t),
          'reversed': lambda: torch.autograd.graph.saved_tensors_hooks(turned, lambda t: t),
          'cpu': lambda: torch.autograd.graph.save_on_cpu(pin_memory=where == 'cuda')}[hook]():
        got = fn(*leaves)
    for a, b in zip(torch.autograd.grad(got, leaves, cot), ref):
        assert torch.equal(a, b)


# ---- second derivatives ----------------------------------------------------------------------------------------------

@where
@pytest.mark.parametrize('name', ['layer_norm', 'window_attention'])
@pytest.mark.parametrize('loss', ['linear', 'square'])
@pytest.mark.parametrize('leaf', [0, 1])
def test_second_derivatives_are_refused_by_name(where, name, loss, leaf):
    """a loss linear in the operator's output (its gradient there is a constant) and one that is not, each with a second term that has a
    second derivative of its own; the derivative asked for one leaf and accumulated for all"""
    fn, leaves = operator(name, where)
    leaves = [t.requires_grad_() for t in leaves]
    y = fn(*leaves).float()
    c = rand(y.shape, where, 4)
    total = ((y if loss == 'linear' else y.pow(2)) * c).sum() + leaves[leaf].float().pow(3).sum()
    g, = torch.autograd.grad(total, leaves[leaf], create_graph=True)
    for second in (lambda: torch.autograd.grad(g.float().pow(2).sum(), leaves[leaf], retain_graph=True), lambda: g.float().sum().backward()):
        with pytest.raises(RuntimeError, match=f'{name}: second derivatives'):
            second()


@where
@pytest.mark.parametrize('name', ['layer_norm', 'window_attention'])
def test_create_graph_alone_is_no_error(where, name):
    """a gradient taken with create_graph=True that nobody differentiates has the bits of the ordinary one"""
    fn, leaves = operator(name, where)
    leaves = [t.requires_grad_() for t in leaves]
    cot = rand(fn(*leaves).shape, where, 4, leaves[0].dtype)
    for a, b in zip(torch.autograd.grad(fn(*leaves), leaves, cot, create_graph=True), torch.autograd.grad(fn(*leaves), leaves, cot)):
        assert torch.equal(a, b) and a.requires_grad


# ---- forward mode ------------------------------------------------------------------------------------------------------

@where
@pytest.mark.parametrize('name', NAMES)
@pytest.mark.parametrize('leaf', [0, 1])
def test_forward_mode_is_refused(where, name, leaf):
    """a tangent is not dropped: the operators have no forward-mode derivatives and say so; without tangents the calls work as ever"""
    fn, leaves = operator(name, where)
    with torch.no_grad():
        ref = fn(*leaves)
        with torch.autograd.forward_ad.dual_level():
            assert torch.equal(fn(*leaves), ref)
            dual = list(leaves)
            dual[leaf] = torch.autograd.forward_ad.make_dual(leaves[leaf], torch.ones_like(leaves[leaf]))
            with pytest.raises(NotImplementedError):
                fn(*dual)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: fn(*leaves[:leaf], t, *leaves[leaf + 1:]), (leaves[leaf],), (torch.ones_like(leaves[leaf]),))
