"""Window attention at the ends of its types' range: values that count although their probability underflows, scores of any size, gradients
that 16 bits hold only scaled. On the host-side emulator and on the GPU."""
import math

import pytest
import torch

from gigagan_pytorch_amd import ops
from test_transformer_ops import DT, att_ref, gen, half_step, normal, qkv, seen, within

WHERE = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
where = pytest.mark.parametrize('where', WHERE)
# queries and keys for the three forward kernels: many rows, few rows, few rows with the keys split over workgroups
SHAPES = [(40, 90), (3, 90), (1, 600)]
shapes = pytest.mark.parametrize('n,m', SHAPES)


@where
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
