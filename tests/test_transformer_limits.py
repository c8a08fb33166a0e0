"""The transformer operators at the ends of what they accept: sizes that no test can hold are put to the host's arithmetic alone."""
import ctypes as C
import random

import pytest
import torch

from gigagan_pytorch_amd import _C, ops

where = pytest.mark.parametrize('where', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])


def window_desc(**kw):
    """a descriptor that the checks accept: its pointers are never followed here"""
    p = torch.zeros(4096).data_ptr()
    d = dict(q=p, k=p, v=p, o=p, o_lo=p, lse=p, d_o=p, dq=p, dk=p, dv=p, dvec=p, B=1, n=1, m=1, h=1, hk=1, d=64, left=-1, right=-1, scale=1.0)
    return _C.WindowDesc(**{**d, **kw})


def test_the_rows_of_a_key_tile():
    """the rows that a key tile's dk and dv visit, over the accepted range of keys (2^28) and rows (2^30): none where every query is far
    behind the tile (keys 2^28 in front of sixteen heads' rows are row -2^32), and the chunks cut them without gap or overlap"""
    lib = _C.lib().lib
    rows = (C.c_int32 * 2)()
    rng = random.Random(0)

    def visited(d, length, k0, chunk=0, chunks=1):
        lib.gg_emu_window_rows(C.byref(d), length, k0, chunk, chunks, rows)
        return (rows[0], rows[1]) if rows[0] <= rows[1] else None
    cases = [(1 << 28, 1, 16, 0, 0, 0, 0), (1 << 28, 5, 100, 7, 3, 0, 128), (1 << 28, 1 << 20, 1024, 0, 0, 0, 1 << 27)]
    for _ in range(2000):
        m, g = round(2 ** rng.uniform(0, 28)), round(2 ** rng.uniform(0, 12))
        n = round(2 ** rng.uniform(0, 30)) // g + 1
        n = min(n, (1 << 30) // g)
        left, right = (rng.choice([-1, 0, round(2 ** rng.uniform(0, 28))]) for _ in range(2))
        cases.append((m, n, g, left, right, rng.choice([0, 0, 1, round(2 ** rng.uniform(0, 28))]), round(2 ** rng.uniform(0, 28)) // 128 * 128 % m // 128 * 128))
    none = 0
    for m, n, g, left, right, sinks, k0 in cases:
        length = rng.choice([m, m, rng.randint(0, m)])
        d = window_desc(m=m, n=n, h=g, left=left, right=right, sinks=sinks)
        # tokens whose position p = length - n + i >= 0 sees a key of the tile that is there
        shift, last = length - n, min(k0 + 127, length - 1)
        lo = max(0, -shift, k0 - right - shift if right >= 0 else 0)
        hi = n - 1 if left < 0 or k0 < min(sinks, m) else min(n - 1, last + left - shift)
        want = (lo * g, hi * g + g - 1) if last >= k0 and lo <= hi else None
        none += want is None
        assert visited(d, length, k0) == want, (m, n, g, left, right, sinks, k0, length)
        if want:
            chunks = rng.randint(2, 64)
            parts = [p for p in (visited(d, length, k0, c, chunks) for c in range(chunks)) if p]
            assert parts[0][0] == want[0] and parts[-1][1] == want[1]
            assert all(b[0] == a[1] + 1 and (b[0] - want[0]) % 64 == 0 for a, b in zip(parts, parts[1:]))
    assert none > 100


def test_the_workspace_query_refuses_what_the_calls_refuse():
    """sizes that no call takes have no workspace: fewer query heads than key heads, head sizes that are not there, products beyond 64 bits"""
    lib = _C.lib().lib
    big = 2 ** 31 - 1
    for bad in (dict(h=1, hk=2), dict(h=3, hk=2), dict(d=48), dict(d=0), dict(m=big), dict(n=big, h=2), dict(B=big, hk=big, h=big), dict(sinks=-1), dict(n=0),
                dict(hk=-1)):
        d = window_desc(**bad)
        for backward in (0, 1):
            assert lib.gg_window_workspace_bytes(C.byref(d), backward) == 0, bad
        assert lib.gg_window_fwd(C.byref(d), None, 0, None) < 0, bad
        assert lib.gg_window_bwd(C.byref(d), None, 0, None) < 0, bad
    assert lib.gg_window_workspace_bytes(C.byref(window_desc(m=8192)), 0) > 0


def test_groups_beyond_the_reciprocal_are_refused():
    """dk / dv turns a row's distance in its tile into tokens by a multiplication with 2^32 / g rounded up: right up to 65504 heads a group,
    wrong from 65537 on, where the call is refused"""
    def quotients(g):
        recip = 0xffffffff // g + 1
        return all((x * recip >> 32) == x // g for x in (0, 1, g - 1, g, g + 1, g + 63))
    assert all(quotients(g) for g in (2, 3, 63, 64, 65, 4097, 65503, 65504)) and not quotients(65537)
    lib = _C.lib().lib
    d = window_desc(h=65505)
    assert lib.gg_window_fwd(C.byref(d), None, 0, None) == -2 and lib.gg_window_bwd(C.byref(d), None, 0, None) == -2
    q, k = torch.zeros(1, 65505, 1, 32, dtype=torch.bfloat16), torch.zeros(1, 1, 1, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='heads a key head'):
        ops.impl.window_attention(q, k, k, scale=1.0)


@pytest.mark.gpu
def test_rotary_of_as_many_tokens_as_a_size_holds():
    """2^31 - 1 tokens of one pair (8 GiB): the tokens at both ends and across the 2^32-byte offsets turn as they do alone"""
    n = 2 ** 31 - 1
    spec = ops.RotarySpec((1,))
    q = torch.zeros((1, 1, n, 2), dtype=torch.bfloat16, device='cuda')
    pos = torch.full((1, 1), 2, dtype=torch.int32, device='cuda')
    at = [0, 1, 1023, 1024, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, n - 1024, n - 1]
    part = torch.randn(1, 1, len(at), 2, device='cuda').to(torch.bfloat16)
    for i, t in enumerate(at):
        q[:, :, t] = part[:, :, i]
    y = ops.impl.rotary(q, pos.expand(n, 1), spec)
    want = ops.impl.rotary(part, pos.expand(len(at), 1), spec)
    assert all(torch.equal(y[:, :, t], want[:, :, i]) for i, t in enumerate(at))
    assert not y[:, :, 2 ** 30 + 2:2 ** 30 + 4096].any() and not y[:, :, 2:1000].any()


def test_row_counts_at_the_end_of_64_bits():
    lib = _C.lib().lib
    p = torch.zeros(4096).data_ptr()
    top = 2 ** 63 - 1
    assert lib.gg_layernorm_fwd(p, 8, p, p, p, None, None, top, 8, 1e-5, 0, None) == -2 and b'too many rows' in lib.gg_last_error()
    assert [lib.gg_layernorm_blocks(r, 512) for r in (1, 4, 5, top - 1, top)] == [1, 1, 2, 512, 512]


def test_the_backward_workspace_is_bounded():
    """at most 1024 chunks of a key tile's fp32 dk and dv (128 MiB with 128 features), however many sinks, rows and heads there are; the
    cases with many sinks asked for 1 to 16 GiB once"""
    lib = _C.lib().lib

    def workspace(B, hk, g, n, m, d, left, right, sinks):
        return lib.gg_window_workspace_bytes(C.byref(window_desc(B=B, h=hk * g, hk=hk, n=n, m=m, d=d, left=left, right=right, sinks=sinks)), 1)
    cases = [(1, 8, 4, 16384, 16384, 128, 127, 0, 4096), (4, 8, 4, 16384, 16384, 128, 127, 0, 4096), (8, 8, 1, 32768, 32768, 128, 127, 0, 1024),
             (8, 8, 1, 32768, 32768, 128, 127, 0, 4096), (1, 8, 1, 16384, 16384, 64, 0, 0, 8192), (1, 8, 4, 16384, 16384, 128, 127, 0, 16384),
             (1, 1, 8, 32640, 32640, 128, 0, 0, 1)]
    rng = random.Random(1)

    def log(bits):
        return round(2 ** rng.uniform(0, bits))
    for _ in range(5000):
        m = log(20)
        n = rng.choice([m, log(20)])
        cases.append((log(6), log(5), log(4), n, m, rng.choice([32, 64, 128]), rng.choice([-1, log(18) - 1]), rng.choice([-1, 0, log(10)]), rng.choice([0, log(18)])))
    for case in cases:
        assert workspace(*case) <= 1024 * 2 * 128 * case[5] * 4, case
    # what was measured keeps its chunks: 11 tiles x 6, one tile x 2, 32 tiles x 16
    for case, chunks in (((3, 2, 3, 777, 1291, 32, 100, 7, 3), 6 * 11 * 6), ((4, 8, 1, 1100, 1100, 32, 40, 0, 3), 32 * 2),
                         ((1, 1, 1, 4096, 4096, 64, -1, 0, 0), 32 * 16), ((8, 8, 1, 4096, 4096, 64, 512, 512, 0), 0)):
        assert workspace(*case) == chunks * 2 * 128 * case[5] * 4, case


@where
@pytest.mark.parametrize('case', [(1, 2, 1, 700, 40, 32, (3, 0), 40), (1, 1, 1, 300, 300, 32, (2, 1), 300), (1, 2, 2, 600, 260, 32, (0, 0), 129)])
def test_many_sinks(where, case):
    """all keys sinks, more rows than keys, a sink tile that is cut beside key tiles that are not: gradients against the definition"""
    from test_transformer_ops import att_run
    att_run(where, case, 'bf16')


@pytest.mark.gpu
@pytest.mark.parametrize('case', [(4, 32, 8, 600, 1500, 64, (31, 0), 1300), (1, 8, 1, 2048, 2048, 128, (15, 0), 1), (2, 4, 2, 3000, 3000, 32, (0, 0), 1000)])
def test_many_sinks_and_heads(case):
    from test_transformer_ops import att_run
    att_run('cuda', case, 'bf16')
