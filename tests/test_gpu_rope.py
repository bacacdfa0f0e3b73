"""kvq.rope.norm_rope on the GPU against its formula in 64 bits, within one rounding to bf16 of fp32 arithmetic."""
import pytest
import torch

import fp4_ref as R
from kvq import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def angles(positions, r, dtype=torch.float32):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / max(r, 1))
    return torch.cat([a.cos(), a.sin()], -1).to(dtype).to(DEV)


def packed(n, hq, hk, d, seed):
    x = torch.randn(n, (hq + 2 * hk) * d, generator=gen(seed)).to(torch.bfloat16).to(DEV)
    return x, x[:, :hq * d].view(n, hq, d), x[:, hq * d:(hq + hk) * d].view(n, hk, d)


@pytest.mark.parametrize("hq,hk,d,r", [(28, 4, 128, 128), (32, 8, 128, 64), (14, 2, 64, 64), (5, 1, 64, 32), (1, 1, 128, 16),
                                       (3, 3, 128, 112), (32, 1, 64, 48), (16, 16, 128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n", [1, 7, 300])
def test_norm_rope(hq, hk, d, r, interleaved, n):
    table_type, weight_type, pos_type = ((torch.float32, torch.bfloat16, torch.int64), (torch.bfloat16, torch.float32, torch.int32))[n % 3 % 2]
    both, q, k = packed(n, hq, hk, d, n)
    before = both.clone()
    w = [(1 + 0.3 * torch.randn(d, generator=gen(s))).to(weight_type).to(DEV) for s in (1, 2)]
    table = angles(5000, r, table_type)
    pos = torch.randint(0, 5000, (n,), generator=gen(3)).to(pos_type).to(DEV)
    qo, ko = torch.empty(n, hq, d, dtype=torch.bfloat16, device=DEV), torch.empty(n, hk, d, dtype=torch.bfloat16, device=DEV)
    a, b = rope.norm_rope(q, k, pos, table, w[0], w[1], 1e-6, interleaved, qo, ko)
    assert a is qo and b is ko and torch.equal(both, before)
    for x, o, weight in ((q, qo, w[0]), (k, ko, w[1])):
        R.check(o, *R.norm_rope(x, pos, table, weight, 1e-6, interleaved))
    # in place: the same bits, and nothing but q and k
    a, b = rope.norm_rope(q, k, pos, table, w[0], w[1], 1e-6, interleaved)
    assert a is q and b is k and torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(both[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_alone(interleaved):
    _, q, k = packed(40, 8, 2, 128, 1)
    table, pos = angles(100, 96), torch.arange(40, device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rope.norm_rope(q, k, pos, table, interleaved=interleaved, q_out=qo, k_out=ko)
    for x, o in ((q, qo), (k, ko)):
        R.check(o, *R.norm_rope(x, pos, table, None, 0.0, interleaved))
    assert torch.equal(qo[..., 96:], q[..., 96:])


def test_positions_that_the_table_does_not_have():
    """Such tokens' rows stay as they are, in either direction and at either width."""
    for t in (torch.int32, torch.int64):
        _, q, k = packed(6, 4, 2, 64, 1)
        qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
        pos = torch.tensor([0, -1, 99, 100, 2 ** 31 - 1, 5]).to(t).to(DEV)
        rope.norm_rope(q, k, pos, angles(100, 64), torch.ones(64, device=DEV), torch.ones(64, device=DEV), q_out=qo, k_out=ko)
        skip = torch.tensor([False, True, False, True, True, False])
        assert bool((qo[skip.to(DEV)] == 9.0).all()) and bool((ko[skip.to(DEV)] == 9.0).all())
        keep = (~skip).to(DEV)
        R.check(qo[keep], *R.norm_rope(q[keep], pos[keep], angles(100, 64), torch.ones(64, device=DEV), 1e-6, False))


def test_rows_of_zeros_and_other_magnitudes():
    _, q, k = packed(5, 2, 1, 128, 1)
    q[0] = 0
    q[1] *= 1e-12
    q[2] *= 1e12
    k[3] *= 2.0 ** -126
    w = torch.ones(128, device=DEV)
    table, pos = angles(10, 128), torch.arange(5, device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rope.norm_rope(q, k, pos, table, w, w, q_out=qo, k_out=ko)
    assert bool((qo[0] == 0).all())
    for x, o in ((q, qo), (k, ko)):
        R.check(o, *R.norm_rope(x, pos, table, w, 1e-6, False))
    # a value that is no number stays in its row and, behind the rotated channels, does not reach others without a norm
    q[4, 0, 100] = float("inf")
    rope.norm_rope(q, k, pos, angles(10, 64), q_out=qo, k_out=ko)
    assert bool(torch.isfinite(qo[4, 0, :100]).all()) and bool(torch.isfinite(qo[4, 1]).all()) and bool(torch.isinf(qo[4, 0, 100]))


def test_many_tokens_and_strided_tables():
    n = 20001
    _, q, k = packed(n, 32, 8, 128, 1)
    wide = torch.zeros(3000, 136, device=DEV)
    wide[:, :128] = angles(3000, 128)
    pos = torch.randint(0, 3000, (n,), generator=gen(3)).to(DEV)
    w = [(1 + 0.3 * torch.randn(128, generator=gen(s))).to(torch.bfloat16).to(DEV) for s in (1, 2)]
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rope.norm_rope(q, k, pos, wide[:, :128], *w, q_out=qo, k_out=ko)
    for x, o, weight in ((q, qo, w[0]), (k, ko, w[1])):
        R.check(o, *R.norm_rope(x, pos, wide[:, :128], weight, 1e-6, False))
