"""GPU: what the attention over the paged cache does to its numbers: weights held in full, large values that stay finite, long stretches of one row."""
import math

import pytest
import torch

import paged_oracle as P

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,width", [(6, None), (900, 200)])  # one tile; shared out over workers, with positions of no weight between
def test_weights_are_held_in_32_bits(dev, fmt, n, width):
    """Values that cancel show the weights' own error. Five positions score 0 (weight 1, exactly), one scores -q: with v1 there and values at the five that
    take away p v1 as far as the cache's numbers allow (2^-4 each, five times), out = (p v1 + sum v) / (5 + p) is what is left.

    u = 2^-24. The score -q log2 e: the constant and the product, 2 u q log2 e <= 3 u for q <= 1, the difference to the maximum 0 is exact; exp2 is off
    by 2 u: p by (3 ln 2 + 2) u <= 5 u of itself. Six terms, their sum of absolute values at most 2.2 p |v1|, added in any order and joined over up
    to eight parts: (6 + 8) u of it. A quotient and a rounding to bf16: 2^-8 of what is left. A weight of 16 bits would be off by up to 2^-17 = 128 u."""
    from merv_amd import ops
    heads, hd = 64, 64
    g = torch.Generator().manual_seed(4)
    q0 = (0.1 + 0.9 * torch.rand(heads, generator=g)).to(torch.bfloat16)
    q = torch.zeros(1, heads, hd, dtype=torch.bfloat16)
    q[0, :, 0] = q0
    p = torch.exp(-q0.to(P.F64))
    at = [3, 7, 131, 450, 700, 899] if n == 900 else [0, 1, 2, 3, 4, 5]  # the first: the position of weight p
    k, v = torch.zeros(n, heads, hd), torch.zeros(n, heads, hd, dtype=P.F64)
    k[:, :, 0] = -2048.0  # a score of -200 or less: no weight
    k[at] = 0.0
    k[at[0], :, 0] = -1.0
    as_held = lambda x: (P.dequantise(*P.quantise(x.to(torch.bfloat16))) if fmt == "e4m3" else x.to(torch.bfloat16).to(P.F64))  # noqa: E731
    v[at[0]] = as_held(0.5 + 0.5 * torch.rand(heads, hd, generator=g, dtype=P.F64))
    left = p[:, None] * v[at[0]]
    for j in at[1:]:
        v[j] = as_held(-left)
        left = left + v[j]
    pool = P.Pool([n], heads, hd, 16, fmt, dev, width=width)
    kk, vv = pool.fill([k.to(torch.bfloat16)], [v.to(torch.bfloat16)])
    assert torch.equal(vv[0], v) and torch.equal(kk[0], k.to(P.F64))
    out = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, pool.table.to(dev), i32([n], dev), scale=1.0, **pool.scales())[0].cpu().to(P.F64)
    total = 5 + p[:, None]
    want = left / total
    terms = p[:, None] * v[at[0]].abs() + v[at[1:]].abs().sum(0)
    assert bool((terms <= 2.2 * p[:, None] * v[at[0]].abs()).all())
    tol = (5 * p[:, None] * v[at[0]].abs() + 14 * terms) * 2.0**-24 / total + 2.0**-8 * want.abs()
    over = (out - want).abs() / tol
    assert bool((over <= 1).all()), (float(over.max()), float((over > 1).double().mean()))
