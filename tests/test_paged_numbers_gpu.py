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


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [None, 300])  # a workgroup for each pair (None: or for the longest rows shared out, too), and shared out
def test_large_values_stay_finite(dev, fmt, width):
    """Values near the largest number, in every position: the result is a mean of them. Scores grow along the row by a little (under what moves the running
    maximum), in one head, and are alike in the other."""
    from merv_amd import ops
    hd, lens = 64, [1, 33, 200, 1100, 2300]
    k, v = P.rows_like(lens, 1, hd, 3)
    for x in k:
        x.zero_()
        x[:, 0, 0] = torch.linspace(0, 4, x.shape[0]).to(torch.bfloat16)  # score 4 = 5.8 in base 2
    for i, x in enumerate(v):
        x[:] = (3.0e38 * torch.where(torch.arange(hd) % 2 == 0, 1.0, -1.0)).to(torch.bfloat16)
        x[:, 0, 10:20] = torch.randn(x.shape[0], 10, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
        x[:, 0, 20:30] *= 2.0**-120
    q = torch.zeros(len(lens), 2, hd, dtype=torch.bfloat16)
    q[:, 0, 0] = 1.0
    pool = P.Pool(lens, 1, hd, 16, fmt, dev, width=width)
    kk, vv = pool.fill(k, v)
    want, want_l, tol, tol_l = P.attention(q, kk, vv, 1.0)
    out, lse = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, pool.table.to(dev), i32(lens, dev), scale=1.0, return_lse=True, **pool.scales())
    out = out.cpu().to(P.F64)
    assert torch.isfinite(out).all()
    assert ((out - want).abs() <= tol).all() and ((lse.cpu().to(P.F64) - want_l).abs() <= tol_l).all()


@pytest.mark.parametrize("fmt,hd", [("bf16", 128), ("bf16", 64), ("e4m3", 128), ("e4m3", 64)])
@pytest.mark.parametrize("window", [0, 5000])
def test_long_stretches_of_one_row(dev, fmt, hd, window):
    """A worker that takes more than 32 units of one pair looks up page numbers anew every 32 tiles. 600 rows of 4096 .. 8200 positions (32, 33, 64 and 65
    units) on the same pages, two pairs each: over 100 units a worker, so that whole rows lie in it. A row whose table has one bad page, before, at
    or behind such a border, is NaN, and no other is."""
    from merv_amd import ops
    H, Hkv, page, B = 4, 2, 16, 600
    kinds = [8200, 4096, 4097, 8192, 4224, 4225, 8191, 5000]
    pool = P.Pool([max(kinds)], Hkv, hd, page, fmt, dev, seed=2)
    kk, vv = pool.fill(*P.rows_like([max(kinds)], Hkv, hd, 1))
    g = torch.Generator().manual_seed(5)
    q = torch.randn(len(kinds), H, hd, generator=g).to(torch.bfloat16)
    want, want_l, tol, tol_l = P.attention(q, [kk[0][:n] for n in kinds], [vv[0][:n] for n in kinds], hd**-0.5, window)
    which = torch.arange(B) % len(kinds)
    lens = torch.tensor(kinds)[which]
    table = pool.table.expand(B, -1).clone()
    bad = {40: 4095, 41: 4095, 80: 4096, 81: 4095, 160: 8191, 163: 8191, 240: 8199, 299: 4999, 300: 4223}  # row: position (all seen)
    for n, (b, pos) in enumerate(bad.items()):
        assert int(lens[b]) - (window or 10**6) <= pos < int(lens[b])
        table[b, pos // page] = [-1, pool.k.shape[0], 2**31 - 1][n % 3]
    out, lse = ops.paged_decode_attention(q[which].to(dev), pool.k, pool.v, table.to(dev), i32(lens.tolist(), dev), window=window, return_lse=True,
                                          **pool.scales())
    out, lse = out.cpu().to(P.F64), lse.cpu().to(P.F64)
    rows = torch.tensor(sorted(bad))
    assert torch.isnan(out[rows]).all() and torch.isnan(lse[rows]).all()
    good = torch.ones(B, dtype=torch.bool)
    good[rows] = False
    w = which[good]
    assert ((out[good] - want[w]).abs() <= tol[w]).all() and ((lse[good] - want_l[w]).abs() <= tol_l[w]).all()


def test_the_largest_numbers_round_to_infinity_in_e4m3(dev):
    """From 248 x 2^120 on the nearest e4m3 number is 256 x 2^120 = 2^128: infinite as bf16, in what is read and what is attended to. Below: finite."""
    from merv_amd import ops
    hd, step = 64, 2.0**120
    x = torch.tensor([255.0, 248.0, 247.0, -255.0, -247.0], dtype=P.F64)[:, None].expand(-1, hd) * step
    pool = P.Pool([5] * 5, 1, hd, 16, "e4m3", dev)
    k = torch.zeros(5, 1, hd, dtype=torch.bfloat16, device=dev)
    v = x.to(torch.bfloat16)[:, None].to(dev)
    assert torch.equal(v[:, 0].cpu().to(P.F64), x)
    table, one = pool.table.to(dev), i32([1] * 5, dev)
    ops.paged_cache_write(k, v, pool.k, pool.v, table, i32([0] * 5, dev), **pool.scales())
    want = torch.tensor([math.inf, math.inf, 240 * step, -math.inf, -240 * step], dtype=P.F64)[:, None].expand(-1, hd)
    _, back = ops.paged_cache_read(pool.k, pool.v, table, None, i32([0, 1, 2, 3, 4, 5], dev), 5, **pool.scales())
    assert torch.equal(back[:, 0].cpu().to(P.F64), want)
    out = ops.paged_decode_attention(torch.ones(5, 1, hd, dtype=torch.bfloat16, device=dev), pool.k, pool.v, table, one, **pool.scales())
    assert torch.equal(out[:, 0].cpu().to(P.F64), want)
