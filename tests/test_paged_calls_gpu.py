"""GPU: calls of the paged key / value cache that are refused, or allowed, by what their operands are beside their shapes."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import paged_oracle as P
from test_paged_gpu import i32, same, tables

pytestmark = pytest.mark.gpu


def test_gradients_and_tangents_are_refused_before_anything_is_written(dev):
    from merv_amd import ops
    pool = P.Pool([20, 9], 2, 64, 16, "bf16", dev)
    table, n = pool.table.to(dev), i32([20, 9], dev)
    k, q = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    cos, sin = (t.to(dev) for t in tables(30, 64))
    before = [pool.k.clone(), pool.v.clone()]
    wants = cos.clone().requires_grad_()
    for c, s in ((wants, sin), (cos, wants)):
        with pytest.raises(ValueError, match="requires a gradient"):
            ops.paged_cache_write(k, k, pool.k, pool.v, table, n, q=q, cos=c, sin=s)
    dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
    with fwd.dual_level():
        for call in (lambda: ops.paged_cache_write(dual(k), k, pool.k, pool.v, table, n), lambda: ops.paged_cache_write(k, k, dual(pool.k), pool.v, table, n),
                     lambda: ops.paged_cache_write(k, k, pool.k, pool.v, table, n, q=q, cos=dual(cos), sin=sin),
                     lambda: ops.paged_decode_attention(dual(q), pool.k, pool.v, table, n), lambda: ops.paged_decode_attention(q, pool.k, dual(pool.v), table, n),
                     lambda: ops.paged_cache_read(dual(pool.k), pool.v, table, None, i32([0, 1, 2], dev), 2)):
            with pytest.raises(ValueError, match="tangent"):
                call()
    assert same(pool.k, before[0]) and same(pool.v, before[1])


def test_outputs_that_are_other_operands_are_refused(dev):
    from merv_amd import ops
    pool = P.Pool([20, 9], 2, 64, 16, "bf16", dev)
    table, n = pool.table.to(dev), i32([20, 9], dev)
    x = torch.zeros(6, 2, 2, 64, dtype=torch.bfloat16, device=dev)
    k, v, q, ko = x[:4]
    cos, sin = (t.to(dev) for t in tables(30, 64))
    before = [pool.k.clone(), pool.v.clone()]
    for kw in (dict(q_out=k), dict(q_out=v), dict(q_out=ko, k_out=ko), dict(k_out=v), dict(k_out=q), dict(q_out=q.transpose(0, 1)), dict(k_out=k.transpose(0, 1))):
        with pytest.raises(ValueError, match="must not share memory"):
            ops.paged_cache_write(k, v, pool.k, pool.v, table, n, q=q, cos=cos, sin=sin, **kw)
    with pytest.raises(ValueError, match="must not share memory"):
        ops.paged_cache_read(pool.k, pool.v, table, None, i32([0, 1, 2], dev), 2, k_out=k, v_out=k)
    with pytest.raises(ValueError, match="must not share memory"):
        ops.paged_decode_attention(q, pool.k, pool.v, table, n, out=q.transpose(0, 1))
    assert same(pool.k, before[0]) and same(pool.v, before[1])


@pytest.mark.parametrize("lens,width", [([300, 0, 41], None), ([1500, 0, 41], 200), ([9000], None)])
def test_attention_over_its_queries(dev, lens, width):
    """out=q: the same bits as into another tensor, whole and shared out."""
    from merv_amd import ops
    pool = P.Pool(lens, 2, 128, 16, "bf16", dev, width=width)
    pool.fill(*P.rows_like(lens, 2, 128, 1))
    q = torch.randn(len(lens), 40, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    table, n = pool.table.to(dev), i32(lens, dev)
    want = ops.paged_decode_attention(q, pool.k, pool.v, table, n)
    got = ops.paged_decode_attention(q, pool.k, pool.v, table, n, out=q)
    assert got is q and torch.equal(got, want)
