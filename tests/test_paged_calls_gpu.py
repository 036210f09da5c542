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
