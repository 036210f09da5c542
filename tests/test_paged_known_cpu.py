"""CPU: the attention of known tokens (prompts beyond a window, 64 dims, extend()) of merv_amd/paged.py against the formula in 64 bits."""
import pytest
import torch


@pytest.mark.parametrize("H,Hkv", [(4, 4), (6, 2), (3, 1)])
@pytest.mark.parametrize("n,past,window", [(1, 0, 0), (7, 0, 0), (5, 40, 0), (1, 33, 8), (40, 0, 8), (9, 30, 8), (30, 3, 100), (25, 60, 25)])
@pytest.mark.parametrize("scores", [1 << 28, 700, 1])
def test_known_attention(monkeypatch, H, Hkv, n, past, window, scores):
    """In 32 bits whatever the heads, never more scores at a time than it says (or one query's), rounded once. A score is a sum of 64 products that are exact in fp32, two
    more roundings of scale and maximum and an exponential: 2^-17 of a weight at scores of up to 8 covers it; then 2^-8 of the result for the rounding to bf16."""
    from merv_amd import paged
    hd = 64
    g = torch.Generator().manual_seed(n + past)
    q, k, v = (torch.randn(m, h, hd, generator=g).to(torch.bfloat16) for m, h in ((n, H), (n + past, Hkv), (n + past, Hkv)))
    seen = []
    sdpa = paged.F.scaled_dot_product_attention

    def spy(q, k, v, **kw):
        assert q.dtype is k.dtype is v.dtype is torch.float32
        assert q.shape[2] == 1 or H * q.shape[2] * k.shape[2] <= scores
        seen.append(q.shape[2])
        return sdpa(q, k, v, **kw)

    monkeypatch.setattr(paged.F, "scaled_dot_product_attention", spy)
    monkeypatch.setattr(paged, "SCORES", scores)
    wide = torch.zeros(n, 2, H, hd, dtype=torch.bfloat16)
    wide[:, 1] = q
    out = paged.known_attention(wide[:, 1], k, v, window)
    assert sum(seen) == n and out.dtype is torch.bfloat16 and out.shape == q.shape and out.is_contiguous()
    qd, kd, vd = q.double(), k.double(), v.double()
    for i in range(n):
        hi = past + i + 1
        lo = max(0, hi - window) if window else 0
        for h in range(H):
            s = kd[lo:hi, h // (H // Hkv)] @ qd[i, h] * hd**-0.5
            assert float(s.abs().max()) < 8
            p = torch.softmax(s, -1)
            x = vd[lo:hi, h // (H // Hkv)]
            want = p @ x
            assert ((out[i, h].double() - want).abs() <= 2.0**-16 * (p @ x.abs()) + 2.0**-8 * want.abs()).all()


def test_a_pool_is_as_large_as_its_rows_need():
    from merv_amd.paged import PagedKVCache, pool_pages
    assert pool_pages([8000] + [50] * 31, 8192) == 256  # 125 + 31 pages, rounded up to 4 a row on the average; 4096 for 32 rows of 8192
    assert pool_pages([1082] * 8, 1280) == 8 * 20  # rows of one length: all of the table
    assert pool_pages([1000, 1000], 1000) == 2 * 16  # never more than the rows' tables name
    assert pool_pages([10**6, 1], 256) == 8 and pool_pages([0, 0], 256) == 0 and pool_pages([], 256) == 0
    assert pool_pages([100], 4096, 1024) == 1 and pool_pages([1, 1, 1], 4096, 16) == 48
    import random
    rng = random.Random(1)
    for _ in range(200):
        page, rows, most = rng.choice([16, 64, 1024]), rng.randint(1, 20), rng.randint(1, 5000)
        lengths = [rng.randint(0, most) for _ in range(rows)]
        c = PagedKVCache(1, rows, most, 1, 64, "cpu", page_size=page, n_pages=0)
        need = sum(-(-n // page) for n in lengths)
        got = pool_pages(lengths, most, page)
        assert need <= got <= rows * c.width and got < need + rows * max(1, 256 // page)
