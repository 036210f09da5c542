"""GPU: the paged key / value cache (csrc/paged.hip through merv_amd.ops) against plain implementations in 64 bits on the CPU (paged_oracle)."""
import math

import pytest
import torch

import paged_oracle as P

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def offsets_of(lens):
    o = [0]
    for n in lens:
        o.append(o[-1] + n)
    return o


def tables(n, hd, seed=3):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(n, hd, generator=g) * 6.28
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


def same(a, b):
    """Equal as numbers, NaN where NaN, and zeros of the same sign."""
    a, b = a.float().cpu(), b.float().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9)) and \
        torch.equal(torch.signbit(a) | torch.isnan(a), torch.signbit(b) | torch.isnan(b))


# ---- write ----
def check_write(dev, news, starts, H, Hkv, hd, page, fmt, rope, layout="phs", prompt=True, seed=0, extra=0):
    """`news[b]` new tokens of row b at starts[b]; `extra` tokens behind the last row."""
    from merv_amd import ops
    lens = [max(0, s) + n for s, n in zip(starts, news)]
    pool = P.Pool(lens, Hkv, hd, page, fmt, dev, seed, layout)
    before = [t.clone() if t is not None else None for t in (pool.k, pool.v, pool.ks, pool.vs)]
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(news) + extra
    wide = torch.randn(T, (H + 2 * Hkv) * hd, generator=g).to(torch.bfloat16)
    q, k, v = wide[:, :H * hd].view(T, H, hd), wide[:, H * hd:(H + Hkv) * hd].view(T, Hkv, hd), wide[:, (H + Hkv) * hd:].view(T, Hkv, hd)
    cos, sin = tables(max(lens) + 3, hd)
    wd = wide.to(dev)
    qd, kd, vd = wd[:, :H * hd].view(T, H, hd), wd[:, H * hd:(H + Hkv) * hd].view(T, Hkv, hd), wd[:, (H + Hkv) * hd:].view(T, Hkv, hd)
    kw = dict(q=qd, cos=cos.to(dev), sin=sin.to(dev)) if rope else {}
    k_out = torch.full((T, Hkv, hd), 7.0, dtype=torch.bfloat16, device=dev)
    q_out = torch.full((T, H, hd), 7.0, dtype=torch.bfloat16, device=dev)
    if rope:
        kw["q_out"] = q_out
    off = i32(offsets_of(news), dev) if prompt else None
    got = ops.paged_cache_write(kd, vd, pool.k, pool.v, pool.table.to(dev), i32(starts, dev), off, k_out=k_out, **pool.scales(), **kw)
    assert (got is q_out) if rope else got is None
    # what should be there
    want_q, want_k = torch.full((T, H, hd), 7.0, dtype=torch.bfloat16), torch.full((T, Hkv, hd), 7.0, dtype=torch.bfloat16)
    want = [before[0].float().cpu(), before[1].float().cpu()]
    want_s = [None if t is None else t.cpu() for t in before[2:]]
    t = 0
    for b, (n, s) in enumerate(zip(news, starts)):
        if s >= 0 and n:
            pos = torch.arange(s, s + n)
            kk = P.rotate(k[t:t + n], cos[pos], sin[pos]) if rope else k[t:t + n]
            if rope:
                want_q[t:t + n] = P.rotate(q[t:t + n], cos[pos], sin[pos])
            want_k[t:t + n] = kk
            at, slot = pool.table[b].long()[pos // page], pos % page
            for i, x in enumerate((kk, v[t:t + n])):
                if fmt == "e4m3":
                    x, sc = P.quantise(x)
                    want_s[i][at, :, slot] = sc
                want[i][at, :, slot] = x.float()
        t += n
    assert same(k_out, want_k)
    assert not rope or same(q_out, want_q)
    assert same(pool.k, want[0]) and same(pool.v, want[1])
    for got_s, w in zip((pool.ks, pool.vs), want_s):
        assert w is None or torch.equal(got_s.cpu(), w)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,Hkv,hd,page", [(32, 8, 128, 64), (28, 4, 128, 16), (5, 5, 64, 32), (16, 1, 64, 128), (40, 40, 128, 1024)])
def test_write_prompts(dev, fmt, H, Hkv, hd, page):
    check_write(dev, [7, 0, 65, 1], [0, 3, 30, page], H, Hkv, hd, page, fmt, rope=True)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("layout", ["phs", "psh", "hps"])
def test_write_layouts(dev, fmt, rope, layout):
    check_write(dev, [33, 2], [0, 15], 8, 2, 128, 16, fmt, rope, layout)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 130])
def test_write_one_token_a_row(dev, rows):
    check_write(dev, [1] * rows, [(37 * i) % 100 for i in range(rows)], 4, 2, 64, 32, "e4m3", True, prompt=False)


def test_write_many_rows_of_prompts(dev):
    check_write(dev, [(i * 5) % 4 for i in range(150)], [(i * 11) % 40 for i in range(150)], 2, 1, 64, 16, "bf16", True)


@pytest.mark.parametrize("prompt", [True, False])
def test_write_leaves_idle_rows_and_tokens_behind_the_last_alone(dev, prompt):
    check_write(dev, [1, 1, 1, 1], [4, -1, 0, -5], 4, 2, 128, 16, "e4m3", True, prompt=prompt, extra=3 if prompt else 0)


def test_write_in_place_and_from_other_strides(dev):
    """Queries and keys rotated where they are; keys and values given head by head ([heads, T, hd] in memory)."""
    from merv_amd import ops
    T, H, Hkv, hd, page = 21, 6, 3, 128, 16
    pool = P.Pool([T], Hkv, hd, page, "bf16", dev)
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(n, T, hd, generator=g).to(torch.bfloat16) for n in (H, Hkv, Hkv))
    cos, sin = tables(T, hd)
    qd, kd, vd = (x.to(dev).transpose(0, 1) for x in (q, k, v))
    got = ops.paged_cache_write(kd, vd, pool.k, pool.v, pool.table.to(dev), i32([0], dev), i32([0, T], dev), q=qd, cos=cos.to(dev), sin=sin.to(dev),
                                q_out=qd, k_out=kd)
    assert got is qd
    kw = P.rotate(k.transpose(0, 1), cos, sin)
    assert same(qd, P.rotate(q.transpose(0, 1), cos, sin)) and same(kd, kw)
    at, slot = pool.table[0].long()[torch.arange(T) // page], torch.arange(T) % page
    assert same(pool.k.cpu()[at, :, slot], kw) and same(pool.v.cpu()[at, :, slot], v.transpose(0, 1))


def test_write_quantises_what_is_odd(dev):
    """Zeros, the smallest and largest bf16 numbers, infinities, NaN, ties of the rounding, and amax just under and over a scale's border."""
    from merv_amd import ops
    hd = 64
    rows = [torch.zeros(hd), torch.full((hd,), -0.0), torch.full((hd,), 2.0**-133), torch.full((hd,), 3.3895e38), torch.full((hd,), math.inf),
            torch.full((hd,), math.nan), torch.tensor([448.0, 17.0, 19.0, 21.0, -17.0, 0.001953125, 0.0009765625, 0.0029296875] * 8),
            torch.tensor([450.0] + [1.0] * 63), torch.tensor([1.75] + [0.01] * 63), torch.tensor([1.7578125] + [0.01] * 63),
            torch.tensor([math.inf, -math.inf, math.nan, 3.0] * 16), torch.tensor([1e38, 1e-38] * 32), torch.tensor([2.0**-126, 2.0**-130] * 32)]
    x = torch.stack(rows).to(torch.bfloat16)[:, None]  # [T, 1, hd]
    T = x.shape[0]
    pool = P.Pool([T], 1, hd, 16, "e4m3", dev)
    ops.paged_cache_write(x.to(dev), x.to(dev), pool.k, pool.v, pool.table.to(dev), i32([0], dev), i32([0, T], dev), **pool.scales())
    val, sc = P.quantise(x)
    page = int(pool.table[0, 0])
    for pages, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
        assert torch.equal(scales[page, 0, :T].cpu(), sc[:, 0])
        assert same(pages[page, 0, :T], val[:, 0].float())


def test_write_without_a_page_shows(dev):
    """A page number out of range, a position behind the table, one behind the rotary tables: nothing is stored elsewhere, and the rotated rows are NaN."""
    from merv_amd import ops
    H, Hkv, hd, page = 4, 2, 64, 16
    pool = P.Pool([40, 40, 40, 40], Hkv, hd, page, "e4m3", dev)
    table = pool.table.clone()
    table[0, 0], table[1, 0] = pool.k.shape[0], -1
    cos, sin = tables(20, hd)
    g = torch.Generator().manual_seed(1)
    k, v, q = (torch.randn(4, n, hd, generator=g).to(torch.bfloat16) for n in (Hkv, Hkv, H))
    k_out = torch.zeros(4, Hkv, hd, dtype=torch.bfloat16, device=dev)
    before = [t.clone() for t in (pool.k, pool.v, pool.ks, pool.vs)]
    got = ops.paged_cache_write(k.to(dev), v.to(dev), pool.k, pool.v, table.to(dev), i32([3, 5, 48, 30], dev), q=q.to(dev), cos=cos.to(dev),
                                sin=sin.to(dev), k_out=k_out, **pool.scales())
    assert torch.isnan(got).all() and torch.isnan(k_out).all()
    want = [t.clone().cpu() for t in before]
    at, slot = pool.place(3, 30)  # the last has a page: its key is NaN there, its value is written
    val, sc = P.quantise(v[3])
    want[0].view(torch.uint8)[at, :, slot] = torch.full((Hkv, hd), math.nan).to(torch.float8_e4m3fn).view(torch.uint8)
    want[2][at, :, slot] = 1
    want[1].view(torch.uint8)[at, :, slot] = val.float().to(torch.float8_e4m3fn).view(torch.uint8)
    want[3][at, :, slot] = sc
    assert same(pool.k, want[0]) and same(pool.v, want[1]) and torch.equal(pool.ks.cpu(), want[2]) and torch.equal(pool.vs.cpu(), want[3])


# ---- read ----
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("Hkv,hd,page,layout", [(8, 128, 64, "phs"), (3, 64, 16, "psh"), (1, 128, 1024, "hps"), (40, 128, 32, "phs")])
def test_read(dev, fmt, Hkv, hd, page, layout):
    """Also from a later position, with an idle row, into given strided outputs whose rows behind the last stay as they were."""
    from merv_amd import ops
    lens = [1, 70, 0, 33, 129]
    pool = P.Pool(lens, Hkv, hd, page, fmt, dev, layout=layout)
    kk, vv = pool.fill(*P.rows_like(lens, Hkv, hd, 2))
    T = sum(lens)
    k, v = ops.paged_cache_read(pool.k, pool.v, pool.table.to(dev), None, i32(offsets_of(lens), dev), T, **pool.scales())
    assert same(k, torch.cat(kk)) and same(v, torch.cat(vv))
    first, news = [0, 30, 0, -1, 128], [1, 40, 0, 4, 1]
    wide = torch.full((sum(news) + 2, 2, Hkv, hd), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.paged_cache_read(pool.k, pool.v, pool.table.to(dev), i32(first, dev), i32(offsets_of(news), dev), sum(news) + 2, k_out=wide[:, 0],
                               v_out=wide[:, 1], **pool.scales())
    assert got[0].data_ptr() == wide.data_ptr()
    for x, rows in ((wide[:, 0], kk), (wide[:, 1], vv)):
        seven = torch.full((1, Hkv, hd), 7.0, dtype=P.F64)
        want = torch.cat([rows[0], rows[1][30:70], seven.expand(4, -1, -1), rows[4][128:129], seven.expand(2, -1, -1)])
        assert same(x, want)


def test_read_without_a_page_is_nan(dev):
    from merv_amd import ops
    pool = P.Pool([40, 20], 2, 64, 16, "e4m3", dev)
    kk, _ = pool.fill(*P.rows_like([40, 20], 2, 64, 2))
    table = pool.table.clone()
    table[0, 1] = 10**9
    k, v = ops.paged_cache_read(pool.k, pool.v, table.to(dev), None, i32([0, 60, 80], dev), 80, **pool.scales())
    want = torch.full((80, 2, 64), math.nan, dtype=P.F64)
    want[:16], want[32:40], want[60:] = kk[0][:16], kk[0][32:], kk[1]  # 48 .. 59: behind the row's table
    assert same(k, want) and torch.isnan(v[16:32]).all() and torch.isnan(v[48:60]).all() and not torch.isnan(v[60:]).any()


# ---- attention ----
def check_attention(dev, lens, H, Hkv, hd, page, fmt, window=0, layout="phs", seed=0, scale=None, width=None, q_gain=1.0):
    from merv_amd import ops
    pool = P.Pool(lens, Hkv, hd, page, fmt, dev, seed, layout, width=width)
    kk, vv = pool.fill(*P.rows_like(lens, Hkv, hd, seed + 1))
    g = torch.Generator().manual_seed(seed + 2)
    q = (q_gain * torch.randn(len(lens), H, hd, generator=g)).to(torch.bfloat16)
    table = pool.table.clone()
    if window:  # pages before the window may be given away
        for b, n in enumerate(lens):
            table[b, :max(0, n - window) // page] = -1
    sc = hd**-0.5 if scale is None else scale
    want, want_l, tol, tol_l = P.attention(q, kk, vv, sc, window)
    got, lse = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, table.to(dev), i32(lens, dev), window=window, return_lse=True, scale=scale,
                                          **pool.scales())
    alone = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, table.to(dev), i32(lens, dev), window=window, scale=scale, **pool.scales())
    assert torch.equal(got, alone)  # the same bits again
    got, lse = got.cpu().to(P.F64), lse.cpu().to(P.F64)
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    assert (over <= 0).all(), (float(over.max()), [int(i) for i in torch.nonzero(over == over.max())[0]])
    empty = torch.tensor([n == 0 for n in lens])
    assert (got[empty] == 0).all() and (lse[empty] == -math.inf).all()
    assert ((lse - want_l).abs()[~empty] <= tol_l[~empty]).all(), float(((lse - want_l).abs() - tol_l)[~empty].max())


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 1, 128, 16), (2, 2, 64, 64), (7, 1, 64, 32), (8, 4, 128, 256)])
def test_attention_lengths(dev, fmt, H, Hkv, hd, page):
    check_attention(dev, EDGES, H, Hkv, hd, page, fmt)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (28, 4), (16, 1), (17, 1), (40, 2), (33, 1), (64, 2)])
def test_attention_heads(dev, fmt, H, Hkv):
    check_attention(dev, [100, 1, 259], H, Hkv, 128, 32, fmt)


@pytest.mark.parametrize("n", EDGES[:8] + [1049, 2500])
def test_attention_one_row(dev, n):
    check_attention(dev, [n], 8, 2, 128, 16, "bf16", width=200)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 128, 1000])
def test_attention_window(dev, fmt, window):
    check_attention(dev, [0, 1, 16, 100, 129, 300, 517, 1200], 4, 2, 64, 16, fmt, window=window)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["psh", "hps"])
def test_attention_layouts(dev, fmt, layout):
    check_attention(dev, [200, 0, 31, 700], 8, 2, 128, 64, fmt, layout=layout)


def test_attention_many_rows(dev):
    """More rows than a block's threads, most of them short, and one long: the long one is split over many blocks, blocks hold many rows."""
    lens = [(i * 7) % 40 for i in range(300)]
    lens[170], lens[299] = 3000, 1
    check_attention(dev, lens, 2, 1, 64, 16, "bf16")


def test_attention_rows_that_fill_the_card(dev):
    check_attention(dev, [150 + 13 * (i % 17) for i in range(70)], 16, 16, 64, 32, "e4m3")


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_attention_short_rows_in_a_large_table(dev, fmt):
    """The table's capacity, which the launch goes by, is far over the lengths, which the kernel goes by: 140 and 520 pairs left whole by the split kernel, 60 and
    4100 pairs of a few units shared out by it."""
    check_attention(dev, [0, 1, 700] + [100 + 9 * i for i in range(32)], 4, 4, 64, 64, fmt, width=100)
    check_attention(dev, [40 + 5 * i for i in range(65)], 8, 8, 64, 64, fmt, width=100)
    check_attention(dev, [513, 129, 0, 1024] * 5, 3, 3, 64, 64, fmt, width=100)
    check_attention(dev, [5, 130] * 21, 100, 100, 64, 64, fmt, width=70)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_attention_pages_of_sixteen_in_unsplit_rows(dev, fmt):
    """Rows of up to 2048 positions, a workgroup for each pair, with more pages than a wave has lanes."""
    check_attention(dev, [2048, 0, 1500] + [33 * i for i in range(1, 30)], 8, 4, 64, 16, fmt)


def test_attention_joins_of_many_parts(dev):
    """One row over all workers: more than 16 partial sums to join, one pair (16 heads) and three; and rows that change within a worker."""
    check_attention(dev, [9000], 16, 1, 64, 32, "bf16")
    check_attention(dev, [5000, 3], 3, 3, 64, 16, "e4m3")
    check_attention(dev, [4000 + 100 * i for i in range(14)], 5, 5, 64, 256, "bf16")


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_attention_split_over_blocks_of_heads(dev, fmt):
    """20 query heads a key head (two blocks of 16 columns) and 128 dims, a row over many workers beside short ones."""
    check_attention(dev, [5000, 3, 0, 130], 40, 2, 128, 32, fmt)


@pytest.mark.parametrize("width", [100, 200])
def test_attention_thousands_of_rows(dev, width):
    """More rows than a lane of the prefix sum has one of, short in a large table. At 100 pages a row one workgroup a row without a plan; at 200 the plan
    leaves 2000 rows whole and shares 4500 out."""
    check_attention(dev, [(i * 7) % 30 for i in range(2000)], 1, 1, 64, 16, "bf16", width=width)
    check_attention(dev, [(i * 11) % 20 for i in range(4500)], 1, 1, 64, 16, "bf16", width=width)


def test_attention_strided_operands(dev):
    """Queries that are columns of a projection, an output that is columns of something wider, a table that is part of a larger one, every other row."""
    from merv_amd import ops
    lens, H, Hkv, hd = [300, 17, 1400], 8, 2, 128
    pool = P.Pool(lens, Hkv, hd, 32, "e4m3", dev)
    kk, vv = pool.fill(*P.rows_like(lens, Hkv, hd, 1))
    wide = torch.randn(6, 3 * H * hd, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    q = wide[::2, H * hd:2 * H * hd].view(3, H, hd)
    out = torch.full((3, 2, H, hd), 7.0, dtype=torch.bfloat16, device=dev)
    big = torch.full((6, pool.width + 5), -9, dtype=torch.int32, device=dev)
    big[::2, 2:2 + pool.width] = pool.table.to(dev)
    got, lse = ops.paged_decode_attention(q, pool.k, pool.v, big[::2, 2:2 + pool.width], i32(lens, dev), out=out[:, 1], return_lse=True, **pool.scales())
    assert got.data_ptr() == out[:, 1].data_ptr() and (out[:, 0] == 7).all()
    want, want_l, tol, tol_l = P.attention(q.cpu(), kk, vv, hd**-0.5)
    assert ((got.cpu().to(P.F64) - want).abs() <= tol).all() and ((lse.cpu().to(P.F64) - want_l).abs() <= tol_l).all()


def test_attention_peaked_and_flat(dev):
    """Scores of some hundreds, where all weight is on one position, and a scale of zero, where all weigh the same."""
    check_attention(dev, [700, 40], 4, 2, 128, 32, "bf16", q_gain=30.0)
    check_attention(dev, [700, 40], 4, 2, 128, 32, "bf16", scale=0.0)


@pytest.mark.parametrize("width", [None, 200])  # left whole, and shared out
def test_attention_bad_rows_are_nan_alone(dev, width):
    from merv_amd import ops
    lens = [300, 300, 300, 300, 0]
    pool = P.Pool(lens, 2, 64, 16, "bf16", dev, width=width)
    pool.fill(*P.rows_like(lens, 2, 64, 1))
    table = pool.table.clone()
    table[1, 9], table[2, 0] = pool.k.shape[0], -1
    g = torch.Generator().manual_seed(2)
    q = torch.randn(5, 4, 64, generator=g).to(torch.bfloat16).to(dev)
    n = i32([300, 300, 300, 16 * table.shape[1] + 1, -3], dev)
    out, lse = ops.paged_decode_attention(q, pool.k, pool.v, table.to(dev), n, return_lse=True)
    good, good_l = ops.paged_decode_attention(q, pool.k, pool.v, pool.table.to(dev), i32(lens, dev), return_lse=True)
    assert torch.isnan(out[1:4]).all() and torch.isnan(lse[1:4]).all()
    assert not torch.isnan(good).any() and (out[4] == 0).all() and (lse[4] == -math.inf).all()
    assert (out[0].float() - good[0].float()).abs().max() <= 2.0**-7 * good[0].abs().max() and torch.allclose(lse[0], good_l[0], atol=1e-5)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_attention_odd_values_in_seen_positions(dev, value, where):
    """They do what they do in the formula: NaN where it has NaN, infinite or finite where it has that."""
    from merv_amd import ops
    n, hd = 200, 64
    pool = P.Pool([n, n], 1, hd, 16, "bf16", dev)
    k, v = P.rows_like([n, n], 1, hd, 1)
    q = torch.randn(2, 2, hd, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    if where == "k":
        q[0, 0, 3], q[0, 1, 3] = 1.0, -1.0  # with an infinity: a score of +inf in one head, of -inf in the other
        k[0][150, 0, 3] = value
    else:
        v[0][150, 0, 5] = value
    kk, vv = pool.fill(k, v)
    out = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, pool.table.to(dev), i32([n, n], dev)).cpu()
    want = []
    for b in range(2):
        p = torch.softmax(q[b].to(P.F64) @ kk[b][:, 0].T * hd**-0.5, -1)
        want.append(p @ vv[b][:, 0])
    want = torch.stack(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.allclose(out[fine].to(P.F64), want[fine], rtol=2.0**-8, atol=1e-4)


def test_attention_all_scores_minus_infinity(dev):
    """Seen positions that all weigh nothing: 0 / 0, as the formula says; a first part that does, with finite scores behind it, does not disturb them."""
    from merv_amd import ops
    hd, n = 64, 900
    k, v = P.rows_like([n, n], 1, hd, 1)
    k[0][:, 0, 0] = -math.inf
    k[1][:700, 0, 0] = -math.inf
    q = torch.ones(2, 1, hd).to(torch.bfloat16)
    pool = P.Pool([n, n], 1, hd, 16, "bf16", dev)
    kk, vv = pool.fill(k, v)
    out = ops.paged_decode_attention(q.to(dev), pool.k, pool.v, pool.table.to(dev), i32([n, n], dev)).cpu()
    p = torch.softmax(kk[1][:, 0] @ q[1, 0].to(P.F64) * hd**-0.5, -1)
    assert torch.isnan(out[0]).all() and torch.allclose(out[1, 0].to(P.F64), p @ vv[1][:, 0], rtol=2.0**-8, atol=1e-4)


def test_offsets_past_32_bits(dev):
    """Pages whose elements lie more than 2^32 from the first: written, read and attended to."""
    from merv_amd import ops
    Hkv, hd, page, n_pages = 8, 128, 64, 70000  # 65536 elements a page: the last starts at 4.6e9
    k_pages = torch.empty(n_pages, Hkv, page, hd, dtype=torch.bfloat16, device=dev)
    v_pages = torch.empty_like(k_pages)
    n = 100
    table = i32([[n_pages - 1, n_pages - 2]], dev)
    k, v = P.rows_like([n], Hkv, hd, 3)
    ops.paged_cache_write(k[0].to(dev), v[0].to(dev), k_pages, v_pages, table, i32([0], dev), i32([0, n], dev))
    assert same(k_pages[-1].transpose(0, 1)[:page], k[0][:page]) and same(v_pages[-2].transpose(0, 1)[:n - page], v[0][page:])
    kr, vr = ops.paged_cache_read(k_pages, v_pages, table, None, i32([0, n], dev), n)
    assert same(kr, k[0]) and same(vr, v[0])
    q = torch.randn(1, 16, hd, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = ops.paged_decode_attention(q.to(dev), k_pages, v_pages, table, i32([n], dev)).cpu().to(P.F64)
    want, _, tol, _ = P.attention(q, k, v, hd**-0.5)
    assert ((out - want).abs() <= tol).all()


# ---- together, as a decoding loop uses them ----
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("graph", [False, True])
def test_prompts_then_steps(dev, fmt, graph):
    """Ragged prompts written, then eight steps of write + attention for the batch (one captured and replayed, its lengths counting on the device, with
    eager work between replays), each against the formula on what the cache holds; at the end the cache is read back."""
    from merv_amd import ops
    H, Hkv, hd, page, steps = 8, 2, 128, 16, 8
    lens = [37, 1, 160, 9]
    total = [n + steps for n in lens]
    pool = P.Pool(total, Hkv, hd, page, fmt, dev)
    table = pool.table.to(dev)
    k, v = P.rows_like(total, Hkv, hd, 4)
    cos, sin = tables(300, hd)
    cosd, sind = cos.to(dev), sin.to(dev)
    stored = [P.rotate(k[b], cos[:total[b]], sin[:total[b]]) for b in range(4)]
    held = [[P.dequantise(*P.quantise(x)) if fmt == "e4m3" else x.to(P.F64) for x in xs] for xs in (stored, v)]
    cat = lambda xs: torch.cat([x[:n] for x, n in zip(xs, lens)]).to(dev)  # noqa: E731
    ops.paged_cache_write(cat(k), cat(v), pool.k, pool.v, table, i32([0] * 4, dev), i32(offsets_of(lens), dev), cos=cosd, sin=sind, **pool.scales())
    g = torch.Generator().manual_seed(9)
    qs = torch.randn(steps, 4, H, hd, generator=g).to(torch.bfloat16)
    q, kn, vn = (torch.empty(4, n, hd, dtype=torch.bfloat16, device=dev) for n in (H, Hkv, Hkv))
    pos, length = i32(lens, dev), i32([n + 1 for n in lens], dev)

    def step():
        rotated = ops.paged_cache_write(kn, vn, pool.k, pool.v, table, pos, q=q, cos=cosd, sin=sind, **pool.scales())
        out = ops.paged_decode_attention(rotated, pool.k, pool.v, table, length, **pool.scales())
        pos.add_(1)
        length.add_(1)
        return out

    def load(s):
        q.copy_(qs[s])
        kn.copy_(torch.stack([k[b][lens[b] + s] for b in range(4)]))
        vn.copy_(torch.stack([v[b][lens[b] + s] for b in range(4)]))

    cg = None
    if graph:
        load(0)
        saved = [t.clone() for t in (pos, length)]
        step()  # warm-up; writes what the first replay writes again
        torch.cuda.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            captured = step()
        pos.copy_(saved[0])
        length.copy_(saved[1])
    for s in range(steps):
        load(s)
        if cg is None:
            out = step()
        else:
            cg.replay()
            out = captured
            torch.randn(1000, device=dev).sum()  # the program's own work
        at = torch.tensor([lens[b] + s for b in range(4)])
        qr = P.rotate(qs[s], cos[at], sin[at])
        want, _, tol, _ = P.attention(qr, [held[0][b][:at[b] + 1] for b in range(4)], [held[1][b][:at[b] + 1] for b in range(4)], hd**-0.5)
        assert ((out.cpu().to(P.F64) - want).abs() <= tol).all(), s
    kr, vr = ops.paged_cache_read(pool.k, pool.v, table, None, i32(offsets_of(total), dev), sum(total), **pool.scales())
    assert same(kr, torch.cat(held[0])) and same(vr, torch.cat(held[1]))


def test_two_streams_at_once(dev):
    """The same call on two streams, over and over, and one graph replayed on each: no state is shared, every result has the same bits."""
    from merv_amd import ops
    lens = [1500, 700, 1, 90]
    pools = [P.Pool(lens, 2, 128, 16, "bf16", dev, seed=i) for i in range(2)]
    qs = []
    for i, pool in enumerate(pools):
        pool.fill(*P.rows_like(lens, 2, 128, i))
        qs.append(torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(dev))
    n, tabs = i32(lens, dev), [pool.table.to(dev) for pool in pools]
    call = lambda i: ops.paged_decode_attention(qs[i], pools[i].k, pools[i].v, tabs[i], n)  # noqa: E731
    first = [call(0).clone(), call(1).clone()]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)], [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=streams[i]):
            outs.append(call(i))
        graphs.append(gr)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, first[i]) for x in got[i])


def test_nothing_to_do(dev):
    from merv_amd import ops
    pool = P.Pool([5], 2, 64, 16, "bf16", dev)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    empty = torch.empty(0, 3, dtype=torch.int32, device=dev)
    ops.paged_cache_write(none, none, pool.k, pool.v, pool.table.to(dev), i32([0], dev), i32([0, 0], dev))
    ops.paged_cache_write(none, none, pool.k, pool.v, empty, i32([], dev))
    k, v = ops.paged_cache_read(pool.k, pool.v, pool.table.to(dev), None, i32([0, 0], dev), 0)
    assert k.shape == (0, 2, 64)
    out, lse = ops.paged_decode_attention(none, pool.k, pool.v, empty, i32([], dev), return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    # a table without columns: every row is empty
    q = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=dev)
    out = ops.paged_decode_attention(q, pool.k, pool.v, torch.empty(2, 0, dtype=torch.int32, device=dev), i32([0, 0], dev))
    assert (out == 0).all()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [4, 200])
def test_a_pool_without_pages(dev, fmt, width):
    """Every position is one without a page: nothing is stored, queries and keys come out as NaN, what is read is NaN; a row of length 0 is as ever."""
    from merv_amd import ops
    kind = torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn
    pages = [torch.empty(0, 2, 16, 64, dtype=kind, device=dev) for _ in range(2)]
    sc = {} if fmt == "bf16" else {n: torch.empty(0, 2, 16, dtype=torch.uint8, device=dev) for n in ("k_scales", "v_scales")}
    table = torch.zeros(3, width, dtype=torch.int32, device=dev)
    k, q = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=dev), torch.ones(3, 4, 64, dtype=torch.bfloat16, device=dev)
    cos, sin = (t.to(dev) for t in tables(64, 64))
    k_out = torch.zeros_like(k)
    q_out = ops.paged_cache_write(k, k, *pages, table, i32([0, 20, 3], dev), q=q, cos=cos, sin=sin, k_out=k_out, **sc)
    assert torch.isnan(q_out).all() and torch.isnan(k_out).all()
    kk, vv = ops.paged_cache_read(*pages, table, None, i32([0, 2, 2, 5], dev), 5, **sc)
    assert torch.isnan(kk).all() and torch.isnan(vv).all()
    out, lse = ops.paged_decode_attention(q, *pages, table, i32([40, 0, 64], dev), return_lse=True, **sc)
    assert torch.isnan(out[[0, 2]]).all() and torch.isnan(lse[[0, 2]]).all() and (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_the_wrappers_refuse(dev):
    """What the tensors alone show, before any launch; nothing is written."""
    from merv_amd import ops
    pool = P.Pool([20, 9], 2, 64, 16, "bf16", dev)
    table, n = pool.table.to(dev), i32([20, 9], dev)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    cos = torch.zeros(30, 64, dtype=torch.bfloat16, device=dev)
    e4 = pool.k.to(torch.float8_e4m3fn)
    sc = torch.zeros(pool.k.shape[:3], dtype=torch.uint8, device=dev)

    def write(k=k, v=k, kp=pool.k, vp=pool.v, table=table, start=n, off=None, **kw):
        ops.paged_cache_write(k, v, kp, vp, table, start, off, **kw)

    def read(start=None, off=i32([0, 1, 2], dev), total=2, **kw):
        ops.paged_cache_read(pool.k, pool.v, table, start, off, total, **kw)

    def att(q=q, kp=pool.k, vp=pool.v, table=table, lens=n, **kw):
        ops.paged_decode_attention(q, kp, vp, table, lens, **kw)

    grad = k.clone().requires_grad_()
    shared = pool.k[:1].expand(4, -1, -1, -1)
    cases = [
        (write, dict(kp=pool.k.float(), vp=pool.v.float()), "float8_e4m3fn"), (write, dict(kp=pool.k[0], vp=pool.v[0]), "CUDA pages"),
        (write, dict(vp=pool.v.transpose(1, 2)), "v_pages"), (write, dict(kp=e4, vp=e4.clone()), "need k_scales"), (write, dict(k_scales=sc, v_scales=sc), "no scales"),
        (write, dict(kp=e4, vp=e4.clone(), k_scales=sc[:1], v_scales=sc[:1]), "uint8 scales"), (write, dict(vp=pool.k), "share memory"),
        (write, dict(kp=e4, vp=e4.clone(), k_scales=sc, v_scales=sc), "share memory"), (write, dict(kp=shared, vp=pool.v[:1].expand(4, -1, -1, -1)), "share memory"),
        (write, dict(table=table.long()), "int32 table"), (write, dict(table=table.cpu()), "int32 table"), (write, dict(k=k[:1], v=k[:1]), "one token for each row"),
        (write, dict(k=k.float()), "k: expected"), (write, dict(v=k[:, :1]), "v: expected"), (write, dict(start=n.long()), "start: expected"),
        (write, dict(start=n[:1]), "start: expected"), (write, dict(off=n), "offsets: expected"), (write, dict(q=q), "q needs them"), (write, dict(cos=cos), "come together"),
        (write, dict(q=q, cos=cos, sin=cos[:5]), "rotary tables"), (write, dict(q=q, cos=cos.float(), sin=cos.float()), "rotary tables"),
        (write, dict(q=q[:1], cos=cos, sin=cos), "q: expected"), (write, dict(q_out=q), "q_out needs q"), (write, dict(k=grad), "requires a gradient"),
        (write, dict(q=q, cos=cos, sin=cos, q_out=q[:, :1].expand(-1, 4, -1)), "share memory"), (write, dict(k_out=k.cpu()), "k_out: expected"),
        (write, dict(kp=pool.k.clone().requires_grad_()), "require a gradient"), (att, dict(vp=pool.v.clone().requires_grad_()), "require a gradient"),
        (write, dict(k=k[:1].expand((1 << 28) + 1, 2, 64), v=k[:1].expand((1 << 28) + 1, 2, 64), off=i32([0, 1, 2], dev)), "at most"), (read, dict(total=1 << 32), "over"),
        (write, dict(k=torch.zeros(2, 2, 68, dtype=torch.bfloat16, device=dev)[..., 4:]), "16-byte"),
        (read, dict(total=-1), "negative"), (read, dict(off=None), "offsets"), (read, dict(off=n), "offsets: expected"), (read, dict(k_out=k.float()), "k_out: expected"),
        (att, dict(q=q[:1]), "q: expected"), (att, dict(q=q[:, :3]), "multiple of 2"), (att, dict(q=q[:, :, :32]), "q: expected"), (att, dict(q=q.half()), "q: expected"),
        (att, dict(window=-1), "window"), (att, dict(lens=n.long()), "lens: expected"), (att, dict(out=q[:, :1].expand(-1, 4, -1)), "share memory"),
        (att, dict(lens=n.cpu()), "lens: expected"), (att, dict(kp=pool.k[:, :, :12], vp=pool.v[:, :, :12]), "page_size"),
    ]
    before = [pool.k.clone(), pool.v.clone()]
    for call, kw, msg in cases:
        with pytest.raises(ValueError, match=msg):
            call(**kw)
    assert same(pool.k, before[0]) and same(pool.v, before[1])
    with torch.no_grad():
        write(k=grad, v=k, start=i32([0, 0], dev))
