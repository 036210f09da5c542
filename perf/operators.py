"""The operators of the paged key / value cache, as they are measured: cases, inputs, plain forms and 64-bit results.

Layout of a cache: pages [n_pages, Hkv, page, hd], bf16 or OCP e4m3; with e4m3 one scale for each token and head, 2^(byte - 127), in
[n_pages, Hkv, page] uint8. table [B, width] int32 names the page of positions i * page ... of row b; entries behind a row's last page are -1.

  write      new keys and values (and queries), rotated by position, into the pages: `offsets` gives each row's range of new tokens (prompts), or there
             is one new token for each row (decoding); e4m3 rows are quantised as they are written
  read       the rows' cached keys and values, one behind the other, as bf16
  attention  one new token for each row over the row's cached positions, with the logarithm of the softmax's sum where a case asks for it
"""
import math
import random

import torch

own = False  # True: `run` makes the framework's calls

MAX_POSITIONS = 4096  # rows of the rotary tables of the write cases


def listed():
    """What each case stands for is said at it. 32 / 32, 32 / 8, 28 / 4 and 16 / 2 heads of 128 are the language models of this repository; 1049
    positions are the prompt of one video (1024 visual tokens and 25 of text)."""
    return [
        # one new token of one sequence: the smallest call, once a layer and token
        dict(name="write 1 token e4m3", op="write", rows=1, tokens=1, heads=32, kv_heads=8, hd=128, page=64, fmt="e4m3", prompt=False),
        # a decoding step of a full batch
        dict(name="write 128 tokens bf16", op="write", rows=128, tokens=1, heads=32, kv_heads=32, hd=128, page=16, fmt="bf16", prompt=False),
        # one video's prompt
        dict(name="write prompt 1049 bf16", op="write", rows=1, tokens=1049, heads=28, kv_heads=4, hd=128, page=32, fmt="bf16", prompt=True),
        # a batch of prompts of different lengths, quantised
        dict(name="write prompts 16x2049 e4m3", op="write", rows=16, tokens=2049, heads=32, kv_heads=8, hd=128, page=64, fmt="e4m3", prompt=True),
        # one video's cache, for a second question on it
        dict(name="read 1049 e4m3", op="read", rows=1, tokens=1049, heads=32, kv_heads=8, hd=128, page=64, fmt="e4m3"),
        # a batch of caches, for instance to move them
        dict(name="read 32x4000 bf16", op="read", rows=32, tokens=4000, heads=16, kv_heads=2, hd=128, page=128, fmt="bf16"),
        # the first tokens of one short text: latency alone
        dict(name="attention 1x77 bf16", op="attention", rows=1, tokens=77, heads=16, kv_heads=2, hd=128, page=16, fmt="bf16", window=0, lse=False),
        # one video, every head with keys of its own
        dict(name="attention 1x1049 bf16 32/32", op="attention", rows=1, tokens=1049, heads=32, kv_heads=32, hd=128, page=64, fmt="bf16", window=0, lse=True),
        # one very long sequence: the length has to be split
        dict(name="attention 1x131072 e4m3", op="attention", rows=1, tokens=131072, heads=32, kv_heads=8, hd=128, page=128, fmt="e4m3", window=0, lse=True),
        # a batch of ragged rows, an odd group of seven heads
        dict(name="attention 33x3001 e4m3 28/4", op="attention", rows=33, tokens=3001, heads=28, kv_heads=4, hd=128, page=32, fmt="e4m3", window=0, lse=False),
        # small heads, and a window that hides all but the newest 1000 positions
        dict(name="attention 24x5000 window 64", op="attention", rows=24, tokens=5000, heads=12, kv_heads=12, hd=64, page=16, fmt="bf16", window=1000, lse=True),
        # a serving batch: the largest call
        dict(name="attention 96x8192 bf16 32/8", op="attention", rows=96, tokens=8192, heads=32, kv_heads=8, hd=128, page=64, fmt="bf16", window=0, lse=False),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """Another case of the same ranges: every operator and both types, 1 to 128 rows, 1 to 131072 positions."""
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (28, 4), (16, 2), (40, 40), (12, 12), (16, 1), (24, 8), (5, 5)])
    case = dict(op=rng.choice(["write", "read", "attention", "attention"]), heads=heads, kv_heads=kv_heads, hd=rng.choice([64, 128, 128]),
                page=rng.choice([16, 32, 64, 128, 256]), fmt=rng.choice(["bf16", "e4m3"]))
    if case["op"] == "write":
        prompt = rng.random() < 0.6
        rows = _spread(rng, 1, 24 if prompt else 128)
        return dict(case, rows=rows, tokens=_spread(rng, 1, min(MAX_POSITIONS, 30000 // rows)) if prompt else 1, prompt=prompt)
    if case["op"] == "read":
        rows = _spread(rng, 1, 48)
        return dict(case, rows=rows, tokens=_spread(rng, 1, 60000 // rows))
    rows = _spread(rng, 1, 128)
    tokens = _spread(rng, 1, min(131072, 3000000 // (rows * kv_heads)))
    return dict(case, rows=rows, tokens=tokens, window=rng.choice([0, 0, 0, max(1, tokens // 3)]), lse=rng.random() < 0.5)


def _lengths(case):
    """Each row's number of positions: the first has them all, the others a part, and in a batch of eight or more one row has one and one is idle."""
    rows, most = case["rows"], case["tokens"]
    if case["op"] == "write" and not case["prompt"]:
        return [1] * rows
    rng = random.Random(rows * 1000003 + most)
    got = [most] + [max(1, int(most * rng.uniform(0.3, 1.0))) for _ in range(rows - 1)]
    if rows >= 8:
        got[-2:] = [1, 0]
    return got


def _starts(case):
    """write: the position of each row's first new token. Prompts begin at 0, or (odd rows) continue a text; a decoding step is anywhere."""
    if not case["prompt"]:
        rng = random.Random(case["rows"] * 7919 + case["page"])
        return [rng.randrange(MAX_POSITIONS) for _ in range(case["rows"])]
    return [0 if i % 2 == 0 else min(37 * i, MAX_POSITIONS - n) for i, n in enumerate(_lengths(case))]


def _quantised(x):
    """[..., hd] fp32 -> e4m3 codes, scale bytes [...]: the smallest power of two under which no element is over 448."""
    m, ex = torch.frexp(x.abs().amax(-1))
    e = (ex - 9 + (m > 0.875).to(ex.dtype)).clamp(min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    return torch.ldexp(x, -e[..., None].expand(x.shape)).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dev = torch.device("cuda")
    B, Hkv, hd, page, e4m3 = case["rows"], case["kv_heads"], case["hd"], case["page"], case["fmt"] == "e4m3"
    lens = _lengths(case)
    starts = _starts(case) if case["op"] == "write" else [0] * B
    need = [-(-(s + n) // page) if n else 0 for s, n in zip(starts, lens)]
    order = list(range(sum(need) + 3))
    rng.shuffle(order)
    width, at, table = max(need), 0, []
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(case=dict(case), table=i32(table), start=i32(starts), lens=i32(lens))
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    s["total"] = T = offsets[-1]
    # channels of unlike size, as keys have them
    gain = torch.exp(0.7 * torch.randn(Hkv, 1, hd, generator=g, device=dev))
    pool = (len(order), Hkv, page, hd)
    if case["op"] == "write":
        if case["prompt"]:
            s["offsets"] = i32(offsets)
        # one projection's output, of which the queries, keys and values are column ranges
        wide = torch.randn(T, (case["heads"] + 2 * Hkv) * hd, generator=g, device=dev)
        wide[:, case["heads"] * hd:(case["heads"] + Hkv) * hd].mul_(gain.reshape(-1))
        wide = wide.to(torch.bfloat16)
        s["q"] = wide[:, :case["heads"] * hd].view(T, case["heads"], hd)
        s["k"] = wide[:, case["heads"] * hd:(case["heads"] + Hkv) * hd].view(T, Hkv, hd)
        s["v"] = wide[:, (case["heads"] + Hkv) * hd:].view(T, Hkv, hd)
        inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd)
        angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device=dev)[:, None] * inv
        angle = torch.cat([angle, angle], -1)
        s["cos"], s["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
        kind = torch.float8_e4m3fn if e4m3 else torch.bfloat16
        s["k_pages"], s["v_pages"] = torch.zeros(pool, dtype=kind, device=dev), torch.zeros(pool, dtype=kind, device=dev)
        s["k_scales"], s["v_scales"] = ((torch.zeros(pool[:3], dtype=torch.uint8, device=dev), torch.zeros(pool[:3], dtype=torch.uint8, device=dev))
                                        if e4m3 else (None, None))
        return s
    s["offsets"] = i32(offsets)
    k = torch.randn(pool, generator=g, device=dev).mul_(gain).to(torch.bfloat16)
    v = torch.randn(pool, generator=g, device=dev).to(torch.bfloat16)
    if e4m3:
        s["k_pages"], s["k_scales"] = _quantised(k.float())
        s["v_pages"], s["v_scales"] = _quantised(v.float())
    else:
        s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"] = k, v, None, None
    if case["op"] == "attention":
        s["q"] = torch.randn(B, case["heads"], hd, generator=g, device=dev).to(torch.bfloat16)
    return s


def _rows_of_tokens(s):
    """Row and position of each new token, as index tensors."""
    dev = s["table"].device
    if "offsets" not in s:
        return torch.arange(s["table"].shape[0], device=dev), s["start"].long()
    row = torch.repeat_interleave(torch.arange(s["table"].shape[0], device=dev), s["lens"].long(), output_size=s["total"])
    return row, s["start"].long()[row] + torch.arange(s["total"], device=dev) - s["offsets"].long()[row]


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _values(pages, scales):
    x = pages.float()
    return x if scales is None else x * torch.ldexp(torch.ones((), device=x.device), scales.to(torch.int32) - 127)[..., None]


def run(state):
    s, case = state, state["case"]
    if own:
        from merv_amd import ops
        if case["op"] == "write":
            q = ops.paged_cache_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], s.get("offsets"), k_scales=s["k_scales"],
                                      v_scales=s["v_scales"], q=s["q"], cos=s["cos"], sin=s["sin"])
            return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        if case["op"] == "read":
            k, v = ops.paged_cache_read(s["k_pages"], s["v_pages"], s["table"], s["start"], s["offsets"], s["total"], k_scales=s["k_scales"],
                                        v_scales=s["v_scales"])
            return dict(k=k, v=v)
        out = ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                                         window=case["window"], return_lse=case["lse"])
        return dict(out=out[0], lse=out[1]) if case["lse"] else dict(out=out)
    page = case["page"]
    if case["op"] == "write":
        row, pos = _rows_of_tokens(s)
        at, slot = s["table"][row, pos // page].long(), pos % page
        cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
        q = _rotated(s["q"].float(), cos, sin).to(torch.bfloat16)
        k, v = _rotated(s["k"].float(), cos, sin).to(torch.bfloat16), s["v"]
        if case["fmt"] == "bf16":
            s["k_pages"][at, :, slot], s["v_pages"][at, :, slot] = k, v
        else:
            u8 = torch.uint8
            (kq, ke), (vq, ve) = _quantised(k.float()), _quantised(v.float())
            s["k_pages"].view(u8)[at, :, slot], s["v_pages"].view(u8)[at, :, slot] = kq.view(u8), vq.view(u8)
            s["k_scales"][at, :, slot], s["v_scales"][at, :, slot] = ke, ve
        return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    if case["op"] == "read":
        row, pos = _rows_of_tokens(s)
        at, slot = s["table"][row, pos // page].long(), pos % page
        if case["fmt"] == "bf16":
            return dict(k=s["k_pages"][at, :, slot], v=s["v_pages"][at, :, slot])
        u8 = torch.uint8
        pick = lambda p, e: _values(p.view(u8)[at, :, slot].view(torch.float8_e4m3fn), e[at, :, slot]).to(torch.bfloat16)  # noqa: E731
        return dict(k=pick(s["k_pages"], s["k_scales"]), v=pick(s["v_pages"], s["v_scales"]))
    B, H, Hkv, hd = case["rows"], case["heads"], case["kv_heads"], case["hd"]
    pages = s["table"].clamp(min=0).long()

    def dense(p, e):  # [B, Hkv, width * page, hd] fp32
        p = p[pages] if e is None else p.view(torch.uint8)[pages].view(torch.float8_e4m3fn)
        return _values(p, None if e is None else e[pages]).transpose(1, 2).reshape(B, Hkv, -1, hd)

    scores = torch.matmul(s["q"].float().view(B, Hkv, H // Hkv, hd), dense(s["k_pages"], s["k_scales"]).transpose(-1, -2)) * hd**-0.5
    j, n = torch.arange(scores.shape[-1], device=scores.device), s["lens"].long()[:, None]
    seen = j < n
    if case["window"]:
        seen = seen & (j >= n - case["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, dense(s["v_pages"], s["v_scales"])) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.view(B, H, hd).to(torch.bfloat16)
    return dict(out=out, lse=(top + torch.log(total)).view(B, H)) if case["lse"] else dict(out=out)


def exact(case, seed):
    """From the definition, row by row and token by token where it matters, in 64 bits."""
    s = prepare(case, seed)
    B, H, Hkv, hd, page = case["rows"], case["heads"], case["kv_heads"], case["hd"], case["page"]
    lens, starts = _lengths(case), _starts(case) if case["op"] == "write" else [0] * case["rows"]
    f64 = torch.float64

    def cached(pages, scales, b, lo, hi):  # positions lo .. hi - 1 of row b: [hi - lo, Hkv, hd]
        ids = s["table"][b, :-(-hi // page)].long()
        x = (pages if scales is None else pages.view(torch.uint8))[ids]
        x = x.to(f64) if scales is None else x.view(torch.float8_e4m3fn).to(f64) * torch.exp2(scales[ids].to(f64) - 127)[..., None]
        return x.permute(0, 2, 1, 3).reshape(-1, Hkv, hd)[lo:hi]

    if case["op"] == "attention":
        out = torch.zeros(B, H, hd, dtype=f64, device="cuda")
        lse = torch.full((B, H), -math.inf, dtype=f64, device="cuda")
        for b, n in enumerate(lens):
            if not n:
                continue
            lo = max(0, n - case["window"]) if case["window"] else 0
            k, v = cached(s["k_pages"], s["k_scales"], b, lo, n), cached(s["v_pages"], s["v_scales"], b, lo, n)
            for h in range(Hkv):
                group = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
                z = s["q"][b, group].to(f64) @ k[:, h].t() / math.sqrt(hd)
                lse[b, group] = torch.logsumexp(z, -1)
                out[b, group] = torch.softmax(z, -1) @ v[:, h]
        return dict(out=out, lse=lse) if case["lse"] else dict(out=out)
    if case["op"] == "read":
        got = [(cached(s["k_pages"], s["k_scales"], b, 0, n), cached(s["v_pages"], s["v_scales"], b, 0, n)) for b, n in enumerate(lens) if n]
        return dict(k=torch.cat([k for k, _ in got]), v=torch.cat([v for _, v in got]))
    # write: x + i y turned by the position's angle, as a product of complex numbers
    k_pages, v_pages = torch.zeros(s["k_pages"].shape, dtype=f64, device="cuda"), torch.zeros(s["v_pages"].shape, dtype=f64, device="cuda")
    q, t = torch.zeros(s["q"].shape, dtype=f64, device="cuda"), 0
    for b, n in enumerate(lens):
        pos = torch.arange(starts[b], starts[b] + n, device="cuda")
        turn = torch.complex(s["cos"][pos, :hd // 2].to(f64), s["sin"][pos, :hd // 2].to(f64))[:, None]

        def turned(x):
            z = torch.complex(x[..., :hd // 2].to(f64), x[..., hd // 2:].to(f64)) * turn
            return torch.cat([z.real, z.imag], -1)

        q[t:t + n] = turned(s["q"][t:t + n])
        k, v = turned(s["k"][t:t + n]).to(torch.bfloat16).to(f64), s["v"][t:t + n].to(f64)  # the cache's keys are bf16 numbers
        ids = s["table"][b, :-(-(starts[b] + n) // page)].long() if n else None
        for x, pages in ((k, k_pages), (v, v_pages)):
            if not n:
                continue
            if case["fmt"] == "e4m3":
                most = x.abs().amax(-1, keepdim=True)
                e = torch.floor(torch.log2(torch.where(most > 0, most, torch.ones_like(most)))) - 8
                e = e + (most > 448 * torch.exp2(e)).to(f64)
                e = torch.where(most > 0, e.clamp(min=-126), torch.full_like(e, -126))
                y = x * torch.exp2(-e)
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)  # distance of e4m3 numbers there
                x = torch.round(y / step) * step  # to the nearest, ties to even
            pages[ids[pos // page], :, pos % page] = x
        t += n
    return dict(q=q, k_pages=k_pages, v_pages=v_pages, k_scales=None, v_scales=None)


def work(case):
    lens, hd, elt = _lengths(case), case["hd"], (1 if case["fmt"] == "e4m3" else 2)
    T, Hkv, H, B = sum(lens), case["kv_heads"], case["heads"], case["rows"]
    row = 2 * Hkv * (hd * elt + (1 if elt == 1 else 0))  # one token's keys and values in the cache
    if case["op"] == "write":
        pages = sum(-(-(s + n) // case["page"]) - s // case["page"] for s, n in zip(_starts(case), lens) if n)
        return dict(bytes=T * (2 * Hkv * hd * 2 + row + 2 * H * hd * 2 + 2 * hd * 2) + 4 * (pages + 2 * B), flops=T * (H + Hkv) * hd * 3)
    pages = sum(-(-n // case["page"]) for n in lens)
    if case["op"] == "read":
        return dict(bytes=T * (row + 2 * Hkv * hd * 2) + 4 * (pages + 2 * B), flops=0)
    seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
    return dict(bytes=seen * row + 2 * B * H * hd * 2 + (4 * B * H if case["lse"] else 0) + 4 * (pages + B), flops=4 * seen * H * hd)
