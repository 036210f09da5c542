"""Plain implementations of the paged key / value cache's operators, on the CPU in 64 bits (rotation and quantisation: every step is exact or rounded
once, so results are equal, not near), and the inputs that the tests of them share."""
import math

import torch

F64 = torch.float64


def quantise(x: torch.Tensor):
    """x [..., hd] (bf16 numbers) -> (values float64, scale bytes uint8): e4m3 under the smallest power of two with no finite element over 448."""
    x = x.to(F64)
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(amax.shape, -126, dtype=torch.int64)
    for n in range(-126, 121):  # the definition: one more for as long as the largest is over 448 of it
        e = torch.where(amax > 448 * 2.0**n, torch.full_like(e, n + 1), e)
    y = x * torch.pow(torch.tensor(2.0, dtype=F64), -e[..., None].to(F64))
    step = torch.pow(torch.tensor(2.0, dtype=F64), torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    y = torch.where(finite, torch.round(y / step) * step, torch.full_like(y, math.nan))
    return y, (e + 127).to(torch.uint8)


def dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return codes.to(F64) * torch.pow(torch.tensor(2.0, dtype=F64), scales.to(F64) - 127)[..., None]


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """[T, heads, hd] bf16 by [T, hd] -> bf16: products of bf16 numbers are exact in fp32, their sum is rounded to fp32 and then to bf16."""
    x, c, s = x.float(), cos.float()[:, None], sin.float()[:, None]
    h = x.shape[-1] // 2
    return (x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * s).to(torch.bfloat16)


def attention(q, k_rows, v_rows, scale, window=0):
    """q [rows, H, hd]; k_rows, v_rows: lists of [len, Hkv, hd]. -> out, lse (float64) and how far a result in fp32 that is rounded to bf16 may be off each.

    With p the softmax, s the scores and u = 2^-24: a score is a sum of hd products, exact in fp32, off by at most (hd + 3) u scale sum |q k| =: d
    (the 3: the factors scale, log2 e and their product), and exp2's argument and result add (|s| + 2) 2^-22; a weight is two bf16
    numbers: cut off after 8 bits, a rest under 2^-7 of it, which is rounded to 8 bits: off by 2^-8 2^-7 = 2^-15; numerator and denominator are sums of len terms, (len + 8) u each (8: joining the parts of a split). out is a quotient, so each counts
    twice, times sum p |v|; then 2^-8 |out| for the rounding to bf16."""
    rows, H, hd = q.shape
    out, lse = torch.zeros(rows, H, hd, dtype=F64), torch.full((rows, H), -math.inf, dtype=F64)
    out_tol, lse_tol = torch.zeros(rows, H, hd, dtype=F64), torch.zeros(rows, H, dtype=F64)
    u = 2.0**-24
    for b in range(rows):
        n = k_rows[b].shape[0]
        lo = max(0, n - window) if window else 0
        if n == 0:
            continue
        k, v = k_rows[b][lo:].to(F64), v_rows[b][lo:].to(F64)
        for h in range(H):
            g = h // (H // k.shape[1])
            x = q[b, h].to(F64)
            s = (k[:, g] @ x) * scale
            p = torch.softmax(s, -1)
            out[b, h], lse[b, h] = p @ v[:, g], torch.logsumexp(s, -1)
            d = (hd + 3) * u * scale * float((k[:, g].abs() @ x.abs()).max()) + (float(s.abs().max()) + 2) * 2.0**-22
            one = d + 2.0**-15 + (n + 8) * u
            out_tol[b, h] = 2 * one * (p @ v[:, g].abs()) + 2.0**-8 * out[b, h].abs() + 1e-30
            lse_tol[b, h] = d + (n + 8) * u + float(lse[b, h].abs() + 1) * 2.0**-22
    return out, lse, out_tol, lse_tol


class Pool:
    """Pages whose every slot holds NaN (and, for e4m3, an arbitrary scale) until a row's positions are put in. layout: the order in which the
    dimensions page, head, slot lie in memory."""

    def __init__(self, lens, kv_heads, hd, page, fmt, dev, seed=0, layout="phs", spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kv_heads, self.hd, self.page, self.fmt, self.dev = list(lens), kv_heads, hd, page, fmt, dev
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        self.width = width or max(need + [1])
        order = torch.randperm(n_pages, generator=g).tolist()
        self.table = torch.full((len(lens), self.width), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.free = order[at:]
        kind = torch.float8_e4m3fn if fmt == "e4m3" else torch.bfloat16
        size, back = {"phs": ((n_pages, kv_heads, page), (0, 1, 2)), "psh": ((n_pages, page, kv_heads), (0, 2, 1)),
                      "hps": ((kv_heads, n_pages, page), (1, 0, 2))}[layout]

        def pages():
            x = torch.full((*size, hd), math.nan).to(kind).to(dev)
            return x.permute(*back, 3)

        self.k, self.v = pages(), pages()
        self.ks = self.vs = None
        if fmt == "e4m3":
            self.ks, self.vs = (torch.randint(0, 256, (n_pages, kv_heads, page), generator=g, dtype=torch.uint8).to(dev) for _ in range(2))

    def place(self, b, pos):
        return int(self.table[b, pos // self.page]), pos % self.page

    def fill(self, k_rows, v_rows):
        """Puts [len, kv_heads, hd] bf16 rows in; -> the values that the cache then stands for, float64."""
        got = []
        for rows, pages, scales in ((k_rows, self.k, self.ks), (v_rows, self.v, self.vs)):
            u8 = pages.view(torch.uint8) if self.fmt == "e4m3" else pages
            host, host_s, back = u8.cpu(), None if scales is None else scales.cpu(), []
            for b, x in enumerate(rows):
                at = self.table[b].long()[torch.arange(x.shape[0]) // self.page]
                slot = torch.arange(x.shape[0]) % self.page
                if self.fmt == "e4m3":
                    val, sc = quantise(x)
                    code = val.float().to(torch.float8_e4m3fn)
                    host[at, :, slot] = code.view(torch.uint8)
                    host_s[at, :, slot] = sc
                    back.append(dequantise(code.float(), sc))
                else:
                    host[at, :, slot] = x
                    back.append(x.to(F64))
            u8.copy_(host)
            if scales is not None:
                scales.copy_(host_s)
            got.append(back)
        return got

    def scales(self):
        return dict(k_scales=self.ks, v_scales=self.vs)


def rows_like(lens, kv_heads, hd, seed):
    """Random keys and values, channels of unlike size, bf16 on the CPU."""
    g = torch.Generator().manual_seed(seed)
    gain = torch.exp(0.7 * torch.randn(kv_heads, hd, generator=g))
    k = [(torch.randn(n, kv_heads, hd, generator=g) * gain).to(torch.bfloat16) for n in lens]
    v = [torch.randn(n, kv_heads, hd, generator=g).to(torch.bfloat16) for n in lens]
    return k, v
