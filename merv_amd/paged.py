"""
Decoding several rows (clips, questions) at once: a paged key / value cache whose rows have lengths of their own, in bf16 or in 8 bits, and the decoder that runs a
Llama / Mistral / Qwen2 module over it. The batch-1 path (llm.HipDecoder) reads every weight once for one token; a batch reads them once for all of its
rows, and what then grows with the rows is the cache: each row's pages are read by ops.paged_decode_attention in one pass, at their own length.

The reference generates one clip at a time through HF's GenerationMixin (merv/models/vidlms/merv.py:818-825); this is the step it would take for a batch.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch
import torch.nn.functional as F

from . import _lib, ops
from ._lib import check, ptr
from .llm import HipDecoder, StaticDecoder


def pool_pages(lengths: Sequence[int], max_len: int, page_size: int = 64) -> int:
    """Pages of a pool for rows of `lengths` positions (at most max_len each), rounded up to whole 256 positions a row, so that a pool also serves batches a little longer."""
    width = -(-max_len // page_size)
    each = len(lengths) * max(1, 256 // page_size)
    need = sum(min(width, -(-int(n) // page_size)) for n in lengths)
    return min(len(lengths) * width, -(-need // each) * each) if need else 0


class PagedKVCache:
    """Pages of all layers and the table that says which of them a row's positions lie in (one table for all layers). fmt "bf16", or "e4m3": 8-bit
    numbers with a power-of-two scale for each token and head. `n_pages` None: enough for every row at `max_len` positions."""

    def __init__(self, layers: int, rows: int, max_len: int, kv_heads: int, head_dim: int, device, fmt: str = "bf16", page_size: int = 64,
                 n_pages: Optional[int] = None) -> None:
        if fmt not in ("bf16", "e4m3"):
            raise ValueError(f"PagedKVCache: unknown format `{fmt}` (bf16 or e4m3)")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("PagedKVCache: page_size must be a power of two from 16 to 1024")
        self.rows, self.max_len, self.page_size, self.fmt = rows, max_len, page_size, fmt
        self.width = -(-max_len // page_size)
        self.n_pages = rows * self.width if n_pages is None else n_pages
        shape = (layers, self.n_pages, kv_heads, page_size, head_dim)
        kind = torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn
        self.k, self.v = torch.empty(shape, dtype=kind, device=device), torch.empty(shape, dtype=kind, device=device)
        self.k_scales = self.v_scales = None
        if fmt == "e4m3":
            self.k_scales, self.v_scales = (torch.empty(shape[:4], dtype=torch.uint8, device=device) for _ in range(2))
        self.table = torch.full((rows, self.width), -1, dtype=torch.int32, device=device)

    def assign(self, lengths: Sequence[int]) -> None:
        """Gives every row the pages of its first lengths[b] positions, and forgets what the cache held. The table stays the same tensor: captured steps
        read it."""
        need = [-(-int(n) // self.page_size) for n in lengths]
        if len(need) != self.rows or max(lengths, default=0) > self.max_len or min(lengths, default=0) < 0:
            raise ValueError(f"PagedKVCache: {self.rows} rows of at most {self.max_len} positions, got {list(lengths)}")
        if sum(need) > self.n_pages:
            raise ValueError(f"PagedKVCache: {sum(need)} pages needed, {self.n_pages} there")
        table, at = torch.full((self.rows, self.width), -1, dtype=torch.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
            at += n
        self.table.copy_(table)

    def layer(self, i: int) -> Dict[str, torch.Tensor]:
        """The arguments that ops.paged_* take for layer i."""
        d = dict(k_pages=self.k[i], v_pages=self.v[i], table=self.table)
        return d if self.k_scales is None else dict(d, k_scales=self.k_scales[i], v_scales=self.v_scales[i])


SCORES = 1 << 28  # of one product in known_attention: 1 GiB


def known_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int) -> torch.Tensor:
    """q [n, H, hd] at the last n of the positions of k, v [positions, Hkv, hd], each over what is at or before it (the newest `window` of that, 0: all) -> [n, H, hd].
    In 32 bits, rounded to q's type at the end: under a mask SDPA may take its batched products, whose 16-bit form with a transposed right operand has faulted the
    GPU with this torch build. Queries in blocks, so that no product has more than SCORES scores."""
    n, H, hd = q.shape
    past, out = k.shape[0] - n, torch.empty_like(q, memory_format=torch.contiguous_format)
    each = max(1, SCORES // (H * k.shape[0]))
    for a in range(0, n, each):
        b = min(n, a + each)
        lo = max(0, past + a - window + 1) if window else 0
        i, j = torch.arange(past + a, past + b, device=q.device)[:, None], torch.arange(lo, past + b, device=q.device)[None]
        mask = (j <= i) & (j > i - window) if window else j <= i
        qb, kb, vb = (x.float().transpose(0, 1)[None] for x in (q[a:b], k[lo:past + b], v[lo:past + b]))
        out[a:b] = F.scaled_dot_product_attention(qb, kb, vb, attn_mask=mask[None, None], enable_gqa=H != k.shape[1])[0].transpose(0, 1)
    return out


class PagedDecoder(StaticDecoder):
    """Prefill and token-by-token decoding of `batch` rows of any prompt lengths. prefill(prompts), then decode(tokens) once a token, as the other decoders;
    extend(more) puts further known tokens behind what the rows hold (a second question on the same clip) without running the first ones again.

    Projections and the MLP's products are library GEMMs over all rows' tokens, everything between them library calls of libmerv_hip.so: norms,
    rotary embedding + cache write (+ quantisation), attention, silu * up. A prompt attends to its own unquantised keys; what is read back
    from the cache, by decode() and extend(), is what the cache holds. A step is captured once in a hipGraph and replayed.

    `n_pages`: the pool that all rows share (None: enough for every row at max_len). A batch that needs more is refused by prefill()."""

    # q / k / v as one product, the module's parameters re-homed once as HipDecoder does it
    fuse_qkv, _qkv_fused = HipDecoder.fuse_qkv, HipDecoder._qkv_fused

    @staticmethod
    def supports(hf_model) -> bool:
        cfg = hf_model.config
        hd = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        p = next(hf_model.parameters())
        mlp = hf_model.model.layers[0].mlp
        mlp_bias = any(getattr(getattr(mlp, n, None), "bias", None) is not None for n in ("gate_proj", "up_proj", "down_proj"))
        return (hd in (64, 128) and p.is_cuda and p.dtype == torch.bfloat16 and not mlp_bias and cfg.hidden_size % 8 == 0 and cfg.hidden_size <= 8192
                and cfg.intermediate_size % 8 == 0)

    def __init__(self, hf_model, max_len: int, batch: int = 1, fmt: str = "bf16", page_size: int = 64, n_pages: Optional[int] = None) -> None:
        if not self.supports(hf_model):
            raise ValueError("PagedDecoder: a bfloat16 CUDA module with head_dim 64 or 128, at most 8192 hidden units and no MLP biases is needed")
        self.cache_args = dict(fmt=fmt, page_size=page_size, n_pages=n_pages)
        super().__init__(hf_model, max_len, batch)
        self.lib = _lib.load()
        for lyr in hf_model.model.layers:
            self._qkv_fused(lyr.self_attn)
        self.pos = torch.full((batch,), -1, dtype=torch.int32, device=self.dev)  # the position that a row's next token takes
        self.held: List[int] = [0] * batch  # the same on the host
        self.room: List[int] = [0] * batch  # positions that a row has pages for
        self.holders = self._holders()
        self.captured_weights: List[int] = []  # where the captured step's parameters lie
        cfg = self.cfg
        win, kinds = getattr(cfg, "sliding_window", None), getattr(cfg, "layer_types", None)
        if not getattr(cfg, "use_sliding_window", True):
            win = None
        self.windows = [int(win) if win is not None and (kinds is None or kinds[i] == "sliding_attention") else 0 for i in range(cfg.num_hidden_layers)]

    def _allocate(self) -> None:
        self.cache = PagedKVCache(self.cfg.num_hidden_layers, self.B, self.max_len, self.Hkv, self.hd, self.dev, **self.cache_args)

    def _holders(self) -> List[torch.nn.Module]:
        return [mod for mod in self.m.modules() if mod._parameters]

    def _drop_stale_step(self) -> None:
        """A captured step holds its parameters' addresses: one captured before a parameter or its storage was replaced is not replayed. Looked at before each
        step (120 us of the host's time for 32 layers, behind a step of milliseconds); modules that were replaced themselves are seen at the next prompt."""
        if self.graph is not None and self._addresses() != self.captured_weights:
            torch.cuda.synchronize(self.dev)  # a replay may be under way
            self.graph = None

    def _addresses(self) -> List[int]:
        return [p.data_ptr() for mod in self.holders for p in mod._parameters.values() if p is not None]

    def _layers(self, x: torch.Tensor, attend) -> torch.Tensor:
        """The decoder stack on x [T, D] (updated in place): attend(li, q, k, v) -> [T, H * hd] with q / k / v column ranges of one projection. Returns x."""
        lib, m, T, D, I = self.lib, self.m, x.shape[0], self.cfg.hidden_size, self.cfg.intermediate_size
        H, Hkv, hd = self.H, self.Hkv, self.hd
        st = torch.cuda.current_stream(self.dev).cuda_stream
        h = torch.empty_like(x)
        layers = m.model.layers
        check(lib.merv_decode_rmsnorm(ptr(x), ptr(layers[0].input_layernorm.weight), ptr(h), T, D, self.eps, st), "merv_decode_rmsnorm")

        def add_rms(delta, w):  # x += delta; h = RMSNorm(x) * w
            check(lib.merv_add_rmsnorm(ptr(x), ptr(delta), ptr(w), ptr(h), T, D, self.eps, st), "merv_add_rmsnorm")

        for li, lyr in enumerate(layers):
            a, mlp = lyr.self_attn, lyr.mlp
            fq = self._qkv_fused(a)
            if fq is not None:
                qkv = F.linear(h, fq[0], fq[1])
            else:
                qkv = torch.cat([F.linear(h, p.weight, p.bias) for p in (a.q_proj, a.k_proj, a.v_proj)], 1)
            q, k, v = qkv[:, :H * hd].view(T, H, hd), qkv[:, H * hd:(H + Hkv) * hd].view(T, Hkv, hd), qkv[:, (H + Hkv) * hd:].view(T, Hkv, hd)
            add_rms(F.linear(attend(li, q, k, v), a.o_proj.weight, a.o_proj.bias), lyr.post_attention_layernorm.weight)
            g, u = F.linear(h, mlp.gate_proj.weight), F.linear(h, mlp.up_proj.weight)
            check(lib.merv_silu_mul(ptr(g), ptr(u), ptr(g), T * I, st), "merv_silu_mul")
            dn = F.linear(g, mlp.down_proj.weight)
            if li + 1 < len(layers):
                add_rms(dn, layers[li + 1].input_layernorm.weight)
            else:
                x += dn
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        last = torch.empty_like(x)
        st = torch.cuda.current_stream(self.dev).cuda_stream
        check(self.lib.merv_decode_rmsnorm(ptr(x), ptr(self.m.model.norm.weight), ptr(last), x.shape[0], x.shape[1], self.eps, st), "merv_decode_rmsnorm")
        return F.linear(last, self.m.lm_head.weight).float()

    def _rows(self, embeds: Sequence[torch.Tensor], what: str) -> List[int]:
        if len(embeds) != self.B or any(e.dim() != 2 or e.shape[1] != self.cfg.hidden_size or e.shape[0] == 0 for e in embeds):
            raise ValueError(f"{what}: expected {self.B} rows of embeddings [tokens, {self.cfg.hidden_size}], one token at least, got "
                             f"{[tuple(e.shape) for e in embeds]}")
        return [e.shape[0] for e in embeds]

    def _known_tokens(self, embeds: Sequence[torch.Tensor], news: List[int]) -> torch.Tensor:
        """Runs known tokens, packed row behind row, behind the self.held positions of each; returns the logits behind each row's last one."""
        H, Hkv, hd, cache = self.H, self.Hkv, self.hd, self.cache
        self.holders = self._holders()
        offsets, ends = [0], []
        for n in news:
            offsets.append(offsets[-1] + n)
        ends = [s + n for s, n in zip(self.held, news)]
        past = any(self.held)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        start, off_d = i32(self.held), i32(offsets)
        if past:
            all_off = [0]
            for n in ends:
                all_off.append(all_off[-1] + n)
            all_off_d = i32(all_off)
        x = torch.cat([e.to(device=self.dev, dtype=self.dt) for e in embeds], 0)  # (a copy, also of one row: the residual stream is updated in place)
        st = torch.cuda.current_stream(self.dev).cuda_stream

        def attend(li, q, k, v):
            ops.paged_cache_write(k, v, start=start, offsets=off_d, q=q, cos=self.cos, sin=self.sin, q_out=q, k_out=k, **cache.layer(li))
            ld, win = q.stride(0), self.windows[li]
            out = torch.empty(q.shape[0], H * hd, dtype=self.dt, device=self.dev)
            if past:
                kc, vc = ops.paged_cache_read(start=None, offsets=all_off_d, total=all_off[-1], **cache.layer(li))
            for b, n in enumerate(news):
                lo, hi = offsets[b], offsets[b + 1]
                if not past and hd == 128 and not (win and n > win):
                    check(self.lib.merv_prefill_attention(q[lo:hi].data_ptr(), k[lo:hi].data_ptr(), v[lo:hi].data_ptr(), out[lo:hi].data_ptr(), n, H, Hkv,
                                                          hd, ld, ld, hd, H * hd, hd**-0.5, st), "merv_prefill_attention")
                    continue
                if past:
                    kb, vb = kc[all_off[b]:all_off[b + 1]].clone(), vc[all_off[b]:all_off[b + 1]].clone()
                    kb[self.held[b]:], vb[self.held[b]:] = k[lo:hi], v[lo:hi]  # its own keys as they are
                else:
                    kb, vb = k[lo:hi], v[lo:hi]
                out[lo:hi] = known_attention(q[lo:hi], kb, vb, win).view(n, H * hd)
            return out

        x = self._layers(x, attend)
        self.held = ends
        self.pos.copy_(i32(ends))  # the same tensor: a captured step keeps reading it
        return self._logits(x[torch.tensor(offsets[1:], device=self.dev) - 1])

    @torch.inference_mode()
    def prefill(self, inputs_embeds, room: Optional[int] = None) -> torch.Tensor:
        """inputs_embeds: [batch, S, D], or a list of [S_b, D], one for each row -> logits behind each row's last position [batch, vocab] (fp32). Every
        row gets pages for its prompt and `room` positions more (None: up to max_len)."""
        news = self._rows(inputs_embeds, "prefill")
        if max(news) >= self.max_len:
            raise ValueError(f"prefill: prompts of {news} tokens, the cache holds {self.max_len} positions a row")
        room = [self.max_len if room is None else min(self.max_len, n + room) for n in news]
        self.cache.assign(room)
        self.room, self.held = room, [0] * self.B
        with torch.cuda.device(self.dev):
            logits = self._known_tokens(inputs_embeds, news)
        return logits

    @torch.inference_mode()
    def extend(self, inputs_embeds) -> torch.Tensor:
        """Further known tokens of every row, behind the positions it holds -> logits behind each row's last one [batch, vocab] (fp32)."""
        news = self._rows(inputs_embeds, "extend")
        if not all(self.held):
            raise ValueError("extend: no prompt is held (prefill first)")
        if any(s + n > r for s, n, r in zip(self.held, news, self.room)):
            raise ValueError(f"extend: rows of {self.held} + {news} positions, room for {self.room}")
        with torch.cuda.device(self.dev):
            return self._known_tokens(inputs_embeds, news)

    def _step(self) -> torch.Tensor:
        cache = self.cache
        lens = self.pos + 1

        def attend(li, q, k, v):
            q = ops.paged_cache_write(k, v, start=self.pos, q=q, cos=self.cos, sin=self.sin, **cache.layer(li))
            return ops.paged_decode_attention(q, lens=lens, window=self.windows[li], **cache.layer(li)).view(self.B, self.H * self.hd)

        with torch.cuda.device(self.dev):
            x = self.m.model.embed_tokens(self.tok).view(self.B, -1)
            return self._logits(self._layers(x, attend))

    def decode(self, token: torch.Tensor, use_graph: bool = True) -> torch.Tensor:
        """token [batch]: each row's token at its position -> logits behind it [batch, vocab] (fp32; a captured step's own tensor, which the next step
        writes over)."""
        if token.shape != (self.B,):
            raise ValueError(f"decode: expected {self.B} tokens, one a row, got {tuple(token.shape)}")
        if not all(self.held) or any(s >= r for s, r in zip(self.held, self.room)):
            raise ValueError(f"decode: rows hold {self.held} positions, with room for {self.room}")
        with torch.cuda.device(self.dev):  # a capture is of the current device's stream
            if use_graph:
                self._drop_stale_step()
            captured = self.graph
            out = super().decode(token, use_graph)
            if self.graph is not captured:
                self.captured_weights = self._addresses()
        self.held = [n + 1 for n in self.held]
        return out
