"""GPU: the batched decoder on the paged cache (merv_amd/paged.py) against the module's formulas in 64 bits on the CPU, with the cache's numbers rounded as it
rounds them; and generation through it."""
import math

import pytest
import torch

import paged_oracle as P
from conftest import rel_l2

pytestmark = pytest.mark.gpu

# A bf16 module rounds each value on the way through a layer a dozen times (norm, projections, rotation, attention, products, residual), each off by 2^-8 / sqrt(3) =
# 2^-8.8 in the mean square at most; three layers and the head: sqrt(40) 2^-8.8 = 1.4e-2 of the result. With an 8-bit cache a tenth of the cached numbers then
# falls on the other side of a rounding border, 2^-3.5 away: 2.8e-2 of a value, averaged over the ten or more positions a token sees: 0.9e-2 more, squared and added: 1.7e-2.
TOL = {"bf16": 2e-2, "e4m3": 3e-2}


def backbone(dev, family="llama", heads=4, kv_heads=2, hidden=256, **kw):
    from merv_amd.llm import LlamaBackbone
    cfg = dict(vocab_size=320, hidden_size=hidden, intermediate_size=512, num_hidden_layers=3, num_attention_heads=heads, num_key_value_heads=kv_heads,
               max_position_embeddings=1024, rms_norm_eps=1e-5, bos_token_id=1, eos_token_id=2, pad_token_id=0)
    cfg.update(kw)
    bb = LlamaBackbone(cfg, device=dev, family=family, seed=3)
    if family == "qwen2":
        with torch.no_grad():
            for lyr in bb.llm.model.layers:
                for p in (lyr.self_attn.q_proj, lyr.self_attn.k_proj, lyr.self_attn.v_proj):
                    p.bias.copy_(0.3 * torch.randn(p.bias.shape, generator=torch.Generator().manual_seed(1)).to(p.bias))
    return bb


class Formula:
    """One row through the module in 64 bits: known tokens attend to unquantised keys of their own call, and to the cache's for what was there before."""

    def __init__(self, bb, cos, sin, fmt, window=0):
        self.m, self.cfg, self.fmt, self.window = bb.llm, bb.config, fmt, window
        self.cos, self.sin = cos.cpu(), sin.cpu()
        L = self.cfg.num_hidden_layers
        self.k, self.v = [[] for _ in range(L)], [[] for _ in range(L)]

    def w(self, p):
        return p.detach().cpu().double()

    def rms(self, x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.cfg.rms_norm_eps) * self.w(w)

    def held(self, xs):
        if self.fmt == "bf16":
            return list(xs)
        val, sc = P.quantise(xs.to(torch.bfloat16))
        return list(P.dequantise(val, sc))

    def run(self, x):
        """x [n, D] -> logits behind the last of the n tokens."""
        x = x.detach().cpu().double()
        n, past = x.shape[0], len(self.k[0])
        H, Hkv = self.cfg.num_attention_heads, self.cfg.num_key_value_heads
        hd = self.cos.shape[1]
        cos, sin = self.cos[past:past + n].double()[:, None], self.sin[past:past + n].double()[:, None]
        rot = lambda y: y * cos + torch.cat([-y[..., hd // 2:], y[..., :hd // 2]], -1) * sin  # noqa: E731
        for li, lyr in enumerate(self.m.model.layers):
            a, mlp = lyr.self_attn, lyr.mlp
            h = self.rms(x, lyr.input_layernorm.weight)
            lin = lambda p: h @ self.w(p.weight).T + (0 if p.bias is None else self.w(p.bias))  # noqa: E731
            q, k, v = rot(lin(a.q_proj).view(n, H, hd)), rot(lin(a.k_proj).view(n, Hkv, hd)), lin(a.v_proj).view(n, Hkv, hd)
            if n == 1:  # a decoding step reads its own token from the cache too
                k, v = torch.stack(self.held(k)), torch.stack(self.held(v))
            ka, va = torch.stack(self.k[li] + list(k)), torch.stack(self.v[li] + list(v))
            o = torch.empty(n, H, hd, dtype=torch.float64)
            for i in range(n):
                hi = past + i + 1
                lo = max(0, hi - self.window) if self.window else 0
                for j in range(H):
                    g = j // (H // Hkv)
                    o[i, j] = torch.softmax(ka[lo:hi, g] @ q[i, j] * hd**-0.5, -1) @ va[lo:hi, g]
            self.k[li] += self.held(k) if n > 1 else list(k)
            self.v[li] += self.held(v) if n > 1 else list(v)
            x = x + o.view(n, H * hd) @ self.w(a.o_proj.weight).T
            h = self.rms(x, lyr.post_attention_layernorm.weight)
            g, u = h @ self.w(mlp.gate_proj.weight).T, h @ self.w(mlp.up_proj.weight).T
            x = x + (g * torch.sigmoid(g) * u) @ self.w(mlp.down_proj.weight).T
        return self.rms(x[-1], self.m.model.norm.weight) @ self.w(self.m.lm_head.weight).T


def prompts(lens, D, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(0.5 * torch.randn(n, D, generator=g)).to(torch.bfloat16).to(dev) for n in lens]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("family,heads,kv_heads,hidden,graph", [("llama", 4, 2, 256, True), ("llama", 4, 1, 512, False), ("qwen2", 4, 4, 512, True)])
def test_steps_follow_the_formula(dev, fmt, family, heads, kv_heads, hidden, graph):
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev, family, heads, kv_heads, hidden)
    dec = PagedDecoder(bb.llm, 256, 4, fmt=fmt, page_size=16)
    for again in range(2):  # the second prefill finds a captured step and other pages
        lens = [[21, 1, 64, 30], [5, 77, 16, 2]][again]
        emb = prompts(lens, hidden, dev, again)
        rows = [Formula(bb, dec.cos, dec.sin, fmt) for _ in lens]
        got = dec.prefill(emb, room=20)
        for b, row in enumerate(rows):
            assert rel_l2(got[b], row.run(emb[b])) < TOL[fmt], b
        toks = torch.randint(3, 320, (6, 4), generator=torch.Generator().manual_seed(7 + again)).to(dev)
        for t in toks:
            got = dec.decode(t, use_graph=graph).clone()
            e = bb.embed_input_ids(t)
            for b, row in enumerate(rows):
                assert rel_l2(got[b], row.run(e[b:b + 1])) < TOL[fmt], b


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_extend_is_what_the_whole_prompt_would_have_been(dev, fmt):
    """A second question behind a held clip: the cache is read back, and decoding goes on behind it."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev, heads=2, kv_heads=1, hidden=256)  # 128 dims a head
    dec = PagedDecoder(bb.llm, 128, 2, fmt=fmt, page_size=32)
    first, second = prompts([40, 3], 256, dev, 1), prompts([5, 21], 256, dev, 2)
    rows = [Formula(bb, dec.cos, dec.sin, fmt) for _ in range(2)]
    dec.prefill(first)
    t = torch.tensor([5, 9], device=dev)
    dec.decode(t)
    got = dec.extend(second)
    last = dec.decode(t)
    for b, row in enumerate(rows):
        row.run(first[b])
        row.run(bb.embed_input_ids(t)[b:b + 1])
        assert rel_l2(got[b], row.run(second[b])) < TOL[fmt]
        assert rel_l2(last[b], row.run(bb.embed_input_ids(t)[b:b + 1])) < TOL[fmt]
    with pytest.raises(ValueError, match="room"):
        dec.extend(prompts([200, 1], 256, dev))


def test_sliding_window(dev):
    """A module whose tokens see the newest 24 positions, prompts on both sides of that, and steps beyond it."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev, "mistral", heads=2, kv_heads=1, hidden=256, sliding_window=24)
    dec = PagedDecoder(bb.llm, 128, 2)
    assert dec.windows == [24] * 3
    emb = prompts([50, 20], 256, dev)
    rows = [Formula(bb, dec.cos, dec.sin, "bf16", 24) for _ in range(2)]
    got = dec.prefill(emb)
    for b, row in enumerate(rows):
        assert rel_l2(got[b], row.run(emb[b])) < TOL["bf16"]
    for s in range(8):
        t = torch.tensor([5 + s, 9 + s], device=dev)
        got = dec.decode(t)
        for b, row in enumerate(rows):
            assert rel_l2(got[b], row.run(bb.embed_input_ids(t)[b:b + 1])) < TOL["bf16"], s


@pytest.mark.parametrize("kv", ["paged", "paged-e4m3"])
def test_generation_of_a_ragged_batch(dev, kv):
    """Every generated token is, but for near ties, the most likely one behind its row's own text (checked with the module's forward on that row alone)."""
    bb = backbone(dev)
    emb = prompts([30, 7, 55], 256, dev)
    ids = bb.generate_from_embeds(emb, max_new_tokens=10, kv_cache=kv)
    assert ids.shape == (3, 10)
    assert torch.equal(ids, bb.generate_from_embeds(emb, max_new_tokens=10, kv_cache=kv))
    assert torch.equal(ids, bb.generate_from_embeds(emb, max_new_tokens=10, kv_cache=kv, use_graph=False))
    for b in range(3):
        with torch.inference_mode():
            text = torch.cat([emb[b], bb.embed_input_ids(ids[b, :-1])])[None]
            lg = bb.llm(inputs_embeds=text).logits[0, emb[b].shape[0] - 1:].float()
        short = lg.max(-1).values - lg.gather(1, ids[b][:, None])[:, 0]
        assert bool((short <= 2 * TOL["e4m3" if kv.endswith("e4m3") else "bf16"] * lg.norm(dim=-1)).all())
    one = bb.generate_from_embeds(emb[0][None], max_new_tokens=4, kv_cache=kv)  # a batch of one, given as a tensor
    assert one.shape == (1, 4) and int(one[0, 0]) == int(ids[0, 0])
    pen = bb.generate_from_embeds(emb, max_new_tokens=6, kv_cache=kv, repetition_penalty=50.0, prompt_ids=[torch.tensor([7, 8], device=dev), torch.tensor([9], device=dev),
                                                                                                             torch.tensor([3, 4, 5], device=dev)])
    assert all(len(set(r)) == 6 for r in pen.tolist())
    got = bb.generate_from_embeds(emb, max_new_tokens=6, kv_cache=kv, do_sample=True, top_k=5, temperature=0.8, generator=torch.Generator(device=dev).manual_seed(0))
    assert got.shape == (3, 6)


def test_replaced_weights_are_seen_by_the_next_prompt(dev):
    """A captured step holds addresses: after a parameter's storage is replaced, by one decoder's leave or another's, the next prompt captures anew."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb, t = prompts([9, 4], 256, dev), torch.tensor([5, 9], device=dev)
    decs = [PagedDecoder(bb.llm, 64, 2) for _ in range(2)]
    for d in decs:
        d.prefill(emb)
        d.decode(t)
    with torch.no_grad():
        for lyr in bb.llm.model.layers:
            for lin in (lyr.self_attn.q_proj, lyr.self_attn.o_proj, lyr.mlp.up_proj):
                lin.weight.data = (lin.weight * 1.5).clone()
    for d in decs:
        d.prefill(emb)
        got = d.decode(t)
        for b in range(2):
            row = Formula(bb, d.cos, d.sin, "bf16")
            row.run(emb[b])
            assert rel_l2(got[b], row.run(bb.embed_input_ids(t)[b:b + 1])) < TOL["bf16"]


def test_static_generation_is_untouched_by_the_paged_one(dev):
    bb = backbone(dev)
    emb = prompts([30], 256, dev)[0][None]
    a = bb.generate_from_embeds(emb, max_new_tokens=8)
    bb.generate_from_embeds(emb, max_new_tokens=8, kv_cache="paged")
    assert torch.equal(a, bb.generate_from_embeds(emb, max_new_tokens=8))


def test_generate_takes_the_cache(dev):
    """MERV.generate(kv_cache=...): the front door over the same path."""
    from test_generate_gpu import _model
    m = _model(dev, ["dinov2-video-all-tokens"], [4])
    m.tokenizer = None
    clip = (torch.randint(0, 256, (40, 3, 64, 80), dtype=torch.uint8, generator=torch.Generator().manual_seed(0)), 25.0)
    for kv in ("paged", "paged-e4m3"):
        ids = m.generate(clip, [1, 9, 8, 7], [4], max_new_tokens=3, kv_cache=kv)
        assert ids.shape == (1, 3)


def test_refusals(dev):
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb = prompts([30, 7], 256, dev)
    with pytest.raises(ValueError, match="several lengths"):
        bb.generate_from_embeds(emb, max_new_tokens=2)
    with pytest.raises(ValueError, match="unknown kv_cache"):
        bb.generate_from_embeds(emb, max_new_tokens=2, kv_cache="paged-int4")
    with pytest.raises(ValueError, match="positions are needed"):
        bb.generate_from_embeds(emb, max_new_tokens=1000, kv_cache="paged")
    dec = PagedDecoder(bb.llm, 64, 2)
    with pytest.raises(ValueError, match="rows hold"):
        dec.decode(torch.tensor([1, 2], device=dev))
    with pytest.raises(ValueError, match="no prompt"):
        dec.extend(emb)
    with pytest.raises(ValueError, match="2 rows"):
        dec.prefill(emb[:1])
    with pytest.raises(ValueError, match="holds 64"):
        dec.prefill(prompts([64, 3], 256, dev))
    dec.prefill(emb, room=2)
    dec.decode(torch.tensor([1, 2], device=dev))
    dec.decode(torch.tensor([1, 2], device=dev))
    with pytest.raises(ValueError, match="rows hold"):
        dec.decode(torch.tensor([1, 2], device=dev))
    with pytest.raises(ValueError, match="PagedDecoder"):
        PagedDecoder(backbone(dev, heads=8).llm, 64, 2)  # 32 dims a head
