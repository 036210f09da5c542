"""GPU: what a PagedDecoder keeps from call to call: its captured step, its pool of pages."""
import pytest
import torch

from conftest import rel_l2
from test_paged_decoder_gpu import TOL, Formula, backbone, prompts

pytestmark = pytest.mark.gpu


def replaced(bb, factor):
    """Other storages for all but q / k / v (whose replacement is seen by their own check); -> the old ones, to put back and to keep alive."""
    old = []
    with torch.no_grad():
        for p in [bb.llm.model.norm.weight] + [lin.weight for lyr in bb.llm.model.layers for lin in (lyr.self_attn.o_proj, lyr.mlp.up_proj, lyr.post_attention_layernorm)]:
            old.append((p, p.data))
            p.data = (p * factor).clone()
    return old


def put_back(old):
    for p, data in old:
        p.data = data


def test_replaced_weights_are_seen_behind_a_held_prompt(dev):
    """prefill, decode (captures), other weights, extend, decode: the step behind extend() uses what extend() used."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb, more, t = prompts([9, 4], 256, dev), prompts([3, 6], 256, dev, 5), torch.tensor([5, 9], device=dev)
    dec = PagedDecoder(bb.llm, 64, 2)
    dec.prefill(emb)
    dec.decode(t)
    rows = [Formula(bb, dec.cos, dec.sin, "bf16") for _ in range(2)]
    for b, row in enumerate(rows):
        row.run(emb[b])
        row.run(bb.embed_input_ids(t)[b:b + 1])
    old = replaced(bb, 1.5)
    got = dec.extend(more)
    last = dec.decode(t).clone()
    for b, row in enumerate(rows):
        assert rel_l2(got[b], row.run(more[b])) < TOL["bf16"]
        assert rel_l2(last[b], row.run(bb.embed_input_ids(t)[b:b + 1])) < TOL["bf16"]
    put_back(old)


@pytest.mark.parametrize("between", ["prefill", "nothing"])
def test_a_step_captured_with_other_weights_is_not_replayed(dev, between):
    """Weights A at the prompt, B at the first step (captured), A again: the next step, behind a new prompt or not, uses A."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb, t = prompts([9, 4], 256, dev), torch.tensor([5, 9], device=dev)
    dec = PagedDecoder(bb.llm, 64, 2)
    dec.prefill(emb)
    old = replaced(bb, 1.5)
    kept = [(p, p.data) for p, _ in old]  # B's storages stay alive
    dec.decode(t)
    put_back(old)
    if between == "prefill":
        dec.prefill(emb)
        got = dec.decode(t)
        want = PagedDecoder(bb.llm, 64, 2)
        want.prefill(emb)
        assert torch.equal(got, want.decode(t, use_graph=False))
    else:
        got = dec.decode(t).clone()
        dec.held = [n - 1 for n in dec.held]
        dec.pos -= 1  # the same step again, not captured
        assert torch.equal(got, dec.decode(t, use_graph=False))
    assert len(kept) == len(old)


def test_a_replaced_parameter_is_seen(dev):
    """Another Parameter object in a module's place, with a captured step alive."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb, t = prompts([9, 4], 256, dev), torch.tensor([5, 9], device=dev)
    dec = PagedDecoder(bb.llm, 64, 2)
    dec.prefill(emb)
    dec.decode(t)
    kept = bb.llm.lm_head.weight
    bb.llm.lm_head.weight = torch.nn.Parameter((kept * -1.0).detach(), requires_grad=False)
    dec.prefill(emb)
    got = dec.decode(t).clone()
    want = PagedDecoder(bb.llm, 64, 2)
    want.prefill(emb)
    assert torch.equal(got, want.decode(t, use_graph=False))


@pytest.mark.parametrize("heads,kv_heads,hidden,window", [(2, 2, 256, None), (4, 4, 256, None), (2, 2, 256, 24), (4, 2, 256, 24), (4, 4, 256, 24)])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_known_tokens_of_heads_of_their_own(dev, fmt, heads, kv_heads, hidden, window):
    """Prompts, steps and further tokens where each query head has its key head (and where two share one), 64 and 128 dims, with and without a window."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev, "mistral" if window else "llama", heads, kv_heads, hidden, **(dict(sliding_window=window) if window else {}))
    dec = PagedDecoder(bb.llm, 128, 2, fmt=fmt, page_size=32)
    first, second, t = prompts([40, 3], hidden, dev, 1), prompts([5, 41], hidden, dev, 2), torch.tensor([5, 9], device=dev)
    rows = [Formula(bb, dec.cos, dec.sin, fmt, window or 0) for _ in range(2)]
    got = [dec.prefill(first), dec.decode(t).clone(), dec.extend(second), dec.decode(t).clone()]
    for b, row in enumerate(rows):
        e = bb.embed_input_ids(t)[b:b + 1]
        for x, known in zip(got, (first[b], e, second[b], e)):
            assert rel_l2(x[b], row.run(known)) < TOL[fmt]


@pytest.mark.parametrize("kv", ["paged", "paged-e4m3"])
def test_a_ragged_batch_takes_the_pages_it_needs(dev, kv):
    """One long prompt beside short ones: a pool for their sum, not for the longest in every row; a batch that needs more gets a larger one, a smaller one the same."""
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb = prompts([700] + [9] * 7, 256, dev)
    ids = bb.generate_from_embeds(emb, max_new_tokens=6, kv_cache=kv)
    dec, = bb._decoders.values()
    assert dec.cache.n_pages == 32 and dec.cache.k.shape[1] == 32  # 12 + 7 pages of 64, rounded up; 8 x 12 for eight rows of 768
    full = PagedDecoder(bb.llm, 768, 8, fmt="e4m3" if kv.endswith("e4m3") else "bf16")
    assert full.cache.n_pages == 96
    tok = full.prefill(emb).argmax(-1)
    for i in range(6):
        assert torch.equal(ids[:, i], tok)
        tok = full.decode(tok).argmax(-1)
    bb.generate_from_embeds(prompts([600] * 4 + [9] * 4, 256, dev), max_new_tokens=100, kv_cache=kv)
    larger, = bb._decoders.values()
    assert larger is not dec and larger.cache.n_pages == 64
    assert torch.equal(ids, bb.generate_from_embeds(emb, max_new_tokens=6, kv_cache=kv))
    assert bb._decoders[next(iter(bb._decoders))] is larger
    small = PagedDecoder(bb.llm, 768, 8, n_pages=18)
    with pytest.raises(ValueError, match="pages needed"):
        small.prefill(emb, room=7)


def test_what_does_not_fit_the_rows_is_refused(dev):
    from merv_amd.paged import PagedDecoder
    bb = backbone(dev)
    emb = prompts([9, 4], 256, dev)
    dec = PagedDecoder(bb.llm, 64, 2)
    dec.prefill(emb)
    for bad in ([5], [5, 6, 7], [[5], [6]]):
        with pytest.raises(ValueError, match="one a row"):
            dec.decode(torch.tensor(bad, device=dev))
    assert dec.held == [9, 4]
    with pytest.raises(ValueError, match="one prompt at least"):
        bb.generate_from_embeds([], max_new_tokens=2, kv_cache="paged")
    ids = torch.tensor([7, 8], device=dev)
    for bad in ([ids], [ids, ids[:0]], [ids, ids, ids]):
        with pytest.raises(ValueError, match="prompt_ids"):
            bb.generate_from_embeds(emb, max_new_tokens=2, kv_cache="paged", repetition_penalty=2.0, prompt_ids=bad)
    none = bb.generate_from_embeds(emb, max_new_tokens=4, kv_cache="paged", repetition_penalty=2.0, prompt_ids=[ids[:0], ids[:0]])
    assert torch.equal(none, bb.generate_from_embeds(emb, max_new_tokens=4, kv_cache="paged", repetition_penalty=2.0))
