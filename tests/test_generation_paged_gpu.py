"""Paged generation on the native path: against the plain forward pass, and captured against eager."""
import pytest
import torch

from lingua_b200.generation import PackedCausalTransformerGeneratorArgs, build_generator
from lingua_b200.models.transformer import LMTransformer, LMTransformerArgs
from lingua_b200.tokenizer import ByteTokenizer

pytestmark = pytest.mark.gpu
PROMPTS = ["hello world, this is a test of a prompt that is longer than a page", "abc", "the quick brown fox jumps over"]


def model_of(seed=0, **kw):
    torch.manual_seed(seed)
    m = LMTransformer(LMTransformerArgs(**{**dict(dim=512, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=258, max_seqlen=512),
                                           **kw}))
    m.init_weights()
    m = m.cuda().bfloat16().eval()
    m.rope_embeddings.reset_parameters()
    return m


def args(**kw):
    return PackedCausalTransformerGeneratorArgs(**{**dict(max_gen_len=16, max_tokens=1024, page_size=16), **kw})


@pytest.mark.parametrize("kw,gkw", [(dict(), dict()), (dict(), dict(prefill_chunk=11)), (dict(n_heads=8, n_kv_heads=8), dict()),
                                    (dict(n_heads=8, n_kv_heads=1), dict(prefill_chunk=30, page_size=32))])
def test_prefill_and_decode_match_full_forward(kw, gkw):
    """Heads of 128 and 64 channels, whole and chunked prompts. Same bound as the contiguous cache's test: bf16 activations
    through two layers."""
    model, ref, tok = model_of(**kw), model_of(**kw), ByteTokenizer()
    gen = build_generator(args(**gkw), model, tok)
    ids = [tok.encode(p, add_bos=True) for p in PROMPTS]
    with torch.inference_mode():
        full = []
        for i in ids:  # in fp32 on the same (rounded) weights: the plain forward takes every head width
            full.append(ref.float()(torch.tensor([i], device="cuda")).float()[0])
        packed = torch.cat([torch.tensor(i[:-1]) for i in ids]).cuda()
        lengths = torch.tensor([len(i) - 1 for i in ids]).cuda()
        pre = gen.prefill(packed.unsqueeze(0), lengths).float()[0]
        nxt = gen.generate_next_token(torch.tensor([[i[-1] for i in ids]], device="cuda")).float()[0]
        gen.release_cache()
    off = 0
    for k, i in enumerate(ids):
        n = len(i) - 1
        scale = full[k].abs().max().item()
        assert (pre[off:off + n] - full[k][:n]).abs().max().item() < 4e-2 * scale
        assert (nxt[k] - full[k][n]).abs().max().item() < 4e-2 * scale
        off += n


@pytest.mark.parametrize("kw", [dict(), dict(attention_window=24, attention_sinks=4), dict(samples_per_prompt=3),
                                dict(repetition_penalty=1.2, frequency_penalty=0.3)])
def test_captured_decode_step_equals_eager(kw):
    """Pages are taken, shared and given back while the captured step is replayed; a second call has another batch."""
    model, tok = model_of(), ByteTokenizer()
    outs = []
    for graph in (False, True):
        gen = build_generator(args(max_gen_len=40, reduce_generation_overhead=graph, **kw), model, tok)
        outs.append([gen.generate(PROMPTS)[0], gen.generate(PROMPTS[:2])[0]])
    assert outs[0] == outs[1]
    assert len(outs[0][0]) == 3 * kw.get("samples_per_prompt", 1)


def test_samples_copy_only_what_they_write():
    model, tok = model_of(), ByteTokenizer()
    gen = build_generator(args(samples_per_prompt=4), model, tok)
    ids = tok.encode(PROMPTS[0], add_bos=True)  # four pages and a part of the fifth
    with torch.inference_mode():
        gen.prefill(torch.tensor([ids]).cuda(), torch.tensor([len(ids)]).cuda())
        used = gen.cache.n_pages - gen.cache.n_free
        a = gen.generate_next_token(torch.tensor([[7, 7, 7, 9]]).cuda())
        assert used == (len(ids) + 15) // 16 and gen.cache.n_pages - gen.cache.n_free == used + 3
        assert torch.equal(a[0, 0], a[0, 1]) and torch.equal(a[0, 0], a[0, 2]) and not torch.equal(a[0, 0], a[0, 3])
    gen.release_cache()


def test_compaction_and_resize_in_mid_generation():
    model, tok = model_of(), ByteTokenizer()
    ids = tok.encode(PROMPTS[0], add_bos=True)
    outs = []
    for move in (False, True):
        gen = build_generator(args(), model, tok)
        with torch.inference_mode():
            gen.prefill(torch.tensor([tok.encode(PROMPTS[2], add_bos=True) + ids]).cuda(),
                        torch.tensor([len(tok.encode(PROMPTS[2], add_bos=True)), len(ids)]).cuda())
            if move:
                gen.cache.free(gen._seqs.pop(0))
                n = gen.cache.compact()
                assert max(gen.cache.pages(gen._seqs[0])) < n
                gen.cache.resize(n + 2)
                gen.setup_generation(None)
                nxt = gen.generate_next_token(torch.tensor([[5]]).cuda())[0, 0]
            else:
                nxt = gen.generate_next_token(torch.tensor([[5, 5]]).cuda())[0, 1]
        outs.append(nxt.clone())
        gen.release_cache()
    assert torch.equal(outs[0], outs[1])


def test_refusals():
    model, tok = model_of(n_heads=16, n_kv_heads=16), ByteTokenizer()  # heads of 32
    with pytest.raises(ValueError):
        build_generator(args(), model, tok)
    with pytest.raises(ValueError):
        build_generator(args(), model_of().float(), tok)
