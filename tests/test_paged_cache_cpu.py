"""Ownership of pages (reference counts, copies on write, compaction) against plain per-sequence copies, and generation on it."""
import random

import pytest
import torch

from lingua_b200.generation import (PackedCausalTransformerGenerator, PackedCausalTransformerGeneratorArgs, build_generator,
                                    sample_tokens)
from lingua_b200.generation_paged import PagedCausalTransformerGenerator
from lingua_b200.models.transformer import LMTransformer, LMTransformerArgs
from lingua_b200.paged_cache import CacheFull, PagedCache
from lingua_b200.tokenizer import ByteTokenizer


def write(cache, seq, at, values):
    """values [n, rows]: stands in for the append kernel, every row of the pool gets the number."""
    P, pages = cache.page_size, cache.pages(seq)
    for i, v in enumerate(values):
        cache.pool[:, pages[(at + i) // P], (at + i) % P] = v


def read(cache, seq):
    P, pages = cache.page_size, cache.pages(seq)
    return [float("nan") if pages[i // P] < 0 else cache.pool[1, pages[i // P], i % P, 0, 0].item()
            for i in range(cache.length(seq))]


def check(cache, shadow):
    for s, want in shadow.items():
        got = read(cache, s)
        assert len(got) == len(want) and all(g == w or w is None for g, w in zip(got, want))
    owned = {}
    for s in shadow:
        for p in cache.pages(s):
            if p >= 0:
                owned[p] = owned.get(p, 0) + 1
    assert sorted(set(range(cache.n_pages)) - set(owned)) == sorted(cache._free)
    assert all(cache._refs[p] == owned.get(p, 0) for p in range(cache.n_pages))


@pytest.mark.parametrize("seed", range(6))
def test_random_life_of_a_cache(seed):
    rng = random.Random(seed)
    cache = PagedCache(1, 40, 16, 1, 2, torch.float32, "cpu")
    shadow, n = {}, 0
    for _ in range(120):
        do = rng.choice(["add", "grow", "grow", "grow", "fork", "free", "behind", "compact", "resize"])
        some = rng.sample(sorted(shadow), min(len(shadow), rng.randint(1, 4)))
        if do == "add":
            shadow[cache.add()] = []
        elif do == "grow" and some:
            new = [rng.choice([0, 1, 1, 15, 16, 33]) for _ in some]
            before = {s: cache.pages(s) for s in shadow}
            try:
                cache.reserve(some, new)
            except CacheFull:
                assert before == {s: cache.pages(s) for s in shadow}
            else:
                for s, k in zip(some, new):
                    vals = [float(n + i + 1) for i in range(k)]
                    n += k
                    write(cache, s, len(shadow[s]), vals)
                    shadow[s] = shadow[s] + vals
        elif do == "fork" and some:
            for s in cache.fork(some[0], 2):
                shadow[s] = list(shadow[some[0]])
        elif do == "free" and some:
            cache.free(some[0])
            del shadow[some[0]]
        elif do == "behind" and some:
            w, k = rng.choice([1, 20, 40]), rng.choice([0, 3, 17])
            cache.release_behind(some[0], w, k)
            L = len(shadow[some[0]])
            shadow[some[0]] = [v if j > L - w or j < k else None for j, v in enumerate(shadow[some[0]])]
        elif do == "compact":
            used = cache.compact()
            assert all(p < used for s in shadow for p in cache.pages(s))
        elif do == "resize":
            try:
                cache.resize(rng.choice([30, 40, 50]))
            except CacheFull:
                pass
        check(cache, shadow)
    for s in list(shadow):
        cache.free(s)
    assert cache.n_free == cache.n_pages


def test_refusals():
    for kw in (dict(page_size=24), dict(n_pages=0), dict(n_layers=0)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(n_layers=1, n_pages=4, page_size=16, n_kv_heads=1, head_dim=2, device="cpu"), **kw})
    cache = PagedCache(1, 4, 16, 1, 2, torch.float32, "cpu")
    s = cache.add()
    for seqs, new in (([s], [1, 2]), ([s, s], [1, 1]), ([s], [-1])):
        with pytest.raises(ValueError):
            cache.reserve(seqs, new)
    with pytest.raises(CacheFull):
        cache.reserve([s], [65])
    assert cache.length(s) == 0 and cache.n_free == 4
    cache.reserve([s], [64])
    with pytest.raises(ValueError):
        cache.table([s], 3)
    assert cache.table([s], 6)[0].tolist() == [0, 1, 2, 3, -1, -1]
    with pytest.raises(CacheFull):
        cache.resize(3)
    with pytest.raises(KeyError):
        cache.free(s + 1)


# ----------------------------------------------------------------------------- generation
def model_of(window=None, seed=0, **kw):
    torch.manual_seed(seed)
    m = LMTransformer(LMTransformerArgs(**{**dict(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=258, max_seqlen=256,
                                                  sliding_window=window), **kw}))
    m.init_weights()
    return m.eval()


def args(**kw):
    return PackedCausalTransformerGeneratorArgs(**{**dict(max_gen_len=20, max_tokens=640, dtype="fp32", device="cpu"), **kw})


PROMPTS = ["hello world, this is a longer prompt", "abc", "the quick brown fox jumps over the lazy dog"]


@pytest.mark.parametrize("kw", [dict(), dict(prefill_chunk=7), dict(prefill_chunk=1), dict(page_size=32, prefill_chunk=50),
                                dict(max_tokens=160)])
def test_same_texts_as_the_contiguous_cache(kw):
    model = model_of()
    want = PackedCausalTransformerGenerator(args(**{k: v for k, v in kw.items() if k == "max_tokens"}), model,
                                            ByteTokenizer()).generate(PROMPTS)
    gen = build_generator(args(**{**dict(page_size=16), **kw}), model, ByteTokenizer())
    assert isinstance(gen, PagedCausalTransformerGenerator)
    got = gen.generate(PROMPTS)
    assert got[0] == want[0]
    for a, b in zip(got[1], want[1]):
        assert torch.allclose(a, b, atol=1e-4)
    assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


@pytest.mark.parametrize("chunk", [None, 5])
def test_window_follows_the_models_own_mask_and_gives_pages_back(chunk):
    model, ref = model_of(window=12, n_layers=1), model_of(window=12, n_layers=1)  # the same weights, no cache attached
    tok = ByteTokenizer()
    gen = build_generator(args(page_size=16, prefill_chunk=chunk), model, tok)
    ids = tok.encode(PROMPTS[0] * 2, add_bos=True)
    with torch.inference_mode():
        out = gen.prefill(torch.tensor([ids]), torch.tensor([len(ids)]))
        assert torch.allclose(out[0], ref(torch.tensor([ids]))[0], atol=1e-4)
        for t in (5, 77, 200, 9) * 10:
            ids.append(t)
            nxt = gen.generate_next_token(torch.tensor([[t]]))
            assert torch.allclose(nxt[0, 0], ref(torch.tensor([ids]))[0, -1], atol=1e-4)
    assert sum(p >= 0 for p in gen.cache.pages(gen._seqs[0])) <= 2
    gen.release_cache()


def test_sinks_stay_visible():
    model = model_of(n_layers=1)
    tok = ByteTokenizer()
    gen = build_generator(args(page_size=16, attention_window=8, attention_sinks=3), model, tok)
    ids = tok.encode(PROMPTS[0] * 2, add_bos=True)
    with torch.inference_mode():
        out = gen.prefill(torch.tensor([ids]), torch.tensor([len(ids)]))[0]
        x = model.tok_embeddings(torch.tensor([ids]))
        at = model.layers[0].attention
        h = model.layers[0].attention_norm(x)
        from lingua_b200.ops.functional import rope_ref

        T = len(ids)
        cs = model.rope_embeddings()
        q, k = (rope_ref(w(h).view(1, T, -1, 16), cs)[0] for w in (at.wq, at.wk))
        v = at.wv(h).view(T, -1, 16)
        i, j = torch.arange(T).view(-1, 1), torch.arange(T).view(1, -1)
        see = (j <= i) & ((j > i - 8) | (j < 3))
        s = torch.einsum("thd,shd->hts", q, k.repeat_interleave(2, 1)) / 4
        o = torch.einsum("hts,shd->thd", torch.softmax(s.masked_fill(~see, float("-inf")), -1), v.repeat_interleave(2, 1))
        y = x + at.wo(o.reshape(1, T, -1))
        y = y + model.layers[0].feed_forward(model.layers[0].ffn_norm(y))
        assert torch.allclose(out, model.output(model.norm(y))[0], atol=1e-4)
    gen.release_cache()


def test_samples_share_their_prompt():
    model = model_of()
    gen = build_generator(args(page_size=16, samples_per_prompt=3), model, ByteTokenizer())
    texts, lls, _ = gen.generate(PROMPTS)
    one = build_generator(args(page_size=16), model, ByteTokenizer()).generate(PROMPTS)
    assert texts == [t for t in one[0] for _ in range(3)] and len(lls) == len(PROMPTS)  # greedy samples agree
    torch.manual_seed(0)
    gen = build_generator(args(page_size=16, samples_per_prompt=4, temperature=2.0), model, ByteTokenizer())
    texts = gen.generate(PROMPTS[:1])[0]
    assert len(set(texts)) > 1  # and go their own ways otherwise


def test_controls_reach_the_sampler():
    model, tok = model_of(), ByteTokenizer()
    free = PackedCausalTransformerGenerator(args(), model, tok).generate(PROMPTS)[0]
    for page in (0, 16):
        same = build_generator(args(page_size=page, presence_penalty=0.0, logit_bias={}), model, tok).generate(PROMPTS)[0]
        assert same == free
        only = build_generator(args(page_size=page, allowed_tokens=[ord("x"), ord("y")]), model, tok).generate(PROMPTS)[0]
        assert all(set(t) <= {"x", "y"} and len(t) == 20 for t in only)
        bias = build_generator(args(page_size=page, logit_bias={ord("q"): 100.0}), model, tok).generate(PROMPTS)[0]
        assert all(t == "q" * 20 for t in bias)
        gen = build_generator(args(page_size=page, presence_penalty=1000.0), model, tok)
        ids = []
        gen.controls.grammar = lambda out: ids.append([list(o) for o in out]) or None
        gen.generate(PROMPTS)
        assert all(len(set(o)) == len(o) for o in ids[-1])  # no token twice
        assert [len(o) for o in ids[-1]] == [19] * 3


def test_penalties_follow_the_history():
    """Greedy with penalties against a loop that recomputes everything."""
    model, tok = model_of(), ByteTokenizer()
    kw = dict(repetition_penalty=1.3, presence_penalty=0.2, frequency_penalty=0.4, max_gen_len=12)
    got = build_generator(args(page_size=16, **kw), model, tok).generate(PROMPTS[1:2])[0][0]
    ids, out = tok.encode(PROMPTS[1], add_bos=True), []
    for _ in range(12):
        z = model(torch.tensor([ids + out]))[0, -1].double()
        for t in set(ids + out):
            z[t] = z[t] / 1.3 if z[t] > 0 else z[t] * 1.3
        for t in set(out):
            z[t] -= 0.2 + 0.4 * out.count(t)
        out.append(int(z.argmax()))
    assert got == tok.decode(out)


def test_generators_refuse_what_they_do_not_do():
    model, tok = model_of(), ByteTokenizer()
    for kw in (dict(page_size=16), dict(samples_per_prompt=2), dict(prefill_chunk=4), dict(attention_sinks=2)):
        with pytest.raises(ValueError):
            PackedCausalTransformerGenerator(args(**kw), model, tok)
    for kw in (dict(page_size=24), dict(page_size=16, samples_per_prompt=0), dict(page_size=16, prefill_chunk=0),
               dict(page_size=16, attention_window=-1)):
        with pytest.raises(ValueError):
            build_generator(args(**kw), model, tok).generate(["a"])
    with pytest.raises(CacheFull):
        build_generator(args(page_size=16, max_tokens=16, max_prompt_len=30), model, tok).generate(PROMPTS)
    assert sample_tokens(torch.zeros(1, 2, 4)).shape == (1, 2)


def test_controls_that_leave_nothing_to_sample():
    model, tok = model_of(), ByteTokenizer()
    nan, inf = float("nan"), float("inf")
    for kw in (dict(allowed_tokens=[]), dict(allowed_tokens=[-1]), dict(logit_bias={-2: 1.0}), dict(logit_bias={1: nan}),
               dict(logit_bias={1: inf}), dict(repetition_penalty=0.0), dict(repetition_penalty=inf),
               dict(presence_penalty=nan), dict(frequency_penalty=-inf)):
        with pytest.raises(ValueError):
            build_generator(args(**kw), model, tok)
    for kw in (dict(allowed_tokens=[3, 258]), dict(logit_bias={300: 1.0}), dict(allowed_tokens=[3], logit_bias={3: -inf})):
        with pytest.raises(ValueError):
            build_generator(args(temperature=1.0, **kw), model, tok).generate(PROMPTS[:1])
    # a grammar that has come to its end allows nothing: no matter for a text that is done, an error for one that goes on
    def only(tokens):
        words = [0] * 9
        for t in tokens:
            words[t // 32] |= 1 << t % 32
        return words

    def grammar(out):
        return torch.tensor([only([ord("a")] if len(out[0]) < 2 else []), only([ord("b")])], dtype=torch.int32)

    for page in (0, 16):
        gen = build_generator(args(temperature=1.0, page_size=page, until=["aa"]), model, tok)
        gen.controls.grammar = grammar
        assert gen.generate(PROMPTS[:2])[0] == ["aa", "b" * 20]
        gen = build_generator(args(temperature=1.0, page_size=page), model, tok)
        gen.controls.grammar = grammar
        with pytest.raises(ValueError):
            gen.generate(PROMPTS[:2])
    never = build_generator(args(temperature=1.0, logit_bias={t: -inf for t in range(258) if t != ord("z")}), model, tok)
    assert never.generate(PROMPTS[:1])[0] == ["z" * 20]


def test_an_error_leaves_no_cache_behind():
    """Generation that fails half way gives the cache back: the model itself and other generators of it work as before."""
    model, tok = model_of(), ByteTokenizer()
    ids = torch.tensor([tok.encode(PROMPTS[0], add_bos=True)])
    want = model(ids)
    free = build_generator(args(), model, tok).generate(PROMPTS)[0]

    def stop(out):
        if len(out[0]) == 3:
            raise RuntimeError("stop")

    for page in (0, 16):
        gen = build_generator(args(page_size=page), model, tok)
        gen.controls.grammar = stop
        with pytest.raises(RuntimeError, match="stop"):
            gen.generate(PROMPTS)
        assert torch.equal(model(ids), want)
        gen.controls.grammar = None
        assert gen.generate(PROMPTS)[0] == free
    # caches of the two kinds do not take each other's place
    paged, flat = build_generator(args(page_size=16), model, tok), build_generator(args(), model, tok)
    lens = torch.tensor([ids.numel()])
    with torch.inference_mode():
        for gen in (paged, flat, paged, flat):
            assert torch.allclose(gen.prefill(ids, lens), want, atol=1e-4)
    flat.release_cache()


@pytest.mark.parametrize("samples,max_tokens", [(1, 100), (3, 160), (4, 203)])
def test_long_prompts_are_cut_to_what_the_cache_holds(samples, max_tokens):
    model, tok = model_of(), ByteTokenizer()
    gen = build_generator(args(page_size=16, max_tokens=max_tokens, samples_per_prompt=samples), model, tok)
    room = gen.prompt_room()
    assert 0 < room <= max_tokens - 20 and all(gen.cache_need(n) <= max_tokens for n in range(1, room + 1))
    texts = gen.generate(["x" * n for n in range(room - 18, room + 3)] + ["y" * 300])[0]
    assert len(texts) == 22 * samples and all(texts)
    with pytest.raises(ValueError):
        build_generator(args(page_size=16, max_tokens=16, samples_per_prompt=samples), model, tok).generate(["a"])
