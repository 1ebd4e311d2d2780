"""Qwen3 over a paged cache: chunks, mixed batches, forked and moved sequences and beam search, against the CPU oracle
run on every sequence from its start (float32 throughout; bfloat16 activations against the oracle that rounds where
the GPU stores).  Logits within 2e-2 as in the other model tests; beams token for token, on prompts whose choices are
apart by at least 1e-3 in the oracle (checked), with scores within 2e-3 per token."""
import numpy as np
import pytest

from kandle_amd import synthetic as syn
from kandle_amd.model_utils import PagedKVCache, Qwen3Config, Qwen3ForCausalLM, init_qwen3_weights
from oracle.qwen3 import Qwen3Oracle

pytestmark = pytest.mark.gpu
ATOL = 2e-2
CFG = dict(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
           num_key_value_heads=2, head_dim=64)


def make(act="float32", seed=3, std=0.1, max_seq=256, **change):
    cfg = Qwen3Config(**{**CFG, **change})
    w = init_qwen3_weights(cfg, seed=seed, std=std)
    return cfg, Qwen3ForCausalLM(cfg, w, max_seq_len=max_seq, activations=act), Qwen3Oracle(cfg, w, max_seq_len=max_seq,
                                                                                           exact=act == "float32")


@pytest.mark.parametrize("act", ["float32", "bfloat16"])
@pytest.mark.parametrize("head_dim,heads,kv", [(64, 4, 2), (128, 6, 2)])
def test_chunks_single_tokens_and_both_together(hip, act, head_dim, heads, kv):
    cfg, model, oracle = make(act, std=0.02, head_dim=head_dim, num_attention_heads=heads, num_key_value_heads=kv)
    cache = model.new_paged_cache(max_sequences=4, num_pages=40)
    ids = [list(syn.randint(10 + s, (150,), 0, cfg.vocab_size)) for s in range(4)]
    at = [0] * 4
    for counts in ([70, 0, 1, 16], [1, 33, 1, 1], [1, 1, 1, 1], [0, 20, 40, 1], [1, 0, 0, 0], [17, 60, 3, 90]):
        packed = sum((ids[s][at[s]:at[s] + n] for s, n in enumerate(counts)), [])
        logits = model.forward_paged(packed, counts, cache).numpy()
        at = [a + n for a, n in zip(at, counts)]
        assert cache.kv_lens.numpy().tolist() == at == cache.lens.tolist()
        for row, s in enumerate(np.flatnonzero(counts)):
            want = oracle.forward(ids[s][:at[s]], 0)
            assert np.abs(logits[row] - want).max() < ATOL, (counts, s)
    cache.dispose()
    model.dispose()


def test_forked_freed_and_moved_sequences(hip):
    cfg, model, oracle = make(std=0.02)
    cache = model.new_paged_cache(max_sequences=3, num_pages=24)
    ids = [list(syn.randint(20, (45,), 0, cfg.vocab_size)), list(syn.randint(21, (30,), 0, cfg.vocab_size)), []]
    model.forward_paged(ids[0] + ids[1], [45, 30, 0], cache).dispose()
    cache.fork([0, 1, 0])                      # a second answer to the first prompt
    ids[2] = list(ids[0])
    used = cache.num_pages - cache.free_pages()
    assert used == 3 + 2                       # shared, not copied
    for step in range(3):
        new = [list(syn.randint(30 + 3 * step + s, (n,), 0, cfg.vocab_size)) for s, n in enumerate((1, 20, 2))]
        ids = [a + b for a, b in zip(ids, new)]
        logits = model.forward_paged(sum(new, []), [1, 20, 2], cache).numpy()
        for s in range(3):
            assert np.abs(logits[s] - oracle.forward(ids[s], 0)).max() < ATOL, (step, s)
        if step == 0:
            cache.free([1])
            ids[1] = []
            live = cache.compact()             # the others' pages move to the front
            assert live == cache.num_pages - cache.free_pages() and cache.page_table.numpy().max() < live
    for bad in ([-1], [3]):
        with pytest.raises(ValueError, match="sequences"):
            cache.free(bad)
    with pytest.raises(ValueError, match="parents"):
        cache.fork([0, 1, 3])
    cache.reset()
    assert cache.free_pages() == 24 and cache.lens.tolist() == [0, 0, 0]
    cache.dispose()
    model.dispose()


def test_a_cache_that_is_too_small_refuses_and_stays(hip):
    cfg, model, oracle = make(std=0.02, max_seq=64)
    cache = model.new_paged_cache(max_sequences=2, num_pages=4)
    ids = list(syn.randint(40, (64,), 0, cfg.vocab_size))
    model.forward_paged(ids[:40], [40, 0], cache).dispose()
    with pytest.raises(RuntimeError, match="pages are missing"):
        model.forward_paged(ids[:30], [0, 30], cache)
    with pytest.raises(ValueError, match="Cache overflow"):
        model.forward_paged(ids[:25], [25, 0], cache)
    with pytest.raises(ValueError, match="counts"):
        model.forward_paged(ids[:3], [3], cache)
    with pytest.raises(ValueError, match="tokens"):
        model.forward_paged(ids[:3], [1, 1], cache)
    logits = model.forward_paged(ids[40:48], [8, 0], cache)
    assert np.abs(logits.numpy()[0] - oracle.forward(ids[:48], 0)).max() < ATOL
    cache.dispose()
    for bad in ((2, 0, 3, 64), (2, 4, 0, 64), (2, 4, 3, 0)):
        with pytest.raises(ValueError):
            PagedKVCache(bad[0], 2, 64, *bad[1:])
    with pytest.raises(ValueError, match="page size"):
        PagedKVCache(2, 2, 64, 4, 3, 64, page_size=24)
    model.dispose()


def beams_of(oracle, prompt, num_beams, steps, eos):
    """Beam search from whole forwards; (tokens, sum) of the last beams, and the smallest gap at a choice."""
    live, gap = [([], 0.0, False)], np.inf
    for _ in range(steps):
        every = []
        for i, (toks, total, done) in enumerate(live):
            if done:
                every.append((total, i, eos))
                continue
            x = oracle.forward(list(prompt) + toks, 0).astype(np.float64)
            x -= x.max()
            x -= np.log(np.exp(x).sum())
            every += [(total + x[t], i, t) for t in range(len(x))]
        every.sort(key=lambda c: (-c[0], c[1], c[2]))
        top = [c[0] for c in every[:num_beams + 1]]
        gap = min(gap, np.diff(top[::-1]).min())
        live = [(live[i][0] + ([] if live[i][2] else [t]), s, live[i][2] or t == eos) for s, i, t in every[:num_beams]]
        if all(d for _, _, d in live):
            break
    return [(t, s) for t, s, _ in live], gap


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("num_beams,eos", [(4, None), (3, "seen"), (1, None)])
def test_beam_search(hip, num_beams, eos, use_graph):
    cfg, model, oracle = make()
    prompts = [list(syn.randint(50 + i, (n,), 0, cfg.vocab_size)) for i, n in enumerate((37, 5, 16))]
    steps = 9
    if eos == "seen":                          # a token that beams of the first prompt reach
        eos = beams_of(oracle, prompts[0], num_beams, 4, None)[0][1][0][2]
    got = model.generate_beams(prompts, num_beams, steps, eos_token_id=eos, length_penalty=0.7, use_graph=use_graph)
    for p, beams in zip(prompts, got):
        want, gap = beams_of(oracle, p, num_beams, steps, eos)
        assert gap > 1e-3
        want = sorted([(t, s / len(t) ** 0.7) for t, s in want], key=lambda x: -x[1])
        assert [t for t, _ in beams] == [t for t, _ in want]
        for (_, a), (t, b) in zip(beams, want):
            assert abs(a - b) < 2e-3 * len(t)
    if num_beams == 1:
        assert got[0][0][0] == model.generate(np.asarray(prompts[0], np.int32), steps)
    model.dispose()


def test_beams_by_graph_are_the_eager_ones_bit_for_bit(hip):
    cfg, model, _ = make("bfloat16", head_dim=128)
    prompts = [list(syn.randint(60 + i, (n,), 0, cfg.vocab_size)) for i, n in enumerate((64, 100))]
    a = model.generate_beams(prompts, 5, 40, use_graph=False)
    b = model.generate_beams(prompts, 5, 40, use_graph=True)
    c = model.generate_beams(prompts, 5, 40, use_graph=True, page_size=64)
    assert a == b
    assert [[t for t, _ in g] for g in a] == [[t for t, _ in g] for g in c]
    model.dispose()


def test_beam_refusals(hip):
    cfg, model, _ = make()
    for bad in (([], 2, 4), ([1, 2], 2, 4), ([[]], 2, 4), ([[1]], 0, 4), ([[1]], 2, 0), ([[1]], 65, 4), ([[1]], 2, 256)):
        with pytest.raises(ValueError):
            model.generate_beams(*bad)
    with pytest.raises(ValueError, match="eos"):
        model.generate_beams([[1]], 2, 4, eos_token_id=500)
    with pytest.raises(RuntimeError, match="pages are missing"):
        model.generate_beams([[1, 2, 3]], 4, 40, num_pages=4)
    model.dispose()


def test_heads_that_paged_attention_does_not_take_are_refused(hip):
    cfg, model, _ = make(head_dim=32)
    with pytest.raises(ValueError, match="64 or 128"):
        model.new_paged_cache(2, 8)
    with pytest.raises(ValueError, match="64 or 128"):
        model.generate_beams([[1, 2]], 2, 4)
    model.dispose()
