"""The model over the paged cache (instantllm_b200/paged_engine.py) against the CPU oracle and against VerifyEngine: prompts in
a batch and in chunks, one token a step, draft trees with their commit."""
import numpy as np
import pytest

from instantllm_b200 import synth

VOCAB = 4096


@pytest.fixture(scope="module")
def model():
    import torch  # noqa: F401

    from instantllm_b200.paged_engine import PagedEngine
    from oracle import qwen_oracle as Q

    w = synth.make_weights("q4", n_layers=2, vocab=VOCAB, seed=21)
    return PagedEngine(w, n_pages=64, page_size=16, max_seqs=6, max_len=160), Q.model_from_weights(w), w


def prompt(n, seed):
    return (synth.make_prompt(n, seed=seed) % VOCAB).tolist()


@pytest.mark.gpu
def test_prompts_chunks_and_steps(model):
    """Logits of a ragged batch, of a second chunk over it, and of single steps: within the passes' own bound of the fp32
    oracle (fp16 activations: 0.05)."""
    from oracle import qwen_oracle as Q

    eng, m, _ = model
    first = {3: prompt(37, 1), 0: prompt(1, 2), 5: prompt(64, 3)}
    second = {0: prompt(20, 4), 5: prompt(3, 5)}
    caches = {s: Q.KVCache(2, 160) for s in first}
    got = eng.prefill(first).cpu().numpy()
    want = [Q.forward_causal(m, caches[s], t, 0) for s, t in first.items()]
    assert np.abs(got - np.stack(want)).max() < 0.05
    got = eng.prefill(second).cpu().numpy()
    want = [Q.forward_causal(m, caches[s], t, len(first[s])) for s, t in second.items()]
    assert np.abs(got - np.stack(want)).max() < 0.05
    pos = {s: len(first[s]) + len(second.get(s, [])) for s in first}
    for step in range(3):
        toks = {s: 7 * step + s for s in first}
        got = eng.decode(toks).cpu().numpy()
        want = [Q.forward_causal(m, caches[s], [toks[s]], pos[s] + step) for s in first]
        assert np.abs(got - np.stack(want)).max() < 0.05
    for s in first:
        eng.release(s)
    eng.kv.check()
    assert eng.kv.free_pages == 64


@pytest.mark.gpu
def test_trees_and_commit(model):
    """Trees of different sizes in one pass: logits against the oracle's tree pass, the committed path and the compacted
    cache against a causal continuation."""
    from oracle import qwen_oracle as Q

    eng, m, _ = model
    rng = np.random.default_rng(9)
    prompts = {1: prompt(30, 6), 2: prompt(50, 7)}
    first = dict(zip(prompts, eng.prefill(prompts).argmax(-1).tolist()))
    caches, truth = {}, {}
    for s, p in prompts.items():
        caches[s] = Q.KVCache(2, 160)
        Q.forward_causal(m, caches[s], p, 0)
        truth[s] = Q.greedy(m, p, 10)[0]
    trees = {1: synth.seeded_tree(rng, truth[1], n=16, p_match=0.9, vocab=VOCAB),
             2: synth.seeded_tree(rng, truth[2], n=5, p_match=0.9, vocab=VOCAB)}
    logits, out = eng.verify(trees, first)
    logits = logits.cpu().numpy()
    for i, s in enumerate(trees):
        n = trees[s]["n"]
        want = Q.tree_pass(m, caches[s].copy(), len(prompts[s]), first[s], trees[s])
        assert np.abs(logits[i, :n] - want).max() < 0.05
        assert len(out[s]) >= 1 and eng.lens[s] == len(prompts[s]) + len(out[s])
        # the cache now holds prompt, root and accepted drafts in order: the next step agrees with a causal run over them
        ids = prompts[s] + [first[s]] + out[s]
        got = eng.decode({s: ids[-1]})[0].cpu().numpy()
        assert np.abs(got - Q.forward_causal(m, Q.KVCache(2, 160), ids, 0)).max() < 0.05
    for s in prompts:
        eng.release(s)
    eng.kv.check()


@pytest.mark.gpu
def test_generate_with_and_without_trees(model):
    """Trees change no token of a greedy decode; VerifyEngine, on the same weights, takes the same ones as long as the two best
    logits are not within rounding of each other."""
    from instantllm_b200.engine import VerifyEngine

    eng, _, w = model
    prompts = [prompt(n, 30 + n) for n in (5, 33, 17, 60)]
    plain = eng.generate(prompts, 12)
    rng = np.random.default_rng(3)

    def tree_fn(s, ids):  # drafts from the known continuation, some of them wrong
        done = len(ids) - len(prompts[s])
        return synth.seeded_tree(rng, (plain[s] + [0] * 20)[done:], n=16, p_match=0.7, vocab=VOCAB)

    assert eng.generate(prompts, 12, tree_fn=tree_fn) == plain
    ve = VerifyEngine(w, max_ctx=160, max_steps=64)
    for p, got in zip(prompts, plain):
        ve.begin(0, 12)
        ve.prefill(p)
        for _ in range(11):
            ve.pass_(synth.root_tree())
        want = ve.tokens(12)
        same = next((i for i, (a, b) in enumerate(zip(got, want)) if a != b), len(got))
        if same < len(got):  # the first difference must be a near tie
            lg = eng.prefill({0: p + got[:same]})[0]
            eng.release(0)
            assert abs(float(lg[got[same]] - lg[want[same]])) < 0.05
    ve.close()


def test_dense_layouts_match_the_oracle():
    """The dequantised weights of every format (CPU)."""
    from instantllm_b200.paged_engine import _dense
    from oracle import qwen_oracle as Q

    rng = np.random.default_rng(0)
    for fmt in ("q4", "q8", "q8g32", "f16"):
        m = synth.make_matrix(fmt, 32, 128, rng)
        assert np.array_equal(_dense(m, "cpu").numpy(), Q.dequant(m).astype(np.float16))


@pytest.mark.gpu
def test_small_trees_beside_large_ones(model):
    """A request whose own tree still fits its row of the table is served beside one with a larger tree, down to a context of one
    token; logits against the oracle's tree pass, tokens and lengths as committed alone, and no page beyond a request's own
    slots."""
    from oracle import qwen_oracle as Q

    eng, m, _ = model
    rng = np.random.default_rng(10)
    prompts = {0: prompt(155, 8), 1: prompt(40, 9), 4: prompt(1, 10), 5: prompt(9, 11)}
    sizes = {0: 5, 1: 16, 4: 1, 5: 7}
    first = dict(zip(prompts, eng.prefill(prompts).argmax(-1).tolist()))
    caches = {}
    for s, p in prompts.items():
        caches[s] = Q.KVCache(2, 180)
        Q.forward_causal(m, caches[s], p, 0)
    trees = {s: synth.seeded_tree(rng, Q.greedy(m, prompts[s], 10)[0], n=k, p_match=0.9, vocab=VOCAB) if k > 1 else synth.root_tree()
             for s, k in sizes.items()}
    logits, out = eng.verify(trees, first)
    eng.kv.check()
    logits = logits.cpu().numpy()
    for i, s in enumerate(trees):
        n = trees[s]["n"]
        want = Q.tree_pass(m, caches[s].copy(), len(prompts[s]), first[s], trees[s])
        assert np.abs(logits[i, :n] - want).max() < 0.05
        assert np.array_equal(logits[i, n:], np.repeat(logits[i, :1], logits.shape[1] - n, 0))
        assert len(eng.kv._pool.held[s]) == -(-(len(prompts[s]) + n) // 16)
        ids = prompts[s] + [first[s]] + out[s]
        assert eng.lens[s] == len(ids) - 1
        if len(ids) <= 160:
            got = eng.decode({s: ids[-1]})[0].cpu().numpy()
            assert np.abs(got - Q.forward_causal(m, Q.KVCache(2, 180), ids, 0)).max() < 0.05
    for s in prompts:
        eng.release(s)
    eng.kv.check()
    assert eng.kv.free_pages == 64


@pytest.mark.gpu
def test_trees_of_different_sizes_under_a_window(model):
    """The same trees in one call and each in its own, over a window that cuts into the padding: the passes' own bound apart."""
    from instantllm_b200.paged_engine import PagedEngine

    w = model[2]
    rng = np.random.default_rng(11)
    sizes = {0: 16, 1: 3, 2: 1, 3: 9}
    prompts = {s: prompt(n, 40 + s) for s, n in {0: 60, 1: 35, 2: 20, 3: 4}.items()}
    for window, sinks in ((6, 2), (20, 0)):
        eng = PagedEngine(w, n_pages=64, page_size=16, max_seqs=4, max_len=160, window=window, sinks=sinks)
        first = dict(zip(prompts, eng.prefill(prompts).argmax(-1).tolist()))
        trees = {s: synth.seeded_tree(rng, [int(x) for x in rng.integers(0, VOCAB, 16)], n=k, vocab=VOCAB) if k > 1 else synth.root_tree()
                 for s, k in sizes.items()}
        got = eng.verify(trees, first, commit=False)[0].cpu().numpy()
        for i, s in enumerate(trees):
            alone = eng.verify({s: trees[s]}, first, commit=False)[0].cpu().numpy()
            assert np.abs(got[i, :sizes[s]] - alone[0]).max() < 0.05
        eng.kv.check()


def test_a_batch_gets_all_its_pages_or_none():
    """Requests that the pool cannot hold together leave no page behind with any of them (host side)."""
    from instantllm_b200 import paged
    from instantllm_b200._lib import VpError

    p = paged.PagePool(6, 16, 3, 4)
    assert p.fits({0: 32, 1: 64}) == 6 and p.fits({0: 0}) == 0
    for bad in ({0: 33, 1: 64}, {0: 16, 2: 65}):
        with pytest.raises(VpError):
            p.fits(bad)
    with pytest.raises(IndexError):
        p.fits({0: 16, -1: 16})
    assert p.held == [[], [], []] and len(p.free) == 6
    p.reserve(0, 20)
    assert p.fits({0: 32, 1: 64}) == 4


@pytest.mark.gpu
def test_a_refused_batch_takes_no_pages(model):
    """The first prompt of a batch fits and the second does not: neither keeps pages, and each alone is served."""
    from instantllm_b200._lib import VpError
    from instantllm_b200.paged_engine import PagedEngine

    eng = PagedEngine(model[2], n_pages=12, page_size=16, max_seqs=3, max_len=160)
    with pytest.raises(VpError, match="pages wanted"):
        eng.prefill({0: prompt(100, 1), 1: prompt(120, 2)})
    assert eng.kv.free_pages == 12 and eng.lens == [0, 0, 0]
    eng.prefill({0: prompt(100, 1)})
    with pytest.raises(VpError, match="pages wanted"):
        eng.prefill({0: prompt(30, 1), 1: prompt(70, 2)})
    assert eng.kv.free_pages == 5 and eng.lens == [100, 0, 0]
    eng.kv.check()


@pytest.mark.gpu
def test_generate_no_tokens(model):
    """A limit of no tokens gives none, and touches no request."""
    eng = model[0]
    free = eng.kv.free_pages
    assert eng.generate([prompt(5, 1), prompt(9, 2)], 0) == [[], []]
    assert [len(t) for t in eng.generate([prompt(5, 1), prompt(9, 2)], 1)] == [1, 1]
    assert eng.kv.free_pages == free and eng.lens == [0] * 6


@pytest.mark.gpu
def test_generate_after_one_that_failed(model):
    """A generate that runs out of pages half way, or whose drafts raise, leaves the engine as it was: the next one gives the tokens
    of a fresh engine. Requests that hold a context are not generated onto."""
    from instantllm_b200._lib import VpError
    from instantllm_b200.paged_engine import PagedEngine

    eng = PagedEngine(model[2], n_pages=5, page_size=16, max_seqs=3, max_len=160)
    prompts = [prompt(30, 1), prompt(17, 2)]
    want = model[0].generate(prompts, 6, eos=())

    def bad(s, ids):
        if len(ids) > 19:
            raise KeyError("draft")
        return synth.root_tree()

    for fails, kind in ((lambda: eng.generate(prompts, 90, eos=()), VpError), (lambda: eng.generate(prompts, 90, tree_fn=bad, eos=()), KeyError),
                        (lambda: eng.generate([prompt(3, i) for i in range(4)], 5), IndexError)):
        with pytest.raises(kind):
            fails()
        assert eng.lens == [0, 0, 0] and eng.kv.free_pages == 5
    assert eng.generate(prompts, 6, eos=()) == want
    eng.prefill({1: prompt(4, 3)})
    with pytest.raises(VpError, match="release"):
        eng.generate(prompts, 6)
    assert eng.lens == [0, 4, 0]
    eng.release(1)
    assert eng.generate([], 5) == []
