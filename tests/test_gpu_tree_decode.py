"""The cache operators together: the tree-decoding example on a synthetic model, held against
the batch engine's logits token by token."""
import importlib.util
import os

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

# relative rounding of a cached element; f32: of what a torch and an engine projection differ by
EPS = {"f32": 2.0 ** -16, "f16": 2.0 ** -11, "q8": 1 / 254}


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("tree_decode", os.path.join(ROOT, "examples", "tree_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def path(sb, workdir):
    p = str(workdir / "tree_decode.gguf")
    sb.synth_gguf(p, n_layers=2, d_model=512, ffn_hidden=768, n_heads=8, n_kv_heads=2, vocab=300, max_seq=512, q4k=False, seed=3)
    return p


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_tree_decoding_follows_the_engine(sb, example, path, kv):
    """Every token that a tree step adds is the engine's greedy choice after the tokens before it,
    up to what the rounding of the cache moves a logit by; steps are saved; a sequence that starts
    from another's saved rows goes on as that one does."""
    model = example.Model(path)
    dec = example.Decoder(model, 3, example.KV[kv])
    prompt = np.random.default_rng(0).integers(0, 300, 77).tolist()
    first = dec.prompt(1, prompt)
    assert dec.ctx == [0, 77, 0]
    K, V = dec.save(1)
    dec.load(0, K, V)
    dec.load(2, K, V)
    if kv != "q8":                                     # 8 bits of 8 bits: the scale may round anew
        for a, b in zip(dec.save(0), (K, V)):
            assert bool((a == b).all())
    texts = [prompt + [t] for t in (first, first, (first + 5) % 300)]
    steps = example.generate(dec, texts, 60)
    assert steps < 60 and [len(t) for t in texts] == [138] * 3
    if kv != "q8":
        assert texts[0] == texts[1]
    eng = sb.LlamaBatch(path, max_batch=16, max_seq=512)
    for t in texts[1:]:
        s = eng.open()
        rc, logits = eng.prefill(s, t[:77])
        assert rc == 0
        checks = [(logits, t[77])] if t is texts[1] else []
        for i in range(77, len(t) - 1):
            rc, _, lg = eng.step([s], [t[i]], want_logits=True)
            assert rc == 0
            checks.append((lg[0], t[i + 1]))
        for lg, chosen in checks:
            # two layers, K and V each: a handful of such errors on the way to a logit
            assert lg[chosen] >= lg.max() - 8 * EPS[kv] * np.abs(lg).max()
        eng.release(s)
    eng.close()


def test_draft(example):
    """The tree's shape: continuations merged, parents before children, 64 nodes at most."""
    parents, tokens = example.draft([1, 2, 3, 4, 1, 2, 3, 5, 1, 2], depth=3)
    paths = set()
    for i in range(len(tokens)):
        p, at = [], i
        while at >= 0:
            p.append(tokens[at])
            at = int(parents[at])
        paths.add(tuple(p[::-1]))
    assert paths == {(2,), (2, 3), (2, 3, 5), (2, 3, 5, 1), (2, 3, 4), (2, 3, 4, 1)}
    parents, tokens = example.draft(list(np.random.default_rng(0).integers(0, 2, 400)), depth=40, branches=50)
    assert len(tokens) == 64 and all(p < i for i, p in enumerate(parents))
    assert example.draft([7], depth=4)[1] == [7] and example.draft([7, 7], depth=0)[1] == [7]


def test_engine_refuses_an_8_bit_cache(sb, path):
    with pytest.raises(RuntimeError, match="8 bits"):
        sb.LlamaBatch(path, kv_dtype=sb.KV_Q8)
