"""The model's step that draws the next tokens on the GPU: the logits are those of
decode_sequences on a twin of each sequence (the same kernels on the same values), the
draw numpy's in 64 bits (test_gpu_sample).  Large vocabularies' logits are copied out in
bands there and stay whole here, so that their sums may be ordered differently: 1e-6 of
a logit's size for the some thousand additions in f32 at most, and twice that, of logits
up to 20, of a probability."""

import sys

import numpy as np
import pytest

import test_gpu_sample as ts
from tvara_amd import native
from tvara_amd import gguf_writer as gf

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def twins(model, rng, n):
    """Two lists of n sequences with the same ragged texts."""
    a, b = ([model.new_sequence() for _ in range(n)] for _ in range(2))
    for x, y in zip(a, b):
        text = [int(t) for t in rng.integers(0, model.vocab_size, int(rng.integers(1, 9)))]
        model.decode_batch(x, text)
        model.decode_batch(y, text)
    return a, b


def expect(logits, u, tokens, chances, bar=2.0 ** -24 + 1e-9, **how):
    each = {k: np.broadcast_to(np.asarray(v), u.shape) for k, v in how.items()}
    for i, row in enumerate(logits):
        token, chance = ts.draw(row, u[i], **{k: v[i] for k, v in each.items()})
        assert tokens[i] == token, (i, tokens[i], token)
        assert abs(chances[i] - chance) <= bar * chance, (i, chances[i], chance)


NAMES = {"t": "temperature", "k": "top_k", "p": "top_p", "m": "min_p"}


@pytest.mark.parametrize("nseq,hidden,vocab", [(1, 64, 100), (2, 64, 100), (41, 128, 500), (70, 128, 500), (1, 128, 34001), (66, 128, 34001),
                                               (3, 40, 90)])
def test_draws(tmp_path, nseq, hidden, vocab):
    say("sample sequences", nseq, hidden, vocab)
    spec = gf.LlamaSpec(matrix_type=gf.T_F32 if hidden == 40 else gf.T_Q8_0, hidden=hidden, intermediate=72 if hidden == 40 else 256,
                        heads=4, kv_heads=2, vocab=vocab)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=16 * nseq, block_tokens=4)
    rng = np.random.default_rng(nseq + vocab)
    a, b = twins(model, rng, nseq)
    tokens = [int(t) for t in rng.integers(0, vocab, nseq)]
    mixed = {"t": rng.uniform(0.3, 2, nseq).astype(np.float32), "k": rng.integers(0, 60, nseq), "p": rng.uniform(0.5, 1, nseq).astype(np.float32),
             "m": rng.uniform(0, 0.1, nseq).astype(np.float32)}
    for how in ({}, {"t": 0.0}, {"t": 0.7, "k": 20}, {"p": 0.9}, {"m": 0.05}, mixed):
        logits = model.decode_sequences(a, tokens)
        u = rng.random(nseq).astype(np.float32)
        got, chances = model.sample_sequences(b, tokens, u, **{NAMES[k]: v for k, v in how.items()})
        expect(logits, u, got, chances, 4e-5 if vocab > 30000 else 2.0 ** -24 + 1e-9, **how)
        if how.get("t") == 0.0 if np.ndim(how.get("t")) == 0 else False:
            assert got == np.argmax(logits, 1).tolist()
        tokens = got  # (the next step's)
    assert model.sample_sequences([], [], [])[0] == []


def test_all_or_nothing(tmp_path):
    say("sample sequences, all or nothing")
    spec = gf.LlamaSpec(context=12)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=14, block_tokens=4)
    a, b, c = (model.new_sequence() for _ in range(3))
    ta, tb, tc = (model.new_sequence() for _ in range(3))
    for s, t, n in ((a, ta, 4), (b, tb, 7), (c, tc, 11)):  # 1 + 2 + 3 blocks, twice
        for x in (s, t):
            model.decode_batch(x, list(range(1, n + 1)))
    u = np.array([0.3, 0.6], np.float32)
    with pytest.raises(ValueError):
        model.sample_sequences([a, b], [1], u)
    with pytest.raises(ValueError):
        model.sample_sequences([a, b], [1, 2], u[:1])
    with pytest.raises(ValueError):
        model.sample_sequences([a, b], [1, spec.vocab], u)
    with pytest.raises(ValueError):
        model.sample_sequences([a, b], [1, 2], u, top_k=-1)
    for bad in (dict(temperature=-1.0), dict(temperature=[1.0, np.nan]), dict(top_p=np.nan), dict(min_p=-0.1),
                dict(uniforms=np.array([0.5, 1.0], np.float32)), dict(uniforms=np.array([np.nan, 0.5], np.float32))):
        with pytest.raises(Exception, match="invalid sampling parameters"):
            model.sample_sequences([a, b], [1, 2], **{"uniforms": u, **bad})
    with pytest.raises(Exception, match="duplicate sequence"):
        model.sample_sequences([a, a], [1, 2], u)
    # c takes its twelfth token, then has no room; b and a have not moved
    got, chances = model.sample_sequences([c], [5], u[:1])
    expect(model.decode_sequences([tc], [5]), u[:1], got, chances)
    with pytest.raises(Exception, match="limits"):
        model.sample_sequences([b, c], [1, 2], u)
    for s, t in ((b, tb), (a, ta)):
        got, chances = model.sample_sequences([s], [9], u[1:])
        expect(model.decode_sequences([t], [9]), u[1:], got, chances)
