"""Trees of drafted tokens through a whole model (tvara_sequences_verify_trees)
against the same model decoding token by token.

A drafted node's logits are those of the token-by-token decode within 1e-4 *
(1 + |logit|) (the batched products against the single ones, the bar of the
model's other passes).  A greedy choice is therefore the same where the largest
logit leads by more than twice that, 2e-4 * (1 + |largest|); trees are drafted
along the choices up to the first that does not, and the tokens expected after
the accepted nodes are compared where theirs does.
"""

import sys

import numpy as np
import pytest

from tvara_amd import gguf_writer as gf
from tvara_amd import native

pytestmark = pytest.mark.gpu
TOL = 1e-4


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def close(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.all(np.abs(got - want) <= TOL * (1 + np.abs(want)))


def choice(logits):
    """The greedy token, and whether it leads clearly."""
    top = np.sort(logits)[-2:].astype(np.float64)
    return int(np.argmax(logits)), bool(top[1] - top[0] > 2 * TOL * (1 + abs(top[1])))


SPECS = {
    "f32-gqa": dict(),
    "f16-split-tied": dict(matrix_type=gf.T_F16, embed_type=gf.T_F16, norm_type=gf.T_F16, rope_layout="split", output=False),
    "q8_0-gqa4": dict(matrix_type=gf.T_Q8_0, heads=8, kv_heads=2, hidden=128, intermediate=256),
    "q8_0-tied-ragged": dict(matrix_type=gf.T_Q8_0, embed_type=gf.T_Q8_0, output=False, vocab=100, hidden=96,
                             intermediate=160, heads=3, kv_heads=1),
    # head_dim 64 and 128: the tiles, in blocks of 16; a vocabulary in several parts
    "q8_0-d64": dict(matrix_type=gf.T_Q8_0, hidden=256, intermediate=512, heads=4, kv_heads=2, vocab=5003),
    "f32-d128": dict(hidden=256, intermediate=256, heads=2, kv_heads=1),
    # widths that the batched products do not take: token by token
    "odd-widths": dict(hidden=40, intermediate=72, heads=4, kv_heads=2),
}


class Greedy:
    """A sequence decoded token by token on its own."""

    def __init__(self, model, prompt):
        self.model, self.seq = model, model.new_sequence()
        for t in prompt:
            self.logits = model.logits(self.seq, t)

    def choices(self, count):
        """Up to `count` greedy tokens, up to the first unclear choice; they are taken back."""
        start, kept, out = self.model.cache().length(self.seq), self.logits, []
        for _ in range(count):
            token, sure = choice(self.logits)
            if not sure:
                break
            out.append(token)
            self.logits = self.model.logits(self.seq, token)
        self.model.truncate(self.seq, start)
        self.logits = kept
        return out

    def take(self, tokens):
        for t in tokens:
            self.logits = self.model.logits(self.seq, t)


def drafted(rng, right, extra, vocab):
    """A tree that holds the path `right` among `extra` wrong nodes: parents,
    tokens, and the path's nodes."""
    parents, tokens, path, at = [], [], [], -1
    spread = sorted(int(x) for x in rng.integers(0, extra + 1, len(right)))
    for step in range(extra + len(right)):
        if len(path) < len(right) and step == spread[len(path)] + len(path):
            parents.append(at)
            tokens.append(right[len(path)])
            at = len(parents) - 1
            path.append(at)
            continue
        p = int(rng.integers(-1, len(parents)))
        avoid = {right[path.index(p) + 1] if p in path and path.index(p) + 1 < len(right) else -1} if p >= 0 else {
            right[0] if right else -1}
        if p == at:  # a child of the last node taken so far
            avoid.add(right[len(path)] if len(path) < len(right) else -1)
        t = int(rng.integers(0, vocab))
        while t in avoid:
            t = (t + 1) % vocab
        parents.append(p)
        tokens.append(t)
    return parents, tokens, path


@pytest.mark.parametrize("block_tokens", [4, 16])
@pytest.mark.parametrize("name", list(SPECS))
def test_trees_match_token_by_token(tmp_path, name, block_tokens):
    say("verify trees", name, block_tokens)
    spec = gf.LlamaSpec(**SPECS[name])
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=400, block_tokens=block_tokens)
    rng = np.random.default_rng(block_tokens)
    prompts = [[int(t) for t in rng.integers(0, spec.vocab, n)] for n in (1, 5, 17, 16, 3, 30)]
    plain = [Greedy(model, p) for p in prompts]
    seqs = [model.new_sequence() for _ in prompts]
    for s, p in zip(seqs, prompts):
        model.prefill(s, p)
    cache = model.cache()
    taken = 0
    # right tokens and wrong ones of each tree: none right, all right, no tree, a single node
    for right, extra in [((0, 3, 5, 1, 0, 4), (6, 4, 0, 0, 0, 28)), ((2, 0, 1, 6, 4, 0), (0, 1, 9, 3, 40, 0)),
                         ((1, 1, 1, 1, 1, 1), (0, 0, 0, 0, 0, 0))]:
        first, trees, ahead = [], [], []
        for g, r, e in zip(plain, right, extra):
            first.append(choice(g.logits)[0])
            path = g.choices(r + 1)
            ahead.append(path)
            trees.append(drafted(rng, path[:r], e, spec.vocab))
            if not path[:r] and trees[-1][1]:  # an unclear first choice: no root has it
                trees[-1] = (trees[-1][0], [(first[-1] + 1) % spec.vocab] * len(trees[-1][1]), [])
        paths, after = model.verify_trees(seqs, [t[0] for t in trees], [t[1] for t in trees], first)
        for i, (g, (parents, tokens, want)) in enumerate(zip(plain, trees)):
            n = len(want)
            assert paths[i][:n] == want, (i, paths[i], want)
            # behind the planted nodes a wrong one may be the unclear choice
            if len(ahead[i]) > n:
                assert paths[i] == want and after[i] == ahead[i][n], i
            got = [tokens[j] for j in paths[i]]
            taken += len(got)
            g.take(got)
            assert choice(g.logits)[0] == after[i] or not choice(g.logits)[1]
            assert cache.length(seqs[i]) == cache.length(g.seq)
        # the appended K/V: what the next token makes of them
        token = [int(t) for t in rng.integers(0, spec.vocab, len(seqs))]
        got = model.decode_sequences(seqs, token)
        for i, (g, t) in enumerate(zip(plain, token)):
            g.take([t])
            assert close(got[i], g.logits), i
    assert taken > 12


def test_generation_equals_greedy(tmp_path):
    """Drafts from a second reading, some wrong: the same text as one token at a time."""
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, hidden=256, intermediate=512, heads=4, kv_heads=2, vocab=700, context=128)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=64, block_tokens=16)
    rng = np.random.default_rng(3)
    prompt = [int(t) for t in rng.integers(0, spec.vocab, 20)]
    g = Greedy(model, prompt)
    want = g.choices(60)
    say("generation", len(want), "clear choices")
    seq = model.new_sequence()
    after = choice(model.prefill(seq, prompt))[0]
    text, steps = [], 0
    while len(text) + 7 < len(want):
        ahead = want[len(text):len(text) + 6]
        wrong = int(rng.integers(1, 7))  # from this draft on
        chain = [t if i < wrong else (t + 1) % spec.vocab for i, t in enumerate(ahead)]
        parents, tokens = [-1, *range(5)] + [0, 0], chain + [(ahead[1] + 2) % spec.vocab, (ahead[1] + 3) % spec.vocab]
        (path,), (after,) = model.verify_trees([seq], [parents], [tokens], [after])
        assert path == list(range(wrong)) and after == want[len(text) + wrong]
        text += [tokens[j] for j in path]
        steps += 1
    assert text == want[:len(text)] and steps <= len(text)
    assert model.cache().length(seq) == len(prompt) + len(text)


def test_fork_copies_on_write(tmp_path):
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, heads=8, kv_heads=2, hidden=128, intermediate=256)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=64, block_tokens=4)
    prompt = [int(t) for t in np.random.default_rng(5).integers(0, spec.vocab, 10)]
    plain = Greedy(model, prompt)
    a = model.new_sequence()
    first = choice(model.prefill(a, prompt))[0]
    cache = model.cache()
    f = cache.fork(a)
    right = plain.choices(3)
    shared = cache.blocks(a)[-1]
    paths, _ = model.verify_trees([f], [[-1, 0, 1][:len(right)]], [right], [first])
    assert paths[0] == list(range(len(right))) and right
    assert cache.blocks(a)[-1] == shared and shared not in cache.blocks(f)
    assert cache.length(a) == len(prompt)
    other = Greedy(model, prompt)
    other.take([7])
    assert close(model.logits(a, 7), other.logits)
    plain.take(right + [9])
    assert close(model.logits(f, 9), plain.logits)


def test_fork_and_its_origin_in_one_call(tmp_path):
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, heads=8, kv_heads=2, hidden=128, intermediate=256)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=64, block_tokens=4)
    prompt = [int(t) for t in np.random.default_rng(6).integers(0, spec.vocab, 9)]
    plain = Greedy(model, prompt)
    a = model.new_sequence()
    first = choice(model.prefill(a, prompt))[0]
    cache = model.cache()
    f = cache.fork(a)
    right = plain.choices(4)
    assert len(right) > 2
    chain = list(range(-1, len(right) - 1))
    paths, after = model.verify_trees([a, f], [chain[:2], chain], [right[:2], right], [first, first])
    assert paths == [[0, 1], list(range(len(right)))] and after[0] == right[2]
    other = Greedy(model, prompt)
    other.take(right[:2] + [5])
    plain.take(right + [7])
    got = model.decode_sequences([a, f], [5, 7])
    assert close(got[0], other.logits) and close(got[1], plain.logits)
    cache.audit()


@pytest.mark.parametrize("nodes,vocab", [(1024, 300), (70, 34001)])
def test_large_trees(tmp_path, nodes, vocab):
    """The most nodes of a tree; logits that are computed in bands."""
    say("verify large trees", nodes, vocab)
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, embed_type=gf.T_Q8_0, output=False, hidden=256, intermediate=512, heads=4,
                        kv_heads=2, vocab=vocab, context=256)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=64, block_tokens=16)
    rng = np.random.default_rng(nodes)
    prompt = [int(t) for t in rng.integers(0, vocab, 40)]
    g = Greedy(model, prompt)
    seq = model.new_sequence()
    first = choice(model.prefill(seq, prompt))[0]
    ahead = g.choices(9)
    right = ahead[:-1]
    parents, tokens, want = drafted(rng, right, nodes - len(right), vocab)
    (path,), (after,) = model.verify_trees([seq], [parents], [tokens], [first])
    assert path == want and after == ahead[-1] and len(want) > 3
    g.take(right + [1])
    assert close(model.logits(seq, 1), g.logits)


def message(fn, *args):
    with pytest.raises((RuntimeError, ValueError)) as e:
        fn(*args)
    return str(e.value)


@pytest.mark.parametrize("hidden", [64, 40])
def test_refusals_change_nothing(tmp_path, hidden):
    spec = gf.LlamaSpec(hidden=hidden, intermediate=128, heads=4, kv_heads=2, context=24)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=6, block_tokens=4)
    a, b = model.new_sequence(), model.new_sequence()
    rng = np.random.default_rng(1)
    pa, pb = ([int(t) for t in rng.integers(0, spec.vocab, n)] for n in (8, 11))
    fa, fb = choice(model.prefill(a, pa))[0], choice(model.prefill(b, pb))[0]
    cache = model.cache()
    chain = [-1, 0, 1, 2, 3]
    verify = model.verify_trees
    assert verify([], [], [], []) == ([], [])
    assert verify([a, b], [[], []], [[], []], [fa, fb]) == ([[], []], [fa, fb])
    assert message(verify, [a, a], [[-1], [-1]], [[1], [1]], [fa, fa]) == "duplicate sequence in decode batch"
    assert message(verify, [a, 99], [[-1], [-1]], [[1], [1]], [fa, fa])
    for bad in ([0], [-1, 1], [-1, 2, 0], [-2]):
        assert message(verify, [a], [bad], [[1] * len(bad)], [fa]) == "invalid token tree", bad
    assert message(verify, [a], [[-1]], [[spec.vocab]], [fa]) == "Invalid token ID"
    assert message(verify, [a], [[-1]], [[1]], [-1]) == "Invalid token ID"
    assert message(verify, [a], [[-1]], [[1, 2]], [fa]) == "one parent per drafted token"
    assert message(verify, [a], [], [], [fa]) == "one tree and one first token per sequence"
    assert message(verify, [a], [[-1] * 1025], [[1] * 1025], [fa]) == "a token tree has at most 1,024 nodes"
    deep = list(range(-1, 16))  # 8 cached + 17 > 24
    assert message(verify, [a], [deep], [[1] * 17], [fa]) == "token tree exceeds the context"
    # the pool: five of six blocks are taken.  Right drafts of both sequences need two
    # more: b's last block has one slot left, a's none
    plain = {}
    for s, p in ((a, pa), (b, pb)):
        start, out = cache.length(s), []
        token = fa if s == a else fb
        for _ in range(2):
            out.append(token)
            token, sure = choice(model.logits(s, token))
            assert sure
        model.truncate(s, start)
        plain[s] = out
    assert message(verify, [a, b], [chain[:2], chain[:2]], [plain[a], plain[b]], [fa, fb])
    assert (cache.length(a), cache.length(b)) == (8, 11)
    paths, _ = verify([a], [chain[:2]], [plain[a]], [fa])
    assert paths == [[0, 1]] and (cache.length(a), cache.length(b)) == (10, 11)
    model.close()
    assert message(verify, [a], [[-1]], [[1]], [fa]) == "Model is closed"


def test_one_deep_tree_among_many_sequences(tmp_path):
    """Sequences times the deepest tree beyond any launch: what is written goes by the
    accepted nodes."""
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, hidden=256, intermediate=512, heads=4, kv_heads=2, vocab=300, context=1100)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=64, block_tokens=16)
    n, prompt = 16400, [int(t) for t in np.random.default_rng(7).integers(0, spec.vocab, 20)]
    seqs = [model.new_sequence() for _ in range(n)]
    plain = Greedy(model, prompt)
    first = [0] * n
    for i in (0, n - 1):
        first[i] = choice(model.prefill(seqs[i], prompt))[0]
    right = plain.choices(6)
    assert len(right) == 6
    wrong = [(right[5] + 1) % spec.vocab] * (1024 - 5)
    parents, tokens = [[] for _ in range(n)], [[] for _ in range(n)]
    parents[0], tokens[0] = [-1, 0], right[:2]
    parents[-1], tokens[-1] = list(range(-1, 1023)), right[:5] + wrong
    paths, after = model.verify_trees(seqs, parents, tokens, first)
    assert paths[0] == [0, 1] and after[0] == right[2]
    assert paths[-1] == list(range(5)) and after[-1] == right[5]
    assert not any(paths[1:-1]) and after[1:-1] == [0] * (n - 2)
    cache = model.cache()
    assert [cache.length(s) for s in (seqs[0], seqs[1], seqs[-1])] == [22, 0, 25]
    plain.take(right[:5] + [9])
    assert close(model.logits(seqs[-1], 9), plain.logits)
    cache.audit()


def test_no_node_accepted(tmp_path):
    spec = gf.LlamaSpec(matrix_type=gf.T_Q8_0, heads=8, kv_heads=2, hidden=128, intermediate=256)
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=8, block_tokens=4)
    prompt = [int(t) for t in np.random.default_rng(5).integers(0, spec.vocab, 10)]
    a = model.new_sequence()
    first = choice(model.prefill(a, prompt))[0]
    wrong = (first + 1) % spec.vocab
    assert model.verify_trees([a], [[-1, 0, -1]], [[wrong] * 3], [first]) == ([[]], [first])
    assert model.cache().length(a) == 10
