"""The speculative loop (speech_to_text_amd/speculative.py) on the CPU: engine and draft are served by a small
table of random logits keyed by the token history, so that what is checked is the loop's own logic - tree
layout, acceptance, the two histories, windows that end at different times - against plain greedy search on
the same table.  Same numbers on both sides, so ids are equal and scores agree to float32 rounding."""
import numpy as np
import pytest
import torch

from speech_to_text_amd import speculative

V, EOS, PAD = 23, 20, 21


class TableEngine(object):
    """The surface of WhisperEngine that speculative.generate uses.  Logits after a history are random
    numbers seeded by it; with probability `error` they are seeded differently (a draft that errs)."""

    def __init__(self, n, max_text_len=64, max_prompt_len=16, error=0.0, eos_bias=0.0):
        self.dims, self.device = {"n_vocab": V}, torch.device("cpu")
        self.max_batch, self.max_beams, self.max_prompt_len, self.max_text_len = n, 1, max_prompt_len, max_text_len
        self._batch, self.error, self.eos_bias = n, error, eos_bias
        self.history, self.nodes, self.passes = None, None, 0

    def logits(self, window, history):
        key = hash((window,) + tuple(int(t) for t in history)) & 0xFFFFFFFF
        rng = np.random.default_rng(key)
        if rng.random() < self.error:
            rng = np.random.default_rng(key ^ 0x55555555)
        z = rng.standard_normal(V).astype(np.float32) * 2
        z[EOS] += self.eos_bias
        return z

    def decode_tree(self, tokens, parents=None, reset=False):
        tokens = np.asarray(tokens)
        n, m = tokens.shape
        assert n == self._batch and n * m <= self.max_batch * self.max_beams * self.max_prompt_len and m <= 64
        if reset:
            self.history = [[] for _ in range(n)]
        out, self.nodes = np.zeros((n, m, V), np.float32), []
        for i in range(n):
            assert len(self.history[i]) + m <= self.max_text_len
            paths = []
            for a in range(m):
                p = a - 1 if parents is None else int(np.asarray(parents)[i, a])
                paths.append((paths[p] if 0 <= p < a else []) + [int(tokens[i, a])])
                out[i, a] = self.logits(i, self.history[i] + paths[a])
            self.nodes.append(paths)
        self.passes += 1
        return torch.from_numpy(out)

    def commit_tree(self, paths):
        for i, p in enumerate(paths):
            assert list(p) == sorted(set(p))
            for j, a in enumerate(p):                    # a path: every node's own path is the prefix up to it
                assert len(self.nodes[i][a]) == j + 1
            self.history[i] = self.history[i] + (self.nodes[i][p[-1]] if p else [])
        self.nodes = None

    def truncate_tree(self, lengths):
        for i, k in enumerate(lengths):
            assert 0 <= k <= len(self.history[i])
            self.history[i] = self.history[i][:int(k)]

    def tree_lengths(self):
        return np.asarray([len(h) for h in self.history], np.int32)


def greedy(engine, prompt, steps, banned=()):
    """Plain greedy search on the table: tokens [n, steps], lengths, scores."""
    n = len(prompt)
    tokens, lens, scores = np.full((n, steps), PAD, np.int32), np.zeros(n, np.int32), np.zeros(n)
    for i in range(n):
        hist = list(prompt[i])
        for t in range(steps):
            z = torch.from_numpy(engine.logits(i, hist))
            z[list(banned)] = float("-inf")
            k = int(z.argmax())
            scores[i] += float(torch.log_softmax(z, 0)[k])
            tokens[i, t] = k
            hist.append(k)
            if k == EOS:
                break
            lens[i] += 1
    return tokens, lens, scores


@pytest.mark.parametrize("n,prompt_len,steps,depth,width,error,eos_bias", [
    (1, 3, 20, 4, 1, 0.0, -5), (1, 3, 20, 4, 1, 0.3, -5), (3, 4, 25, 3, 2, 0.4, 0), (4, 1, 30, 5, 3, 0.5, 1), (2, 7, 40, 1, 1, 0.2, 0),
    (5, 2, 12, 2, 4, 1.0, 0), (2, 30, 20, 4, 2, 0.3, -5), (3, 3, 1, 4, 1, 0.3, 0), (3, 3, 2, 4, 2, 0.3, 0), (1, 24, 40, 15, 1, 0.1, -5)])
def test_ids_are_those_of_greedy_search(n, prompt_len, steps, depth, width, error, eos_bias):
    for seed in range(4):
        prompt = np.random.default_rng(seed).integers(0, 20, (n, prompt_len)).astype(np.int32)
        engine, draft = TableEngine(n, eos_bias=eos_bias), TableEngine(n, error=error, eos_bias=eos_bias)
        want = greedy(engine, prompt, steps)
        extras = {}
        got = speculative.generate(engine, draft, prompt, max_new_tokens=steps, eos_token=EOS, pad_token=PAD, draft_tokens=depth,
                                   draft_width=width, extras=extras)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert np.abs(got[2] - want[2]).max() < 1e-4
        if error == 0.0 and steps > 2 * depth:               # a draft that is always right: depth + 1 tokens a pass
            assert extras["speculation"]["passes"] <= -(-steps // (depth + 1)) + 1
        assert extras["speculation"]["tokens"] == sum(min(steps, int(k) + 1) for k in got[1]) - n


def test_suppressed_ids_and_exactly_full_capacity():
    prompt = np.array([[1, 2, 3, 4]] * 2, np.int32)
    engine, draft = TableEngine(2, max_text_len=24, eos_bias=-9), TableEngine(2, max_text_len=24, error=0.5, eos_bias=-9)
    banned = [0, 5, 6, 7, 8]
    got = speculative.generate(engine, draft, prompt, max_new_tokens=20, eos_token=EOS, pad_token=PAD, draft_tokens=3, draft_width=4,
                               suppress=banned)
    assert np.array_equal(got[0], greedy(engine, prompt, 20, banned)[0])
    assert not np.isin(got[0], banned).any()


def test_tree_layout_and_walk():
    assert speculative.tree_layout(3, 2).tolist() == [-1, 0, 0, 1, 1, 3, 3]
    assert speculative.tree_layout(0, 2).tolist() == [-1]
    tokens = [9, 4, 5, 6, 7, 2, 3]
    # 4 (trunk), 6 (trunk), then 3: a leaf
    assert speculative.walk([4, 6, 0, 3, 0, 0, 0], tokens, 3, 2) == [0, 1, 3, 6]
    # 5 is a leaf: nothing follows it
    assert speculative.walk([5, 6, 6, 3, 0, 0, 0], tokens, 3, 2) == [0, 2]
    assert speculative.walk([1, 6, 6, 3, 0, 0, 0], tokens, 3, 2) == [0]


@pytest.mark.parametrize("change", [dict(draft_tokens=0), dict(draft_width=0), dict(draft_tokens=32, draft_width=2), dict(max_new_tokens=0),
                                    dict(max_new_tokens=62), dict(same=True), dict(vocab=True), dict(batch=True), dict(rows=True)])
def test_refusals(change):
    engine, draft = TableEngine(2), TableEngine(2)
    kw = dict(max_new_tokens=5, eos_token=EOS, pad_token=PAD)
    if change.pop("same", False):
        draft = engine
    if change.pop("vocab", False):
        draft.dims = {"n_vocab": V + 1}
    if change.pop("batch", False):
        draft._batch = 3
    if change.pop("rows", False):
        engine.max_prompt_len = 1
    with pytest.raises(ValueError):
        speculative.generate(engine, draft, np.zeros((2, 3), np.int32), **dict(kw, **change))
