"""stt_decode_tree and what is built on it (commit, truncate, speculative greedy search), and engines whose
weight matrices are held in 4 bits, against oracle/model.py."""
import numpy as np
import pytest
import torch

from oracle import model as om
from tests import _operators as O
from tests import _parity as P

pytestmark = pytest.mark.gpu

EOS = PAD = 999
DIMS = om.Dims(n_mels=80, n_audio_ctx=1500, n_audio_state=128, n_audio_head=2, n_audio_layer=2, n_vocab=1000, n_text_ctx=64,
               n_text_state=128, n_text_head=2, n_text_layer=2)


@pytest.fixture(scope="module")
def small():
    from speech_to_text_amd.engine import WhisperEngine
    w = P.bf16_round(om.random_weights(DIMS, seed=0, style="peaked"))
    engine = WhisperEngine(P.dims_dict(DIMS), w, max_batch=3, max_beams=1, max_text_len=60, max_prompt_len=20)
    oracle = om.Whisper(DIMS, w)
    mel = torch.rand(3, 3000, 80, generator=torch.Generator().manual_seed(1)) * 2 - 1
    with torch.no_grad():
        enc = oracle.encoder(mel)
    return w, engine, oracle, mel, enc


def _oracle_last(oracle, enc, window, tokens):
    """float32 logits after `tokens` of one window."""
    with torch.no_grad():
        cross = [(k[window: window + 1], v[window: window + 1]) for k, v in oracle.cross_kv(enc)]
        return oracle.decoder(torch.tensor([tokens]).long(), cross)[0][0, -1].numpy()


def test_every_node_sees_its_own_path(small):
    """Prompt, then trees of which paths of different lengths join the histories, a truncation and more trees: the
    logits after each node are the oracle's for the sequence history + path (the bf16 tolerance of _parity)."""
    w, engine, oracle, mel, enc = small
    engine.encode(mel)
    rng = np.random.default_rng(3)
    history = [[int(t) for t in rng.integers(0, 998, 5)] for _ in range(3)]
    z = engine.decode_tree(np.asarray(history, np.int32), reset=True).cpu().numpy()
    want = np.stack([[_oracle_last(oracle, enc, i, history[i][: j + 1]) for j in range(5)] for i in range(3)])
    assert P.rel_l2(z, want) < 2e-2
    engine.commit_tree([[0, 1, 2, 3, 4]] * 3)
    for step in range(4):
        m = [9, 1, 20, 6][step]
        tokens = rng.integers(0, 998, (3, m)).astype(np.int32)
        parents = np.stack([[-1] + [int(rng.integers(-1, a)) for a in range(1, m)] for _ in range(3)]).astype(np.int32)
        z = engine.decode_tree(tokens, parents).cpu().numpy()
        paths = []
        for i in range(3):
            nodes = []
            for a in range(m):
                nodes.append((nodes[parents[i, a]] if parents[i, a] >= 0 else []) + [a])
            want = np.stack([_oracle_last(oracle, enc, i, history[i] + [int(tokens[i, b]) for b in nodes[a]]) for a in range(m)])
            assert P.rel_l2(z[i], want) < 2e-2, (step, i)
            best = max(nodes, key=len)
            paths.append(best[: len(best) - i] if i < len(best) else [])
            history[i] = history[i] + [int(tokens[i, b]) for b in paths[i]]
        engine.commit_tree(paths)
        assert engine.tree_lengths().tolist() == [len(h) for h in history]
        if step == 1:
            keep = [len(h) - (2 * i) for i, h in enumerate(history)]
            engine.truncate_tree(keep)
            history = [h[:k] for h, k in zip(history, keep)]
    # an uncommitted pass leaves no trace, and a second one gives the same bits
    a = engine.decode_tree(tokens, parents)
    assert torch.equal(a, engine.decode_tree(tokens, parents))


def test_tree_steps_and_plain_steps_agree(small):
    """A chain of single-token trees is the plain cached step: same cache contents up to rounding of another
    kernel, so the logits agree to the bf16 tolerance; and each kind of history ends the other."""
    from speech_to_text_amd._lib import SttError
    w, engine, oracle, mel, enc = small
    engine.encode(mel)
    toks = np.random.default_rng(5).integers(0, 998, (3, 8)).astype(np.int32)
    plain = [engine.decode_step(toks[:, :4], reset=True)] + [engine.decode_step(toks[:, j: j + 1]) for j in range(4, 8)]
    tree = [engine.decode_tree(toks[:, :4], reset=True)[:, -1]]
    engine.commit_tree([[0, 1, 2, 3]] * 3)
    for j in range(4, 8):
        tree.append(engine.decode_tree(toks[:, j: j + 1])[:, 0])
        engine.commit_tree([[0]] * 3)
    for a, b in zip(plain, tree):
        assert P.rel_l2(a.cpu(), b.cpu()) < 2e-2
    with pytest.raises(SttError):
        engine.decode_step(toks[:, :1])                          # the plain history is gone
    engine.decode_step(toks[:, :1], reset=True)
    with pytest.raises(SttError):
        engine.decode_tree(toks[:, :1])                          # and now the tree history
    engine.decode_tree(toks[:, :1], reset=True)
    engine.encode(mel)
    with pytest.raises(SttError):
        engine.decode_tree(toks[:, :1])


def test_argument_checks(small):
    from speech_to_text_amd._lib import SttError
    w, engine, oracle, mel, enc = small
    engine.encode(mel)
    t = np.zeros((3, 4), np.int32)
    with pytest.raises(SttError):
        engine.decode_tree(t)                                    # no history
    with pytest.raises(ValueError):
        engine.commit_tree([[0]] * 3)
    with pytest.raises(SttError):
        engine.decode_tree(t[:2], reset=True)                    # two sequences for three windows
    with pytest.raises(SttError):
        engine.decode_tree(np.zeros((3, 21), np.int32), reset=True)      # more rows than reserved
    with pytest.raises(ValueError):
        engine.decode_tree(t, parents=t[:, :2])
    engine.decode_tree(t, reset=True)
    for paths in ([[0, 0]] * 3, [[1, 0]] * 3, [[4]] * 3, [[-1]] * 3):
        with pytest.raises(SttError):
            engine.commit_tree(paths)
    for paths in ([[0]] * 2, [[0, 1, 2, 3, 3]] * 3):
        with pytest.raises(ValueError):
            engine.commit_tree(paths)
    engine.commit_tree([[0, 1, 2, 3], [], [0]])
    with pytest.raises(SttError):
        engine.commit_tree([[0]] * 3)                            # already committed
    with pytest.raises(SttError):
        engine.truncate_tree([5, 0, 1])
    with pytest.raises(ValueError):
        engine.truncate_tree([1, 0])
    engine.truncate_tree([4, 0, 0])
    for _ in range(2):
        engine.decode_tree(np.zeros((3, 20), np.int32))
        engine.commit_tree([list(range(20))] * 3)
    with pytest.raises(SttError):
        engine.decode_tree(np.zeros((3, 17), np.int32))          # 44 + 17 > 60 positions
    engine.decode_tree(np.zeros((3, 16), np.int32))


def test_tree_passes_are_not_recorded_into_graphs(small):
    """Their lengths are host values: recording one is refused and leaves the history as it was."""
    from speech_to_text_amd import _lib
    w, engine, oracle, mel, enc = small
    engine.encode(mel)
    tokens = torch.tensor([[5, 6, 7]] * 3, dtype=torch.int32, device=engine.device)
    want = engine.decode_tree(tokens, reset=True).clone()
    engine.commit_tree([[0, 1, 2]] * 3)
    after = engine.decode_tree(tokens).clone()
    torch.cuda.synchronize()
    for call in (lambda: engine.decode_tree(tokens), lambda: engine.truncate_tree([0, 0, 0]), lambda: engine.commit_tree([[0]] * 3)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(_lib.SttError, match="graph"):
                call()
    assert engine.tree_lengths().tolist() == [3, 3, 3]
    assert torch.equal(engine.decode_tree(tokens), after)
    assert torch.equal(engine.decode_tree(tokens, reset=True), want)


def _four_bit(w, names):
    """The weights with the named matrices replaced by what their 4-bit form stands for."""
    out = dict(w)
    for k in w:
        if names(k):
            out[k] = torch.from_numpy(O.values_of(*O.quantize_reference(w[k].double().numpy()))).float()
    return out


def _decoder_matrix(k):
    return k.startswith("decoder.blocks.") and k.endswith(".weight") and "_ln" not in k and \
        not k.endswith(("cross_attn.key.weight", "cross_attn.value.weight"))


@pytest.mark.parametrize("erf", [False, True])
def test_four_bit_decoder_is_the_oracle_on_the_values_it_stands_for(small, erf):
    from speech_to_text_amd.engine import WhisperEngine
    w, _, _, mel, enc = small
    engine = WhisperEngine(P.dims_dict(DIMS), w, max_batch=3, max_text_len=60, max_prompt_len=59, gelu_tanh=not erf, decoder_format="mxfp4")
    oracle = om.Whisper(DIMS, _four_bit(w, _decoder_matrix), "none" if erf else "tanh")
    with torch.no_grad():
        enc = oracle.encoder(mel)
    got_enc = engine.encode(mel, return_output=True).cpu().numpy()
    assert P.rel_l2(got_enc, enc.numpy()) < 1e-2                   # the encoder is the bf16 one
    rng = np.random.default_rng(7)
    for length in (1, 3, 40):                                     # 3, 9 and 120 rows
        toks = rng.integers(0, 998, (3, length)).astype(np.int32)
        with torch.no_grad():
            want, _ = oracle.decoder(torch.from_numpy(toks).long(), oracle.cross_kv(enc))
        assert P.rel_l2(engine.decoder_logits(toks).cpu(), want.numpy()) < 2e-2, length
    engine.encode(mel[:1])                                        # one row per step (the fused LayerNorm path of bf16 engines)
    a = engine.decode_step(np.array([[5, 6, 7]], np.int32), reset=True)
    b = engine.decode_step(np.array([[8]], np.int32))
    with torch.no_grad():
        want, _ = oracle.decoder(torch.tensor([[5, 6, 7, 8]]), oracle.cross_kv(enc[:1]))
    assert P.rel_l2(torch.stack([a[0], b[0]]).cpu(), want[0, 2:].numpy()) < 2e-2
    prompt = np.array([[1, 2, 3]] * 3, np.int32)
    engine.encode(mel)
    tokens, lengths, scores = engine.generate(prompt, max_new_tokens=16, eos_token=EOS, pad_token=PAD, early_stopping=False)
    with torch.no_grad():
        exact, total = P.check_greedy_steps(oracle, enc, prompt, tokens, EOS, PAD, scores=scores)
    assert total == 48 and exact >= 43


class _FourBitMlp(om.Whisper):
    """The oracle with the encoder MLP's activations in 4 bits where the engine has them."""

    def _mlp_block(self, x, p):
        if not p.startswith("encoder."):
            return super()._mlp_block(x, p)
        def four(t):
            flat = t.to(torch.bfloat16).double().reshape(-1, t.shape[-1]).numpy()
            return torch.from_numpy(O.values_of(*O.quantize_reference(flat))).float().reshape(t.shape)
        h = four(om.layer_norm(x, self.w, p + "mlp_ln"))
        return x + om.linear(four(om.gelu(om.linear(h, self.w, p + "mlp.0"), self.act)), self.w, p + "mlp.2")


def test_four_bit_encoder_mlp(small):
    """Against the oracle with the same weights and with activations quantised at the same two places.  Rounding
    amplifies differences: an activation that differs by e (relative to the rms) lands on another code with
    probability 0.8 e / s, s = 0.4 being the mean spacing of the codes relative to the rms, and then moves by
    s, so the quantised values differ by sqrt(0.8 e s) = sqrt(0.32 e).  With the encoder's stated bf16
    tolerance e = 1e-2 that is 5.7 % at the first place; at the second e = 5.7e-2 gives 13.5 %, together
    14.6 % of the MLP's output.  It joins a residual stream at least as large (/ sqrt 2) and there are two
    layers (* sqrt 2): 0.146.  What the 4 bits cost against the plain oracle is larger than what is left
    of that in the mean: s / sqrt 12 = 11.5 % for each of two activations and two matrices, 23 %."""
    from speech_to_text_amd.engine import WhisperEngine
    w, _, plain, mel, enc = small
    engine = WhisperEngine(P.dims_dict(DIMS), w, max_batch=2, max_text_len=60, max_prompt_len=20, encoder_mlp_format="mxfp4")
    oracle = _FourBitMlp(DIMS, _four_bit(w, lambda k: k.startswith("encoder.blocks.") and k.endswith(("mlp.0.weight", "mlp.2.weight"))))
    with torch.no_grad():
        want = oracle.encoder(mel[:2]).numpy()
    first = None
    for _ in range(2):
        got = engine.encode(mel[:2], return_output=True).cpu().numpy()
        assert P.rel_l2(got, want) < 0.146
        assert P.rel_l2(got, want) < 0.7 * P.rel_l2(got, enc[:2].numpy())    # it is the 4-bit network, not the other one
        assert first is None or np.array_equal(first, got)
        first = got
    one = engine.encode(mel[1:2], return_output=True).cpu().numpy()
    assert P.rel_l2(one, want[1:2]) < 0.146


@pytest.mark.parametrize("width,tokens_ahead", [(1, 4), (3, 3), (2, 9)])
@pytest.mark.parametrize("kind", ["mxfp4", "other"])
def test_speculative_greedy_follows_the_full_engine(small, kind, width, tokens_ahead):
    """Ids and scores are those of the full model's greedy search, step by step (near-ties as in _parity), with a 4-bit
    copy of the model and with an unrelated model as the draft; the copy saves passes."""
    from speech_to_text_amd.engine import WhisperEngine
    w, engine, oracle, mel, enc = small
    if kind == "mxfp4":
        draft = WhisperEngine(P.dims_dict(DIMS), w, max_batch=3, max_text_len=60, max_prompt_len=20, decoder_format="mxfp4",
                              encoder_mlp_format="mxfp4")
    else:
        draft = WhisperEngine(P.dims_dict(DIMS), P.bf16_round(om.random_weights(DIMS, seed=9, style="peaked")), max_batch=3,
                              max_text_len=60, max_prompt_len=4)
    engine.encode(mel)
    draft.encode(mel)
    prompt = np.array([[1, 2, 3], [4, 5, 6], [7, 8, 9]], np.int32)
    extras = {}
    tokens, lengths, scores = engine.generate(prompt, max_new_tokens=40, eos_token=EOS, pad_token=PAD, draft=draft,
                                              draft_tokens=tokens_ahead, draft_width=width, extras=extras)
    with torch.no_grad():
        exact, total = P.check_greedy_steps(oracle, enc, prompt, tokens, EOS, PAD, scores=scores)
    assert exact >= 0.9 * total
    spec = extras["speculation"]
    assert spec["passes"] <= 40 and spec["tokens"] == total - 3
    if kind == "mxfp4" and total == 120:
        assert spec["passes"] < 39                                 # some drafts were accepted in every window
    with pytest.raises(ValueError):
        engine.generate(prompt, max_new_tokens=4, eos_token=EOS, pad_token=PAD, draft=draft, method="beam", num_beams=2)
    with pytest.raises(ValueError):
        engine.generate(prompt, max_new_tokens=4, eos_token=EOS, pad_token=PAD, draft=draft, return_logits=True)


def test_runtime_with_a_draft():
    """Two runtimes over the same seeded weights, one in 4 bits: the call with `draft` returns what the plain one does,
    up to near-ties (the scores of both are compared where the ids differ)."""
    from speech_to_text_amd.runtimes import build_runtime
    full = build_runtime("mi355x", "random:tiny:3:peaked")
    draft = build_runtime("mi355x", "random:tiny:3:peaked", decoder_format="mxfp4", encoder_mlp_format="mxfp4")
    assert draft.engine is not full.engine and draft.engine.formats["decoder_format"] == "mxfp4"
    assert build_runtime("mi355x", "random:tiny:3:peaked", decoder_format="mxfp4", encoder_mlp_format="mxfp4").engine is draft.engine
    for r in (full, draft):
        r.set_tokens(sos_token=50258, eos_token=50257, pad_token=50257)
    mel = torch.rand(2, 3000, 80, generator=torch.Generator().manual_seed(4)) * 2 - 1
    prompt = np.array([[50258, 50259, 50359]] * 2, np.int32)
    plain = full(mel, tokens=prompt, max_new_tokens=24)
    spec = full(mel, tokens=prompt, max_new_tokens=24, draft=draft, draft_tokens=5, draft_width=2)
    assert spec.tokens.shape == plain.tokens.shape
    # a near-tie may part the two; up to there they are the same
    for a, b in zip(plain.tokens, spec.tokens):
        diff = np.flatnonzero(a != b)
        assert diff.size == 0 or diff[0] >= 4
    same = [np.array_equal(a, b) for a, b in zip(plain.tokens, spec.tokens)]
    for s, x, y in zip(same, plain.scores, spec.scores):
        assert not s or abs(x - y) < 0.2
    with pytest.raises(ValueError):
        full(mel, tokens=prompt, draft=full)
    with pytest.raises(ValueError):
        build_runtime("mi355x", "random:tiny:3:peaked", decoder_format="int8")
