"""Speculative calls through the runtime and the wrapper: every emitted token against the float32 oracle on the emitted
history, at the sizes the runtime reserves by itself."""
import numpy as np
import pytest
import torch

from oracle import model as om
from tests import _parity as P

pytestmark = pytest.mark.gpu

EOS = PAD = 50257
SOS = [50258, 50259, 50359]
NO_TIMESTAMPS = list(range(50364, 51865))


@pytest.fixture(scope="module")
def trio():
    """A runtime, its 4-bit draft, and the oracle of the runtime's weights as it holds them (bf16)."""
    from speech_to_text_amd.runtimes import build_runtime
    full = build_runtime("mi355x", "random:tiny:3:peaked")
    draft = build_runtime("mi355x", "random:tiny:3:peaked", decoder_format="mxfp4", encoder_mlp_format="mxfp4")
    for r in (full, draft):
        r.set_tokens(sos_token=SOS[0], eos_token=EOS, pad_token=PAD)
    oracle = om.Whisper(om.Dims.named("tiny"), P.bf16_round(full.engine.weights))
    return full, draft, oracle


@pytest.mark.parametrize("windows,ahead,width,steps", [(1, 4, 1, 60), (3, 5, 2, 40), (12, 3, 3, 30)])
def test_every_emitted_token_is_the_full_models(trio, windows, ahead, width, steps):
    """A wrong commit, truncation or position shows from the first token after it on: each choice has to be the
    oracle's after what was emitted so far, or lose to it by less than the near-tie allowance, and the sum of the
    log-probabilities has to be the oracle's."""
    full, draft, oracle = trio
    mel = torch.rand(windows, 3000, 80, generator=torch.Generator().manual_seed(windows)) * 2 - 1
    with torch.no_grad():
        enc = oracle.encoder(mel)
    prompt = np.array([SOS] * windows, np.int32)
    for _ in range(2):                              # the second call finds the engines as the first left them
        got = full(mel, tokens=prompt, max_new_tokens=steps, draft=draft, draft_tokens=ahead, draft_width=width)
        assert got.tokens.shape == (windows, steps)
        with torch.no_grad():
            exact, total = P.check_greedy_steps(oracle, enc, prompt, got.tokens, EOS, PAD, scores=got.scores)
        assert total >= windows * 2 and exact >= 0.9 * total


def test_two_replicas_with_a_draft_equal_one():
    """Six windows in batches of two, alternated over two pairs of engines: the tokens of a single pair."""
    from speech_to_text_amd.stt import Whisper
    model = Whisper(pretrained="tiny", path="random:tiny:3:peaked", max_batch=2)
    draft = Whisper(pretrained="tiny", path="random:tiny:3:peaked", max_batch=2, decoder_format="mxfp4")
    mel = torch.rand(17000, 80, generator=torch.Generator().manual_seed(8)).cuda() * 2 - 1
    options = dict(lang="en", batch_size=2, max_length=24, logits_filter=NO_TIMESTAMPS, draft=draft, draft_width=2)
    one = model.infer_windows(mel, **options)
    two = model.infer_windows(mel, replicas=2, **options)
    assert sorted(one) == sorted(two) == list(range(6))
    for w in one:
        assert len(one[w]["tokens"]) and np.array_equal(one[w]["tokens"], two[w]["tokens"])
