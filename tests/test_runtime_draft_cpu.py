"""MI355XRuntime calls with `draft = `: what reaches the engines and what is refused (no GPU: the engines are records of
their calls)."""
import numpy as np
import pytest
import torch

from speech_to_text_amd.eager import EngineState
from speech_to_text_amd.runtimes import mi355x_runtime as M


class Device(object):
    """A device engine that notes what happens to it."""

    _epoch, max_text_len, dims = 0, 64, {'n_vocab': 7, 'n_text_layer': 1}

    def __init__(self, calls, name):
        self.calls, self.name = calls, name

    def step_state(self):
        return 2, 1, 5

    def encode(self, mel):
        self.calls.append((self.name, 'encode', mel.shape[0]))

    def generate(self, tokens, **kwargs):
        self.calls.append((self.name, 'generate', kwargs))
        n = len(tokens)
        return np.zeros((n, 3), np.int32), np.full(n, 3, np.int32), np.zeros(n, np.float32)


class Engine(M._Engine):
    def __init__(self, calls, name):
        super().__init__({'n_vocab': 7, 'n_text_ctx': 64}, {})
        self.device = Device(calls, name)

    def get(self, batch, beams, text_len, prompt_len, replica=0):
        return self.device


@pytest.fixture
def pair():
    calls = []
    made = []
    for name in ('full', 'draft'):
        r = M.MI355XRuntime('p', engine=Engine(calls, name))
        r.set_tokens(sos_token=1, eos_token=2, pad_token=2)
        made.append(r)
    return made[0], made[1], calls


MEL, PROMPT = torch.zeros(2, 30, 80), np.array([[1, 3], [1, 3]], np.int32)


def test_an_earlier_state_and_a_draft_are_refused_together(pair):
    full, draft, calls = pair
    state = EngineState(full.engine.device)
    full(None, tokens=PROMPT, max_new_tokens=3, initial_state=state)
    assert [c[:2] for c in calls] == [('full', 'generate')]
    with pytest.raises(ValueError):
        full(None, tokens=PROMPT, max_new_tokens=3, draft=draft, initial_state=state)
    assert len(calls) == 1


def test_on_encoded_is_called_once_both_encoder_passes_are_enqueued(pair, monkeypatch):
    """infer_windows(replicas = 2) starts its second engine on it."""
    full, draft, calls = pair

    class Event(object):
        def record(self):
            calls.append(('event', 'record'))
    monkeypatch.setattr(torch.cuda, 'Event', Event)
    full(MEL, tokens=PROMPT, max_new_tokens=3, draft=draft, on_encoded=lambda ev: calls.append(('caller', type(ev))))
    assert [c[:2] for c in calls] == [('full', 'encode'), ('draft', 'encode'), ('event', 'record'), ('caller', Event),
                                      ('full', 'generate')]
