"""Outputs and caches that share memory with themselves are refused by paged.tree_attention (several blocks would write
one place); layouts that only reorder or pad are not."""
import pytest
import torch

from speech_to_text_amd import paged

BF = torch.bfloat16


def _call(cache=None, out=None):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = torch.zeros(6, 2, 16, 64, dtype=BF) if cache is None else cache
    return paged.tree_attention(torch.zeros(5, 4, 64, dtype=BF), torch.zeros(5, 2, 64, dtype=BF), torch.zeros(5, 2, 64, dtype=BF),
                                cache, cache, i(3, 2), i(3), i(4), torch.zeros(5, dtype=torch.int64), max_nodes=4, out=out)


@pytest.mark.parametrize("change", [
    dict(out=torch.zeros(5, 1, 64, dtype=BF).expand(5, 4, 64)), dict(out=torch.zeros(1, 4, 64, dtype=BF).expand(5, 4, 64)),
    dict(out=torch.zeros(4096, dtype=BF).as_strided((5, 4, 64), (256, 32, 1))),
    dict(cache=torch.zeros(6, 1, 16, 64, dtype=BF).expand(6, 2, 16, 64)), dict(cache=torch.zeros(1, 2, 16, 64, dtype=BF).expand(6, 2, 16, 64)),
    dict(cache=torch.zeros(8192, dtype=BF).as_strided((6, 2, 16, 64), (1024, 512, 64, 1)))])
def test_overlapping_outputs_and_caches_are_refused(change):
    with pytest.raises(ValueError, match="overlap"):
        _call(**change)


@pytest.mark.parametrize("change", [
    dict(), dict(out=torch.zeros(4, 5, 64, dtype=BF).transpose(0, 1)), dict(out=torch.zeros(5, 6, 72, dtype=BF)[:, 1:5, :64]),
    dict(cache=torch.zeros(6, 16, 2, 64, dtype=BF).transpose(1, 2)), dict(cache=torch.zeros(2, 6, 16, 64, dtype=BF).transpose(0, 1)),
    dict(cache=torch.zeros(9, 3, 20, 80, dtype=BF)[::2, :2, :16, :64][:5])])
def test_reordered_and_padded_layouts_are_not(change):
    with pytest.raises(ValueError, match="on a GPU"):              # everything in order but the device
        _call(**change)
