"""Row counts that the C entry point has no room for are refused by paged.plan before anything is allocated."""
import pytest
import torch

from speech_to_text_amd import paged


@pytest.mark.parametrize("rows", [-1, 2 ** 31, 2 ** 32 + 5])
def test_row_counts_that_do_not_fit_are_refused(rows):
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        paged.plan(ints(2), ints(2), ints(2, 3), ints(2), ints(8), torch.zeros(2, dtype=torch.int64), block_size=16, rows=rows)
