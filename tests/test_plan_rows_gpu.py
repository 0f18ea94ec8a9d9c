"""Plans in which few requests bring most of the new rows (prompts beside token steps), against the request-by-request form."""
import numpy as np
import pytest

from tests import _operators as O
from tests.test_paged_gpu import _run_plan

pytestmark = pytest.mark.gpu


def _state(cached, new, held, block, spare, seed):
    rng = np.random.default_rng(seed)
    cached, new, held = (np.asarray(v) for v in (cached, new, held))
    need = -(-(cached + new) // block)
    n_ring = int(held.sum() + np.maximum(need - held, 0).sum() + spare)
    ids, at = rng.permutation(n_ring), 0
    table = np.full((len(cached), int(max(held.max(), need.max())) + 1), -1)
    for i, h in enumerate(held):
        table[i, :h] = ids[at: at + h]
        at += h
    free, head = np.full(n_ring, -1), int(rng.integers(0, 3 * n_ring))
    free[(head + np.arange(n_ring - at)) % n_ring] = ids[at:]
    return dict(cached=cached, new=new, held=held, table=table, free=free, ring=np.array([head, head + n_ring - at]))


@pytest.mark.parametrize("block", [1, 16, 64])
@pytest.mark.parametrize("new", [[20000], [16384, 0, 1], [1, 1, 7001, 1], [0, 5000, 4999, 0, 0, 1] + [1] * 300, [40000] + [1] * 2000])
def test_one_request_with_thousands_of_new_rows(new, block):
    cached = [(37 * i) % 300 for i in range(len(new))]
    held = [-(-c // block) + (1 if i % 4 == 3 else 0) for i, c in enumerate(cached)]
    s = _state(cached, new, held, block, spare=3, seed=len(new) + block)
    rows = sum(new) + 70
    want = O.plan_reference(s["cached"], s["new"], s["table"], s["held"], s["free"], s["ring"], block, rows)
    got, _, _ = _run_plan(s, block, rows)
    assert got["status"][0] == 0
    for name, v in want.items():
        assert np.array_equal(got[name], v), name
