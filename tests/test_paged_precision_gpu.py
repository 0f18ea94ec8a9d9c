"""How exact paged.tree_attention is: float32 softmax weights reach the product with the values, and values of
visible positions that are not finite do what the formula says.

Bound per output element, with w the exact weights, v the values, A = sum w |v|, eps the step of the storage
type, u = 2^-24, c keys, head size d:
  * the result is rounded once: eps / 2 * |out|;
  * a weight meets v as the sum of two numbers of the storage type: the first is off by at most eps / 2 of the
    weight, the second holds that remainder (exact in float32) to eps / 2 of itself: (eps / 2)^2 * A;
  * float16 only, whose smallest step is 2^-24: weights are scaled so that the largest key's is at least 2^7, so
    half a step is at most 2^-25 / 2^7 = 2^-32 of the largest weight: 2^-32 * max w * sum |v|;
  * a score is a float32 sum of d products, times scale, times log2 e: |error| <= (d + 4) u S with S the largest
    scale * sum |q_i k_i|; it moves the weight and the normaliser by that much each, exp2 adds 2 u each:
    2 ((d + 4) S + 2) u * A;
  * numerator and denominator are float32 sums over c keys (the numerator of 2 c products) in some order, every
    partial sum rescaled by a rounded factor at most once per 32 keys: (3 c + c / 8 + 16) u * A.
"""
import math

import numpy as np
import pytest
import torch

from tests import _operators as O
from tests.test_paged_gpu import _call, _to_gpu, _tree_state

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _exact(s, scale=None):
    """(out, bound) in float64 of every (row, head).  A key whose score is -inf has no weight; a value that is
    not finite and has some makes the output that infinity, or NaN where both infinities or a NaN meet."""
    q, k, v, kc, vc = (s[x].double() for x in ("q", "k", "v", "k_cache", "v_cache"))
    table, cached, starts = s["table"], s["cached"].tolist(), s["starts"].tolist()
    (rows, heads, d), block = q.shape, kc.shape[2]
    group, eps = heads // k.shape[1], torch.finfo(s["q"].dtype).eps
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.full((rows, heads, d), float("nan"), dtype=torch.float64), torch.zeros(rows, heads, d, dtype=torch.float64)
    for i in range(len(cached)):
        lo, hi = starts[i], starts[i + 1]
        at = torch.arange(cached[i])
        blk, off = table[i][at // block].long(), at % block
        hk, hv = kc[blk, :, off], vc[blk, :, off]
        seen = O.tree_paths(None if s["parents"] is None else s["parents"][lo:hi], hi - lo)
        for a in range(hi - lo):
            mine = torch.from_numpy(np.nonzero(seen[a])[0])
            keys, vals = torch.cat([hk, k[lo:hi][mine]]), torch.cat([hv, v[lo:hi][mine]])
            for h in range(heads):
                kk, vv = keys[:, h // group], vals[:, h // group]
                z = (kk * q[lo + a, h]).sum(dim=1) * scale
                w = torch.softmax(z, dim=0)
                has = z > -math.inf
                bad = has[:, None] & ~torch.isfinite(vv)
                clean = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
                o, big = w @ clean, w @ clean.abs()
                if bad.any():
                    up, down = (bad & (vv == math.inf)).any(dim=0), (bad & (vv == -math.inf)).any(dim=0)
                    nan = (bad & torch.isnan(vv)).any(dim=0) | (up & down)
                    o = torch.where(up, torch.full_like(o, math.inf), torch.where(down, torch.full_like(o, -math.inf), o))
                    o = torch.where(nan, torch.full_like(o, math.nan), o)
                fine = torch.isfinite(z)
                top = float((kk[fine].abs() @ q[lo + a, h].abs()).max()) * abs(scale) if fine.any() else 0.0
                c = len(z)
                out[lo + a, h] = o
                bound[lo + a, h] = eps / 2 * o.abs() + ((eps / 2) ** 2 + (2 * ((d + 4) * top + 2) + 3 * c + c / 8 + 16) * O.U) * big
                if s["q"].dtype == HF:
                    bound[lo + a, h] += 2.0 ** -32 * float(w.max()) * clean.abs().sum(dim=0)
    return out, bound


def _check(s, scale=None, **kw):
    want, bound = _exact(s, scale)
    rows = int(s["starts"][-1])
    nodes = int((s["starts"][1:] - s["starts"][:-1]).max())
    got = _call(_to_gpu(s), nodes, scale=scale, **kw).double().cpu()[:rows]
    want, bound = want[:rows], bound[:rows]
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    err = (got - want)[~odd].abs()
    assert (err <= bound[~odd]).all(), "off by %g, %.2f of the bound" % (float(err.max()), float((err / bound[~odd]).max()))
    return got


# every kernel variant: few rows per KV head with four waves and with one (2 048 units and more), 64, 128, 256 rows
# and two row tiles; histories of one slice and of several; blocks smaller than what a wave load covers
VARIANTS = [
    (64, 2, 2, [9, 5, 3, 16], [0, 7, 70, 700], 16), (128, 4, 2, [4, 1, 8, 5], [33, 1, 40, 5000], 32),
    (64, 16, 16, [1] * 130, list(range(1, 131)), 16), (64, 3, 3, [40, 33, 17], [70, 0, 300], 16),
    (128, 2, 1, [33, 60], [64, 97], 2), (64, 6, 2, [33, 40], [100, 2], 1), (128, 4, 1, [64, 40], [100, 2000], 64),
    (64, 5, 1, [64, 61], [31, 600], 16)]


def _variant(dtype, which, seed):
    dim, heads, kv, nodes, cached, block = VARIANTS[which]
    return _tree_state(cached, nodes, heads, kv, dim, block, dtype, seed=seed)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("which", range(len(VARIANTS)))
def test_weights_are_not_rounded_to_the_storage_type(dtype, which):
    """Small scores, so that nothing but the rounding of the weights could pass the bound."""
    s = _variant(dtype, which, seed=20 + which)
    _check(s, scale=1 / 64)
    _check(s)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("which", range(len(VARIANTS)))
def test_visible_history_values_that_are_not_finite(dtype, which):
    s = _variant(dtype, which, seed=40 + which)
    block, g = s["k_cache"].shape[2], torch.Generator().manual_seed(which)
    hit = 0
    for i, c in enumerate(s["cached"].tolist()):
        if c < 7 or i % 5 == 4:
            continue
        at = torch.randperm(c, generator=g)[:7].tolist()
        for p, f, x in zip(at, (3, 9, 17, 30, 30, 31, 31), (math.inf, -math.inf, math.nan, math.inf, -math.inf, math.inf, math.inf)):
            s["v_cache"][int(s["table"][i, p // block]), 0, p % block, f] = x
        hit += 1
    got = _check(s)
    assert hit and not torch.isfinite(got[:, 0, 3]).all() and torch.isfinite(got[..., 0]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("which", range(len(VARIANTS)))
def test_visible_history_keys_that_are_not_finite(dtype, which):
    """A NaN spoils the rows of its KV head; an infinity too where its score is +inf, and drops its own key where that is -inf."""
    s = _variant(dtype, which, seed=60 + which)
    block = s["k_cache"].shape[2]
    for i, c in enumerate(s["cached"].tolist()):
        if c < 2 or i % 3 == 2:
            continue
        p = c - 2
        s["k_cache"][int(s["table"][i, p // block]), 0, p % block, 5] = math.inf if i % 3 == 0 else math.nan
    got = _check(s)
    assert torch.isnan(got).any() and torch.isfinite(got).any()


def _one_dominant(n_keys, dim=64, block=64):
    """One key 17.5 nats above all others (2^-25.2 each), whose own value is zero: the output is what the others weigh."""
    n_blocks = -(-(n_keys + 1) // block)
    kc, vc = torch.zeros(n_blocks, 1, block, dim, dtype=HF), torch.ones(n_blocks, 1, block, dim, dtype=HF)
    q, k, v = torch.zeros(1, 1, dim, dtype=HF), torch.zeros(1, 1, dim, dtype=HF), torch.zeros(1, 1, dim, dtype=HF)
    q[0, 0, 0], k[0, 0, 0] = 4.375, 4.0
    return dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, table=torch.arange(n_blocks).int()[None], cached=torch.tensor([n_keys]).int(),
                starts=torch.tensor([0, 1]).int(), slots=torch.tensor([n_keys]), parents=None, layout="hnd", fused=False)


@pytest.mark.parametrize("n_keys", [300, 16000])
def test_small_float16_weights_add_up(n_keys):
    got = _check(_one_dominant(n_keys), scale=1.0)
    assert (got > 0.9 * n_keys * math.exp(-17.5)).all()


def test_an_infinite_value_under_a_small_float16_weight():
    s = _one_dominant(300)
    s["v_cache"][2, 0, 3, 7] = -math.inf
    assert float(_check(s, scale=1.0)[0, 0, 7]) == -math.inf


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("which", range(len(VARIANTS)))
def test_values_that_are_not_finite_under_weights_that_underflow(dtype, which):
    """Scores of hundreds: between tiles, waves and slices most weights are zero in float32, their keys are seen all the same."""
    s = _variant(dtype, which, seed=80 + which)
    s["q"] = (s["q"].float() * 40).to(dtype)
    block, g = s["k_cache"].shape[2], torch.Generator().manual_seed(100 + which)
    for i, c in enumerate(s["cached"].tolist()):
        if c < 4 or i % 4 == 3:
            continue
        at = torch.randperm(c, generator=g)[:4].tolist()
        for p, f, x in zip(at, (2, 11, 20, 29), (math.inf, -math.inf, math.nan, math.inf)):
            s["v_cache"][int(s["table"][i, p // block]), 0, p % block, f] = x
    got = _check(s)
    assert torch.isinf(got).any() and torch.isnan(got).any()


@pytest.mark.parametrize("n_keys", [300, 16000])
def test_an_infinite_value_far_below_the_largest_score(n_keys):
    s = _one_dominant(n_keys)
    s["q"][0, 0, 0], s["k"][0, 0, 0] = 12.5, 12.0
    for block, f in ((0, 3), (2, 4), (n_keys // 64 - 1, 5)):
        s["v_cache"][block, 0, 9, f] = math.inf
    assert torch.isinf(_check(s, scale=1.0)[0, 0, 3:6]).all()
