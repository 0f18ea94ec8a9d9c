"""Argument checks of paged.py, mxfp4.py and the C entry points below them: every refusal is decided on
the host before anything touches a GPU.  Also the 64-bit references against cases worked by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

from speech_to_text_amd import _lib, mxfp4, paged
from tests import _operators as O


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _plan_args(**change):
    a = dict(cached=_i32(3), new=_i32(3), table=_i32(3, 4), held=_i32(3), free=_i32(8), ring=torch.zeros(2, dtype=torch.int64))
    k = dict(block_size=16, rows=5)
    for name, v in change.items():
        (k if name in k else a)[name] = v
    return a, k


@pytest.mark.parametrize("change", [
    dict(block_size=0), dict(block_size=24), dict(block_size=131072), dict(rows=-1), dict(cached=_i32(0)),
    dict(cached=_i32(8193)), dict(cached=_i32(1, 3)), dict(new=_i32(4)), dict(new=_i32(3).long()), dict(held=_i32(2)),
    dict(table=_i32(2, 4)), dict(table=_i32(3)), dict(table=_i32(3, 0)), dict(table=_i32(3, 8)[:, ::2]), dict(free=_i32(0)),
    dict(ring=_i32(2)), dict(ring=torch.zeros(3, dtype=torch.int64)),
    dict()])                                        # all in order, but on the CPU
def test_plan_refusals(change):
    a, k = _plan_args(**change)
    with pytest.raises(ValueError):
        paged.plan(a["cached"], a["new"], a["table"], a["held"], a["free"], a["ring"], **k)


def _tree_args(**change):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(5, 4, 64, dtype=bf), k=torch.zeros(5, 2, 64, dtype=bf), v=torch.zeros(5, 2, 64, dtype=bf),
             k_cache=torch.zeros(6, 2, 16, 64, dtype=bf), v_cache=torch.zeros(6, 2, 16, 64, dtype=bf), table=_i32(3, 2),
             cached=_i32(3), starts=_i32(4), slots=torch.zeros(5, dtype=torch.int64), parents=_i32(5))
    k = dict(max_nodes=4, out=None)
    for name, v in change.items():
        (k if name in k else a)[name] = v
    return a, k


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(5, 4, 64)), dict(q=torch.zeros(5, 4, 96, dtype=torch.bfloat16)), dict(q=torch.zeros(5, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 3, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(5, 4, 128, dtype=torch.bfloat16)[..., ::2]),
    dict(q=torch.zeros(5, 4 * 64 + 4, dtype=torch.bfloat16)[:, :256].unflatten(1, (4, 64))),
    dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)),
    dict(v=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), dict(k_cache=torch.zeros(6, 2, 12, 64, dtype=torch.bfloat16)),
    dict(k_cache=torch.zeros(6, 2, 16, 64)), dict(v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)),
    dict(v_cache=torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16).transpose(1, 2)), dict(table=_i32(3, 2).long()),
    dict(cached=_i32(4)), dict(starts=_i32(3)), dict(slots=_i32(5)), dict(parents=_i32(4)), dict(max_nodes=0), dict(max_nodes=65),
    dict(out=torch.zeros(5, 4, 64)), dict()])
def test_tree_attention_refusals(change):
    a, k = _tree_args(**change)
    with pytest.raises(ValueError):
        paged.tree_attention(*a.values(), **k)


@pytest.mark.parametrize("codes,scales", [
    (torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.uint8)),
    (torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)),
    (torch.zeros(2, 32, dtype=torch.uint8)[:, ::2], torch.zeros(2, 1, dtype=torch.uint8)),
    (torch.zeros(16, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8))])
def test_mxfp4_tensor_refusals(codes, scales):
    with pytest.raises(ValueError):
        mxfp4.Mxfp4Tensor(codes, scales)


@pytest.mark.parametrize("x", [torch.zeros(2, 33), torch.zeros(32), torch.zeros(2, 32, dtype=torch.float64),
                               torch.zeros(2, 64)[:, ::2], torch.zeros(2, 34)[:, :32], torch.zeros(1, 32).expand(3, 32),
                               torch.zeros(2, 32)])
def test_quantize_refusals(x):
    with pytest.raises(ValueError):
        mxfp4.quantize(x)


def test_matmul_refusals():
    w = mxfp4.Mxfp4Weight.__new__(mxfp4.Mxfp4Weight)             # a weight of the right shape without a GPU behind it
    w.shape, w.packed = torch.Size((3, 64)), torch.zeros(16, dtype=torch.uint8)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    bad = [dict(x=x.float()), dict(x=x[:, :32]), dict(x=torch.zeros(2, 68, dtype=torch.bfloat16)[:, :64]), dict(x=x[0]), dict(w=x),
           dict(gelu="sigmoid"), dict(out_dtype=torch.float16), dict(bias=torch.zeros(4)), dict(bias=torch.zeros(3, dtype=torch.bfloat16)),
           dict(out=torch.zeros(2, 4)), dict(out=torch.zeros(3, 2).t()), dict(accumulate=True),
           dict(accumulate=True, out=torch.zeros(2, 3, dtype=torch.bfloat16)), dict(accumulate=True, out=torch.zeros(2, 3), gelu="erf")]
    for change in bad:
        args = dict(dict(x=x, w=w), **change)
        with pytest.raises(ValueError):
            mxfp4.matmul(args.pop("x"), args.pop("w"), **args)


def test_c_entry_points_refuse_before_any_launch():
    """Codes and messages of the C ABI; made-up pointers, none of which is followed."""
    lib = paged._library()
    mxfp4._library()
    p = 0x10000
    ok = [p, p, 3, 16, p, 4, p, 8, p, p + 64, p, p + 64, 5, p, p, p, p, None]
    for at, v, code in [(2, 0, -2), (2, 8193, -2), (3, 3, -2), (5, 0, -1), (7, 0, -1), (12, -1, -1), (0, None, -1), (9, p, -1), (11, p, -1),
                        (16, None, -1), (13, None, -1)]:
        bad = list(ok)
        bad[at] = v
        assert lib.stt_paged_plan(*bad) == code, (at, v)
        assert _lib.load().stt_last_error()
    good = dict(d_q=p, d_k=p, d_v=p, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, d_k_cache=p, d_v_cache=p,
                block_stride=2048, head_stride=1024, pos_stride=64, d_table=p, d_cached=p, d_starts=p, d_slots=p, d_out=p,
                out_row=256, out_head=64, scale=1.0, dtype=1, n_seq=3, rows=5, n_heads=4, n_kv_heads=2, head_dim=64, n_blocks=6,
                block_size=16, width=2, max_nodes=4, max_cached=0)
    for change, code in [(dict(dtype=0), -2), (dict(head_dim=80), -2), (dict(n_heads=3), -1), (dict(n_kv_heads=0), -1), (dict(n_seq=-1), -1),
                         (dict(block_size=48), -2), (dict(max_nodes=65), -2), (dict(max_nodes=0), -2), (dict(d_q=None), -1),
                         (dict(d_q=p + 8), -1), (dict(q_head=68), -1), (dict(pos_stride=4), -1), (dict(width=2 ** 27, block_size=16), -2),
                         (dict(d_slots=None), -1), (dict(d_k_cache=None), -1)]:
        a = paged.TreeAttentionArgs(**dict(good, **change))
        assert lib.stt_tree_attention(C.byref(a), None, 0, None) == code, change
    assert lib.stt_tree_attention(None, None, 0, None) == -1
    a = paged.TreeAttentionArgs(**dict(good, n_seq=0))
    assert lib.stt_tree_attention(C.byref(a), None, 0, None) == 0            # nothing to do, nothing launched
    assert lib.stt_mxfp4_quantize(p, 0, 2, 33, 64, p, p, None) == -1
    assert lib.stt_mxfp4_quantize(p, 3, 2, 32, 64, p, p, None) == -2
    assert lib.stt_mxfp4_quantize(p + 4, 0, 2, 32, 64, p, p, None) == -1
    assert lib.stt_mxfp4_quantize(p, 1, 2, 32, 36, p, p, None) == -1
    assert lib.stt_mxfp4_quantize(p, 1, 2, 32, 0, p, p, None) == -1
    assert lib.stt_mxfp4_quantize(p, 1, 0, 32, 32, p, p, None) == 0
    assert lib.stt_mxfp4_dequantize(p, p, 2, 32, p, 2, None) == -2
    assert lib.stt_mxfp4_dequantize(p, p, 2, 40, p, 0, None) == -1
    assert lib.stt_mxfp4_pack(p, None, 2, 32, p, None) == -1
    assert lib.stt_mxfp4_packed_bytes(17, 160) == 2 * 2 * (1024 + 64)
    m = dict(d_x=p, x_row=64, d_w=p, d_out=p, out_row=3, out_dtype=1, gelu=0, accumulate=0, m=2, n=3, k=64)
    for change, code in [(dict(k=0), -1), (dict(k=48), -1), (dict(m=-1), -1), (dict(out_dtype=2), -2), (dict(gelu=3), -2),
                         (dict(accumulate=1), -2), (dict(accumulate=1, out_dtype=0, gelu=1), -2), (dict(d_x=None), -1),
                         (dict(d_x=p + 2), -1), (dict(x_row=60), -1), (dict(out_row=2), -1)]:
        a = mxfp4.MatmulArgs(**dict(m, **change))
        assert lib.stt_mxfp4_matmul(C.byref(a), None) == code, change
    assert lib.stt_mxfp4_matmul(C.byref(mxfp4.MatmulArgs(**dict(m, m=0))), None) == 0


def test_references_on_cases_worked_by_hand():
    # ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4; 7 saturates at 6
    x = np.zeros((1, 32))
    x[0, :10] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.3]
    codes, scales = O.quantize_reference(x)
    assert scales[0, 0] == 127
    assert O.values_of(codes, scales)[0, :10].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.5]
    assert O.quantize_reference(np.zeros((1, 32)))[1][0, 0] == 0
    # node 2 hangs under 0, 3 under 1; -1, 7 and 5 (not earlier) are roots
    seen = O.tree_paths([-1, 7, 0, 1, 5], 5)
    assert [np.nonzero(r)[0].tolist() for r in seen] == [[0], [1], [0, 2], [1, 3], [4]]
    # three requests, blocks of 4: the first grows by one block, the second has ended, the third stays
    r = O.plan_reference([3, 0, 1], [2, 0, 3], np.array([[5, -1], [2, 7], [1, -1]]), [1, 2, 1], np.array([-1, 0, 9, -1]), [1, 3], 4, 6)
    assert r["table"].tolist() == [[5, 0], [2, 7], [1, -1]] and r["free"].tolist() == [7, 0, 9, 2]
    assert r["ring"].tolist() == [2, 5] and r["held"].tolist() == [2, 0, 1] and r["starts"].tolist() == [0, 2, 2, 5]
    assert r["slots"].tolist() == [23, 0, 5, 6, 7, -1] and r["positions"].tolist() == [3, 4, 1, 2, 3, -1]
