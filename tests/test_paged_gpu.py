"""paged.plan and paged.tree_attention on the GPU against the 64-bit references of tests/_operators.py,
at the sizes, layouts and masks where they can go wrong."""
import numpy as np
import pytest
import torch

from tests import _operators as O

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------------------------- plan
def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _plan_state(n, block, longest, new_hi, seed, idle=0.2, spare=7):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, longest + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    held = -(-cached // block) + (rng.random(n) < 0.3)
    gone = rng.random(n) < idle
    cached[gone] = new[gone] = 0
    need = -(-(cached + new) // block)
    width = int(max(held.max(), need.max(), 1)) + 2
    n_ring = int(held.sum() + np.maximum(need - held, 0).sum() + spare)
    ids = rng.permutation(n_ring)
    table = np.full((n, width), -1)
    at = 0
    for i in range(n):
        table[i, :held[i]] = ids[at: at + held[i]]
        at += held[i]
    free = np.full(n_ring, -1)
    head = int(rng.integers(0, 5 * n_ring))
    free[(head + np.arange(n_ring - at)) % n_ring] = ids[at:]
    return dict(cached=cached, new=new, held=held, table=table, free=free, ring=np.array([head, head + n_ring - at]))


def _run_plan(s, block, rows):
    from speech_to_text_amd import paged
    dev = {k: _i32(v) for k, v in s.items() if k != "ring"}
    ring = torch.tensor(s["ring"], dtype=torch.int64, device="cuda")
    r = paged.plan(dev["cached"], dev["new"], dev["table"], dev["held"], dev["free"], ring, block_size=block, rows=rows)
    got = dict(r._asdict(), table=dev["table"], free=dev["free"])
    return {k: v.cpu().numpy() for k, v in got.items()}, dev, ring


@pytest.mark.parametrize("n,block,longest,new_hi", [
    (1, 16, 0, 1), (1, 1, 50, 3), (3, 16, 31, 9), (63, 4, 200, 1), (64, 64, 500, 70), (65, 8, 100, 0), (1000, 32, 3000, 40),
    (1025, 16, 448, 9), (8192, 128, 5000, 3), (37, 65536, 100000, 200)])
def test_plan_equals_the_request_by_request_form(n, block, longest, new_hi):
    s = _plan_state(n, block, longest, new_hi, seed=n + block)
    rows = int(s["new"].sum()) + 5
    want = O.plan_reference(s["cached"], s["new"], s["table"], s["held"], s["free"], s["ring"], block, rows)
    got, dev, ring = _run_plan(s, block, rows)
    assert got["status"][0] == 0
    for name, v in want.items():
        assert np.array_equal(got[name], v), name
    # what it was given is untouched, so the step can be planned again with the same result
    assert np.array_equal(dev["held"].cpu().numpy(), s["held"]) and np.array_equal(ring.cpu().numpy(), s["ring"])
    again, _, _ = _run_plan(dict(s, table=got["table"], free=got["free"]), block, rows)
    for name, v in want.items():
        assert np.array_equal(again[name], v), name


def test_plan_refuses_on_the_device_and_changes_nothing():
    base = _plan_state(70, 16, 300, 5, seed=1)
    rows = int(base["new"].sum())
    need = np.maximum(-(-(base["cached"] + base["new"]) // 16) - base["held"], 0).sum()
    assert need > 0

    def with_(**change):
        s = {k: v.copy() for k, v in base.items()}
        for k, (at, v) in change.items():
            s[k][at] = v
        return s
    short = with_(ring=(1, base["ring"][0] + need - 1))
    cases = [(short, rows, 1), (with_(cached=(69, 16 * base["table"].shape[1])), rows, 2), (with_(cached=(3, 2 ** 31 - 1)), rows, 2),
             (base, rows - 1, 3), (with_(new=(0, -1)), rows, 4), (with_(cached=(64, -5)), rows, 4), (with_(held=(9, -1)), rows, 4),
             (with_(held=(9, base["table"].shape[1] + 1)), rows, 4), (with_(ring=(1, base["ring"][0] - 1)), rows, 4),
             (with_(ring=(1, base["ring"][0] + len(base["free"]) + 1)), rows, 4), (with_(ring=(0, -1)), rows, 4)]
    for s, r, status in cases:
        got, _, _ = _run_plan(s, 16, r)
        assert got["status"][0] == status, (status, got["status"])
        for name in ("table", "free", "held", "ring"):
            assert np.array_equal(got[name], s[name]), (status, name)
        assert (got["slots"] == -1).all() and (got["positions"] == -1).all() and (got["starts"] == 0).all()
    exact = with_(ring=(1, base["ring"][0] + need))                          # just enough
    assert _run_plan(exact, 16, rows)[0]["status"][0] == 0


def test_plan_over_many_steps_never_shares_or_loses_a_block():
    """Requests grow, end and are replaced for 30 steps; every block is in exactly one place throughout."""
    from speech_to_text_amd import paged
    rng = np.random.default_rng(4)
    n, block, width, n_ring = 40, 8, 12, 300
    table, held = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), _i32(np.zeros(n))
    free = _i32(rng.permutation(n_ring))
    ring = torch.tensor([0, n_ring], dtype=torch.int64, device="cuda")
    cached = np.zeros(n, dtype=np.int64)
    for step in range(30):
        new = rng.integers(0, 7, n)
        over = (cached + new > block * width) | (rng.random(n) < 0.1)
        cached[over] = new[over] = 0
        r = paged.plan(_i32(cached), _i32(new), table, held, free, ring, block_size=block, rows=6 * n)
        held, ring = r.held, r.ring
        assert int(r.status) == 0
        t, h = table.cpu().numpy(), held.cpu().numpy()
        lo, hi = ring.tolist()
        f = free.cpu().numpy()
        have = [b for i in range(n) for b in t[i, :h[i]]] + [f[j % n_ring] for j in range(lo, hi)]
        assert sorted(have) == list(range(n_ring)), step
        # accepted: some of the new tokens stay
        cached = cached + np.minimum(new, rng.integers(0, 7, n))


# ------------------------------------------------------------------------------------ tree attention
def _tree_state(cached, nodes, heads, kv, dim, block, dtype, seed, layout="hnd", chain=False, fused=False, spare=3, fill=None):
    """Random inputs on the CPU (made in float32, rounded once); `fill`: what cache positions nobody may see
    and nodes' K/V behind the last sequence hold."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    cached, nodes = np.asarray(cached), np.asarray(nodes)
    n, rows = len(cached), int(nodes.sum()) + spare
    blocks = -(-(cached + nodes) // block)
    width, n_blocks = max(int(blocks.max()), 1), int(blocks.sum()) + 2
    ids = rng.permutation(n_blocks)
    table = np.full((n, width), -1)
    at = 0
    for i in range(n):
        table[i, :blocks[i]] = ids[at: at + blocks[i]]
        at += blocks[i]
    starts = np.concatenate([[0], np.cumsum(nodes)])
    slots = np.full(rows, -1)
    parents = np.full(rows, -1)
    for i in range(n):
        for a in range(nodes[i]):
            p = cached[i] + a
            slots[starts[i] + a] = table[i, p // block] * block + p % block
            parents[starts[i] + a] = rng.integers(-1, a) if a else -1
    rand = lambda *s: torch.randn(s, generator=g).to(dtype)
    shape = (n_blocks, kv, block, dim)
    kc, vc = rand(*shape), rand(*shape)
    if fill is not None:
        used = torch.zeros(n_blocks, block, dtype=torch.bool)
        for i in range(n):
            for p in range(cached[i]):
                used[table[i, p // block], p % block] = True
        for c in (kc, vc):
            c.permute(0, 2, 1, 3)[~used] = fill
    q, k, v = rand(rows, heads, dim), rand(rows, kv, dim), rand(rows, kv, dim)
    if fill is not None and spare:
        k[-spare:], v[-spare:] = fill, fill
    return dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, table=torch.from_numpy(table).int(), cached=torch.from_numpy(cached).int(),
                starts=torch.from_numpy(starts).int(), slots=torch.from_numpy(slots).long(),
                parents=None if chain else torch.from_numpy(parents).int(), layout=layout, fused=fused)


def _to_gpu(s):
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if s["layout"] == "nhd":                       # [block][position][head][dim] in memory
        for name in ("k_cache", "v_cache"):
            d[name] = d[name].transpose(1, 2).contiguous().transpose(1, 2)
    if s["fused"]:                                 # q | k | v of a row side by side, as a projection leaves them
        rows, heads, dim = s["q"].shape
        kv = s["k"].shape[1]
        row = torch.cat([d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1)], dim=1)
        d["q"] = row[:, :heads * dim].unflatten(1, (heads, dim))
        d["k"] = row[:, heads * dim: (heads + kv) * dim].unflatten(1, (kv, dim))
        d["v"] = row[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
    return d


def _call(d, max_nodes, **kw):
    from speech_to_text_amd import paged
    return paged.tree_attention(d["q"], d["k"], d["v"], d["k_cache"], d["v_cache"], d["table"], d["cached"], d["starts"],
                                d["slots"], d["parents"], max_nodes=max_nodes, **kw)


def _same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def _check(s, max_nodes=None, want=None, **kw):
    nodes = (s["starts"][1:] - s["starts"][:-1]).tolist()
    max_nodes = max_nodes or max(max(nodes), 1)
    want, bound, kc, vc = want or O.tree_reference(*[s[k] for k in ("q", "k", "v", "k_cache", "v_cache", "table", "cached", "starts", "slots", "parents")],
                                                   scale=kw.get("scale"))
    d = _to_gpu(s)
    keep = torch.full_like(d["q"].contiguous(), 7.5)
    out = _call(d, max_nodes, out=keep, **kw)
    got = out.double().cpu()
    live = ~torch.isnan(bound.sum(dim=(1, 2)) + want.sum(dim=(1, 2)))
    assert live[: int(s["starts"][-1])].all()
    err = (got[live] - want[live]).abs()
    assert (err <= bound[live]).all(), "off by %g, %.2f of the bound" % (float(err.max()), float((err / bound[live]).max()))
    assert (got[~live] == 7.5).all()                                          # rows of no sequence stay
    assert _same(d["k_cache"], kc) and _same(d["v_cache"], vc)
    return out, d


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 4])
def test_tree_lengths_around_every_tile_edge(dtype, dim, group):
    cached = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300]
    nodes = [1, 2, 15, 16, 17, 3, 32, 33, 1, 31, 5, 64, 9, 48]
    s = _tree_state(cached, nodes, 2 * group, 2, dim, 16, dtype, seed=dim + group)
    _check(s)


@pytest.mark.parametrize("block", [1, 2, 8, 32, 64, 256])
@pytest.mark.parametrize("layout,fused", [("hnd", False), ("nhd", True)])
def test_tree_block_sizes_and_layouts(block, layout, fused):
    s = _tree_state([0, 5, 100, 257, 64], [3, 1, 20, 9, 7], 6, 2, 64, block, BF, seed=block, layout=layout, fused=fused)
    _check(s)
    _check(dict(s, parents=None))                  # the same rows as chains


@pytest.mark.parametrize("heads,kv", [(1, 1), (20, 20), (5, 1), (16, 2), (12, 4), (48, 3)])
def test_tree_head_groups(heads, kv):
    _check(_tree_state([70, 0, 33], [11, 64, 1], heads, kv, 64, 16, BF, seed=heads))


@pytest.mark.parametrize("dtype,dim,group,nodes", [(BF, 128, 4, 64), (HF, 128, 5, 33), (BF, 64, 3, 61), (HF, 64, 9, 40)])
def test_tree_many_rows_of_a_head(dtype, dim, group, nodes):
    # more than 128 rows: one image for eight waves, and every remainder of its pipeline of four tiles
    cached = [0, 1, 31, 32, 33, 63, 64, 96, 97, 127, 128, 129, 159, 161, 192, 224, 255, 256, 257, 300]
    _check(_tree_state(cached, [nodes - i % 5 for i in range(len(cached))], 2 * group, 2, dim, 16, dtype, seed=nodes))


@pytest.mark.parametrize("dtype,dim,group,nodes", [(BF, 128, 4, 64), (HF, 64, 3, 64), (BF, 128, 2, 33), (HF, 128, 1, 40), (BF, 64, 1, 3)])
def test_tree_slices_of_every_variant(dtype, dim, group, nodes):
    _check(_tree_state([5000, 257, 0, 513, 1025], [nodes, 1, nodes, 2, nodes - 1], group, 1, dim, 32, dtype, seed=group))


@pytest.mark.parametrize("max_cached", [0, 1, 5000, 100000])
def test_tree_long_histories_whatever_the_hint(max_cached):
    """The bound on the history chooses the split only: too small, right or too large, same result."""
    s = _tree_state([5000, 1, 2047, 4096], [9, 4, 33, 1], 4, 2, 128, 32, BF, seed=9)
    _check(s, max_cached=max_cached)


def test_tree_single_tokens_of_many_sequences():
    rng = np.random.default_rng(2)
    _check(_tree_state(rng.integers(0, 90, 150), np.ones(150, dtype=int), 3, 3, 64, 16, HF, seed=3))


def test_tree_sequences_without_rows_and_larger_max_nodes():
    s = _tree_state([9, 40, 0, 17], [0, 5, 0, 2], 2, 1, 64, 16, BF, seed=5)
    _check(s, max_nodes=64)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_tree_unseen_positions_may_hold_anything(fill):
    """Stale positions behind the histories, blocks of nobody, rows behind the last sequence."""
    s = _tree_state([0, 5, 100, 31, 64], [3, 1, 20, 9, 33], 4, 2, 64, 16, BF, seed=6, fill=fill)
    _check(s)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim,heads", [(64, 2), (128, 8)])
def test_tree_a_bad_node_spoils_only_those_that_see_it(bad, dim, heads):
    s = _tree_state([37, 0, 200], [40, 9, 64], heads, 2, dim, 16, BF, seed=7)
    parents = s["parents"]
    want = O.tree_reference(*[s[k] for k in ("q", "k", "v", "k_cache", "v_cache", "table", "cached", "starts", "slots", "parents")])
    d = _to_gpu(s)
    for first, node in ((0, 7), (40, 2), (49, 33)):
        d["v"][first + node, 1, 5] = bad
        d["k"][first + node, 0] = bad
    out = _call(d, 64).double().cpu()
    hit = torch.zeros(113, dtype=torch.bool)
    for i, (lo, hi, node) in enumerate(((0, 40, 7), (40, 49, 2), (49, 113, 33))):
        hit[lo:hi] = torch.from_numpy(O.tree_paths(parents[lo:hi], hi - lo)[:, node])
    ok = torch.nonzero(~hit)[:, 0]
    assert len(ok) > 50 and hit[7] and hit[42] and hit[82]
    assert ((out[ok] - want[0][ok]).abs() <= want[1][ok]).all()
    per = heads // 2
    assert torch.isnan(out[7, :per]).all()                       # KV head 0: a bad key makes every feature of those heads NaN
    assert not torch.isfinite(out[7, per:, 5]).any()             # KV head 1: one bad value feature
    good = [f for f in range(dim) if f != 5]
    assert ((out[7, per:][:, good] - want[0][7, per:][:, good]).abs() <= want[1][7, per:][:, good]).all()


def test_tree_bad_table_entries_and_parents():
    """Entries outside the cache leave their positions out, parents that are not earlier nodes are roots, and
    slots outside the cache store nothing."""
    s = _tree_state([64, 100, 40], [6, 5, 7], 2, 2, 64, 16, BF, seed=8)
    s["table"][0, 1] = -1
    s["table"][1, 0] = 10 ** 6
    s["table"][2, 0] = -2 ** 31
    s["parents"][3], s["parents"][8], s["parents"][13] = 3, 2 ** 31 - 1, -2 ** 31
    s["slots"][0], s["slots"][7], s["slots"][12] = -5, 2 ** 40, s["k_cache"].shape[0] * 16
    _check(s)


def test_tree_table_narrower_than_the_history():
    s = _tree_state([100, 20], [3, 3], 2, 1, 64, 16, BF, seed=10)
    s["table"] = s["table"][:, :4].contiguous()                  # 64 of the 100 positions have an entry
    _check(s)


def test_tree_scale_and_large_scores():
    """Scores of several hundred: the softmax has one survivor and nothing overflows."""
    s = _tree_state([80, 3], [10, 10], 2, 2, 64, 16, HF, seed=11)
    s["q"] = (s["q"].float() * 40).to(HF)
    _check(s, scale=0.9)
    _check(s, scale=0.0)
    _check(s, scale=-0.125)


def test_tree_offsets_beyond_32_bits():
    """A cache whose second half starts 2^32 elements in: block 1 of two, 9 GB apart."""
    s = _tree_state([30, 9], [4, 5], 2, 1, 64, 32, BF, seed=12, spare=0)
    n_blocks = s["k_cache"].shape[0]
    d = _to_gpu(s)
    stride = 2 ** 32 // (n_blocks - 1) // 8 * 8 + 4096
    big = [torch.empty((n_blocks - 1) * stride + 32 * 64, dtype=BF, device="cuda") for _ in range(2)]
    for name, store in zip(("k_cache", "v_cache"), big):
        view = store.as_strided(s[name].shape, (stride, 32 * 64, 64, 1))
        view.copy_(d[name])
        d[name] = view
    want, bound, kc, vc = O.tree_reference(*[s[k] for k in ("q", "k", "v", "k_cache", "v_cache", "table", "cached", "starts", "slots", "parents")])
    out = _call(d, 5).double().cpu()
    assert ((out - want).abs() <= bound).all()
    assert _same(d["k_cache"], kc) and _same(d["v_cache"], vc)


def test_tree_results_do_not_depend_on_the_run():
    s = _tree_state([3000, 10, 700], [17, 64, 3], 8, 2, 128, 16, BF, seed=13)
    d = _to_gpu(s)
    first = _call(d, 64)
    for _ in range(3):
        assert torch.equal(first[:84], _call(d, 64)[:84])


def test_plan_and_tree_on_another_stream_and_in_graphs():
    """Two captured steps (plan, then attention over what it planned) replayed in turn with eager work in
    between: each replay equals the eager result."""
    from speech_to_text_amd import paged
    block, n = 16, 3
    s = _tree_state([20, 0, 500], [5, 5, 5], 4, 2, 64, block, BF, seed=14, spare=0)
    d = _to_gpu(s)
    n_blocks = d["k_cache"].shape[0]

    def fresh(cached):
        held = -(-np.asarray(cached) // block)
        table = np.full((n, 40), -1)
        table[:, :] = -1
        at = 0
        for i in range(n):
            table[i, :held[i]] = np.arange(at, at + held[i])
            at += held[i]
        free = np.full(n_blocks, -1)
        free[: n_blocks - at] = np.arange(at, n_blocks)
        # a cache each: the blocks one step writes are history of the other
        return dict(cached=_i32(cached), new=_i32([5] * n), table=_i32(table), held=_i32(held), free=_i32(free),
                    ring=torch.tensor([0, n_blocks - at], dtype=torch.int64, device="cuda"),
                    k_cache=d["k_cache"].clone(), v_cache=d["v_cache"].clone())

    def step(p):
        r = paged.plan(p["cached"], p["new"], p["table"], p["held"], p["free"], p["ring"], block_size=block, rows=15)
        return paged.tree_attention(d["q"], d["k"], d["v"], p["k_cache"], p["v_cache"], p["table"], p["cached"], r.starts,
                                    r.slots, d["parents"], max_nodes=5, max_cached=500)
    plans = [fresh([20, 0, 500]), fresh([17, 33, 64])]
    eager = [step(p).clone() for p in plans]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for p, e in zip(plans, eager):
            got = step(p)
            side.synchronize()
            assert torch.equal(got, e)
    graphs, outs = [], []
    for p in plans:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(p))
        graphs.append(g)
    for turn in range(4):
        for g, o, p, e in zip(graphs, outs, plans, eager):
            o.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, e), turn
            assert torch.equal(step(p), e)


def test_plan_and_tree_run_as_decoding_does():
    """Three requests of different lengths: a prompt as a chain, then trees of which a path is accepted (its K/V
    moved to the front by the caller), six steps.  The output of every accepted token equals attention over
    the whole accepted sequence."""
    from speech_to_text_amd import paged
    rng = np.random.default_rng(15)
    g = torch.Generator().manual_seed(15)
    heads, kv, dim, block, n, n_blocks, width = 4, 2, 64, 8, 3, 64, 16
    kc, vc = (torch.full((n_blocks, kv, block, dim), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    table, held = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), _i32(np.zeros(n))
    free, ring = _i32(rng.permutation(n_blocks)), torch.tensor([0, n_blocks], dtype=torch.int64, device="cuda")
    cached = np.zeros(n, dtype=int)
    story = [[] for _ in range(n)]                  # accepted (k, v) per request
    for step in range(6):
        nodes = np.array([9, 1, 20]) if step == 0 else rng.integers(1, 12, n)
        rows = int(nodes.sum())
        q, k, v = (torch.randn(rows, h, dim, generator=g).to(BF) for h in (heads, kv, kv))
        r = paged.plan(_i32(cached), _i32(nodes), table, held, free, ring, block_size=block, rows=rows)
        held, ring = r.held, r.ring
        starts = np.concatenate([[0], np.cumsum(nodes)])
        par = np.concatenate([[-1 if a == 0 else (a - 1 if step == 0 else int(rng.integers(0, a))) for a in range(m)] for m in nodes])
        out = paged.tree_attention(q.cuda(), k.cuda(), v.cuda(), kc, vc, table, _i32(cached), r.starts, r.slots,
                                   None if step == 0 else _i32(par), max_nodes=int(nodes.max())).double().cpu()
        slots = r.slots.tolist()
        for i in range(n):
            lo = starts[i]
            path = [int(nodes[i]) - 1]
            while 0 <= par[lo + path[0]]:
                path.insert(0, int(par[lo + path[0]]))
            for j, a in enumerate(path):
                story[i].append((k[lo + a], v[lo + a]))
                keys = torch.stack([x[0] for x in story[i]]).double()
                vals = torch.stack([x[1] for x in story[i]]).double()
                for h in range(heads):
                    w = torch.softmax(keys[:, h // 2] @ q[lo + a, h].double() * dim ** -0.5, dim=0)
                    o, big = w @ vals[:, h // 2], w @ vals[:, h // 2].abs()
                    eps = torch.finfo(BF).eps
                    assert ((out[lo + a, h] - o).abs() <= eps / 2 * o.abs() + (eps / 2 + 1e-4) * big).all(), (step, i, a, h)
                src, dst = slots[lo + a], slots[lo + j]          # path[j] >= j: moved towards the front
                for c in (kc, vc):
                    c[dst // block, :, dst % block] = c[src // block, :, src % block].clone()
            cached[i] += len(path)
