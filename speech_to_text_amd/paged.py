"""Paged K/V cache on the GPU: block tables and slot maps from request lengths, and attention of drafted
token trees over the cache (stt_paged_plan and stt_tree_attention of include/stt_mi355x.h).

What a step of speculative decoding needs beside the engine's fixed cache: sequences of different
lengths, blocks of positions from a common pool, and attention in which a drafted token sees its own
path only.  `WhisperEngine.decode_tree` runs on both; they work for any decoder with heads of 64 or
128.  No counterpart in the reference.

Every call runs on the current stream of the tensors' device and returns without waiting for it.
"""
import collections
import ctypes as C
import struct

import torch

from . import _lib

MAX_NODES = 64            # STT_TREE_MAX_NODES
MAX_REQUESTS = 8192       # STT_PLAN_MAX_REQUESTS
PLAN_OK, PLAN_NO_BLOCKS, PLAN_TOO_LONG, PLAN_TOO_MANY_ROWS, PLAN_BAD_STATE = range(5)

Plan = collections.namedtuple("Plan", ["starts", "slots", "positions", "held", "ring", "status"])

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}


class TreeAttentionArgs(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in ("d_q", "d_k", "d_v")] + \
        [(k, C.c_int64) for k in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")] + \
        [(k, C.c_void_p) for k in ("d_k_cache", "d_v_cache")] + \
        [(k, C.c_int64) for k in ("block_stride", "head_stride", "pos_stride")] + \
        [(k, C.c_void_p) for k in ("d_table", "d_cached", "d_starts", "d_slots", "d_parents", "d_out")] + \
        [(k, C.c_int64) for k in ("out_row", "out_head")] + [("scale", C.c_float)] + \
        [(k, C.c_int32) for k in ("dtype", "n_seq", "rows", "n_heads", "n_kv_heads", "head_dim", "n_blocks",
                                  "block_size", "width", "max_nodes", "max_cached")]


# the same layout as bytes: packing them takes the host a quarter of the time of filling the structure
_PACKED = struct.Struct("@3P6q2P3q6P2qf11i")
assert _PACKED.size == C.sizeof(TreeAttentionArgs)


def _whole(name, t, dtype, shape):
    """`t` must be a contiguous tensor of this type and shape (None: any size)."""
    if t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return
    if t.dtype != dtype or t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError("%s must be %s %s, got %s %s" % (
            name, dtype, ["any" if s is None else s for s in shape], t.dtype, list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


def _one_gpu(first, *rest):
    """The common device of the tensors (None entries are skipped)."""
    dev = first.device
    if not first.is_cuda:
        raise ValueError("tensors must be on a GPU, got %s" % dev)
    for t in rest:
        if t is not None and t.device != dev:
            raise ValueError("tensors on %s and %s" % (dev, t.device))
    return dev


def _power_of_two(name, v):
    if v < 1 or v & (v - 1) or v > 65536:
        raise ValueError("%s must be a power of two up to 65536, got %d" % (name, v))


def plan(cached, new, table, held, free, ring, *, block_size, rows):
    """One step's block tables and slot map, built on the GPU.

    cached, new, held: int32 [n], positions in the cache, tokens about to be added, blocks held by each
    of the requests; table int32 [n, width], the blocks a request holds in its row's first entries;
    free int32 [n_ring] and ring int64 [2]: the free block ids are entries ring[0] .. ring[1] - 1 of
    `free`, modulo its length.  `rows`: capacity of the per-token outputs.

    Missing blocks are taken from the ring in request order, surplus ones (a request that has ended has
    both lengths 0) go back to its end.  `table` and `free` are updated in place, `held` and `ring` are
    left alone: the returned ones replace them.  Returns Plan(starts int32 [n + 1], slots int64 [rows],
    positions int32 [rows], held, ring, status int32 [1]).  status 0 means done; otherwise
    (PLAN_NO_BLOCKS, PLAN_TOO_LONG, PLAN_TOO_MANY_ROWS, PLAN_BAD_STATE) nothing has changed and every
    row is -1.  It stays on the device: reading it waits for the step."""
    n = cached.shape[0] if cached.dim() == 1 else -1
    if not 1 <= n <= MAX_REQUESTS:
        raise ValueError("1 to %d requests, got lengths %s" % (MAX_REQUESTS, list(cached.shape)))
    block_size, rows = int(block_size), int(rows)
    _power_of_two("block_size", block_size)
    if not 0 <= rows < 2 ** 31:
        raise ValueError("rows must be 0 to 2^31 - 1, got %d" % rows)
    _whole("cached", cached, torch.int32, (n,))
    _whole("new", new, torch.int32, (n,))
    _whole("held", held, torch.int32, (n,))
    _whole("table", table, torch.int32, (n, None))
    _whole("free", free, torch.int32, (None,))
    _whole("ring", ring, torch.int64, (2,))
    width, n_ring = table.shape[1], free.shape[0]
    if width < 1 or not 1 <= n_ring < 2 ** 31 or width * block_size > 2 ** 31 - 1:
        raise ValueError("table of %d blocks of %d positions, ring of %d" % (width, block_size, n_ring))
    dev = _one_gpu(cached, new, held, table, free, ring)
    lib = _library()
    with _lib.on(dev):
        # one allocation for the outputs, longs first: a view costs the host less than an allocation
        words = (2 * n + 3 + rows) // 2
        ring_out, slots, ints = torch.split_with_sizes(
            torch.empty(2 + rows + words, dtype=torch.int64, device=dev), (2, rows, words))
        sizes = (n, n + 1, 1, rows) if rows & 1 == 0 else (n, n + 1, 1, rows, 1)
        held_out, starts, status, positions = torch.split_with_sizes(ints.view(torch.int32), sizes)[:4]
        _lib.check(lib.stt_paged_plan(
            cached.data_ptr(), new.data_ptr(), n, block_size, table.data_ptr(), width, free.data_ptr(), n_ring,
            ring.data_ptr(), ring_out.data_ptr(), held.data_ptr(), held_out.data_ptr(), rows, starts.data_ptr(),
            slots.data_ptr(), positions.data_ptr(), status.data_ptr(), _lib.stream(dev)))
    return Plan(starts, slots, positions, held_out, ring_out, status)


def _rows_of(name, t, dtype, shape):
    """`t` must be of this type and shape, its rows and heads 16-byte aligned; returns their strides."""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError("%s must be %s %s, got %s %s" % (name, dtype, list(shape), t.dtype, list(t.shape)))
    row, head, last = t.stride()
    if (last != 1 or (row | head) % 8 or t.data_ptr() % 16) and t.numel():
        raise ValueError("%s: the last dimension must be contiguous, rows and heads 16-byte aligned (strides %s)" % (
            name, t.stride()))
    return row, head


def _apart(name, t):
    """What is written must not share memory with itself (an expanded tensor, overlapping windows)."""
    if t.is_contiguous():
        return
    end = t.shape[-1]
    for stride, size in sorted(zip(t.stride()[:-1], t.shape[:-1])):
        if size > 1:
            if stride < end:
                raise ValueError("%s: elements overlap (strides %s)" % (name, t.stride()))
            end += stride * (size - 1)


def tree_attention(q, k, v, k_cache, v_cache, table, cached, starts, slots, parents=None, *, max_nodes, max_cached=0,
                   scale=None, out=None):
    """Attention of the new tokens of every sequence over its cached positions and its drafted tree, and
    the store of their K/V into the cache, in one call.

    q [rows, n_heads, d], k, v [rows, n_kv_heads, d] (bfloat16 or float16, d 64 or 128): the new
    tokens of all sequences; sequence i owns rows starts[i] .. starts[i + 1] - 1, the nodes of its tree,
    at most `max_nodes` (<= 64) of them.  parents int32 [rows]: a node's parent, an earlier node of its
    tree, or -1 for a root; None: every token follows the one before it.  A node sees the sequence's
    cached positions, its ancestors and itself.

    k_cache, v_cache [n_blocks, n_kv_heads, block_size, d] (any strides that keep d contiguous, 16-byte
    alignment and elements apart, the same for both); table int32 [n, width], cached int32 [n], starts int32 [n + 1], slots
    int64 [rows] as `plan` makes them; row r's K/V go to slots[r] unless that is negative.
    `max_cached`: the largest entry of `cached` if the host knows it; it decides how the work is split
    and nothing else.  scale: 1 / sqrt(d) unless given.

    Returns out [rows, n_heads, d] (a given `out` must not overlap the other tensors); rows that belong to no
    sequence are left as they are."""
    if q.dim() != 3 or q.dtype not in _DTYPES:
        raise ValueError("q must be bfloat16 or float16 [rows, heads, dim], got %s %s" % (q.dtype, list(q.shape)))
    rows, heads, dim = q.shape
    if dim not in (64, 128):
        raise ValueError("head size %d: 64 or 128" % dim)
    if k_cache.dim() != 4 or k_cache.dtype != q.dtype or k_cache.shape[3] != dim:
        raise ValueError("k_cache must be %s [blocks, kv heads, block size, %d], got %s %s" % (
            q.dtype, dim, k_cache.dtype, list(k_cache.shape)))
    n_blocks, kv_heads, block_size, _ = k_cache.shape
    strides = k_cache.stride()
    if n_blocks >= 2 ** 31:
        raise ValueError("cache of %d blocks" % n_blocks)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("%d heads over %d KV heads" % (heads, kv_heads))
    _power_of_two("block size", block_size)
    if v_cache.dtype != q.dtype or v_cache.shape != k_cache.shape or v_cache.stride() != strides:
        raise ValueError("v_cache must be laid out like k_cache")
    bs, hs, ps, ds = strides
    if (ds != 1 or (bs | hs | ps) % 8 or (k_cache.data_ptr() | v_cache.data_ptr()) % 16) and k_cache.numel():
        raise ValueError("cache: the last dimension must be contiguous, positions 16-byte aligned (strides %s)" % (strides,))
    _apart("cache", k_cache)
    max_nodes, max_cached = int(max_nodes), min(max(int(max_cached), 0), 2 ** 31 - 1)
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError("max_nodes must be 1 to %d, got %d" % (MAX_NODES, max_nodes))
    dtype = q.dtype
    q_row, q_head = _rows_of("q", q, dtype, (rows, heads, dim))
    k_row, k_head = _rows_of("k", k, dtype, (rows, kv_heads, dim))
    v_row, v_head = _rows_of("v", v, dtype, (rows, kv_heads, dim))
    n, width = table.shape if table.dim() == 2 else (-1, -1)
    _whole("table", table, torch.int32, (n, width))
    _whole("cached", cached, torch.int32, (n,))
    _whole("starts", starts, torch.int32, (n + 1,))
    _whole("slots", slots, torch.int64, (rows,))
    if parents is not None:
        _whole("parents", parents, torch.int32, (rows,))
    if out is not None:
        _rows_of("out", out, dtype, (rows, heads, dim))
        _apart("out", out)
    dev = _one_gpu(q, k, v, k_cache, v_cache, table, cached, starts, slots, parents, out)
    lib = _library()
    with _lib.on(dev):
        if out is None:
            out = torch.empty((rows, heads, dim), dtype=dtype, device=dev)
            out_row, out_head = heads * dim, dim
        else:
            out_row, out_head, _ = out.stride()
        a = _PACKED.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q_row, q_head, k_row, k_head, v_row, v_head,
            k_cache.data_ptr(), v_cache.data_ptr(), bs, hs, ps, table.data_ptr(), cached.data_ptr(), starts.data_ptr(),
            slots.data_ptr(), parents.data_ptr() if parents is not None else 0, out.data_ptr(), out_row, out_head,
            dim ** -0.5 if scale is None else float(scale), _DTYPES[dtype], n, rows, heads, kv_heads, dim, n_blocks, block_size,
            width, max_nodes, max_cached)
        need = lib.stt_tree_attention_workspace_bytes(a)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.stt_tree_attention(a, work.data_ptr() if need else None, need, _lib.stream(dev)))
    return out


SYMBOLS = ("stt_paged_plan", "stt_tree_attention", "stt_tree_attention_workspace_bytes")
_declared = False


def _library():
    global _declared
    lib = _lib.load()
    if not _declared:
        vp, i32 = C.c_void_p, C.c_int
        lib.stt_paged_plan.restype = i32
        lib.stt_paged_plan.argtypes = [vp, vp, i32, i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, vp, vp, vp, vp]
        lib.stt_tree_attention.restype = i32
        lib.stt_tree_attention.argtypes = [vp, vp, C.c_size_t, vp]
        lib.stt_tree_attention_workspace_bytes.restype = C.c_size_t
        lib.stt_tree_attention_workspace_bytes.argtypes = [vp]
        _declared = True
    return lib
